"""The C++ tests of the 8-bit KV cache, tree attention and their plans (tests/cpp/), built by build()."""
import pytest

from test_cpp import _run


def test_cache_plans():
    _run("cache_plan_cpu_test")


@pytest.mark.gpu
def test_quantized_kv_cache():
    _run("quantized_kv_cache_gpu_test", timeout=300)
