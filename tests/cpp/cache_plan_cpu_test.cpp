// The plans of the attention over a cache with a length for each sequence
// (csrc/kernels/dispatch.hpp): a workspace sized for the cache's length holds the
// slices of every shorter one, slices are whole tiles and few enough to merge,
// and a call that may not cut its keys does not; and the kernels' divisions.
#include "../../qwen3-runtime-byyourself_amd/csrc/kernels/dispatch.hpp"
#include "test_util.hpp"

#include <string>

using test::require;

namespace
{
    // x / d by the kernels' multiplication, at and around multiples of d up to 2^31 - 1.
    void divisions()
    {
        using namespace q3k;
        for (int64_t d = 1; d <= INT32_MAX; d += d < 3000 ? 1 : d / 7)
            for (const int64_t by : {d - 1, d, d + 1})
            {
                if (by < 1 || by > INT32_MAX)
                    continue;
                const Divisor v = divisor(by);
                for (int64_t q = 0; q * by <= INT32_MAX; q += 1 + q / 5)
                    for (const int64_t x : {q * by - 1, q * by, q * by + 1, q * by + by / 2})
                        if (x >= 0 && x <= INT32_MAX)
                            require(static_cast<int32_t>(x) / v == x / by && static_cast<int32_t>(x) % v == x % by,
                                    std::to_string(x) + " / " + std::to_string(by));
                require(INT32_MAX / v == INT32_MAX / by, "2^31 - 1 / " + std::to_string(by));
            }
    }

    void body()
    {
        using namespace q3k;
        divisions();
        const int32_t heads[][2] = {{16, 8}, {32, 8}, {40, 8}, {64, 8}, {2, 1}, {4, 1}, {5, 1}, {8, 1}, {32, 1}};
        int64_t cut = 0, whole = 0, waves[9] = {};
        for (const auto &h : heads)
            for (const int64_t B : {1, 2, 5, 16, 40, 64, 200, 3000})
                for (const int64_t S : {1, 2, 7, 33, 100, 256, 1000})
                {
                    int64_t before = 0;
                    for (int64_t cached = 1; cached <= 40000; cached += cached / 24 + 1)
                    {
                        const int64_t bytes = cache_attention_workspace_bytes(B, S, h[0], h[1], cached);
                        require(bytes >= before, "less workspace than for a shorter cache");
                        before = bytes;
                        for (int form = 0; form < 8; ++form)
                        {
                            const bool e4m3 = (form & 1) != 0, tree = (form & 2) != 0, ragged = (form & 4) != 0;
                            const std::string what = std::to_string(h[0]) + "/" + std::to_string(h[1]) + " heads, B " +
                                                     std::to_string(B) + ", S " + std::to_string(S) + ", " +
                                                     std::to_string(cached) + " rows, form " + std::to_string(form);
                            const CacheAttnPlan p = plan_cache_attention(B, S, h[0], h[1], cached, e4m3, tree, ragged, true);
                            const bool decode = S * (h[0] / h[1]) <= kAttColsPerWave;
                            require((p.decode_waves > 0) == decode, what + ": kernel");
                            require(!decode || p.decode_waves == 1 || p.decode_waves == 4 || (e4m3 && p.decode_waves == 8),
                                    what + ": a block of waves that is not built");
                            require(decode || p.key_groups == 1 || p.key_groups == 4, what + ": key groups that are not built");
                            waves[decode ? p.decode_waves : 0] += 1;
                            require((p.splits > 1) == (p.bytes > 0), what + ": a size without slices, or slices without");
                            require(p.bytes <= bytes, what + ": the slices need more than the workspace");
                            require(p.bytes == 0 || p.bytes == p.splits * B * S * h[0] * (kAttHeadDim + 2) * 4, what + ": size");
                            require(p.splits <= kAttMaxSplits, what + ": more slices than the merge holds");
                            if (p.splits > 1)
                            {
                                require(p.split_keys % (decode ? kCacheDecodeTile : kCacheBlockTile) == 0, what + ": half a tile");
                                const int64_t rows = decode || cached > S ? cached : S;
                                require(static_cast<int64_t>(p.splits) * p.split_keys >= rows &&
                                            static_cast<int64_t>(p.splits - 1) * p.split_keys < rows,
                                        what + ": slices do not cover the rows");
                            }
                            (p.splits > 1 ? cut : whole) += 1;
                            const CacheAttnPlan q = plan_cache_attention(B, S, h[0], h[1], cached, e4m3, tree, ragged, false);
                            require(q.splits == 1 && q.bytes == 0, what + ": cut without a workspace");
                        }
                    }
                }
        require(cut > 10000 && whole > 10000, "the shapes cover whole and cut keys");
        require(waves[1] > 0 && waves[4] > 0 && waves[8] > 0 && waves[0] > 0, "the shapes cover every kernel");
    }
} // namespace

int main() { return test::run("cache attention plan test", body); }
