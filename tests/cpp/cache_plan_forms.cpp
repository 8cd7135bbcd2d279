// Prints the plan of each call of the attention over a cache that standard input
// names, a line a call: "B S Hq Hkv cached e4m3 tree ragged can_split" gives
// "decode_waves key_groups splits merged_by_rows" (csrc/kernels/dispatch.hpp).
#include "../../qwen3-runtime-byyourself_amd/csrc/kernels/dispatch.hpp"

#include <iostream>

int main()
{
    int64_t B = 0, S = 0, cached = 0;
    int32_t Hq = 0, Hkv = 0;
    bool e4m3 = false, tree = false, ragged = false, can_split = false;
    while (std::cin >> B >> S >> Hq >> Hkv >> cached >> e4m3 >> tree >> ragged >> can_split)
    {
        const q3k::CacheAttnPlan p = q3k::plan_cache_attention(B, S, Hq, Hkv, cached, e4m3, tree, ragged, can_split);
        std::cout << p.decode_waves << ' ' << p.key_groups << ' ' << p.splits << ' ' << (B * S * Hq > q3k::kAttBlockMergeRows)
                  << '\n';
    }
    return 0;
}
