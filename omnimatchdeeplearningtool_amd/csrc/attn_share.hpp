// attn_share.hpp — how many workgroups share a walk of the attention kernels for
// training (host code, no device needed).
#pragma once

#include <algorithm>

namespace omhip {

// Workgroups that share a block's walk of `tiles` 64-row tiles: as many as make `room` of them in all and no more (one
// workgroup past what the CUs hold starts a second round: 1 x 2048 x 5 heads of 128 causal backward 75.3 us, rounded up 89.4),
// of four tiles at least. So a grid that fills the room is not shared, which bounds the parts' fp32 sums of every row
// and what the launches of their workgroups and of their join start. Room is
//  * two workgroups a CU, the long walk of one block and the short one of another, which make a causal grid even; dK / dV of
//    head dimensions up to 64 hold two workgroups a CU at once and ask for four. (2 x 4096 x 16 heads on 4 of 128 backward
//    499 us with two a CU, 516 with four, about 730 unshared.)
//  * in a window, whose walks are alike, what the CUs hold at once. Backward, causal, us:
//                                                            unshared   2    3    4    8
//      1 x 8192, 8 heads on 2 of 128, window 1024, 128 blocks   188   148  175  162  188    (2 fill the room)
//      1 x 4096, 4 heads of 32, window 1024, 128 blocks          40    35   35   35   41    (4)
//      2 x 4160, 16 heads on 4 of 128, window 1024, 264 blocks  249   277  289  302  365    (1)
//      2 x 6144, the same, 384 blocks                           430   418  438  453  549    (1)
//      4 x 8320, 32 heads on 8 of 128, window 2048, 2080 blocks 3563 3759 3859 3980 4578    (1; 2 keep 545 MB of sums)
inline int walkParts(long long blocks, int tiles, long long room) {
    if (blocks == 0 || tiles == 0) return 1;
    return (int)std::clamp<long long>(room / blocks, 1, std::max(1, tiles / 4));
}

}  // namespace omhip
