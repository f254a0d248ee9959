// attn_share.hpp — how many workgroups share a walk of the attention kernels for
// training, where all blocks' walks are alike (host code, no device needed).
#pragma once

#include <algorithm>

namespace omhip {

// Workgroups that share a block's walk of `tiles` 64-row tiles, all blocks' walks alike: those with which the last one ends
// first where `room` of them run at once. A walk's start and end are as long as four tiles, the join of parts as eight.
// No more than a launch takes, which drops the bits of its threads' number above 2^32 silently: 512 threads a workgroup, and
// in the join one for each 8 of a block's 128 x up to 128 values.
inline int evenParts(long long blocks, int tiles, long long room) {
    constexpr long long kMostThreads = 0xffffffffLL;
    int best = 1;
    long long least = 0;
    for (int parts = 1; parts <= std::min(16, std::max(1, tiles / 4)); ++parts) {
        if (parts > 1 && (blocks * parts * 512 > kMostThreads || blocks * (128 * 128 / 8) > kMostThreads)) break;
        const long long rounds = (blocks * parts + room - 1) / room;
        const long long time = rounds * ((tiles + parts - 1) / parts + 4) + (parts > 1 ? 8 : 0);
        if (parts == 1 || time < least) best = parts, least = time;
    }
    return best;
}

}  // namespace omhip
