// CPU test of omhip::walkParts, the number of workgroups that share a walk of the attention kernels for training: no choice,
// over grids from one block of 128 keys to as many as a call may have, starts more threads in a launch than it takes (512
// for a workgroup of the walk, one for 8 values of a key in the join of the parts), shares a grid past the room that it
// is given, or keeps more sums than that room's (dK and dV, 128 keys of 128 values in fp32, of each workgroup).
// Exit status 0 = all checks passed.
#include <cstdio>

#include "../../omnimatchdeeplearningtool_amd/csrc/attn_share.hpp"

static int g_fail = 0;

static void check(long long blocks, int tiles, long long room) {
    const int parts = omhip::walkParts(blocks, tiles, room);
    const long long most = 0xffffffffLL, walk = blocks * parts * 512, join = parts > 1 ? blocks * 128 * (128 / 8) : 0;
    const long long sums = parts > 1 ? blocks * parts * 128 * 128 * 8 : 0;
    if (parts < 1 || walk > most || join > most || (parts > 1 && blocks * parts > room) || parts > std::max(1, tiles / 4) ||
        sums > room * 128 * 128 * 8) {
        std::printf("FAIL blocks %lld tiles %d room %lld: %d parts, %lld threads, %lld of the join, %lld bytes of sums\n", blocks, tiles,
                    room, parts, walk, join, sums);
        ++g_fail;
    }
}

int main() {
    // 128 heads on 2 of 8, 65600 queries in a window of 65600 over 2^28 + 128 keys: 2^21 + 1 blocks of either key head
    check(2 * ((1LL << 21) + 1), 1025 * 64, 512);
    // 4 x 8320 tokens, 32 heads on 8 of 128, window 2048: grids of many rounds are not shared
    check(4 * 8 * 65, 35 * 4, 256);
    check(257 * 8, 67 * 4, 256);     // 1 x 32896, window 4096
    check(1025 * 8, 515 * 4, 256);   // 1 x 131200, window 32768
    if (omhip::walkParts(128, 76, 256) != 2 || omhip::walkParts(9, 44, 512) != 11 || omhip::walkParts(264, 76, 256) != 1) {
        std::printf("FAIL: grids below the room\n");
        ++g_fail;
    }
    constexpr long long kMostBlocks = 0xffffffffLL / 512;   // of a call
    for (long long room : {1LL, 256LL, 304LL, 512LL, 608LL, 1024LL})
        for (long long blocks = 1; blocks <= kMostBlocks; blocks += 1 + blocks / 7)
            for (int tiles : {0, 1, 3, 4, 7, 8, 9, 16, 33, 64, 257, 1000, 4099, 65600, 1 << 20, 1 << 28}) {
                check(blocks, tiles, room);
                check(std::min(kMostBlocks, (blocks + room - 1) / room * room + 1), tiles, room);   // one past whole rounds
            }
    check(kMostBlocks, 1 << 28, 512);
    if (g_fail == 0) std::printf("ALL PASSED\n");
    return g_fail ? 1 : 0;
}
