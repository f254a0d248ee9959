// CPU test of omhip::evenParts, the number of workgroups that share a walk of the windowed attention's dK and dV: no choice,
// over grids from one block of 128 keys to as many as a call may have, starts more threads in a launch than it takes (512
// for a workgroup of the walk, one for 8 values of a key in the join of the parts).
// Exit status 0 = all checks passed.
#include <cstdio>

#include "../../omnimatchdeeplearningtool_amd/csrc/attn_share.hpp"

static int g_fail = 0;

static void check(long long blocks, int tiles, long long room) {
    const int parts = omhip::evenParts(blocks, tiles, room);
    const long long most = 0xffffffffLL, walk = blocks * parts * 512, join = parts > 1 ? blocks * 128 * (128 / 8) : 0;
    if (parts < 1 || parts > 16 || walk > most || join > most) {
        std::printf("FAIL blocks %lld tiles %d room %lld: %d parts, %lld threads, %lld of the join\n", blocks, tiles, room, parts, walk,
                    join);
        ++g_fail;
    }
}

int main() {
    // 128 heads on 2 of 8, 65600 queries in a window of 65600 over 2^28 + 128 keys: 2^21 + 1 blocks of either key head
    check(2 * ((1LL << 21) + 1), 1025 * 64, 512);
    constexpr long long kMostBlocks = 0xffffffffLL / 512;   // of a call
    for (long long room : {1LL, 256LL, 304LL, 512LL, 608LL})
        for (long long blocks = 1; blocks <= kMostBlocks; blocks += 1 + blocks / 7)
            for (int tiles : {0, 1, 3, 4, 7, 8, 9, 16, 33, 64, 257, 1000, 4099, 65600, 1 << 20, 1 << 28}) {
                check(blocks, tiles, room);
                check(std::min(kMostBlocks, (blocks + room - 1) / room * room + 1), tiles, room);   // one past whole rounds
            }
    check(kMostBlocks, 1 << 28, 512);
    if (g_fail == 0) std::printf("ALL PASSED\n");
    return g_fail ? 1 : 0;
}
