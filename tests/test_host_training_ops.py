"""The C++ class offers the attention block's training operators (no GPU needed)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include "omhip_backend.hpp"
using om::HIPBackend;
void step(const uint16_t* qkv, uint16_t* ctx, float* lse, const uint16_t* dctx, uint16_t* dqkv, const int* lens, const void* x,
          void* y, float* f, const uint64_t* rng) {
    const long long ld = 3 * 64;
    HIPBackend::groupNormNhwc(0, x, f, f, y, f, f, 2, 49, 64, 8, 1e-5f, 2);
    HIPBackend::attentionTrainForwardHalf(0, qkv, qkv + 64, qkv + 128, ld, 50 * ld, ld, 50 * ld, lens, lens, true, ctx, lse, 2, 50,
                                          50, 1, 1, 64, 0.125f);
    HIPBackend::dropout(0, x, f, x, y, 100, 64, 0.1f, rng, 0);
    HIPBackend::dropoutBackward(0, x, y, f, 100, 64, 0.1f, rng, 0);
    HIPBackend::attentionBackwardHalf(0, qkv, qkv + 64, qkv + 128, ld, 50 * ld, ld, 50 * ld, lens, lens, true, ctx, lse, dctx,
                                      dqkv, dqkv + 64, dqkv + 128, 2, 50, 50, 1, 1, 64, 0.125f);
    HIPBackend::groupNormNhwcBackward(0, x, x, nullptr, f, f, f, f, y, f, f, 2, 49, 64, 8, 2);
}
"""


def test_cpp_class_compiles(tmp_path):
    src = tmp_path / "step.cpp"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++23", "-Wall", "-Werror", f"-I{ROOT}/include", "-c", str(src), "-o", str(tmp_path / "step.o")],
                   check=True)
