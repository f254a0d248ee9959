"""The C++ class offers the operators that tell an attention block where its tokens are (no GPU needed)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include "omhip_backend.hpp"
using om::HIPBackend;
void step(const uint16_t* qkv, uint16_t* turned, uint16_t* ctx, float* lse, const uint16_t* dctx, uint16_t* dturned, uint16_t* dqkv,
          const int* lens, const float* f, float* g, const int* at) {
    const long long ld = 3 * 64, im = 50 * ld;
    HIPBackend::qkNormRotary(0, qkv, qkv + 64, ld, im, ld, im, f, f, f, f, at, turned, turned + 64, ld, im, ld, im, 2, 50, 1, 1, 64, 64,
                             50, 1e-6f, false);
    HIPBackend::attentionWindowForwardHalf(0, turned, turned + 64, qkv + 128, ld, im, ld, im, lens, lens, true, 16, 1, ctx, lse, 2, 50,
                                           50, 1, 1, 64, 0.125f);
    HIPBackend::attentionWindowBackwardHalf(0, turned, turned + 64, qkv + 128, ld, im, ld, im, lens, lens, true, 16, 1, ctx, lse, dctx,
                                            dturned, dturned + 64, dqkv + 128, 2, 50, 50, 1, 1, 64, 0.125f);
    HIPBackend::attentionBiasForwardHalf(0, turned, turned + 64, qkv + 128, ld, im, ld, im, lens, lens, false, f, at, at, at, 9, 9, 4,
                                         ctx, lse, 2, 50, 50, 1, 1, 64, 0.125f);
    HIPBackend::attentionBiasBackwardHalf(0, turned, turned + 64, qkv + 128, ld, im, ld, im, lens, lens, false, f, at, at, at, 9, 9, 4,
                                          ctx, lse, dctx, dturned, dturned + 64, dqkv + 128, g, 2, 50, 50, 1, 1, 64, 0.125f);
    HIPBackend::qkNormRotaryBackward(0, dturned, dturned + 64, ld, im, ld, im, qkv, qkv + 64, ld, im, ld, im, f, f, f, f, at, dqkv,
                                     dqkv + 64, g, g, 2, 50, 1, 1, 64, 64, 50, 1e-6f, false);
}
"""


def test_cpp_class_compiles(tmp_path):
    src = tmp_path / "step.cpp"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++23", "-Wall", "-Werror", f"-I{ROOT}/include", "-c", str(src), "-o", str(tmp_path / "step.o")],
                   check=True)
