"""What a launch gave up on reads as NaN: the rows that attention over prompts marks, and results of the 4-bit cache's decode that a part
without a sum of weights went into.  No wait runs out here: the marks and the joining are called for themselves."""
import os
import shutil
import subprocess

import pytest

pytestmark = pytest.mark.gpu
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ojasx-vector-24x96_b200", "csrc")

SOURCE = r"""
#include <cstdio>
#include <cmath>
#include <vector>
#include "packed.cuh"
#include "q4kv_decode.cu"
namespace ojx {
void count_launch(int) {}
int num_sms() { return 1; }
void set_last_error(const char*, cudaError_t) {}
}
using namespace ojx;
constexpr int kRows = 9, kHeads = 6, kHd = 64;
template <class T> __global__ void mark(T* out) { packed_give_up<kHd>(out, 2, 5, 2, 3, kHeads, threadIdx.x, blockDim.x); }
template <class T> int marks() {
    std::vector<T> h(kRows * kHeads * kHd, T(1.0f));
    T* d;
    cudaMalloc(&d, h.size() * sizeof(T));
    cudaMemcpy(d, h.data(), h.size() * sizeof(T), cudaMemcpyHostToDevice);
    mark<<<1, 256>>>(d);
    if (cudaMemcpy(h.data(), d, h.size() * sizeof(T), cudaMemcpyDeviceToHost) != cudaSuccess) return 1;
    for (int r = 0; r < kRows; ++r)
        for (int e = 0; e < kHeads * kHd; ++e) {
            const bool in = r >= 2 && r < 7 && e / kHd >= 2 && e / kHd < 5;
            if (std::isnan((float)h[r * kHeads * kHd + e]) != in) return 2;
        }
    return 0;
}
int joins() {   // one item of two query heads in two parts; the second part of head 1 gave up
    constexpr int row = kHd + 2;
    std::vector<float> parts(2 * 2 * kQdHeads * row, 0.0f);
    for (int c = 0; c < 2; ++c)
        for (int h = 0; h < 2; ++h) {
            float* p = parts.data() + ((c * 2 + (c == 0 ? 1 : 0)) * kQdHeads + h) * row;
            p[1] = c == 1 && h == 1 ? NAN : 2.0f;
            for (int d = 0; d < kHd; ++d) p[2 + d] = 6.0f;
        }
    const int2 pieces[2] = {make_int2(0, 1), make_int2(-1, 0)};
    Q4DecodeProblem P{};
    float* out;
    cudaMalloc(&P.partials, parts.size() * 4);
    cudaMalloc(&P.pieces, sizeof(pieces));
    cudaMalloc(&out, 2 * kHd * 4);
    cudaMemcpy(P.partials, parts.data(), parts.size() * 4, cudaMemcpyHostToDevice);
    cudaMemcpy(P.pieces, pieces, sizeof(pieces), cudaMemcpyHostToDevice);
    P.out = out;
    P.cache.kv_heads = P.blocks = P.batch = 1;
    P.q_heads = P.share = 2;
    q4_combine_kernel<kHd, false><<<2, kQcThreads>>>(P);
    float h[2 * kHd];
    if (cudaMemcpy(h, out, sizeof(h), cudaMemcpyDeviceToHost) != cudaSuccess) return 3;
    for (int d = 0; d < kHd; ++d) if (h[d] != 3.0f || !std::isnan(h[kHd + d])) return 4;
    return 0;
}
int main() {
    const int a = marks<float>(), b = marks<__nv_bfloat16>(), c = joins();
    printf("%d %d %d\n", a, b, c);
    return a || b || c;
}
"""


def test_results_that_were_given_up_are_nan(cuda, tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("needs nvcc")
    (tmp_path / "marks.cu").write_text(SOURCE)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr", "-I", CSRC, "-o", str(tmp_path / "marks"),
                    str(tmp_path / "marks.cu")], check=True, timeout=300)
    run = subprocess.run([str(tmp_path / "marks")], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout + run.stderr
