// Causal attention over whole prompts: packed sequences of different lengths, grouped query heads, softmax(q k^T * scale) v.
//
// The last query of a sequence sees its last key: with n queries and m keys query i sees the keys up to i + m - n, none where that is
// negative.  The rows of a tile are (position, query head of the KV head), so that the heads that share keys share their tiles too.
#include <algorithm>
#include <cmath>

#include "handles.h"
#include "launch.h"
#include "packed.cuh"
#include "../../include/ojasx_lut_b200.h"

namespace ojx {

struct PromptProblem {
    const void *q, *k, *v;
    void* out;                                     // [n_rows][q_heads][head_dim]
    long long q_row, q_head, k_row, k_head, v_row, v_head;   // strides in elements
    const int *ends, *key_ends;
    int batch, n_rows, n_keys, q_heads, kv_heads, share;
    float scale;
};

// fp32 tiles of 64 rows x 64 keys, sixteen threads to four rows, four keys of a thread.
template <int HD, bool kBf16>
__global__ void __launch_bounds__(256) prompt_tile_kernel(const __grid_constant__ PromptProblem P) {
    constexpr int R = 64, C = 64, W = HD + 4;
    extern __shared__ __align__(16) float sm[];
    float *qs = sm, *ks = qs + R * W, *vs = ks + C * W, *ps = vs + C * W;   // ps [R][C + 4]
    __shared__ int s_seq, s_part;
    chain_begin();
    const int per = R / P.share, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, head = blockIdx.y;
    if (tid < 32) {
        int seq = -1, part = 0;
        const bool in = packed_part(P.batch, blockIdx.x, [&](int b) { return (packed_range(P.ends, b, P.n_rows).count + per - 1) / per; }, seq, part);
        if (tid == 0) { s_seq = in ? seq : -1; s_part = part; }
    }
    __syncthreads();
    if (s_seq < 0) return;
    const PackedRange rows = packed_range(P.ends, s_seq, P.n_rows), keys = packed_range(P.key_ends, s_seq, P.n_keys);
    const int p0 = s_part * per, live = min(per, rows.count - p0) * P.share, ahead = keys.count - rows.count;
    auto load = [](const void* p, size_t i) { return kBf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]) : reinterpret_cast<const float*>(p)[i]; };
    for (int i = tid; i < R * HD; i += 256) {
        const int r = i / HD, d = i % HD;
        qs[r * W + d] = r < live ? load(P.q, (size_t)(rows.first + p0 + r / P.share) * P.q_row + (size_t)(head * P.share + r % P.share) * P.q_head + d) * P.scale : 0.0f;
    }
    float m[4], l[4], o[4][HD / 16];
    int last[4];   // last key that the row sees
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i;
        m[i] = -INFINITY; l[i] = 0.0f;
        last[i] = r < live ? p0 + r / P.share + ahead : -1;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) o[i][j] = 0.0f;
    }
    const int n = min(keys.count, p0 + (live - 1) / P.share + ahead + 1);
    for (int k0 = 0; k0 < n; k0 += C) {
        __syncthreads();
        for (int i = tid; i < C * HD; i += 256) {
            const int c = i / HD, d = i % HD;
            const bool in = k0 + c < n;
            ks[c * W + d] = in ? load(P.k, (size_t)(keys.first + k0 + c) * P.k_row + (size_t)head * P.k_head + d) : 0.0f;
            vs[c * W + d] = in ? load(P.v, (size_t)(keys.first + k0 + c) * P.v_row + (size_t)head * P.v_head + d) : 0.0f;
        }
        __syncthreads();
        float s[4][4] = {};
        for (int d = 0; d < HD; d += 4) {
            float4 a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = *reinterpret_cast<const float4*>(qs + (ty * 4 + i) * W + d);
                b[i] = *reinterpret_cast<const float4*>(ks + (tx + 16 * i) * W + d);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][j] = fmaf(a[i].x, b[j].x, fmaf(a[i].y, b[j].y, fmaf(a[i].z, b[j].z, fmaf(a[i].w, b[j].w, s[i][j]))));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (k0 + tx + 16 * j > last[i]) s[i][j] = -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int off = 8; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            const float base = top == -INFINITY ? 0.0f : top, keep = __expf(m[i] - base);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = __expf(s[i][j] - base);
                sum += p;
                ps[(ty * 4 + i) * (C + 4) + tx + 16 * j] = p;
            }
#pragma unroll
            for (int off = 8; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            l[i] = fmaf(l[i], keep, sum);
            m[i] = top;
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) o[i][j] *= keep;
        }
        __syncwarp();   // (a row's sixteen threads are in one warp)
        for (int c = 0; c < C; ++c) {
            float v[HD / 16];
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) v[j] = vs[c * W + tx + 16 * j];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = ps[(ty * 4 + i) * (C + 4) + c];
                if (k0 + c > last[i]) continue;   // (what a row does not see may be infinite)
#pragma unroll
                for (int j = 0; j < HD / 16; ++j) o[i][j] = fmaf(p, v[j], o[i][j]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i;
        if (r >= live) continue;
        const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
        const size_t to = ((size_t)(rows.first + p0 + r / P.share) * P.q_heads + head * P.share + r % P.share) * HD;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
            const float x = o[i][j] * inv;
            if (kBf16) reinterpret_cast<__nv_bfloat16*>(P.out)[to + tx + 16 * j] = __float2bfloat16_rn(x);
            else reinterpret_cast<float*>(P.out)[to + tx + 16 * j] = x;
        }
    }
}

template <int HD>
constexpr size_t prompt_tile_smem() { return sizeof(float) * (3 * 64 * (HD + 4) + 64 * 68); }

template <int HD, bool kBf16>
static int launch_prompt_tile(const PromptProblem& P, cudaStream_t s) {
    static std::atomic<bool> opted[64];
    constexpr size_t smem = prompt_tile_smem<HD>();
    OJX_CUDA_TRY(opt_in_smem(reinterpret_cast<const void*>(prompt_tile_kernel<HD, kBf16>), smem, opted));
    const int per = 64 / P.share;
    // as many tiles as the sequences can have: each has at most one that is not full
    const long long tiles = P.n_rows / per + std::min(P.batch, P.n_rows);
    if (tiles > 0x7fffffffLL) return OJX_ERR_TOO_LARGE;
    OJX_CUDA_TRY(launch_chained(prompt_tile_kernel<HD, kBf16>, dim3((unsigned)tiles, P.kv_heads), 256, smem, s, P));
    count_launch(1);
    return OJX_OK;
}

}  // namespace ojx

using namespace ojx;

extern "C" int ojasx_b200_prompt_attention(const void* d_q, long long q_row, long long q_head, const void* d_k, long long k_row,
                                           long long k_head, const void* d_v, long long v_row, long long v_head, void* d_out,
                                           const int* d_ends, const int* d_key_ends, int batch, int n_rows, int n_keys, int q_heads,
                                           int kv_heads, int head_dim, float scale, int io_dtype, void* stream) {
    if (!d_q || !d_k || !d_v || !d_out || !d_ends || !d_key_ends || batch <= 0 || n_rows < 0 || n_keys < 0 || kv_heads <= 0 || q_heads <= 0 ||
        q_heads % kv_heads)
        return OJX_ERR_ARG;
    if (io_dtype != OJX_F32 && io_dtype != OJX_BF16) return OJX_ERR_ARG;
    if ((head_dim != 64 && head_dim != 128) || q_heads / kv_heads > 64) return OJX_ERR_UNSUPPORTED;
    if (kv_heads > 65535) return OJX_ERR_TOO_LARGE;
    if (n_rows == 0) return OJX_OK;
    PromptProblem P{};
    P.q = d_q; P.k = d_k; P.v = d_v; P.out = d_out;
    P.q_row = q_row; P.q_head = q_head; P.k_row = k_row; P.k_head = k_head; P.v_row = v_row; P.v_head = v_head;
    P.ends = d_ends; P.key_ends = d_key_ends; P.batch = batch; P.n_rows = n_rows; P.n_keys = n_keys;
    P.q_heads = q_heads; P.kv_heads = kv_heads; P.share = q_heads / kv_heads;
    P.scale = scale > 0.0f ? scale : 1.0f / sqrtf((float)head_dim);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (io_dtype == OJX_BF16) return head_dim == 64 ? launch_prompt_tile<64, true>(P, s) : launch_prompt_tile<128, true>(P, s);
    return head_dim == 64 ? launch_prompt_tile<64, false>(P, s) : launch_prompt_tile<128, false>(P, s);
}
