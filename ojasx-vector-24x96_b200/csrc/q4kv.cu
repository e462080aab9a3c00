// 4-bit paged KV cache: appending with the position rotation on the way, and reading back.  Layout and format: q4kv.cuh; attention of
// single tokens: q4kv_decode.cu.
#include <cmath>

#include "handles.h"
#include "launch.h"
#include "packed.cuh"
#include "q4kv.cuh"
#include "../../include/ojasx_lut_b200.h"

namespace ojx {

__device__ __forceinline__ float4 q4_load4(const void* p, size_t i, bool bf16) {
    if (!bf16) return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
    const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(p) + i);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
}
__device__ __forceinline__ void q4_store4(void* p, size_t i, bool bf16, float4 v) {
    if (!bf16) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = v;
        return;
    }
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p) + i) =
        make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}

// Four values of a group whose other 28 are with the neighbouring seven lanes, as nibbles; `meta`: the group's minimum and scale.
__device__ __forceinline__ unsigned q4_encode(float4 x, unsigned& meta) {
    float lo = fminf(fminf(x.x, x.y), fminf(x.z, x.w)), hi = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
    float odd = (x.x - x.x) + (x.y - x.y) + (x.z - x.z) + (x.w - x.w);   // NaN for an infinity or a NaN (which the maxima pass over)
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
        odd += __shfl_xor_sync(0xffffffffu, odd, off);
    }
    const __nv_bfloat16 mb = __float2bfloat16_rd(lo);
    const float m = __bfloat162float(mb);
    const float range = hi - m;
    const bool wide = isinf(range);   // beyond fp32: quotients first, then their difference
    const __nv_bfloat16 sb = __float2bfloat16_ru(wide ? hi / 15.0f - m / 15.0f : __fdiv_rn(range, 15.0f));
    const float s = __bfloat162float(sb);
    if (!(odd == 0.0f) || isinf(m) || isinf(s)) {
        meta = 0x7fff0000u;
        return 0u;
    }
    meta = (unsigned)__bfloat16_as_ushort(mb) << 16 | __bfloat16_as_ushort(sb);
    const float d = s > 0.0f ? s : 1.0f;   // a group of one value that bf16 holds has no steps
    auto code = [&](float v) { return (unsigned)fminf(fmaxf(rintf(wide ? v / d - m / d : __fdiv_rn(v - m, d)), 0.0f), 15.0f); };
    return code(x.x) | code(x.y) << 4 | code(x.z) << 8 | code(x.w) << 12;
}

struct Q4AppendProblem {
    Q4Cache cache;
    const void *k, *v, *q;      // [n_tokens][heads][head_dim] with row strides in elements
    void* q_out;                // [n_tokens][q_heads][head_dim]
    long long k_stride, v_stride, q_stride;
    const int* positions;       // [batch] tokens that are cached already
    const int* ends;            // [batch + 1] or null: token i is one of sequence i
    const double* turns;        // [head_dim / 2] turns per position, or null: no rotation
    int n_tokens, batch, q_heads;
};

// cos and sin of four angles, given in turns: whole turns are dropped in 64 bits, where a position of 2^31 is still exact to 2^-22.
__device__ __forceinline__ void q4_angles(const double* turns, int j, int pos, float (&c)[4], float (&s)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double t = (double)pos * turns[j + i];
        sincospif(2.0f * (float)(t - rint(t)), &s[i], &c[i]);
    }
}

// One token per CTA; HD / 8 lanes share a vector, each with four dimensions of either half (a rotated pair is in one lane, a group
// is eight lanes).  Keys and queries are turned by position * turns[j], keys and values go to the cache as 4 bits.
template <int HD, bool kBf16>
__global__ void __launch_bounds__(128) q4_append_kernel(const __grid_constant__ Q4AppendProblem P) {
    constexpr int L = HD / 8, G = HD / 32;
    using T = Q4Layout<HD>;
    chain_begin();
    const int token = blockIdx.x, l = threadIdx.x % L, task0 = threadIdx.x / L, step = 128 / L;
    int b = token, pos;
    if (P.ends) {
        b = packed_owner(P.ends, P.batch, token);
        if (b < 0) return;
        pos = P.positions[b] + token - P.ends[b];
    } else {
        pos = P.positions[b];
    }
    float c[4] = {1.0f, 1.0f, 1.0f, 1.0f}, s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (P.turns) q4_angles(P.turns, 4 * l, pos, c, s);
    const int kv = P.cache.kv_heads, tasks = 2 * kv + (P.q ? P.q_heads : 0);
    const int rounds = (tasks + step - 1) / step;
    for (int r = 0; r < rounds; ++r) {
        const int task = min(r * step + task0, tasks - 1);      // (the lanes of a warp stay together for the shuffles)
        const bool live = r * step + task0 < tasks;
        const int kind = task < kv ? 0 : task < 2 * kv ? 1 : 2, head = kind == 2 ? task - 2 * kv : task - kind * kv;
        const void* src = kind == 0 ? P.k : kind == 1 ? P.v : P.q;
        const long long stride = kind == 0 ? P.k_stride : kind == 1 ? P.v_stride : P.q_stride;
        const size_t at = (size_t)token * stride + (size_t)head * HD + 4 * l;
        float4 a = q4_load4(src, at, kBf16), d = q4_load4(src, at + HD / 2, kBf16);
        if (kind != 1 && P.turns) {
            const float4 x = a, y = d;
            a = make_float4(x.x * c[0] - y.x * s[0], x.y * c[1] - y.y * s[1], x.z * c[2] - y.z * s[2], x.w * c[3] - y.w * s[3]);
            d = make_float4(y.x * c[0] + x.x * s[0], y.y * c[1] + x.y * s[1], y.z * c[2] + x.z * s[2], y.w * c[3] + x.w * s[3]);
        }
        unsigned meta[2];
        const unsigned code[2] = {q4_encode(a, meta[0]), q4_encode(d, meta[1])};
        if (!live) continue;
        if (kind == 2) {
            const size_t to = ((size_t)token * P.q_heads + head) * HD + 4 * l;
            q4_store4(P.q_out, to, kBf16, a);
            q4_store4(P.q_out, to + HD / 2, kBf16, d);
            continue;
        }
        uint8_t* tile = q4_tile<HD>(P.cache, b, head, pos);
        if (!tile) {
            if (l == 0) atomicExch(P.cache.status, 1);
            continue;
        }
        const int in = pos % kQ4Tile;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int g = h * (G / 2) + l / 8;
            *reinterpret_cast<unsigned short*>(tile + (kind ? T::value_at(in, g, l % 8) : T::key_at(in, g, l % 8))) = (unsigned short)code[h];
            if (l % 8 == 0) *reinterpret_cast<unsigned*>(tile + (kind ? T::value_meta : T::key_meta) + T::meta_at(in, g)) = meta[h];
        }
    }
}

struct Q4ReadProblem {
    Q4Cache cache;
    void *k, *v;                // [n_tokens][kv_heads][head_dim]
    const int *ends, *positions;   // positions null: from the first token
    int n_tokens, batch;
};

// One token per CTA, a lane per four dimensions.  Tokens without a page are read as zeros.
template <int HD, bool kBf16>
__global__ void __launch_bounds__(128) q4_read_kernel(const __grid_constant__ Q4ReadProblem P) {
    using T = Q4Layout<HD>;
    chain_begin();
    const int token = blockIdx.x, b = packed_owner(P.ends, P.batch, token), kv = P.cache.kv_heads;
    if (b < 0) return;
    const int pos = (P.positions ? P.positions[b] : 0) + token - P.ends[b], in = pos & (kQ4Tile - 1);
    for (int i = threadIdx.x; i < 2 * kv * (HD / 4); i += 128) {
        const int which = i / (kv * (HD / 4)), rem = i - which * kv * (HD / 4), head = rem / (HD / 4), d4 = rem % (HD / 4), g = d4 >> 3;
        const uint8_t* tile = q4_tile<HD>(P.cache, b, head, pos);
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (tile) {
            const unsigned w = *reinterpret_cast<const unsigned short*>(tile + (which ? T::value_at(in, g, d4 & 7) : T::key_at(in, g, d4 & 7)));
            const unsigned meta = *reinterpret_cast<const unsigned*>(tile + (which ? T::value_meta : T::key_meta) + T::meta_at(in, g));
            const float s = q4_scale(meta), m = q4_min(meta);
            x = make_float4(fmaf((float)(w & 15), s, m), fmaf((float)(w >> 4 & 15), s, m), fmaf((float)(w >> 8 & 15), s, m), fmaf((float)(w >> 12), s, m));
        } else {
            atomicExch(P.cache.status, 1);
        }
        q4_store4(which ? P.v : P.k, ((size_t)token * kv + head) * HD + d4 * 4, kBf16, x);
    }
}

}  // namespace ojx

using namespace ojx;

extern "C" {

size_t ojasx_b200_q4kv_page_bytes(int kv_heads, int page_size, int head_dim) {
    if (kv_heads <= 0 || page_size <= 0 || page_size % kQ4Tile || (head_dim != 64 && head_dim != 128)) return 0;
    return (size_t)kv_heads * (page_size / kQ4Tile) * (head_dim == 64 ? Q4Layout<64>::bytes : Q4Layout<128>::bytes);
}

int ojasx_b200_q4kv_append(const void* d_k, long long k_stride, const void* d_v, long long v_stride, const void* d_q, long long q_stride,
                           void* d_q_out, void* d_pool, const int* d_block_table, const int* d_positions, const int* d_ends,
                           const double* d_turns, int* d_status, int n_tokens, int batch, int max_pages, int num_pages, int page_size,
                           int kv_heads, int q_heads, int head_dim, int io_dtype, void* stream) {
    const int rc = q4_check(d_pool, d_block_table, max_pages, num_pages, page_size, kv_heads, head_dim, batch, io_dtype, d_status);
    if (rc != OJX_OK) return rc;
    if (!d_k || !d_v || !d_positions || n_tokens < 0 || (d_q && (!d_q_out || q_heads <= 0)) || (!d_ends && n_tokens != batch)) return OJX_ERR_ARG;
    if (!q4_aligned(d_k) || !q4_aligned(d_v) || !q4_aligned(d_q) || !q4_aligned(d_q_out) || k_stride % 4 || v_stride % 4 || q_stride % 4) return OJX_ERR_ARG;
    if (n_tokens == 0) return OJX_OK;
    Q4AppendProblem P{};
    P.cache = {static_cast<uint8_t*>(d_pool), d_block_table, d_status, max_pages, num_pages, page_size, kv_heads};
    P.k = d_k; P.v = d_v; P.q = d_q; P.q_out = d_q_out; P.k_stride = k_stride; P.v_stride = v_stride; P.q_stride = q_stride;
    P.positions = d_positions; P.ends = d_ends; P.turns = d_turns; P.n_tokens = n_tokens; P.batch = batch; P.q_heads = q_heads;
    const bool bf = io_dtype == OJX_BF16;
    auto kernel = head_dim == 64 ? (bf ? q4_append_kernel<64, true> : q4_append_kernel<64, false>)
                                 : (bf ? q4_append_kernel<128, true> : q4_append_kernel<128, false>);
    OJX_CUDA_TRY(launch_chained(kernel, n_tokens, 128, 0, static_cast<cudaStream_t>(stream), P));
    count_launch(1);
    return OJX_OK;
}

int ojasx_b200_q4kv_read(const void* d_pool, const int* d_block_table, const int* d_ends, const int* d_positions, void* d_k, void* d_v,
                         int* d_status, int n_tokens, int batch, int max_pages, int num_pages, int page_size, int kv_heads, int head_dim,
                         int io_dtype, void* stream) {
    const int rc = q4_check(d_pool, d_block_table, max_pages, num_pages, page_size, kv_heads, head_dim, batch, io_dtype, d_status);
    if (rc != OJX_OK) return rc;
    if (!d_ends || !d_k || !d_v || n_tokens < 0 || !q4_aligned(d_k) || !q4_aligned(d_v)) return OJX_ERR_ARG;
    if (n_tokens == 0) return OJX_OK;
    Q4ReadProblem P{};
    P.cache = {static_cast<uint8_t*>(const_cast<void*>(d_pool)), d_block_table, d_status, max_pages, num_pages, page_size, kv_heads};
    P.k = d_k; P.v = d_v; P.ends = d_ends; P.positions = d_positions; P.n_tokens = n_tokens; P.batch = batch;
    const bool bf = io_dtype == OJX_BF16;
    auto kernel = head_dim == 64 ? (bf ? q4_read_kernel<64, true> : q4_read_kernel<64, false>)
                                 : (bf ? q4_read_kernel<128, true> : q4_read_kernel<128, false>);
    OJX_CUDA_TRY(launch_chained(kernel, n_tokens, 128, 0, static_cast<cudaStream_t>(stream), P));
    count_launch(1);
    return OJX_OK;
}

}  // extern "C"
