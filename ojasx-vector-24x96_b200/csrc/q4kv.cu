// 4-bit paged KV cache: appending with the position rotation on the way, and reading back.  Layout and format: q4kv.cuh; attention of
// single tokens: q4kv_decode.cu.
#include <algorithm>
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
__device__ __forceinline__ void q4_load8(const void* p, size_t i, bool bf16, float4& a, float4& b) {
    if (!bf16) {
        a = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i)[0];
        b = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i)[1];
        return;
    }
    const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p) + i);
    a = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
    b = make_float4(__uint_as_float(w.z << 16), __uint_as_float(w.z & 0xffff0000u), __uint_as_float(w.w << 16), __uint_as_float(w.w & 0xffff0000u));
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

// Minimum and maximum that a NaN makes NaN.
__device__ __forceinline__ float q4_less(float a, float b) {
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
    return a;
}
__device__ __forceinline__ float q4_more(float a, float b) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
    return a;
}

// Eight consecutive values of a group whose other 24 are with the lanes whose numbers differ in bits 1 and 2, as nibbles of a word;
// `meta`: the group's minimum and scale.
// Quotients are those of IEEE division: with the rounded reciprocal r of s, q = v r, and q + (v - q s) r is v / s rounded (Markstein's
// theorem) where nothing leaves the range of fp32, which the branch sees to.  v - minimum is not negative and at most 15 scales.
__device__ __forceinline__ unsigned q4_encode(const float (&x)[8], unsigned& meta) {
    float lo = q4_less(q4_less(q4_less(x[0], x[1]), q4_less(x[2], x[3])), q4_less(q4_less(x[4], x[5]), q4_less(x[6], x[7])));
    float hi = q4_more(q4_more(q4_more(x[0], x[1]), q4_more(x[2], x[3])), q4_more(q4_more(x[4], x[5]), q4_more(x[6], x[7])));
#pragma unroll
    for (int off = 2; off < 8; off <<= 1) {
        lo = q4_less(lo, __shfl_xor_sync(0xffffffffu, lo, off));
        hi = q4_more(hi, __shfl_xor_sync(0xffffffffu, hi, off));
    }
    const unsigned lb = __float_as_uint(lo), mb = (lb + ((unsigned)((int)lb >> 31) & 0xffffu)) & 0xffff0000u;   // down to bf16
    const float m = __uint_as_float(mb), range = hi - m;
    unsigned sb = (__float_as_uint(__fdiv_rn(range, 15.0f)) + 0xffffu) & 0xffff0000u;                          // up
    float s = __uint_as_float(sb);
    unsigned code = 0;
    if (s > 0x1p-90f && s < 0x1p90f) {
        const float r = __frcp_rn(s);
        // rounded by an addition, which leaves a code in the lowest bits; what is above them adds up to a constant
        constexpr float round = 12582912.0f;
        constexpr unsigned above = 0x4b400000u * 0x11111111u;
#pragma unroll
        for (int i = 7; i >= 0; --i) {
            const float d = x[i] - m, q = d * r;
            code = code * 16u + __float_as_uint(fmaf(fmaf(-q, s, d), r, q) + round);
        }
        code -= above;
    } else {
        if (!isfinite(lo) || !isfinite(hi)) {
            meta = 0x7fff0000u;
            return 0u;
        }
        const bool wide = isinf(range);   // beyond fp32: quotients first, then their difference
        if (wide) sb = (__float_as_uint(hi / 15.0f - m / 15.0f) + 0xffffu) & 0xffff0000u;
        s = __uint_as_float(sb);
        if (isinf(m) || isinf(s)) {
            meta = 0x7fff0000u;
            return 0u;
        }
        const float d = s > 0.0f ? s : 1.0f;   // a group of one value that bf16 holds has no steps
#pragma unroll
        for (int i = 7; i >= 0; --i) code = code << 4 | (unsigned)fminf(fmaxf(rintf(wide ? x[i] / d - m / d : __fdiv_rn(x[i] - m, d)), 0.0f), 15.0f);
    }
    meta = mb | sb >> 16;
    return code;
}
// From four values of either half of a vector (as the rotation has them) to eight consecutive ones: even lanes get the first half's.
template <int HD>
__device__ __forceinline__ void q4_gather(float4 a, float4 d, int l, float (&x)[8]) {
    const bool odd = l & 1;
    const float4 give = odd ? a : d;
    const float4 got = make_float4(__shfl_xor_sync(0xffffffffu, give.x, 1), __shfl_xor_sync(0xffffffffu, give.y, 1), __shfl_xor_sync(0xffffffffu, give.z, 1),
                                   __shfl_xor_sync(0xffffffffu, give.w, 1));
    const float4 u = odd ? got : a, v = odd ? d : got;
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
}
// The dimensions that lane l has then begin at this one.
template <int HD>
__device__ __forceinline__ int q4_first(int l) { return (l & 1) * (HD / 2) + (l >> 1) * 8; }

// A token's eight dimensions from `d0` on, and their group's scale and minimum, into its tile.
template <int HD>
__device__ __forceinline__ void q4_put(unsigned char* tile, bool value, int in, int d0, unsigned code, unsigned meta) {
    using T = Q4Layout<HD>;
    const int g = d0 / 32, c = d0 % 32 / 4;
    if (value) {
        *reinterpret_cast<unsigned short*>(tile + T::value_at(in, g, c)) = (unsigned short)code;
        *reinterpret_cast<unsigned short*>(tile + T::value_at(in, g, c + 1)) = (unsigned short)(code >> 16);
    } else {
        *reinterpret_cast<unsigned*>(tile + T::key_at(in, g, c)) = code;
    }
    if (c == 0) {
        *reinterpret_cast<unsigned short*>(tile + (value ? T::value_scales : T::key_scales) + T::meta_at(in, g)) = (unsigned short)meta;
        *reinterpret_cast<unsigned short*>(tile + (value ? T::value_mins : T::key_mins) + T::meta_at(in, g)) = (unsigned short)(meta >> 16);
    }
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

__device__ __forceinline__ void q4_rotate(float4& a, float4& d, const float (&c)[4], const float (&s)[4]) {
    const float4 x = a, y = d;
    a = make_float4(x.x * c[0] - y.x * s[0], x.y * c[1] - y.y * s[1], x.z * c[2] - y.z * s[2], x.w * c[3] - y.w * s[3]);
    d = make_float4(y.x * c[0] + x.x * s[0], y.y * c[1] + x.y * s[1], y.z * c[2] + x.z * s[2], y.w * c[3] + x.w * s[3]);
}

// Few tokens: 1024 / HD vectors (keys, values and queries of one token) per CTA, HD / 8 lanes to a vector, each with four dimensions of
// either half (a rotated pair is in one lane, a group is eight lanes).  Bound by latency: everything that does not wait for the
// position is asked for before it, the page while the angles are made.  One token of 8 KV heads and 32 query heads of 128: 2.3 us.
template <int HD, bool kBf16>
__global__ void __launch_bounds__(128) q4_append_kernel(const __grid_constant__ Q4AppendProblem P) {
    constexpr int L = HD / 8, V = 128 / L;
    chain_begin();
    const int kv = P.cache.kv_heads, tasks = 2 * kv + (P.q ? P.q_heads : 0), parts = (tasks + V - 1) / V;
    const int token = blockIdx.x / parts, l = threadIdx.x % L, first = blockIdx.x % parts * V + threadIdx.x / L;
    const int task = min(first, tasks - 1);      // (the lanes of a warp stay together for the shuffles)
    const int kind = task < kv ? 0 : task < 2 * kv ? 1 : 2, head = kind == 2 ? task - 2 * kv : task - kind * kv;
    const void* src = kind == 0 ? P.k : kind == 1 ? P.v : P.q;
    const size_t at = (size_t)token * (kind == 0 ? P.k_stride : kind == 1 ? P.v_stride : P.q_stride) + (size_t)head * HD + 4 * l;
    float4 a = q4_load4(src, at, kBf16), d = q4_load4(src, at + HD / 2, kBf16);
    int b = token, pos;
    if (P.ends) {
        b = packed_owner(P.ends, P.batch, token);
        if (b < 0) return;   // (of the whole CTA)
        pos = P.positions[b] < 0 ? -1 : P.positions[b] + token - P.ends[b];   // (a sequence that begins nowhere has no place at all)
    } else {
        pos = P.positions[b];
    }
    uint8_t* tile = kind == 2 ? nullptr : q4_tile<HD>(P.cache, b, head, pos);
    if (kind != 1 && P.turns) {
        float c[4], s[4];
        q4_angles(P.turns, 4 * l, pos, c, s);
        q4_rotate(a, d, c, s);
    }
    float x[8];
    q4_gather<HD>(a, d, l, x);
    unsigned meta;
    const unsigned code = q4_encode(x, meta);
    if (first >= tasks) return;
    if (kind == 2) {
        const size_t to = ((size_t)token * P.q_heads + head) * HD + 4 * l;
        q4_store4(P.q_out, to, kBf16, a);
        q4_store4(P.q_out, to + HD / 2, kBf16, d);
    } else if (tile) {
        q4_put<HD>(tile, kind == 1, pos % kQ4Tile, q4_first<HD>(l), code, meta);
    } else if (l == 0) {
        atomicExch(P.cache.status, 1);
    }
}

// A tile of the cache that tokens `from` to `to` (in it) of a CTA's rows lie in: its sequence, the first one's row and position.
struct Q4Span { int b, row, pos, from, to; };

// Span `index` of the tiles that the packed tokens of all sequences touch; all lanes of a warp call it together.  A sequence that begins
// at a negative position has none, which `status` tells.
__device__ __forceinline__ bool q4_span(const int* ends, const int* positions, int batch, int rows, int index, int* status, Q4Span& S) {
    int part = 0;
    auto tiles = [&](int b) {
        const PackedRange r = packed_range(ends, b, rows);
        if (r.count == 0) return 0;
        if (positions && positions[b] < 0) {
            atomicExch(status, 1);
            return 0;
        }
        const int in = (positions ? positions[b] : 0) % kQ4Tile;
        return (in + r.count + kQ4Tile - 1) / kQ4Tile;
    };
    if (!packed_part(batch, index, tiles, S.b, part)) return false;
    const PackedRange r = packed_range(ends, S.b, rows);
    const int begin = positions ? positions[S.b] : 0, in = begin % kQ4Tile;
    S.from = part == 0 ? in : 0;
    S.to = min(kQ4Tile, in + r.count - part * kQ4Tile);
    S.pos = begin - in + part * kQ4Tile;     // of the tile's first token
    S.row = r.first - in + part * kQ4Tile;   // (whose row may be another sequence's)
    return true;
}
// Tiles that packed tokens can touch.
static long long q4_spans(int rows, int batch) { return rows / kQ4Tile + 2LL * std::min(rows, batch); }

// Prompts: a tile of 16 tokens per CTA and some of the heads, a token to HD / 8 lanes (or two of them at head_dim 64), which make its
// angles once.  A head's tile is put together in shared memory and written in 16-byte pieces: its words hold two tokens each.  No pipe is
// full (integer pipe 43 %): warps wait for their loads, one vector ahead in 64 registers, and at the barrier of every turn of heads.
// 16384 tokens of 8 KV heads of 128 in bf16 take 36.9 us, 88 MB; with 32 query heads 78, 357 MB, against 190 by single vectors, each of
// which makes its angles anew.  In fp32 it spills 8 to 20 bytes.
template <int HD, bool kBf16>
__global__ void __launch_bounds__(256, 4) q4_append_tile_kernel(const __grid_constant__ Q4AppendProblem P, int slices) {
    constexpr int L = HD / 8, G = HD / 32, W = 256 / (kQ4Tile * L);   // W: vectors of a token at a time
    using T = Q4Layout<HD>;
    __shared__ __align__(16) unsigned char s_tile[2][W * T::bytes];
    __shared__ Q4Span s_span;
    chain_begin();
    if (threadIdx.x < 32) {
        Q4Span S{-1, 0, 0, 0, 0};
        if (!q4_span(P.ends, P.positions, P.batch, P.n_tokens, blockIdx.x / slices, P.cache.status, S)) S.b = -1;
        if (threadIdx.x == 0) s_span = S;
    }
    __syncthreads();
    const Q4Span S = s_span;
    if (S.b < 0) return;
    const int kv = P.cache.kv_heads, slice = blockIdx.x % slices, l = threadIdx.x % L, w = threadIdx.x / L % W, in = threadIdx.x / (L * W);
    const bool live = in >= S.from && in < S.to;
    const size_t row = (size_t)(S.row + (live ? in : S.from));   // (the lanes of a warp stay together for the shuffles)
    float c[4] = {}, s[4] = {};
    if (P.turns) q4_angles(P.turns, 4 * l, S.pos + in, c, s);
    uint8_t* const tile = q4_tile<HD>(P.cache, S.b, 0, S.pos);
    if (!tile && threadIdx.x == 0) atomicExch(P.cache.status, 1);
    const size_t head_bytes = (size_t)(P.cache.page_size / kQ4Tile) * T::bytes;

    if (P.q) {
        const int h1 = (int)((long long)P.q_heads * (slice + 1) / slices);
        for (int h = (int)((long long)P.q_heads * slice / slices) + w; h < h1; h += 4 * W) {
            float4 a[4], d[4];   // loads ahead of what is done with them
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const size_t at = row * P.q_stride + (size_t)min(h + u * W, h1 - 1) * HD + 4 * l;
                a[u] = q4_load4(P.q, at, kBf16);
                d[u] = q4_load4(P.q, at + HD / 2, kBf16);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (!live || h + u * W >= h1) continue;
                if (P.turns) q4_rotate(a[u], d[u], c, s);
                const size_t to = (row * P.q_heads + h + u * W) * HD + 4 * l;
                q4_store4(P.q_out, to, kBf16, a[u]);
                q4_store4(P.q_out, to + HD / 2, kBf16, d[u]);
            }
        }
    }
    const int h0 = (int)((long long)kv * slice / slices), h1 = (int)((long long)kv * (slice + 1) / slices);
    if (!tile || h0 >= h1) return;
    // keys as the rotation wants them, values as they are encoded
    const int d0 = q4_first<HD>(l);
    float4 x[4];
    auto load = [&](int h) {
        const size_t key = row * P.k_stride + (size_t)min(h, h1 - 1) * HD + 4 * l, value = row * P.v_stride + (size_t)min(h, h1 - 1) * HD + d0;
        x[0] = q4_load4(P.k, key, kBf16);
        x[1] = q4_load4(P.k, key + HD / 2, kBf16);
        q4_load8(P.v, value, kBf16, x[2], x[3]);
    };
    load(h0 + w);
    int turn = 0;
    for (int h = h0; h < h1; h += W, turn ^= 1) {
        unsigned char* to = s_tile[turn] + w * T::bytes;
        float4 a = x[0], d = x[1];
        const float values[8] = {x[2].x, x[2].y, x[2].z, x[2].w, x[3].x, x[3].y, x[3].z, x[3].w};
        if (h + W < h1) load(h + W + w);
        if (P.turns) q4_rotate(a, d, c, s);
        float keys[8];
        q4_gather<HD>(a, d, l, keys);
        unsigned meta;
        unsigned code = q4_encode(keys, meta);
        q4_put<HD>(to, false, in, d0, code, meta);
        code = q4_encode(values, meta);
        q4_put<HD>(to, true, in, d0, code, meta);
        __syncthreads();   // (the other buffer's pieces were read before the barrier of the turn before)
        const int heads = min(W, h1 - h);
        if (S.from == 0 && S.to == kQ4Tile) {
            for (int i = threadIdx.x; i < heads * (T::bytes / 16); i += 256) {
                const int head = i / (T::bytes / 16), piece = i % (T::bytes / 16);
                *reinterpret_cast<uint4*>(tile + (h + head) * head_bytes + piece * 16) = *reinterpret_cast<const uint4*>(s_tile[turn] + i * 16);
            }
        } else {   // only these tokens' parts
            constexpr int pieces = 2 * (8 * G + 2 * G);   // of 16 bits, of a token
            for (int i = threadIdx.x; i < heads * kQ4Tile * pieces; i += 256) {
                const int head = i / (kQ4Tile * pieces), token = i / pieces % kQ4Tile, piece = i % pieces, which = piece / (10 * G), p = piece % (10 * G);
                if (token < S.from || token >= S.to) continue;
                const int at = p < 8 * G ? (which ? T::value_at(token, p / 8, p % 8) : T::key_at(token, p / 8, p % 8))
                                         : (p < 9 * G ? (which ? T::value_scales : T::key_scales) - 8 * G * 2 : (which ? T::value_mins : T::key_mins) - 9 * G * 2) + T::meta_at(token, 0) + p * 2;
                *reinterpret_cast<unsigned short*>(tile + (h + head) * head_bytes + at) = *reinterpret_cast<const unsigned short*>(s_tile[turn] + head * T::bytes + at);
            }
        }
    }
}

struct Q4ReadProblem {
    Q4Cache cache;
    void *k, *v;                // [n_tokens][kv_heads][head_dim]
    const int *ends, *positions;   // positions null: from the first token
    unsigned char* none;        // [n_tokens] or null: 1 for a token without a page, 0 for the others
    int n_tokens, batch;
};

// A tile of 16 tokens and up to eight KV heads per CTA: the tiles of the heads come in 16-byte pieces, eight values of a token go out in
// one or two.  Tokens without a page are read as zeros.  Bound by what it writes: 16384 tokens of 8 heads of 128 as bf16 in 19 us, 88 MB.
constexpr int kQ4ReadHeads = 8;

template <int HD, bool kBf16>
__global__ void __launch_bounds__(256) q4_read_kernel(const __grid_constant__ Q4ReadProblem P) {
    using T = Q4Layout<HD>;
    __shared__ __align__(16) unsigned char s_tile[kQ4ReadHeads * T::bytes];
    __shared__ Q4Span s_span;
    chain_begin();
    if (threadIdx.x < 32) {
        Q4Span S{-1, 0, 0, 0, 0};
        if (!q4_span(P.ends, P.positions, P.batch, P.n_tokens, blockIdx.x, P.cache.status, S)) S.b = -1;
        if (threadIdx.x == 0) s_span = S;
    }
    __syncthreads();
    const Q4Span S = s_span;
    if (S.b < 0) return;
    const int kv = P.cache.kv_heads, h0 = blockIdx.y * kQ4ReadHeads, heads = min(kQ4ReadHeads, kv - h0);
    const uint8_t* tile = q4_tile<HD>(P.cache, S.b, h0, S.pos);
    const size_t head_bytes = (size_t)(P.cache.page_size / kQ4Tile) * T::bytes;
    if (tile) {
        for (int i = threadIdx.x; i < heads * (T::bytes / 16); i += 256)
            *reinterpret_cast<uint4*>(s_tile + i * 16) = *reinterpret_cast<const uint4*>(tile + i / (T::bytes / 16) * head_bytes + i % (T::bytes / 16) * 16);
    } else if (threadIdx.x == 0) {
        atomicExch(P.cache.status, 1);
    }
    if (P.none && blockIdx.y == 0 && threadIdx.x >= S.from && threadIdx.x < S.to) P.none[S.row + threadIdx.x] = tile ? 0 : 1;
    __syncthreads();
    // eight dimensions of a token and head per thread
    constexpr int E = HD / 8, R = 256 / (2 * kQ4ReadHeads * E);   // R: tokens at a time
    const int d8 = threadIdx.x % E, head = threadIdx.x / E % kQ4ReadHeads, which = threadIdx.x / (E * kQ4ReadHeads) % 2, g = d8 / 4, c = d8 % 4 * 2;
    if (head >= heads) return;
    const unsigned char* from = s_tile + head * T::bytes;
    const size_t to0 = ((size_t)S.row * kv + h0 + head) * HD + d8 * 8;
    for (int token = S.from + threadIdx.x / (E * kQ4ReadHeads * 2); token < S.to; token += R) {
        float x[8];
        if (tile) {
            unsigned word;
            if (which) word = *reinterpret_cast<const unsigned short*>(from + T::value_at(token, g, c)) | (unsigned)*reinterpret_cast<const unsigned short*>(from + T::value_at(token, g, c + 1)) << 16;
            else word = *reinterpret_cast<const unsigned*>(from + T::key_at(token, g, c));
            const float s = q4_bf16(*reinterpret_cast<const unsigned short*>(from + (which ? T::value_scales : T::key_scales) + T::meta_at(token, g)));
            const float m = q4_bf16(*reinterpret_cast<const unsigned short*>(from + (which ? T::value_mins : T::key_mins) + T::meta_at(token, g)));
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = fmaf(__uint_as_float(0x4b000000u | (word >> (4 * u) & 15u)) - 8388608.0f, s, m);
        } else {
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = 0.0f;
        }
        void* out = which ? P.v : P.k;
        const size_t to = to0 + (size_t)token * kv * HD;
        if (kBf16) {
            unsigned w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * u], x[2 * u + 1]);
                w[u] = *reinterpret_cast<const unsigned*>(&p);
            }
            *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(out) + to) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            float4* f = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + to);
            f[0] = make_float4(x[0], x[1], x[2], x[3]);
            f[1] = make_float4(x[4], x[5], x[6], x[7]);
        }
    }
}

}  // namespace ojx

using namespace ojx;

extern "C" {

size_t ojasx_b200_q4kv_page_bytes(int kv_heads, int page_size, int head_dim) {
    if (kv_heads <= 0 || page_size <= 0 || page_size % kQ4Tile || (head_dim != 64 && head_dim != 128)) return 0;
    return (size_t)kv_heads * (page_size / kQ4Tile) * (head_dim == 64 ? Q4Layout<64>::bytes : Q4Layout<128>::bytes);
}

int ojasx_b200_q4kv_append(const OjasxQ4Cache* cache, const void* d_k, long long k_stride, const void* d_v, long long v_stride, const void* d_q,
                           long long q_stride, void* d_q_out, const int* d_block_table, int max_pages, const int* d_positions,
                           const int* d_ends, int n_tokens, int batch, int io_dtype, void* stream) {
    const int rc = q4_check(cache, d_block_table, max_pages, batch, io_dtype);
    if (rc != OJX_OK) return rc;
    if (!d_k || !d_v || !d_positions || n_tokens < 0 || (d_q && !d_q_out) || (!d_ends && n_tokens != batch)) return OJX_ERR_ARG;
    if (!q4_aligned(d_k) || !q4_aligned(d_v) || !q4_aligned(d_q) || !q4_aligned(d_q_out) || (k_stride | v_stride | q_stride) % (io_dtype == OJX_BF16 ? 8 : 4)) return OJX_ERR_ARG;
    const int kv_heads = cache->kv_heads, q_heads = cache->q_heads, head_dim = cache->head_dim;
    if (n_tokens == 0) return OJX_OK;
    Q4AppendProblem P{};
    P.cache = q4_cache(cache, d_block_table, max_pages);
    P.k = d_k; P.v = d_v; P.q = d_q; P.q_out = d_q_out; P.k_stride = k_stride; P.v_stride = v_stride; P.q_stride = q_stride;
    P.positions = d_positions; P.ends = d_ends; P.turns = cache->turns; P.n_tokens = n_tokens; P.batch = batch; P.q_heads = q_heads;
    const bool bf = io_dtype == OJX_BF16;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int vectors = 1024 / head_dim, parts = (2 * kv_heads + (d_q ? q_heads : 0) + vectors - 1) / vectors;
    // Few tokens by vectors, many by tiles, each sequence of which begins and ends with a part of one.  us of the two at 8 KV heads and 32
    // query heads of 128 in bf16: one sequence of 64 tokens 2.9 and 4.7, 256 5.6 and 4.9, 1024 13.2 and 7.9; 16 sequences of 16 6.4 and 8.1,
    // of 32 8.9 and 8.9, of 64 15.0 and 10.9; 64 of 4 7.1 and 8.9, of 16 15.9 and 14.5, of 64 55.7 and 28.4.
    if (d_ends && (long long)n_tokens * parts > 12LL * num_sms() + 48LL * batch) {
        const long long tiles = q4_spans(n_tokens, batch);
        // equal slices of the heads while the CTAs are at most three times what the GPU holds (us with 8 heads in 1, 2 and 3 slices for one
        // sequence of 16384 tokens without queries: 36.2, 39.1 and 43.9; in 4 and 7 for 64 of 16: 14.0 and 16.6; in 2 and 4 for 64 of 64: 30.0 and 28.1)
        int slices = kv_heads;
        while (slices > 1 && (kv_heads % slices || tiles * slices > 12LL * num_sms())) --slices;
        if (tiles * slices > 0x7fffffffLL) return OJX_ERR_TOO_LARGE;
        auto kernel = head_dim == 64 ? (bf ? q4_append_tile_kernel<64, true> : q4_append_tile_kernel<64, false>)
                                     : (bf ? q4_append_tile_kernel<128, true> : q4_append_tile_kernel<128, false>);
        OJX_CUDA_TRY(launch_chained(kernel, dim3((unsigned)(tiles * slices)), 256, 0, s, P, slices));
    } else {
        if ((long long)n_tokens * parts > 0x7fffffffLL) return OJX_ERR_TOO_LARGE;
        auto kernel = head_dim == 64 ? (bf ? q4_append_kernel<64, true> : q4_append_kernel<64, false>)
                                     : (bf ? q4_append_kernel<128, true> : q4_append_kernel<128, false>);
        OJX_CUDA_TRY(launch_chained(kernel, dim3((unsigned)(n_tokens * parts)), 128, 0, s, P));
    }
    count_launch(1);
    return OJX_OK;
}

int ojasx_b200_q4kv_read(const OjasxQ4Cache* cache, const int* d_block_table, int max_pages, const int* d_ends, const int* d_positions, void* d_k,
                         void* d_v, int n_tokens, int batch, int io_dtype, void* stream) {
    return ojasx_b200_q4kv_read_marked(cache, d_block_table, max_pages, d_ends, d_positions, d_k, d_v, nullptr, n_tokens, batch, io_dtype, stream);
}

int ojasx_b200_q4kv_read_marked(const OjasxQ4Cache* cache, const int* d_block_table, int max_pages, const int* d_ends, const int* d_positions,
                                void* d_k, void* d_v, unsigned char* d_none, int n_tokens, int batch, int io_dtype, void* stream) {
    const int rc = q4_check(cache, d_block_table, max_pages, batch, io_dtype);
    if (rc != OJX_OK) return rc;
    if (!d_ends || !d_k || !d_v || n_tokens < 0 || !q4_aligned(d_k) || !q4_aligned(d_v) || !q4_aligned(d_none)) return OJX_ERR_ARG;
    const int kv_heads = cache->kv_heads, head_dim = cache->head_dim;
    if (n_tokens == 0) return OJX_OK;
    Q4ReadProblem P{};
    P.cache = q4_cache(cache, d_block_table, max_pages);
    P.k = d_k; P.v = d_v; P.ends = d_ends; P.positions = d_positions; P.none = d_none; P.n_tokens = n_tokens; P.batch = batch;
    const bool bf = io_dtype == OJX_BF16;
    auto kernel = head_dim == 64 ? (bf ? q4_read_kernel<64, true> : q4_read_kernel<64, false>)
                                 : (bf ? q4_read_kernel<128, true> : q4_read_kernel<128, false>);
    const long long tiles = q4_spans(n_tokens, batch);
    if (tiles > 0x7fffffffLL || kv_heads > 65535 * kQ4ReadHeads) return OJX_ERR_TOO_LARGE;
    OJX_CUDA_TRY(launch_chained(kernel, dim3((unsigned)tiles, (kv_heads + kQ4ReadHeads - 1) / kQ4ReadHeads), 256, 0, static_cast<cudaStream_t>(stream), P));
    count_launch(1);
    return OJX_OK;
}

}  // extern "C"
