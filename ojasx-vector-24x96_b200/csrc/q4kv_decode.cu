// Attention of single tokens over the 4-bit paged cache: softmax(q K^T * scale) V of up to eight query heads per KV head at a time.
//
// With the codes c, scales s and minima m of a token's groups of 32 dimensions, a score is sum_g (s_g (q_g . c_g) + m_g sum(q_g)) and
// the result sum_t p_t (s_tg c_t + m_tg) per dimension of group g: both products take the codes as they are on mma.sync m16n8k16, and
// the scales join in fp32 (those of the values before their product, as p * s).  A nibble in the lowest bits of an fp16 number is the
// subnormal c * 2^-24, in the next ones 16 times that: a word of eight codes becomes operands with five integer instructions, and the
// powers of two are taken out of the queries and the results (12 instructions for bf16 numbers, which need an exponent and its
// subtraction: 295 against 211 us at 16 sequences of 32768 tokens, 8 KV heads of 4 query heads of 128).  The tensor cores line up what
// they add by exponents that a subnormal does not have: sums of them keep 16 bits, enough for bf16 activations.  For fp32 ones the
// codes are made whole numbers around zero, 1024 + c less 1032, and the minima m + 8 s: the two parts of a result are then of its own
// size and do not cancel (2e-5 off 64 bits with subnormals, 8e-7 with c itself, 2e-7 so).
// A warp takes tiles of 16 tokens:
//   S[token][head]  = codes of K (16 x 16 a step) x q (16 x 8)           a group's steps have sums of their own
//   O[dim][head]   += codes of V, transposed (16 x 16) x p * s_g (16 x 8)    p * s_g turned by movmatrix
// A bf16 query is one fp16 number where a power of two brings the head's largest to 2^15 (what is 2^29 below it loses bits), an fp32
// one two of them (22 bits); so is p * s * 2^u, one with bf16 activations (11 bits, below the rounding of the result), two with fp32.
// Each head has an exponent u for each group of dimensions, which goes down where a product would pass 2^14, so that the largest so far is at
// 2^5: scales that differ from token to token or from group to group, by 2^22 in the tests, cost one another no bits.  (One exponent for
// all of them, that of the largest scale met so far, took 64 and 145 us in the place of the 67 and 149 below, but a token of large scale and next to
// no weight cost all others theirs: 1.4e-4 off 64 bits at 2^16, 8e-3 at 2^22.)  u is 100 at most: scales below 2^-100 weigh nothing.
//
// Work: units of 128 tokens of a (sequence, KV head, eight query heads), all of them in a row, in equal shares for the CTAs whatever the
// lengths are; the four warps of a CTA take two tiles of a unit each, from rings of their own that bulk copies fill.  A share that begins
// or ends inside a sequence leaves its sums to q4_combine_kernel.
//
// No pipe is full (integer pipe 55 %, tensor pipe 20 %, 12 warps an SM, 391 instructions a tile and warp): warps wait for their chains of
// product, exponential and product, next to the copies, which alone take 111 to 130 us: 16 sequences of 32768 tokens, 671 MB, in 149 us
// (4.5 TB/s) with 8 KV heads of 4 query heads of 128 in bf16; 48 of up to 20011, 4 heads of 7 of 64 in fp32, 106 MB, in 67 us, where the
// second planes of queries and weights double the products.  fp32 at head_dim 128 spills 48 bytes (168 registers for three CTAs an SM).
#include <algorithm>
#include <cmath>

#include "gather_mma.cuh"
#include "handles.h"
#include "launch.h"
#include "q4kv.cuh"
#include "../../include/ojasx_lut_b200.h"

namespace ojx {

constexpr int kQdThreads = 128, kQdWarps = 4, kQdStages = 2, kQdHeads = 8, kQdPair = 2;
constexpr int kQdUnit = kQdWarps * kQdPair * kQ4Tile;   // tokens
constexpr float kQdLowest = -3.0e38f;         // finite: scores of -inf weigh nothing, a NaN makes its head's result one
constexpr float kQdSlack = 8.0f;              // weights are relative to a reference, until a score is 2^8 above it
constexpr int kQdRoom = 5;                    // the largest p * s * 2^u is 2^5 to 2^6 when u is set ...
constexpr unsigned kQdTooLarge = 0x74007400u; // ... and 2^14 at most (two fp16 numbers)
constexpr int kQdMost = 127 + 100;            // u at most, as the exponent of a float

static __device__ int g_q4_error;   // raised when a bounded wait inside a kernel ran out

struct Q4DecodeProblem {
    Q4Cache cache;
    const void* q;              // [batch][q_heads][head_dim]
    void* out;
    const int* lengths;         // [batch]
    int2* pieces;               // [CTAs] item that begins and does not end in the CTA's share (-1: none), last CTA with a part of it
    float* partials;            // [CTAs][2][8][head_dim + 2]: of an item that began before the share, of one that does not end in it
    int batch, q_heads, share, blocks;   // blocks: of eight query heads per KV head
    float scale;                // times log2(e)
};

template <int N> struct Q4Words;
template <> struct Q4Words<1> { using type = unsigned; };
template <> struct Q4Words<2> { using type = uint2; };
template <> struct Q4Words<4> { using type = uint4; };

__device__ __forceinline__ void q4_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned q4_turn(unsigned v) {   // an 8 x 8 matrix of 16-bit numbers, a pair per lane
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// Nibbles i and i + 4 of a word as fp16 numbers, 16 times as large for odd i: c * 2^-24 (kSub) or c - 8.
template <bool kSub>
__device__ __forceinline__ void q4_codes(unsigned w, unsigned (&c)[4]) {
    const unsigned v = w >> 8, one = kSub ? 0u : 0x64006400u;   // 1024
    c[0] = (w & 0x000f000fu) | one;
    c[1] = (w & 0x00f000f0u) | one;
    c[2] = (v & 0x000f000fu) | one;
    c[3] = (v & 0x00f000f0u) | one;
    if (!kSub) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float zero = i & 1 ? 1024.0f + 16 * 8.0f : 1024.0f + 8.0f;
            const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&c[i]), __floats2half2_rn(zero, zero));
            c[i] = *reinterpret_cast<const unsigned*>(&h);
        }
    }
}
__device__ __forceinline__ float q4_exp2(float x) {
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
    return x;
}
// The next fp16 part of two numbers, which keep the rest.
__device__ __forceinline__ unsigned q4_part(float& a, float& b) {
    const __half2 h = __floats2half2_rn(a, b);
    a -= __low2float(h);
    b -= __high2float(h);
    return *reinterpret_cast<const unsigned*>(&h);
}
// Two products in one instruction.
__device__ __forceinline__ float2 q4_mul2(float2 a, float2 b) {
    float2 c;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(c.x), "=f"(c.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return c;
}
// The power of two with this exponent field (zero where the field would be negative), and the field of a number that is not negative.
__device__ __forceinline__ float q4_power(int field) { return __uint_as_float((unsigned)max(field, 0) << 23); }
__device__ __forceinline__ int q4_bits(float x) { return (int)(__float_as_uint(x) >> 23); }

// Quotient of numbers that are not negative (64-bit division takes some hundred instructions).
__device__ __forceinline__ long long q4_quotient(long long a, long long b) {
    return (unsigned long long)a >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
}
// All units in shares that differ by one at most, none of them empty.
struct Q4Shares {
    long long least, more;   // units of a share; shares with one more, the first ones
    int n;
    __device__ __forceinline__ Q4Shares(long long all, int ctas) : n((int)min((long long)ctas, all)) {
        least = n ? q4_quotient(all, n) : 0;
        more = all - least * n;
    }
    __device__ __forceinline__ long long first(int cta) const { return least * min(cta, n) + min((long long)min(cta, n), more); }
    __device__ __forceinline__ int owner(long long unit) const {
        const long long big = more * (least + 1);
        return (int)(unit < big ? q4_quotient(unit, least + 1) : more + q4_quotient(unit - big, least));
    }
};

// A place in the row of units: unit `u` of the `units` of sequence b for (KV head, block of query heads) `hh`.
struct Q4Place {
    int b, hh, u, units;
    __device__ __forceinline__ void skip(const Q4DecodeProblem& P, int heads) {   // to the next unit, on through sequences without any
        if (++u < units) return;
        u = 0;
        if (++hh < heads) return;
        hh = 0;
        do ++b;
        while (b < P.batch && (units = length_units(P, b)) == 0);
    }
    static __device__ __forceinline__ int length(const Q4DecodeProblem& P, int b) {
        return min(max(P.lengths[b], 0), P.cache.max_pages * P.cache.page_size);
    }
    static __device__ __forceinline__ int length_units(const Q4DecodeProblem& P, int b) { return (length(P, b) + kQdUnit - 1) / kQdUnit; }
};

template <int HD>
struct QdSmem {
    static constexpr int stage = kQdPair * Q4Layout<HD>::bytes, ring = kQdStages * stage;    // of a warp
    static constexpr int row = HD + 8;                              // of a head's sums
    static constexpr int bytes(int heads) { return kQdWarps * (ring + heads * row * 4); }
};

constexpr int kQdCtas = 3;   // per SM (16 sequences of 32768 tokens, with one exponent for all groups: 151 us; 2: 154, 4: 159)

template <int HD, bool kBf16>
__global__ void __launch_bounds__(kQdThreads, kQdCtas) q4_decode_kernel(const __grid_constant__ Q4DecodeProblem P) {
    constexpr int G = HD / 32, NP = kBf16 ? 1 : 2;
    constexpr float kCode = kBf16 ? 16777216.0f : 1.0f;   // what the operands are less than their codes
    using T = Q4Layout<HD>;
    using M = QdSmem<HD>;
    using Words = typename Q4Words<G>::type;
    using Metas = typename Q4Words<G / 2>::type;   // a token's scales or minima
    extern __shared__ __align__(128) unsigned char qd_smem[];
    constexpr int kAtOnce = kBf16 ? kQdPair : 1;   // tiles whose weights are looked at together
    __shared__ float s_m[kQdWarps][kQdHeads], s_l[kQdWarps][kQdHeads];
    __shared__ __align__(8) float s_up[kQdWarps][G * kQdHeads];   // [group][head] 2^u
    __shared__ __align__(8) unsigned long long s_bar[kQdWarps][kQdStages];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, t = lane & 3, sum_heads = min(P.share, kQdHeads);
    unsigned char* ring = qd_smem + warp * M::ring;
    float* sums = reinterpret_cast<float*>(qd_smem + kQdWarps * M::ring);
    const unsigned ring_at = static_cast<unsigned>(__cvta_generic_to_shared(ring)), bar_at = static_cast<unsigned>(__cvta_generic_to_shared(&s_bar[warp][0]));
    if (lane == 0) {
        for (int i = 0; i < kQdStages; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar_at + 8 * i) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    chain_begin();
    const int heads = P.cache.kv_heads * P.blocks;

    // this CTA's share of all units, and the place where it begins
    long long total = 0;
    int mine = 0, upto = 0;   // units of the lane's sequence (of the last 32), and with those before it
    for (int b0 = 0; b0 < P.batch; b0 += 32) {
        mine = upto = b0 + lane < P.batch ? Q4Place::length_units(P, b0 + lane) : 0;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, off);
            if (lane >= off) upto += o;
        }
        total += __shfl_sync(0xffffffffu, upto, 31);
    }
    // an empty sequence has no units: its zeros come from here
    for (int b = blockIdx.x; b < P.batch; b += gridDim.x) {
        const int length = Q4Place::length(P, b);
        if (tid == 0 && P.lengths[b] > length) atomicExch(P.cache.status, 1);   // more tokens than the table has room for
        if (length > 0) continue;
        for (int i = tid; i < P.q_heads * HD; i += kQdThreads) {
            if (kBf16) reinterpret_cast<__nv_bfloat16*>(P.out)[(size_t)b * P.q_heads * HD + i] = __float2bfloat16_rn(0.0f);
            else reinterpret_cast<float*>(P.out)[(size_t)b * P.q_heads * HD + i] = 0.0f;
        }
    }
    if (tid == 0) P.pieces[blockIdx.x] = make_int2(-1, 0);
    const Q4Shares shares(total * heads, gridDim.x);
    const long long first = shares.first(blockIdx.x), last = shares.first(blockIdx.x + 1);
    if (first >= last) return;
    Q4Place at{0, 0, 0, 0};
    {
        long long before = 0;
        for (int b0 = 0; b0 < P.batch; b0 += 32) {
            if (P.batch > 32) {   // (else they are there still)
                mine = upto = b0 + lane < P.batch ? Q4Place::length_units(P, b0 + lane) : 0;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int o = __shfl_up_sync(0xffffffffu, upto, off);
                    if (lane >= off) upto += o;
                }
            }
            const unsigned in = __ballot_sync(0xffffffffu, first < (before + upto) * heads);
            if (in) {
                const int src = __ffs(in) - 1;
                at.b = b0 + src;
                at.units = __shfl_sync(0xffffffffu, mine, src);
                const long long rest = first - (before + __shfl_sync(0xffffffffu, upto - mine, src)) * heads;
                at.hh = (int)q4_quotient(rest, at.units);
                at.u = (int)(rest - (long long)at.hh * at.units);
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    __syncwarp();

    // Copies run ahead by the stages of the ring, two tiles each: lanes 0 and 1 have a tile to themselves (the others do as they do).  A
    // pair that begins before its sequence's end has a stage; a tile behind the end or without a page stays as it is, the latter is
    // marked.  The pages of the next copies are looked up a pair ahead.
    Q4Place ahead = at;
    int rest = (int)(last - first);    // units from `ahead` on
    int left, in, id;                  // tiles of the sequence from this lane's next one on, that one's place in its page, the page's id
    const int* page;                   // its entry in the table
    const uint8_t* head;               // the head's part of page 0
    const int page_tiles = P.cache.page_size / kQ4Tile, step_pages = kQdWarps * kQdPair / page_tiles, step_in = kQdWarps * kQdPair % page_tiles;
    const size_t head_bytes = (size_t)page_tiles * T::bytes, page_bytes = head_bytes * P.cache.kv_heads;
    unsigned missing = 0;     // two bits for each stage
    auto enter = [&]() {   // an item, at its unit `ahead.u`
        const int tile = (ahead.u * kQdWarps + warp) * kQdPair + (lane & 1);
        left = (Q4Place::length(P, ahead.b) + kQ4Tile - 1) / kQ4Tile - tile;
        page = P.cache.block_table + (size_t)ahead.b * P.cache.max_pages + tile / page_tiles;
        head = P.cache.pool + ahead.hh / P.blocks * head_bytes;
        in = tile % page_tiles;
        id = left > 0 ? *page : 0;
    };
    auto next = [&]() {
        --rest;
        if (ahead.u + 1 < ahead.units) {
            ++ahead.u;
            left -= kQdWarps * kQdPair;
            in += step_in;
            page += step_pages;
            if (in >= page_tiles) { in -= page_tiles; ++page; }
            __syncwarp();
            if (left > 0) id = *page;
        } else if (rest > 0) {
            ahead.skip(P, heads);
            enter();
        }
    };
    auto fill = [&](int stage) {   // true: there was a pair
        while (rest > 0 && left + (lane & 1) <= 0) next();
        if (rest <= 0) return false;
        const bool there = left > 0 && (unsigned)id < (unsigned)P.cache.num_pages;
        const unsigned none = __ballot_sync(0xffffffffu, left > 0 && !there) & 3u, copies = __ballot_sync(0xffffffffu, there) & 3u;
        missing = (missing & ~(3u << (2 * stage))) | none << (2 * stage);
        const unsigned bar = bar_at + 8 * stage;
        if (lane == 0) {
            if (copies) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(__popc(copies) * T::bytes) : "memory");
            else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
            if (none) atomicExch(P.cache.status, 1);
        }
        __syncwarp();
        if (lane < kQdPair && there)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(ring_at + stage * M::stage + lane * T::bytes),
                         "l"(head + (size_t)id * page_bytes + in * T::bytes), "n"(T::bytes), "r"(bar)
                         : "memory");
        next();
        return true;
    };
    int filled = 0, taken = 0;
    {   // the first item's queries come while the pages are looked up
        const int h0 = (at.hh % P.blocks) * kQdHeads;
        const char* q = reinterpret_cast<const char*>(P.q) + (((size_t)at.b * P.q_heads + at.hh / P.blocks * P.share + h0 + gq) * HD + 8 * t) * (kBf16 ? 2 : 4);
        if (h0 + gq < P.share)
#pragma unroll
            for (int g = 0; g < G; ++g) asm volatile("prefetch.global.L1 [%0];" ::"l"(q + g * 32 * (kBf16 ? 2 : 4)));
    }
    enter();
    for (int i = 0; i < kQdStages; ++i) filled += fill(i);

    bool ok = true;
    for (long long unit = first; unit < last;) {
        const int head = at.hh / P.blocks, h0 = (at.hh % P.blocks) * kQdHeads, n_heads = min(kQdHeads, P.share - h0), length = Q4Place::length(P, at.b);
        const size_t row0 = ((size_t)at.b * P.q_heads + head * P.share + h0) * HD;
        const bool begins = at.u == 0;
        // the queries as the second operand: lane (head gq, t) has the dimensions 32 g + 8 t + 0..7, pairs i and i + 4
        unsigned qf[NP][G][4];
        unsigned qs[2];       // bf16: sums over the groups in three bf16 parts, as an operand: k = 4 part + group
        float qsum[G][2];     // fp32: sums for the heads 2 t and 2 t + 1
        float unscale[2];
        {
            float x[G][8];
            unsigned most = 0;
#pragma unroll
            for (int g = 0; g < G; ++g) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[g][e] = 0.0f;
                if (gq < n_heads) {
                    const size_t i = row0 + gq * HD + 32 * g + 8 * t;
                    if (kBf16) {
                        const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(P.q) + i);
                        const unsigned ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) { x[g][2 * e] = __uint_as_float(ws[e] << 16); x[g][2 * e + 1] = __uint_as_float(ws[e] & 0xffff0000u); }
                    } else {
                        const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(P.q) + i);
                        const float4 c = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(P.q) + i + 4);
                        x[g][0] = a.x; x[g][1] = a.y; x[g][2] = a.z; x[g][3] = a.w; x[g][4] = c.x; x[g][5] = c.y; x[g][6] = c.z; x[g][7] = c.w;
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(x[g][e]) & 0x7fffffffu);
            }
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            float grow, down;
            gm_scale(most, grow, down);
            // what a score comes out of the products with
            const float back = fminf(fmaxf(down * (P.scale * kCode), 0x1p-126f), 3.0e38f);   // (not zero: what is not seen is -inf times it)
            unscale[0] = __shfl_sync(0xffffffffu, back, 8 * t);        // heads 2 t and 2 t + 1
            unscale[1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
            float total[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < G; ++g) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[g][e] *= grow;
                float sum = ((x[g][0] + x[g][1]) + (x[g][2] + x[g][3])) + ((x[g][4] + x[g][5]) + (x[g][6] + x[g][7]));
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sum *= 1.0f / kCode;
                total[g] = sum;
                if (!kBf16) {
                    qsum[g][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
                    qsum[g][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
                }
#pragma unroll
                for (int i = 1; i < 8; i += 2) x[g][i] *= 0.0625f;     // (the codes of odd nibbles are 16 times as large)
#pragma unroll
                for (int p = 0; p < NP; ++p)
#pragma unroll
                    for (int i = 0; i < 4; ++i) qf[p][g][i] = q4_part(x[g][i], x[g][i + 4]);
            }
            // lane t has k = 2 t and 2 t + 1 (parts 0 and 1), and 8 on (part 2)
            float s0 = t & 1 ? total[2] : total[0], s1 = t & 1 ? total[3] : total[1];
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(s0, s1);
                s0 -= __low2float(h);
                s1 -= __high2float(h);
                const unsigned w = *reinterpret_cast<const unsigned*>(&h);
                if (p == 2) qs[1] = t < 2 ? w : 0u;
                else if (p == t >> 1) qs[0] = w;
            }
        }
        float top[2] = {kQdLowest, kQdLowest}, l[2] = {0.0f, 0.0f}, o[2 * G][4], mins[G][2];
#pragma unroll
        for (int m = 0; m < 2 * G; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[m][e] = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) mins[g][0] = mins[g][1] = 0.0f;

        if (lane < kQdHeads * G) s_up[warp][lane] = 1.0f;
        __syncwarp();
        float2* const up = reinterpret_cast<float2*>(s_up[warp]) + t;   // of group g at 4 g: 2^u for the heads 2 t and 2 t + 1
        const int u0 = at.u, u1 = (int)min((long long)at.units, at.u + (last - unit));
        for (int u = u0; u < u1 && ok; ++u) {
            const int token = (u * kQdWarps + warp) * kQdPair * kQ4Tile;
            if (token >= length) break;
            const int from = taken % kQdStages;
            if (!(ok = __all_sync(0xffffffffu, bar_wait(bar_at + 8 * from, taken / kQdStages & 1)))) break;
            const unsigned char* stage = ring + from * M::stage;
            const unsigned none = missing >> (2 * from) & 3u;
            // tokens of the two tiles that are there
            const int seen[2] = {none & 1 ? 0 : length - token, none & 2 ? 0 : length - token - kQ4Tile};
            const bool part = min(seen[0], seen[1]) < kQ4Tile;
            float x[kQdPair][4];
            float now[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < kQdPair; ++i) {
                const unsigned char* tile = stage + i * T::bytes;
                const Words ka = *reinterpret_cast<const Words*>(tile + (gq * 4 + t) * (4 * G)), kb = *reinterpret_cast<const Words*>(tile + ((gq + 8) * 4 + t) * (4 * G));
                const Metas ma = *reinterpret_cast<const Metas*>(tile + T::key_scales + T::meta_at(gq, 0)), mb = *reinterpret_cast<const Metas*>(tile + T::key_scales + T::meta_at(gq + 8, 0));
                const unsigned *wa = reinterpret_cast<const unsigned*>(&ka), *wb = reinterpret_cast<const unsigned*>(&kb);
                const unsigned *ca = reinterpret_cast<const unsigned*>(&ma), *cb = reinterpret_cast<const unsigned*>(&mb);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][e] = 0.0f;
                if (kBf16) {   // sum_g m_g sum(q_g): the minima, bf16 as they are, times the sums in three parts
                    const int pair = G == 4 ? (t & 1) * 2 : 0;
                    const unsigned a = *reinterpret_cast<const unsigned*>(tile + T::key_mins + T::meta_at(gq, pair)), b = *reinterpret_cast<const unsigned*>(tile + T::key_mins + T::meta_at(gq + 8, pair));
                    q4_mma(x[i], a, b, a, b, qs[0], qs[1]);
                }
                Metas la{}, lb{};
                if (!kBf16) {
                    la = *reinterpret_cast<const Metas*>(tile + T::key_mins + T::meta_at(gq, 0));
                    lb = *reinterpret_cast<const Metas*>(tile + T::key_mins + T::meta_at(gq + 8, 0));
                }
                const unsigned *oa = reinterpret_cast<const unsigned*>(&la), *ob = reinterpret_cast<const unsigned*>(&lb);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    unsigned a[4], b[4];
                    q4_codes<kBf16>(wa[g], a);
                    q4_codes<kBf16>(wb[g], b);
                    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) {
                        gm_mma(c, {a[0], b[0], a[1], b[1]}, qf[p][g][0], qf[p][g][1]);
                        gm_mma(c, {a[2], b[2], a[3], b[3]}, qf[p][g][2], qf[p][g][3]);
                    }
                    const float low = g & 1 ? q4_high(ca[g / 2]) : q4_low(ca[g / 2]), high = g & 1 ? q4_high(cb[g / 2]) : q4_low(cb[g / 2]);
                    if (!kBf16) {
                        const float za = fmaf(8.0f, low, g & 1 ? q4_high(oa[g / 2]) : q4_low(oa[g / 2])), zb = fmaf(8.0f, high, g & 1 ? q4_high(ob[g / 2]) : q4_low(ob[g / 2]));
                        x[i][0] = fmaf(za, qsum[g][0], x[i][0]);
                        x[i][1] = fmaf(za, qsum[g][1], x[i][1]);
                        x[i][2] = fmaf(zb, qsum[g][0], x[i][2]);
                        x[i][3] = fmaf(zb, qsum[g][1], x[i][3]);
                    }
                    x[i][0] = fmaf(low, c[0], x[i][0]);
                    x[i][1] = fmaf(low, c[1], x[i][1]);
                    x[i][2] = fmaf(high, c[2], x[i][2]);
                    x[i][3] = fmaf(high, c[3], x[i][3]);
                }
                if (part) {   // what is behind the last token may be anything
                    if (gq >= seen[i]) x[i][0] = x[i][1] = -INFINITY;
                    if (gq + 8 >= seen[i]) x[i][2] = x[i][3] = -INFINITY;
                }
                now[0] = fmaxf(now[0], fmaxf(x[i][0], x[i][2]));
                now[1] = fmaxf(now[1], fmaxf(x[i][1], x[i][3]));
            }
            // the reference moves where a lane sees a score too far above it; by a whole number, so that all factors are powers of two
            int rise[2] = {0, 0};
            bool update = __any_sync(0xffffffffu, fmaf(now[0], unscale[0], -kQdSlack) > top[0] || fmaf(now[1], unscale[1], -kQdSlack) > top[1]);
            if (update) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) now[h] = fmaxf(now[h], __shfl_xor_sync(0xffffffffu, now[h], off));
                    const float to = fmaf(now[h], unscale[h], -kQdSlack) > top[h] ? ceilf(now[h] * unscale[h]) : top[h];
                    rise[h] = (int)fminf(to - top[h], 1000.0f);
                    top[h] = to;
                }
                if (u > u0) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float keep = q4_power(127 - rise[h]);
                        l[h] *= keep;
#pragma unroll
                        for (int g = 0; g < G; ++g) mins[g][h] *= keep;
                    }
                }
            }
#pragma unroll
            for (int i0 = 0; i0 < kQdPair; i0 += kAtOnce) {
                // a token's scales, or minima, as far as it is there
                auto metas = [&](int i, int at, Metas& a, Metas& b) {
                    const unsigned char* tile = stage + (i0 + i) * T::bytes;
                    a = *reinterpret_cast<const Metas*>(tile + at + T::meta_at(gq, 0));
                    b = *reinterpret_cast<const Metas*>(tile + at + T::meta_at(gq + 8, 0));
                    if (part) {
                        if (gq >= seen[i0 + i]) a = Metas{};
                        if (gq + 8 >= seen[i0 + i]) b = Metas{};
                    }
                };
                auto of_group = [](const Metas& m, int g) {
                    const unsigned w = reinterpret_cast<const unsigned*>(&m)[g / 2];
                    return g & 1 ? q4_high(w) : q4_low(w);
                };
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    float (&p)[4] = x[i0 + i];
                    Metas sa, sb, ma, mb;
                    if (!kBf16) metas(i, T::value_scales, sa, sb);
                    metas(i, T::value_mins, ma, mb);
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = q4_exp2(fmaf(p[e], unscale[e & 1], -top[e & 1]));
                    l[0] += p[0] + p[2];
                    l[1] += p[1] + p[3];
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        float low = of_group(ma, g), high = of_group(mb, g);
                        if (!kBf16) {
                            low = fmaf(8.0f, of_group(sa, g), low);
                            high = fmaf(8.0f, of_group(sb, g), high);
                        }
                        mins[g][0] = fmaf(p[0], low, fmaf(p[2], high, mins[g][0]));
                        mins[g][1] = fmaf(p[1], low, fmaf(p[3], high, mins[g][1]));
                    }
                }
                // p * s * 2^u as fp16 parts.  Where the reference has risen, u has with it, and the sums stay; u goes down where a product would be
                // too large (of the first ones always), and the sums with it.
                unsigned y[kAtOnce][G][NP][2];
                for (;; update = true) {
                    if (update) {
                        float high[G][2];
                        int was[G][2];
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            const float2 f = up[g * 4];
                            was[g][0] = q4_bits(f.x) + rise[0];
                            was[g][1] = q4_bits(f.y) + rise[1];
                            high[g][0] = high[g][1] = 0.0f;
                        }
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i) {
                            Metas sa, sb;
                            metas(i, T::value_scales, sa, sb);
#pragma unroll
                            for (int g = 0; g < G; ++g)
#pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    high[g][h] = fmaxf(high[g][h], fmaxf(fabsf(x[i0 + i][h] * of_group(sa, g)), fabsf(x[i0 + i][h + 2] * of_group(sb, g))));
                        }
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1)
#pragma unroll
                            for (int g = 0; g < G; ++g)
#pragma unroll
                                for (int h = 0; h < 2; ++h) high[g][h] = fmaxf(high[g][h], __shfl_xor_sync(0xffffffffu, high[g][h], off));
                        __syncwarp();
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            int to[2];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                to[h] = min(min(was[g][h], kQdMost), 254 + kQdRoom - q4_bits(high[g][h]));
                                was[g][h] = to[h] - was[g][h];
                            }
                            if (gq == 0) up[g * 4] = make_float2(q4_power(to[0]), q4_power(to[1]));
                        }
                        if (u > u0 || i0 > 0) {   // (there are no sums before)
#pragma unroll
                            for (int g = 0; g < G; ++g)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const float keep = q4_power(127 + was[g][h]);
#pragma unroll
                                    for (int m = 2 * g; m < 2 * g + 2; ++m) { o[m][h] *= keep; o[m][h + 2] *= keep; }
                                }
                        }
                        __syncwarp();
                    }
                    unsigned most = 0;
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        const float (&p)[4] = x[i0 + i];
                        Metas sa, sb;
                        metas(i, T::value_scales, sa, sb);
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            const float2 f = up[g * 4];
                            const float a = of_group(sa, g), b = of_group(sb, g);
                            float2 w0 = q4_mul2(q4_mul2(make_float2(p[0], p[1]), make_float2(a, a)), f);
                            float2 w1 = q4_mul2(q4_mul2(make_float2(p[2], p[3]), make_float2(b, b)), f);
#pragma unroll
                            for (int n = 0; n < NP; ++n) { y[i][g][n][0] = q4_part(w0.x, w0.y); y[i][g][n][1] = q4_part(w1.x, w1.y); }
                            most = __vimax3_u16x2(most, y[i][g][0][0], y[i][g][0][1]);
                        }
                    }
                    if (update || !__any_sync(0xffffffffu, (most + (0x80008000u - kQdTooLarge)) & 0x80008000u)) break;
                }
                update = false;
                rise[0] = rise[1] = 0;
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    const unsigned char* tile = stage + (i0 + i) * T::bytes;
                    const Words va = *reinterpret_cast<const Words*>(tile + T::values + (gq * 4 + t) * (4 * G)),
                                vb = *reinterpret_cast<const Words*>(tile + T::values + (32 + gq * 4 + t) * (4 * G));
                    const unsigned *wa = reinterpret_cast<const unsigned*>(&va), *wb = reinterpret_cast<const unsigned*>(&vb);
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        unsigned b0[NP], b1[NP], a[4], b[4];
#pragma unroll
                        for (int n = 0; n < NP; ++n) { b0[n] = q4_turn(y[i][g][n][0]); b1[n] = q4_turn(y[i][g][n][1]); }
                        q4_codes<kBf16>(wa[g], a);
                        q4_codes<kBf16>(wb[g], b);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (NP == 1) {
                                gm_mma(o[2 * g + h], {a[2 * h], a[2 * h + 1], b[2 * h], b[2 * h + 1]}, b0[0], b1[0]);
                            } else {   // (the tensor cores cut what they add to a sum: a tile's products are summed on their own)
                                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                                for (int n = NP - 1; n >= 0; --n) gm_mma(c, {a[2 * h], a[2 * h + 1], b[2 * h], b[2 * h + 1]}, b0[n], b1[n]);
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[2 * g + h][e] += c[e];
                            }
                        }
                    }
                }
            }
            ++taken;
            __syncwarp();   // the stage has been read
            filled += fill(from);
        }

        // the warps' sums joined, and out
        float down[G][2];   // 2^-u
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float2 f = up[g * 4];
            down[g][0] = q4_power(254 - q4_bits(f.x));
            down[g][1] = q4_power(254 - q4_bits(f.y));
        }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], off);
#pragma unroll
                for (int g = 0; g < G; ++g) mins[g][h] += __shfl_xor_sync(0xffffffffu, mins[g][h], off);
            }
        if (gq == 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) { s_m[warp][2 * t + h] = top[h]; s_l[warp][2 * t + h] = ok ? l[h] : NAN; }   // (a wait ran out: no result)
        }
#pragma unroll
        for (int m = 0; m < 2 * G; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (2 * t + h >= sum_heads) continue;
                float* to = sums + (warp * sum_heads + 2 * t + h) * M::row + 32 * (m >> 1) + 4 * gq + 2 * (m & 1);
                *reinterpret_cast<float2*>(to) = make_float2(fmaf(o[m][h] * down[m >> 1][h], kCode, mins[m >> 1][h]), fmaf(o[m][h + 2] * down[m >> 1][h], kCode / 16.0f, mins[m >> 1][h]));
            }
        __syncthreads();
        unit += u1 - u0;
        const bool ends = u1 == at.units;
        float* part = P.partials + ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * kQdHeads * (HD + 2);
        for (int i = tid; i < n_heads * HD; i += kQdThreads) {
            const int h = i / HD, d = i % HD;
            float most = kQdLowest, acc = 0.0f, weight = 0.0f;
#pragma unroll
            for (int w = 0; w < kQdWarps; ++w) most = fmaxf(most, s_m[w][h]);
#pragma unroll
            for (int w = 0; w < kQdWarps; ++w) {
                const float keep = q4_exp2(s_m[w][h] - most);
                acc = fmaf(sums[(w * sum_heads + h) * M::row + d], keep, acc);
                weight = fmaf(s_l[w][h], keep, weight);
            }
            if (begins && ends) {
                acc = weight == 0.0f ? 0.0f : acc / weight;
                if (kBf16) reinterpret_cast<__nv_bfloat16*>(P.out)[row0 + i] = __float2bfloat16_rn(acc);
                else reinterpret_cast<float*>(P.out)[row0 + i] = acc;
            } else {
                part[h * (HD + 2) + 2 + d] = acc;
                if (d == 0) { part[h * (HD + 2)] = most; part[h * (HD + 2) + 1] = weight; }
            }
        }
        if (begins && !ends && tid == 0) {
            P.pieces[blockIdx.x] = make_int2(at.b * heads + at.hh, shares.owner(unit + (at.units - u1) - 1));
        }
        __syncthreads();   // the sums have been read
        at.u = u1 - 1;
        if (unit < last) at.skip(P, heads);
    }
    if (!ok) {
        for (int i = taken; i < filled; ++i) bar_wait(bar_at + 8 * (i % kQdStages), (i / kQdStages) & 1);   // nothing may land after the CTA has left
        atomicExch(&g_q4_error, 1);
    }
}

// Items that several CTAs have parts of; a CTA per CTA of the decode, a thread per result.  Bound by latency: eight parts are asked for
// at a time.
constexpr int kQcThreads = 256;

template <int HD, bool kBf16>
__global__ void __launch_bounds__(kQcThreads) q4_combine_kernel(const __grid_constant__ Q4DecodeProblem P) {
    chain_begin();
    const int2 piece = P.pieces[blockIdx.x];
    if (piece.x < 0) return;
    const int heads = P.cache.kv_heads * P.blocks, b = piece.x / heads, hh = piece.x % heads, h0 = (hh % P.blocks) * kQdHeads;
    const int n_heads = min(kQdHeads, P.share - h0), first = blockIdx.x;
    const size_t row0 = ((size_t)b * P.q_heads + hh / P.blocks * P.share + h0) * HD;
    for (int i = threadIdx.x; i < n_heads * HD; i += kQcThreads) {
        const int h = i / HD, d = i % HD;
        float most = kQdLowest, acc = 0.0f, weight = 0.0f;
        for (int c0 = first; c0 <= piece.y; c0 += 8) {
            float m[8], w[8], v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int c = min(c0 + u, piece.y);
                const float* p = P.partials + (((size_t)c * 2 + (c == first ? 1 : 0)) * kQdHeads + h) * (HD + 2);
                m[u] = p[0];
                w[u] = p[1];
                v[u] = p[2 + d];
            }
            float top = most;
#pragma unroll
            for (int u = 0; u < 8; ++u) top = fmaxf(top, m[u]);
            const float keep = q4_exp2(most - top);
            acc *= keep;
            weight *= keep;
            most = top;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (c0 + u > piece.y) continue;
                const float k = q4_exp2(m[u] - top);
                acc = fmaf(v[u], k, acc);
                weight = fmaf(w[u], k, weight);
            }
        }
        acc = weight == 0.0f ? 0.0f : acc / weight;
        if (kBf16) reinterpret_cast<__nv_bfloat16*>(P.out)[row0 + i] = __float2bfloat16_rn(acc);
        else reinterpret_cast<float*>(P.out)[row0 + i] = acc;
    }
}

// CTAs of a decode: what the GPU holds at a time, or a unit each where the tables have room for fewer.
static int q4_decode_ctas(int batch, int max_pages, int page_size, int kv_heads, int share) {
    const long long units = (long long)batch * kv_heads * ((share + kQdHeads - 1) / kQdHeads) * (((long long)max_pages * page_size + kQdUnit - 1) / kQdUnit);
    const int most = num_sms() * kQdCtas;
    return units < most ? (int)units : most;
}
static size_t q4_decode_bytes(int ctas, int head_dim) {
    return ((size_t)ctas * sizeof(int2) + 15) / 16 * 16 + (size_t)ctas * 2 * kQdHeads * (head_dim + 2) * sizeof(float);
}

template <int HD, bool kBf16>
static int launch_q4_decode(const Q4DecodeProblem& P, int ctas, cudaStream_t s) {
    static std::atomic<bool> opted[64];
    OJX_CUDA_TRY(opt_in_smem(reinterpret_cast<const void*>(q4_decode_kernel<HD, kBf16>), QdSmem<HD>::bytes(kQdHeads), opted));
    OJX_CUDA_TRY(launch_chained(q4_decode_kernel<HD, kBf16>, ctas, kQdThreads, QdSmem<HD>::bytes(std::min(P.share, kQdHeads)), s, P));
    OJX_CUDA_TRY(launch_chained(q4_combine_kernel<HD, kBf16>, ctas, kQcThreads, 0, s, P));
    count_launch(2);
    return OJX_OK;
}

int take_q4_error(int* out) {
    int v = 0, zero = 0;
    OJX_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_q4_error, sizeof(int)));
    if (v) OJX_CUDA_TRY(cudaMemcpyToSymbol(g_q4_error, &zero, sizeof(int)));
    *out = v;
    return OJX_OK;
}

}  // namespace ojx

using namespace ojx;

extern "C" {

size_t ojasx_b200_q4kv_decode_workspace(const OjasxQ4Cache* cache, int batch, int max_pages, int io_dtype) {
    if (!cache || batch <= 0 || max_pages <= 0 || cache->page_size <= 0 || cache->kv_heads <= 0 || cache->q_heads <= 0) return 0;
    if (io_dtype != OJX_F32 && io_dtype != OJX_BF16) return 0;
    return q4_decode_bytes(q4_decode_ctas(batch, max_pages, cache->page_size, cache->kv_heads, cache->q_heads / cache->kv_heads), cache->head_dim);
}

int ojasx_b200_q4kv_decode(const OjasxQ4Cache* cache, const void* d_q, void* d_out, const int* d_block_table, int max_pages, const int* d_lengths,
                           int batch, float scale, int io_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = q4_check(cache, d_block_table, max_pages, batch, io_dtype);
    if (rc != OJX_OK) return rc;
    const int kv_heads = cache->kv_heads, q_heads = cache->q_heads, head_dim = cache->head_dim;
    if (!d_q || !d_out || !d_lengths || !q4_aligned(d_q) || !q4_aligned(d_out)) return OJX_ERR_ARG;
    const int share = q_heads / kv_heads, ctas = q4_decode_ctas(batch, max_pages, cache->page_size, kv_heads, share);
    if (!workspace || !q4_aligned(workspace) || workspace_bytes < q4_decode_bytes(ctas, head_dim)) return OJX_ERR_ARG;
    if ((long long)batch * q_heads > 0x7fffffffLL) return OJX_ERR_TOO_LARGE;
    Q4DecodeProblem P{};
    P.cache = q4_cache(cache, d_block_table, max_pages);
    P.q = d_q; P.out = d_out; P.lengths = d_lengths; P.batch = batch; P.q_heads = q_heads; P.share = share;
    P.blocks = (share + kQdHeads - 1) / kQdHeads;
    P.pieces = static_cast<int2*>(workspace);
    P.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + ((size_t)ctas * sizeof(int2) + 15) / 16 * 16);
    P.scale = (scale > 0.0f ? scale : 1.0f / sqrtf((float)head_dim)) * 1.4426950408889634f;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (io_dtype == OJX_BF16) return head_dim == 64 ? launch_q4_decode<64, true>(P, ctas, s) : launch_q4_decode<128, true>(P, ctas, s);
    return head_dim == 64 ? launch_q4_decode<64, false>(P, ctas, s) : launch_q4_decode<128, false>(P, ctas, s);
}

}  // extern "C"
