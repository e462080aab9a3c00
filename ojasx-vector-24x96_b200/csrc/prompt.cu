// Causal attention over whole prompts: packed sequences of different lengths, grouped query heads, softmax(q k^T * scale) v.
//
// The last query of a sequence sees its last key: with n queries and m keys query i sees the keys up to i + m - n, none where that is
// negative.  The rows of a tile are (position, query head of the KV head), so that the heads that share keys share their tiles too.
#include <algorithm>
#include <cmath>

#include "handles.h"
#include "launch.h"
#include "packed.cuh"
#include "tc.cuh"
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
template <int HD>
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
    auto load = [](const void* p, size_t i) { return reinterpret_cast<const float*>(p)[i]; };
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
            reinterpret_cast<float*>(P.out)[to + tx + 16 * j] = o[i][j] * inv;
        }
    }
}

template <int HD>
constexpr size_t prompt_tile_smem() { return sizeof(float) * (3 * 64 * (HD + 4) + 64 * 68); }

template <int HD>
static int launch_prompt_tile(const PromptProblem& P, cudaStream_t s) {
    static std::atomic<bool> opted[64];
    constexpr size_t smem = prompt_tile_smem<HD>();
    OJX_CUDA_TRY(opt_in_smem(reinterpret_cast<const void*>(prompt_tile_kernel<HD>), smem, opted));
    const int per = 64 / P.share;
    // as many tiles as the sequences can have: each has at most one that is not full
    const long long tiles = P.n_rows / per + std::min(P.batch, P.n_rows);
    if (tiles > 0x7fffffffLL) return OJX_ERR_TOO_LARGE;
    OJX_CUDA_TRY(launch_chained(prompt_tile_kernel<HD>, dim3((unsigned)tiles, P.kv_heads), 256, smem, s, P));
    count_launch(1);
    return OJX_OK;
}

// ------------------------------------------------------------------------------------ bf16 on the 5th-generation tensor cores
//
// A CTA has two tiles of 128 rows of one sequence and KV head (rows are (position, head of the KV head)) and walks the keys 128 at a
// time.  Per tile and step: S = Q K^T into tensor memory, one thread per row takes the maximum, the exponentials and their sum, writes
// the weights back over S as bf16, O += P V with P read from tensor memory.  The two tiles take turns: while the tensor cores are at
// one, 128 threads are at the other's exponentials.
//   warps 0..3, 4..7: the rows of the two tiles; warp 8: issues the products; warp 9: the copies of Q, K and V (K and V in a ring);
//   warps 10, 11: none (registers are moved between groups of four warps: 384 * 168 = 64512 are 2 * 128 * 216 + 128 * 64 and some)
// Maxima are left behind: a row's sums are relative to the maximum it had when a score was last more than 2^8 above it, so that
// O is rescaled a few times per row and not once per step (weights up to 2^8 cost nothing in bf16 or in fp32 sums).
constexpr int kPaRows = 128, kPaKeys = 128, kPaThreads = 384;
constexpr float kPaSlack = 8.0f;

template <int HD>
struct PaSmem {
    static constexpr int tile = 128 * HD * 2;                     // 128 rows or keys
    static constexpr int slots = HD == 128 ? 5 : 8;
    static constexpr int ring = 2 * tile, bars = ring + slots * tile;
    static constexpr int bytes = bars + 256 + 1024;               // (swizzled tiles begin on 1024 bytes)
};

static __device__ int g_prompt_error;   // raised when a bounded wait inside a kernel ran out

template <int HD>
__global__ void __launch_bounds__(kPaThreads, 1) prompt_tc_kernel(const __grid_constant__ PromptProblem P, const __grid_constant__ CUtensorMap q_map,
                                                                  const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using M = PaSmem<HD>;
    constexpr int NS = M::slots, C = HD / 64;
    extern __shared__ unsigned char pa_raw[];
    unsigned char* smem = pa_raw + ((1024u - (tc_smem(pa_raw) & 1023u)) & 1023u);
    __shared__ int s_seq, s_part, s_gone, s_odd[2];
    __shared__ unsigned s_tmem;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned base = tc_smem(smem), bars = base + M::bars;
    const unsigned full = bars, empty = bars + 8 * NS, q_full = empty + 8 * NS, s_full = q_full + 16, p_full = s_full + 16, o_full = p_full + 16,
                   checked = o_full + 16, ended = checked + 16, gone = tc_smem(&s_gone);
    const int head = blockIdx.x % P.kv_heads, per = kPaRows / P.share;
    if (tid == 0) {
        for (int i = 0; i < NS; ++i) { tc_bar_init(full + 8 * i, 1); tc_bar_init(empty + 8 * i, 1); }
        for (int i = 0; i < 2; ++i) {
            tc_bar_init(q_full + 8 * i, 1);
            tc_bar_init(s_full + 8 * i, 1);
            tc_bar_init(p_full + 8 * i, 4);
            tc_bar_init(o_full + 8 * i, 1);
            tc_bar_init(checked + 8 * i, 4);
            s_odd[i] = 0;
        }
        tc_bar_init(ended, 1);
        s_gone = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    chain_begin();
    if (warp == 0) {
        // the last parts of a sequence, which see the most keys, first
        int seq = -1, part = 0;
        const bool in = packed_part(P.batch, (int)(gridDim.x / P.kv_heads) - 1 - (int)blockIdx.x / P.kv_heads,
                                    [&](int b) { return (packed_range(P.ends, b, P.n_rows).count + 2 * per - 1) / (2 * per); }, seq, part);
        if (lane == 0) { s_seq = in ? seq : -1; s_part = part; }
    }
    __syncthreads();
    if (s_seq < 0) return;
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tc_smem(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const unsigned tmem = s_tmem;
    const PackedRange rows = packed_range(P.ends, s_seq, P.n_rows), keys = packed_range(P.key_ends, s_seq, P.n_keys);
    const int ahead = keys.count - rows.count;
    int pos[2], live[2], steps[2];   // first position, positions and steps of the tiles
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        pos[i] = (s_part * 2 + i) * per;
        live[i] = max(0, min(per, rows.count - pos[i]));
        steps[i] = live[i] > 0 ? max(0, pos[i] + live[i] + ahead + kPaKeys - 1) / kPaKeys : 0;
    }
    const int n = max(steps[0], steps[1]);
    bool ok = true;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 9 && lane == 0) {
            for (int i = 0; i < 2; ++i) {
                if (!steps[i]) continue;
                tc_bar_expect(q_full + 8 * i, per * P.share * HD * 2);
                for (int c = 0; c < C; ++c) tc_load3(base + i * M::tile + c * (M::tile / C), &q_map, 64 * c, head * P.share, rows.first + pos[i], q_full + 8 * i);
            }
            int s = 0;
            for (; s < 2 * n; ++s) {   // K of step 0, V of step 0, K of step 1, ...
                const int slot = s % NS;
                if (s >= NS && !(ok = bar_wait(empty + 8 * slot, (s / NS - 1) & 1, gone))) break;
                tc_bar_expect(full + 8 * slot, M::tile);
                for (int c = 0; c < C; ++c)
                    tc_load3(base + M::ring + slot * M::tile + c * (M::tile / C), s & 1 ? &v_map : &k_map, 64 * c, head, keys.first + (s >> 1) * kPaKeys, full + 8 * slot);
            }
            if (!ok) {   // nothing may land after the CTA has left
                for (int u = max(0, s - NS); u < s; ++u) bar_wait(full + 8 * (u % NS), (u / NS) & 1);
                for (int i = 0; i < 2; ++i) if (steps[i]) bar_wait(q_full + 8 * i, 0);
            }
        }
        if (warp == 8 && lane == 0) {
            constexpr unsigned iq = tc_idesc<true, false>(kPaKeys), iv = tc_idesc<true, true>(HD);
            auto slot_at = [&](int s) { return base + M::ring + (s % NS) * M::tile; };
            auto wait_slot = [&](int s) { return bar_wait(full + 8 * (s % NS), (s / NS) & 1, gone); };
            auto scores = [&](int i, int j) {
                const unsigned a = base + i * M::tile, b = slot_at(2 * j);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k)
                    tc_mma(tmem + i * 128, tc_desc(a + (k / 4) * (M::tile / C) + (k % 4) * 32), tc_desc(b + (k / 4) * (M::tile / C) + (k % 4) * 32), iq, k > 0);
                tc_commit(s_full + 8 * i);
            };
            if (n > 0) ok = wait_slot(0);
            for (int i = 0; i < 2 && ok; ++i)
                if (steps[i]) {
                    ok = bar_wait(q_full + 8 * i, 0, gone);
                    if (ok) scores(i, 0);
                }
            if (n > 0 && ok) tc_commit(empty);
            for (int j = 0; j < n && ok; ++j) {
                if (j + 1 < n) ok = wait_slot(2 * j + 2);
                if (ok) ok = wait_slot(2 * j + 1);
                for (int i = 0; i < 2 && ok; ++i) {
                    if (j >= steps[i]) continue;
                    if (!(ok = bar_wait(p_full + 8 * i, j & 1, gone))) break;
                    tc_after();
                    if (*reinterpret_cast<volatile int*>(&s_odd[i]) != j + 1) {   // (else the rows have added their products themselves)
                        const unsigned b = slot_at(2 * j + 1);
#pragma unroll
                        for (int k = 0; k < kPaKeys / 16; ++k)
                            tc_mma_ts(tmem + 256 + i * 128, tmem + i * 128 + k * 8, tc_desc(b + k * 2048, M::tile / C), iv, j > 0 || k > 0);
                    }
                    if (j + 1 < steps[i]) scores(i, j + 1);   // (in order: its commit says that O is up to date, too)
                    else tc_commit(o_full + 8 * i);
                }
                if (!ok) break;
                tc_commit(empty + 8 * ((2 * j + 1) % NS));
                if (j + 1 < n) tc_commit(empty + 8 * ((2 * j + 2) % NS));
            }
            if (!ok) {
                tc_commit(ended);
                bar_wait(ended, 0);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int i = warp >> 2, row = tid & 127;   // the row's lane of tensor memory is its place in the tile
        const int at = min(row, max(live[i] * P.share - 1, 0)), last = pos[i] + at / P.share + ahead;   // last key that the row sees
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16, st = tmem + i * 128 + lanes, ot = tmem + 256 + i * 128 + lanes;
        const float scale = P.scale * 1.4426950408889634f;
        float top = 0.0f, sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        int checks = 0;
        auto wait = [&](unsigned bar, unsigned parity) { return (bool)__all_sync(0xffffffffu, bar_wait(bar, parity, gone)); };
        auto rescale = [&](float by) {   // the warp's rows of O
            for (int c = 0; c < HD; c += 32) {
                unsigned o[32];
                tc_ld32(ot + c, o);
                tc_wait_ld();
                tc_pin32(o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * by);
                tc_st32(ot + c, o);
            }
        };
        for (int j = 0; j < steps[i]; ++j) {
            if (!(ok = wait(s_full + 8 * i, j & 1))) break;
            tc_after();
            unsigned s[128];
#pragma unroll
            for (int c = 0; c < 4; ++c) tc_ld32(st + 32 * c, s + 32 * c);
            tc_wait_ld();
#pragma unroll
            for (int c = 0; c < 4; ++c) tc_pin32(s + 32 * c);
            const bool masked = (j + 1) * kPaKeys - 1 > pos[i] + ahead;   // some row does not see all of these keys
            if (masked) {
                const int see = last - j * kPaKeys;
#pragma unroll
                for (int e = 0; e < 128; ++e) s[e] = e > see ? 0xff800000u : s[e];
            }
            float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 128; e += 4)
#pragma unroll
                for (int u = 0; u < 4; ++u) m[u] = fmaxf(m[u], __uint_as_float(s[e + u]));
            const float now = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
            const bool up = (now - top) * scale > kPaSlack;   // (by the row's own scores: its result does not depend on its neighbours)
            if (j == 0) {
                top = now;
            } else if (__any_sync(0xffffffffu, up)) {
                const float to = up ? now : top, by = up ? exp2f((top - now) * scale) : 1.0f;
                rescale(by);
#pragma unroll
                for (int u = 0; u < 4; ++u) sum[u] *= by;
                top = to;
            }
            const float off = top == -INFINITY ? 0.0f : top * scale;   // (a row that has seen nothing: its weights are exp(-inf))
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                unsigned w[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    float a = fmaf(__uint_as_float(s[64 * c + 2 * e]), scale, -off), b = fmaf(__uint_as_float(s[64 * c + 2 * e + 1]), scale, -off);
                    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
                    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
                    sum[e & 1] += a;
                    sum[2 + (e & 1)] += b;
                    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
                    w[e] = *reinterpret_cast<const unsigned*>(&h);
                }
                tc_st32(st + 32 * c, w);
            }
            if (masked) {
                // A weight of zero times an infinity is a NaN, and the products take all keys of the step.  Where a value among them is
                // not finite (padding behind a sequence, another sequence's rows) each row adds the values that it sees itself.
                if (!(ok = wait(full + 8 * ((2 * j + 1) % NS), ((2 * j + 1) / NS) & 1))) break;
                const unsigned char* v = smem + M::ring + ((2 * j + 1) % NS) * M::tile;
                unsigned odd = 0;
                for (int e = row; e < M::tile / 16; e += 128) {
                    const uint4 x = reinterpret_cast<const uint4*>(v)[e];   // an exponent of all ones carries into the sign's place
                    odd |= (((x.x & 0x7f807f80u) + 0x00800080u) | ((x.y & 0x7f807f80u) + 0x00800080u) | ((x.z & 0x7f807f80u) + 0x00800080u) |
                            ((x.w & 0x7f807f80u) + 0x00800080u)) & 0x80008000u;
                }
                odd = __reduce_or_sync(0xffffffffu, odd);
                if (lane == 0) {
                    if (odd) *reinterpret_cast<volatile int*>(&s_odd[i]) = j + 1;
                    tc_bar_arrive(checked + 8 * i);
                }
                if (!(ok = wait(checked + 8 * i, checks++ & 1))) break;
                if (*reinterpret_cast<volatile int*>(&s_odd[i]) == j + 1) {
                    tc_wait_st();
                    const int see = min(last - j * kPaKeys, kPaKeys - 1);
                    for (int c = 0; c < HD; c += 32) {
                        float o[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0.0f;
                        for (int k = 0; k < kPaKeys; ++k) {
                            unsigned w = tc_ld1(st + (k >> 1));
                            tc_wait_ld();
                            asm volatile("" : "+r"(w));
                            if (k <= see) {
                                const float p = __uint_as_float(k & 1 ? w & 0xffff0000u : w << 16);
                                const unsigned char* line = v + (c / 64) * (M::tile / C) + k * 128;
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const uint4 x = *reinterpret_cast<const uint4*>(line + (((c % 64) / 8 + e) ^ (k & 7)) * 16);
                                    const unsigned xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                                    for (int h = 0; h < 4; ++h) {
                                        o[8 * e + 2 * h] = fmaf(p, __uint_as_float(xs[h] << 16), o[8 * e + 2 * h]);
                                        o[8 * e + 2 * h + 1] = fmaf(p, __uint_as_float(xs[h] & 0xffff0000u), o[8 * e + 2 * h + 1]);
                                    }
                                }
                            }
                            __syncwarp();
                        }
                        unsigned r[32];
                        if (j > 0) {
                            tc_ld32(ot + c, r);
                            tc_wait_ld();
                            tc_pin32(r);
                        }
#pragma unroll
                        for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(o[e] + (j > 0 ? __uint_as_float(r[e]) : 0.0f));
                        tc_st32(ot + c, r);
                    }
                }
            }
            tc_wait_st();
            tc_before();
            __syncwarp();
            if (lane == 0) tc_bar_arrive(p_full + 8 * i);
        }
        if (ok && live[i] > 0) {
            const int position = row / P.share;
            const bool out = position < live[i] && row < per * P.share;
            const float total = (sum[0] + sum[1]) + (sum[2] + sum[3]), inv = total == 0.0f ? 0.0f : 1.0f / total;
            uint4* to = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(P.out) +
                                                 ((size_t)(rows.first + pos[i] + (out ? position : 0)) * P.q_heads + head * P.share + (out ? row % P.share : 0)) * HD);
            if (steps[i]) {
                ok = wait(o_full + 8 * i, 0);
                tc_after();
            }
            for (int c = 0; c < HD && ok; c += 32) {
                unsigned o[32];
                if (steps[i]) {
                    tc_ld32(ot + c, o);
                    tc_wait_ld();
                    tc_pin32(o);
                }
                if (!out) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    unsigned w[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        // (a row whose weights are all zero has a sum of zero: nothing it saw, or scores of -inf)
                        const float x = steps[i] ? __uint_as_float(o[8 * e + 2 * h]) * inv : 0.0f, y = steps[i] ? __uint_as_float(o[8 * e + 2 * h + 1]) * inv : 0.0f;
                        const __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
                        w[h] = *reinterpret_cast<const unsigned*>(&p);
                    }
                    to[c / 8 + e] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
    }
    if (!ok) atomicExch(&g_prompt_error, 1);
    tc_before();
    __syncthreads();
    if (warp == 8) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <int HD>
static int launch_prompt_tc(const PromptProblem& P, cudaStream_t s) {
    static std::atomic<bool> opted[64];
    constexpr int smem = PaSmem<HD>::bytes;
    OJX_CUDA_TRY(opt_in_smem(reinterpret_cast<const void*>(prompt_tc_kernel<HD>), smem, opted));
    const int per = kPaRows / P.share;
    const long long parts = P.n_rows / (2 * per) + std::min(P.batch, P.n_rows);
    if (parts * P.kv_heads > 0x7fffffffLL) return OJX_ERR_TOO_LARGE;
    CUtensorMap q, k, v;
    const bool none = P.n_keys == 0;
    if (!tc_map3(&q, true, P.q, HD, P.q_heads, P.n_rows, P.q_head, P.q_row, 64, P.share, per) ||
        !tc_map3(&k, true, none ? P.q : P.k, HD, none ? 1 : P.kv_heads, none ? 1 : P.n_keys, none ? HD : P.k_head, none ? HD : P.k_row, 64, 1, kPaKeys) ||
        !tc_map3(&v, true, none ? P.q : P.v, HD, none ? 1 : P.kv_heads, none ? 1 : P.n_keys, none ? HD : P.v_head, none ? HD : P.v_row, 64, 1, kPaKeys)) {
        set_last_error_msg("prompt attention: the tensors' strides do not make a tensor map");
        return OJX_ERR_ARG;
    }
    OJX_CUDA_TRY(launch_chained(prompt_tc_kernel<HD>, dim3((unsigned)(parts * P.kv_heads)), kPaThreads, smem, s, P, q, k, v));
    count_launch(1);
    return OJX_OK;
}

int take_prompt_error(int* out) {
    int v = 0, zero = 0;
    OJX_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_prompt_error, sizeof(int)));
    if (v) OJX_CUDA_TRY(cudaMemcpyToSymbol(g_prompt_error, &zero, sizeof(int)));
    *out = v;
    return OJX_OK;
}

}  // namespace ojx

using namespace ojx;

extern "C" int ojasx_b200_prompt_attention(const void* d_q, long long q_row, long long q_head, const void* d_k, long long k_row,
                                           long long k_head, const void* d_v, long long v_row, long long v_head, void* d_out,
                                           const int* d_ends, const int* d_key_ends, int batch, int n_rows, int n_keys, int q_heads,
                                           int kv_heads, int head_dim, float scale, int io_dtype, void* stream) {
    if (!d_q || (n_keys > 0 && (!d_k || !d_v)) || !d_out || !d_ends || !d_key_ends || batch <= 0 || n_rows < 0 || n_keys < 0 || kv_heads <= 0 || q_heads <= 0 ||
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
    if (io_dtype == OJX_BF16) return head_dim == 64 ? launch_prompt_tc<64>(P, s) : launch_prompt_tc<128>(P, s);
    return head_dim == 64 ? launch_prompt_tile<64>(P, s) : launch_prompt_tile<128>(P, s);
}
