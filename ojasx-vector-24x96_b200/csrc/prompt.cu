// Causal attention over whole prompts: packed sequences of different lengths, grouped query heads, softmax(q k^T * scale) v.
//
// The last query of a sequence sees its last key: with n queries and m keys query i sees the keys up to i + m - n, none where that is
// negative.  The rows of a tile are (position, query head of the KV head), so that the heads that share keys share their tiles too.
#include <algorithm>
#include <cmath>

#include "gather_mma.cuh"
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
    const unsigned char* none;                     // [n_keys, up to a multiple of 16] or null: not zero for keys that nobody sees
    int batch, n_rows, n_keys, q_heads, kv_heads, share;
    float scale;
};

// ------------------------------------------------------------------------------------ bf16 on the 5th-generation tensor cores
//
// A CTA has two tiles of 128 rows of one sequence and KV head (rows are (position, head of the KV head)) and walks the keys 64 at a
// time.  Per tile and step: S = Q K^T into tensor memory, one thread per row takes the maximum, the exponentials and their sum, writes
// the weights back over S as bf16, O += P V with P read from tensor memory.  A tile has S twice: the products of a step are made while
// the row's threads are at the step before, and those of the tiles go on in turn.  (With one S of 128 keys a tile, whose products wait
// for its weights: 139 against 129 us for packed prompts, 306 against 299 for 1024 positions behind 7000.)
//   warps 0..3, 4..7: the rows of the two tiles; warp 8: issues the products; warp 9: the copies of Q, K and V (K and V in a ring);
//   warp 11: what to do next, so that a CTA's copies and products for one part of the prompts begin while it is at the last results of
//   another (packed prompts 171 us without and 154 with it, when they were that slow); warp 10: none.  Registers move between groups of four warps: 384 * 168 are
//   2 * 128 * 200 + 128 * 96 and some.
// Maxima are left behind: a row's sums are relative to the maximum it had when a score was last more than 2^8 above it, so that
// O is rescaled a few times per row and not once per step (weights up to 2^8 cost nothing in bf16 or in fp32 sums).
// Weights are rounded to bf16, below the rounding of the result.  Bound by the chain from a product through maximum and exponentials to the
// next one (tensor pipe 56 %, exponentials 56 % of their pipe): 8192 positions of 32 query heads and 8 KV heads of 128 take 497 to 523 us by
// CUDA events, call after call, on several GPUs whose power limit sets their clocks (1.66 GHz), 1050 to 1110 TFLOP/s.  Products issued
// by a warp as a whole with an elected lane, and not by one lane in a branch: 610 -> 562.
constexpr int kPaRows = 128, kPaKeys = 64, kPaThreads = 384;
constexpr float kPaSlack = 8.0f;
constexpr long long kPaPartClocks = 1LL << 35;   // 18 s: a step of 64 keys takes a microsecond, and 10^9 keys do not fit into the memory

template <int HD>
struct PaSmem {
    static constexpr int tile = 128 * HD * 2, part = kPaKeys * HD * 2;     // of Q, and of K or V
    static constexpr int slots = 10;
    static constexpr int ring = 2 * tile, bars = ring + slots * part;
    static constexpr int bytes = bars + 384 + 1024;               // (swizzled tiles begin on 1024 bytes)
};

// Two fp32 numbers in one register pair: half the instructions for what is done to all scores.
__device__ __forceinline__ unsigned long long pa_pair(float a, float b) { return (unsigned long long)__float_as_uint(b) << 32 | __float_as_uint(a); }
__device__ __forceinline__ unsigned long long pa_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long pa_add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ unsigned long long pa_mul2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float pa_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ unsigned long long pa_exp2(unsigned long long x) {
    float a = __uint_as_float((unsigned)x), b = __uint_as_float((unsigned)(x >> 32));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    return pa_pair(a, b);
}
static __device__ int g_prompt_error;   // raised when a bounded wait inside a kernel ran out

// ---- Few rows over many keys: the CTAs of a cluster have the same rows and a share of the keys each.  Their sums go into their own shared
// memory (copies and products are done by then), and after a cluster barrier every CTA joins the sums of some of the rows, in the
// shares' order, and writes them.
__device__ __forceinline__ void pa_cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int pa_cluster_rank() {
    unsigned rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    return (int)rank;
}
__device__ __forceinline__ int pa_cluster_size() {
    unsigned size;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    return (int)size;
}
__device__ __forceinline__ void pa_rows_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }   // the rows' threads of both tiles
// Steps of the keys that this CTA has of the n of its rows.
struct PaShare {
    int first, count;
    __device__ __forceinline__ PaShare(int n, int rank, int size)
        : first((int)((long long)n * rank / size)), count((int)((long long)n * (rank + 1) / size) - first) {}
};
// A row's sums: its products, and the reference of its weights (in powers of two) and their sum behind those of all rows.
template <int HD> struct PaParts {
    static constexpr int row = HD + 4, heads = 256 * row * 4, bytes = heads + 256 * 8;
};
template <int HD, bool kBf16>
__device__ __forceinline__ void pa_join(const PromptProblem& P, const unsigned char* parts, int first_row, int head, int per, int live0, int live1, float unit) {
    const int rank = pa_cluster_rank(), size = pa_cluster_size(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned at = static_cast<unsigned>(__cvta_generic_to_shared(parts));
    constexpr int W = HD / 32;   // values of a lane
    auto map = [](unsigned local, int z) {
        unsigned far;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(local), "r"(z));
        return far;
    };
    for (int r = rank + size * warp; r < 2 * kPaRows; r += size * 8) {
        const int tile = r / kPaRows, row = r % kPaRows, position = row / P.share;
        if (row >= per * P.share || position >= (tile ? live1 : live0)) continue;
        float top = -INFINITY, sum = 0.0f;
        if (lane < size) asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(top), "=f"(sum) : "r"(map(at + PaParts<HD>::heads + r * 8, lane)) : "memory");
        float most = top;
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
        const float keep = top == -INFINITY ? 0.0f : exp2f(top - most);   // (a share without keys for the row)
        float x[W], total = 0.0f;
#pragma unroll
        for (int e = 0; e < W; ++e) x[e] = 0.0f;
        for (int z = 0; z < size; ++z) {
            const float k = __shfl_sync(0xffffffffu, keep, z);
            const unsigned from = map(at + (r * PaParts<HD>::row + lane * W) * 4, z);
            float y[W];
            if constexpr (W == 4) asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(y[0]), "=f"(y[1]), "=f"(y[2]), "=f"(y[3]) : "r"(from) : "memory");
            else asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(y[0]), "=f"(y[1]) : "r"(from) : "memory");
#pragma unroll
            for (int e = 0; e < W; ++e) x[e] = fmaf(y[e], k, x[e]);
            total = fmaf(__shfl_sync(0xffffffffu, sum, z), k, total);
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / (total * unit);
        const size_t to = ((size_t)(first_row + tile * per + position) * P.q_heads + head * P.share + row % P.share) * HD + lane * W;
        if constexpr (kBf16) {
            unsigned w[W / 2];
#pragma unroll
            for (int e = 0; e < W / 2; ++e) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * e] * inv, x[2 * e + 1] * inv);
                w[e] = *reinterpret_cast<const unsigned*>(&h);
            }
            unsigned* out = reinterpret_cast<unsigned*>(reinterpret_cast<__nv_bfloat16*>(P.out) + to);
#pragma unroll
            for (int e = 0; e < W / 2; ++e) out[e] = w[e];
        } else {
            float* out = reinterpret_cast<float*>(P.out) + to;
#pragma unroll
            for (int e = 0; e < W; ++e) out[e] = x[e] * inv;
        }
    }
}

// kHoles: P.none may name keys.  In a kernel of its own, since the test of it in every step costs the others 2 to 6 %.
template <int HD, bool kShares, bool kHoles>
__global__ void __launch_bounds__(kPaThreads, 1) prompt_tc_kernel(const __grid_constant__ PromptProblem P, const __grid_constant__ CUtensorMap q_map,
                                                                  const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using M = PaSmem<HD>;
    constexpr int NS = M::slots, C = HD / 64;
    extern __shared__ unsigned char pa_raw[];
    unsigned char* smem = pa_raw + ((1024u - (tc_smem(pa_raw) & 1023u)) & 1023u);
    __shared__ int s_gone, s_odd[2][2];   // s_odd: of either S of a tile, since its rows may be a step ahead of the products
    __shared__ unsigned s_tmem;
    __shared__ __align__(16) int s_item[3][8];   // two in turn, and one that was found when a wait had run out
    __shared__ __align__(16) int s_stolen[4];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;   // (the same for a warp, as the compiler sees)
    const unsigned base = tc_smem(smem), bars = base + M::bars;
    const unsigned full = bars, empty = bars + 8 * NS, q_full = empty + 8 * NS, s_full = q_full + 16, p_full = s_full + 32, o_full = p_full + 32,
                   checked = o_full + 32, q_empty = checked + 16, item_full = q_empty + 16, item_empty = item_full + 16,
                   want = item_empty + 16, steal = want + 8, ended = steal + 8, gone = tc_smem(&s_gone);
    const int per = kPaRows / P.share;
    if (tid == 0) {
        for (int i = 0; i < NS; ++i) { tc_bar_init(full + 8 * i, 1); tc_bar_init(empty + 8 * i, 1); }
        for (int i = 0; i < 2; ++i) {
            tc_bar_init(q_full + 8 * i, 1);
            tc_bar_init(s_full + 16 * i, 1);
            tc_bar_init(s_full + 16 * i + 8, 1);
            tc_bar_init(p_full + 16 * i, 4);
            tc_bar_init(p_full + 16 * i + 8, 4);
            tc_bar_init(o_full + 16 * i, 1);
            tc_bar_init(o_full + 16 * i + 8, 1);
            tc_bar_init(checked + 8 * i, 4);
            tc_bar_init(q_empty + 8 * i, 1);
            tc_bar_init(item_full + 8 * i, 1);
            tc_bar_init(item_empty + 8 * i, 10);
            s_odd[i][0] = s_odd[i][1] = 0;
            s_item[i][0] = s_item[2][0] = -1;
        }
        tc_bar_init(want, 1);
        tc_bar_init(steal, 1);
        tc_bar_init(ended, 1);
        s_gone = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    chain_begin();
    __syncthreads();
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tc_smem(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const unsigned tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    bool ok = true;
    auto wait = [&](unsigned bar, unsigned parity) { return tc_wait(bar, parity, gone); };
    // For the end of what another warp does with all keys of a part: its own waits end soon, and this one with them.
    auto wait_part = [&](unsigned bar, unsigned parity) { return tc_wait(bar, parity, gone, kPaPartClocks); };
    // Item `number` of the CTA, as warp 11 has put it down; false behind the last one (or where a wait ran out).
    struct { int row, key, ahead, head, pos[2], live[2], steps[2], n; } item;   // first row and key; first position, positions and steps of the tiles
    auto take = [&](int number) {
        if (!(ok = wait_part(item_full + 8 * (number & 1), (number >> 1) & 1))) return false;
        const int4 a = *reinterpret_cast<const int4*>(s_item[number & 1]), b = *reinterpret_cast<const int4*>(s_item[number & 1] + 4);
        __syncwarp();
        if (lane == 0) tc_bar_arrive(item_empty + 8 * (number & 1));
        item.row = a.x; item.key = a.y; item.ahead = a.z; item.head = a.w;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            item.pos[i] = b.x + i * per;
            item.live[i] = i ? b.z : b.y;
            item.steps[i] = item.live[i] > 0 ? max(0, item.pos[i] + item.live[i] + item.ahead + kPaKeys - 1) / kPaKeys : 0;
            if (kShares) item.steps[i] = min(item.steps[i], b.w);
        }
        item.n = max(item.steps[0], item.steps[1]);
        return item.row >= 0;
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        if (warp == 11) {
            // Work: the CTA's own part of the prompts, and then those of CTAs that have not begun, asked for when the copies of the last one
            // have been issued.  The last parts of a sequence, which see the most keys, come first.
            const int size = kShares ? pa_cluster_size() : 1, rank = kShares ? pa_cluster_rank() : 0;
            int cta = kShares ? (int)blockIdx.x / size : (int)blockIdx.x, number = 0;
            unsigned asked = 0;
            bool room = true;   // false: a wait ran out
            for (;;) {
                int seq = -1, part = 0;
                const bool in = cta >= 0 && packed_part(P.batch, (int)((kShares ? gridDim.x / size : gridDim.x) / P.kv_heads) - 1 - cta / P.kv_heads,
                                                        [&](int b) { return (packed_range(P.ends, b, P.n_rows).count + 2 * per - 1) / (2 * per); }, seq, part);
                if (in || cta < 0) {
                    room = room && (number < 2 || wait(item_empty + 8 * (number & 1), ((number >> 1) - 1) & 1));
                    if (lane == 0) {
                        int4 a = make_int4(-1, 0, 0, 0), b = make_int4(0, 0, 0, 0);
                        if (in) {
                            const PackedRange rows = packed_range(P.ends, seq, P.n_rows), keys = packed_range(P.key_ends, seq, P.n_keys);
                            const int pos = part * 2 * per;
                            a = make_int4(rows.first, keys.first, keys.count - rows.count, cta % P.kv_heads);
                            b = make_int4(pos, min(per, rows.count - pos), max(0, min(per, rows.count - pos - per)), 0);
                            if (kShares) {   // the keys begin with the first of this CTA's
                                const PaShare share(max(0, pos + b.y + b.z + a.z + kPaKeys - 1) / kPaKeys, rank, size);
                                a.y += share.first * kPaKeys;
                                a.z -= share.first * kPaKeys;
                                b.w = share.count;
                            }
                        }
                        int* const to = s_item[room ? number & 1 : 2];
                        *reinterpret_cast<int4*>(to) = a;
                        *reinterpret_cast<int4*>(to + 4) = b;
                        if (room) tc_bar_arrive(item_full + 8 * (number & 1));
                    }
                    __syncwarp();
                    if (!(ok = room) || cta < 0 || !(ok = wait_part(want, number & 1))) break;
                    ++number;
                }
                if (!(ok = room)) break;
                if constexpr (kShares) {   // (the CTAs of a cluster stay at one part)
                    cta = -1;
                    continue;
                }
                if (lane == 0) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    tc_bar_expect(steal, 16);
                    tc_steal(tc_smem(s_stolen), steal);
                }
                __syncwarp();
                room = wait(steal, asked & 1);
                if (!room && !__all_sync(0xffffffffu, bar_wait(steal, asked & 1))) {   // nothing may land after the CTA has left
                    ok = false;
                    break;
                }
                ++asked;
                cta = tc_stolen(tc_smem(s_stolen));
                __syncwarp();
            }
        }
        if (warp == 9) {
            TcRing<NS> ring{0, 1};   // (of the phases that free the slots: none is waited for the first time round)
            int quota = NS, loads[2] = {0, 0};
            for (int number = 0; take(number); ++number) {
                auto stage = [&](bool value, int j) {
                    if (quota > 0) --quota;
                    else if (!(ok = wait(empty + 8 * ring.slot, ring.parity))) return;
                    if (lane == 0) {
                        tc_bar_expect(full + 8 * ring.slot, M::part);
                        for (int c = 0; c < C; ++c)
                            tc_load3(base + M::ring + ring.slot * M::part + c * (M::part / C), value ? &v_map : &k_map, 64 * c, item.head, item.key + j * kPaKeys,
                                     full + 8 * ring.slot);
                    }
                    __syncwarp();
                    ring.next(1);
                };
                for (int j = 0; j < item.n && ok; ++j) {   // K of step 0, Q, V of step 0, K of step 1, ...
                    stage(false, j);
                    for (int i = 0; i < 2 && j == 0 && ok; ++i) {
                        if (!item.steps[i]) continue;
                        if (loads[i] > 0 && !(ok = wait(q_empty + 8 * i, (loads[i] - 1) & 1))) break;
                        ++loads[i];
                        if (lane == 0) {
                            tc_bar_expect(q_full + 8 * i, per * P.share * HD * 2);
                            for (int c = 0; c < C; ++c)
                                tc_load3(base + i * M::tile + c * (M::tile / C), &q_map, 64 * c, item.head * P.share, item.row + item.pos[i], q_full + 8 * i);
                        }
                        __syncwarp();
                    }
                    if (ok) stage(true, j);
                }
                if (!ok) break;
                if (lane == 0) tc_bar_arrive(want);
            }
            if (!ok) {   // nothing may land after the CTA has left
                for (int u = 0; u < NS; ++u) { bar_wait(full + 8 * u, 0); bar_wait(full + 8 * u, 1); }
                for (int i = 0; i < 2; ++i) { bar_wait(q_full + 8 * i, 0); bar_wait(q_full + 8 * i, 1); }
            }
        }
        if (warp == 8) {
            const unsigned lead = tc_lead();
            constexpr unsigned iq = tc_idesc<true, false>(kPaKeys), iv = tc_idesc<true, true>(HD);
            const unsigned long long ring_k = tc_desc(base + M::ring), ring_v = tc_desc(base + M::ring, M::part / C), q_desc = tc_desc(base);
            auto scores = [&](int i, int half, int slot) {
                const unsigned long long a = tc_at(q_desc, i * M::tile), b = tc_at(ring_k, slot * M::part);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k)
                    tc_mma(lead, tmem + i * 128 + half * 64, tc_at(a, (k / 4) * (M::tile / C) + (k % 4) * 32), tc_at(b, (k / 4) * (M::part / C) + (k % 4) * 32), iq, k > 0);
                tc_commit(lead, s_full + 16 * i + 8 * half);
            };
            TcRing<NS> kr{0, 0}, vr{1, 0};
            unsigned done[2] = {0, 0}, halves[2] = {0, 0}, items[2] = {0, 0};   // steps of the tiles so far, those with either S (a bit each), and items
            for (int number = 0; take(number); ++number) {
                const int n = item.n;
#pragma unroll
                for (int j = 0; j < 2; ++j) {   // the scores of two steps ahead
                    if (j >= n || !ok) continue;
                    ok = wait(full + 8 * kr.slot, kr.parity);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (j >= item.steps[i] || !ok) continue;
                        if (j == 0) {
                            if (!(ok = wait(q_full + 8 * i, items[i]++ & 1))) continue;
                            tc_after();
                        }
                        scores(i, j, kr.slot);
                        if (j + 1 == item.steps[i]) tc_commit(lead, q_empty + 8 * i);
                    }
                    tc_commit(lead, empty + 8 * kr.slot);
                    kr.next(2);
                }
                for (int j = 0; j < n && ok; ++j) {
                    bool loaded = false;   // K of the step after the next
                    ok = wait(full + 8 * vr.slot, vr.parity);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (j >= item.steps[i] || !ok) continue;
                        const unsigned step = ++done[i];
                        if (!(ok = wait(p_full + 16 * i + 8 * (j & 1), halves[i] >> (j & 1) & 1))) continue;
                        halves[i] ^= 1u << (j & 1);
                        tc_after();
                        // (values that are not finite behind what is seen: the rows have added their products themselves)
                        if (!((j + 1) * kPaKeys - 1 > item.pos[i] + item.ahead && *reinterpret_cast<volatile int*>(&s_odd[i][j & 1]) == (int)step)) {
                            const unsigned long long b = tc_at(ring_v, vr.slot * M::part);
#pragma unroll
                            for (int k = 0; k < kPaKeys / 16; ++k)
                                tc_mma_ts(lead, tmem + 256 + i * 128, tmem + i * 128 + (j & 1) * 64 + k * 8, tc_at(b, k * 2048), iv, j > 0 || k > 0);
                        }
                        tc_commit(lead, o_full + 16 * i + 8 * (j & 1));
                        if (j + 2 < item.steps[i]) {
                            if (!loaded && !(ok = wait(full + 8 * kr.slot, kr.parity))) continue;
                            loaded = true;
                            scores(i, j & 1, kr.slot);   // (behind the products that read the weights in their place)
                            if (j + 3 == item.steps[i]) tc_commit(lead, q_empty + 8 * i);
                        }
                    }
                    if (!ok) break;
                    tc_commit(lead, empty + 8 * vr.slot);
                    vr.next(2);
                    if (j + 2 < n) {
                        tc_commit(lead, empty + 8 * kr.slot);
                        kr.next(2);
                    }
                }
                if (!ok) break;
            }
            if (!ok) {
                tc_commit(lead, ended);
                bar_wait(ended, 0);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int i = warp >> 2, row = tid & 127;   // the row's lane of tensor memory is its place in the tile
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16, st = tmem + i * 128 + lanes, ot = tmem + 256 + i * 128 + lanes;
        const float scale = P.scale * 1.4426950408889634f;
        int checks = 0;
        bool met = false;   // (of the tiles' threads)
        unsigned done = 0, halves = 0, before = 0;   // steps of the tile so far, those with either S (a bit each), and the CTA's
        // The products of step j, whose scores were the last that the row has waited for, or those before them.  (Either S has a barrier for its
        // products: the scores of a step tell that the products of the second step before are done, not those of the one before.)
        auto products = [&](int j) { return wait(o_full + 16 * i + 8 * (j & 1), (halves >> (j & 1) & 1) ^ 1); };
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
        for (int number = 0;; ++number) {
            // (read again where it is needed: registers are short between)
            const volatile int* const what = s_item[number & 1];
            if (!(ok = wait_part(item_full + 8 * (number & 1), (number >> 1) & 1)) || what[0] < 0) break;
            int steps, last, first, n;   // of the tile; last key that the row sees, and that the tile's first row sees; steps of both tiles
            {
                const int pos = what[4] + i * per, live = what[5 + i], ahead = what[2], end = pos + live + ahead;
                steps = live > 0 ? max(0, end + kPaKeys - 1) / kPaKeys : 0;
                first = pos + ahead;
                last = first + min(row, max(live * P.share - 1, 0)) / P.share;
                const int other = what[6 - i], to = what[4] + (1 - i) * per + other + ahead;
                n = max(steps, other > 0 ? max(0, to + kPaKeys - 1) / kPaKeys : 0);
                if (kShares) steps = min(steps, what[7]);   // (n is for the parts behind this one, and there are none)
            }
            bool holes = false;   // keys among the tile's that nobody sees (or some of the 15 before and behind them, as they are read)
            if constexpr (kHoles) {
                unsigned some = 0;
                const long long to = min((long long)what[1] + steps * kPaKeys, (long long)P.n_keys);
                for (long long key = (what[1] & ~15) + 16 * lane; key < to; key += 512) {
                    const uint4 x = *reinterpret_cast<const uint4*>(P.none + key);
                    some |= x.x | x.y | x.z | x.w;
                }
                holes = __any_sync(0xffffffffu, some != 0);
            }
            float top = 0.0f;
            unsigned long long sum2[2] = {0, 0};
            for (int j = 0; j < steps; ++j) {
                const unsigned step = ++done;
                const unsigned at = st + (j & 1) * 64;
                if (!(ok = wait(s_full + 16 * i + 8 * (j & 1), halves >> (j & 1) & 1))) break;
                halves ^= 1u << (j & 1);
                tc_after();
                unsigned s[64];
                tc_ld32(at, s);
                tc_ld32(at + 32, s + 32);
                tc_wait_ld();
                tc_pin32(s);
                tc_pin32(s + 32);
                const bool masked = (j + 1) * kPaKeys - 1 > first;   // some row does not see all of these keys
                if (kHoles ? masked || holes : masked) {
                    const int see = masked ? last - j * kPaKeys : kPaKeys;
                    if constexpr (kHoles) {
                        const long long key = (long long)what[1] + j * kPaKeys + lane;
                        unsigned long long not_seen = see < 0 ? ~0ull : see < 63 ? ~0ull << (see + 1) : 0ull;
                        if (holes)
                            not_seen |= __ballot_sync(0xffffffffu, key < P.n_keys && P.none[key]) |
                                        (unsigned long long)__ballot_sync(0xffffffffu, key + 32 < P.n_keys && P.none[key + 32]) << 32;
#pragma unroll
                        for (int e = 0; e < 64; ++e) s[e] = not_seen >> e & 1u ? 0xff800000u : s[e];
                    } else {
#pragma unroll
                        for (int e = 0; e < 64; ++e) s[e] = e > see ? 0xff800000u : s[e];
                    }
                }
                float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 64; e += 8)
#pragma unroll
                    for (int u = 0; u < 4; ++u) m[u] = pa_max3(m[u], __uint_as_float(s[e + 2 * u]), __uint_as_float(s[e + 2 * u + 1]));
                const float now = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
                const bool up = (now - top) * scale > kPaSlack;   // (by the row's own scores: its result does not depend on its neighbours)
                if (j == 0) {
                    top = now;
                } else if (__any_sync(0xffffffffu, up)) {
                    if (!(ok = products(j - 1))) break;
                    tc_after();
                    const float to = up ? now : top, by = up ? exp2f((top - now) * scale) : 1.0f;
                    rescale(by);
                    sum2[0] = pa_mul2(sum2[0], pa_pair(by, by));
                    sum2[1] = pa_mul2(sum2[1], pa_pair(by, by));
                    top = to;
                }
                const float off = top == -INFINITY ? 0.0f : top * scale;   // (a row that has seen nothing: its weights are exp(-inf))
                const unsigned long long scale2 = pa_pair(scale, scale), off2 = pa_pair(-off, -off);
                unsigned w[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const unsigned long long x = pa_exp2(pa_fma2((unsigned long long)s[2 * e + 1] << 32 | s[2 * e], scale2, off2));
                    sum2[e & 1] = pa_add2(sum2[e & 1], x);
                    const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float((unsigned)x), __uint_as_float((unsigned)(x >> 32)));
                    w[e] = *reinterpret_cast<const unsigned*>(&h);
                }
                tc_st32(at, w);
                if (masked) {
                    // A weight of zero times an infinity is a NaN, and the products take all keys of the step.  Where a value among them is
                    // not finite (padding behind a sequence, another sequence's rows) each row adds the values that it sees itself.
                    const unsigned place = 2 * (before + j) + 1;
                    if (!(ok = wait(full + 8 * (place % NS), place / NS & 1))) break;
                    const unsigned char* v = smem + M::ring + place % NS * M::part;
                    unsigned odd = 0;
                    for (int e = row; e < M::part / 16; e += 128) {
                        const uint4 x = reinterpret_cast<const uint4*>(v)[e];   // an exponent of all ones carries into the sign's place
                        odd |= (((x.x & 0x7f807f80u) + 0x00800080u) | ((x.y & 0x7f807f80u) + 0x00800080u) | ((x.z & 0x7f807f80u) + 0x00800080u) |
                                ((x.w & 0x7f807f80u) + 0x00800080u)) & 0x80008000u;
                    }
                    odd = __reduce_or_sync(0xffffffffu, odd);
                    if (lane == 0) {
                        if (odd) *reinterpret_cast<volatile int*>(&s_odd[i][j & 1]) = (int)step;
                        tc_bar_arrive(checked + 8 * i);
                    }
                    if (!(ok = wait(checked + 8 * i, checks++ & 1))) break;
                    if (*reinterpret_cast<volatile int*>(&s_odd[i][j & 1]) == (int)step) {
                        if (j > 0 && !(ok = products(j - 1))) break;
                        tc_after();
                        tc_wait_st();
                        const int see = min(last - j * kPaKeys, kPaKeys - 1);
                        for (int c = 0; c < HD; c += 32) {
                            float o[32];
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = 0.0f;
                            for (int k = 0; k < kPaKeys; ++k) {
                                unsigned w = tc_ld1(at + (k >> 1));
                                tc_wait_ld();
                                asm volatile("" : "+r"(w));
                                if (k <= see) {
                                    const float p = __uint_as_float(k & 1 ? w & 0xffff0000u : w << 16);
                                    const unsigned char* line = v + (c / 64) * (M::part / C) + k * 128;
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
                if (lane == 0) tc_bar_arrive(p_full + 16 * i + 8 * (j & 1));
            }
            const int live = what[5 + i];
            if constexpr (kShares) {
                if (ok && steps) {
                    ok = products(steps - 1);
                    tc_after();
                }
                pa_rows_sync();   // (where Q, K and V were)
                met = true;
                sum2[0] = pa_add2(sum2[0], sum2[1]);
                float* const parts = reinterpret_cast<float*>(smem);
                for (int c = 0; c < HD; c += 32) {
                    unsigned o[32];
                    if (steps) {
                        tc_ld32(ot + c, o);
                        tc_wait_ld();
                        tc_pin32(o);
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<uint4*>(parts + tid * PaParts<HD>::row + c + e) =
                            steps ? make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]) : make_uint4(0u, 0u, 0u, 0u);
                }
                reinterpret_cast<float2*>(smem + PaParts<HD>::heads)[tid] =
                    steps ? make_float2(top * scale, __uint_as_float((unsigned)sum2[0]) + __uint_as_float((unsigned)(sum2[0] >> 32))) : make_float2(-INFINITY, 0.0f);
            }
            if (!kShares && ok && live > 0) {
                const int position = row / P.share;
                const bool out = position < live && row < per * P.share;
                sum2[0] = pa_add2(sum2[0], sum2[1]);
                const float total = __uint_as_float((unsigned)sum2[0]) + __uint_as_float((unsigned)(sum2[0] >> 32)), inv = total == 0.0f ? 0.0f : 1.0f / total;
                uint4* to = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(P.out) +
                                                     ((size_t)(what[0] + what[4] + i * per + (out ? position : 0)) * P.q_heads + what[3] * P.share + (out ? row % P.share : 0)) * HD);
                if (steps) {
                    ok = products(steps - 1);
                    tc_after();
                }
                for (int c = 0; c < HD && ok; c += 32) {
                    unsigned o[32];
                    if (steps) {
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
                            const float x = steps ? __uint_as_float(o[8 * e + 2 * h]) * inv : 0.0f, y = steps ? __uint_as_float(o[8 * e + 2 * h + 1]) * inv : 0.0f;
                            const __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
                            w[h] = *reinterpret_cast<const unsigned*>(&p);
                        }
                        to[c / 8 + e] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            if (!ok) break;
            before += n;
            __syncwarp();
            if (lane == 0) tc_bar_arrive(item_empty + 8 * (number & 1));
        }
        if (kShares && !met) pa_rows_sync();   // (a warp that gave up must not leave the others waiting)
    }
    if (!ok) atomicExch(&g_prompt_error, 1);
    tc_before();
    __syncthreads();
    if (warp == 8) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if constexpr (kShares) {
        pa_cluster_sync();   // the sums of every share are in place
        const volatile int* const what = s_item[0];
        if (warp < 8 && what[0] >= 0) pa_join<HD, true>(P, smem, what[0] + what[4], what[3], per, what[5], what[6], 1.0f);
        pa_cluster_sync();   // nobody leaves while its sums may still be read
    }
    if (*reinterpret_cast<volatile int*>(&s_gone) && threadIdx.x < 256)   // what the CTA had last and before, and what it took from another one
        for (int i = 0; i < 3; ++i) {
            const volatile int* const what = s_item[i];
            if (what[0] >= 0)
                packed_give_up<HD>(static_cast<__nv_bfloat16*>(P.out), (size_t)(what[0] + what[4]), what[5] + what[6], what[3] * P.share, P.share, P.q_heads, threadIdx.x, 256);
        }
}

// CTAs that share the keys of a part of the rows: as many as the GPU holds next to one another, with four steps of keys each on average.  The
// cluster's launch and the joining cost 8 us in bf16, where there is also no work to take over, and 2 us next to the longer steps of fp32.
// us without and with shares, 8 KV heads of 4 query heads of 128: 256 positions behind 768 cached ones 22 and 27 in bf16, 60 and 52 in
// fp32, 300 behind 1700 37 and 34, 104 and 77, 64 behind 7936 124 and 30, 367 and 85; 512 alone 15 and 23, 38 and 40.
static int prompt_shares(const PromptProblem& P, long long parts, bool bf16) {
    const long long steps = (long long)P.n_keys / std::min(P.batch, P.n_rows) / 64;
    int shares = 1;
    if (steps < (bf16 ? 24 : 12)) return 1;
    while (shares < 8 && parts * shares * 2 <= num_sms() && steps >= 8LL * shares) shares *= 2;
    return shares;
}
static_assert(kPaKeys == 64, "steps of keys");

template <int HD>
static int launch_prompt_tc(const PromptProblem& P, cudaStream_t s) {
    static std::atomic<bool> opted[4][64];
    constexpr int smem = PaSmem<HD>::bytes;
    static_assert(PaParts<HD>::bytes <= PaSmem<HD>::bars, "the sums of the rows lie where Q, K and V were");
    const int per = kPaRows / P.share;
    const long long parts = P.n_rows / (2 * per) + std::min(P.batch, P.n_rows);
    if (parts * P.kv_heads > 0x7fffffffLL) return OJX_ERR_TOO_LARGE;   // (with shares there are at most as many as SMs)
    CUtensorMap q, k, v;
    const bool none = P.n_keys == 0;
    if (!tc_map3(&q, true, P.q, HD, P.q_heads, P.n_rows, P.q_head, P.q_row, 64, P.share, per) ||
        !tc_map3(&k, true, none ? P.q : P.k, HD, none ? 1 : P.kv_heads, none ? 1 : P.n_keys, none ? HD : P.k_head, none ? HD : P.k_row, 64, 1, kPaKeys) ||
        !tc_map3(&v, true, none ? P.q : P.v, HD, none ? 1 : P.kv_heads, none ? 1 : P.n_keys, none ? HD : P.v_head, none ? HD : P.v_row, 64, 1, kPaKeys)) {
        set_last_error_msg("prompt attention: the tensors' strides do not make a tensor map");
        return OJX_ERR_ARG;
    }
    const int shares = prompt_shares(P, parts * P.kv_heads, true);
    auto kernel = P.none ? (shares > 1 ? prompt_tc_kernel<HD, true, true> : prompt_tc_kernel<HD, false, true>)
                         : (shares > 1 ? prompt_tc_kernel<HD, true, false> : prompt_tc_kernel<HD, false, false>);
    OJX_CUDA_TRY(opt_in_smem(reinterpret_cast<const void*>(kernel), smem, opted[(shares > 1) + 2 * (P.none != nullptr)]));
    if (shares > 1) OJX_CUDA_TRY(launch_chained_cluster(kernel, dim3((unsigned)(parts * P.kv_heads * shares)), kPaThreads, smem, s, (unsigned)shares, P, q, k, v));
    else OJX_CUDA_TRY(launch_chained(kernel, dim3((unsigned)(parts * P.kv_heads)), kPaThreads, smem, s, P, q, k, v));
    count_launch(1);
    return OJX_OK;
}

// ------------------------------------------------------------------------------------ fp32 on the 5th-generation tensor cores
//
// The bf16 kernel's two tiles and turns, on operands that are two fp16 numbers each, x = (hi + lo) / scale: 22 bits, and three products
// for one (lo hi, hi lo, hi hi).  Every row of Q, K and V has a power of two of its own that brings its largest element to 2^14..2^15:
//   those of Q and K are taken out of the scores (a factor per row, a factor per key);
//   those of V go into the weights, y = 2^(x + e - reference) with e the exponent of the key's largest value, so that a weight times its
//   value is what it is, and the sum of weights takes y * 2^-e.  e stays in -20..100: the values of a smaller row keep fewer bits.
// The high parts of Q are in tensor memory, where products take them without the shared memory's bandwidth; the low ones, and K and V
// in steps of 64 keys, are in shared memory.  The tensor cores cut what they add to a sum, so a step's products with V are summed on
// their own and join the row's fp32 sums, which are in its thread's registers.  Bound by what a row's thread does for a step (the two parts
// of 64 weights, O of the step before, and at head_dim 128 some of the 312 bytes that do not fit into its registers, 116 at 64); the tensor
// pipe is 41 % busy.  Two prompts of 2048 with 32 query heads and 8 KV heads of 128: 263 to 272 us, 253 to 261 TFLOP/s of the formula, three
// times as many of fp16 products (4750 us with fp32 FMA, 364 with all of Q in shared memory).  Two S of 32 keys a tile, so
// that products and exponentials overlap within a tile too, took a fifth longer: every step has its waits, whatever its length.
constexpr int kPpKeys = 64;
constexpr float kPpRoom = 5.0f;   // y is 2^5 at most when the reference is set, 2^13 later on

template <int HD>
struct PpSmem {
    static constexpr int tile = 128 * HD * 2;                                 // of Q: the low parts
    static constexpr int part = kPpKeys * HD * 2, slot = 2 * part;            // of K or V: two planes
    static constexpr int slots = HD == 128 ? 4 : 8;
    static constexpr int ring = 2 * tile, factors = ring + slots * slot;      // [2][3][64]: of K, e, 2^-e
    static constexpr int bars = factors + 2 * 3 * kPpKeys * 4;
    static constexpr int bytes = bars + 256 + 1024;
};

struct PromptSplit {
    __half* planes[4];      // K hi, K lo, V hi, V lo: [n_keys][kv_heads][head_dim]
    float2* factors;        // [kv_heads][n_keys]: 1 / scale of the key's row of K, e of its row of V
};

// A row of K or V per HD / 8 lanes, 16 bytes in and out; bound by the instructions of the split and the latency of its loads.  (With HD / 4
// lanes to a row the two kernels took 285.4 us for two prompts of 2048, with HD / 8 283.3 then.)
template <int HD>
__global__ void __launch_bounds__(256) prompt_split_kernel(const __grid_constant__ PromptProblem P, const __grid_constant__ PromptSplit S) {
    constexpr int L = HD / 8;
    chain_begin();
    const long long row = ((long long)blockIdx.x * 256 + threadIdx.x) / L, rows = (long long)P.n_keys * P.kv_heads;
    const int l = threadIdx.x % L;
    if (row >= 2 * rows) return;   // (all L lanes of a row, within which the shuffles stay)
    const bool values = row >= rows;
    const long long r = values ? row - rows : row;
    const long long key = r / P.kv_heads;
    const int head = (int)(r - key * P.kv_heads);
    const float4* from = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(values ? P.v : P.k) + key * (values ? P.v_row : P.k_row) +
                                                         head * (values ? P.v_head : P.k_head) + 8 * l);
    const float4 x = from[0], y = from[1];
    float xs[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    unsigned most = 0;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const unsigned b = __float_as_uint(xs[e]) & 0x7fffffffu;
        if (b < 0x7f800000u) most = max(most, b);
        else odd = true;
    }
    const unsigned lanes = ((1u << L) - 1u) << (threadIdx.x % 32 / L * L);   // the row's: they are all here, or none of them
#pragma unroll
    for (int off = L / 2; off >= 1; off >>= 1) most = max(most, __shfl_xor_sync(lanes, most, off));
    float up, down, e = 0.0f;
    if (values) {
        const int p = min(max((int)(most >> 23) - 127, -20), 100);
        up = __uint_as_float((unsigned)(127 + 14 - p) << 23);
        e = P.none && P.none[key] ? -INFINITY : (float)p;   // a key that nobody sees: its scores, which e is added to, are -inf
    } else {
        gm_scale(most, up, down);
        // A key with infinities: their signs alone, times infinity, so that its scores are infinite or, where the query is zero, NaN.  (Two
        // infinities that cancel in a score, as far as the queries' sizes let them, are taken for the larger one.)
        if (__any_sync(lanes, odd)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) xs[i] = isinf(xs[i]) ? copysignf(1.0f, xs[i]) : isnan(xs[i]) ? xs[i] : 0.0f;
            up = 1.0f;
            down = INFINITY;
        }
    }
    unsigned hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = xs[2 * i] * up, b = xs[2 * i + 1] * up;
        const __half2 h = __floats2half2_rn(a, b);
        hi[i] = *reinterpret_cast<const unsigned*>(&h);
        lo[i] = gm_pack(a - __low2float(h), b - __high2float(h));
    }
    const size_t to = (size_t)r * HD + 8 * l;
    *reinterpret_cast<uint4*>(S.planes[values ? 2 : 0] + to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(S.planes[values ? 3 : 1] + to) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    // (a value is 2^(14 - e) times as large, its weight 2^e: 2^14 is left for the end)
    if (l == 0) {
        float* f = reinterpret_cast<float*>(S.factors + (size_t)head * P.n_keys + key);
        f[values] = values ? e : down;
    }
}

template <int HD, bool kShares>
__global__ void __launch_bounds__(kPaThreads, 1) prompt_pair_kernel(const __grid_constant__ PromptProblem P, const __grid_constant__ PromptSplit S,
                                                                    const __grid_constant__ CUtensorMap k_hi, const __grid_constant__ CUtensorMap k_lo,
                                                                    const __grid_constant__ CUtensorMap v_hi, const __grid_constant__ CUtensorMap v_lo) {
    using M = PpSmem<HD>;
    constexpr int NS = M::slots, C = HD / 64, N = kPpKeys;
    extern __shared__ unsigned char pa_raw[];
    unsigned char* smem = pa_raw + ((1024u - (tc_smem(pa_raw) & 1023u)) & 1023u);
    __shared__ int s_seq, s_part, s_gone, s_odd[2];
    __shared__ unsigned s_tmem;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;   // (the same for a warp, as the compiler sees)
    const unsigned base = tc_smem(smem), bars = base + M::bars;
    const unsigned full = bars, empty = bars + 8 * NS, q_full = empty + 8 * NS, s_full = q_full + 16, p_full = s_full + 16, o_full = p_full + 16,
                   checked = o_full + 16, f_full = checked + 16, f_empty = f_full + 16, ended = f_empty + 16, gone = tc_smem(&s_gone);
    const int size = kShares ? pa_cluster_size() : 1, unit = (int)blockIdx.x / size, units = (int)gridDim.x / size;
    const int head = unit % P.kv_heads, per = kPaRows / P.share;
    if (tid == 0) {
        for (int i = 0; i < NS; ++i) { tc_bar_init(full + 8 * i, 1); tc_bar_init(empty + 8 * i, 1); }
        for (int i = 0; i < 2; ++i) {
            tc_bar_init(q_full + 8 * i, 4);
            tc_bar_init(s_full + 8 * i, 1);
            tc_bar_init(p_full + 8 * i, 4);
            tc_bar_init(o_full + 8 * i, 1);
            tc_bar_init(checked + 8 * i, 4);
            tc_bar_init(f_full + 8 * i, 32);
            tc_bar_init(f_empty + 8 * i, 8);
            s_odd[i] = 0;
        }
        tc_bar_init(ended, 1);
        s_gone = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    chain_begin();
    if (warp == 0) {
        int seq = -1, part = 0;   // (the last parts first)
        const bool in = packed_part(P.batch, units / P.kv_heads - 1 - unit / P.kv_heads,
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
    // S and then the weights of tile i at 64 i (hi 32 columns, lo 32), Q's high parts at 128 + 64 i, a step's O at 256 + 128 i
    const unsigned tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    const PackedRange rows = packed_range(P.ends, s_seq, P.n_rows);
    PackedRange keys = packed_range(P.key_ends, s_seq, P.n_keys);
    int ahead = keys.count - rows.count, pos[2], live[2], steps[2], most = 0x7fffffff;
    if (kShares) {   // the keys begin with the first of this CTA's
        const int end = min(rows.count, (s_part + 1) * 2 * per);
        const PaShare share(max(0, end + ahead + N - 1) / N, pa_cluster_rank(), size);
        keys.first += share.first * N;
        keys.count -= share.first * N;
        ahead -= share.first * N;
        most = share.count;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        pos[i] = (s_part * 2 + i) * per;
        live[i] = max(0, min(per, rows.count - pos[i]));
        steps[i] = live[i] > 0 ? min(max(0, pos[i] + live[i] + ahead + N - 1) / N, most) : 0;
    }
    const int n = max(steps[0], steps[1]);
    bool ok = true;
    auto wait = [&](unsigned bar, unsigned parity) { return tc_wait(bar, parity, gone); };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 9 && lane == 0) {
            int s = 0;
            for (; s < 2 * n; ++s) {   // K of step 0, V of step 0, K of step 1, ...
                const int slot = s % NS;
                if (s >= NS && !(ok = bar_wait(empty + 8 * slot, (s / NS - 1) & 1, gone))) break;
                tc_bar_expect(full + 8 * slot, M::slot);
                for (int c = 0; c < C; ++c)
                    for (int p = 0; p < 2; ++p)
                        tc_load3(base + M::ring + slot * M::slot + p * M::part + c * (M::part / C), s & 1 ? (p ? &v_lo : &v_hi) : (p ? &k_lo : &k_hi), 64 * c,
                                 head, keys.first + (s >> 1) * N, full + 8 * slot);
            }
            if (!ok)   // nothing may land after the CTA has left
                for (int u = max(0, s - NS); u < s; ++u) bar_wait(full + 8 * (u % NS), (u / NS) & 1);
        }
        if (warp == 10) {
            for (int j = 0; j < n; ++j) {
                if (j >= 2 && !(ok = bar_wait(f_empty + 8 * (j & 1), (j / 2 - 1) & 1, gone))) break;
                float* f = reinterpret_cast<float*>(smem + M::factors) + (j & 1) * 3 * N;
                for (int c = lane; c < N; c += 32) {
                    const int key = j * N + c;
                    const float2 x = key < keys.count ? S.factors[(size_t)head * P.n_keys + keys.first + key] : make_float2(0.0f, 0.0f);
                    f[c] = x.x;
                    f[N + c] = x.y;
                    f[2 * N + c] = x.y == -INFINITY ? 1.0f : __uint_as_float((unsigned)(127 - (int)x.y) << 23);
                }
                tc_bar_arrive(f_full + 8 * (j & 1));
            }
        }
        if (warp == 8) {
            const unsigned lead = tc_lead();
            constexpr unsigned iq = tc_idesc<false, false>(N), iv = tc_idesc<false, true>(HD);
            const unsigned long long ring_k = tc_desc(base + M::ring), ring_v = tc_desc(base + M::ring, M::part / C), q_desc = tc_desc(base);
            auto scores = [&](int i, int slot) {
                const unsigned long long a = tc_at(q_desc, i * M::tile), b = tc_at(ring_k, slot * M::slot);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k)   // lo hi
                    tc_mma(lead, tmem + i * 64, tc_at(a, (k / 4) * (M::tile / C) + (k % 4) * 32), tc_at(b, (k / 4) * (M::part / C) + (k % 4) * 32), iq, k > 0);
#pragma unroll
                for (int p = 1; p >= 0; --p)        // hi lo, hi hi
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k)
                        tc_mma_ts(lead, tmem + i * 64, tmem + 128 + i * 64 + k * 8, tc_at(b, p * M::part + (k / 4) * (M::part / C) + (k % 4) * 32), iq, true);
                tc_commit(lead, s_full + 8 * i);
            };
            TcRing<NS> kr{0, 0}, vr{1, 0};
            if (n > 0) ok = wait(full, 0);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (ok && steps[i]) {
                    ok = wait(q_full + 8 * i, 0);
                    tc_after();
                    if (ok) scores(i, 0);
                }
            if (n > 0 && ok) tc_commit(lead, empty);
            for (int j = 0; j < n && ok; ++j) {
                kr.next(2);
                bool loaded = false;
                ok = wait(full + 8 * vr.slot, vr.parity);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (j >= steps[i] || !ok) continue;
                    if (!(ok = wait(p_full + 8 * i, j & 1))) continue;
                    tc_after();
                    if (!((j + 1) * N - 1 > pos[i] + ahead && *reinterpret_cast<volatile int*>(&s_odd[i]) == j + 1)) {
                        const unsigned long long b = tc_at(ring_v, vr.slot * M::slot);
#pragma unroll
                        for (int p = 0; p < 3; ++p)
#pragma unroll
                            for (int k = 0; k < N / 16; ++k)
                                tc_mma_ts(lead, tmem + 256 + i * 128, tmem + i * 64 + (p == 0) * (N / 2) + k * 8, tc_at(b, (p == 1) * M::part + k * 2048), iv, p > 0 || k > 0);
                    }
                    if (j + 1 < steps[i]) {
                        if (!loaded && !(ok = wait(full + 8 * kr.slot, kr.parity))) continue;
                        loaded = true;
                        scores(i, kr.slot);   // (in order: its commit says that O is there, too)
                    } else {
                        tc_commit(lead, o_full + 8 * i);
                    }
                }
                if (!ok) break;
                tc_commit(lead, empty + 8 * vr.slot);
                if (j + 1 < n) tc_commit(lead, empty + 8 * kr.slot);
                vr.next(2);
            }
            if (!ok) {
                tc_commit(lead, ended);
                bar_wait(ended, 0);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        const int i = warp >> 2, row = tid & 127;
        const int at = min(row, max(live[i] * P.share - 1, 0)), last = pos[i] + at / P.share + ahead;
        const bool out = row < live[i] * P.share;
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16, st = tmem + i * 64 + lanes, ot = tmem + 256 + i * 128 + lanes;
        const size_t where = out ? (size_t)(rows.first + pos[i] + row / P.share) : 0;
        const int q_head = head * P.share + (out ? row % P.share : 0);
        int checks = 0;
        float unscale = 0.0f;
        if (steps[i]) {   // the warp's rows of Q, HD / 4 lanes to a row: the high parts through shared memory to tensor memory, then the low ones
            constexpr int L = HD / 4, R = 32 / L;
            const int l = lane % L, sub = lane / L;
            const long long from = out ? (long long)where * P.q_row + (long long)q_head * P.q_head : -1;   // of the thread's own row
            float4 x[32 / R];
#pragma unroll
            for (int r = 0; r < 32 / R; ++r) {   // (all loads before the first is waited for)
                const long long at_row = __shfl_sync(0xffffffffu, from, r * R + sub);
                x[r] = at_row >= 0 ? *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(P.q) + at_row + 4 * l) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int r = 0; r < 32 / R; ++r) {
                unsigned most = max(max(__float_as_uint(x[r].x) & 0x7fffffffu, __float_as_uint(x[r].y) & 0x7fffffffu),
                                    max(__float_as_uint(x[r].z) & 0x7fffffffu, __float_as_uint(x[r].w) & 0x7fffffffu));
#pragma unroll
                for (int off = L / 2; off >= 1; off >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, off));
                float up, down;
                gm_scale(most, up, down);
                x[r] = make_float4(x[r].x * up, x[r].y * up, x[r].z * up, x[r].w * up);
                const float back = __shfl_sync(0xffffffffu, down, (lane % R) * L);   // lane r * R + k takes that of the k-th row of these
                if (lane / R == r) unscale = back;
            }
#pragma unroll
            for (int low = 0; low < 2; ++low) {
#pragma unroll
                for (int r = 0; r < 32 / R; ++r) {
                    const int mine = (warp & 3) * 32 + r * R + sub;
                    const __half2 h0 = __floats2half2_rn(x[r].x, x[r].y), h1 = __floats2half2_rn(x[r].z, x[r].w);
                    *reinterpret_cast<uint2*>(smem + i * M::tile + (4 * l / 64) * (M::tile / C) + mine * 128 + (((l % 16) / 2 ^ (mine & 7)) << 4) + (l & 1) * 8) =
                        make_uint2(*reinterpret_cast<const unsigned*>(&h0), *reinterpret_cast<const unsigned*>(&h1));
                    x[r] = make_float4(x[r].x - __low2float(h0), x[r].y - __high2float(h0), x[r].z - __low2float(h1), x[r].w - __high2float(h1));
                }
                __syncwarp();
                if (low) break;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    unsigned w[32];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        *reinterpret_cast<uint4*>(w + 4 * e) = *reinterpret_cast<const uint4*>(smem + i * M::tile + c * (M::tile / C) + row * 128 + ((e ^ (row & 7)) << 4));
                    tc_st32(tmem + 128 + i * 64 + lanes + 32 * c, w);
                }
                tc_wait_st();
                __syncwarp();
            }
            unscale *= P.scale * 1.4426950408889634f;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc_before();
            __syncwarp();
            if (lane == 0) tc_bar_arrive(q_full + 8 * i);
        }
        float top = -INFINITY;
        unsigned long long sum = 0, o[HD / 2];
#pragma unroll
        for (int d = 0; d < HD / 2; ++d) o[d] = 0;
        bool parted = false;   // a step's O is in tensor memory
        auto join = [&]() {
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                unsigned x[32];
                tc_ld32(ot + c, x);
                tc_wait_ld();
                tc_pin32(x);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[c / 2 + e] = pa_add2(o[c / 2 + e], (unsigned long long)x[2 * e + 1] << 32 | x[2 * e]);
            }
        };
        for (int j = 0; j < n; ++j) {
            if (j >= steps[i]) {   // (the other tile has more steps: the keys' factors have to go on)
                if (!(ok = wait(f_full + 8 * (j & 1), (j / 2) & 1))) break;
                __syncwarp();
                if (lane == 0) tc_bar_arrive(f_empty + 8 * (j & 1));
                continue;
            }
            if (!(ok = wait(s_full + 8 * i, j & 1))) break;
            tc_after();
            if (parted) join();
            unsigned s[N];
            tc_ld32(st, s);
            tc_ld32(st + 32, s + 32);
            if (!(ok = wait(f_full + 8 * (j & 1), (j / 2) & 1))) break;
            tc_wait_ld();
            tc_pin32(s);
            tc_pin32(s + 32);
            const float* f = reinterpret_cast<const float*>(smem + M::factors) + (j & 1) * 3 * N;
            const bool masked = (j + 1) * N - 1 > pos[i] + ahead;
            const int see = last - j * N;
            const unsigned long long unscale2 = pa_pair(unscale, unscale);
            float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const ulonglong2 kf = *reinterpret_cast<const ulonglong2*>(f + e), ex = *reinterpret_cast<const ulonglong2*>(f + N + e);
                const unsigned long long x = pa_fma2(pa_mul2((unsigned long long)s[e + 1] << 32 | s[e], kf.x), unscale2, ex.x);
                const unsigned long long y = pa_fma2(pa_mul2((unsigned long long)s[e + 3] << 32 | s[e + 2], kf.y), unscale2, ex.y);
                s[e] = (unsigned)x; s[e + 1] = (unsigned)(x >> 32); s[e + 2] = (unsigned)y; s[e + 3] = (unsigned)(y >> 32);
                if (masked) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) s[e + u] = e + u > see ? 0xff800000u : s[e + u];
                }
                m[0] = pa_max3(m[0], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
                m[1] = pa_max3(m[1], __uint_as_float(s[e + 2]), __uint_as_float(s[e + 3]));
            }
            const float now = fmaxf(m[0], m[1]) - kPpRoom;
            const bool up = now > top + kPaSlack;
            if (j == 0) {
                top = now;
            } else if (__any_sync(0xffffffffu, up)) {
                const float by = up ? exp2f(top - now) : 1.0f;
                const unsigned long long by2 = pa_pair(by, by);
                top = up ? now : top;
                sum = pa_mul2(sum, by2);
#pragma unroll
                for (int d = 0; d < HD / 2; ++d) o[d] = pa_mul2(o[d], by2);
            }
            const float off = top == -INFINITY ? 0.0f : top;
            const unsigned long long off2 = pa_pair(-off, -off);
#pragma unroll
            for (int c = 0; c < N; c += 32) {
                unsigned hi[16], lo[16];
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const ulonglong2 vf = *reinterpret_cast<const ulonglong2*>(f + 2 * N + c + e);
                    const unsigned long long vfs[2] = {vf.x, vf.y};
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const unsigned long long y = pa_exp2(pa_add2((unsigned long long)s[c + e + 2 * u + 1] << 32 | s[c + e + 2 * u], off2));
                        sum = pa_fma2(y, vfs[u], sum);
                        // the high part is cut to 11 bits, which fp16 holds as they are (266 us with a
                        // rounded one, which has to come back from fp16, and 254.5 so on one box; 3.3e-7 and 3.4e-7 off 64 bits)
                        const unsigned yl = (unsigned)y & 0xffffe000u, yh = (unsigned)(y >> 32) & 0xffffe000u;
                        const __half2 h = __floats2half2_rn(__uint_as_float(yl), __uint_as_float(yh));
                        const unsigned long long rest = pa_fma2((unsigned long long)yh << 32 | yl, pa_pair(-1.0f, -1.0f), y);
                        hi[e / 2 + u] = *reinterpret_cast<const unsigned*>(&h);
                        lo[e / 2 + u] = gm_pack(__uint_as_float((unsigned)rest), __uint_as_float((unsigned)(rest >> 32)));
                    }
                }
                tc_st16(st + c / 2, hi);
                tc_st16(st + N / 2 + c / 2, lo);
            }
            parted = true;
            if (masked) {   // (as in the bf16 kernel: values that are not finite among those that are not seen)
                if (!(ok = wait(full + 8 * ((2 * j + 1) % NS), ((2 * j + 1) / NS) & 1))) break;
                const unsigned char* v = smem + M::ring + ((2 * j + 1) % NS) * M::slot;
                unsigned odd = 0;
                for (int e = row; e < M::part / 16; e += 128) {
                    const uint4 x = reinterpret_cast<const uint4*>(v)[e];
                    odd |= (((x.x & 0x7c007c00u) + 0x04000400u) | ((x.y & 0x7c007c00u) + 0x04000400u) | ((x.z & 0x7c007c00u) + 0x04000400u) |
                            ((x.w & 0x7c007c00u) + 0x04000400u)) & 0x80008000u;
                }
                odd = __reduce_or_sync(0xffffffffu, odd);
                if (lane == 0) {
                    if (odd) *reinterpret_cast<volatile int*>(&s_odd[i]) = j + 1;
                    tc_bar_arrive(checked + 8 * i);
                }
                if (!(ok = wait(checked + 8 * i, checks++ & 1))) break;
                if (*reinterpret_cast<volatile int*>(&s_odd[i]) == j + 1) {
                    tc_wait_st();
                    parted = false;
                    const int end = min(see, N - 1);
#pragma unroll
                    for (int c = 0; c < HD; c += 32)
                        for (int k = 0; k < N; ++k) {
                            unsigned hi = tc_ld1(st + (k >> 1)), lo = tc_ld1(st + N / 2 + (k >> 1));
                            tc_wait_ld();
                            asm volatile("" : "+r"(hi), "+r"(lo));
                            if (k <= end) {
                                const __half2 a = *reinterpret_cast<const __half2*>(&hi), b = *reinterpret_cast<const __half2*>(&lo);
                                const float y = k & 1 ? __high2float(a) + __high2float(b) : __low2float(a) + __low2float(b);
                                const unsigned char* line = v + (c / 64) * (M::part / C) + k * 128;
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int piece = (((c % 64) / 8 + e) ^ (k & 7)) * 16;
                                    const uint4 xh = *reinterpret_cast<const uint4*>(line + piece), xl = *reinterpret_cast<const uint4*>(line + M::part + piece);
                                    const unsigned hs[4] = {xh.x, xh.y, xh.z, xh.w}, ls[4] = {xl.x, xl.y, xl.z, xl.w};
#pragma unroll
                                    for (int h = 0; h < 4; ++h) {
                                        const __half2 vh = *reinterpret_cast<const __half2*>(&hs[h]), vl = *reinterpret_cast<const __half2*>(&ls[h]);
                                        o[c / 2 + 4 * e + h] = pa_fma2(pa_pair(y, y), pa_pair(__low2float(vh) + __low2float(vl), __high2float(vh) + __high2float(vl)), o[c / 2 + 4 * e + h]);
                                    }
                                }
                            }
                            __syncwarp();
                        }
                }
            }
            tc_wait_st();
            tc_before();
            __syncwarp();
            if (lane == 0) {
                tc_bar_arrive(f_empty + 8 * (j & 1));
                tc_bar_arrive(p_full + 8 * i);
            }
        }
        if constexpr (kShares) {
            if (ok && steps[i]) {
                ok = wait(o_full + 8 * i, 0);
                tc_after();
                if (ok && parted) join();
            }
            pa_rows_sync();   // (where Q, K and V were)
            float* const to = reinterpret_cast<float*>(smem) + tid * PaParts<HD>::row;
#pragma unroll
            for (int d = 0; d < HD / 2; d += 2) *reinterpret_cast<ulonglong2*>(to + 2 * d) = make_ulonglong2(o[d], o[d + 1]);
            reinterpret_cast<float2*>(smem + PaParts<HD>::heads)[tid] =
                make_float2(top, __uint_as_float((unsigned)sum) + __uint_as_float((unsigned)(sum >> 32)));
        }
        if (!kShares && ok && live[i] > 0) {
            if (steps[i]) {
                ok = wait(o_full + 8 * i, 0);
                tc_after();
                if (ok && parted) join();
            }
            const float total = __uint_as_float((unsigned)sum) + __uint_as_float((unsigned)(sum >> 32)), inv = total == 0.0f ? 0.0f : 1.0f / (total * 16384.0f);   // (values are 2^14 times as large as their exponents say)
            if (ok && out) {
                float4* to = reinterpret_cast<float4*>(reinterpret_cast<float*>(P.out) + (where * P.q_heads + q_head) * HD);
#pragma unroll
                for (int d = 0; d < HD / 2; d += 2)
                    to[d / 2] = make_float4(__uint_as_float((unsigned)o[d]) * inv, __uint_as_float((unsigned)(o[d] >> 32)) * inv,
                                            __uint_as_float((unsigned)o[d + 1]) * inv, __uint_as_float((unsigned)(o[d + 1] >> 32)) * inv);
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
    if constexpr (kShares) {
        pa_cluster_sync();   // the sums of every share are in place
        if (warp < 8) pa_join<HD, false>(P, smem, rows.first + pos[0], head, per, live[0], live[1], 16384.0f);
        pa_cluster_sync();   // nobody leaves while its sums may still be read
    }
    if (*reinterpret_cast<volatile int*>(&s_gone) && threadIdx.x < 256) {
        const PackedRange of = packed_range(P.ends, s_seq, P.n_rows);
        const int first = s_part * 2 * (kPaRows / P.share), share = P.share;
        packed_give_up<HD>(static_cast<float*>(P.out), (size_t)(of.first + first), min(2 * (kPaRows / share), of.count - first),
                           (int)blockIdx.x / (kShares ? pa_cluster_size() : 1) % P.kv_heads * share, share, P.q_heads, threadIdx.x, 256);
    }
}

// Bytes of the planes and factors of K and V.
static size_t prompt_split_plane(int n_keys, int kv_heads, int head_dim) { return ((size_t)std::max(n_keys, 1) * kv_heads * head_dim * 2 + 255) / 256 * 256; }

template <int HD>
static int launch_prompt_pair(const PromptProblem& P, void* workspace, cudaStream_t s) {
    static std::atomic<bool> opted[2][64];
    constexpr int smem = PpSmem<HD>::bytes;
    static_assert(PaParts<HD>::bytes <= PpSmem<HD>::factors, "the sums of the rows lie where Q, K and V were");
    const int per = kPaRows / P.share;
    const long long parts = P.n_rows / (2 * per) + std::min(P.batch, P.n_rows);
    const long long split = ((long long)P.n_keys * P.kv_heads * 2 * (HD / 8) + 255) / 256;
    if (parts * P.kv_heads > 0x7fffffffLL || split > 0x7fffffffLL) return OJX_ERR_TOO_LARGE;
    PromptSplit S{};
    const size_t plane = prompt_split_plane(P.n_keys, P.kv_heads, HD);
    char* at = static_cast<char*>(workspace);
    CUtensorMap maps[4];
    for (int i = 0; i < 4; ++i, at += plane) {
        S.planes[i] = reinterpret_cast<__half*>(at);
        if (!tc_map3(&maps[i], false, at, HD, P.kv_heads, std::max(P.n_keys, 1), HD, (unsigned long long)P.kv_heads * HD, 64, 1, kPpKeys)) {
            set_last_error_msg("prompt attention: no tensor map");
            return OJX_ERR_CUDA;
        }
    }
    S.factors = reinterpret_cast<float2*>(at);
    if (split) {
        OJX_CUDA_TRY(launch_chained(prompt_split_kernel<HD>, dim3((unsigned)split), 256, 0, s, P, S));
        count_launch(1);
    }
    const int shares = prompt_shares(P, parts * P.kv_heads, false);
    auto kernel = shares > 1 ? prompt_pair_kernel<HD, true> : prompt_pair_kernel<HD, false>;
    OJX_CUDA_TRY(opt_in_smem(reinterpret_cast<const void*>(kernel), smem, opted[shares > 1]));
    if (shares > 1)
        OJX_CUDA_TRY(launch_chained_cluster(kernel, dim3((unsigned)(parts * P.kv_heads * shares)), kPaThreads, smem, s, (unsigned)shares, P, S, maps[0], maps[1],
                                            maps[2], maps[3]));
    else OJX_CUDA_TRY(launch_chained(kernel, dim3((unsigned)(parts * P.kv_heads)), kPaThreads, smem, s, P, S, maps[0], maps[1], maps[2], maps[3]));
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

extern "C" {

size_t ojasx_b200_prompt_workspace(int n_keys, int kv_heads, int head_dim, int io_dtype) {
    if (io_dtype != OJX_F32 || n_keys < 0 || kv_heads <= 0 || head_dim <= 0) return 0;
    return 4 * prompt_split_plane(n_keys, kv_heads, head_dim) + (size_t)n_keys * kv_heads * sizeof(float2);
}

int ojasx_b200_prompt_attention(const void* d_q, long long q_row, long long q_head, const void* d_k, long long k_row, long long k_head,
                                const void* d_v, long long v_row, long long v_head, void* d_out, const int* d_ends, const int* d_key_ends,
                                int batch, int n_rows, int n_keys, int q_heads, int kv_heads, int head_dim, float scale, int io_dtype,
                                void* workspace, size_t workspace_bytes, void* stream) {
    return ojasx_b200_prompt_attention_marked(d_q, q_row, q_head, d_k, k_row, k_head, d_v, v_row, v_head, d_out, d_ends, d_key_ends, nullptr, batch, n_rows,
                                              n_keys, q_heads, kv_heads, head_dim, scale, io_dtype, workspace, workspace_bytes, stream);
}

int ojasx_b200_prompt_attention_marked(const void* d_q, long long q_row, long long q_head, const void* d_k, long long k_row, long long k_head,
                                       const void* d_v, long long v_row, long long v_head, void* d_out, const int* d_ends, const int* d_key_ends,
                                       const unsigned char* d_none, int batch, int n_rows, int n_keys, int q_heads, int kv_heads, int head_dim,
                                       float scale, int io_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (!d_q || (n_keys > 0 && (!d_k || !d_v)) || !d_out || !d_ends || !d_key_ends || batch <= 0 || n_rows < 0 || n_keys < 0 || kv_heads <= 0 ||
        q_heads <= 0 || q_heads % kv_heads)
        return OJX_ERR_ARG;
    if (io_dtype != OJX_F32 && io_dtype != OJX_BF16) return OJX_ERR_ARG;
    const int unit = io_dtype == OJX_F32 ? 4 : 8;   // elements of 16 bytes
    for (const long long stride : {q_row, q_head, k_row, k_head, v_row, v_head})
        if (stride < 0 || stride % unit) return OJX_ERR_ARG;
    for (const void* p : {d_q, d_k, d_v, static_cast<const void*>(d_out), static_cast<const void*>(d_none)})
        if (reinterpret_cast<uintptr_t>(p) & 15) return OJX_ERR_ARG;
    if ((head_dim != 64 && head_dim != 128) || q_heads / kv_heads > 64) return OJX_ERR_UNSUPPORTED;
    const size_t need = ojasx_b200_prompt_workspace(n_keys, kv_heads, head_dim, io_dtype);
    if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < need)) return OJX_ERR_ARG;
    if (n_rows == 0) return OJX_OK;
    PromptProblem P{};
    P.q = d_q; P.k = d_k; P.v = d_v; P.out = d_out;
    P.q_row = q_row; P.q_head = q_head; P.k_row = k_row; P.k_head = k_head; P.v_row = v_row; P.v_head = v_head;
    P.ends = d_ends; P.key_ends = d_key_ends; P.none = d_none; P.batch = batch; P.n_rows = n_rows; P.n_keys = n_keys;
    P.q_heads = q_heads; P.kv_heads = kv_heads; P.share = q_heads / kv_heads;
    P.scale = scale > 0.0f ? scale : 1.0f / sqrtf((float)head_dim);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (io_dtype == OJX_BF16) return head_dim == 64 ? launch_prompt_tc<64>(P, s) : launch_prompt_tc<128>(P, s);
    return head_dim == 64 ? launch_prompt_pair<64>(P, workspace, s) : launch_prompt_pair<128>(P, workspace, s);
}

}  // extern "C"
