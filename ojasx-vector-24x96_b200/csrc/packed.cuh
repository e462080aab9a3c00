// Packed sequences: row r of a [rows, ...] tensor belongs to the sequence b with ends[b] <= r < ends[b + 1].
#pragma once
#include "common.cuh"

namespace ojx {

struct PackedRange { int first, count; };

// Rows of sequence b, kept inside the tensor whatever `ends` holds.
__device__ __forceinline__ PackedRange packed_range(const int* __restrict__ ends, int b, int rows) {
    const int first = min(max(ends[b], 0), rows);
    return {first, min(max(ends[b + 1], first), rows) - first};
}

// Sequence of a row, or -1 for a row behind the last one.  `ends` ascends from 0.
__device__ __forceinline__ int packed_owner(const int* __restrict__ ends, int batch, int row) {
    int lo = 0, hi = batch;   // ends[lo] <= row < ends[hi], if any
    if (row < ends[0] || row >= ends[batch]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] <= row) lo = mid; else hi = mid;
    }
    return lo;
}

// Part `index` of all sequences, cut into `parts(b)` parts each, in order: its sequence and its number there.  All lanes of a warp
// call it together; false behind the last part.
template <class Parts>
__device__ __forceinline__ bool packed_part(int batch, int index, Parts parts, int& seq, int& part) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int b0 = 0; b0 < batch; b0 += 32) {
        const int mine = b0 + lane < batch ? parts(b0 + lane) : 0;
        int sum = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, sum, off);
            if (lane >= off) sum += o;
        }
        const unsigned in = __ballot_sync(0xffffffffu, index < before + sum);
        if (in) {
            const int src = __ffs(in) - 1;
            seq = b0 + src;
            part = index - before - __shfl_sync(0xffffffffu, sum - mine, src);
            return true;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return false;
}

// NaN for results that a launch gave up on: `heads` heads from `head` on of `rows` rows from `row` on of a [.., all_heads, HD] tensor.
// `thread` of `threads` that call it.
template <int HD, class T>
__device__ __forceinline__ void packed_give_up(T* out, size_t row, int rows, int head, int heads, int all_heads, int thread, int threads) {
    for (int i = thread; i < rows * heads * HD; i += threads) {
        const int r = i / (heads * HD);
        out[((row + r) * all_heads + head) * HD + i - r * (heads * HD)] = T(__int_as_float(0x7fffffff));
    }
}

}  // namespace ojx
