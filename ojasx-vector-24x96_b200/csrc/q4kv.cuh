// Layout of the 4-bit paged KV cache.
//
// 32 consecutive dimensions of a token's key or value form a group with a bf16 minimum and a bf16 scale: minimum = floor(min x) and
// scale = ceil((max x - minimum) / 15), to the neighbouring bf16 number, code = round((x - minimum) / scale) in 0..15.  Rounding the
// two outwards keeps every x of the group inside the 16 steps, so that it is read back within half a step.  A group with a value
// that is not finite, or below the lowest bf16 number, has a scale of zero and a NaN for its minimum, and is read back as NaN.  (The
// largest code of a group whose maximum is beyond 3.37e38 may stand for an infinity.)
//
// A page of one KV head is page_size / 16 tiles of 16 tokens, each contiguous (2560 bytes at head_dim 128), pools are
// [pages][kv_heads][tiles].  A tile is laid out as the operands of mma.sync m16n8k16 that the decode kernel makes of it, so that
// every lane reads whole 8- or 16-byte pieces, G = head_dim / 32 groups:
//   keys     [token][t = 0..3][g]: words; word (t, g) holds dimensions 32 g + 8 t + j in nibble j
//   their    scales, minima [token][g]
//   values   [half][c = 0..7][pair = 0..3][g]: words; tokens 8 half + 2 pair (low 16 bits) and + 1 (high 16 bits), dimensions
//            32 g + 4 c + i in nibble i of either
//   their    scales, minima [token][g]
#pragma once
#include "common.cuh"
#include "../../include/ojasx_lut_b200.h"

namespace ojx {

constexpr int kQ4Group = 32;
constexpr int kQ4Tile = 16;    // tokens of a tile

template <int HD>
struct Q4Layout {
    static constexpr int G = HD / kQ4Group;
    static constexpr int codes = kQ4Tile * HD / 2, metas = kQ4Tile * G * 2;
    static constexpr int key_scales = codes, key_mins = key_scales + metas;
    static constexpr int values = key_mins + metas;
    static constexpr int value_scales = values + codes, value_mins = value_scales + metas;
    static constexpr int bytes = value_mins + metas;
    // dimensions 32 g + 4 c .. + 3 of a token, as 16 bits
    __host__ __device__ static constexpr int key_at(int token, int g, int c) { return ((token * 4 + (c >> 1)) * G + g) * 4 + (c & 1) * 2; }
    __host__ __device__ static constexpr int value_at(int token, int g, int c) {
        return values + ((((token >> 3) * 8 + c) * 4 + ((token >> 1) & 3)) * G + g) * 4 + (token & 1) * 2;
    }
    __host__ __device__ static constexpr int meta_at(int token, int g) { return (token * G + g) * 2; }   // from any of the four
};

struct Q4Cache {
    uint8_t* pool;              // [num_pages][kv_heads][page_size / 16][tile]
    const int* block_table;     // [batch][max_pages] page ids; ids outside [0, num_pages) hold nothing
    int* status;                // set to 1 where a token has no page
    int max_pages, num_pages, page_size, kv_heads;
};

// Tile of `token` of sequence b for one KV head, or null where the table has no page for it.
template <int HD>
__device__ __forceinline__ uint8_t* q4_tile(const Q4Cache& C, int b, int head, int token) {
    const int p = token / C.page_size;
    if (token < 0 || p >= C.max_pages) return nullptr;
    const int id = C.block_table[(size_t)b * C.max_pages + p];
    if ((unsigned)id >= (unsigned)C.num_pages) return nullptr;
    const int tiles = C.page_size / kQ4Tile;
    return C.pool + (((size_t)id * C.kv_heads + head) * tiles + (token - p * C.page_size) / kQ4Tile) * Q4Layout<HD>::bytes;
}

// A scale or minimum, and the two in a word.
__device__ __forceinline__ float q4_bf16(unsigned short b) { return __uint_as_float((unsigned)b << 16); }
__device__ __forceinline__ float q4_low(unsigned w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float q4_high(unsigned w) { return __uint_as_float(w & 0xffff0000u); }

// What every entry point asks of a cache.
inline int q4_check(const OjasxQ4Cache* c, const int* table, int max_pages, int batch, int dtype) {
    if (!c || !c->pool || !c->status || !table || max_pages <= 0 || c->num_pages <= 0 || c->kv_heads <= 0 || c->q_heads <= 0 || c->q_heads % c->kv_heads || batch <= 0)
        return OJX_ERR_ARG;
    if (dtype != OJX_F32 && dtype != OJX_BF16) return OJX_ERR_ARG;
    if (c->page_size <= 0 || c->page_size % kQ4Tile || (c->head_dim != 64 && c->head_dim != 128)) return OJX_ERR_UNSUPPORTED;
    if ((long long)max_pages * c->page_size > 0x7fffffffLL) return OJX_ERR_TOO_LARGE;
    return (reinterpret_cast<uintptr_t>(c->pool) & 15) ? OJX_ERR_ARG : OJX_OK;
}
inline Q4Cache q4_cache(const OjasxQ4Cache* c, const int* table, int max_pages) {
    return {static_cast<uint8_t*>(c->pool), table, c->status, max_pages, c->num_pages, c->page_size, c->kv_heads};
}
inline bool q4_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace ojx
