// The cache that holds keys and values in 4 bits: its layout and its numbers, shared by the kernels that write and read it.
//
// Of a token's key (value) of one kv head, D numbers x, are kept a scale s = bf16(max x / 15 - min x / 15), a minimum
// m = bf16(min x) and a code n = round((x - m) / s) in 0 .. 15 per number; a code stands for m + s n. One scale and one minimum per
// vector: 8 bytes for a key and its value beside D bytes of codes (136 bytes at D = 128, where 16 bits take 512), and the scores and sums
// can be taken on the codes alone, s and m coming in once per (row, key).
//
// A layer's cache is uint8 [pages, kv heads, page size, W], W = 32 C + 8 bytes per token, C = ceil(D / 32) chunks of 32 numbers.
// Eight tokens of one page and kv head, positions 8i .. 8i + 7, lie together (page sizes are multiples of 8), so that any run of them is
// contiguous whatever the page size, and a chunk of eight tokens is 128 bytes that ldmatrix reads without a bank conflict:
//   [C][8 tokens][16 bytes]   codes of the keys; byte b of a chunk: number 2b in its low four bits, 2b + 1 in its high ones
//   [C][8 tokens][16 bytes]   codes of the values
//   [8 tokens][4 bfloat16]    s and m of the key, s and m of the value
// What D leaves of the last chunk holds zeros.
#pragma once
#include "common.cuh"

namespace vob_kv4 {

constexpr int GROUP = 8;                                                            // tokens that lie together
__host__ __device__ constexpr int chunks(int hd) { return (hd + 31) / 32; }
__host__ __device__ constexpr int token_bytes(int hd) { return 32 * chunks(hd) + 8; }

// First byte of the group of eight tokens that holds token `off` of a page.
__device__ __forceinline__ size_t group_at(size_t page, int head, int off, int kv_heads, int page_size, int width) {
    return ((page * kv_heads + head) * page_size + (off & ~7)) * (size_t)width;
}

// s and m of a key or value from the two bfloat16 of one 32-bit word.
__device__ __forceinline__ float2 scale_min(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ bool is_finite2(float2 a) { return isfinite(a.x) && isfinite(a.y); }

// s and m of a key and its value, as attention takes them. A value that is not finite (its token's projection was not) is taken as 0
// and its key as NaN: the rows that see the token become NaN through their scores, and no other row does, as 0 * NaN would make them
// where a product is taken over tokens that a row's mask hides.
__device__ __forceinline__ void attend_scales(uint2 p, float2& key, float2& val) {
    key = scale_min(p.x);
    val = scale_min(p.y);
    if (!is_finite2(val)) {
        key = make_float2(NAN, NAN);
        val = make_float2(0.f, 0.f);
    }
}

}  // namespace vob_kv4
