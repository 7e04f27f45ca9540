// The 4-bit key/value cache: layout, index arithmetic and conversions shared by its kernels (sm_100a).
//
// A page record holds page_size rows of one key/value head, 34 words a position:
//   key codes [page_size][16] | value codes [page_size][16] | key (scale, zero) [page_size] | value (scale, zero) [page_size]
// A row is 128 values quantised as one group with a zero point: value = (code - 8) * scale + zero; its 16 words are packed as
// the library's weight words are (element j of a word at bit {0, 8, 16, 24, 4, 12, 20, 28}[j]); (scale, zero) is an fp16 pair
// with the scale in the low half.  8 is subtracted for the same reason as in the weights: the products of a long sum then
// have both signs, and the 32-bit accumulators of the tensor cores do not grow with its length.
//
// Every index that comes from device memory is checked before it forms an address: lengths are cut at what the block table
// can hold, a page number outside the pool makes its positions unreadable (append drops them, read gives zero, attention does
// not see them).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "w4a16_common.cuh"

namespace w4 {

constexpr int kKvDim = 128;              // values of a head
constexpr int kKvRowWords = 16;          // words of codes of a row
constexpr int kKvSlotWords = 34;         // words of a position in a record
constexpr int kKvTile = 16;              // positions that lie in one page for certain

struct Kv4View {
    uint32_t* pages;
    float* key_weight;                   // [num_pages][kv_heads][page_size] or null
    const int32_t* table;                // [num_seqs][max_pages]
    const int32_t* lens;                 // [num_seqs]
    const int32_t* qstart;               // [num_seqs + 1] or null: one token a sequence
    int num_pages, kv_heads, page_shift, num_seqs, max_pages, num_tokens;
    // No launch that may still run when this one starts writes table, lens, qstart or the positions of the call: they are read before
    // the wait for the launches in front.  The decode sweep can promise it (its graph writes none of them), a single call cannot: a
    // sampler that counts a position on may be two early launches ahead.
    bool settled = false;
};

// New tokens of sequence b: first row of the batch and count, both inside the batch whatever the array holds.
__device__ __forceinline__ int2 kv4_new_tokens(const Kv4View& c, int b) {
    if (c.qstart == nullptr) return make_int2(b, b < c.num_tokens ? 1 : 0);
    const int first = min(max(__ldcg(c.qstart + b), 0), c.num_tokens);
    const int end = min(max(__ldcg(c.qstart + b + 1), first), c.num_tokens);
    return make_int2(first, end - first);
}
__device__ __forceinline__ int kv4_capacity(const Kv4View& c) {
    return c.max_pages << c.page_shift;       // at most 2^30: the entry points see to it
}
// The record of position `at` of a sequence and head; null where the table has no page of the pool there.
__device__ __forceinline__ uint32_t* kv4_record_of_page(const Kv4View& c, int page, int head) {
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(c.num_pages)) return nullptr;
    const size_t record = static_cast<size_t>(page) * c.kv_heads + head;
    return c.pages + ((record * kKvSlotWords) << c.page_shift);
}
__device__ __forceinline__ int kv4_page(const Kv4View& c, int b, int at) {
    return __ldcg(c.table + static_cast<size_t>(b) * c.max_pages + (at >> c.page_shift));
}
__device__ __forceinline__ size_t kv4_weight_index(const Kv4View& c, int page, int head, int at) {
    return (((static_cast<size_t>(page) * c.kv_heads + head) << c.page_shift) | (at & ((1 << c.page_shift) - 1)));
}

// Sequence of a token: how many sequences end at or before it.  A whole warp calls it; one round trip for up to 32 sequences.
__device__ __forceinline__ int kv4_seq_of_token(const Kv4View& c, int token) {
    if (c.qstart == nullptr) return token;
    int before = 0;
    for (int i = threadIdx.x & 31; i < c.num_seqs; i += 32) before += __ldcg(c.qstart + i + 1) <= token;
    return __reduce_add_sync(0xFFFFFFFFu, before);
}

__device__ __forceinline__ float kv4_scale(uint32_t params) { return __half2float(__ushort_as_half(static_cast<unsigned short>(params))); }
__device__ __forceinline__ float kv4_zero(uint32_t params) { return __half2float(__ushort_as_half(static_cast<unsigned short>(params >> 16))); }

// Four pairs (code - 8) out of a word as fp16: pair n holds the nibbles at bits 4 n and 16 + 4 n.  0x6400 | c is 1024 + c and
// 0x6400 | c << 4 is 1024 + 16 c, so one addition or one fma gives c - 8, exactly.  (In the low bits of a half a nibble is a subnormal
// number already, and a mask would do for keys; but the tensor core lines products up by their exponents, a subnormal's has leading
// zeros behind it, and 32-bit results were off by 2e-6 where they are now by 3e-7, for 3 % of a large batch's time.)
__device__ __forceinline__ void kv4_centred_codes(uint32_t w, uint32_t (&out)[4]) {
    const __half2 a = __float2half2_rn(-1032.0f), m = __float2half2_rn(0.0625f), b = __float2half2_rn(-72.0f);
    const uint32_t u = w >> 8;
    uint32_t r[4];
    asm("lop3.b32 %0, %1, 0x000F000F, 0x64006400, 0xEA;" : "=r"(r[0]) : "r"(w));
    asm("lop3.b32 %0, %1, 0x00F000F0, 0x64006400, 0xEA;" : "=r"(r[1]) : "r"(w));
    asm("lop3.b32 %0, %1, 0x000F000F, 0x64006400, 0xEA;" : "=r"(r[2]) : "r"(u));
    asm("lop3.b32 %0, %1, 0x00F000F0, 0x64006400, 0xEA;" : "=r"(r[3]) : "r"(u));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 c = *reinterpret_cast<const __half2*>(&r[i]), v = i & 1 ? __hfma2(c, m, b) : __hadd2(c, a);
        out[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
}
// The same for values, whose nibble places are different rows of A: pair n holds (code - 7.5) times 2^-9 (n even) or 2^-5
// (n odd), which the row's sums carry to the end.  One fma takes the subnormal numbers there; codes taken around 7.5, their mean, leave sums that do not grow with the number of positions, where the
// tensor core's truncation would all go one way (at 131 001 positions the output's error against 64 bits fell from 6.5e-6).
__device__ __forceinline__ void kv4_value_codes_to_half2(uint32_t w, uint32_t (&out)[4]) {
    const __half2 m = __float2half2_rn(32768.0f), lo = __float2half2_rn(-7.5f / 512.0f), hi = __float2half2_rn(-7.5f / 32.0f);
    const uint32_t u = w >> 8;
    const uint32_t r[4] = {w & 0x000F000Fu, w & 0x00F000F0u, u & 0x000F000Fu, u & 0x00F000F0u};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&r[i]), m, i & 1 ? hi : lo);
        out[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
}
__device__ __forceinline__ float kv4_value_undo(int pair) { return pair & 1 ? 32.0f : 512.0f; }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace w4
