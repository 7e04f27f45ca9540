// How the attention kernels over the 4-bit key/value cache cut a batch: query rows, units of positions, and the place of a CTA.
#pragma once

#include "kv4.cuh"

namespace w4 {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// A unit is 64 positions (16 a warp) against one tile of query rows and one head; units are numbered by
// sequence, tile, head, position, and every CTA of a persistent grid takes the same number of consecutive ones.  So the CTAs
// finish together whatever the lengths are (they live on the device, the host does not know them), and a CTA has at most two
// parts of a (tile, head) that others have parts of too: its first and its last one.
constexpr int kUnit = 64;

struct SeqWork {
    int first, n;                 // rows of the batch
    int past;                     // positions in front of the first new token (negative: tokens without a position)
    int tiles, units;             // tiles of query rows; units of one tile and head
};
__device__ __forceinline__ SeqWork seq_work(const Kv4View& c, int b, int group, int tile_rows) {
    SeqWork w;
    const int2 mine = kv4_new_tokens(c, b);
    const int len = max(__ldcg(c.lens + b), 0);
    w.first = mine.x;
    w.n = mine.y;
    w.past = len - mine.y;
    w.tiles = (mine.y * group + tile_rows - 1) / tile_rows;
    w.units = max(1, (min(len, kv4_capacity(c)) + kUnit - 1) / kUnit);
    return w;
}
// A place in the order of the units.
struct Place {
    SeqWork w;
    int seq;
    long long in_seq;             // unit (or tile and head) of the sequence
    long long units_before;       // units of the sequences in front
};
template <int THREADS>
struct FindScratch {
    longlong2 sums[THREADS / 32]; // units; units or tiles and heads
    Place found;
};
__device__ __forceinline__ long long ceil_div(long long a, int b) {
    // a division of 64 bits is a long subroutine in the way of the first load
    return a >> 31 == 0 ? static_cast<long long>((static_cast<uint32_t>(a) + static_cast<uint32_t>(b) - 1u) / static_cast<uint32_t>(b)) : (a + b - 1) / b;
}
// Units of the whole batch, per = ceil(all / parts), and the place of unit `per * index` or, with BY_TILE, of the (tile, head)
// number `index`; false where there is none.  All threads of the CTA call it.  One round trip, for up to THREADS sequences.
template <int THREADS, bool BY_TILE = false>
__device__ __forceinline__ bool find_unit(const Kv4View& c, int group, int tile_rows, int index, int parts, FindScratch<THREADS>& s, long long* per, long long* all, Place* out) {
    const int tid = threadIdx.x, lane = tid & 31, each = (c.num_seqs + THREADS - 1) / THREADS;
    const int b0 = min(tid * each, c.num_seqs), b1 = min(b0 + each, c.num_seqs);
    longlong2 mine = {0, 0};
    SeqWork w{};
    auto count = [&](longlong2& n) {
        const long long tiles = static_cast<long long>(w.tiles) * c.kv_heads;
        n.x += tiles * w.units;
        n.y += tiles;
    };
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
        w = seq_work(c, b, group, tile_rows);
        count(mine);
    }
    longlong2 upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long x = __shfl_up_sync(0xFFFFFFFFu, upto.x, d), y = BY_TILE ? __shfl_up_sync(0xFFFFFFFFu, upto.y, d) : 0;
        if (lane >= d) { upto.x += x; upto.y += y; }
    }
    if (lane == 31) s.sums[tid >> 5] = upto;
    __syncthreads();
    longlong2 total = {0, 0};
    longlong2 at = {upto.x - mine.x, upto.y - mine.y};
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
        if (i == tid >> 5) { at.x += total.x; at.y += total.y; }
        total.x += s.sums[i].x;
        total.y += s.sums[i].y;
    }
    *all = total.x;
    *per = ceil_div(total.x, parts);
    const long long want = BY_TILE ? index : *per * index;
    if (want >= (BY_TILE ? total.y : total.x)) return false;
    if ((BY_TILE ? at.y : at.x) <= want && want < (BY_TILE ? at.y + mine.y : at.x + mine.x)) {        // the sequence is one of this thread's
        for (int b = b0; b < b1; ++b) {
            if (each > 1) w = seq_work(c, b, group, tile_rows);
            longlong2 next = at;
            count(next);
            if (want < (BY_TILE ? next.y : next.x)) {
                s.found = Place{w, b, want - (BY_TILE ? at.y : at.x), at.x};
                break;
            }
            at = next;
        }
    }
    __syncthreads();
    *out = s.found;
    return true;
}

// Output row r of a tile.
__device__ __forceinline__ size_t out_row(const SeqWork& w, int heads, int group, int head, int row) {
    return static_cast<size_t>(w.first + row / group) * (static_cast<size_t>(heads) * group) + head * group + row % group;
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Results: an average of finite values can step over fp16's end by the roundings of scales, zeros and weights; it is cut there.
__device__ __forceinline__ uint32_t pack_result(float a, float b) {
    const __half2 end = __float2half2_rn(65504.0f), h = __hmax2_nan(__hmin2_nan(__floats2half2_rn(a, b), end), __hneg2(end));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float sum_half8(const uint4& w) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        s += f.x + f.y;
    }
    return s;
}
// One part's four dimensions, with its maximum and sum, into a sum around `top` (the largest maximum).  A part without any
// position has maximum -infinity and sum 0; where all parts are such, the factor is 1 and what is added is 0.
__device__ __forceinline__ void add_part(float4& x, float& sum, const float4& p, float2 ml, float top) {
    const float f = ml.x == top ? 1.0f : ex2(ml.x - top);
    sum = fmaf(ml.y, f, sum);
    x.x = fmaf(p.x, f, x.x);
    x.y = fmaf(p.y, f, x.y);
    x.z = fmaf(p.z, f, x.z);
    x.w = fmaf(p.w, f, x.w);
}
// top + log2(sum).  The sum may be far from 1, and its exponent goes to top first, where the two cancel.
__device__ __forceinline__ float log2_of_sum(float top, float sum) {
    const uint32_t bits = __float_as_uint(sum);
    const int e = static_cast<int>(bits >> 23 & 255u) - 127; // 128: an infinity or a NaN
    return e == 128 ? top + sum : (top + static_cast<float>(e)) + log2f(__uint_as_float((bits & 0x007FFFFFu) | 0x3F800000u));
}
// A finished row: a warp, four dimensions a lane.
template <bool F32>
__device__ __forceinline__ void store_row(void* out, float* lse, size_t row, const float4& x, float top, float sum) {
    const int lane = threadIdx.x & 31;
    const float f = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
    const float4 y = sum == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
    if constexpr (F32) {
        reinterpret_cast<float4*>(static_cast<float*>(out) + row * kKvDim)[lane] = y;
    } else {
        const uint2 h = make_uint2(pack_result(y.x, y.y), pack_result(y.z, y.w));
        reinterpret_cast<uint2*>(static_cast<__half*>(out) + row * kKvDim)[lane] = h;
    }
    if (lane == 0 && lse != nullptr) lse[row] = sum == 0.0f ? -INFINITY : log2_of_sum(top, sum) * kLn2;
}

}  // namespace
}  // namespace w4
