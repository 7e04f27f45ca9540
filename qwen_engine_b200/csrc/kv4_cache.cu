// The 4-bit key/value cache: rows in (bias, rotary position, quantisation), rows back as numbers, and eviction to fresh pages.
#include "kv4.cuh"
#include "kv4_attention.hpp"
#include "kv4_select.hpp"
#include "w4a16_internal.hpp"

namespace w4 {
namespace {

constexpr int kRowThreads = 16;          // a row is a half-warp's
constexpr int kAppendThreads = 256;      // 16 rows a CTA

struct AppendArgs {
    Kv4View c;
    const __half *q, *k, *v, *q_bias, *k_bias, *v_bias;
    __half* q_out;
    const int32_t* positions;
    const float* inv_freq;
    int q_heads, q_stride, kv_stride, blocks_per_token;
};

__device__ __forceinline__ void half4_to_float(uint2 w, float* x) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    x[0] = a.x;
    x[1] = a.y;
    x[2] = b.x;
    x[3] = b.y;
}
__device__ __forceinline__ uint4 float_to_half8(const float (&x)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// A row of 128 fp16 values in a half-warp: lane hl has 4 hl .. 4 hl + 3 and the same + 64, so that both values of a rotated pair are its
// own.  Returns the code word that the lane stores, number kv4_word_of(hl), and the row's (scale, zero).  Both halves of a warp call it.
// The codes are those of the formula in IEEE arithmetic: zero lies in the row's range, which is 15 scales and a half more where the scale is
// subnormal, so |quotient| < 23, and a product with the reciprocal is off by less than 5e-6 (three roundings); only where one lands
// nearer than 2e-5 to a border between two codes are the divisions made.  A row with an infinity or a NaN gets
// a NaN scale: it reads back as NaN instead of as finite values that it does not hold.
__device__ __forceinline__ int kv4_word_of(int hl) { return (hl & 1) * 8 + (hl >> 1); }
__device__ __forceinline__ uint32_t kv4_quantise_lane(const __half2 (&h)[4], int hl, uint32_t* params) {
    __half2 lo2 = __hmin2_nan(__hmin2_nan(h[0], h[1]), __hmin2_nan(h[2], h[3])), hi2 = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    // (smallest, minus the largest), so that one minimum reduces both
    __half2 ends = __halves2half2(__hmin_nan(__low2half(lo2), __high2half(lo2)), __hneg(__hmax_nan(__low2half(hi2), __high2half(hi2))));
#pragma unroll
    for (int m = 8; m > 0; m >>= 1) ends = __hmin2_nan(ends, __shfl_xor_sync(0xFFFFFFFFu, ends, m));
    const float lo = __low2float(ends), hi = -__high2float(ends);
    const bool finite = lo >= -65504.0f && hi <= 65504.0f;                  // false for a NaN
    __half scale = __float2half_rn(__fdiv_rn(hi - lo, 15.0f));
    const float s = __half2float(scale);
    __half zero = __float2half_rn(__fadd_rn(lo, 8.0f * s));
    const float z = __half2float(zero);
    uint32_t part[2] = {0x08080808u, 0x08080808u};
    if (finite && s > 0.0f) {
        const float inv = __frcp_rn(s);
        constexpr float kRound = 12582912.0f;                               // 1.5 * 2^23: adding it leaves the nearest integer in the low bits
        float d[8], t[8], off = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(h[j]);
            d[2 * j] = f.x - z;
            d[2 * j + 1] = f.y - z;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            t[j] = d[j] * inv;
            off = fmaxf(off, fabsf(t[j] - (__fadd_rn(t[j], kRound) - kRound)));
        }
        if (off > 0.5f - 2e-5f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = __fdiv_rn(d[j], s);
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            part[q] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float r = fminf(fmaxf(t[4 * q + j], -8.0f), 7.0f);     // rounds to the same code as what it cuts off
                part[q] |= (__float_as_uint(__fadd_rn(r, kRound + 8.0f)) & 15u) << (8 * j);
            }
        }
    }
    if (!finite) scale = zero = __ushort_as_half(0x7FFF);
    *params = static_cast<uint32_t>(__half_as_ushort(scale)) | (static_cast<uint32_t>(__half_as_ushort(zero)) << 16);
    // an even lane has elements 0..3 of its words, an odd one 4..7; the even one finishes the first word, the odd one the second
    const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, hl & 1 ? part[0] : part[1], 1);
    return hl & 1 ? (part[1] << 4) | other : part[0] | (other << 4);
}

// Where a token of the batch goes.
struct Spot {
    int seq, at, page;       // seq < 0: the token belongs to no sequence; page < 0: it has no place in the cache
};
__device__ __forceinline__ Spot find_spot(const Kv4View& c, int token) {     // a whole warp calls it
    Spot s{-1, 0, -1};
    if (token >= c.num_tokens) return s;
    const int seq = kv4_seq_of_token(c, token);
    if (seq >= c.num_seqs) return s;
    const int2 mine = kv4_new_tokens(c, seq);
    if (token < mine.x || token >= mine.x + mine.y) return s;
    s.seq = seq;
    s.at = __ldcg(c.lens + seq) - mine.y + (token - mine.x);
    if (s.at >= 0 && s.at < kv4_capacity(c)) {
        const int page = kv4_page(c, seq, s.at);
        if (static_cast<unsigned>(page) < static_cast<unsigned>(c.num_pages)) s.page = page;
    }
    return s;
}

// The rows of TOK tokens: q_heads of q (rotated into q_out), kv_heads of k (rotated, quantised), kv_heads of v (quantised).
// A CTA takes 16 of a token's rows; all its rows are requested first, then a warp a token finds its place (three dependent
// round trips), then the threads share the tokens' 64 angles.  Angles are position * inv_freq in 64 bits, reduced to a turn
// there (a 32-bit angle of position 100 000 is off by 0.004 rad), and so are their sines; the products round one by one.  A rotated value is
// then the 32-bit formula's bit for bit, and no code of a key beside a border between two codes depends on how it was computed (32-bit
// sines and fused products moved one key in some millions by a whole step of its row; they cost 1 us less of 52).  What bounds a prompt are those round trips: with one token a
// CTA instead of four 4 prompts of up to 4100 tokens took 79 us.
template <int TOK>
__global__ void __launch_bounds__(kAppendThreads, 6) kv4_append_kernel(const __grid_constant__ AppendArgs a) {
    __shared__ __align__(16) float2 s_turn[TOK][kKvDim / 2];     // cosine, sine
    __shared__ Spot s_spot[TOK];
    __shared__ int s_pos[TOK];
    const Kv4View& c = a.c;
    const int token0 = blockIdx.x / a.blocks_per_token * TOK;
    const int row = (blockIdx.x % a.blocks_per_token) * (kAppendThreads / kRowThreads) + (threadIdx.x >> 4);
    const int hl = threadIdx.x & 15, warp = threadIdx.x >> 5;
    const int n_q = a.q != nullptr ? a.q_heads : 0, rows = n_q + 2 * c.kv_heads;
    // what the row is: 0 q, 1 k, 2 v
    const int kind = row < n_q ? 0 : row < n_q + c.kv_heads ? 1 : 2;
    const int head = row - (kind == 0 ? 0 : kind == 1 ? n_q : n_q + c.kv_heads);
    const bool on = row < rows;
    const __half* src = (kind == 0 ? a.q : kind == 1 ? a.k : a.v) + head * kKvDim + hl * 4;
    const int stride = kind == 0 ? a.q_stride : a.kv_stride;
    uint2 raw[TOK][2], bias[2] = {make_uint2(0, 0), make_uint2(0, 0)};
    auto fetch = [&]() {
        pdl_wait_prior_grids();
        pdl_release_dependents();
#pragma unroll
        for (int i = 0; i < TOK; ++i)
#pragma unroll
            for (int p = 0; p < 2; ++p)
                raw[i][p] = on && token0 + i < c.num_tokens ? __ldcg(reinterpret_cast<const uint2*>(src + static_cast<size_t>(token0 + i) * stride + 64 * p)) : make_uint2(0, 0);
        const __half* b = kind == 0 ? a.q_bias : kind == 1 ? a.k_bias : a.v_bias;
        if (on && b != nullptr) {
#pragma unroll
            for (int p = 0; p < 2; ++p) bias[p] = __ldcg(reinterpret_cast<const uint2*>(b + head * kKvDim + hl * 4 + 64 * p));
        }
    };
    const bool late = TOK == 1 && c.settled;                     // a decode step: place and angles in front of the wait
    if (!late) fetch();
    if (warp < TOK) {
        const int token = token0 + warp;
        int pos = 0;
        if (a.positions != nullptr && token < c.num_tokens) pos = __ldcg(a.positions + token);
        const Spot s = find_spot(c, token);
        if ((threadIdx.x & 31) == 0) {
            s_spot[warp] = s;
            s_pos[warp] = a.positions != nullptr ? pos : s.at;
        }
    }
    __syncthreads();
    if (a.inv_freq != nullptr) {
        for (int i = threadIdx.x; i < TOK * kKvDim / 2; i += kAppendThreads) {
            const double turns = static_cast<double>(s_pos[i >> 6]) * static_cast<double>(__ldcg(a.inv_freq + (i & 63))) * 0.15915494309189533577;
            double sn, cs;
            sincospi(2.0 * (turns - rint(turns)), &sn, &cs);
            s_turn[i >> 6][i & 63] = make_float2(static_cast<float>(cs), static_cast<float>(sn));
        }
    }
    if (late) fetch();
    __syncthreads();
    float bf[8];
    half4_to_float(bias[0], bf);
    half4_to_float(bias[1], bf + 4);
    const int ps = 1 << c.page_shift, part = kind - 1;
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
        const Spot s = s_spot[i];
        if (s.seq < 0) continue;                                 // behind the last sequence: left as it is
        float x[8];                                              // four values and the four 64 behind them
        half4_to_float(raw[i][0], x);
        half4_to_float(raw[i][1], x + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] += bf[j];
        if (a.inv_freq != nullptr && kind != 2) {
            const float4 t01 = reinterpret_cast<const float4*>(s_turn[i])[2 * hl], t23 = reinterpret_cast<const float4*>(s_turn[i])[2 * hl + 1];
            const float cs[4] = {t01.x, t01.z, t23.x, t23.z}, sn[4] = {t01.y, t01.w, t23.y, t23.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float u = x[j], v = x[j + 4];
                x[j] = __fsub_rn(__fmul_rn(u, cs[j]), __fmul_rn(v, sn[j]));
                x[j + 4] = __fadd_rn(__fmul_rn(v, cs[j]), __fmul_rn(u, sn[j]));
            }
        }
        const __half2 h[4] = {__floats2half2_rn(x[0], x[1]), __floats2half2_rn(x[2], x[3]), __floats2half2_rn(x[4], x[5]), __floats2half2_rn(x[6], x[7])};
        if (on && kind == 0) {
            __half* out = a.q_out + static_cast<size_t>(token0 + i) * a.q_stride + head * kKvDim + hl * 4;
            *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<const uint32_t*>(&h[0]), *reinterpret_cast<const uint32_t*>(&h[1]));
            *reinterpret_cast<uint2*>(out + 64) = make_uint2(*reinterpret_cast<const uint32_t*>(&h[2]), *reinterpret_cast<const uint32_t*>(&h[3]));
        }
        const bool stored = on && kind != 0 && s.page >= 0;
        if (__any_sync(0xFFFFFFFFu, stored)) {
            uint32_t params;
            const uint32_t word = kv4_quantise_lane(h, hl, &params);
            if (stored) {
                uint32_t* record = kv4_record_of_page(c, s.page, head);
                const int slot = s.at & (ps - 1);
                record[(part * ps + slot) * kKvRowWords + kv4_word_of(hl)] = word;
                if (hl == 0) {
                    record[(32 + part) * ps + slot] = params;
                    if (kind == 1 && c.key_weight != nullptr) c.key_weight[kv4_weight_index(c, s.page, head, s.at)] = 0.0f;
                }
            }
        }
    }
}

// The rows that an append of this batch writes, as fp16.  A half-warp a row, TOK tokens a CTA as above.
template <int TOK>
__global__ void __launch_bounds__(kAppendThreads) kv4_read_kernel(const __grid_constant__ Kv4View c, __half* k_out, __half* v_out, int blocks_per_token) {
    __shared__ Spot s_spot[TOK];
    pdl_wait_prior_grids();
    pdl_release_dependents();
    const int token0 = blockIdx.x / blocks_per_token * TOK;
    const int row = (blockIdx.x % blocks_per_token) * (kAppendThreads / kRowThreads) + (threadIdx.x >> 4);
    const int hl = threadIdx.x & 15, warp = threadIdx.x >> 5;
    if (warp < TOK) {
        const Spot s = find_spot(c, token0 + warp);
        if ((threadIdx.x & 31) == 0) s_spot[warp] = s;
    }
    __syncthreads();
    const int part = row >= c.kv_heads, head = row - part * c.kv_heads, ps = 1 << c.page_shift;
    __half* out = part ? v_out : k_out;
    if (row >= 2 * c.kv_heads || out == nullptr) return;
    uint32_t word[TOK], params[TOK];
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
        word[i] = params[i] = 0;                                 // a scale of zero: zeros
        const Spot s = s_spot[i];
        if (s.page < 0) continue;
        const uint32_t* record = kv4_record_of_page(c, s.page, head);
        const int slot = s.at & (ps - 1);
        word[i] = __ldcg(record + (part * ps + slot) * kKvRowWords + hl);
        params[i] = __ldcg(record + (32 + part) * ps + slot);
    }
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
        if (s_spot[i].seq < 0) continue;
        const float s = kv4_scale(params[i]), z = kv4_zero(params[i]);
        constexpr int kShift[8] = {0, 8, 16, 24, 4, 12, 20, 28};
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = fmaf(static_cast<float>(static_cast<int>((word[i] >> kShift[j]) & 15u) - 8), s, z);
            if (fabsf(x[j]) > 65504.0f) x[j] = copysignf(65504.0f, x[j]);    // the rounding of scale and zero may step over fp16's end
        }
        *reinterpret_cast<uint4*>(out + (static_cast<size_t>(token0 + i) * c.kv_heads + head) * kKvDim + hl * 8) = float_to_half8(x);
    }
}

// ---- eviction ------------------------------------------------------------------------------------------------

struct EvictArgs {
    Kv4View c;
    const int32_t* dst_table;
    int32_t* new_lens;
    int32_t* kept;                       // [num_seqs][kv_heads][budget]
    int dst_pages, budget, sink, recent;
    int cluster;                         // CTAs of a sequence and head
};

// Order of the weights as unsigned numbers: larger weight, larger key; a NaN is below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (!(w == w)) return 0u;
    w = w + 0.0f;                        // -0 and 0 are equal
    const uint32_t u = __float_as_uint(w);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Choice and copy in one launch, a cluster of CTAs for each sequence and head, a CTA for a slice of its positions:
//   1. the weights' keys into shared memory, four a thread and request (or, where a slice is longer, read again in every pass);
//   2. the n-th largest key of the middle part, narrowed down by histograms of 2048 bins over the range that is left.  The first
//      range is the weights from 2^-32 to 2^32, 32 bins an octave, with what is outside in the end bins: as many bins
//      over all 32 bits would be 4 an octave, where the lanes' additions meet.  The histograms stay where they are; the cluster
//      exchanges sums of 32 bins, then the 32 bins that matter (all bins of 7 other CTAs took 5 us a round);
//   3. every warp counts what stays of its run of positions; scans over warps and CTAs give each its first new position;
//   4. the same run again: new positions by ballot, the old ones written down in order;
//   5. the rows copied, shared out evenly over the cluster, eight lanes a position (16 bytes each), four positions in flight.
// Integer counts and a fixed order throughout, so equal weights fall the same way every time.
constexpr int kEvictThreads = 1024, kEvictWarps = kEvictThreads / 32;
constexpr int kEvictCoarse = kEvictBins / 32;
constexpr int kEvictCached = 16384;      // keys of a slice in shared memory
constexpr int kEvictMaxCluster = 8;

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t ld_cluster(const void* mine, uint32_t rank) {
    uint32_t at, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

__global__ void __launch_bounds__(kEvictThreads, 1) kv4_evict_kernel(const __grid_constant__ EvictArgs a) {
    extern __shared__ __align__(16) uint32_t s_keys[];           // [kEvictCached], written four at a time
    __shared__ uint32_t s_hist[kEvictBins], s_coarse[kEvictCoarse];
    __shared__ uint32_t s_warp[2][kEvictWarps];
    __shared__ uint32_t s_found[2], s_total[2];
    pdl_wait_prior_grids();
    pdl_release_dependents();
    const Kv4View& c = a.c;
    const uint32_t ranks = a.cluster, rank = ranks > 1 ? cluster_rank() : 0;
    const int pair = blockIdx.x / a.cluster, b = pair / c.kv_heads, head = pair - b * c.kv_heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto barrier = [&]() { if (ranks > 1) cluster_barrier(); else __syncthreads(); };
    const int len = min(max(__ldcg(c.lens + b), 0), kv4_capacity(c));
    const int keep = min(len, a.budget);
    int32_t* kept = a.kept + (static_cast<size_t>(b) * c.kv_heads + head) * a.budget;
    if (rank == 0) {
        if (head == 0 && tid == 0) a.new_lens[b] = keep;
        for (int i = keep + tid; i < a.budget; i += kEvictThreads) kept[i] = -1;
    }
    const bool all_stay = len <= a.budget;
    const int lo = all_stay ? len : a.sink, hi = all_stay ? len : len - a.recent;      // the middle: sink + recent <= budget < len
    const uint32_t want = all_stay ? 0u : static_cast<uint32_t>(a.budget - a.sink - a.recent);
    const int slice = (len / static_cast<int>(ranks) + 32) & ~31;                      // multiple of 32, times ranks above len - 1
    const int s0 = min(slice * static_cast<int>(rank), len), s1 = min(s0 + slice, len);
    const bool cached = slice <= kEvictCached;
    auto page_at = [&](int i) { return kv4_page(c, b, i); };
    auto key_from = [&](int i) -> uint32_t {
        const int page = page_at(i);
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(c.num_pages)) return 0u;
        return weight_key(__ldcg(c.key_weight + kv4_weight_index(c, page, head, i)));
    };
    auto key_at = [&](int i) -> uint32_t { return cached ? s_keys[i - s0] : key_from(i); };
    const int m0 = max(s0, lo), m1 = min(s1, hi);                                      // this CTA's share of the middle
    KeyRange range;
    uint32_t need = want;
    if (want > 0) {
        if (cached) {
            // quads lie in one page, and a page's weights are there whatever the length is
            constexpr int kDeep = 2;
            for (int i0 = s0 + 4 * tid; i0 < s1; i0 += kDeep * 4 * kEvictThreads) {
                int page[kDeep];
                float4 w[kDeep];
#pragma unroll
                for (int d = 0; d < kDeep; ++d) page[d] = i0 + d * 4 * kEvictThreads < s1 ? page_at(i0 + d * 4 * kEvictThreads) : -1;
#pragma unroll
                for (int d = 0; d < kDeep; ++d) {
                    const float none = __int_as_float(0x7FC00000);
                    w[d] = make_float4(none, none, none, none);
                    if (static_cast<unsigned>(page[d]) < static_cast<unsigned>(c.num_pages))
                        w[d] = __ldcg(reinterpret_cast<const float4*>(c.key_weight + kv4_weight_index(c, page[d], head, i0 + d * 4 * kEvictThreads)));
                }
#pragma unroll
                for (int d = 0; d < kDeep; ++d)
                    if (i0 + d * 4 * kEvictThreads < s1)
                        *reinterpret_cast<uint4*>(s_keys + i0 + d * 4 * kEvictThreads - s0) =
                            make_uint4(weight_key(w[d].x), weight_key(w[d].y), weight_key(w[d].z), weight_key(w[d].w));
            }
        }
        while (true) {
            for (int i = tid; i < kEvictBins; i += kEvictThreads) s_hist[i] = 0;
            __syncthreads();
            for (int i = m0 + tid; i < m1; i += kEvictThreads) {
                uint32_t k = key_at(i);
                if (range.clamp) k = min(max(k, range.first), range.last);
                if (k >= range.first && k <= range.last) atomicAdd(&s_hist[(k - range.first) >> range.shift], 1u);
            }
            __syncthreads();
            for (int k = warp; k < kEvictCoarse; k += kEvictWarps) {
                const uint32_t n = __reduce_add_sync(0xFFFFFFFFu, s_hist[32 * k + lane]);
                if (lane == 0) s_coarse[k] = n;
            }
            barrier();
            if (warp == 0) {
                // from the top: the group of 32 bins, then the bin, in which the count reaches `need`
                uint32_t left = need, group = 0;
#pragma unroll 1
                for (int level = 0; level < 3; ++level) {        // the upper half of the groups, the lower, the bins of the group found
                    const uint32_t* at = level < 2 ? &s_coarse[kEvictCoarse - 1 - 32 * level - lane] : &s_hist[32 * group + 31 - lane];
                    uint32_t n = 0, more[kEvictMaxCluster];
#pragma unroll
                    for (uint32_t r = 0; r < kEvictMaxCluster; ++r) more[r] = r < ranks ? (ranks > 1 ? ld_cluster(at, r) : *at) : 0u;
#pragma unroll
                    for (uint32_t r = 0; r < kEvictMaxCluster; ++r) n += more[r];
                    uint32_t upto = n;
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
                        if (lane >= d) upto += o;
                    }
                    const uint32_t reached = __ballot_sync(0xFFFFFFFFu, upto >= left);
                    if (reached == 0) {                          // the upper half does not reach it
                        left -= __shfl_sync(0xFFFFFFFFu, upto, 31);
                        continue;
                    }
                    const int l = __ffs(reached) - 1;
                    left -= __shfl_sync(0xFFFFFFFFu, upto - n, l);
                    if (level < 2) {
                        group = static_cast<uint32_t>(kEvictCoarse - 1 - 32 * level - l);
                        level = 1;
                    } else if (lane == 0) {
                        s_found[0] = 32 * group + 31 - l;
                        s_found[1] = left;
                    }
                }
            }
            barrier();                                           // and the histograms may be cleared
            const uint32_t bin = s_found[0];
            need = s_found[1];
            range = narrowed(range, bin);
            if (range.first == range.last) break;
            __syncthreads();                                     // s_found has been read
        }
    }
    const uint32_t prefix = range.first;
    // what stays: outside the middle, keys above `prefix`, and the first `need` of those equal to it
    const int run = ((s1 - s0 + kEvictWarps - 1) / kEvictWarps + 31) & ~31;
    const int r0 = min(s0 + warp * run, s1), r1 = min(r0 + run, s1);
    uint32_t above = 0, equal = 0;
    for (int i = r0 + lane; i < r1; i += 32) {
        if (i < lo || i >= hi) {
            ++above;
        } else if (want > 0) {
            const uint32_t k = key_at(i);
            above += k > prefix;
            equal += k == prefix;
        }
    }
    above = __reduce_add_sync(0xFFFFFFFFu, above);
    equal = __reduce_add_sync(0xFFFFFFFFu, equal);
    if (lane == 0) { s_warp[0][warp] = above; s_warp[1][warp] = equal; }
    __syncthreads();
    const uint32_t wa = lane < kEvictWarps ? s_warp[0][lane] : 0u, we = lane < kEvictWarps ? s_warp[1][lane] : 0u;
    if (tid < 32) {
        const uint32_t ta = __reduce_add_sync(0xFFFFFFFFu, wa), te = __reduce_add_sync(0xFFFFFFFFu, we);
        if (tid == 0) { s_total[0] = ta; s_total[1] = te; }
    }
    barrier();
    uint32_t at_above = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? wa : 0u), at_equal = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? we : 0u);
    for (uint32_t r = 0; r < rank; ++r) {
        at_above += ld_cluster(&s_total[0], r);
        at_equal += ld_cluster(&s_total[1], r);
    }
    for (int i0 = r0; i0 < r1; i0 += 32) {
        const int i = i0 + lane;
        bool more = false, same = false;
        if (i < r1) {
            if (i < lo || i >= hi) more = true;
            else if (want > 0) {
                const uint32_t k = key_at(i);
                more = k > prefix;
                same = k == prefix;
            }
        }
        const uint32_t mm = __ballot_sync(0xFFFFFFFFu, more), ms = __ballot_sync(0xFFFFFFFFu, same);
        const uint32_t below = (1u << lane) - 1u;
        const uint32_t eq = at_equal + __popc(ms & below);       // equal keys in front of this one
        const bool stay = more || (same && eq < need);
        const int at = static_cast<int>(at_above + __popc(mm & below) + min(eq, need));
        at_above += __popc(mm);
        at_equal += __popc(ms);
        if (stay && at < keep) __stcg(kept + at, i);
    }
    barrier();                                                   // the cluster's list is complete, and no CTA leaves while its totals are read
    const int ps = 1 << c.page_shift, sub = lane & 7, part = sub >> 2;
    constexpr int kMove = 4;
    const int groups = static_cast<int>(ranks) * (kEvictThreads / 8);
    for (int j0 = static_cast<int>(rank) * (kEvictThreads / 8) + (tid >> 3); j0 < keep; j0 += kMove * groups) {
        int i[kMove], from[kMove], to[kMove];
#pragma unroll
        for (int u = 0; u < kMove; ++u) {
            i[u] = j0 + u * groups < keep ? __ldcg(kept + j0 + u * groups) : -1;
            // weights that change while they are read can leave the list short: what it held before is no position
            if (static_cast<unsigned>(i[u]) >= static_cast<unsigned>(len)) i[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < kMove; ++u) {
            from[u] = to[u] = -1;
            if (i[u] >= 0) {
                from[u] = page_at(i[u]);
                to[u] = __ldcg(a.dst_table + static_cast<size_t>(b) * a.dst_pages + ((j0 + u * groups) >> c.page_shift));
            }
        }
        uint4 w[kMove];
        uint32_t extra[kMove];
#pragma unroll
        for (int u = 0; u < kMove; ++u) {
            // a page outside the pool moves nothing
            if (static_cast<unsigned>(to[u]) >= static_cast<unsigned>(c.num_pages)) from[u] = -1;
            const uint32_t* old = kv4_record_of_page(c, from[u], head);
            w[u] = make_uint4(0, 0, 0, 0);
            extra[u] = 0;
            if (old != nullptr) {
                const int slot = i[u] & (ps - 1);
                w[u] = __ldcg(reinterpret_cast<const uint4*>(old + (part * ps + slot) * kKvRowWords) + (sub & 3));
                if (sub < 2) extra[u] = __ldcg(old + (32 + sub) * ps + slot);
                if (sub == 2) extra[u] = __ldcg(reinterpret_cast<const uint32_t*>(c.key_weight) + kv4_weight_index(c, from[u], head, i[u]));
            }
        }
#pragma unroll
        for (int u = 0; u < kMove; ++u) {
            if (static_cast<unsigned>(from[u]) >= static_cast<unsigned>(c.num_pages)) continue;
            uint32_t* fresh = kv4_record_of_page(c, to[u], head);
            const int j = j0 + u * groups, slot = j & (ps - 1);
            *(reinterpret_cast<uint4*>(fresh + (part * ps + slot) * kKvRowWords) + (sub & 3)) = w[u];
            if (sub < 2) fresh[(32 + sub) * ps + slot] = extra[u];
            if (sub == 2) reinterpret_cast<uint32_t*>(c.key_weight)[kv4_weight_index(c, to[u], head, j)] = extra[u];
        }
    }
}

}  // namespace

// Four tokens a CTA where that leaves every SM enough CTAs: one token 4.9 us an append + read, either way; 4 prompts of 2100 to
// 4100 tokens see the kernel.
static int tokens_per_cta(int num_tokens, int blocks_per_token) { return static_cast<long long>(num_tokens) * blocks_per_token >= 4 * 148 * 4 ? 4 : 1; }

int kv4_append(const Kv4View& c, const Kv4AppendArgs& x, cudaStream_t stream) {
    AppendArgs a{c, x.q, x.k, x.v, x.q_bias, x.k_bias, x.v_bias, x.q_out, x.positions, x.inv_freq, x.q_heads, x.q_stride, x.kv_stride, 0};
    const int rows = (x.q != nullptr ? x.q_heads : 0) + 2 * c.kv_heads;
    a.blocks_per_token = (rows + 15) / 16;
    const int tok = tokens_per_cta(c.num_tokens, a.blocks_per_token);
    const long long blocks = static_cast<long long>(a.blocks_per_token) * ((c.num_tokens + tok - 1) / tok);
    if (blocks > 0x7FFFFFFFll) return W4A16_ERR_TOO_LARGE;
    return static_cast<int>(launch_kernel(tok == 4 ? kv4_append_kernel<4> : kv4_append_kernel<1>, dim3(static_cast<unsigned>(blocks)), dim3(kAppendThreads), 0,
                                          stream, pdl_enabled(), a));
}

int kv4_read(const Kv4View& c, __half* k_out, __half* v_out, cudaStream_t stream) {
    const int per = (2 * c.kv_heads + 15) / 16, tok = tokens_per_cta(c.num_tokens, per);
    const long long blocks = static_cast<long long>(per) * ((c.num_tokens + tok - 1) / tok);
    if (blocks > 0x7FFFFFFFll) return W4A16_ERR_TOO_LARGE;
    return static_cast<int>(launch_kernel(tok == 4 ? kv4_read_kernel<4> : kv4_read_kernel<1>, dim3(static_cast<unsigned>(blocks)), dim3(kAppendThreads), 0, stream,
                                          pdl_enabled(), c, k_out, v_out, per));
}

int kv4_set_attributes() {
    return static_cast<int>(cudaFuncSetAttribute(kv4_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvictCached * 4));
}

int kv4_evict(const Kv4View& c, const Kv4EvictArgs& x, cudaStream_t stream) {
    EvictArgs a{c, x.dst_table, x.new_lens, x.kept, x.dst_pages, x.budget, x.sink, x.recent, 1};
    // CTAs of a (sequence, head): about 4096 positions each while all have an SM of their own (clusters of 8 fill no more than 96:
    // 16 of them took 35 us for what 16 of 4 do in 26), and as many more as it takes to keep the keys in shared memory
    const long long capacity = static_cast<long long>(c.max_pages) << c.page_shift, pairs = static_cast<long long>(c.num_seqs) * c.kv_heads;
    while (a.cluster < kEvictMaxCluster && capacity > 4096ll * a.cluster && (pairs * a.cluster * 2 <= (a.cluster < 4 ? 148 : 96) || capacity > static_cast<long long>(kEvictCached) * a.cluster))
        a.cluster *= 2;
    if (pairs * a.cluster > 0x7FFFFFFFll) return W4A16_ERR_TOO_LARGE;
    const long long slice = capacity / a.cluster + 64;
    const size_t smem = static_cast<size_t>(slice < kEvictCached ? slice : kEvictCached) * 4;
    return static_cast<int>(launch_kernel_cluster(kv4_evict_kernel, dim3(static_cast<unsigned>(pairs * a.cluster)), dim3(kEvictThreads), smem, stream, pdl_enabled(),
                                                  dim3(a.cluster), a));
}

}  // namespace w4
