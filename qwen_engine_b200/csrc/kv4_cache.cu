// The 4-bit key/value cache: rows in (bias, rotary position, quantisation), rows back as numbers, and eviction to fresh pages.
#include "kv4.cuh"
#include "kv4_attention.hpp"
#include "w4a16_internal.hpp"

namespace w4 {
namespace {

constexpr int kRowThreads = 16;          // a row is a half-warp's: 8 values a lane
constexpr int kAppendThreads = 256;      // 16 rows a CTA

struct AppendArgs {
    Kv4View c;
    const __half *q, *k, *v, *q_bias, *k_bias, *v_bias;
    __half* q_out;
    const int32_t* positions;
    const float* inv_freq;
    int q_heads, q_stride, kv_stride, blocks_per_token;
};

__device__ __forceinline__ void half8_to_float(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
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

// One row of 128 fp16 values, 8 a lane of a half-warp, to its code word and (scale, zero).  Both halves of a warp call it.
// IEEE division and rounding throughout, so the codes are those of the formula.  A row with an infinity or a NaN gets a
// NaN scale: it reads back as NaN instead of as finite values that it does not hold.
__device__ __forceinline__ uint32_t kv4_quantise_lane(const float (&x)[8], uint32_t* params) {
    float lo = x[0], hi = x[0];
    bool finite = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
        finite = finite && fabsf(x[j]) <= 65504.0f;
    }
#pragma unroll
    for (int m = 8; m > 0; m >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, m));
        hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, m));
    }
    const uint32_t all = __ballot_sync(0xFFFFFFFFu, finite);
    const bool row_finite = ((threadIdx.x & 16 ? all >> 16 : all) & 0xFFFFu) == 0xFFFFu;
    __half scale = __float2half_rn(__fdiv_rn(hi - lo, 15.0f));
    const float s = __half2float(scale);
    __half zero = __float2half_rn(__fadd_rn(lo, 8.0f * s));
    const float z = __half2float(zero);
    uint32_t word = 0;
    constexpr int kShift[8] = {0, 8, 16, 24, 4, 12, 20, 28};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        int code = 8;
        if (row_finite && s > 0.0f) code = min(max(__float2int_rn(__fdiv_rn(x[j] - z, s)) + 8, 0), 15);
        word |= static_cast<uint32_t>(code) << kShift[j];
    }
    if (!row_finite) scale = zero = __ushort_as_half(0x7FFF);
    *params = static_cast<uint32_t>(__half_as_ushort(scale)) | (static_cast<uint32_t>(__half_as_ushort(zero)) << 16);
    return word;
}

// One token's rows: q_heads of q (rotated into q_out), kv_heads of k (rotated, quantised), kv_heads of v (quantised).
// A CTA takes 16 of them.  Angles are position * inv_freq in 64 bits, reduced to a turn there (a 32-bit angle of
// position 100 000 is off by 0.004 rad), the 64 sines and cosines of a token worked out once a CTA.
__global__ void __launch_bounds__(kAppendThreads) kv4_append_kernel(const __grid_constant__ AppendArgs a) {
    __shared__ float2 s_turn[kKvDim / 2];
    pdl_wait_prior_grids();
    pdl_release_dependents();
    const Kv4View& c = a.c;
    const int token = blockIdx.x / a.blocks_per_token;
    const int row = (blockIdx.x - token * a.blocks_per_token) * (kAppendThreads / kRowThreads) + (threadIdx.x >> 4);
    const int hl = threadIdx.x & 15;
    const int n_q = a.q != nullptr ? a.q_heads : 0, rows = n_q + 2 * c.kv_heads;
    // what the row is: 0 q, 1 k, 2 v
    const int kind = row < n_q ? 0 : row < n_q + c.kv_heads ? 1 : 2;
    const int head = row - (kind == 0 ? 0 : kind == 1 ? n_q : n_q + c.kv_heads);
    const bool on = row < rows;
    uint4 raw = make_uint4(0, 0, 0, 0), bias = raw;
    if (on) {
        const __half* src = kind == 0 ? a.q + static_cast<size_t>(token) * a.q_stride
                                      : (kind == 1 ? a.k : a.v) + static_cast<size_t>(token) * a.kv_stride;
        raw = __ldcg(reinterpret_cast<const uint4*>(src + head * kKvDim + hl * 8));
        const __half* b = kind == 0 ? a.q_bias : kind == 1 ? a.k_bias : a.v_bias;
        if (b != nullptr) bias = __ldcg(reinterpret_cast<const uint4*>(b + head * kKvDim + hl * 8));
    }
    const int seq = kv4_seq_of_token(c, token);
    if (seq >= c.num_seqs) return;                               // behind the last sequence: left as it is
    const int2 mine = kv4_new_tokens(c, seq);
    const int at = __ldcg(c.lens + seq) - mine.y + (token - mine.x);
    if (token < mine.x || token >= mine.x + mine.y) return;
    if (a.inv_freq != nullptr && threadIdx.x < kKvDim / 2) {
        const int pos = a.positions != nullptr ? __ldcg(a.positions + token) : at;
        const double turns = static_cast<double>(pos) * static_cast<double>(__ldcg(a.inv_freq + threadIdx.x)) * 0.15915494309189533577;
        float sn, cs;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sn, &cs);
        s_turn[threadIdx.x] = make_float2(cs, sn);
    }
    __syncthreads();
    float x[8], b[8];
    half8_to_float(raw, x);
    half8_to_float(bias, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] += b[j];
    if (a.inv_freq != nullptr) {
        // values d and d + 64 are a pair: lanes hl and hl ^ 8
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float other = __shfl_xor_sync(0xFFFFFFFFu, x[j], 8);
            const float2 t = s_turn[(hl & 7) * 8 + j];
            if (kind != 2) x[j] = hl < 8 ? x[j] * t.x - other * t.y : x[j] * t.x + other * t.y;
        }
    }
    const uint4 rounded = float_to_half8(x);
    if (on && kind == 0)
        *reinterpret_cast<uint4*>(a.q_out + static_cast<size_t>(token) * a.q_stride + head * kKvDim + hl * 8) = rounded;
    half8_to_float(rounded, x);
    uint32_t params;
    const uint32_t word = kv4_quantise_lane(x, &params);
    if (!on || kind == 0 || at < 0 || at >= kv4_capacity(c)) return;
    const int page = kv4_page(c, seq, at);
    uint32_t* record = kv4_record_of_page(c, page, head);
    if (record == nullptr) return;
    const int ps = 1 << c.page_shift, slot = at & (ps - 1), part = kind - 1;
    record[(part * ps + slot) * kKvRowWords + hl] = word;
    if (hl == 0) {
        record[(32 + part) * ps + slot] = params;
        if (kind == 1 && c.key_weight != nullptr) c.key_weight[kv4_weight_index(c, page, head, at)] = 0.0f;
    }
}

// The rows that an append of this batch writes, as fp16.  A half-warp a row.
__global__ void __launch_bounds__(kAppendThreads) kv4_read_kernel(const __grid_constant__ Kv4View c, __half* k_out, __half* v_out, int blocks_per_token) {
    pdl_wait_prior_grids();
    pdl_release_dependents();
    const int token = blockIdx.x / blocks_per_token;
    const int row = (blockIdx.x - token * blocks_per_token) * (kAppendThreads / kRowThreads) + (threadIdx.x >> 4);
    const int hl = threadIdx.x & 15;
    const int seq = kv4_seq_of_token(c, token);
    if (seq >= c.num_seqs || row >= 2 * c.kv_heads) return;
    const int2 mine = kv4_new_tokens(c, seq);
    if (token < mine.x || token >= mine.x + mine.y) return;
    const int part = row >= c.kv_heads, head = row - part * c.kv_heads;
    __half* out = part ? v_out : k_out;
    if (out == nullptr) return;
    const int at = __ldcg(c.lens + seq) - mine.y + (token - mine.x);
    uint4 got = make_uint4(0, 0, 0, 0);
    const uint32_t* record = at >= 0 && at < kv4_capacity(c) ? kv4_record_of_page(c, kv4_page(c, seq, at), head) : nullptr;
    if (record != nullptr) {
        const int ps = 1 << c.page_shift, slot = at & (ps - 1);
        const uint32_t word = __ldcg(record + (part * ps + slot) * kKvRowWords + hl);
        const uint32_t params = __ldcg(record + (32 + part) * ps + slot);
        const float s = kv4_scale(params), z = kv4_zero(params);
        constexpr int kShift[8] = {0, 8, 16, 24, 4, 12, 20, 28};
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = fmaf(static_cast<float>(static_cast<int>((word >> kShift[j]) & 15u) - 8), s, z);
            if (fabsf(x[j]) > 65504.0f) x[j] = copysignf(65504.0f, x[j]);    // the rounding of scale and zero may step over fp16's end
        }
        got = float_to_half8(x);
    }
    *reinterpret_cast<uint4*>(out + (static_cast<size_t>(token) * c.kv_heads + head) * kKvDim + hl * 8) = got;
}

// ---- eviction ------------------------------------------------------------------------------------------------

struct EvictArgs {
    Kv4View c;
    const int32_t* dst_table;
    int32_t* new_lens;
    int32_t* kept;                       // [num_seqs][kv_heads][budget]
    int dst_pages, budget, sink, recent;
};

// Order of the weights as unsigned numbers: larger weight, larger key; a NaN is below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (!(w == w)) return 0u;
    w = w + 0.0f;                        // -0 and 0 are equal
    const uint32_t u = __float_as_uint(w);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024;

// Which positions of one sequence and head stay, in order.  The n-th largest key of the middle part by a radix search, a byte
// a round; then one ordered pass that numbers what stays.
__global__ void __launch_bounds__(kSelectThreads) kv4_select_kernel(const __grid_constant__ EvictArgs a) {
    __shared__ uint32_t s_hist[256];
    __shared__ uint32_t s_prefix, s_need;
    __shared__ int s_warp[2][32];
    pdl_wait_prior_grids();
    pdl_release_dependents();
    const Kv4View& c = a.c;
    const int b = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int len = min(max(__ldcg(c.lens + b), 0), kv4_capacity(c));
    const int keep = min(len, a.budget);
    int32_t* kept = a.kept + (static_cast<size_t>(b) * c.kv_heads + head) * a.budget;
    if (head == 0 && tid == 0) a.new_lens[b] = keep;
    for (int i = keep + tid; i < a.budget; i += kSelectThreads) kept[i] = -1;
    if (len <= a.budget) {
        for (int i = tid; i < keep; i += kSelectThreads) kept[i] = i;
        return;
    }
    const int lo = a.sink, hi = len - a.recent;                 // the middle: sink + recent <= budget < len
    const uint32_t want = static_cast<uint32_t>(a.budget - a.sink - a.recent);
    auto key_at = [&](int i) -> uint32_t {
        const int page = kv4_page(c, b, i);
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(c.num_pages)) return 0u;
        return weight_key(__ldcg(c.key_weight + kv4_weight_index(c, page, head, i)));
    };
    if (tid == 0) { s_prefix = 0; s_need = want; }
    uint32_t prefix = 0, need = want;
    for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
        for (int i = tid; i < 256; i += kSelectThreads) s_hist[i] = 0;
        __syncthreads();
        for (int i = lo + tid; i < hi; i += kSelectThreads) {
            const uint32_t k = key_at(i);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_hist[(k >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t above = 0;
            int d = 255;
            while (d > 0 && above + s_hist[d] < need) above += s_hist[d--];
            s_prefix = prefix | (static_cast<uint32_t>(d) << shift);
            s_need = need - above;
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
    }
    // keys above `prefix` stay, and the first `need` of those equal to it
    int base = 0, equal_base = 0;
    for (int i0 = 0; i0 < len; i0 += kSelectThreads) {
        const int i = i0 + tid;
        bool stay = i < len && (i < lo || i >= hi), equal = false;
        if (i >= lo && i < hi && want > 0) {
            const uint32_t k = key_at(i);
            stay = k > prefix;
            equal = k == prefix;
        }
        const uint32_t eq = __ballot_sync(0xFFFFFFFFu, equal);
        if (lane == 0) s_warp[0][warp] = __popc(eq);
        __syncthreads();
        int before = equal_base, total_eq = 0;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) before += s_warp[0][w];
            total_eq += s_warp[0][w];
        }
        before += __popc(eq & ((1u << lane) - 1u));
        if (equal && before < static_cast<int>(need)) stay = true;
        equal_base += total_eq;
        const uint32_t st = __ballot_sync(0xFFFFFFFFu, stay);
        if (lane == 0) s_warp[1][warp] = __popc(st);
        __syncthreads();
        int at = base, total = 0;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) at += s_warp[1][w];
            total += s_warp[1][w];
        }
        at += __popc(st & ((1u << lane) - 1u));
        if (stay && at < a.budget) kept[at] = i;
        base += total;
    }
}

// The kept rows to their fresh pages: a half-warp moves a position, two 64-byte rows, their parameters and the weight.
__global__ void __launch_bounds__(256) kv4_move_kernel(const __grid_constant__ EvictArgs a) {
    pdl_wait_prior_grids();
    pdl_release_dependents();
    const Kv4View& c = a.c;
    const int b = blockIdx.z, head = blockIdx.y, hl = threadIdx.x & 15;
    const int j = blockIdx.x * 16 + (threadIdx.x >> 4);
    if (j >= a.budget) return;
    const int i = __ldcg(a.kept + (static_cast<size_t>(b) * c.kv_heads + head) * a.budget + j);
    if (i < 0) return;
    const int old_page = kv4_page(c, b, i), ps = 1 << c.page_shift;
    const int new_page = __ldcg(a.dst_table + static_cast<size_t>(b) * a.dst_pages + (j >> c.page_shift));
    const uint32_t* from = kv4_record_of_page(c, old_page, head);
    uint32_t* to = kv4_record_of_page(c, new_page, head);
    if (from == nullptr || to == nullptr) return;
    const int s0 = i & (ps - 1), s1 = j & (ps - 1);
    to[s1 * kKvRowWords + hl] = __ldcg(from + s0 * kKvRowWords + hl);
    to[(ps + s1) * kKvRowWords + hl] = __ldcg(from + (ps + s0) * kKvRowWords + hl);
    if (hl < 2) to[(32 + hl) * ps + s1] = __ldcg(from + (32 + hl) * ps + s0);
    if (hl == 2) c.key_weight[kv4_weight_index(c, new_page, head, j)] = __ldcg(c.key_weight + kv4_weight_index(c, old_page, head, i));
}

}  // namespace

int kv4_append(const Kv4View& c, const Kv4AppendArgs& x, cudaStream_t stream) {
    AppendArgs a{c, x.q, x.k, x.v, x.q_bias, x.k_bias, x.v_bias, x.q_out, x.positions, x.inv_freq, x.q_heads, x.q_stride, x.kv_stride, 0};
    const int rows = (x.q != nullptr ? x.q_heads : 0) + 2 * c.kv_heads;
    a.blocks_per_token = (rows + 15) / 16;
    const long long blocks = static_cast<long long>(a.blocks_per_token) * c.num_tokens;
    if (blocks > 0x7FFFFFFFll) return W4A16_ERR_TOO_LARGE;
    return static_cast<int>(launch_kernel(kv4_append_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kAppendThreads), 0, stream, pdl_enabled(), a));
}

int kv4_read(const Kv4View& c, __half* k_out, __half* v_out, cudaStream_t stream) {
    const int per = (2 * c.kv_heads + 15) / 16;
    const long long blocks = static_cast<long long>(per) * c.num_tokens;
    if (blocks > 0x7FFFFFFFll) return W4A16_ERR_TOO_LARGE;
    return static_cast<int>(launch_kernel(kv4_read_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kAppendThreads), 0, stream, pdl_enabled(), c, k_out, v_out, per));
}

int kv4_evict(const Kv4View& c, const Kv4EvictArgs& x, cudaStream_t stream) {
    EvictArgs a{c, x.dst_table, x.new_lens, x.kept, x.dst_pages, x.budget, x.sink, x.recent};
    cudaError_t e = launch_kernel(kv4_select_kernel, dim3(c.num_seqs, c.kv_heads), dim3(kSelectThreads), 0, stream, pdl_enabled(), a);
    if (e != cudaSuccess) return static_cast<int>(e);
    const dim3 grid((x.budget + 15) / 16, c.kv_heads, c.num_seqs);
    return static_cast<int>(launch_kernel(kv4_move_kernel, grid, dim3(256), 0, stream, pdl_enabled(), a));
}

}  // namespace w4
