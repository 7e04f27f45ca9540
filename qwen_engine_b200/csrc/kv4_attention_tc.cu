// Attention of many query rows over the 4-bit key/value cache (chunks of a prompt), fp16 out, on tcgen05.
//
// A CTA has 256 query rows of one key/value head (token major, so the heads that share it lie side by side) as two tiles of 128,
// and walks over the positions 128 at a time:
//   S_i [128 rows x 128 positions] = Q_i . K^T      both from shared memory
//   P_i = 2^(S_i c - m), fp16, over S_i in tensor memory; m follows the running maximum, for the next step where it falls 8 behind, at
//       once (the step's weights are worked out again) where 15, as fp16 ends at 2^16.  Weights below 2^-24 of the largest are lost
//   O_i [128 rows x 128 dims] += P_i . V            P from tensor memory, V (transposed: positions contiguous) from shared memory
// While the softmax warps of one tile work the tensor core has the other one.  Keys and values become fp16 once for both tiles.  A
// value is (code - 8) * scale + zero by one fma behind an exact conversion, so has one rounding (in two parts: 2.6e-4 instead of 3.3e-4 of a
// result, but 970 us instead of 750 for a chunk of 1000 tokens at 32 100 positions and 32 heads on 8).  A key has none: (code - 8) * scale
// has 15 bits at most and is the sum of two fp16 numbers, the product and what its rounding left (one fma), which are two operands;
// its zero comes in as 16 more columns that all hold it, against the sum of q in two parts, an eighth in each of eight columns.
// (Keys rounded to fp16 left 4e-4 in the lse of short sequences.  Exact codes as the operand and scale and zero in the softmax need two
// numbers a position in every thread: from shared memory they took 200 of 910 us, through the same queue as the exponentials.)
//
// What bounds it: the exponentials (16 a cycle and SM: 2048 cycles for 256 x 128) and the tensor core (2048 cycles) alike, and
// behind them the issue slots of the softmax.
//
//   warps 0..3, 4..7 : softmax of tile 0 and 1, a thread a row; at the end they store O
//   warps 8..15      : operands.  Keys, half a row a thread, from global memory by way of registers, a step ahead; values' codes through a
//                      staging buffer, then a thread takes 8 dims x 8 positions and stores them as rows of 8 positions.  Every access
//                      of both is free of bank conflicts (chunks of 16 bytes are xor-ed).  Keys have one slot, so the next step's wait
//                      for the scores of this one and come first (four warps for keys and four for values: 880 us)
//   warp 16          : tensor memory; one thread issues the MMAs
// Within a word the elements come out as 0 2 4 6 1 3 5 7; the queries are put into the same order once.
//
// Rows that some query must not see: a position outside the split, the sequence or the pool is zeros in shared memory and a cleared
// bit in the mask of its step; one whose value scale is NaN is zeros too, and a bit in a second mask that makes the weight of a
// row that does see it NaN (0 * NaN would reach the others).
#include "kv4_attention.hpp"
#include "kv4_work.cuh"
#include "tc_ptx.cuh"
#include "w4a16_internal.hpp"

namespace w4 {
namespace {

constexpr int kTile = 128, kChunkRows = 2 * kTile, kChunkKeys = 128;
constexpr int kSoftWarps = 8, kOperandWarp = 8, kMmaWarp = 16, kChunkThreads = 20 * 32;
// Registers: a launch of 20 warps has 96 a thread (61 440); the warpgroups share them as 128 (softmax, two), 80 (keys, values) and 64
// (the issuing warp's): 256 * 128 + 256 * 80 + 128 * 64 = 61 440.
constexpr int kSoftRegs = 128, kOperandRegs = 80, kIssueRegs = 64;
static_assert(256 * kSoftRegs + 256 * kOperandRegs + 128 * kIssueRegs <= kChunkThreads * 96);
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
constexpr int kOperand = kTile * kKvDim * 2;              // bytes of a 128 x 128 operand: two panels of 64 columns, 128-byte swizzle
constexpr int kPanel = kOperand / 2;
constexpr int kValueStage = kChunkKeys * 64;
constexpr int kExtra = kTile * 32;                        // 16 more columns, 32-byte swizzle
// queries of both tiles; keys, first and second part; values, two slots; the extra columns of queries and keys; values' codes and parameters
constexpr int kSmemK = 2 * kOperand, kSmemV = 4 * kOperand, kSmemQx = 6 * kOperand, kSmemKx = kSmemQx + 2 * kExtra, kSmemStage = kSmemKx + kExtra,
              kSmemParam = kSmemStage + 2 * kValueStage, kChunkSmem = kSmemParam + 2 * kChunkKeys * 4;
static_assert(kChunkSmem + 1024 + 2048 <= 227 * 1024);
constexpr int kTmemO = 256;                               // S_0, S_1, O_0, O_1: 128 columns each

// The two products, with descriptors given by their low words (address): the high word is the same for every operand here, and as
// 64-bit values the 64 of them that the unrolled loop uses were kept in registers, and spilled.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);      // rows of 128 bytes in groups of 8, 128-byte swizzle
constexpr uint32_t kDescHighExtra = (256u >> 4) | (1u << 14) | (6u << 29);  // rows of 32 bytes in groups of 8, 32-byte swizzle
__device__ __forceinline__ uint32_t desc_low(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | (1u << 16); }
template <uint32_t HIGH = kDescHigh>
__device__ __forceinline__ void mma_ss(uint32_t tmem_d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(HIGH)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
                 : "r"(taddr)
                 : "memory");
}
// Bounded waits that leave the issue slots to others: a try that parks the thread for up to 20 us, and the abort flag looked at
// between tries only.  (With the short tries of mbar_wait, and its flag at each, waiting warps issued 6000 of a step's 14 000
// instructions.)
__device__ __forceinline__ bool park_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    if (mbar_test_wait(bar, parity)) return true;      // a try costs more even where the phase is complete (663 us without this, 615 with)
    for (unsigned it = 0; it < (1u << 16); ++it) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity), "r"(20000u)
            : "memory");
        if (ok) return true;
        if (*abort_flag) return false;
    }
    *abort_flag = 1;
    atomicAdd(&g_tc_wait_timeouts, 1u);
    return false;
}
// The whole warp waits, every lane by itself: all see what the barrier's arrivals announce.  (One lane's wait behind a branch made the
// whole kernel a third slower, 817 us for 615: what follows it is no longer known to be converged.)
__device__ __forceinline__ bool park_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    return __all_sync(0xFFFFFFFFu, park_wait(bar, parity, abort_flag));
}
// Barrier of the operand warps: whether all of them are well.  A warp whose wait ran out comes here too, so none is left waiting.
__device__ __forceinline__ bool all_of_256(bool ok) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"(static_cast<uint32_t>(ok)) : "memory");
    return r != 0;
}
// Two 32-bit operations in one instruction, the exponential and the conversion, all volatile: their order is the software pipeline
// of softmax_pass.
__device__ __forceinline__ void fma2(float& x, float& y, float2 b, float2 c) {
    asm volatile("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tmov.b64 c, {%4, %5};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
                 : "+f"(x), "+f"(y) : "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
}
__device__ __forceinline__ void add_to2(float& x, float& y, float2 b) {
    asm volatile("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
                 : "+f"(x), "+f"(y) : "f"(b.x), "f"(b.y));
}
__device__ __forceinline__ void add2(float2& s, float x, float y) {
    asm volatile("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
                 : "+f"(s.x), "+f"(s.y) : "f"(x), "f"(y));
}
__device__ __forceinline__ void ex2_here(float& x) { asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(x)); }
__device__ __forceinline__ uint32_t pack_here(float lo, float hi) {
    uint32_t d;
    asm volatile("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// Waits for the tensor-memory loads in flight and hands the values on: whatever uses them depends on the wait.
__device__ __forceinline__ void tmem_take32(float (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])
                 :: "memory");
    asm volatile("" : "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31]) :: "memory");
}

// A row of 128 scores to weights p = 2^(score * scale2 - mu), as fp16 pairs, their sum, and the largest exponent.  What bounds it is
// the exponential, 8 cycles a warp; so it is one stream of them, with a pair's scaling eight pairs ahead of its exponential and its sum
// and conversion three behind.  (As loops that the compiler orders a row took 2200 cycles alone on its scheduler.)  The wait for
// tensor-memory loads is one for all that are in flight, so 32 columns are asked for behind the wait for the 32 before them and
// have all of their exponentials' time; asked for in eighths, later, each wait stalled (2200 cycles again, 1300 without loads).
// SIMPLE: the row sees every position, and rest2 is not used; else those of `sees`, and rest2 is added.
template <bool SIMPLE>
__device__ __forceinline__ float softmax_pass(uint32_t t_s, float2 scale2, float2 mu2, float2 rest2, const uint32_t (&sees)[4], uint32_t (&p)[64], float* total) {
    float s[2][32];
    float2 sum[2] = {};
    float top[2] = {-INFINITY, -INFINITY};
    auto scale = [&](int c, int k) {
        float &x = s[c & 1][2 * k], &y = s[c & 1][2 * k + 1];
        fma2(x, y, scale2, mu2);
        if (!SIMPLE) {
            add_to2(x, y, rest2);
            if (!(sees[c] >> (2 * k) & 1u)) x = -INFINITY;
            if (!(sees[c] >> (2 * k) & 2u)) y = -INFINITY;
        }
        top[k & 1] = fmaxf(top[k & 1], fmaxf(x, y));
    };
    auto finish = [&](int c, int k) {
        float &x = s[c & 1][2 * k], &y = s[c & 1][2 * k + 1];
        add2(sum[k & 1], x, y);
        p[16 * c + k] = pack_here(x, y);
    };
    constexpr int kAhead = 8, kBehind = 3;
    tmem_ld32(t_s, s[0]);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        tmem_take32(s[c & 1]);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) scale(c, k);
        if (c > 0) {
#pragma unroll
            for (int k = 16 - kBehind; k < 16; ++k) finish(c - 1, k);
        }
        if (c < 3) tmem_ld32(t_s + 32u * (c + 1), s[(c + 1) & 1]);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            ex2_here(s[c & 1][2 * k]);
            ex2_here(s[c & 1][2 * k + 1]);
            if (k + kAhead < 16) scale(c, k + kAhead);
            if (k >= kBehind) finish(c, k - kBehind);
        }
    }
#pragma unroll
    for (int k = 16 - kBehind; k < 16; ++k) finish(3, k);
    *total = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    return fmaxf(top[0], top[1]);
}

// (scale, zero) of a row that becomes fp16 values: where rounding took its ends past 65504 both shrink a little, so that none is
// infinite.  A NaN stays.
__device__ __forceinline__ uint32_t finite_params(uint32_t p) {
    const float s = kv4_scale(p), z = kv4_zero(p);
    const float end = fmaxf(fabsf(fmaf(-8.0f, s, z)), fabsf(fmaf(7.0f, s, z)));
    if (!(end > 65504.0f)) return p;
    const float f = 65504.0f / end;
    return static_cast<uint32_t>(__half_as_ushort(__float2half_rz(s * f))) | (static_cast<uint32_t>(__half_as_ushort(__float2half_rz(z * f))) << 16);
}
__device__ __forceinline__ bool nan_params(uint32_t p) { return kv4_scale(p) != kv4_scale(p) || kv4_zero(p) != kv4_zero(p); }

// Four pairs of values of a word's nibbles (bits 4 n and 16 + 4 n) with their scales and zeros.
__device__ __forceinline__ void dequantise(uint32_t w, __half2 s, __half2 z, uint32_t (&out)[4]) {
    kv4_centred_codes(w, out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&out[i]), s, z);
        out[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
}
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ uint32_t sixteenth(uint32_t x) {
    const __half2 y = __hmul2(as_half2(x), __float2half2_rn(0.0625f));
    return *reinterpret_cast<const uint32_t*>(&y);
}

// Row and 16-byte chunk (8 columns) of an operand in shared memory.
__device__ __forceinline__ uint32_t operand_at(int row, int chunk) {
    return static_cast<uint32_t>((chunk >> 3) * kPanel + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

__device__ __forceinline__ uint32_t extra_at(int row, int chunk) { return static_cast<uint32_t>(row * 32 + ((chunk ^ ((row >> 2) & 1)) << 4)); }

// The (tile, head) of a CTA.  (All steps of the batch shared evenly by 148 persistent CTAs took 780 us where this takes 765 and 102 where it
// takes 57, for all that 20 and 50 of the SMs have nothing to do here: a piece costs 14 us beside its steps, for queries, first scores,
// the second pass over the first step and its parts.)  Long ones first, which are the last ones of a sequence.
struct ChunkPlace {
    SeqWork w;
    int seq, head, row0, rows;
};
template <int THREADS>
__device__ __forceinline__ bool find_chunk(const Kv4View& c, int group, int index, FindScratch<THREADS>& s, ChunkPlace* out) {
    long long per, all;
    Place pl;
    if (!find_unit<THREADS, true>(c, group, kChunkRows, index, 1, s, &per, &all, &pl)) return false;
    const int th = static_cast<int>(pl.in_seq), tile = pl.w.tiles - 1 - th / c.kv_heads;
    out->w = pl.w;
    out->seq = pl.seq;
    out->head = th % c.kv_heads;
    out->row0 = tile * kChunkRows;
    out->rows = min(kChunkRows, pl.w.n * group - out->row0);
    return true;
}
// Positions of a (tile, head): what its last row sees, and the steps of one split.
__device__ __forceinline__ int chunk_seen(const Kv4View& c, const ChunkPlace& p, int group) {
    return min(max(p.w.past + (p.row0 + p.rows - 1) / group + 1, 0), kv4_capacity(c));
}
__device__ __forceinline__ int chunk_steps(int seen, int splits) { return ((seen + kChunkKeys - 1) / kChunkKeys + splits - 1) / splits; }

__global__ void __launch_bounds__(kChunkThreads, 1) kv4_chunk_kernel(const __grid_constant__ Kv4ChunkArgs a) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ uint64_t s_bar[14];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort_word;
    __shared__ __align__(16) uint32_t s_mask[4][2][4];     // [step % 4][there, poisoned][32 positions]
    __shared__ FindScratch<kChunkThreads> s_find;
    volatile int* s_abort = &s_abort_word;
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t smem0 = smem_u32(smem), bar0 = smem_u32(s_bar);
    const uint32_t k_full = bar0, k_empty = bar0 + 8u * 2;
    auto v_full = [&](int i) { return bar0 + 8u * (4 + i); };
    auto v_empty = [&](int i) { return bar0 + 8u * (6 + i); };
    auto s_full = [&](int i) { return bar0 + 8u * (8 + i); };
    auto p_full = [&](int i) { return bar0 + 8u * (10 + i); };
    const uint32_t q_full = bar0 + 8u * 12, finished = bar0 + 8u * 13;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (warp == kMmaWarp) {
        if (lane < 2) {
            mbar_init(v_full(lane), 8);
            mbar_init(v_empty(lane), 1);
            mbar_init(s_full(lane), 1);
            mbar_init(p_full(lane), 4);
        }
        if (lane == 0) {
            mbar_init(k_full, 8);
            mbar_init(k_empty, 1);
            mbar_init(q_full, kSoftWarps);
            mbar_init(finished, 1);
            *s_abort = 0;
        }
        fence_barrier_init();
        __syncwarp();
        tmem_alloc(smem_u32(&s_tmem), 512);
        tmem_relinquish();
    }
    pdl_wait_prior_grids();
    const Kv4View& c = a.c;
    const int index = blockIdx.x / a.splits, split = blockIdx.x - index * a.splits;
    ChunkPlace pl;
    const bool work = find_chunk<kChunkThreads>(c, a.group, index, s_find, &pl);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0;        // all 512 columns are this CTA's, so they begin at 0; a constant keeps the issuing thread's operands uniform
    pdl_release_dependents();           // not before: a CTA of the next launch must not take this one's tensor memory
    const int seen = work ? chunk_seen(c, pl, a.group) : 0, steps_each = chunk_steps(seen, a.splits);
    const int k0 = split * steps_each * kChunkKeys, k1 = min(seen, k0 + steps_each * kChunkKeys);
    const int steps = work && k1 > k0 ? (k1 - k0 + kChunkKeys - 1) / kChunkKeys : 0;
    const int tiles = work && pl.rows > kTile ? 2 : 1;
    const int32_t* table = c.table + static_cast<size_t>(work ? pl.seq : 0) * c.max_pages;
    const int ps = 1 << c.page_shift;

    if (warp < kSoftWarps) {
        // ================= softmax: thread = row = tensor-memory lane =================
        more_registers<kSoftRegs>();
        const int i = warp >> 2, r = tid & 127, row = i * kTile + r;
        const bool mine = work && row < pl.rows;
        const size_t at_row = mine ? out_row(pl.w, c.kv_heads, a.group, pl.head, pl.row0 + row) : 0;
        const int limit = mine ? pl.w.past + (pl.row0 + row) / a.group + 1 : 0x7FFFFFFF;
        float to_log2 = a.scale * kLog2e;
        if (steps > 0 && i < tiles) {
            uint4 w[16];
            float qsum = 0.0f;
            const __half* src = a.q;
            if (mine) src += static_cast<size_t>(pl.w.first + (pl.row0 + row) / a.group) * a.q_stride + (pl.head * a.group + (pl.row0 + row) % a.group) * kKvDim;
#pragma unroll
            for (int k = 0; k < 16; ++k) w[k] = mine ? __ldcg(reinterpret_cast<const uint4*>(src) + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < 16; ++k)
                *reinterpret_cast<uint4*>(smem + i * kOperand + operand_at(r, k)) =
                    make_uint4(__byte_perm(w[k].x, w[k].y, 0x5410), __byte_perm(w[k].z, w[k].w, 0x5410), __byte_perm(w[k].x, w[k].y, 0x7632),
                               __byte_perm(w[k].z, w[k].w, 0x7632));
#pragma unroll
            for (int k = 0; k < 16; ++k) qsum += sum_half8(w[k]);
            if (fabsf(qsum) > 8.0f * 65504.0f) {
                // an eighth of the sum is no fp16 number any more: the row a sixteenth of its size (128 * 65504 / 16 is in range again), its scores
                // the other way.  Exact but for elements below 2^-10, where it is off by 2^-21, in a row whose mean is above 4094.
#pragma unroll 1
                for (int k = 0; k < 16; ++k) {
                    uint4* at = reinterpret_cast<uint4*>(smem + i * kOperand + operand_at(r, k));
                    *at = make_uint4(sixteenth(at->x), sixteenth(at->y), sixteenth(at->z), sixteenth(at->w));
                }
                qsum *= 0.0625f;
                to_log2 *= 16.0f;
            }
            const __half part = __float2half_rn(qsum * 0.125f), rest = __float2half_rn(fmaf(qsum, 0.125f, -__half2float(part)));
            const uint32_t pp = pack_half2(__half2float(part), __half2float(part)), rr = pack_half2(__half2float(rest), __half2float(rest));
            *reinterpret_cast<uint4*>(smem + kSmemQx + i * kExtra + extra_at(r, 0)) = make_uint4(pp, pp, pp, pp);
            *reinterpret_cast<uint4*>(smem + kSmemQx + i * kExtra + extra_at(r, 1)) = make_uint4(rr, rr, rr, rr);
            fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t t_s = lanes + static_cast<uint32_t>(i * 128), t_o = lanes + static_cast<uint32_t>(kTmemO + i * 128);
        // m: reference of the exponents, at most 15 below the row's largest so far and renewed where it is 8 below; grow: by how much, at
        // the next step.  Rows that have seen nothing have -infinity.
        // From 2^23 on a 32-bit number's neighbours are 1 and more away.  The exponents are rounded once, behind the subtraction, so there the
        // reference is m + rest, and m is taken from below, so that what is left to grow is above zero.
        constexpr float kFar = 8388608.0f;
        auto from_below = [&](float x) { return fabsf(x) < kFar ? x : __int_as_float(__float_as_int(x) + (x > 0.0f ? -1 : 1)); };
        float m = -INFINITY, l = 0.0f, grow = 0.0f, rest = 0.0f;
        bool ok = true;
        for (int j = 0; j < (i < tiles ? steps : 0); ++j) {
            ok = park_warp(s_full(i), j & 1, s_abort);
            if (!ok) break;
            tc_fence_after();
            const int base = k0 + j * kChunkKeys;
            uint32_t sees[4];
            bool simple, poisoned;
            {
                const uint4 there = *reinterpret_cast<const uint4*>(s_mask[j & 3][0]), poison = *reinterpret_cast<const uint4*>(s_mask[j & 3][1]);
                const uint32_t all = there.x & there.y & there.z & there.w, any = poison.x | poison.y | poison.z | poison.w;
                simple = __all_sync(0xFFFFFFFFu, base + kChunkKeys <= limit && all == ~0u);
                poisoned = any != 0;
                const uint32_t th[4] = {there.x, there.y, there.z, there.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int n = limit - base - 32 * q;
                    sees[q] = th[q] & (n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u);
                }
            }
            uint32_t p[64];
            float sum;
            for (int turns = 0; turns < 3; ++turns) {       // the third one from 2^23 on
                if (__any_sync(0xFFFFFFFFu, grow > 0.0f)) {
                    const float t = rest + grow, fresh = m + t, step = fresh - m;
                    const float left = fabsf(fresh) < kFar ? 0.0f : (m - (fresh - step)) + (t - step);
                    const float f = grow > 0.0f ? ex2(rest - left - step) : 1.0f;
                    if (grow > 0.0f) {
                        m = fresh;
                        rest = left;
                    }
                    l *= f;
                    grow = 0.0f;
                    if (j > 0) {
                        // the product of the step before is complete: s_full of this step was committed behind it
#pragma unroll 1
                        for (int q = 0; q < 4; ++q) {
                            float x[32];
                            tmem_ld32(t_o + 32u * q, x);
                            tmem_take32(x);
                            uint32_t y[2][16];
#pragma unroll
                            for (int k = 0; k < 32; ++k) y[k >> 4][k & 15] = __float_as_uint(x[k] * f);
                            tmem_st16(t_o + 32u * q, y[0]);
                            tmem_st16(t_o + 32u * q + 16u, y[1]);
                        }
                    }
                }
                const float mu = m == -INFINITY ? 0.0f : m;
                const float2 scale2 = make_float2(to_log2, to_log2), mu2 = make_float2(-mu, -mu);
                const float top = simple && __all_sync(0xFFFFFFFFu, fabsf(mu) < kFar) ? softmax_pass<true>(t_s, scale2, mu2, mu2, sees, p, &sum)
                                                                                      : softmax_pass<false>(t_s, scale2, mu2, make_float2(-rest, -rest), sees, p, &sum);
                // too large for fp16, or the row's first positions: again with the maximum known
                const bool fresh = m == -INFINITY && top > -INFINITY, again = fresh || top > 15.0f;
                if (fresh) m = from_below(top);
                else if (top > 8.0f) grow = from_below(top);
                if (!__any_sync(0xFFFFFFFFu, again)) break;
            }
            if (poisoned) {                 // behind the sum, which the values have no part in
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t bad = sees[q] & s_mask[j & 3][1][q];
#pragma unroll
                    for (int k = 0; k < 16; ++k) p[16 * q + k] |= (bad >> (2 * k) & 1u ? 0x00007E00u : 0u) | (bad >> (2 * k) & 2u ? 0x7E000000u : 0u);
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t y[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) y[k] = p[16 * q + k];
                tmem_st16(t_s + 16u * q, y);
            }
            l += sum;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(i));
        }
        if (ok && steps > 0 && i < tiles) ok = park_warp(finished, 0, s_abort);
        if (work && ok && i < tiles) {
            tc_fence_after();
            const bool whole = a.splits == 1;
            const float f = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
            const size_t part = (static_cast<size_t>(blockIdx.x) * kChunkRows + row);
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
                float x[32] = {};
                if (steps > 0) {
                    tmem_ld32(t_o + 32u * q, x);
                    tmem_take32(x);
                }
                if (!mine) continue;
                if (whole) {
                    __half* out = a.out + at_row * kKvDim + 32 * q;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = l == 0.0f ? 0u : pack_result(x[8 * k + 2 * e] * f, x[8 * k + 2 * e + 1] * f);
                        reinterpret_cast<uint4*>(out)[k] = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                } else {
                    float4* out = reinterpret_cast<float4*>(a.part_o + part * kKvDim + 32 * q);
#pragma unroll
                    for (int k = 0; k < 8; ++k) __stcg(out + k, make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]));
                }
            }
            if (mine && whole && a.lse != nullptr) a.lse[at_row] = l == 0.0f ? -INFINITY : (m + (rest + log2f(l))) * kLn2;
            if (mine && !whole) __stcg(a.part_ml + part, make_float2(m + rest, l));
        }
    } else if (warp < kMmaWarp) {
        // ================= operands: two threads a position =================
        fewer_registers<kOperandRegs>();
        const int t = tid & 127, part = (warp - kOperandWarp) >> 2;      // keys: words 8 part ..; values: positions 64 part ..
        const int word = (lane >> 3) + 4 * (warp & 3), oct = t >> 3;
        uint4 w[2];
        uint32_t kp = 0, vp = 0;
        bool there = false;
        int page = -1;
        auto page_of = [&](int j) { const int at = k0 + j * kChunkKeys + t; return j < steps && at < k1 ? __ldcg(table + (at >> c.page_shift)) : -1; };
        // position t's key codes and parameters into registers, its value codes into the staging buffer
        const uint32_t stage_to = smem0 + static_cast<uint32_t>(kSmemStage + (t ^ ((oct >> 2) & 1)) * 64);
        auto fetch = [&](int j) {
            const uint32_t* record = kv4_record_of_page(c, page, pl.head);
            there = record != nullptr;
            kp = vp = 0;
            w[0] = w[1] = make_uint4(0, 0, 0, 0);
            if (there) {
                const int slot = (k0 + j * kChunkKeys + t) & (ps - 1);
                const uint32_t* keys = record + slot * kKvRowWords + 8 * part;
                w[0] = __ldcg(reinterpret_cast<const uint4*>(keys));
                w[1] = __ldcg(reinterpret_cast<const uint4*>(keys) + 1);
                kp = __ldcg(record + 32 * ps + slot);
                vp = __ldcg(record + 33 * ps + slot);
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                 ::"r"(stage_to + static_cast<uint32_t>((j & 1) * kValueStage + (((2 * part + k) ^ (oct & 3)) << 4))),
                                 "l"(keys + ps * kKvRowWords + 4 * k) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            page = page_of(j + 1);
        };
        if (steps > 0) {
            page = page_of(0);
            fetch(0);
        }
        bool ok = true;
        for (int j = 0; j < steps; ++j) {
            const int slot = j & 1;
            // ---- keys, first: the scores of the next step wait for them ----
            ok = ok && park_warp(k_empty, (j & 1) ^ 1, s_abort);
            const uint32_t here = __ballot_sync(0xFFFFFFFFu, there), bad = __ballot_sync(0xFFFFFFFFu, nan_params(vp));
            if (part == 0 && lane == 0) {
                s_mask[j & 3][0][warp & 3] = here;
                s_mask[j & 3][1][warp & 3] = bad;
            }
            {
                const __half2 s = __half2half2(__ushort_as_half(static_cast<unsigned short>(kp)));
                const uint32_t zero = __byte_perm(kp, kp, 0x3232);
                *reinterpret_cast<uint4*>(smem + kSmemKx + t * 32 + 16 * part) = make_uint4(zero, zero, zero, zero);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t words[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t o[4], hi[4], lo[4];
                        kv4_centred_codes(words[e], o);         // pairs (0, 2), (4, 6), (1, 3), (5, 7)
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            // in a row that spans more than 15 * 8188 the product of the lowest code is below fp16's end: it is cut there, and
                            // what is left, a multiple of 32 below 4400, is a second part like any other
                            const __half2 h = __hmax2_nan(__hmul2(as_half2(o[n]), s), __float2half2_rn(-65504.0f)), l = __hfma2(as_half2(o[n]), s, __hneg2(h));
                            hi[n] = *reinterpret_cast<const uint32_t*>(&h);
                            lo[n] = *reinterpret_cast<const uint32_t*>(&l);
                        }
                        uint8_t* to = smem + kSmemK + operand_at(t, 8 * part + 4 * k + e);
                        *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4*>(to + kOperand) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(k_full);
            // ---- values ----
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            uint32_t* params = reinterpret_cast<uint32_t*>(smem + kSmemParam) + slot * kChunkKeys;
            if (part == 0) params[t] = nan_params(vp) ? 0u : finite_params(vp);
            if (!all_of_256(ok)) break;         // every position's codes and parameters are there, and the step before has been read
            if (j + 1 < steps) fetch(j + 1);
            ok = park_warp(v_empty(slot), ((j >> 1) & 1) ^ 1, s_abort);
            if (!ok) continue;
            uint8_t* to = smem + kSmemV + slot * kOperand;
            const uint8_t* stage = smem + kSmemStage + slot * kValueStage;
            const int o8 = (lane & 7) + 8 * part;               // eight positions
            const uint4 p0 = reinterpret_cast<const uint4*>(params)[2 * o8], p1 = reinterpret_cast<const uint4*>(params)[2 * o8 + 1];
            const uint32_t pr[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
            uint32_t vw[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                vw[e] = *reinterpret_cast<const uint32_t*>(stage + ((8 * o8 + e) ^ ((o8 >> 2) & 1)) * 64 + (((word >> 2) ^ (o8 & 3)) << 4) + (word & 3) * 4);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t v[4][4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    dequantise(__byte_perm(vw[2 * e], vw[2 * e + 1], half ? 0x7632 : 0x5410), as_half2(__byte_perm(pr[2 * e], pr[2 * e + 1], 0x5410)),
                               as_half2(__byte_perm(pr[2 * e], pr[2 * e + 1], 0x7632)), v[e]);
                constexpr int kElement[2][4] = {{0, 4, 1, 5}, {2, 6, 3, 7}};
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    *reinterpret_cast<uint4*>(to + operand_at(8 * word + kElement[half][n], o8)) = make_uint4(v[0][n], v[1][n], v[2][n], v[3][n]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(v_full(slot));
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
        // ================= MMA issue: one thread =================
        fewer_registers<kIssueRegs>();
        if (warp == kMmaWarp && steps > 0 && elect_one()) {
            constexpr uint32_t idesc = (1u << 4) | ((kTile >> 3) << 17) | ((kTile >> 4) << 24);      // D fp32, A and B fp16, both K-major
            const uint32_t qd = desc_low(smem0), kd = desc_low(smem0 + kSmemK), vd = desc_low(smem0 + kSmemV), qx = desc_low(smem0 + kSmemQx), kx = desc_low(smem0 + kSmemKx);
            constexpr uint32_t kNext = kOperand >> 4, kPanelNext = kPanel >> 4, kExtraNext = kExtra >> 4;
            // tile and slot are constants, so that nothing but the loop's own counters is computed here
            auto scores = [&]<int I>() {
                mma_ss<kDescHighExtra>(tmem + static_cast<uint32_t>(I * 128), qx + I * kExtraNext, kx, idesc, 0);
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const uint32_t off = (ks >= 4 ? kPanelNext : 0) + 2u * (ks & 3);
                        mma_ss(tmem + static_cast<uint32_t>(I * 128), qd + (I * kNext + off), kd + (part * kNext + off), idesc, 1);
                    }
                tc_commit(s_full(I));
            };
            bool ok = park_wait(q_full, 0, s_abort) && park_wait(k_full, 0, s_abort);
            if (ok) {
                tc_fence_after();
                scores.template operator()<0>();
                if (tiles == 2) scores.template operator()<1>();
                tc_commit(k_empty);
            }
            auto outputs = [&]<int I, int SLOT>(int j) {
                if (!park_wait(p_full(I), j & 1, s_abort)) return false;
                tc_fence_after();
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
                    mma_ts(tmem + static_cast<uint32_t>(kTmemO + I * 128), tmem + static_cast<uint32_t>(I * 128 + 8 * ks),
                           vd + (SLOT * kNext + (ks >= 4 ? kPanelNext : 0) + 2u * (ks & 3)), idesc, j != 0 || ks != 0);
                if (j + 1 < steps) {
                    if (I == 0) {
                        if (!park_wait(k_full, (j + 1) & 1, s_abort)) return false;
                        tc_fence_after();
                    }
                    scores.template operator()<I>();
                }
                return true;
            };
            auto step = [&]<int SLOT>(int j) {
                ok = park_wait(v_full(SLOT), (j >> 1) & 1, s_abort) && outputs.template operator()<0, SLOT>(j) &&
                     (tiles == 1 || outputs.template operator()<1, SLOT>(j));
                if (j + 1 < steps) tc_commit(k_empty);
                tc_commit(v_empty(SLOT));
            };
            for (int j = 0; ok && j < steps; j += 2) {
                step.template operator()<0>(j);
                if (ok && j + 1 < steps) step.template operator()<1>(j + 1);
            }
            tc_commit(finished);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (*s_abort) __nanosleep(500000);      // a bounded wait ran out: what is in flight lands before the memory goes
    if (warp == kMmaWarp) tmem_dealloc(s_tmem, 512);
}

// The splits of a (tile, head) joined, a warp a row.
constexpr int kChunkJoinWarps = 8;
__global__ void __launch_bounds__(32 * kChunkJoinWarps) kv4_chunk_join_kernel(const __grid_constant__ Kv4ChunkArgs a) {
    __shared__ FindScratch<32 * kChunkJoinWarps> s_find;
    const int lane = threadIdx.x & 31, row = blockIdx.y * kChunkJoinWarps + (threadIdx.x >> 5);
    ChunkPlace pl;
    // released behind the wait of the launch in front, as the other form's join
    const bool work = find_chunk<32 * kChunkJoinWarps>(a.c, a.group, blockIdx.x, s_find, &pl);
    pdl_wait_prior_grids();
    pdl_release_dependents();
    if (!work || row >= pl.rows) return;
    const int seen = chunk_seen(a.c, pl, a.group), each = chunk_steps(seen, a.splits) * kChunkKeys;
    const int used = each > 0 ? (seen + each - 1) / each : 0;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float top = -INFINITY, sum = 0.0f;
    auto part = [&](int s) { return (static_cast<size_t>(blockIdx.x) * a.splits + s) * kChunkRows + row; };
    for (int s = 0; s < used; ++s) top = fmaxf(top, __ldcg(&a.part_ml[part(s)].x));
#pragma unroll 4
    for (int s = 0; s < used; ++s)
        add_part(x, sum, __ldcg(reinterpret_cast<const float4*>(a.part_o + part(s) * kKvDim) + lane), __ldcg(a.part_ml + part(s)), top);
    store_row<false>(a.out, a.lse, out_row(pl.w, a.c.kv_heads, a.group, pl.head, pl.row0 + row), x, top, sum);
}

}  // namespace

int kv4_chunk_set_attributes() {
    // the warpgroups trade registers against what a launch has: with fewer than 96 a thread they would wait for each other
    cudaFuncAttributes f{};
    const cudaError_t e = cudaFuncGetAttributes(&f, kv4_chunk_kernel);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (f.numRegs != 96) return static_cast<int>(cudaErrorInvalidKernelImage);
    return static_cast<int>(cudaFuncSetAttribute(kv4_chunk_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kChunkSmem + 1024));
}
int kv4_chunk_timeouts(unsigned int* out) { return static_cast<int>(cudaMemcpyFromSymbol(out, g_tc_wait_timeouts, sizeof(unsigned int))); }

Kv4ChunkPlan kv4_chunk_plan(int num_tokens, int num_seqs, int q_heads, int kv_heads) {
    Kv4ChunkPlan p;
    const long long group = q_heads / kv_heads, rows = group * num_tokens;
    const long long by_token = num_tokens * ((group + kChunkRows - 1) / kChunkRows), by_rows = rows / kChunkRows + num_seqs;
    p.tile_heads = (by_token < by_rows ? by_token : by_rows) * kv_heads;
    p.splits = static_cast<int>(p.tile_heads >= 74 ? 1 : 148 / p.tile_heads);
    const long long parts = p.splits > 1 ? p.tile_heads * p.splits * kChunkRows : 0;
    p.ml_offset = parts * kKvDim * 4;
    p.bytes = p.ml_offset + parts * 8;
    return p;
}

int kv4_chunk_attention(Kv4ChunkArgs a, int q_heads, void* workspace, cudaStream_t stream) {
    const Kv4ChunkPlan p = kv4_chunk_plan(a.c.num_tokens, a.c.num_seqs, q_heads, a.c.kv_heads);
    if (p.tile_heads * p.splits > 0x7FFFFFFFll) return W4A16_ERR_TOO_LARGE;
    a.splits = p.splits;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + p.ml_offset);
    cudaError_t e = launch_kernel(kv4_chunk_kernel, dim3(static_cast<unsigned>(p.tile_heads * p.splits)), dim3(kChunkThreads), kChunkSmem + 1024, stream, pdl_enabled(), a);
    if (e != cudaSuccess || p.splits == 1) return static_cast<int>(e);
    return static_cast<int>(launch_kernel(kv4_chunk_join_kernel, dim3(static_cast<unsigned>(p.tile_heads), kChunkRows / kChunkJoinWarps), dim3(32 * kChunkJoinWarps), 0,
                                          stream, pdl_enabled(), a));
}

}  // namespace w4
