// Attention of many query rows over the 4-bit key/value cache (chunks of a prompt), fp16 out, on tcgen05.
//
// A CTA has 256 query rows of one key/value head (token major, so the heads that share it lie side by side) as two tiles of 128,
// and walks over the positions 128 at a time:
//   S_i [128 rows x 128 positions] = Q_i . K^T      Q and K from shared memory
//   P_i = 2^(S_i c - m), fp16, over S_i in tensor memory; m is the running maximum, renewed only where a score exceeds it by 2^8
//   O_i [128 rows x 128 dims] += P_i . V            P from tensor memory, V (transposed: positions contiguous) from shared memory
// While the softmax warps of one tile work the tensor core has the other one.  Keys and values become fp16 once for both tiles:
// value = (code - 8) * scale + zero by one fma behind an exact conversion, so with one rounding.
//
// What bounds it: the exponentials (16 a cycle and SM: 2048 cycles for 256 x 128) and the tensor core (2048 cycles) alike, and
// behind them the issue slots of the softmax.
//
//   warps 0..3, 4..7 : softmax of tile 0 and 1, a thread a row; at the end they store O
//   warps 8..11      : keys, a thread a position: its row from global memory a step ahead in registers, to shared memory as fp16
//   warps 12..15     : values: codes through a staging buffer, then a thread takes 8 dims x 8 positions twice and stores them as
//                      rows of 8 positions.  Every access of both is free of bank conflicts (chunks of 16 bytes are xor-ed).
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
constexpr int kSoftWarps = 8, kKeyWarp = 8, kValueWarp = 12, kMmaWarp = 16, kChunkThreads = 17 * 32;
constexpr int kOperand = kTile * kKvDim * 2;              // bytes of a 128 x 128 operand: two panels of 64 columns, 128-byte swizzle
constexpr int kPanel = kOperand / 2;
constexpr int kValueStage = kChunkKeys * 64;
constexpr int kSmemK = 2 * kOperand, kSmemV = 4 * kOperand, kSmemStage = 6 * kOperand, kSmemParam = kSmemStage + 2 * kValueStage;
constexpr int kChunkSmem = kSmemParam + 2 * kChunkKeys * 4;
constexpr int kTmemO = 256;                               // S_0, S_1, O_0, O_1: 128 columns each

__device__ __forceinline__ void tc_mma_f16_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]),
          "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]),
          "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]),
          "=f"(r[31])
        : "r"(taddr)
        : "memory");
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
    const __half2 a = __float2half2_rn(-1032.0f), m = __float2half2_rn(0.0625f), b = __float2half2_rn(-72.0f);
    const uint32_t u = w >> 8;
    uint32_t r[4];
    asm("lop3.b32 %0, %1, 0x000F000F, 0x64006400, 0xEA;" : "=r"(r[0]) : "r"(w));      // 1024 + code
    asm("lop3.b32 %0, %1, 0x00F000F0, 0x64006400, 0xEA;" : "=r"(r[1]) : "r"(w));      // 1024 + 16 code
    asm("lop3.b32 %0, %1, 0x000F000F, 0x64006400, 0xEA;" : "=r"(r[2]) : "r"(u));
    asm("lop3.b32 %0, %1, 0x00F000F0, 0x64006400, 0xEA;" : "=r"(r[3]) : "r"(u));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 c = *reinterpret_cast<const __half2*>(&r[i]);
        const __half2 v = __hfma2(i & 1 ? __hfma2(c, m, b) : __hadd2(c, a), s, z);
        out[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
}
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }

// Row and 16-byte chunk (8 columns) of an operand in shared memory.
__device__ __forceinline__ uint32_t operand_at(int row, int chunk) {
    return static_cast<uint32_t>((chunk >> 3) * kPanel + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// The (tile, head) of a CTA: long ones first, which are the last ones of a sequence.
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
    auto k_full = [&](int i) { return bar0 + 8u * i; };
    auto k_empty = [&](int i) { return bar0 + 8u * (2 + i); };
    auto v_full = [&](int i) { return bar0 + 8u * (4 + i); };
    auto v_empty = [&](int i) { return bar0 + 8u * (6 + i); };
    auto s_full = [&](int i) { return bar0 + 8u * (8 + i); };
    auto p_full = [&](int i) { return bar0 + 8u * (10 + i); };
    const uint32_t q_full = bar0 + 8u * 12, finished = bar0 + 8u * 13;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (warp == kMmaWarp) {
        if (lane < 2) {
            mbar_init(k_full(lane), 4);
            mbar_init(k_empty(lane), 1);
            mbar_init(v_full(lane), 4);
            mbar_init(v_empty(lane), 1);
            mbar_init(s_full(lane), 1);
            mbar_init(p_full(lane), 4);
        }
        if (lane == 0) {
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
    const uint32_t tmem = s_tmem;
    pdl_release_dependents();           // not before: a CTA of the next launch must not take this one's tensor memory
    const int seen = work ? chunk_seen(c, pl, a.group) : 0, steps_each = chunk_steps(seen, a.splits);
    const int k0 = split * steps_each * kChunkKeys, k1 = min(seen, k0 + steps_each * kChunkKeys);
    const int steps = work && k1 > k0 ? (k1 - k0 + kChunkKeys - 1) / kChunkKeys : 0;
    const int tiles = work && pl.rows > kTile ? 2 : 1;
    const int32_t* table = c.table + static_cast<size_t>(work ? pl.seq : 0) * c.max_pages;
    const int ps = 1 << c.page_shift;

    if (warp < kSoftWarps) {
        // ================= softmax: thread = row = tensor-memory lane =================
        const int i = warp >> 2, r = tid & 127, row = i * kTile + r;
        const bool mine = work && row < pl.rows;
        const size_t at_row = mine ? out_row(pl.w, c.kv_heads, a.group, pl.head, pl.row0 + row) : 0;
        const int limit = mine ? pl.w.past + (pl.row0 + row) / a.group + 1 : 0x7FFFFFFF;
        if (steps > 0 && i < tiles) {
            uint4 w[16];
            const __half* src = a.q;
            if (mine) src += static_cast<size_t>(pl.w.first + (pl.row0 + row) / a.group) * a.q_stride + (pl.head * a.group + (pl.row0 + row) % a.group) * kKvDim;
#pragma unroll
            for (int k = 0; k < 16; ++k) w[k] = mine ? __ldcg(reinterpret_cast<const uint4*>(src) + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < 16; ++k)
                *reinterpret_cast<uint4*>(smem + i * kOperand + operand_at(r, k)) =
                    make_uint4(__byte_perm(w[k].x, w[k].y, 0x5410), __byte_perm(w[k].z, w[k].w, 0x5410), __byte_perm(w[k].x, w[k].y, 0x7632),
                               __byte_perm(w[k].z, w[k].w, 0x7632));
            fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        const float to_log2 = a.scale * kLog2e;
        const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t t_s = lanes + static_cast<uint32_t>(i * 128), t_o = lanes + static_cast<uint32_t>(kTmemO + i * 128);
        float m = -INFINITY, mu = 0.0f, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < (i < tiles ? steps : 0); ++j) {
            ok = warp_wait(s_full(i), j & 1, s_abort, lane);
            if (!ok) break;
            tc_fence_after();
            const int base = k0 + j * kChunkKeys;
            const uint4 there = *reinterpret_cast<const uint4*>(s_mask[j & 3][0]), poison = *reinterpret_cast<const uint4*>(s_mask[j & 3][1]);
            const uint32_t all = there.x & there.y & there.z & there.w, any = poison.x | poison.y | poison.z | poison.w;
            const bool simple = __all_sync(0xFFFFFFFFu, base + kChunkKeys <= limit && all == ~0u && any == 0);
            const uint32_t th[4] = {there.x, there.y, there.z, there.w}, po[4] = {poison.x, poison.y, poison.z, poison.w};
            auto sees = [&](int q) -> uint32_t {        // the row's positions of quarter q
                const int n = limit - base - 32 * q;
                return th[q] & (n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u);
            };
            float x[2][32];
            float top = -INFINITY;
            tmem_ld32(t_s, x[0]);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                tmem_ld_wait();
                if (q < 3) tmem_ld32(t_s + 32u * (q + 1), x[(q + 1) & 1]);
                float (&v)[32] = x[q & 1];
                if (!simple) {
                    const uint32_t bits = sees(q);
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] = bits >> k & 1u ? v[k] : -INFINITY;
                }
                float t4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (int k = 4; k < 32; ++k) t4[k & 3] = fmaxf(t4[k & 3], v[k]);
                top = fmaxf(top, fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])));
            }
            top *= to_log2;
            if (__any_sync(0xFFFFFFFFu, top > m + 8.0f)) {
                const float fresh = fmaxf(m, top), f = fresh == m ? 1.0f : ex2(m - fresh);
                m = fresh;
                mu = fresh == -INFINITY ? 0.0f : fresh;
                l *= f;
                if (j > 0) {
                    // the product of the step before is complete: s_full of this step was committed behind it
#pragma unroll 1
                    for (int q = 0; q < 4; ++q) {
                        tmem_ld32(t_o + 32u * q, x[0]);
                        tmem_ld_wait();
                        uint32_t y[2][16];
#pragma unroll
                        for (int k = 0; k < 32; ++k) y[k >> 4][k & 15] = __float_as_uint(x[0][k] * f);
                        tmem_st16(t_o + 32u * q, y[0]);
                        tmem_st16(t_o + 32u * q + 16u, y[1]);
                    }
                }
            }
            float sum[4] = {};
            tmem_ld32(t_s, x[0]);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                tmem_ld_wait();
                if (q < 3) tmem_ld32(t_s + 32u * (q + 1), x[(q + 1) & 1]);
                float (&v)[32] = x[q & 1];
                uint32_t p[16];
                if (simple) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] = ex2(fmaf(v[k], to_log2, -mu));
                } else {
                    const uint32_t bits = sees(q), bad = bits & po[q];
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        const float e = ex2(fmaf(v[k], to_log2, -mu));
                        v[k] = bits >> k & 1u ? (bad >> k & 1u ? __int_as_float(0x7FC00000) : e) : 0.0f;
                    }
                }
#pragma unroll
                for (int k = 0; k < 32; ++k) sum[k & 3] += v[k];
#pragma unroll
                for (int k = 0; k < 16; ++k) p[k] = pack_half2(v[2 * k], v[2 * k + 1]);
                tmem_st16(t_s + 16u * q, p);             // over the quarter before it, which has been read
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(i));
        }
        if (ok && steps > 0 && i < tiles) ok = warp_wait(finished, 0, s_abort, lane);
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
                    tmem_ld_wait();
                }
                if (!mine) continue;
                if (whole) {
                    __half* out = a.out + at_row * kKvDim + 32 * q;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = l == 0.0f ? 0u : pack_half2(x[8 * k + 2 * e] * f, x[8 * k + 2 * e + 1] * f);
                        reinterpret_cast<uint4*>(out)[k] = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                } else {
                    float4* out = reinterpret_cast<float4*>(a.part_o + part * kKvDim + 32 * q);
#pragma unroll
                    for (int k = 0; k < 8; ++k) __stcg(out + k, make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]));
                }
            }
            if (mine && whole && a.lse != nullptr) a.lse[at_row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
            if (mine && !whole) __stcg(a.part_ml + part, make_float2(m, l));
        }
    } else if (warp < kValueWarp) {
        // ================= keys: thread = position = row of the operand =================
        const int t = tid & 127;
        uint4 w[4];
        uint32_t kp = 0, vp = 0;
        bool there = false;
        int page = -1;
        auto page_of = [&](int j) { const int at = k0 + j * kChunkKeys + t; return j < steps && at < k1 ? __ldcg(table + (at >> c.page_shift)) : -1; };
        auto fetch = [&](int j) {
            const uint32_t* record = kv4_record_of_page(c, page, pl.head);
            there = record != nullptr;
            kp = vp = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = make_uint4(0, 0, 0, 0);
            if (there) {
                const int slot = (k0 + j * kChunkKeys + t) & (ps - 1);
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = __ldcg(reinterpret_cast<const uint4*>(record + slot * kKvRowWords) + k);
                kp = __ldcg(record + 32 * ps + slot);
                vp = __ldcg(record + 33 * ps + slot);
            }
            page = page_of(j + 1);
        };
        if (steps > 0) {
            page = page_of(0);
            fetch(0);
        }
        for (int j = 0; j < steps; ++j) {
            const int slot = j & 1;
            if (!warp_wait(k_empty(slot), ((j >> 1) & 1) ^ 1, s_abort, lane)) break;
            const uint32_t p = finite_params(kp);
            const __half2 s = __half2half2(__ushort_as_half(static_cast<unsigned short>(p))), z = __half2half2(__ushort_as_half(static_cast<unsigned short>(p >> 16)));
            const uint32_t here = __ballot_sync(0xFFFFFFFFu, there), bad = __ballot_sync(0xFFFFFFFFu, nan_params(vp));
            if (lane == 0) {
                s_mask[j & 3][0][warp - kKeyWarp] = here;
                s_mask[j & 3][1][warp - kKeyWarp] = bad;
            }
            uint8_t* to = smem + kSmemK + slot * kOperand;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t words[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t o[4];
                    dequantise(words[e], s, z, o);          // pairs (0, 2), (4, 6), (1, 3), (5, 7)
                    *reinterpret_cast<uint4*>(to + operand_at(t, 4 * k + e)) = make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
            if (j + 1 < steps) fetch(j + 1);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(k_full(slot));
        }
    } else if (warp < kMmaWarp) {
        // ================= values =================
        const int t = tid & 127, word = (lane >> 3) + 4 * (warp - kValueWarp);
        uint32_t vp = 0;
        int page = -1;
        auto page_of = [&](int j) { const int at = k0 + j * kChunkKeys + t; return j < steps && at < k1 ? __ldcg(table + (at >> c.page_shift)) : -1; };
        // position t's codes into the staging buffer, its parameters into a register
        const int oct = t >> 3;
        const uint32_t stage_to = smem0 + static_cast<uint32_t>(kSmemStage + (t ^ ((oct >> 2) & 1)) * 64);
        auto fetch = [&](int j) {
            const uint32_t* record = kv4_record_of_page(c, page, pl.head);
            vp = 0;
            if (record != nullptr) {
                const int slot = (k0 + j * kChunkKeys + t) & (ps - 1);
                const uint32_t* codes = record + (ps + slot) * kKvRowWords;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(stage_to + static_cast<uint32_t>((j & 1) * kValueStage + ((k ^ (oct & 3)) << 4))),
                                 "l"(codes + 4 * k) : "memory");
                vp = __ldcg(record + 33 * ps + slot);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            page = page_of(j + 1);
        };
        if (steps > 0) {
            page = page_of(0);
            fetch(0);
        }
        for (int j = 0; j < steps; ++j) {
            const int slot = j & 1;
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            uint32_t* params = reinterpret_cast<uint32_t*>(smem + kSmemParam) + slot * kChunkKeys;
            params[t] = nan_params(vp) ? 0u : finite_params(vp);
            asm volatile("bar.sync 1, 128;" ::: "memory");        // every position's codes and parameters are there, and the step before has been read
            if (j + 1 < steps) fetch(j + 1);
            if (!warp_wait(v_empty(slot), ((j >> 1) & 1) ^ 1, s_abort, lane)) break;
            uint8_t* to = smem + kSmemV + slot * kOperand;
            const uint8_t* stage = smem + kSmemStage + slot * kValueStage;
#pragma unroll
            for (int job = 0; job < 2; ++job) {
                const int o8 = (lane & 7) + 8 * job;               // eight positions
                const uint4 p0 = reinterpret_cast<const uint4*>(params)[2 * o8], p1 = reinterpret_cast<const uint4*>(params)[2 * o8 + 1];
                const uint32_t pr[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    w[e] = *reinterpret_cast<const uint32_t*>(stage + ((8 * o8 + e) ^ ((o8 >> 2) & 1)) * 64 + (((word >> 2) ^ (o8 & 3)) << 4) + (word & 3) * 4);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t v[4][4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        dequantise(__byte_perm(w[2 * e], w[2 * e + 1], half ? 0x7632 : 0x5410), as_half2(__byte_perm(pr[2 * e], pr[2 * e + 1], 0x5410)),
                                   as_half2(__byte_perm(pr[2 * e], pr[2 * e + 1], 0x7632)), v[e]);
                    constexpr int kElement[2][4] = {{0, 4, 1, 5}, {2, 6, 3, 7}};
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        *reinterpret_cast<uint4*>(to + operand_at(8 * word + kElement[half][n], o8)) = make_uint4(v[0][n], v[1][n], v[2][n], v[3][n]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(v_full(slot));
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else if (steps > 0) {
        // ================= MMA issue: one thread =================
        if (elect_one()) {
            const uint32_t idesc = make_idesc(kTile);
            auto scores = [&](int i, int slot) {
                const uint64_t qd = make_smem_desc(smem0 + static_cast<uint32_t>(i * kOperand)), kd = make_smem_desc(smem0 + static_cast<uint32_t>(kSmemK + slot * kOperand));
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const uint32_t off = (ks >= 4 ? kPanel >> 4 : 0) + 2u * (ks & 3);
                    tc_mma_f16_ss(tmem + static_cast<uint32_t>(i * 128), qd + off, kd + off, idesc, ks != 0);
                }
                tc_commit(s_full(i));
            };
            bool ok = mbar_wait(q_full, 0, s_abort) && mbar_wait(k_full(0), 0, s_abort);
            if (ok) {
                tc_fence_after();
                for (int i = 0; i < tiles; ++i) scores(i, 0);
                tc_commit(k_empty(0));
            }
            for (int j = 0; ok && j < steps; ++j) {
                const int slot = j & 1, next = slot ^ 1;
                ok = mbar_wait(v_full(slot), (j >> 1) & 1, s_abort);
                for (int i = 0; ok && i < tiles; ++i) {
                    ok = mbar_wait(p_full(i), j & 1, s_abort);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t vd = make_smem_desc(smem0 + static_cast<uint32_t>(kSmemV + slot * kOperand));
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)
                        tc_mma_f16_ts(tmem + static_cast<uint32_t>(kTmemO + i * 128), tmem + static_cast<uint32_t>(i * 128 + 8 * ks),
                                      vd + ((ks >= 4 ? kPanel >> 4 : 0) + 2u * (ks & 3)), idesc, j != 0 || ks != 0);
                    if (j + 1 < steps) {
                        if (i == 0) {
                            ok = mbar_wait(k_full(next), ((j + 1) >> 1) & 1, s_abort);
                            if (!ok) break;
                            tc_fence_after();
                        }
                        scores(i, next);
                    }
                }
                if (j + 1 < steps) tc_commit(k_empty(next));
                tc_commit(v_empty(slot));
            }
            tc_commit(finished);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (*s_abort) __nanosleep(500000);      // a bounded wait ran out: what is in flight lands before the memory goes
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// The splits of a (tile, head) joined, a warp a row.
constexpr int kChunkJoinWarps = 8;
__global__ void __launch_bounds__(32 * kChunkJoinWarps) kv4_chunk_join_kernel(const __grid_constant__ Kv4ChunkArgs a) {
    __shared__ FindScratch<32 * kChunkJoinWarps> s_find;
    pdl_wait_prior_grids();
    pdl_release_dependents();
    const int lane = threadIdx.x & 31, row = blockIdx.y * kChunkJoinWarps + (threadIdx.x >> 5);
    ChunkPlace pl;
    if (!find_chunk<32 * kChunkJoinWarps>(a.c, a.group, blockIdx.x, s_find, &pl) || row >= pl.rows) return;
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
