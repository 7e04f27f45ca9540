// Attention over the 4-bit key/value cache for single tokens and small groups of them, and the attention weight of every
// cached position.
//
// Both contract small sets of query rows with the cached rows on mma.sync.m16n8k16, the cached positions (or the values'
// dimensions) as the 16 rows of A and the queries as the 8 columns of B: a decode step has as many query rows as a key/value
// head has query heads, and these, not the positions, are what is padded.  The rows of a head (token major) are cut into tiles
// of 8 or 16; a tile's positions are split over CTAs, a CTA's over its four warps, 16 positions at a time.
//
//   scores^T [16 positions x 8 queries] = codes [16 x 128] . q^T;  then scale * score + zero * (sum of q), because a row is
//       (code - 8) * scale + zero: the codes are exact in fp16 and no key is ever rounded.
//   out^T [128 x 8] += codes^T [128 x 16] . (p * value scale)^T: for a 32-bit result the weight enters as two fp16 numbers
//       whose sum has 22 bits, for an fp16 result as one: its rounding and the result's own make 3.0e-4 where the
//       latter is 2.1e-4 (64 sequences of up to 8190 positions: 100 us, with both parts 106); zeros enter as one 32-bit sum a query.
//   reference of the exponents: not the largest score but the largest log2(p * value scale), so that what fp16 holds best is what counts most
//       in the result, whatever the value scales are (rows that get most of the attention often have the smallest values).  Renewed
//       where an fp16 weight could pass 2^15, which a vote finds, and set so that the largest is 2^6: a weight is off by 2^-31 of the
//       largest at most, or by 2^-22 of itself.  p itself is a 32-bit number that may be as large as 2^15 over the scale.
#include "kv4.cuh"
#include "kv4_attention.hpp"
#include "kv4_work.cuh"
#include "w4a16_internal.hpp"

namespace w4 {
namespace {

constexpr int kAttnWarps = 4, kAttnThreads = 32 * kAttnWarps;
static_assert(kUnit == kKvTile * kAttnWarps);

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// A warp's 16 positions in shared memory, copied there by itself (cp.async, 5 a lane) several steps ahead: what is in flight
// is what bounds this kernel (with one step ahead, in registers, 64 sequences of up to 8190 positions took 115 us), and registers
// are short.  Chunks of 16 bytes are placed so that no access meets another in a bank:
//   keys: the row of A number r holds position key_position(r), which makes the columns of p^T that the transposition leaves with
//         a lane the positions t, 4 + t, 8 + t and 12 + t; rows lie in order of r;
//   values: a lane reads 8 bytes of the rows t, 4 + t, ...; rows 2 and 3 of four have their halves swapped.
constexpr int kStageBytes = kKvTile * 136, kStages = 4;
constexpr int kStageValues = 1024, kStageKeyParams = 2048, kStageValueParams = 2112;
__device__ __forceinline__ int key_position(int r) { return ((r >> 1) & 3) + 4 * (r & 1) + (r & 8); }
__device__ __forceinline__ int key_row(int position) { return 2 * (position & 3) + ((position >> 2) & 1) + (position & 8); }

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
struct TileCopy {
    const char *keys, *values, *params;      // the lane's first chunk of each in the head's record of page 0
    size_t page;                             // bytes from page to page
    int in_page;                             // positions of a page, less one
    uint32_t key_to, value_to, param_to;     // where they go; the second ones lie 512 bytes on, as in the record

    __device__ __forceinline__ TileCopy(const Kv4View& c, int head_no, int lane, uint32_t ring) {
        const size_t record = static_cast<size_t>(kKvSlotWords * 4) << c.page_shift;
        const int ps = 1 << c.page_shift;
        const char* head = reinterpret_cast<const char*>(c.pages) + head_no * record;
        keys = head + 16 * lane;
        values = keys + 64 * ps;
        params = head + 128 * ps + 16 * (lane & 3) + (lane & 4) * ps;
        page = record * c.kv_heads;
        in_page = ps - 1;
        const int row = lane >> 2, chunk = lane & 3;          // and row + 8
        key_to = ring + static_cast<uint32_t>(key_row(row) * 64 + chunk * 16);
        value_to = ring + static_cast<uint32_t>(kStageValues + row * 64 + (chunk ^ (row & 2)) * 16);
        param_to = ring + static_cast<uint32_t>(kStageKeyParams + 16 * lane);
    }
    __device__ __forceinline__ void issue(uint32_t stage, int page_no, int at, int lane) const {
        const int s = at & in_page;
        const size_t rows = page_no * page + 64 * s;
        cp_async_16(key_to + stage, keys + rows);
        cp_async_16(key_to + stage + 512, keys + rows + 512);
        cp_async_16(value_to + stage, values + rows);
        cp_async_16(value_to + stage + 512, values + rows + 512);
        if (lane < 8) cp_async_16(param_to + stage, params + rows - 60 * s);
    }
};

// B fragments of eight query rows for the eight k steps: steps 2 j and 2 j + 1 take the elements of word 4 t + j in the order in
// which the code conversion gives them, 0 2 1 3 and 4 6 5 7.
__device__ __forceinline__ uint4 query_words(const uint4& w) {
    return make_uint4(__byte_perm(w.x, w.y, 0x5410), __byte_perm(w.x, w.y, 0x7632), __byte_perm(w.z, w.w, 0x5410), __byte_perm(w.z, w.w, 0x7632));
}
template <int NT, bool F32>
__global__ void __launch_bounds__(kAttnThreads, NT == 1 ? 4 : 2) kv4_attention_kernel(const __grid_constant__ Kv4AttentionArgs a) {
    constexpr int R = 8 * NT, kPitch = kKvDim + 4;
    __shared__ __align__(128) uint8_t s_ring[kAttnWarps][kStages * kStageBytes];     // and, behind the last position, the warps' sums
    __shared__ uint4 s_q[NT][4][32];         // the queries as B fragments; in registers they would leave too few for the rest
    __shared__ float2 s_ml[kAttnWarps][R];
    __shared__ FindScratch<kAttnThreads> s_find;
    static_assert(R * kPitch * 4 <= kStages * kStageBytes);
    auto s_o = [&](int w, int r, int d) -> float& { return reinterpret_cast<float*>(s_ring[w])[r * kPitch + d]; };
    const Kv4View& c = a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    long long per, all;
    Place pl;
    if (!c.settled) pdl_wait_prior_grids();
    const bool work = find_unit<kAttnThreads>(c, a.group, R, blockIdx.x, gridDim.x, s_find, &per, &all, &pl);
    if (c.settled) pdl_wait_prior_grids();
    pdl_release_dependents();               // the join reads lengths before its own wait, so not before this one's
    if (!work) return;
    long long left = min(per, all - per * blockIdx.x);
    for (bool first_part = true; left > 0; first_part = false) {
    while (pl.in_seq >= static_cast<long long>(pl.w.tiles) * c.kv_heads * pl.w.units) {      // past the sequence: the next one with work
        pl.w = seq_work(c, ++pl.seq, a.group, R);
        pl.in_seq = 0;
    }
    const int tile_head = static_cast<int>(pl.in_seq / pl.w.units), unit0 = static_cast<int>(pl.in_seq - static_cast<long long>(tile_head) * pl.w.units);
    const int head = tile_head % c.kv_heads, row0 = tile_head / c.kv_heads * R;
    const int units = static_cast<int>(min(left, static_cast<long long>(pl.w.units - unit0)));
    const bool whole = units == pl.w.units;
    left -= units;
    pl.in_seq += units;
    struct { int seq, first_token, row0, rows, past; } q = {pl.seq, pl.w.first, row0, min(R, pl.w.n * a.group - row0), pl.w.past};
    const int seen = min(max(q.past + (q.row0 + q.rows - 1) / a.group + 1, 0), kv4_capacity(c));
    const int k0 = unit0 * kUnit, k1 = min(k0 + units * kUnit, seen);

    // A page outside the pool is a step without copies.
    const uint8_t* ring = s_ring[warp];
    const TileCopy copy(c, head, lane, static_cast<uint32_t>(__cvta_generic_to_shared(ring)));
    const int32_t* table = c.table + static_cast<size_t>(q.seq) * c.max_pages;
    const int first_at = k0 + warp * kKvTile, steps = first_at < k1 ? (k1 - first_at + kUnit - 1) / kUnit : 0;
    auto page_of = [&](int step) { return step < steps ? __ldcg(table + ((first_at + step * kUnit) >> c.page_shift)) : -1; };
    auto start = [&](int step, int page) {
        const bool ok = static_cast<unsigned>(page) < static_cast<unsigned>(c.num_pages);
        if (ok) copy.issue(static_cast<uint32_t>(step % kStages) * kStageBytes, page, first_at + step * kUnit, lane);
        return ok;
    };
    // EARLY: page numbers of the first steps at once, all queries, and the rows on their way before the queries are used, instead of five
    // to nine round trips one behind the other: 8 sequences of 3 to 5 tokens 24.0 -> 20.6 us, 64 sequences 103 -> 100.6.  Eight
    // 32-bit rows have all registers in use, and what follows gets slower by more: one sequence of 131 001 positions 26.3 us
    // instead of 25.7, of 32 000 in the decode sweep 866 instead of 814 (of 1021: 610 instead of 620).
    constexpr bool EARLY = NT == 2 || !F32;
    static_assert(kStages == 4);
    int page[kStages] = {page_of(0), -1, -1, -1};
    if constexpr (EARLY) {
#pragma unroll
        for (int i = 1; i < kStages; ++i) page[i] = page_of(i);
    }

    // queries: B fragments of rows g (+ 8), and for the lane's columns 2 t, 2 t + 1 the sum of q and how far the row sees
    float qsum[NT][2];
    int limit[NT][2];
    const float to_log2 = a.scale * kLog2e;
    [[maybe_unused]] uint4 qw[NT][4];
    if constexpr (EARLY) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = n * 8 + g, row = q.row0 + r, token = q.first_token + row / a.group, h = head * a.group + row % a.group;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                qw[n][j] = r < q.rows ? __ldcg(reinterpret_cast<const uint4*>(a.q + static_cast<size_t>(token) * a.q_stride + h * kKvDim + 32 * t + 8 * j))
                                      : make_uint4(0, 0, 0, 0);
        }
    }
    uint32_t there = 0;                                     // bit i: the step i from now has rows
    auto begin = [&](int i) {
        if (start(i, page[i])) there |= 1u << i;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if constexpr (EARLY) {
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) begin(i);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if constexpr (EARLY) {
                w = qw[n][j];
            } else {
                const int r = n * 8 + g, row = q.row0 + r;
                if (r < q.rows) {
                    const int token = q.first_token + row / a.group, h = head * a.group + row % a.group;
                    w = __ldcg(reinterpret_cast<const uint4*>(a.q + static_cast<size_t>(token) * a.q_stride + h * kKvDim + 32 * t + 8 * j));
                }
            }
            s += sum_half8(w);
            if (j == warp) s_q[n][j][lane] = query_words(w);
        }
        s += __shfl_xor_sync(0xFFFFFFFFu, s, 1);
        s += __shfl_xor_sync(0xFFFFFFFFu, s, 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            qsum[n][e] = __shfl_sync(0xFFFFFFFFu, s, 4 * (2 * t + e)) * to_log2;
            limit[n][e] = q.past + (q.row0 + min(n * 8 + 2 * t + e, q.rows - 1)) / a.group + 1;
        }
    }
    const int all_see = q.past + q.row0 / a.group + 1;      // positions that every row of the tile sees
    __syncthreads();

    // m: reference of the exponents, renewed where a weight's logarithm is above `above` (m, or -infinity: by every step)
    constexpr float kNothingSeen = -3e38f;                  // finite: -infinity less it is -infinity
    float o[NT][8][4] = {}, m[NT][2], above[NT][2], l[NT][2] = {}, zacc[NT][2] = {};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            m[n][e] = kNothingSeen;
            above[n][e] = -INFINITY;
        }
    const int pos = key_position(g);                        // positions of rows g and g + 8 of A: pos and pos + 8
    const int value_from = kStageValues + 64 * t + ((8 * g) ^ (16 * (t & 2)));
    // CUT: some row does not see some of these positions
    auto take = [&]<bool CUT>(const uint8_t* st, int at) {
        struct { uint4 k[2]; uint2 v[4]; uint32_t kp[2], vp[2]; } r;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            r.k[i] = *reinterpret_cast<const uint4*>(st + 512 * i + 64 * g + 16 * t);
            r.kp[i] = *reinterpret_cast<const uint32_t*>(st + kStageKeyParams + 4 * pos + 32 * i);
            r.vp[i] = *reinterpret_cast<const uint32_t*>(st + kStageValueParams + 4 * pos + 32 * i);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[i] = *reinterpret_cast<const uint2*>(st + value_from + 256 * i);
        float s[NT][4] = {};
        const uint32_t kw0[4] = {r.k[0].x, r.k[0].y, r.k[0].z, r.k[0].w}, kw1[4] = {r.k[1].x, r.k[1].y, r.k[1].z, r.k[1].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t lo[4], hi[4];
            kv4_centred_codes(kw0[j], lo);
            kv4_centred_codes(kw1[j], hi);
            const uint32_t a0[4] = {lo[0], hi[0], lo[2], hi[2]}, a1[4] = {lo[1], hi[1], lo[3], hi[3]};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint4 b = s_q[n][j][lane];
                mma_16816(s[n], a0, b.x, b.y);
                mma_16816(s[n], a1, b.z, b.w);
            }
        }
        float ks[2], kz[2], vs[2], vz[2], lv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            ks[i] = kv4_scale(r.kp[i]);
            kz[i] = kv4_zero(r.kp[i]);
            ks[i] *= to_log2;
            vs[i] = kv4_scale(r.vp[i]);
            vz[i] = fmaf(-0.5f, vs[i], kv4_zero(r.vp[i]));  // codes are taken around 7.5
            // log2 of the scale less 15: exponent and seven bits of the mantissa as a number, at most 0.1 too small.  A scale of zero, or a
            // NaN, counts as 2^-60.
            lv[i] = fmaf(__uint_as_float(__byte_perm(__float_as_uint(fmaxf(vs[i], 0x1p-60f)), 0x4B000000u, 0x7632)), 0.0078125f, -(65536.0f + 127.0f + 15.0f));
        }
        bool renew = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = fmaf(s[n][e], ks[e >> 1], kz[e >> 1] * qsum[n][e & 1]);
        if constexpr (CUT) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (at + pos + 8 * (e >> 1) >= limit[n][e & 1]) s[n][e] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (at + pos + 8 * i >= k1) vs[i] = vz[i] = 0.0f;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) renew = renew || fmaxf(s[n][e] + lv[0], s[n][e + 2] + lv[1]) > above[n][e];
        if (__any_sync(0xFFFFFFFFu, renew)) {
            // From 2^23 on a score's neighbours are 1 and more away, and what is added to one is lost or rounded up: there the reference is the
            // largest score itself, at every step, so that a weight is the scale at most.
            constexpr float kFar = 8388608.0f;
            auto reference = [&](float score, float l) { return fabsf(score) < kFar ? score + (l + (15.0f - 6.0f)) : score; };
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = fmaxf(reference(s[n][e], lv[0]), reference(s[n][e + 2], lv[1]));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, d));
                    const float fresh = fmaxf(m[n][e], x);
                    const float f = fresh == m[n][e] ? 1.0f : ex2(m[n][e] - fresh);
                    m[n][e] = fresh;
                    above[n][e] = fabsf(fresh) < kFar ? fresh : -INFINITY;
                    l[n][e] *= f;
                    zacc[n][e] *= f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        o[n][i][e] *= f;
                        o[n][i][e + 2] *= f;
                    }
                }
        }
        uint32_t ph[NT][2];
        [[maybe_unused]] uint32_t pl[NT][2];                      // p * value scale in one or two fp16 parts, columns = positions
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = ex2(s[n][e] - m[n][e & 1]);
                l[n][e & 1] += p;
                x[e] = p * vs[e >> 1];
                float z = p * vz[e >> 1];
                if (CUT && at + pos + 8 * (e >> 1) >= limit[n][e & 1]) x[e] = z = 0.0f;   // whatever the row holds
                zacc[n][e & 1] += z;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                ph[n][i] = transpose_8x8(*reinterpret_cast<const uint32_t*>(&h));
                if constexpr (F32) {
                    const float2 b = __half22float2(h);
                    pl[n][i] = transpose_8x8(pack_half2(x[2 * i] - b.x, x[2 * i + 1] - b.y));
                }
            }
        }
        // values: pair two positions' words by 16-bit halves, then each nibble place is one dimension of both
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7632u : 0x5410u;
            uint32_t w[4][4];
            kv4_value_codes_to_half2(__byte_perm(r.v[0].x, r.v[1].x, sel), w[0]);
            kv4_value_codes_to_half2(__byte_perm(r.v[0].y, r.v[1].y, sel), w[1]);
            kv4_value_codes_to_half2(__byte_perm(r.v[2].x, r.v[3].x, sel), w[2]);
            kv4_value_codes_to_half2(__byte_perm(r.v[2].y, r.v[3].y, sel), w[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t av[4] = {w[0][i], w[1][i], w[2][i], w[3][i]};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma_16816(o[n][half * 4 + i], av, ph[n][0], ph[n][1]);
                    if constexpr (F32) mma_16816(o[n][half * 4 + i], av, pl[n][0], pl[n][1]);
                }
            }
        }
    };

    if constexpr (!EARLY) {
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) {
            begin(i);
            page[i + 1] = page_of(i + 1);
        }
    }
    int next_page = page[kStages - 1];
    // a page number is fetched one step before the copies that need it
    auto ahead = [&](int step) {
        const bool ok = step < steps && static_cast<unsigned>(next_page) < static_cast<unsigned>(c.num_pages);
        if (ok) copy.issue(static_cast<uint32_t>(step % kStages) * kStageBytes, next_page, first_at + step * kUnit, lane);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (step + 1 < steps) next_page = __ldcg(table + ((first_at + (step + 1) * kUnit) >> c.page_shift));
        there |= (ok ? 1u : 0u) << (kStages - 1);
    };
    for (int i = 0; i < steps; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncwarp();                                       // every lane's copies are there, and the slot of the step before has been read
        ahead(i + kStages - 1);
        if (there & 1u) {
            const int at = first_at + i * kUnit;
            const uint8_t* st = ring + (i % kStages) * kStageBytes;
            if (at + kKvTile > all_see) take.template operator()<true>(st, at);
            else take.template operator()<false>(st, at);
        }
        there >>= 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();

    // the warps' parts into shared memory: a lane has dimensions 16 g .. 16 g + 15 of queries 2 t and 2 t + 1
    constexpr int kElement[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float ls = l[n][e], zs = zacc[n][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                ls += __shfl_xor_sync(0xFFFFFFFFu, ls, d);
                zs += __shfl_xor_sync(0xFFFFFFFFu, zs, d);
            }
            const int r = n * 8 + 2 * t + e;
            if (g == 0) s_ml[warp][r] = make_float2(m[n][e] == kNothingSeen ? -INFINITY : m[n][e], ls);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s_o(warp, r, 16 * g + kElement[i]) = fmaf(o[n][i][e], kv4_value_undo(i), zs);
                s_o(warp, r, 16 * g + 8 + kElement[i]) = fmaf(o[n][i][e + 2], kv4_value_undo(i), zs);
            }
        }
    __syncthreads();
    const size_t part = 2 * static_cast<size_t>(blockIdx.x) + (first_part ? 0 : 1);
    // a warp a row, four dimensions a lane
    for (int r = warp; r < q.rows; r += kAttnWarps) {
        float2 ml[kAttnWarps];
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
            ml[w] = s_ml[w][r];
            top = fmaxf(top, ml[w].x);
        }
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) add_part(x, sum, *reinterpret_cast<const float4*>(&s_o(w, r, 4 * lane)), ml[w], top);
        if (whole) {
            store_row<F32>(a.out, a.lse, out_row(pl.w, c.kv_heads, a.group, head, q.row0 + r), x, top, sum);
        } else {
            __stcg(reinterpret_cast<float4*>(a.part_o + (part * R + r) * kKvDim + 4 * lane), x);
            if (lane == 0) __stcg(a.part_ml + part * R + r, make_float2(top, sum));
        }
    }
    __syncthreads();
    }
}

// The parts of a (tile, head) joined.  SPLIT: there are few (tile, head), so of many parts each; a CTA joins one row (blockIdx.y) of
// one (blockIdx.x), its warps sharing the parts.  Else a CTA stands at the boundary of the CTAs blockIdx.x and blockIdx.x + 1 of the
// launch above, works if that is the first boundary inside a (tile, head), and a warp joins the rows of its number.
constexpr int kJoinWarps = 16;
template <bool F32, bool SPLIT>
__global__ void __launch_bounds__(32 * kJoinWarps) kv4_attention_join_kernel(const __grid_constant__ Kv4AttentionArgs a, int tile_rows, int parts) {
    __shared__ FindScratch<32 * kJoinWarps> s_find;
    __shared__ float4 s_x[kJoinWarps][32];
    __shared__ float2 s_ml[kJoinWarps];
    const Kv4View& c = a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long per, all;
    Place pl;
    const int boundary = blockIdx.x + 1;
    // the attention in front releases this launch behind its own wait: what it read of the lengths is settled
    const bool work = find_unit<32 * kJoinWarps, SPLIT>(c, a.group, tile_rows, SPLIT ? blockIdx.x : boundary, parts, s_find, &per, &all, &pl);
    pdl_wait_prior_grids();
    pdl_release_dependents();
    if (!work) return;
    const int tile_head = static_cast<int>(SPLIT ? pl.in_seq : pl.in_seq / pl.w.units);
    const long long unit0 = pl.units_before + static_cast<long long>(tile_head) * pl.w.units;
    if (!SPLIT && (unit0 == per * boundary || unit0 < per * (boundary - 1))) return;
    const int c0 = SPLIT ? static_cast<int>(unit0 / per) : boundary - 1, c1 = static_cast<int>((unit0 + pl.w.units - 1) / per);
    if (c0 == c1) return;                // one CTA had it all
    const int head = tile_head % c.kv_heads, row0 = tile_head / c.kv_heads * tile_rows, rows = min(tile_rows, pl.w.n * a.group - row0);
    constexpr int kDeep = SPLIT ? 8 : 4, kStride = SPLIT ? kJoinWarps : 1;
    for (int r = SPLIT ? blockIdx.y : warp; r < rows; r += SPLIT ? tile_rows : kJoinWarps) {
        // part of CTA i: its first, unless the (tile, head) begins inside of it
        auto part_row = [&](int i) { return (2 * static_cast<size_t>(i) + (i == c0 && unit0 != per * c0 ? 1 : 0)) * tile_rows + r; };
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float top = -INFINITY, sum = 0.0f;
        for (int i0 = c0 + (SPLIT ? warp : 0); i0 <= c1; i0 += kStride * kDeep) {
            float4 p[kDeep];
            float2 ml[kDeep];
            float fresh = top;
#pragma unroll
            for (int d = 0; d < kDeep; ++d) {
                const int i = i0 + d * kStride;
                ml[d] = make_float2(-INFINITY, 0.0f);
                p[d] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (i <= c1) {
                    ml[d] = __ldcg(a.part_ml + part_row(i));
                    p[d] = __ldcg(reinterpret_cast<const float4*>(a.part_o + part_row(i) * kKvDim) + lane);
                }
            }
#pragma unroll
            for (int d = 0; d < kDeep; ++d) fresh = fmaxf(fresh, ml[d].x);
            const float4 old = x;
            const float2 old_ml = make_float2(top, sum);
            x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            sum = 0.0f;
            top = fresh;
            add_part(x, sum, old, old_ml, top);
#pragma unroll
            for (int d = 0; d < kDeep; ++d) add_part(x, sum, p[d], ml[d], top);
        }
        if constexpr (SPLIT) {
            s_x[warp][lane] = x;
            if (lane == 0) s_ml[warp] = make_float2(top, sum);
            __syncthreads();
            if (warp != 0) return;
            top = -INFINITY;
            sum = 0.0f;
            x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, s_ml[w].x);
#pragma unroll
            for (int w = 0; w < kJoinWarps; ++w) add_part(x, sum, s_x[w][lane], s_ml[w], top);
        }
        store_row<F32>(a.out, a.lse, out_row(pl.w, c.kv_heads, a.group, head, row0 + r), x, top, sum);
    }
}

// ---- attention weight of the cached positions ------------------------------------------------------------------

// A warp takes 32 positions of a head and adds up, over all query rows of the sequence, exp(score - lse), and
// adds that to the position's weight: one addition in memory for each block of rows, atomic because sequences may share pages (a common
// prefix).  Positions of one sequence alone get the same bits every time, as one thread makes all their additions.  The queries pass through shared memory in blocks of up to
// 128 rows, in fragment order, and stay there while the CTA walks over its positions; the codes of the next 32 are on their way
// meanwhile.  What bounds it is the rate of mma.sync (with a block of rows staged for each 128 positions it was the staging: the last 32
// tokens of two sequences of 32 000 and 20 000 positions, 32 heads on 8, took 111 us).
constexpr int kWeightRows = 128, kWeightPositions = 32 * kAttnWarps;

__global__ void __launch_bounds__(kAttnThreads, 3) kv4_key_weight_kernel(const __grid_constant__ Kv4WeightArgs a) {
    __shared__ uint4 s_q[kWeightRows / 8][4][32];
    __shared__ float2 s_row[kWeightRows];                    // sum of q, -lse, both in the exponent's units
    const Kv4View& c = a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    if (!c.settled) pdl_wait_prior_grids();
    const int head = blockIdx.y, b = blockIdx.z, ps = 1 << c.page_shift;
    const int first = blockIdx.x * a.positions + warp * 32;
    const int2 mine = kv4_new_tokens(c, b);
    const int len = max(__ldcg(c.lens + b), 0), past = len - mine.y;
    const int rows = mine.y * a.group, end = min(min(len, kv4_capacity(c)), (static_cast<int>(blockIdx.x) + 1) * a.positions);
    const float to_log2 = a.scale * kLog2e;
    const int32_t* table = c.table + static_cast<size_t>(b) * c.max_pages;
    if (c.settled) pdl_wait_prior_grids();
    pdl_release_dependents();
    if (blockIdx.x * a.positions >= end || rows <= 0) return;
    // what the lane needs of 32 positions: rows at + g + {0, 8, 16, 24}
    struct Raw {
        uint4 w[4];
        uint32_t params[4];
        int page[2];
    } raw;
    auto pages = [&](int at, int (&p)[2]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) p[u] = at + 16 * u < end ? __ldcg(table + ((at + 16 * u) >> c.page_shift)) : -1;
    };
    auto fetch = [&](int at) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t* record = kv4_record_of_page(c, raw.page[u], head);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                raw.w[2 * u + i] = make_uint4(0, 0, 0, 0);
                raw.params[2 * u + i] = 0;
                if (record != nullptr) {
                    const int s = ((at + 16 * u) & (ps - 1)) + g + 8 * i;
                    raw.w[2 * u + i] = __ldcg(reinterpret_cast<const uint4*>(record + s * kKvRowWords + 4 * t));
                    raw.params[2 * u + i] = __ldcg(record + 32 * ps + s);
                }
            }
        }
    };
    for (int r0 = 0; r0 < rows; r0 += kWeightRows) {
        int next[2];
        pages(first, raw.page);
        // a row is 16 pieces of 16 bytes; half-warps take rows
        const int staged = min((rows - r0 + 7) & ~7, kWeightRows);
        __syncthreads();
        for (int r = threadIdx.x >> 4; r < staged; r += kAttnThreads / 16) {
            const int piece = threadIdx.x & 15, row = r0 + r;
            uint4 w = make_uint4(0, 0, 0, 0);
            float lse = INFINITY;
            if (row < rows) {
                const int token = mine.x + row / a.group, h = head * a.group + row % a.group;
                w = __ldcg(reinterpret_cast<const uint4*>(a.q + static_cast<size_t>(token) * a.q_stride + h * kKvDim + 8 * piece));
                lse = __ldcg(a.lse + static_cast<size_t>(token) * c.kv_heads * a.group + h);
            }
            float s = sum_half8(w);
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
            s_q[r >> 3][piece & 3][(r & 7) * 4 + (piece >> 2)] = query_words(w);
            if (piece == 0) s_row[r] = make_float2(s * to_log2, -lse * kLog2e);
        }
        fetch(first);
        pages(first + kWeightPositions, next);
        __syncthreads();
        for (int at = first; at < end; at += kWeightPositions) {
            uint32_t codes[2][4][2][4];
            float ks[4], kz[4], got[4] = {};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                ks[k] = kv4_scale(raw.params[k]);
                kz[k] = kv4_zero(raw.params[k]);
                ks[k] *= to_log2;
                kv4_centred_codes(raw.w[k].x, codes[k >> 1][0][k & 1]);
                kv4_centred_codes(raw.w[k].y, codes[k >> 1][1][k & 1]);
                kv4_centred_codes(raw.w[k].z, codes[k >> 1][2][k & 1]);
                kv4_centred_codes(raw.w[k].w, codes[k >> 1][3][k & 1]);
            }
            // the lane's position in the end: 8 t + g, so that a warp's additions are one instruction on 128 bytes
            const int mine_at = at + 8 * t + g, mine_page = t < 2 ? raw.page[0] : raw.page[1];
            float* weight = nullptr;
            if (mine_at < end && static_cast<unsigned>(mine_page) < static_cast<unsigned>(c.num_pages)) weight = c.key_weight + kv4_weight_index(c, mine_page, head, mine_at);
            raw.page[0] = next[0];
            raw.page[1] = next[1];
            fetch(at + kWeightPositions);
            pages(at + 2 * kWeightPositions, next);
            auto add_rows = [&]<bool CUT>() {               // CUT: some row does not see some of these positions
                for (int n = 0; n < staged / 8; ++n) {
                    float s[2][4] = {};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 f = s_q[n][j][lane];
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const uint32_t a0[4] = {codes[u][j][0][0], codes[u][j][1][0], codes[u][j][0][2], codes[u][j][1][2]};
                            const uint32_t a1[4] = {codes[u][j][0][1], codes[u][j][1][1], codes[u][j][0][3], codes[u][j][1][3]};
                            mma_16816(s[u], a0, f.x, f.y);
                            mma_16816(s[u], a1, f.z, f.w);
                        }
                    }
                    const float4 row = *reinterpret_cast<const float4*>(&s_row[n * 8 + 2 * t]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float qs = e ? row.z : row.x, less = e ? row.w : row.y;
                        int limit = 0;
                        if constexpr (CUT) {
                            const int r = r0 + n * 8 + 2 * t + e;
                            limit = r < rows ? past + r / a.group + 1 : 0;
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float x = fmaf(s[k >> 1][2 * (k & 1) + e], ks[k], fmaf(kz[k], qs, less));
                            const float p = ex2(x);
                            if (!CUT || at + 8 * k + g < limit) got[k] += p;
                        }
                    }
                }
            };
            if (at + 32 <= past + r0 / a.group + 1) add_rows.template operator()<false>();
            else add_rows.template operator()<true>();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                got[k] += __shfl_xor_sync(0xFFFFFFFFu, got[k], 1);
                got[k] += __shfl_xor_sync(0xFFFFFFFFu, got[k], 2);
            }
            const float sum = t < 2 ? (t == 0 ? got[0] : got[1]) : t == 2 ? got[2] : got[3];
            if (weight != nullptr && sum != 0.0f) atomicAdd(weight, sum);
        }
    }
}

}  // namespace

Kv4AttentionPlan kv4_attention_plan(int num_tokens, int num_seqs, int q_heads, int kv_heads) {
    Kv4AttentionPlan p;
    const long long group = q_heads / kv_heads, rows = group * num_tokens;
    p.nt = rows > 8ll * num_seqs ? 2 : 1;
    p.ctas = 148 * (p.nt == 1 ? 4 : 2);
    const long long R = 8 * p.nt, by_token = num_tokens * ((group + R - 1) / R), by_rows = rows / R + num_seqs;
    p.tile_heads = (by_token < by_rows ? by_token : by_rows) * kv_heads;
    const long long parts = 2ll * p.ctas * R;
    p.ml_offset = parts * kKvDim * 4;
    p.bytes = p.ml_offset + parts * 8;
    return p;
}

int kv4_attention(Kv4AttentionArgs a, int q_heads, bool f32, void* workspace, cudaStream_t stream) {
    const Kv4View& c = a.c;
    const Kv4AttentionPlan p = kv4_attention_plan(c.num_tokens, c.num_seqs, q_heads, c.kv_heads);
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + p.ml_offset);
    auto kernel = p.nt == 1 ? (f32 ? kv4_attention_kernel<1, true> : kv4_attention_kernel<1, false>)
                            : (f32 ? kv4_attention_kernel<2, true> : kv4_attention_kernel<2, false>);
    // no more CTAs than there can be units
    const long long most = p.tile_heads * (((static_cast<long long>(c.max_pages) << c.page_shift) + kUnit - 1) / kUnit);
    const int ctas = static_cast<int>(most < p.ctas ? most : p.ctas);
    cudaError_t e = launch_kernel(kernel, dim3(ctas), dim3(kAttnThreads), 0, stream, pdl_enabled(), a);
    if (e != cudaSuccess || ctas == 1) return static_cast<int>(e);
    const bool split = p.tile_heads * 8 <= ctas;     // more than eight parts each
    auto join = split ? (f32 ? kv4_attention_join_kernel<true, true> : kv4_attention_join_kernel<false, true>)
                      : (f32 ? kv4_attention_join_kernel<true, false> : kv4_attention_join_kernel<false, false>);
    return static_cast<int>(launch_kernel(join, split ? dim3(static_cast<unsigned>(p.tile_heads), 8 * p.nt) : dim3(ctas - 1), dim3(32 * kJoinWarps), 0, stream, pdl_enabled(), a, 8 * p.nt, ctas));
}

int kv4_add_key_weights(Kv4WeightArgs a, cudaStream_t stream) {
    const Kv4View& c = a.c;
    // as many positions a CTA as leave each SM six CTAs, two rounds of three, where the tables are as long as the sequences; 128 at
    // least, 2048 at most
    const long long capacity = static_cast<long long>(c.max_pages) << c.page_shift;
    const long long each = capacity * c.kv_heads * c.num_seqs / (148 * 6);
    a.positions = static_cast<int>(each < kWeightPositions ? kWeightPositions : each > 2048 ? 2048 : each / kWeightPositions * kWeightPositions);
    const long long blocks = (capacity + a.positions - 1) / a.positions;
    const dim3 grid(static_cast<unsigned>(blocks), c.kv_heads, c.num_seqs);
    return static_cast<int>(launch_kernel(kv4_key_weight_kernel, grid, dim3(kAttnThreads), 0, stream, pdl_enabled(), a));
}

}  // namespace w4
