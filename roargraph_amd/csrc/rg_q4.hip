// rg_q4.hip -- a base in 4 bits with one scale (and minimum) per group of elements: packing, unpacking, exhaustive scores.
//
//   y_ij = sum_k q_ik v_jk,   v_jk = s_jg (c_jk - 8)   or   s_jg c_jk + m_jg = s_jg (c_jk - 8) + (m_jg + 8 s_jg)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "rg.h"
#include "rg_internal.h"
#include "rg_rows.h"

namespace rg {
namespace {

constexpr uint32_t kMaxDim = 4096;

__device__ __forceinline__ float half_bits(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// eight elements of a row from k on (n of them exist)
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T *row, uint32_t k, uint32_t n, float (&v)[8]) {
    if (n == 8) {                                    // (wide loads take any address)
        if constexpr (DT == RG_DTYPE_F32) {
            typedef f32x4 f32x4_a4 __attribute__((aligned(4)));
            const f32x4 a = *reinterpret_cast<const f32x4_a4 *>(row + k), b = *reinterpret_cast<const f32x4_a4 *>(row + k + 4);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < 4 ? a[i % 4] : b[i % 4];
        } else {
            typedef typename std::conditional<DT == RG_DTYPE_F16, half8, bf8>::type V;
            typedef V V_a2 __attribute__((aligned(2)));
            const V a = *reinterpret_cast<const V_a2 *>(row + k);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)row[k + min((uint32_t)i, n - 1)];      // (behind the row: its last element, which changes no extremum)
    }
}

// Packing: bound by reading the rows.  A lane holds eight elements, a group is 4, 8 or 16 neighbouring lanes.  The nearest level comes from an
// fp32 quotient wherever that is not close to the border of two; there (one wave in a hundred) 64 bits decide, in which x, minimum and
// code * scale are exact; ties go to the even code.
template <int DT>
__global__ void __launch_bounds__(256) rg_q4_pack_kernel(const void *rows, uint32_t nb, uint64_t stride, uint32_t dim, uint32_t group, uint8_t *codes, uint64_t cstride,
                                                         uint16_t *scales, uint16_t *mins, uint64_t sstride) {
    typedef typename Elem<DT>::T T;
    const uint32_t lanes = group / 8, D = (dim + 7) / 8, per_row = (D + lanes - 1) / lanes * lanes;
    const int first = mins ? 0 : -8;
    // (whole waves turn together: per_row * nb rounded up to them)
    const uint64_t total = (uint64_t)nb * per_row;
    uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    uint32_t j = (uint32_t)(at / per_row), l = (uint32_t)(at % per_row);
    const uint64_t hop = (uint64_t)gridDim.x * 256;
    const uint32_t hop_rows = (uint32_t)(hop / per_row), hop_lanes = (uint32_t)(hop % per_row);
    for (; at - threadIdx.x % 64 < total; at += hop) {
        const bool here = at < total && l < D;
        const uint32_t row = min(j, nb - 1), k = min(l, D - 1) * 8, n = min(8u, dim - k);
        float v[8];
        load8<DT>(static_cast<const T *>(rows) + (size_t)row * stride, k, n, v);
        float lo = v[0], hi = v[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) { lo = fminf(lo, v[i]); hi = fmaxf(hi, v[i]); }
        // (a lane behind the row holds the row's last eight again: of the same group as the lanes before it, or alone in a group that is none)
        for (uint32_t d = 1; d < lanes; d <<= 1) { lo = fminf(lo, __shfl_xor(lo, d)); hi = fmaxf(hi, __shfl_xor(hi, d)); }
        const _Float16 s16 = (_Float16)(mins ? (hi - lo) * (1.0f / 15.0f) : fmaxf(fabsf(lo), fabsf(hi)) * (1.0f / 7.0f)), m16 = (_Float16)(mins ? lo : 0.0f);
        const float s = (float)s16, m = (float)m16, inv = s > 0.0f ? 1.0f / s : 0.0f;
        // how far the fp32 quotient can be off: half a step of x - m and a few of the quotient
        const float off = (fabsf(m) * inv + 32.0f) * 0x1p-22f;
        float c[8];
        bool close = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float t = (v[i] - m) * inv;        // (a scale of zero: all are level 0)
            c[i] = rintf(t);
            close |= fabsf(fabsf(t - c[i]) - 0.5f) <= off;
        }
        if (__any(close)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double r = fma(-(double)c[i], (double)s, (double)v[i] - (double)m), half = 0.5 * (double)s;
                const bool odd = ((int)c[i] & 1) != 0;
                if (s == 0.0f) continue;             // (one level)
                if (r > half || (r == half && odd)) c[i] += 1.0f;
                else if (r < -half || (r == -half && odd)) c[i] -= 1.0f;
            }
        }
        float half[2] = {0.0f, 0.0f};                // four codes each (codes and their sums are whole numbers)
#pragma unroll
        for (int i = 7; i >= 0; --i) {
            const float code = __builtin_amdgcn_fmed3f(c[i], (float)first, (float)(first + 15)) - (float)first;
            half[i / 4] = fmaf(half[i / 4], 16.0f, (uint32_t)i < n ? code : 0.0f);
        }
        const uint32_t w = (uint32_t)half[0] | (uint32_t)half[1] << 16;
        if (here) {
            *reinterpret_cast<uint32_t *>(codes + (size_t)j * cstride + l * 4) = w;
            if (l % lanes == 0) {
                scales[(size_t)j * sstride + l / lanes] = __builtin_bit_cast(uint16_t, s16);
                if (mins) mins[(size_t)j * sstride + l / lanes] = __builtin_bit_cast(uint16_t, m16);
            }
        }
        l += hop_lanes;
        j += hop_rows;
        if (l >= per_row) { l -= per_row; ++j; }
    }
}

// Unpacking: bound by writing the values, eight a lane, past the caches (nobody reads them soon) and at any alignment; the last lane of a row
// writes what is left of it.  (One value a lane where rows are not 16-byte aligned: 100,003 x 301 55 us, now 27 us.)
__global__ void __launch_bounds__(256) rg_q4_unpack_kernel(const uint8_t *codes, uint64_t cstride, const uint16_t *scales, const uint16_t *mins, uint64_t sstride, uint32_t nb, uint32_t dim,
                                                           uint32_t group, const uint32_t *ids, uint32_t n, float *out, uint64_t ostride) {
    typedef f32x4 f32x4_a4 __attribute__((aligned(4)));
    const bool whole = ((uintptr_t)out | ostride * 4) % 16 == 0;
    const uint32_t per_row = (dim + 7) / 8;
    uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    uint32_t i = (uint32_t)(at / per_row), l = (uint32_t)(at % per_row);
    const uint64_t hop = (uint64_t)gridDim.x * 256;
    const uint32_t hop_rows = (uint32_t)(hop / per_row), hop_lanes = (uint32_t)(hop % per_row);
    for (; at < (uint64_t)n * per_row; at += hop) {
        const uint32_t j = ids ? ids[i] : i, k = 8 * l;
        float v[8];
        if (j < nb) {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(codes + (size_t)j * cstride + l * 4);
            const float s = half_bits(scales[(size_t)j * sstride + k / group]), m = mins ? half_bits(mins[(size_t)j * sstride + k / group]) : 0.0f;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                const uint32_t c = w >> (4 * e) & 15u;
                v[e] = mins ? (float)c * s + m : (float)((int)c - 8) * s;
            }
        } else {                                     // no such row
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) v[e] = NAN;
        }
        float *to = out + (size_t)i * ostride + k;
        if (k + 8 <= dim && !whole) {                // (lines shared by two rows are put together in the cache)
            *reinterpret_cast<f32x4_a4 *>(to) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4_a4 *>(to + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else if (k + 8 <= dim) {
            __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4_a4 *>(to));
            __builtin_nontemporal_store(f32x4{v[4], v[5], v[6], v[7]}, reinterpret_cast<f32x4_a4 *>(to + 4));
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 7; ++e)
                if (k + e < dim) to[e] = v[e];
        }
        l += hop_lanes;
        i += hop_rows;
        if (l >= per_row) { l -= per_row; ++i; }
    }
}

// ---------------------------------------------------------------- scores
//
// Bound by reading the codes; the arithmetic has to stay out of the way.  v_mfma_f32_16x16x32_f16 with queries as the A operand -- rows 2 q and
// 2 q + 1 are the halves of query q, x = 2^e (hi + lo), 22 bits relative to its largest element, so that eight fp32 queries cost what one
// costs -- and 16 rows of the base as the B operand.
//
//   a code needs no conversion: its four bits, moved to the top of the fraction of an fp16, are the subnormal c 2^-18, which the matrix core
//   takes exactly.  Eight instructions make eight operands of a dword.  (At the bottom, where they lie -- c 2^-24 and 16 c 2^-24, five
//   instructions -- the products were right, but not the sums: they are aligned by the operands' exponents, and a subnormal's is 2^-14
//   whatever its leading zeros, so 6 and more bits of each fell off: an error of 9e-7 of the scores' norm instead of 8e-8, for 287 us instead
//   of 294 us, one query on 10M x 200.)
//   the partial sum of a group starts at -8 times the queries' sum over it, so that it is that of c - 8, and is then multiplied by the
//   row's scale in fp32: lane (n, g) holds it for row n and queries 2 g, 2 g + 1
//   minima: s c + m = s (c - 8) + (m + 8 s), and the queries' sum is at hand
//
// A wave takes 32 rows at a time; lane (n, g) reads 16 bytes = 32 codes of row n, chunk 4 j + g of the row.  (A row's last chunk is moved back
// to end with the row; what the chunk before it holds already meets zeros in the query.)  One product must see one group only: for
// groups of 128 the chunks of a step are that, for 32 and 64 the dwords change lanes first (permlane swaps).  kScoreDepth steps are
// on their way while one is multiplied.  A dword's codes come out in the order 0 4 1 5 2 6 3 7, and the queries lie in LDS in that order.
//
// (A first form made s (c - 8) of every code, exactly, as a pair of halves: 21 vector instructions a dword, 72 % of the vector units' time and 3.3 TB/s.)
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));

struct ScoreArgs {
    const uint8_t *codes;
    const uint16_t *scales, *mins;
    const void *queries;
    float *out;
    uint64_t cstride, sstride, qstride, ostride;
    uint32_t nb, nq, dim, groups;
    int dtype;
};

constexpr int kScoreThreads = 512, kScoreRows = 32, kScoreDepth = 2;

// where product u of a step finds its dword in lane group g: (lane group it was read by, dword of the 16 bytes)
template <int GS> __device__ __forceinline__ constexpr uint32_t from_group(uint32_t u, uint32_t g) { return GS == 0 ? u : GS == 1 ? (u & 1) * 2 + (g & 1) : g; }
template <int GS> __device__ __forceinline__ constexpr uint32_t from_dword(uint32_t u, uint32_t g) { return GS == 0 ? g : GS == 1 ? (u & 2) + (g >> 1) : u; }
template <int GS>
__device__ __forceinline__ void exchange(u32x4 &c) {
    if constexpr (GS < 2) {
        auto p = __builtin_amdgcn_permlane32_swap(c[0], c[1], false, false), q = __builtin_amdgcn_permlane32_swap(c[2], c[3], false, false);
        if constexpr (GS == 1) {
            c = u32x4{p[0], p[1], q[0], q[1]};
        } else {                                     // lane groups (0 1 | 2 3) -> a 4 x 4 transpose
            p = __builtin_amdgcn_permlane32_swap(c[0], c[2], false, false);
            q = __builtin_amdgcn_permlane32_swap(c[1], c[3], false, false);
            const auto a = __builtin_amdgcn_permlane16_swap(p[0], q[0], false, false), b = __builtin_amdgcn_permlane16_swap(p[1], q[1], false, false);
            c = u32x4{a[0], a[1], b[0], b[1]};
        }
    }
}

// a row's values of the groups of a step, from the lane groups that read them to every lane
template <int GS>
__device__ __forceinline__ void spread(uint32_t v, uint32_t (&out)[4 >> GS]) {
    if constexpr (GS == 2) {
        out[0] = v;
    } else {
        const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        if constexpr (GS == 1) {
            out[0] = p[0];
            out[1] = p[1];
        } else {
            const auto a = __builtin_amdgcn_permlane16_swap(p[0], p[0], false, false), b = __builtin_amdgcn_permlane16_swap(p[1], p[1], false, false);
            out[0] = a[0];
            out[1] = a[1];
            out[2] = b[0];
            out[3] = b[1];
        }
    }
}

// element i of the eight holds element order(i) of the dword
__device__ __forceinline__ constexpr int code_order(int i) { return i % 2 * 4 + i / 2; }
__device__ __forceinline__ half8 codes8(uint32_t w) {
    return __builtin_bit_cast(half8, u32x4{w << 6 & 0x03c003c0u, w << 2 & 0x03c003c0u, w >> 2 & 0x03c003c0u, w >> 6 & 0x03c003c0u});
}

// NQB blocks of eight queries at a time; groups of 32 << GS elements
template <int NQB, int GS, bool MINS>
__global__ void __launch_bounds__(kScoreThreads, NQB == 1 ? 4 : 2) rg_q4_score_kernel(ScoreArgs A) {
    constexpr uint32_t NS = 4 >> GS;                  // groups of a step
    extern __shared__ char lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
    const uint32_t dim = A.dim, D = (dim + 7) / 8, chunks = (D + 3) / 4, steps = (chunks + 3) / 4;       // dwords, chunks, steps of four chunks of a row
    half8 *X = reinterpret_cast<half8 *>(lds);                                        // [block][step][product][lane]
    f32x4 *seed = reinterpret_cast<f32x4 *>(lds + (size_t)NQB * steps * 4096);        // [block][step][group][lane group]: what a partial sum starts at
    float *factor = reinterpret_cast<float *>(seed + NQB * steps * NS * 4);           // [query]

    struct Stage {
        u32x4 c[2];
        uint32_t s[2], m[2];                         // of the group lane group g reads: 4 j + g, 2 j + g / 2 or j
    };
    Stage ring[kScoreDepth];
    const uint32_t waves = kScoreThreads / 64, tiles = (A.nb + kScoreRows - 1) / kScoreRows;
    const uint32_t stride = gridDim.x * waves, first = wave * gridDim.x + blockIdx.x;
    const uint32_t mine = first < tiles ? (tiles - first - 1) / stride + 1 : 0;
    const uint32_t total = mine * steps;             // (the host's rule: below 2^32)
    // What is fetched next: a uniform address of the tile and 32-bit offsets of the lanes, so that a step's loads cost a few vector
    // instructions.  In the last tile rows behind the last one are read as the last.
    uint32_t ptile = first, pstep = 0, asked = 0;
    uint32_t code_at[2], scale_at[2];
    auto rows_of = [&](uint32_t tile) {
        const uint32_t last = min((uint32_t)kScoreRows, A.nb - tile * kScoreRows) - 1;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            code_at[r] = min(16 * r + n, last) * (uint32_t)A.cstride;
            scale_at[r] = min(16 * r + n, last) * (uint32_t)A.sstride * 2;
        }
    };
    if (mine) rows_of(first);
    auto fetch = [&](Stage &st) {
        if (asked == total) return;
        ++asked;
        const char *codes = reinterpret_cast<const char *>(A.codes + (size_t)ptile * kScoreRows * A.cstride);
        const char *scales = reinterpret_cast<const char *>(A.scales + (size_t)ptile * kScoreRows * A.sstride), *mins = reinterpret_cast<const char *>(A.mins + (size_t)ptile * kScoreRows * A.sstride);
        const uint32_t chunk = 4 * pstep + g, group2 = min(chunk >> GS, A.groups - 1) * 2;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (D >= 4) {
                st.c[r] = *reinterpret_cast<const u32x4_a4 *>(codes + (code_at[r] + min(16 * chunk, 4 * D - 16)));
            } else {
#pragma unroll
                for (int t = 0; t < 4; ++t) st.c[r][t] = *reinterpret_cast<const uint32_t *>(codes + (code_at[r] + 4 * min((uint32_t)t, D - 1)));
            }
            st.s[r] = *reinterpret_cast<const uint16_t *>(scales + (scale_at[r] + group2));
            if (MINS) st.m[r] = *reinterpret_cast<const uint16_t *>(mins + (scale_at[r] + group2));
        }
        if (++pstep == steps) {
            pstep = 0;
            ptile += stride;
            if (ptile == tiles - 1) rows_of(ptile);
        }
    };
#pragma unroll
    for (int d = 0; d < kScoreDepth; ++d) fetch(ring[d]);

    // N elements of a query from element k on, behind dim the last one again (nothing waits between the loads)
    auto values = [&](uint32_t q, uint32_t k, uint32_t apart, auto &v) {
        constexpr int N = sizeof(v) / sizeof(v[0]);
        const char *row = static_cast<const char *>(A.queries) + (size_t)q * A.qstride * (A.dtype == RG_DTYPE_F32 ? 4 : 2);
        if (A.dtype == RG_DTYPE_F32) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = reinterpret_cast<const float *>(row)[min(k + i * apart, dim - 1)];
        } else if (A.dtype == RG_DTYPE_F16) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = (float)reinterpret_cast<const _Float16 *>(row)[min(k + i * apart, dim - 1)];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = (float)reinterpret_cast<const __bf16 *>(row)[min(k + i * apart, dim - 1)];
        }
    };
    for (uint32_t q0 = 0; q0 < A.nq; q0 += 8 * NQB) {
        // queries: the largest element of each, then halves in operand order (zeros behind dim and behind the last query) and sums of groups
        for (uint32_t q = wave; q < 8 * NQB; q += waves) {
            uint32_t m = 0;
            if (q0 + q < A.nq)
                for (uint32_t k = lane; k < dim; k += 256) {
                    float v[4];
                    values(q0 + q, k, 64, v);
#pragma unroll
                    for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
                }
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
            if (lane == 0) factor[q] = __uint_as_float(m);
        }
        __syncthreads();
        for (uint32_t i = tid; i < NQB * steps * 4 * 4 * 8; i += kScoreThreads) {
            const uint32_t q = i % 8, gg = i / 8 % 4, u = i / 32 % 4, j = i / 128 % steps, qb = i / 128 / steps;
            const float top = factor[qb * 8 + q], down = pow2(-row_exponent(top));
            const uint32_t c = 4 * j + from_group<GS>(u, gg), d = (D >= 4 ? min(4 * c, D - 4) : 0) + from_dword<GS>(u, gg);
            const bool any = q0 + qb * 8 + q < A.nq && d >= 4 * c && d < D;
            float v[8];
            values(any ? q0 + qb * 8 + q : q0, 8 * min(d, D - 1), 1, v);
            half8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float x = v[code_order(e)];          // scaled; of a query that is not finite the signs of its infinities
                x = top < INFINITY ? x * down : fabsf(x) < INFINITY ? 0.0f : fabsf(x) == INFINITY ? copysignf(1.0f, x) : x;
                x = any && 8 * d + code_order(e) < dim ? x : 0.0f;
                hi[e] = (_Float16)x;
                lo[e] = (_Float16)(x - (float)hi[e]);
            }
            half8 *at = X + ((size_t)(qb * steps + j) * 4 + u) * 64 + gg * 16 + 2 * q;
            at[0] = hi;
            at[1] = lo;
        }
        __syncthreads();
        for (uint32_t i = tid; i < NQB * steps * NS * 16; i += kScoreThreads) {
            const uint32_t h = i % 16, u = i / 16 % NS, j = i / 16 / NS % steps, qb = i / 16 / NS / steps;
            float sum = 0.0f;                        // of the halves as they are multiplied
#pragma unroll
            for (uint32_t p = 0; p < (1u << GS); ++p)
#pragma unroll
                for (uint32_t gg = 0; gg < 4; ++gg) {
                    const half8 x = X[((size_t)(qb * steps + j) * 4 + u + p * NS) * 64 + gg * 16 + h];
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum += (float)x[e];
                }
            reinterpret_cast<float *>(seed + ((size_t)(qb * steps + j) * NS + u) * 4)[h] = sum * -0x1p-15f;      // -8 x 2^-18
        }
        __syncthreads();

        if (q0) {                                    // the base once more for the next queries
            ptile = first;
            pstep = asked = 0;
            if (mine) rows_of(first);
#pragma unroll
            for (int d = 0; d < kScoreDepth; ++d) fetch(ring[d]);
        }
        f32x4 acc[2][NQB];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int b = 0; b < NQB; ++b) acc[r][b] = f32x4{0, 0, 0, 0};
        uint32_t tile = first, step = 0;
        for (uint32_t it = 0; it < total; it += kScoreDepth) {
#pragma unroll
            for (int d = 0; d < kScoreDepth; ++d) {
                if (it + d >= total) break;
                Stage st = ring[d];
                fetch(ring[d]);
                uint32_t scale[2][NS], low[2][NS];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    exchange<GS>(st.c[r]);
                    spread<GS>(st.s[r], scale[r]);
                    if (MINS) spread<GS>(st.m[r], low[r]);
                }
#pragma unroll
                for (int b = 0; b < NQB; ++b) {
                    half8 x[4];
                    f32x4 start[NS];
#pragma unroll
                    for (int u = 0; u < 4; ++u) x[u] = X[((size_t)(b * steps + step) * 4 + u) * 64 + lane];
#pragma unroll
                    for (uint32_t u = 0; u < NS; ++u) start[u] = seed[((size_t)(b * steps + step) * NS + u) * 4 + g];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        f32x4 sum[NS];
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const int v = GS == 0 ? u : GS == 1 ? u & 1 : 0;
                            sum[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[u], codes8(st.c[r][u]), u == v ? start[v] : sum[v], 0, 0, 0);
                        }
#pragma unroll
                        for (uint32_t u = 0; u < NS; ++u) {
                            const float s = half_bits((uint16_t)scale[r][u]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[r][b][i] = fmaf(s, sum[u][i], acc[r][b][i]);
                            if (MINS) {
                                const float off = fmaf(half_bits((uint16_t)low[r][u]), -0.125f, -s);      // -(m + 8 s) / 8
#pragma unroll
                                for (int i = 0; i < 4; ++i) acc[r][b][i] = fmaf(off, start[u][i], acc[r][b][i]);
                            }
                        }
                    }
                }
                if (++step == steps) {
                    step = 0;
#pragma unroll
                    for (int b = 0; b < NQB; ++b)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t q = b * 8 + 2 * g + h;
                            const float top = factor[q], up = row_factor(top, row_exponent(top));
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const uint32_t row = tile * kScoreRows + 16 * r + n;
                                if (q0 + q < A.nq && row < A.nb) A.out[(size_t)(q0 + q) * A.ostride + row] = (acc[r][b][2 * h] + acc[r][b][2 * h + 1]) * 0x1p18f * up;
                            }
                        }
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int b = 0; b < NQB; ++b) acc[r][b] = f32x4{0, 0, 0, 0};
                    tile += stride;
                }
            }
        }
        __syncthreads();
    }
}

size_t score_lds(uint32_t dim, int nqb, uint32_t group) {
    const size_t steps = (((dim + 7) / 8 + 3) / 4 + 3) / 4;
    return nqb * (steps * (4096 + 128 / group * 64) + 32);
}

template <int NQB, int GS>
rg_status launch_score(const ScoreArgs &A, size_t lds, hipStream_t s) {
    auto kern = A.mins ? rg_q4_score_kernel<NQB, GS, true> : rg_q4_score_kernel<NQB, GS, false>;
    if (lds > 64 * 1024) RG_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    const uint32_t tiles = (A.nb + kScoreRows - 1) / kScoreRows, per_cu = std::max<uint32_t>(1, std::min<uint32_t>(2, (uint32_t)(160 * 1024 / lds)));
    hipLaunchKernelGGL(kern, dim3(std::min(tiles, 256u * per_cu)), dim3(kScoreThreads), lds, s, A);
    RG_HIP(hipGetLastError());
    return RG_OK;
}
template <int GS>
rg_status launch_score_gs(const ScoreArgs &A, hipStream_t s) {
    // as many queries per reading of the base as there are, and as LDS holds
    const uint32_t group = 32 << GS;
    int nqb = A.nq > 16 ? 4 : A.nq > 8 ? 2 : 1;
    while (score_lds(A.dim, nqb, group) > 160 * 1024) nqb /= 2;
    const size_t lds = score_lds(A.dim, nqb, group);
    return nqb == 4 ? launch_score<4, GS>(A, lds, s) : nqb == 2 ? launch_score<2, GS>(A, lds, s) : launch_score<1, GS>(A, lds, s);
}

rg_status check_form(const void *codes, uint64_t cstride, const void *scales, const void *mins, uint64_t sstride, uint32_t nb, uint32_t dim, uint32_t group) {
    if (group != 32 && group != 64 && group != 128) return set_error(RG_ERR_ARG, "4-bit base: groups of 32, 64 or 128 elements");
    if (dim == 0 || dim > kMaxDim) return set_error(RG_ERR_ARG, "4-bit base: dim must be in [1, 4096]");
    if (nb > 0x7fffffffu) return set_error(RG_ERR_ARG, "4-bit base: at most 2^31 - 1 rows");
    if (cstride > 1u << 26 || sstride > 1u << 25) return set_error(RG_ERR_ARG, "4-bit base: row strides of at most 64 MB");
    if (nb == 0) return RG_OK;
    if (!codes || !scales) return set_error(RG_ERR_ARG, "null argument");
    if (cstride % 4 || cstride < (uint64_t)aligned_dim(dim) / 2 || (uintptr_t)codes % 4) return set_error(RG_ERR_ARG, "4-bit base: code rows are 4-byte aligned and hold dim rounded up to 8 elements");
    if (sstride < (dim + group - 1) / group || (uintptr_t)scales % 2 || (uintptr_t)mins % 2) return set_error(RG_ERR_ARG, "4-bit base: one fp16 scale (and minimum) per group of a row");
    return RG_OK;
}

}  // namespace
}  // namespace rg

using namespace rg;

extern "C" {

rg_status rg_q4_pack_dev(const void *d_rows, uint32_t nb, uint64_t stride, uint32_t dim, int dtype, uint32_t group, uint8_t *d_codes,
                         uint64_t cstride, uint16_t *d_scales, uint16_t *d_mins, uint64_t sstride, int device, void *stream) {
    rg_status st = check_form(d_codes, cstride, d_scales, d_mins, sstride, nb, dim, group);
    if (st != RG_OK) return st;
    if (!known_dtype(dtype)) return set_error(RG_ERR_ARG, "unknown dtype");
    if (nb == 0) return RG_OK;
    if (!d_rows) return set_error(RG_ERR_ARG, "null argument");
    if (stride < dim || (uintptr_t)d_rows % elem_bytes(dtype)) return set_error(RG_ERR_ARG, "rows: stride smaller than dim, or not aligned to their elements");
    OnDevice on(device);
    if (on.st != RG_OK) return on.st;
    const uint64_t n = (uint64_t)nb * ((dim + group - 1) / group) * (group / 8);
    auto kern = dtype == RG_DTYPE_F32 ? rg_q4_pack_kernel<RG_DTYPE_F32> : dtype == RG_DTYPE_F16 ? rg_q4_pack_kernel<RG_DTYPE_F16> : rg_q4_pack_kernel<RG_DTYPE_BF16>;
    hipLaunchKernelGGL(kern, dim3((uint32_t)std::min<uint64_t>((n + 255) / 256, 256u * 32u)), dim3(256), 0, (hipStream_t)stream, d_rows, nb, stride, dim, group, d_codes, cstride, d_scales, d_mins, sstride);
    RG_HIP(hipGetLastError());
    return RG_OK;
}

rg_status rg_q4_unpack_dev(const uint8_t *d_codes, uint64_t cstride, const uint16_t *d_scales, const uint16_t *d_mins, uint64_t sstride,
                           uint32_t nb, uint32_t dim, uint32_t group, const uint32_t *d_ids, uint32_t n, float *d_out, uint64_t ostride,
                           int device, void *stream) {
    rg_status st = check_form(d_codes, cstride, d_scales, d_mins, sstride, nb, dim, group);
    if (st != RG_OK) return st;
    if (!d_ids && n > nb) return set_error(RG_ERR_ARG, "more rows asked for than there are");
    if (n > 0x7fffffffu) return set_error(RG_ERR_ARG, "4-bit base: at most 2^31 - 1 rows");
    if (n == 0) return RG_OK;
    if (!d_out) return set_error(RG_ERR_ARG, "null argument");
    if (ostride < dim || (uintptr_t)d_out % 4) return set_error(RG_ERR_ARG, "output rows: stride smaller than dim, or not aligned to their elements");
    OnDevice on(device);
    if (on.st != RG_OK) return on.st;
    const uint64_t items = (uint64_t)n * ((dim + 7) / 8);
    hipLaunchKernelGGL(rg_q4_unpack_kernel, dim3((uint32_t)std::min<uint64_t>((items + 255) / 256, 256u * 32u)), dim3(256), 0, (hipStream_t)stream, d_codes, cstride, d_scales, d_mins, sstride, nb, dim,
                       group, d_ids, n, d_out, ostride);
    RG_HIP(hipGetLastError());
    return RG_OK;
}

rg_status rg_q4_score_dev(const uint8_t *d_codes, uint64_t cstride, const uint16_t *d_scales, const uint16_t *d_mins, uint64_t sstride,
                          uint32_t nb, uint32_t dim, uint32_t group, const void *d_queries, uint32_t nq, uint64_t qstride, int dtype,
                          float *d_out, uint64_t ostride, int device, void *stream) {
    rg_status st = check_form(d_codes, cstride, d_scales, d_mins, sstride, nb, dim, group);
    if (st != RG_OK) return st;
    if (!known_dtype(dtype)) return set_error(RG_ERR_ARG, "unknown dtype");
    if (nq > 0x7fffffffu) return set_error(RG_ERR_ARG, "4-bit base: at most 2^31 - 1 queries");
    if (nb == 0 || nq == 0) return RG_OK;
    if (!d_queries || !d_out) return set_error(RG_ERR_ARG, "null argument");
    if (qstride < dim || (uintptr_t)d_queries % elem_bytes(dtype)) return set_error(RG_ERR_ARG, "queries: stride smaller than dim, or not aligned to their elements");
    if (ostride < nb || (uintptr_t)d_out % 4) return set_error(RG_ERR_ARG, "scores: stride smaller than the number of rows, or not aligned to their elements");
    OnDevice on(device);
    if (on.st != RG_OK) return on.st;
    ScoreArgs A;
    A.codes = d_codes; A.scales = d_scales; A.mins = d_mins; A.queries = d_queries; A.out = d_out;
    A.cstride = cstride; A.sstride = sstride; A.qstride = qstride; A.ostride = ostride;
    A.nb = nb; A.nq = nq; A.dim = dim; A.groups = (dim + group - 1) / group; A.dtype = dtype;
    hipStream_t s = (hipStream_t)stream;
    return group == 32 ? launch_score_gs<0>(A, s) : group == 64 ? launch_score_gs<1>(A, s) : launch_score_gs<2>(A, s);
}

}  // extern "C"
