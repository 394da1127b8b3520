// rg_q4.hip -- a base in 4 bits with one scale (and minimum) per group of elements: packing, unpacking, exhaustive scores.
//
//   y_ij = sum_k q_ik v_jk,   v_jk = s_jg (c_jk - 8)   or   s_jg c_jk + m_jg = s_jg (c_jk - 8) + (m_jg + 8 s_jg)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "rg.h"
#include "rg_internal.h"
#include "rg_rows.h"

namespace rg {
namespace {

constexpr uint32_t kMaxDim = 4096;

__device__ __forceinline__ float half_bits(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }

// one thread per group of a row.  The nearest level is decided exactly: x, minimum, scale and code have few enough bits that
// x - min - code * scale is exact in 64 bits, and its distance to half a scale decides (ties to the even code).
template <int DT>
__global__ void __launch_bounds__(256) rg_q4_pack_kernel(const void *rows, uint32_t nb, uint64_t stride, uint32_t dim, uint32_t group, uint8_t *codes, uint64_t cstride,
                                                         uint16_t *scales, uint16_t *mins, uint64_t sstride) {
    typedef typename Elem<DT>::T T;
    const uint32_t ng = (dim + group - 1) / group;
    for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < (uint64_t)nb * ng; at += (uint64_t)gridDim.x * 256) {
    const uint32_t j = (uint32_t)(at / ng), g = (uint32_t)(at % ng), k0 = g * group, n = min(group, dim - k0);
    const T *x = static_cast<const T *>(rows) + (size_t)j * stride + k0;
    float lo = INFINITY, hi = -INFINITY, top = 0.0f;
    for (uint32_t k = 0; k < n; ++k) { const float v = (float)x[k]; lo = fminf(lo, v); hi = fmaxf(hi, v); top = fmaxf(top, fabsf(v)); }
    const _Float16 s16 = (_Float16)(mins ? (hi - lo) * (1.0f / 15.0f) : top * (1.0f / 7.0f)), m16 = (_Float16)(mins ? lo : 0.0f);
    const double s = (double)(float)s16, m = (double)(float)m16;
    const int first = mins ? 0 : -8;
    scales[(size_t)j * sstride + g] = __builtin_bit_cast(uint16_t, s16);
    if (mins) mins[(size_t)j * sstride + g] = __builtin_bit_cast(uint16_t, m16);
    uint8_t *out = codes + (size_t)j * cstride + k0 / 2;
    for (uint32_t k = 0; k < n; k += 2) {
        uint32_t b = 0;
        for (uint32_t e = 0; e < 2; ++e) {
            if (k + e >= n) continue;
            int c = 0;
            if (s > 0) c = max(first, min(first + 15, (int)rint(((double)(float)x[k + e] - m) / s)));
            b |= (uint32_t)(c - first) << (4 * e);
        }
        out[k / 2] = (uint8_t)b;
    }
    if (g == ng - 1)
        for (uint32_t b = (dim + 1) / 2; b < (dim + 7) / 8 * 4; ++b) codes[(size_t)j * cstride + b] = 0;
    }
}

__global__ void __launch_bounds__(256) rg_q4_unpack_kernel(const uint8_t *codes, uint64_t cstride, const uint16_t *scales, const uint16_t *mins, uint64_t sstride, uint32_t nb, uint32_t dim,
                                                           uint32_t group, const uint32_t *ids, uint32_t n, float *out, uint64_t ostride) {
    for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < (uint64_t)n * dim; at += (uint64_t)gridDim.x * 256) {
    const uint32_t i = (uint32_t)(at / dim), k = (uint32_t)(at % dim), j = ids ? ids[i] : i;
    float v = NAN;                              // no such row
    if (j < nb) {
        const uint32_t c = codes[(size_t)j * cstride + k / 2] >> (4 * (k & 1)) & 15u, g = k / group;
        const float s = half_bits(scales[(size_t)j * sstride + g]);
        v = mins ? (float)c * s + half_bits(mins[(size_t)j * sstride + g]) : (float)((int)c - 8) * s;
    }
    out[(size_t)i * ostride + k] = v;
    }
}

// ---------------------------------------------------------------- scores
//
// Bound by reading the codes; the arithmetic has to stay out of the way.  Rows are the A operand of v_mfma_f32_16x16x32_f16 (16 rows x 32
// elements), queries its B operand: column n < 8 holds the upper half of query n, column n + 8 the lower (x = 2^e (hi + lo), 22 bits relative
// to the query's largest element), so eight fp32 queries cost what one costs.
//
//   a code becomes s (c - 8) in fp16 exactly, as two halves: s has 11 bits and c - 8 four, hi = fl(s (c - 8)), lo = s (c - 8) - hi, and no multiple
//   of 2^-24 is lost; products and sums are the matrix core's, in fp32, over the whole row -- no scale is applied to partial sums
//   minima: s c + m = s (c - 8) + (m + 8 s), and sum_k (m + 8 s) x_k over 32 elements is one slot of one more product per 128 elements
//
// A wave takes 32 rows at a time; lane (n, g) reads 16 bytes = 32 codes of row n, chunk 4 j + g of the row, with their scale.  (A row's last chunk is
// moved back to end with the row; what the chunk before it holds already meets zeros in the query.)  DEPTH such steps are on their way
// while one is multiplied.  The dword's codes come out in the order 0 4 1 5 2 6 3 7, and the queries lie in LDS in that order.
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct ScoreArgs {
    const uint8_t *codes;
    const uint16_t *scales, *mins;
    const void *queries;
    float *out;
    uint64_t cstride, sstride, qstride, ostride;
    uint32_t nb, nq, dim, chunk_shift, groups;          // chunks of 32 elements, 2^chunk_shift to a group
};

constexpr int kScoreThreads = 512, kScoreRows = 32, kScoreDepth = 4;

__device__ __forceinline__ void dequant(uint32_t w, half2 s, half8 &hi, half8 &lo) {
    const uint32_t w8 = w >> 8;
    const half2 c8 = {-1032.0f, -1032.0f}, sixteenth = {0.0625f, 0.0625f}, c72 = {-72.0f, -72.0f};
    half2 v[4];
    v[0] = __builtin_bit_cast(half2, (w & 0x000f000fu) | 0x64006400u) + c8;                                          // 1024 + c
    v[1] = __builtin_elementwise_fma(__builtin_bit_cast(half2, (w & 0x00f000f0u) | 0x64006400u), sixteenth, c72);     // 1024 + 16 c
    v[2] = __builtin_bit_cast(half2, (w8 & 0x000f000fu) | 0x64006400u) + c8;
    v[3] = __builtin_elementwise_fma(__builtin_bit_cast(half2, (w8 & 0x00f000f0u) | 0x64006400u), sixteenth, c72);
    half2 h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = v[i] * s;
        l[i] = __builtin_elementwise_fma(v[i], s, -h[i]);
    }
    hi = __builtin_bit_cast(half8, h);
    lo = __builtin_bit_cast(half8, l);
}

// element i of the B operand's eight holds element order(i) of the dword
__device__ __forceinline__ constexpr int code_order(int i) { return i % 2 * 4 + i / 2; }

// NQB blocks of eight queries at a time
template <int DT, int NQB, bool MINS>
__global__ void __launch_bounds__(kScoreThreads) rg_q4_score_kernel(ScoreArgs A) {
    typedef typename Elem<DT>::T T;
    extern __shared__ char lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
    const uint32_t dim = A.dim, D = (dim + 7) / 8, chunks = (D + 3) / 4, steps = (chunks + 3) / 4;       // dwords, chunks, steps of four chunks of a row
    half8 *X = reinterpret_cast<half8 *>(lds);                                        // [block][step][t][lane]
    uint32_t *XG = reinterpret_cast<uint32_t *>(lds + (size_t)NQB * steps * 4096);    // [block][step][lane]: the chunk's sum, twice
    float *factor = reinterpret_cast<float *>(XG + (MINS ? NQB * steps * 64 : 0));    // [query]

    struct Stage {
        u32x4 c[2];
        uint32_t s[2], m[2];
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
        const uint32_t q = 4 * pstep + g, group2 = min(q >> A.chunk_shift, A.groups - 1) * 2;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (D >= 4) {
                typedef u32x4 u32x4_dw __attribute__((aligned(4)));
                st.c[r] = *reinterpret_cast<const u32x4_dw *>(codes + (code_at[r] + min(16 * q, 4 * D - 16)));
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

    for (uint32_t q0 = 0; q0 < A.nq; q0 += 8 * NQB) {
        // queries: the largest element of each, then halves in operand order (zeros behind dim and behind the last query)
        for (uint32_t q = wave; q < 8 * NQB; q += waves) {
            uint32_t m = 0;
            if (q0 + q < A.nq)
                for (uint32_t k = lane; k < dim; k += 64) m = max(m, __float_as_uint((float)static_cast<const T *>(A.queries)[(size_t)(q0 + q) * A.qstride + k]) & 0x7fffffffu);
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
            if (lane == 0) factor[q] = __uint_as_float(m);
        }
        __syncthreads();
        auto element = [&](uint32_t q, uint32_t k, float top, float down) {      // a query's element, scaled; of one that is not finite the signs of its infinities
            if (q0 + q >= A.nq || k >= dim) return 0.0f;
            const float v = (float)static_cast<const T *>(A.queries)[(size_t)(q0 + q) * A.qstride + k];
            if (top < INFINITY) return v * down;
            return fabsf(v) < INFINITY ? 0.0f : fabsf(v) == INFINITY ? copysignf(1.0f, v) : v;
        };
        for (uint32_t i = tid; i < NQB * steps * 4 * 4 * 8; i += kScoreThreads) {
            const uint32_t q = i % 8, gg = i / 8 % 4, t = i / 32 % 4, j = i / 128 % steps, qb = i / 128 / steps;
            const float top = factor[qb * 8 + q], down = pow2(-row_exponent(top));
            const uint32_t c = 4 * j + gg, d = D >= 4 ? min(4 * c, D - 4) + t : t;
            half8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = d >= 4 * c && d < D ? element(qb * 8 + q, 8 * d + code_order(e), top, down) : 0.0f;
                hi[e] = (_Float16)v;
                lo[e] = (_Float16)(v - (float)hi[e]);
            }
            half8 *at = X + ((size_t)(qb * steps + j) * 4 + t) * 64 + gg * 16 + q;
            at[0] = hi;
            at[8] = lo;
        }
        if (MINS)
            for (uint32_t i = tid; i < NQB * steps * 4 * 8; i += kScoreThreads) {
                const uint32_t q = i % 8, gg = i / 8 % 4, j = i / 32 % steps, qb = i / 32 / steps;
                const float top = factor[qb * 8 + q], down = pow2(-row_exponent(top));
                float v = 0.0f;
                for (uint32_t k = 32 * (4 * j + gg); k < min(32 * (4 * j + gg) + 32, dim); ++k) v += element(qb * 8 + q, k, top, down);
                const _Float16 h = (_Float16)v, l = (_Float16)(v - (float)h);
                uint32_t *at = XG + (qb * steps + j) * 64 + gg * 16 + q;
                at[0] = 0x10001u * __builtin_bit_cast(uint16_t, h);
                at[8] = 0x10001u * __builtin_bit_cast(uint16_t, l);
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
                const Stage st = ring[d];
                fetch(ring[d]);
                half2 s[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) s[r] = __builtin_bit_cast(half2, st.s[r] * 0x10001u);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    half8 x[NQB];
#pragma unroll
                    for (int b = 0; b < NQB; ++b) x[b] = X[((size_t)(b * steps + step) * 4 + t) * 64 + lane];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        half8 hi, lo;
                        dequant(st.c[r][t], s[r], hi, lo);
#pragma unroll
                        for (int b = 0; b < NQB; ++b) {
                            acc[r][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, x[b], acc[r][b], 0, 0, 0);
                            acc[r][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, x[b], acc[r][b], 0, 0, 0);
                        }
                    }
                }
                if (MINS) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float off = fmaf(half_bits((uint16_t)st.s[r]), 8.0f, half_bits((uint16_t)st.m[r]));
                        half8 o = {0, 0, 0, 0, 0, 0, 0, 0};
                        o[0] = (_Float16)off;
                        o[1] = (_Float16)(off - (float)o[0]);
#pragma unroll
                        for (int b = 0; b < NQB; ++b) {
                            const u32x4 v = {XG[(b * steps + step) * 64 + lane], 0, 0, 0};
                            acc[r][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(o, __builtin_bit_cast(half8, v), acc[r][b], 0, 0, 0);
                        }
                    }
                }
                if (++step == steps) {
                    step = 0;
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int b = 0; b < NQB; ++b) {
                            f32x4 v = acc[r][b];
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[i] += __shfl_xor(v[i], 8);
                            const uint32_t q = q0 + b * 8 + n, row = tile * kScoreRows + 16 * r + 4 * g;
                            if (n < 8 && q < A.nq && row < A.nb) {
                                const float top = factor[b * 8 + n], up = row_factor(top, row_exponent(top));
                                float *to = A.out + q * A.ostride + row;
                                if (row + 4 <= A.nb) {
                                    typedef f32x4 f32x4_dw __attribute__((aligned(4)));
                                    *reinterpret_cast<f32x4_dw *>(to) = v * up;
                                } else {
#pragma unroll
                                    for (int i = 0; i < 4; ++i)
                                        if (row + i < A.nb) to[i] = v[i] * up;
                                }
                            }
                            acc[r][b] = f32x4{0, 0, 0, 0};
                        }
                    tile += stride;
                }
            }
        }
        __syncthreads();
    }
}

size_t score_lds(uint32_t dim, int nqb, bool mins) {
    const size_t steps = (((dim + 7) / 8 + 3) / 4 + 3) / 4;
    return nqb * steps * (4096 + (mins ? 256 : 0)) + nqb * 32;
}

template <int DT, int NQB>
rg_status launch_score(const ScoreArgs &A, hipStream_t s) {
    auto kern = A.mins ? rg_q4_score_kernel<DT, NQB, true> : rg_q4_score_kernel<DT, NQB, false>;
    const size_t lds = score_lds(A.dim, NQB, A.mins != nullptr);
    RG_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    const uint32_t tiles = (A.nb + kScoreRows - 1) / kScoreRows, per_cu = std::max<uint32_t>(1, std::min<uint32_t>(2, (uint32_t)(160 * 1024 / lds)));
    hipLaunchKernelGGL(kern, dim3(std::min(tiles, 256u * per_cu)), dim3(kScoreThreads), lds, s, A);
    RG_HIP(hipGetLastError());
    return RG_OK;
}
template <int DT>
rg_status launch_score_dt(const ScoreArgs &A, hipStream_t s) {
    // as many queries per reading of the base as there are, and as LDS holds
    const bool mins = A.mins != nullptr;
    if (A.nq > 16 && score_lds(A.dim, 4, mins) <= 160 * 1024) return launch_score<DT, 4>(A, s);
    if (A.nq > 8 && score_lds(A.dim, 2, mins) <= 160 * 1024) return launch_score<DT, 2>(A, s);
    return launch_score<DT, 1>(A, s);
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
    const uint64_t n = (uint64_t)nb * ((dim + group - 1) / group);
    auto kern = dtype == RG_DTYPE_F32 ? rg_q4_pack_kernel<RG_DTYPE_F32> : dtype == RG_DTYPE_F16 ? rg_q4_pack_kernel<RG_DTYPE_F16> : rg_q4_pack_kernel<RG_DTYPE_BF16>;
    hipLaunchKernelGGL(kern, dim3((uint32_t)std::min<uint64_t>((n + 255) / 256, 1u << 20)), dim3(256), 0, (hipStream_t)stream, d_rows, nb, stride, dim, group, d_codes, cstride, d_scales, d_mins, sstride);
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
    hipLaunchKernelGGL(rg_q4_unpack_kernel, dim3((uint32_t)std::min<uint64_t>(((uint64_t)n * dim + 255) / 256, 1u << 20)), dim3(256), 0, (hipStream_t)stream, d_codes, cstride, d_scales, d_mins, sstride, nb, dim, group, d_ids,
                       n, d_out, ostride);
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
    A.nb = nb; A.nq = nq; A.dim = dim; A.chunk_shift = group == 32 ? 0 : group == 64 ? 1 : 2; A.groups = (dim + group - 1) / group;
    hipStream_t s = (hipStream_t)stream;
    return dtype == RG_DTYPE_F32 ? launch_score_dt<RG_DTYPE_F32>(A, s) : dtype == RG_DTYPE_F16 ? launch_score_dt<RG_DTYPE_F16>(A, s) : launch_score_dt<RG_DTYPE_BF16>(A, s);
}

}  // extern "C"
