// rg_softmax_pass.h -- the pass of the softmax operators (rg_softmax.hip): stationary rows x against streamed rows y.
//
// A wave owns NX blocks of 16 rows x (or a part of their dimensions), held in registers as MFMA operands for the whole pass; its workgroup streams rows y
// through LDS, 32 at a time.  Per tile and wave:
//
//   S^T[y][x] = Y X^T       v_mfma_f32_16x16x32: A = 16 rows y (ds_read_b128), B = 16 rows x (registers)
//   P = 2^(S k + bias - M)  in the accumulator's layout: a lane holds 4 + 4 weights of ONE row x
//   O^T[d][x] += Y^T P^T    A = 16 dims x 32 rows y of the same LDS tile (ds_read_b64_tr_b16 transposes on the way), B = the weights as they
//                           lie: slot (g, e) of the 32-deep product is row y = 16 (e / 4) + 4 g + e % 4, for both operands
//
// so a tile is read from memory once for both products and no weight crosses lanes.  fp32 rows are split into two fp16 halves, each row
// scaled by its own power of two to the top of fp16's range: x = 2^e (hi + lo), 22 bits; a product is hi hi + hi lo + lo hi (what is left out is 2^-22 of it).
// Weights are rounded to the 16-bit type they are multiplied in -- bf16 as such, fp16 with 2^7 .. 2^15 at the top of its range, fp32 rows
// as two halves again; sums of weights are taken before that rounding, and every accumulation is fp32.  What O is divided by is the sum of the
// weights as they were multiplied: divided by the others' sum, the mean is off by up to half a step of itself, which shows where a query's
// gradient is the small difference of mean and target (bf16, rows 0.1 beside the target: 0.012 of the gradient's norm, now 0.0017).
//
// M is a reference, not the running maximum: it moves only when a weight would pass 2^15 (a branch no wave takes on most tiles), so sums
// are rescaled a few times per pass instead of once per tile.
//
// LDS: a row of a plane is KS * 64 bytes in 16-byte chunks, pitch a multiple of 256 bytes, chunk c of row y at slot c ^ swizzle(y) within its 256
// bytes.  The second product's reads touch 8 rows 32 bytes wide: those need distinct pairs of slots.  The first product's touch 16 rows at one
// chunk and are served 16 lanes at a time as lanes 0-3, 12-15, 20-23, 24-27 (and so on), that is rows 0-3, 12-15 at chunk c and rows 4-11 at
// chunk c + 1: rows r and r ^ 12 share a pair.  (With 2 (y % 8) + y / 8 instead every such read took twice its time: 34 % of the LDS cycles.)
#pragma once
#include <hip/hip_runtime.h>

#include "rg.h"
#include "rg_rows.h"

namespace rg {

enum { kStats = 0, kMean = 1, kRows = 2 };

struct PassArgs {
    const void *x, *y;                 // stationary and streamed rows (wide: y as 16-bit planes)
    uint64_t xstride, ystride;         // in elements
    uint32_t nx, ny, dim, ydim;        // ydim: what of a row of y may be read
    float k;                           // scale * log2 e
    uint32_t nsplit, rows_per_split;   // of y
    uint32_t opitch;                   // floats of a row of o
    uint32_t resume;                   // the slots hold what earlier pieces of y left
    float4 *ml;                        // [slot][nx] reference and sum of the weights, reference of O, what O is divided by under the first (kMean, kStats; kRows in pieces: the third)
    float *o;                          // [slot][nx][opitch] (kMean, kRows in pieces)
    const uint32_t *targets;           // kStats, kMean: per x (global ids)
    uint32_t id_base;
    float *own2;                       // kStats, kMean: z2 of the target, written where it is met
    const float *yinfo;                // fp32 rows and kRows, per 32 rows y: 32 factors and biases of a logit, signs of the weight, target rows (bits)
    const float *ytarget;              // kRows, per y: the biased logit of its own row, log2(|w| (1 - p_target))
    void *out;                         // kRows in one piece: the gradient itself
    uint64_t ostride;
    float oscale;
};

// an instantiation: rows x of a workgroup, blocks of 16 output dims, bytes of LDS, waves per SIMD, threads (rg_softmax_inst_*.hip)
struct SoftmaxKernel {
    const void *kern;
    uint32_t xt, ob, lds, wps, threads;
};
#define RG_SOFTMAX_KERNELS(DT)                    \
    SoftmaxKernel softmax_thin_##DT##_stats(int ks); \
    SoftmaxKernel softmax_thin_##DT##_mean(int ks);  \
    SoftmaxKernel softmax_wide_##DT##_stats(int ks); \
    SoftmaxKernel softmax_wide_##DT##_mean(int ks);  \
    SoftmaxKernel softmax_wide_##DT##_rows(int ks);
RG_SOFTMAX_KERNELS(f32)
RG_SOFTMAX_KERNELS(f16)
RG_SOFTMAX_KERNELS(bf16)
#undef RG_SOFTMAX_KERNELS

constexpr uint32_t kNoTarget = 0xffffffffu;
constexpr float kNothing = -3.0e38f;   // M before the first row (an infinity would make NaN of a logit of -inf)

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The sums of a product over the dimensions are made in this many parts, whichever kernel and waves make them: the logits
// of all modes have the same bits.
constexpr int softmax_parts(int dt, int ks) { return dt == RG_DTYPE_F32 ? (ks <= 8 ? 1 : ks <= 16 ? 2 : 4) : ks <= 16 ? 1 : 4; }

template <int DT> struct Frag { typedef half8 V; };
template <> struct Frag<RG_DTYPE_BF16> { typedef bf8 V; };

__device__ __forceinline__ f32x4 mma(half8 a, half8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(bf8 a, bf8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ uint32_t swizzle(uint32_t y) { return (((y & 7) ^ (y >> 1 & 4)) << 1) | (y >> 3 & 1); }

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// 8 elements of a row from element k on (zeros from dim on, or where nothing is to be taken): as they are for 16-bit types, as floats for
// fp32.  Rows need no other alignment than their elements': the memory units take wide accesses at any address.  A chunk that ends behind
// the row is the row's last 8 elements, moved down (its single elements took up to 7 loads more: loss of 20 bf16 queries on 1M x 301 238 us, now 145 us).
// SMALL: rows may be shorter than that.
template <int DT> struct Chunk { u32x4 v; };
template <> struct Chunk<RG_DTYPE_F32> { f32x4 a, b; };
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef f32x4 f32x4_a4 __attribute__((aligned(4)));

template <int DT, bool SMALL>
__device__ __forceinline__ Chunk<DT> fetch_chunk(const void *row, uint32_t k, uint32_t dim, bool take) {
    Chunk<DT> c;
    take &= k < dim;
    const uint32_t at = min(k, dim - 8);
    if constexpr (DT == RG_DTYPE_F32) {
        const float *p = static_cast<const float *>(row);
        c.a = c.b = f32x4{0, 0, 0, 0};
        if (!SMALL || dim >= 8) {
            if (take) {
                c.a = *reinterpret_cast<const f32x4_a4 *>(p + at);
                c.b = *reinterpret_cast<const f32x4_a4 *>(p + at + 4);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (take && k + i < dim) c.a[i] = p[k + i];
                if (take && k + 4 + i < dim) c.b[i] = p[k + 4 + i];
            }
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(row);
        c.v = u32x4{0, 0, 0, 0};
        if (!SMALL || dim >= 8) {
            if (take) c.v = *reinterpret_cast<const u32x4_a2 *>(p + at);
        } else {
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (take && k + i < dim) c.v[i / 2] |= (uint32_t)p[k + i] << (16 * (i % 2));
        }
    }
    return c;
}
// ... moved down, where it is used, and only where rows are ragged -- asked once for all chunks that are on their way: whoever moves one waits for it
template <bool SMALL> __device__ __forceinline__ bool ragged(uint32_t dim) { return dim % 8 != 0 && (!SMALL || dim > 8); }
template <int DT>
__device__ __forceinline__ Chunk<DT> settle(Chunk<DT> c, uint32_t k, uint32_t dim) {
    const uint32_t s = k < dim ? k - min(k, dim - 8) : 0;
    if constexpr (DT == RG_DTYPE_F32) {
        if (s & 4) { c.a = c.b; c.b = f32x4{0, 0, 0, 0}; }
        if (s & 2) { c.a = f32x4{c.a[2], c.a[3], c.b[0], c.b[1]}; c.b = f32x4{c.b[2], c.b[3], 0, 0}; }
        if (s & 1) { c.a = f32x4{c.a[1], c.a[2], c.a[3], c.b[0]}; c.b = f32x4{c.b[1], c.b[2], c.b[3], 0}; }
    } else {
        if (s & 4) c.v = u32x4{c.v[2], c.v[3], 0, 0};
        if (s & 2) c.v = u32x4{c.v[1], c.v[2], c.v[3], 0};
        if (s & 1) c.v = u32x4{c.v[0] >> 16 | c.v[1] << 16, c.v[1] >> 16 | c.v[2] << 16, c.v[2] >> 16 | c.v[3] << 16, c.v[3] >> 16};
    }
    return c;
}
// a lane's N chunks of a row, from element k on and `apart` elements from each other
template <int DT, bool SMALL, int N>
__device__ __forceinline__ void load_chunks(Chunk<DT> (&c)[N], const void *row, uint32_t k, uint32_t apart, uint32_t dim, bool take) {
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = fetch_chunk<DT, SMALL>(row, k + i * apart, dim, take);
    if (ragged<SMALL>(dim))
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = settle<DT>(c[i], k + i * apart, dim);
}

// the largest absolute value of a chunk; NaN counts as infinity
__device__ __forceinline__ float absmax(const Chunk<RG_DTYPE_F32> &c) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(max(m, __float_as_uint(c.a[i]) & 0x7fffffffu), __float_as_uint(c.b[i]) & 0x7fffffffu);
    return __uint_as_float(m);
}
__device__ __forceinline__ void split8(Chunk<RG_DTYPE_F32> c, float top, float s, half8 &hi, half8 &lo) {
    if (!(top < INFINITY)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float v = i < 4 ? c.a[i % 4] : c.b[i % 4];
            v = fabsf(v) < INFINITY ? 0.0f : fabsf(v) == INFINITY ? copysignf(1.0f, v) : v;
            if (i < 4) c.a[i % 4] = v;
            else c.b[i % 4] = v;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = (i < 4 ? c.a[i % 4] : c.b[i % 4]) * s;
        const _Float16 h = (_Float16)v;
        hi[i] = h;
        lo[i] = (_Float16)(v - (float)h);
    }
}

// the bias of a streamed fp32 row's logits in kMean, its scale.  Of a row that is not finite the second product would take the signs: with logits of -inf,
// which leave the loss alone, its weight is 0, and 0 times infinity is no number.
__device__ __forceinline__ float row_bias(float top, int e) { return top < INFINITY ? (float)e : NAN; }

// stationary operands of row x: lane (n, g) holds elements 32 ks + 8 g .. + 7 of part kq of KQ of the row; returns what its logits are
// multiplied by
template <int DT, int KS, int KQ, int NP>
__device__ __forceinline__ float load_stationary(const PassArgs &A, uint32_t x, uint32_t g, typename Frag<DT>::V (&X)[KS][NP], uint32_t kq = 0) {
    const char *row = static_cast<const char *>(A.x) + (size_t)x * A.xstride * sizeof(typename Elem<DT>::T);
    constexpr bool SMALL = KS * KQ <= 2;
    const bool take = x < A.nx;
    const uint32_t k0 = 32 * KS * kq + 8 * g;
    if constexpr (DT == RG_DTYPE_F32) {
        // the largest element of the row, all its parts (where chunks end behind the row, elements that count anyway), then this part -- at once where
        // it is all of it, else once more from the caches: it would not fit with the registers of a wide row's part
        uint32_t m = 0;
        Chunk<DT> c[KQ == 1 ? KS : 1];
        if (KQ == 1) {
            load_chunks<DT, SMALL>(c, row, k0, 32, A.dim, take);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) m = max(m, __float_as_uint(absmax(c[KQ == 1 ? ks : 0])));
        } else {
#pragma unroll 4
            for (uint32_t ks = 0; ks < KS * KQ; ++ks) m = max(m, __float_as_uint(absmax(fetch_chunk<DT, SMALL>(row, 32 * ks + 8 * g, A.dim, take))));
        }
        m = max(m, (uint32_t)__shfl_xor((int)m, 16));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32));
        const float top = __uint_as_float(m);
        const int e = row_exponent(top);
        if constexpr (KQ == 1) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) split8(c[KQ == 1 ? ks : 0], top, pow2(-e), X[ks][0], X[ks][1]);
        } else {
            constexpr int G = KS % 4 == 0 ? 4 : KS % 3 == 0 ? 3 : 2;      // chunks on their way
            static_assert(KS % G == 0, "parts are whole groups");
#pragma unroll
            for (int ks = 0; ks < KS; ks += G) {
                Chunk<DT> d[G];
                load_chunks<DT, SMALL>(d, row, k0 + 32 * ks, 32, A.dim, take);
#pragma unroll
                for (int i = 0; i < G; ++i) split8(d[i], top, pow2(-e), X[ks + i][0], X[ks + i][1]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        return A.k * row_factor(top, e);
    } else {
        Chunk<DT> c[KS];
        load_chunks<DT, SMALL>(c, row, k0, 32, A.dim, take);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) X[ks][0] = __builtin_bit_cast(typename Frag<DT>::V, c[ks].v);
        return A.k;
    }
}

// the sum of a lane's weights as they are multiplied (16-bit subnormals count)
__device__ __forceinline__ float sum_of(half8 w) {
    typedef _Float16 half2 __attribute__((ext_vector_type(2)));
    const half2 one{(_Float16)1.0f, (_Float16)1.0f};
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_fdot2(half2{w[2 * e], w[2 * e + 1]}, one, s, false);
    return s;
}
__device__ __forceinline__ float sum_of(bf8 w) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    const bf2 one{(__bf16)1.0f, (__bf16)1.0f};
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_fdot2_f32_bf16(bf2{w[2 * e], w[2 * e + 1]}, one, s, false);
    return s;
}
// kMean, 16-bit rows: such a sum is kept beside l (fp32 rows' weights are 22 bits of themselves, and l serves)
constexpr bool softmax_sums_rounded(int dt, int mode) { return mode == kMean && dt != RG_DTYPE_F32; }

// what an earlier piece left in a wave's slot
template <int DT, int MODE, int OB, int NX, int NO>
__device__ __forceinline__ void take_up(const PassArgs &A, uint32_t x0, uint32_t n, uint32_t g, uint32_t kq, uint32_t split, float (&M)[NX], float (&Ml)[NX], float (&l)[NX], float (&R)[NX], f32x4 (&O)[NO][NX]) {
#pragma unroll
    for (int j = 0; j < NX; ++j) {
        const uint32_t x = x0 + j * 16 + n;
        if (x >= A.nx) continue;
        const size_t at = (size_t)split * A.nx + x;
        const float4 v = A.ml[at];
        Ml[j] = v.x;
        M[j] = v.z;
        l[j] = g == 0 ? v.y : 0.0f;                  // (finish adds the four up)
        if (softmax_sums_rounded(DT, MODE)) R[j] = g == 0 ? v.w : 0.0f;
        if constexpr (MODE != kStats)
#pragma unroll
            for (int ob = 0; ob < OB; ++ob) {
                const uint32_t d = (kq * OB + ob) * 16 + 4 * g;
                if (d < A.dim) O[ob][j] = *reinterpret_cast<const f32x4 *>(A.o + at * A.opitch + d);
            }
    }
}

// what a wave (with part kq of the output blocks) leaves behind: references and sums, and the sums of rows (partial results, or the gradient itself)
template <int DT, int MODE, int OB, int NX, int NO>
__device__ __forceinline__ void finish(const PassArgs &A, uint32_t x0, uint32_t n, uint32_t g, uint32_t kq, uint32_t split, const float (&M)[NX], const float (&Ml)[NX], const float (&l)[NX],
                                       const float (&R)[NX], const f32x4 (&O)[NO][NX]) {
    typedef typename Elem<DT>::T T;
#pragma unroll
    for (int j = 0; j < NX; ++j) {
        const uint32_t x = x0 + j * 16 + n;
        float s = l[j];
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        float r = s;
        if (softmax_sums_rounded(DT, MODE)) {
            r = R[j];
            r += __shfl_xor(r, 16);
            r += __shfl_xor(r, 32);
        }
        if (x >= A.nx) continue;
        const size_t at = (size_t)split * A.nx + x;
        const bool direct = MODE == kRows && A.nsplit == 1;
        if (!direct && g == 0 && kq == 0) A.ml[at] = make_float4(Ml[j], s, M[j], r);
        if constexpr (MODE != kStats) {
            const float f = direct ? exp2_hw(0.5f * M[j]) : 1.0f;      // 2^M in two steps: it may lie below the normal range
#pragma unroll
            for (int ob = 0; ob < OB; ++ob) {
                const uint32_t d = (kq * OB + ob) * 16 + 4 * g;
                if (d >= A.dim) continue;
                if (!direct) {
                    *reinterpret_cast<f32x4 *>(A.o + at * A.opitch + d) = O[ob][j];
                } else {
                    T *out = static_cast<T *>(A.out) + (size_t)x * A.ostride + d;
                    typedef T T4 __attribute__((ext_vector_type(4)));
                    typedef T4 T4_any __attribute__((aligned(sizeof(T))));
                    T4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = (T)(O[ob][j][i] * f * (f * A.oscale));
                    if (d + 4 <= A.dim) {
                        *reinterpret_cast<T4_any *>(out) = v;
                    } else {
#pragma unroll
                        for (int i = 0; i < 3; ++i)
                            if (d + i < A.dim) out[i] = v[i];
                    }
                }
            }
        }
    }
}

// workgroups are handed out to the eight XCDs in turn: give each XCD (an L2 of its own) a stretch of neighbouring work instead, so that
// what neighbours stream is fetched once per XCD
__device__ __forceinline__ uint32_t xcd_block(uint32_t b, uint32_t total) {
    const uint32_t per = total / 8, extra = total % 8, xcd = b % 8;
    return xcd * per + min(xcd, extra) + b / 8;
}

}  // namespace rg
