// rg_softmax_pass.h -- the pass of the softmax operators (rg_softmax.hip) on the matrix cores.
//
// A workgroup of four waves owns 64 * NX stationary rows x (NX blocks of 16 per wave, held in registers as MFMA operands for the whole
// pass) and streams rows y through LDS, 32 at a time.  Per tile and wave:
//
//   S^T[y][x] = Y X^T       v_mfma_f32_16x16x32: A = 16 rows y (ds_read_b128), B = 16 rows x (registers)
//   P = 2^(S k + bias - M)  in the accumulator's layout: a lane holds 4 + 4 weights of ONE row x
//   O^T[d][x] += Y^T P^T    A = 16 dims x 32 rows y of the same LDS tile (ds_read_b64_tr_b16 transposes on the way), B = the weights as they
//                           lie: slot (g, e) of the 32-deep product is row y = 16 (e / 4) + 4 g + e % 4, for both operands
//
// so a tile is read from memory once for both products and no weight crosses lanes.  fp32 rows are split into two fp16 halves, each row
// scaled by its own power of two to [1, 2): x = 2^e (hi + lo), 22 bits; a product is hi hi + hi lo + lo hi.
//
// M is a reference, not the running maximum: it moves only when a weight would pass 2^15 (a branch no wave takes on most tiles), so sums
// are rescaled a few times per pass instead of once per tile.
//
// LDS: a row of a plane is KS * 64 bytes in 16-byte chunks, pitch a multiple of 256 bytes, chunk c of row y at slot
// c ^ (2 (y % 8) + y / 8 % 2) within its 256 bytes: 16 rows read at one chunk (first product) and 8 rows read 32 bytes wide (second)
// both touch every bank once.
#pragma once
#include <hip/hip_runtime.h>

#include "rg.h"
#include "rg_rows.h"

namespace rg {

enum { kStats = 0, kMean = 1, kRows = 2 };

struct PassArgs {
    const void *x, *y;                 // stationary and streamed rows
    uint64_t xstride, ystride;
    uint32_t nx, ny, dim;
    float k;                           // scale * log2 e
    uint32_t nsplit, rows_per_split;   // of y
    uint32_t nslices;                  // of the dimensions of O
    uint32_t opitch;                   // floats of a row of o
    float4 *ml;                        // [slot][nx] reference and sum of the weights, reference of O, -- (kMean, kStats; kRows in pieces: the third)
    float *o;                          // [slot][nx][opitch] (kMean, kRows in pieces)
    const uint32_t *targets;           // kStats, kMean: per x (global ids)
    uint32_t id_base;
    float *own2;                       // kStats, kMean: z2 of the target, written where it is met
    const float4 *yparam;              // kRows, per y: bias, log2(|w| (1 - p_target)), sign, target row of the shard (bits)
    void *out;                         // kRows in one piece: the gradient itself
    uint64_t ostride;
    float oscale;
};

constexpr uint32_t kNoTarget = 0xffffffffu;
constexpr float kNothing = -3.0e38f;   // M before the first row (an infinity would make NaN of a logit of -inf)

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// the kernel of a type, mode and number of 32-element steps (rg_softmax_inst_*.hip)
#define RG_SOFTMAX_KERNELS(DT)                   \
    const void *softmax_kernel_##DT##_stats(int ks); \
    const void *softmax_kernel_##DT##_mean(int ks);  \
    const void *softmax_kernel_##DT##_rows(int ks);
RG_SOFTMAX_KERNELS(f32)
RG_SOFTMAX_KERNELS(f16)
RG_SOFTMAX_KERNELS(bf16)
#undef RG_SOFTMAX_KERNELS

// what an instantiation holds: NX blocks of x per wave, OB blocks of 16 output dims per slice, waves per SIMD
template <int DT, int KS>
struct PassCfg {
    static constexpr int NP = DT == RG_DTYPE_F32 ? 2 : 1;
    static constexpr int NX = DT == RG_DTYPE_F32 ? (KS <= 8 ? 2 : 1) : (KS <= 4 ? 4 : KS <= 16 ? 2 : 1);
    static constexpr int OB = KS == 7 ? 13 : (DT == RG_DTYPE_F32 && KS == 32) ? 32 : 2 * KS;
    static constexpr int XT = 64 * NX;
    static constexpr int TY = 32;
    static constexpr int PITCH = (KS * 64 + 255) / 256 * 256;
    static constexpr int PLANE = TY * PITCH;
    static constexpr int BUF = NP * PLANE;
    static constexpr int NBUF = 2 * BUF <= 128 * 1024 ? 2 : 1;
    static constexpr int YV = TY * 4 * 4;                       // per buffer: factor, bias, sign, target of the rows
    static constexpr int LDS = NBUF * (BUF + YV);
    static constexpr int WPS = (DT == RG_DTYPE_F32 ? KS <= 4 : KS <= 8) ? 2 : 1;
};

template <int DT> struct Frag { typedef half8 V; };
template <> struct Frag<RG_DTYPE_BF16> { typedef bf8 V; };

__device__ __forceinline__ f32x4 mma(half8 a, half8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(bf8 a, bf8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// 8 elements of a row from element k on (zeros from dim on): as they are for 16-bit types, as floats for fp32
template <int DT> struct Chunk { u32x4 v; };
template <> struct Chunk<RG_DTYPE_F32> { f32x4 a, b; };

template <int DT>
__device__ __forceinline__ Chunk<DT> load_chunk(const void *row, uint32_t k, uint32_t dim, bool vec) {
    const uint16_t *p = static_cast<const uint16_t *>(row) + k;
    Chunk<DT> c;
    c.v = u32x4{0, 0, 0, 0};
    if (k + 8 <= dim && vec) {
        c.v = *reinterpret_cast<const u32x4 *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < dim) c.v[i / 2] |= (uint32_t)p[i] << (16 * (i % 2));
    }
    return c;
}
template <>
__device__ __forceinline__ Chunk<RG_DTYPE_F32> load_chunk<RG_DTYPE_F32>(const void *row, uint32_t k, uint32_t dim, bool vec) {
    const float *p = static_cast<const float *>(row) + k;
    Chunk<RG_DTYPE_F32> c;
    c.a = c.b = f32x4{0, 0, 0, 0};
    if (k + 8 <= dim && vec) {
        c.a = *reinterpret_cast<const f32x4 *>(p);
        c.b = *reinterpret_cast<const f32x4 *>(p + 4);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (k + i < dim) c.a[i] = p[i];
            if (k + 4 + i < dim) c.b[i] = p[4 + i];
        }
    }
    return c;
}

// the largest absolute value of a chunk; NaN counts as infinity
__device__ __forceinline__ float absmax(const Chunk<RG_DTYPE_F32> &c) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(max(m, __float_as_uint(c.a[i]) & 0x7fffffffu), __float_as_uint(c.b[i]) & 0x7fffffffu);
    return __uint_as_float(m);
}
// exponent e of a row's largest value: 2^-e brings the row to [1, 2)
__device__ __forceinline__ int row_exponent(float top) {
    const uint32_t u = __float_as_uint(top) >> 23;
    return u >= 255 ? 0 : u ? (int)u - 127 : top == 0.0f ? 0 : -126;       // (subnormal rows: 2^126 is the largest factor)
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

// a row that is not finite keeps the signs of its infinities (and its NaN) and nothing else; its logits are multiplied by infinity
__device__ __forceinline__ float row_factor(float top, int e) { return top < INFINITY ? pow2(e) : INFINITY; }

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

template <int DT, int KS, int MODE>
__global__ void __launch_bounds__(256, (PassCfg<DT, KS>::WPS)) rg_softmax_pass_kernel(PassArgs A) {
    typedef PassCfg<DT, KS> C;
    typedef typename Elem<DT>::T T;
    typedef typename Frag<DT>::V V;
    constexpr int NP = C::NP, NX = C::NX, OB = C::OB, PITCH = C::PITCH, CI = (KS + 3) / 4;
    constexpr bool F32 = DT == RG_DTYPE_F32;
    constexpr float kTop = 15.0f, kStart = DT == RG_DTYPE_BF16 ? 0.0f : 7.0f;   // a weight is at most 2^15; the first largest one 2^0 / 2^7
    extern __shared__ char lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const uint32_t ntx = (A.nx + C::XT - 1) / C::XT;
    uint32_t b = blockIdx.x;
    const uint32_t xt = b % ntx;
    b /= ntx;
    const uint32_t slice = MODE == kStats ? 0 : b % A.nslices, split = MODE == kStats ? b : b / A.nslices;
    const uint32_t ybeg = min(A.ny, split * A.rows_per_split), yend = min(A.ny, ybeg + A.rows_per_split);
    const uint32_t x0 = xt * C::XT + wave * 16 * NX;
    const bool live = x0 < A.nx;                                // waves behind the last row only help to load
    const uint32_t dim = A.dim;
    const size_t esz = sizeof(T);
    const bool xvec = ((uintptr_t)A.x | A.xstride * esz) % 16 == 0, yvec = ((uintptr_t)A.y | A.ystride * esz) % 16 == 0;

    // stationary operands: lane (n, g) holds elements 32 ks + 8 g .. + 7 of row n of every block
    V X[NX][KS][NP];
    float kx[NX];
    uint32_t target[NX];
#pragma unroll
    for (int j = 0; j < NX; ++j) {
        const uint32_t x = x0 + j * 16 + n;
        const char *row = static_cast<const char *>(A.x) + (size_t)x * A.xstride * esz;
        kx[j] = A.k;
        if constexpr (F32) {
            float top = 0.0f;
            Chunk<DT> c[KS];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                c[ks] = load_chunk<DT>(row, 32 * ks + 8 * g, x < A.nx ? dim : 0, xvec);
                top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(absmax(c[ks]))));
            }
            top = __uint_as_float(max(__float_as_uint(top), (uint32_t)__shfl_xor((int)__float_as_uint(top), 16)));
            top = __uint_as_float(max(__float_as_uint(top), (uint32_t)__shfl_xor((int)__float_as_uint(top), 32)));
            const int e = row_exponent(top);
            const float s = pow2(-e);
            kx[j] *= row_factor(top, e);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) split8(c[ks], top, s, X[j][ks][0], X[j][ks][1]);
        } else {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) X[j][ks][0] = __builtin_bit_cast(V, load_chunk<DT>(row, 32 * ks + 8 * g, x < A.nx ? dim : 0, xvec).v);
        }
        target[j] = kNoTarget;
        if (MODE != kRows && x < A.nx) {
            const uint32_t t = A.targets[x];
            if (t != kNoTarget && t >= A.id_base && t - A.id_base >= ybeg && t - A.id_base < yend) target[j] = t - A.id_base;
        }
    }

    f32x4 O[MODE == kStats ? 1 : OB][NX];
    // M: reference of the weights of O; with fp32 rows those carry the rows' scales, so that the sum l has a reference Ml of its own
    constexpr bool TWO = F32 && MODE == kMean;
    float M[NX], l[NX], Ml[NX];
#pragma unroll
    for (int j = 0; j < NX; ++j) {
        M[j] = Ml[j] = kNothing;
        l[j] = 0.0f;
        if (MODE != kStats)
#pragma unroll
            for (int ob = 0; ob < OB; ++ob) O[ob][j] = f32x4{0, 0, 0, 0};
    }

    // streaming: 16 lanes per row, two rows per thread (r, r + 16)
    const uint32_t lr = tid >> 4, lc = tid & 15;
    Chunk<DT> stage[2][CI];
    float4 param[2];
    auto fetch = [&](uint32_t y0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t y = y0 + lr + 16 * h;
            const char *row = static_cast<const char *>(A.y) + (size_t)y * A.ystride * esz;
#pragma unroll
            for (int i = 0; i < CI; ++i) stage[h][i] = load_chunk<DT>(row, 8 * (lc + 16 * i), y < yend ? dim : 0, yvec);
            if (MODE == kRows) param[h] = lc == 0 && y < yend ? A.yparam[y] : make_float4(0.0f, 0.0f, 1.0f, __uint_as_float(kNoTarget));
        }
    };
    auto commit = [&](uint32_t buf) {
        char *tile = lds + buf * C::BUF;
        float *yv = reinterpret_cast<float *>(lds + C::NBUF * C::BUF) + buf * C::TY * 4;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t r = lr + 16 * h, sw = ((r & 7) << 1) | ((r >> 3) & 1);
            int e = 0;
            float top = 0.0f;
            if constexpr (F32) {
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < CI; ++i) m = max(m, __float_as_uint(absmax(stage[h][i])));
#pragma unroll
                for (int d = 1; d < 16; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
                top = __uint_as_float(m);
                e = row_exponent(top);
            }
            const float s = F32 ? pow2(-e) : 1.0f;
#pragma unroll
            for (int i = 0; i < CI; ++i) {
                const uint32_t c = lc + 16 * i;
                if (KS * 4 % 16 == 0 || c < (uint32_t)KS * 4) {
                    char *at = tile + r * PITCH + i * 256 + ((lc ^ sw) << 4);
                    if constexpr (F32) {
                        half8 hi, lo;
                        split8(stage[h][i], top, s, hi, lo);
                        *reinterpret_cast<half8 *>(at) = hi;
                        *reinterpret_cast<half8 *>(at + C::PLANE) = lo;
                    } else {
                        *reinterpret_cast<u32x4 *>(at) = stage[h][i].v;
                    }
                }
            }
            if (lc == 0 && (F32 || MODE == kRows)) {            // what a logit is multiplied by and what is added to it; sign and target
                float bias = F32 && MODE != kStats ? (float)e : 0.0f;
                if (MODE == kRows) {
                    bias += param[h].x;
                    yv[64 + r] = param[h].z;
                    yv[96 + r] = param[h].w;
                }
                yv[r] = row_factor(top, e);
                yv[32 + r] = bias;
            }
        }
    };

    auto compute = [&](uint32_t buf, uint32_t y0) {
        const char *tile = lds + buf * C::BUF;
        const float *yv = reinterpret_cast<const float *>(lds + C::NBUF * C::BUF) + buf * C::TY * 4;
        f32x4 S[2][NX];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < NX; ++j) S[h][j] = f32x4{0, 0, 0, 0};
        {
            const uint32_t sw = ((n & 7) << 1) | (n >> 3);      // (row + 16: the same swizzle)
            const char *row = tile + n * PITCH;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const uint32_t c = 4 * ks + g;
                const char *at = row + (c & ~15u) * 16 + (((c & 15) ^ sw) << 4);
                V a[2][NP];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int p = 0; p < NP; ++p) a[h][p] = *reinterpret_cast<const V *>(at + h * 16 * PITCH + p * C::PLANE);
                if constexpr (F32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < NX; ++j) S[h][j] = mma(a[h][1], X[j][ks][0], S[h][j]);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < NX; ++j) S[h][j] = mma(a[h][0], X[j][ks][1], S[h][j]);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < NX; ++j) S[h][j] = mma(a[h][0], X[j][ks][0], S[h][j]);
            }
        }
        f32x4 ky[2], bias[2];
        if (F32 || MODE == kRows)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                ky[h] = *reinterpret_cast<const f32x4 *>(yv + 16 * h + 4 * g);
                bias[h] = *reinterpret_cast<const f32x4 *>(yv + 32 + 16 * h + 4 * g);
            }
        const bool tail = y0 + 32 > yend;
        bool met = false, neg = false;                          // a target of these rows lies in the tile; a weight is negative
        if (MODE != kRows) {
#pragma unroll
            for (int j = 0; j < NX; ++j) met |= target[j] - y0 < 32;
            met = __any(met);
        } else {
            met = __any(__float_as_uint(yv[96 + (lane & 31)]) - x0 < 16 * NX);
            neg = __any(yv[64 + (lane & 31)] < 0.0f);
        }
        constexpr bool BIAS = TWO || MODE == kRows;
#pragma unroll
        for (int j = 0; j < NX; ++j) {
            const uint32_t x = x0 + j * 16 + n;
            uint32_t dead = 0, hit = 0;                         // bits of the elements (h, i) that take no part / that are a query's own row
            if (met || tail) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t r = 16 * h + 4 * g + i;
                        if (MODE != kRows && y0 + r == target[j]) {
                            float z = S[h][j][i];
                            if (F32) z *= ky[h][i];
                            if (slice == 0) A.own2[x] = z * kx[j];
                            dead |= 1u << (4 * h + i);
                        }
                        if (MODE == kRows && __float_as_uint(yv[96 + r]) == x) hit |= 1u << (4 * h + i);
                        if (y0 + r >= yend) dead |= 1u << (4 * h + i);
                    }
            }
            // the logit of element (h, i), in units of log 2, minus a reference
            auto logit = [&](int h, int i, bool biased, float ref) {
                float z = S[h][j][i];
                if (F32) z *= ky[h][i];
                z = fmaf(z, kx[j], biased ? bias[h][i] - ref : -ref);
                if (met || tail) {
                    if (MODE == kRows && (hit >> (4 * h + i) & 1)) z = A.yparam[y0 + 16 * h + 4 * g + i].y + (F32 ? log2f(ky[h][i]) : 0.0f) - ref;
                    if (dead >> (4 * h + i) & 1) z = -INFINITY;
                }
                return z;
            };
            // weights 2^(logit - ref) under a reference that moves where one would pass 2^kTop; true where it moved, by a factor `old`
            auto weigh = [&](bool biased, float &ref, float &old, float (&p)[2][4]) {
                float top = kNothing;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        p[h][i] = logit(h, i, biased, ref);
                        top = fmaxf(top, p[h][i]);
                    }
                const bool move = __any(top > kTop);
                if (move) {
                    float z = kNothing;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            p[h][i] = logit(h, i, biased, 0.0f);
                            z = fmaxf(z, p[h][i]);
                        }
                    z = fmaxf(z, __shfl_xor(z, 16));
                    z = fmaxf(z, __shfl_xor(z, 32));
                    const float to = z - ref > kTop ? z - kStart : ref;
                    old = exp2_hw(ref - to);
                    ref = to;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[h][i] -= to;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[h][i] = exp2_hw(p[h][i]);
                return move;
            };
            float p[2][4], old = 1.0f;
            if (TWO) {
                if (weigh(false, Ml[j], old, p)) l[j] *= old;
                l[j] += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
            }
            if (weigh(BIAS, M[j], old, p)) {
                if (!TWO) l[j] *= old;
                if (MODE != kStats)
#pragma unroll
                    for (int ob = 0; ob < OB; ++ob) O[ob][j] *= old;
            }
            if (MODE != kRows && !TWO) l[j] += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
            if constexpr (MODE != kStats) {
                if (MODE == kRows && (neg || met)) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            p[h][i] *= yv[64 + 16 * h + 4 * g + i];
                            if (hit >> (4 * h + i) & 1) p[h][i] = -p[h][i];
                        }
                }
                V w, wl;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (DT == RG_DTYPE_BF16) {
                            w[4 * h + i] = (__bf16)p[h][i];
                        } else {
                            w[4 * h + i] = (_Float16)p[h][i];
                            if (F32) wl[4 * h + i] = (_Float16)(p[h][i] - (float)w[4 * h + i]);
                        }
                    }
                S[0][j] = __builtin_bit_cast(f32x4, w);
                if (F32) S[1][j] = __builtin_bit_cast(f32x4, wl);
            }
        }
        if constexpr (MODE != kStats) {
            // lane (n, g) reads 8 bytes of row 4 g + n / 4 (and + 16) at dims 4 (n % 4) of the block, and receives dim n of rows 4 g .. + 3
            typedef __attribute__((address_space(3))) s16x4 *tr_ptr;
            const uint32_t r = 4 * g + (n >> 2), sw = ((r & 7) << 1) | ((r >> 3) & 1);     // (row + 16: the same swizzle)
            const char *row = tile + r * PITCH + (n & 1) * 8;
#pragma unroll
            for (int ob = 0; ob < OB; ++ob) {
                const uint32_t c = 2 * (slice * OB + ob) + ((n >> 1) & 1);
                const char *at = row + (c & ~15u) * 16 + (((c & 15) ^ sw) << 4);
                V a[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(const_cast<char *>(at) + p * C::PLANE));
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(const_cast<char *>(at) + p * C::PLANE + 16 * PITCH));
                    a[p] = __builtin_bit_cast(V, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                }
#pragma unroll
                for (int j = 0; j < NX; ++j) {
                    if constexpr (F32) {
                        O[ob][j] = mma(a[1], __builtin_bit_cast(V, S[0][j]), O[ob][j]);
                        O[ob][j] = mma(a[0], __builtin_bit_cast(V, S[1][j]), O[ob][j]);
                    }
                    O[ob][j] = mma(a[0], __builtin_bit_cast(V, S[0][j]), O[ob][j]);
                }
            }
        }
    };

    if (ybeg < yend) {
        if constexpr (C::NBUF == 2) {
            fetch(ybeg);
            commit(0);
            __syncthreads();
            uint32_t buf = 0;
            for (uint32_t y0 = ybeg; y0 < yend; y0 += 32, buf ^= 1) {
                const bool more = y0 + 32 < yend;
                if (more) fetch(y0 + 32);
                if (live) compute(buf, y0);
                if (more) commit(buf ^ 1);
                __syncthreads();
            }
        } else {
            for (uint32_t y0 = ybeg; y0 < yend; y0 += 32) {
                fetch(y0);
                commit(0);
                __syncthreads();
                if (live) compute(0, y0);
                __syncthreads();
            }
        }
    }

#pragma unroll
    for (int j = 0; j < NX; ++j) {
        const uint32_t x = x0 + j * 16 + n;
        if (x >= A.nx) continue;
        float s = l[j];
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        const size_t at = (size_t)split * A.nx + x;
        const bool direct = MODE == kRows && A.nsplit == 1;
        if (!direct && g == 0 && slice == 0) A.ml[at] = make_float4(TWO ? Ml[j] : M[j], s, M[j], 0.0f);
        if constexpr (MODE != kStats) {
            const float f = direct ? exp2_hw(0.5f * M[j]) : 1.0f;      // 2^M in two steps: it may lie below the normal range
#pragma unroll
            for (int ob = 0; ob < OB; ++ob) {
                const uint32_t d = (slice * OB + ob) * 16 + 4 * g;
                if (d >= dim) continue;
                if (!direct) {
                    *reinterpret_cast<f32x4 *>(A.o + at * A.opitch + d) = O[ob][j];
                } else {
                    T *out = static_cast<T *>(A.out) + (size_t)x * A.ostride + d;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (d + i < dim) out[i] = (T)(O[ob][j][i] * f * (f * A.oscale));
                }
            }
        }
    }
}

}  // namespace rg
