// rg_softmax.hip -- softmax cross entropy over all rows of a base, and its gradients, without storing the logits.
//
// With z_ij = scale <q_i, b_j> (kept in units of log 2: z2 = z log2 e, so that every exponential is one v_exp_f32):
//
//   statistics + mean   for each query i one pass over the rows j != target with a running reference M, sums l, R and sum O:
//                         P = 2^(z2 - M),  l += P,  W = P in the rows' type,  R += W,  O += W b_j      rest = ln 2 (M + log2 l),  mean = O / R
//                       the target's own logit is set aside, so that loss = log(1 + e^(rest - own)) keeps its digits where it is small
//   gradient of rows    for each row j one pass over the queries i -- the same pass with the roles exchanged:
//                         G = w_i 2^(z2 - lse2_i) = +-2^(z2 + bias_i),   bias_i = log2|w_i| - lse2_i
//                         (at j = t_i: -w_i (1 - e^-loss_i)),            db_j = scale sum_i G q_i
//   gradient of queries dq_i = w_i scale (e^(rest - lse) mean_i - (1 - e^-loss) b_target): one small kernel, the product is in the mean
//
// so one kernel serves both: a tile of stationary rows x, streamed rows y, weights 2^(z2 + bias_y), sum of weights times y.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "rg.h"
#include "rg_internal.h"
#include "rg_rows.h"
#include "rg_softmax_pass.h"

namespace rg {
namespace {

constexpr uint32_t kMaxDim = 1024, kMaxQueries = (1u << 24) - 1;     // (a workgroup of 256 each, and a launch holds less than 2^32 threads)
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;

__device__ __forceinline__ bool target_here(uint32_t t, uint32_t id_base, uint32_t nb) { return t != kNoTarget && t >= id_base && t - id_base < nb; }

// log(1 + e^d) without overflow: loss of a target d below the others' log sum
__device__ __forceinline__ float softplus(float d) { return d > 15.0f ? d + log1pf(expf(-d)) : log1pf(expf(d)); }

// the loss of a target whose logit is `own`, d below the others' log sum, and the log sum r with it: a logit of +inf is infinity less infinity, no
// perfect answer; one of -inf takes no part in the sum
__device__ __forceinline__ float loss_of(float own, float d) { return own == INFINITY ? NAN : own == -INFINITY ? INFINITY : softplus(d); }
__device__ __forceinline__ float lse_of(float own, float loss, float r) { return own == -INFINITY ? r : own + loss; }

// joins the slots of a query: rest, target logit, lse, loss, mean of the others.  One workgroup per query, or, where queries are few, per query
// and kJoinDims of the mean's elements; with many slots, sixteen groups of lanes share them
// (244 slots of 333 queries x 93: four groups of single elements 25 us, now 12 us).
constexpr uint32_t kJoinDims = 64, kJoinSlots = 16;
__global__ void __launch_bounds__(256) rg_softmax_join_kernel(const float4 *ml, const float *o, uint32_t opitch, uint32_t nslots, uint32_t nq, uint32_t dim, uint32_t nb, uint32_t id_base, const float *own2,
                                                              const uint32_t *targets, float *rest, float *own, float *lse, float *loss, float *mean) {
    const uint32_t i = blockIdx.x, tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    __shared__ float red[8], weight[256];
    __shared__ __attribute__((aligned(16))) float part[16][kJoinDims];
    float M = kNothing, Mo = kNothing;
    for (uint32_t s = tid; s < nslots; s += 256) {
        const float4 v = ml[(size_t)s * nq + i];
        M = fmaxf(M, v.x);
        Mo = fmaxf(Mo, v.z);
    }
    for (int d = 1; d < 64; d <<= 1) {
        M = fmaxf(M, __shfl_xor(M, d));
        Mo = fmaxf(Mo, __shfl_xor(Mo, d));
    }
    if (lane == 0) { red[wave] = M; red[4 + wave] = Mo; }
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    Mo = fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]));
    float l = 0.0f, div = 0.0f;            // sum of the weights; what the mean is divided by (the weights as they were multiplied)
    for (uint32_t s = tid; s < nslots; s += 256) {
        const float4 v = ml[(size_t)s * nq + i];
        const float f = exp2f(v.x - M);
        l += v.y * f;
        div += v.w * f;
    }
    for (int d = 1; d < 64; d <<= 1) {
        l += __shfl_xor(l, d);
        div += __shfl_xor(div, d);
    }
    __syncthreads();
    if (lane == 0) { red[wave] = l; red[4 + wave] = div; }
    __syncthreads();
    l = red[0] + red[1] + red[2] + red[3];
    div = red[4] + red[5] + red[6] + red[7];
    const bool none = M == kNothing && l == 0.0f;       // no other row than the target (where all logits are NaN the reference has not moved either, but l is NaN)
    if (tid == 0 && blockIdx.y == 0) {
        const uint32_t t = targets[i];
        const bool here = target_here(t, id_base, nb);
        // (in 64 bits: the instruction behind log2f rounds down, which a small loss shows)
        const double r2 = none ? -INFINITY : (double)M + log2((double)l), z2 = here ? own2[i] : -INFINITY;
        const float r = (float)(r2 * kLn2), z = (float)(z2 * kLn2);
        const float v = t == kNoTarget ? 0.0f : r != r ? r : here ? loss_of(z, (float)((r2 - z2) * kLn2)) : INFINITY;
        rest[i] = r;
        own[i] = z;
        if (lse) lse[i] = here ? lse_of(z, v, r) : r;
        if (loss) loss[i] = v;
    }
    if (mean) {
        const float f = none ? 0.0f : exp2f(Mo - M) / div;
        const bool many = nslots >= kJoinSlots;
        const uint32_t width = many ? kJoinDims : 256, group = tid / 16;
        for (uint32_t k0 = blockIdx.y * width; k0 < dim; k0 += gridDim.y * width) {
            const uint32_t k = k0 + (many ? tid % 16 * 4 : tid);
            float s = 0.0f;
            f32x4 s4{0.0f, 0.0f, 0.0f, 0.0f};
            for (uint32_t e0 = 0; e0 < nslots; e0 += 256) {
                __syncthreads();
                if (e0 + tid < nslots) weight[tid] = exp2f(ml[(size_t)(e0 + tid) * nq + i].z - Mo);
                __syncthreads();
                const uint32_t n = min(256u, nslots - e0);
                const float *row = o + ((size_t)e0 * nq + i) * opitch + k;
                if (k >= dim) continue;
                if (many) {
#pragma unroll 8
                    for (uint32_t e = group; e < n; e += 16) s4 += weight[e] * *reinterpret_cast<const f32x4 *>(row + (size_t)e * nq * opitch);
                } else {
                    for (uint32_t e = 0; e < n; ++e) s = fmaf(weight[e], row[(size_t)e * nq * opitch], s);
                }
            }
            if (many) {
                *reinterpret_cast<f32x4 *>(&part[group][tid % 16 * 4]) = s4;
                __syncthreads();
                if (tid < kJoinDims)
#pragma unroll
                    for (uint32_t g = 0; g < 16; ++g) s += part[g][tid];
            }
            const uint32_t d = k0 + tid;
            if (tid < width && d < dim) mean[(size_t)i * dim + d] = s * f;
        }
    }
}

__global__ void __launch_bounds__(256) rg_softmax_merge_kernel(const float *rest_in, const float *own_in, uint32_t nlists, uint32_t nq, const uint32_t *targets, float *lse, float *loss) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= nq) return;
    float m = -INFINITY, own = -INFINITY;
    for (uint32_t s = 0; s < nlists; ++s) {
        m = fmaxf(m, rest_in[(size_t)s * nq + i]);
        const float z = own_in[(size_t)s * nq + i];
        own = z != z || z > own ? z : own;             // (once NaN, it stays)
    }
    float l = 0.0f;
    const float ref = m == -INFINITY ? 0.0f : m;
    for (uint32_t s = 0; s < nlists; ++s) l += expf(rest_in[(size_t)s * nq + i] - ref);       // (NaN where a shard's rest is)
    const double r2 = l == 0.0f ? -INFINITY : (double)ref + log((double)l);        // (in 64 bits, as in the join: a sum near the target's logit keeps its digits)
    const float r = (float)r2;
    const float v = targets[i] == kNoTarget ? 0.0f : r != r ? r : loss_of(own, (float)(r2 - own));
    lse[i] = targets[i] == kNoTarget ? r : lse_of(own, v, r);
    loss[i] = v;
}

// what a pass needs of a streamed row, 32 rows at a time: factors, biases, signs, targets (PassArgs::yinfo)
__device__ __forceinline__ void put_info(float *info, uint64_t y, float factor, float bias, float sign, uint32_t target) {
    float *at = info + (y / 32 * 128 + y % 32);
    at[0] = factor;
    at[32] = bias;
    at[64] = sign;
    at[96] = __uint_as_float(target);
}

// per query: what the pass over the rows needs of it (info, ytarget and, where queries cannot be read where they lie, planes; padded to whole tiles),
// and dq.  One wave per query.
template <int DT>
__global__ void __launch_bounds__(64) rg_softmax_dq_kernel(const void *queries, uint64_t qstride, const void *base, uint64_t bstride, uint32_t nb, uint32_t id_base, uint32_t nq, uint32_t dim, float scale,
                                                           const uint32_t *targets, const float *lse, const float *loss, const float *rest, const float *mean,
                                                           const float *weights, void *dq, uint64_t dqstride, float *info, float *ytarget, uint16_t *planes, uint32_t ks) {
    typedef typename Elem<DT>::T T;
    constexpr uint32_t NP = DT == RG_DTYPE_F32 ? 2 : 1;
    const uint32_t i = blockIdx.x;
    if (i >= nq) {
        if (threadIdx.x == 0) {
            put_info(info, i, 1.0f, -INFINITY, 0.0f, kNoTarget);     // (copies of the last query: they take no part, whatever that holds)
            ytarget[i] = -INFINITY;
        }
        if (planes)
            for (uint32_t c = threadIdx.x; c < NP * ks * 4; c += 64) reinterpret_cast<u32x4 *>(planes + (size_t)i * NP * ks * 32)[c] = u32x4{0, 0, 0, 0};
        return;
    }
    const uint32_t t = targets[i], row = t - id_base;
    const bool here = target_here(t, id_base, nb);
    const float w = t == kNoTarget ? 0.0f : weights[i], miss = here ? -expm1f(-loss[i]) : 0.0f;      // 1 - p_target
    bool whole = true;                  // a query that takes no part may hold anything: the pass over the rows is told (sign 0)
    if (info && t == kNoTarget) {
        for (uint32_t k = threadIdx.x; k < dim; k += 64) whole &= fabsf((float)static_cast<const T *>(queries)[(size_t)i * qstride + k]) < INFINITY;
        whole = __all(whole);
    }
    float factor = 1.0f;
    if (planes) {                       // (zeros of a query that is not finite and takes no part)
        Chunk<DT> c[2];
        load_chunks<DT, true>(c, static_cast<const T *>(queries) + (size_t)i * qstride, 8 * threadIdx.x, 512, dim, whole);
        uint16_t *out = planes + (size_t)i * NP * ks * 32;
        if constexpr (DT == RG_DTYPE_F32) {
            uint32_t m = max(__float_as_uint(absmax(c[0])), __float_as_uint(absmax(c[1])));
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
            const float top = __uint_as_float(m);
            const int e = row_exponent(top);
            factor = row_factor(top, e);
#pragma unroll
            for (uint32_t u = 0; u < 2; ++u) {
                if (threadIdx.x + 64 * u >= ks * 4) continue;
                half8 hi, lo;
                split8(c[u], top, pow2(-e), hi, lo);
                *reinterpret_cast<half8 *>(out + 8 * (threadIdx.x + 64 * u)) = hi;
                *reinterpret_cast<half8 *>(out + ks * 32 + 8 * (threadIdx.x + 64 * u)) = lo;
            }
        } else {
#pragma unroll
            for (uint32_t u = 0; u < 2; ++u)
                if (threadIdx.x + 64 * u < ks * 4) *reinterpret_cast<u32x4 *>(out + 8 * (threadIdx.x + 64 * u)) = c[u].v;
        }
    }
    if (info && threadIdx.x == 0) {
        const float lw = (float)log2((double)fabsf(w));
        put_info(info, i, factor, t == kNoTarget ? -INFINITY : lw - lse[i] * kLog2e, w < 0.0f ? -1.0f : whole ? 1.0f : 0.0f, here ? row : kNoTarget);
        ytarget[i] = lw + (float)log2((double)miss);
    }
    if (!dq) return;
    const float part = rest[i] == -INFINITY ? 0.0f : expf(rest[i] - lse[i]);
    for (uint32_t k = threadIdx.x; k < dim; k += 64) {
        float v = 0.0f;
        if (t != kNoTarget) {
            v = part * mean[(size_t)i * dim + k];
            if (here) v = fmaf(-miss, (float)static_cast<const T *>(base)[(size_t)row * bstride + k], v);
            v *= w * scale;
        }
        static_cast<T *>(dq)[(size_t)i * dqstride + k] = (T)v;
    }
}

// rows as the wide pass streams them: 16-bit planes of 32 ks elements, zeros behind dim and behind the last row; fp32 as two halves scaled by the
// row's power of two, whose factor and exponent go to `info`.  16 lanes per row, CI chunks of 8 elements a lane.
template <int DT, int CI>
__global__ void __launch_bounds__(256) rg_softmax_planes_kernel(const void *rows, uint64_t stride, uint32_t n, uint32_t npad, uint32_t dim, uint32_t ks, uint16_t *planes, float *info) {
    typedef typename Elem<DT>::T T;
    constexpr int NP = DT == RG_DTYPE_F32 ? 2 : 1;
    const uint32_t lc = threadIdx.x % 16;
    for (uint64_t r = (uint64_t)blockIdx.x * 16 + threadIdx.x / 16; r < npad; r += (uint64_t)gridDim.x * 16) {
        const char *row = static_cast<const char *>(rows) + (size_t)r * stride * sizeof(T);
        uint16_t *out = planes + (size_t)r * NP * ks * 32;
        Chunk<DT> c[CI];
        const bool take = r < n;
        load_chunks<DT, CI == 1>(c, row, 8 * lc, 128, dim, take);
        if constexpr (DT == RG_DTYPE_F32) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < CI; ++i) m = max(m, __float_as_uint(absmax(c[i])));
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
            const float top = __uint_as_float(m);
            const int e = row_exponent(top);
#pragma unroll
            for (int i = 0; i < CI; ++i) {
                if (lc + 16 * i >= ks * 4) continue;
                half8 hi, lo;
                split8(c[i], top, pow2(-e), hi, lo);
                *reinterpret_cast<half8 *>(out + 8 * (lc + 16 * i)) = hi;
                *reinterpret_cast<half8 *>(out + ks * 32 + 8 * (lc + 16 * i)) = lo;
            }
            if (lc == 0) put_info(info, r, row_factor(top, e), row_bias(top, e), 1.0f, kNoTarget);
        } else {
#pragma unroll
            for (int i = 0; i < CI; ++i)
                if (lc + 16 * i < ks * 4) *reinterpret_cast<u32x4 *>(out + 8 * (lc + 16 * i)) = c[i].v;
        }
    }
}

// db from the slots of the pass over the queries
template <int DT>
__global__ void __launch_bounds__(256) rg_softmax_db_kernel(const float4 *ml, const float *o, uint32_t opitch, uint32_t nslots, uint32_t nb, uint32_t dim, float scale, void *db, uint64_t dbstride) {
    typedef typename Elem<DT>::T T;
    for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < (uint64_t)nb * dim; at += (uint64_t)gridDim.x * 256) {
        const uint32_t j = (uint32_t)(at / dim), k = (uint32_t)(at % dim);
        float s = 0.0f;
        for (uint32_t e = 0; e < nslots; ++e) {
            const float f = exp2f(0.5f * ml[(size_t)e * nb + j].z);     // 2^M in two steps: it may lie below the normal range
            s = fmaf(f, f * o[((size_t)e * nb + j) * opitch + k], s);
        }
        static_cast<T *>(db)[(size_t)j * dbstride + k] = (T)(s * scale);
    }
}

uint64_t up256(uint64_t n) { return (n + 255) / 256 * 256; }
uint32_t up32(uint32_t n) { return (n + 31) / 32 * 32; }
uint32_t opitch_of(uint32_t dim) { return (dim + 15) / 16 * 16; }

// the instantiation a width runs in, as the number of 32-element steps that holds it (7: its output blocks end at 208)
int steps_of(uint32_t dim) {
    if (dim > 192 && dim <= 208) return 7;
    for (int ks : {2, 4, 8, 12, 16, 24})
        if (dim <= 32u * ks) return ks;
    return 32;
}

// at most this many bytes of planes at a time: a large base is streamed piece by piece
constexpr uint64_t kPieceBytes = 1ull << 30;

SoftmaxKernel kernel_of(int dtype, int mode, bool thin, int ks) {
    typedef SoftmaxKernel (*Pick)(int);
    static const Pick wide[3][3] = {{softmax_wide_f32_stats, softmax_wide_f32_mean, softmax_wide_f32_rows},
                                    {softmax_wide_f16_stats, softmax_wide_f16_mean, softmax_wide_f16_rows},
                                    {softmax_wide_bf16_stats, softmax_wide_bf16_mean, softmax_wide_bf16_rows}};
    static const Pick few[3][2] = {{softmax_thin_f32_stats, softmax_thin_f32_mean}, {softmax_thin_f16_stats, softmax_thin_f16_mean}, {softmax_thin_bf16_stats, softmax_thin_bf16_mean}};
    return thin ? few[dtype][mode](ks) : wide[dtype][mode](ks);
}

// how a pass is cut: into pieces of y that are made into planes one after another (planes), each split into slots whose partial results are
// joined at the end (a slot goes on from piece to piece).  More slots fill the workgroup places of the device, and each costs the writing and reading of its results: the cheapest
// number is taken, in bytes of the device's traffic, one of which it moves while its matrix cores do kOpsPerByte operations of a pass (measured:
// 600 Top/s of the 16-bit passes, 4 TB/s).  333 fp16 queries on 70001 rows of 93 dims: 3 slots, which leave fewer places empty, took
// 80 us + 29 us to join for the gradient of the rows, 1 slot 58 us.
// With and without the mean, a call is cut alike (for the sum of both costs), so that both give the same loss.
constexpr double kOpsPerByte = 150, kLaunchCost = 16e6;     // (bytes of the 4 us of a launch)
struct Use {                          // of the device by a kernel
    uint64_t nt, places;              // workgroups of a slot; workgroups that run at once
    double row_cost;                  // bytes of a row y, were all places used
    double busy(uint32_t rows, uint32_t n) const {
        const uint64_t rounds = (n * nt + places - 1) / places;
        return row_cost * rows * (double)(rounds * places) / ((double)nt * n);
    }
};
struct Plan {
    SoftmaxKernel k;
    int ks;
    bool thin, planes;
    uint32_t nx, ny, ntx, piece, nslots;
    uint64_t row_bytes;               // of a row of planes
    Use use[2];
    int nuse;
    double slot_cost;                 // bytes of a slot
    bool free_slot;                   // a single slot needs no joining
    struct Cut {
        uint32_t nsplit, rows;
    };
    Cut cut(uint32_t rows) const {
        const uint32_t most = std::max(1u, rows / 32);
        uint32_t best = 1;
        double least = HUGE_VAL;
        auto look = [&](uint64_t n_) {
            const uint32_t n = (uint32_t)std::clamp<uint64_t>(n_, 1, most);
            double cost = n == 1 && free_slot ? 0.0 : nuse * n * slot_cost + (free_slot ? kLaunchCost : 0.0);
            for (int u = 0; u < nuse; ++u) cost += use[u].busy(rows, n);
            if (cost < least || (cost == least && n < best)) { least = cost; best = n; }
        };
        look(1);
        for (int u = 0; u < nuse; ++u) {
            const Use &U = use[u];
            look((uint64_t)std::sqrt(U.row_cost * rows * (double)U.places / ((double)U.nt * slot_cost)));     // where one round does: the least of busy / n + n slot_cost
            for (uint64_t first = (U.nt + U.places - 1) / U.places, rounds = first; rounds <= first + 3; ++rounds) look(rounds * U.places / U.nt);     // the most slots of so many rounds
        }
        Cut c;
        c.rows = up32((std::max(rows, 1u) + best - 1) / best);
        c.nsplit = std::max(1u, (rows + c.rows - 1) / c.rows);
        return c;
    }
};

// The kernel of a mode.  Few rows x: the pass is bound by reading y, and the thin kernel, which reads fp32 rows and rows of any alignment where
// they lie, once for 64 rows x, beats planes made first, read and read again (1.25M x 200 fp32: 64 queries 349 us against 660 us, 128 queries
// 613 / 772 us, 256 1138 / 1124 us; 16-bit rows that need planes gain more: 830k x 301 bf16, 256 queries 488 / 570 us) -- and of short 16-bit rows
// that need none it still does up to 128 (2M x 64 bf16 179 / 226 us; 1.25M x 200, where the wide kernel reads in place what fills its tiles, 250 / 197 us).
// It holds a row in a wave's registers: of wide rows the sums no longer fit, and the wide kernel is faster even with planes (fp32 x 768, 64
// queries: 994 against 669 us; 488k x 512 559 / 622 us, with 128 queries 1042 / 802 us; fp16 500k x 512 in place, 8 - 64 queries 209 - 241 / 113 - 127 us).  Statistics alone
// are the thin kernel's up to 512 elements in place (111 / 121 us; x 1024 131 / 122 us) and at all widths with planes.
bool thin_of(int dtype, int mode, int ks, uint32_t nx, bool direct) {
    const bool f32 = dtype == RG_DTYPE_F32;
    if (mode == kRows || nx > (direct ? (ks <= 2 ? 128 : 64) : f32 ? 128 : 256)) return false;
    return mode == kStats ? ks <= 16 || !direct : ks <= (direct || (f32 && nx > 64) ? 8 : 16);
}

// direct: the streamed rows can be read where they lie (16-bit rows of whole 16-byte chunks, 16-byte aligned)
Plan plan_of(int dtype, int mode, uint32_t dim, uint32_t nx, uint32_t ny, bool direct) {
    Plan p;
    p.ks = steps_of(dim);
    p.thin = thin_of(dtype, mode, p.ks, nx, direct);
    p.k = kernel_of(dtype, mode, p.thin, p.ks);
    p.planes = !p.thin && !direct;
    p.nx = nx;
    p.ny = ny;
    p.ntx = std::max(1u, (uint32_t)(((uint64_t)nx + p.k.xt - 1) / p.k.xt));
    p.row_bytes = (uint64_t)(dtype == RG_DTYPE_F32 ? 2 : 1) * p.ks * 64;
    p.nuse = 0;
    bool any_planes = false;
    for (int m = mode == kRows ? kRows : kStats; m <= (mode == kRows ? kRows : kMean); ++m) {
        const bool thin = thin_of(dtype, m, p.ks, nx, direct);
        const SoftmaxKernel k = kernel_of(dtype, m, thin, p.ks);
        Use &u = p.use[p.nuse++];
        u.nt = std::max<uint64_t>(1, ((uint64_t)nx + k.xt - 1) / k.xt);
        u.places = 256ull * std::min<uint32_t>(k.wps * 256 / k.threads, 160 * 1024 / k.lds);     // (256 CUs)
        const double ops = 2.0 * (dtype == RG_DTYPE_F32 ? 3 : 1) * (double)(u.nt * k.xt) * (32.0 * p.ks + (m == kStats ? 0.0 : 16.0 * k.ob));     // of a row y
        u.row_cost = std::max(thin || direct ? (double)dim * elem_bytes(dtype) * (thin ? (double)u.nt : 1.0) : 0.0, thin ? 0.0 : ops / kOpsPerByte);
        any_planes |= !thin && !direct;
    }
    p.slot_cost = 8.0 * opitch_of(dim) * std::max(nx, 1u);
    p.free_slot = mode == kRows;
    p.piece = ny;
    if (any_planes && mode != kRows) p.piece = (uint32_t)std::min<uint64_t>(ny, kPieceBytes / p.row_bytes / 32 * 32);
    p.nslots = p.cut(p.piece).nsplit;
    return p;
}

// the parts of the scratch: references and sums of the slots, sums of rows of the slots, per query its target's logit or its parameters,
// parameters of the streamed rows, planes
struct Layout {
    uint64_t ml, o, aux, info, planes, total;
};
Layout layout_of(const Plan &p, int mode, int dtype, uint32_t dim) {
    Layout L;
    const bool pieces = mode != kRows || p.nslots > 1;
    uint64_t at = 0;
    auto part = [&](uint64_t bytes) { const uint64_t was = at; at += up256(bytes); return was; };
    L.ml = part(pieces ? (uint64_t)p.nslots * p.nx * 16 : 0);
    L.o = part(pieces && mode != kStats ? (uint64_t)p.nslots * p.nx * opitch_of(dim) * 4 : 0);
    L.aux = part(mode == kRows ? (uint64_t)up32(p.ny) * 4 : (uint64_t)p.nx * 4);
    L.info = part(mode == kRows ? (uint64_t)up32(p.ny) * 16 : p.planes && dtype == RG_DTYPE_F32 ? (uint64_t)up32(p.piece) * 16 : 0);
    L.planes = part(p.planes ? up32(p.piece) * p.row_bytes : 0);
    L.total = at;
    return L;
}
// of a call whose pointers are not known yet
uint64_t scratch_of(int mode, uint32_t nb, uint32_t nq, uint32_t dim, int dtype) {
    const uint32_t nx = mode == kRows ? nb : nq, ny = mode == kRows ? nq : nb;
    uint64_t n = layout_of(plan_of(dtype, mode, dim, nx, ny, false), mode, dtype, dim).total;
    if (dtype != RG_DTYPE_F32 && dim % 8 == 0) n = std::max(n, layout_of(plan_of(dtype, mode, dim, nx, ny, true), mode, dtype, dim).total);
    return n;
}
bool direct_rows(const void *rows, uint64_t stride, uint32_t dim, int dtype) {
    return dtype != RG_DTYPE_F32 && dim % 8 == 0 && stride % 8 == 0 && stride < (1u << 25) && (uintptr_t)rows % 16 == 0;     // (32 rows' bytes in 32 bits)
}
template <int DT>
rg_status make_planes(const void *rows, uint64_t stride, uint32_t n, uint32_t dim, int ks, void *planes, float *info, hipStream_t s) {
    auto kern = ks <= 4 ? rg_softmax_planes_kernel<DT, 1> : ks <= 8 ? rg_softmax_planes_kernel<DT, 2> : ks <= 16 ? rg_softmax_planes_kernel<DT, 4> : rg_softmax_planes_kernel<DT, 8>;
    const uint32_t npad = up32(n);
    hipLaunchKernelGGL(kern, dim3(std::min(npad / 16, 1u << 16)), dim3(256), 0, s, rows, stride, n, npad, dim, (uint32_t)ks, static_cast<uint16_t *>(planes), info);
    RG_HIP(hipGetLastError());
    return RG_OK;
}

rg_status launch_pass(const Plan &p, const PassArgs &A, hipStream_t s) {
    const uint64_t grid = (uint64_t)p.ntx * A.nsplit;
    if (grid * p.k.threads > 0xffffffffull) return set_error(RG_ERR_ARG, "softmax over a base: too many rows for one launch");
    if (p.k.lds > 64 * 1024) RG_HIP(hipFuncSetAttribute(p.k.kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.k.lds));
    void *args[] = {const_cast<PassArgs *>(&A)};
    RG_HIP(hipLaunchKernel(p.k.kern, dim3((uint32_t)grid), dim3(p.k.threads), args, p.k.lds, s));
    return RG_OK;
}

rg_status check_shapes(uint32_t nb, uint32_t nq, uint32_t dim, int dtype) {
    if (!known_dtype(dtype)) return set_error(RG_ERR_ARG, "unknown dtype");
    if (dim == 0 || dim > kMaxDim) return set_error(RG_ERR_ARG, "softmax over a base: dim must be in [1, 1024]");
    if (nb > 0x7fffffffu || nq > kMaxQueries) return set_error(RG_ERR_ARG, "softmax over a base: at most 2^31 - 1 rows and 2^24 - 1 queries");
    return RG_OK;
}
rg_status check_rows(const void *p, uint32_t n, uint64_t stride, uint32_t dim, int dtype, const char *name) {
    if (n == 0) return RG_OK;
    if (!p) return set_error(RG_ERR_ARG, "null argument");
    if (stride < dim) return set_error(RG_ERR_ARG, std::string(name) + ": row stride smaller than dim");
    if ((uintptr_t)p % elem_bytes(dtype)) return set_error(RG_ERR_ARG, std::string(name) + ": not aligned to its elements");
    return RG_OK;
}

rg_status check_call(uint32_t nb, const void *base, uint64_t bstride, uint32_t nq, const void *queries, uint64_t qstride, uint32_t dim, int dtype, float scale, uint32_t id_base) {
    rg_status st = check_shapes(nb, nq, dim, dtype);
    if (st == RG_OK) st = check_rows(base, nb, bstride, dim, dtype, "base");
    if (st == RG_OK) st = check_rows(queries, nq, qstride, dim, dtype, "queries");
    if (st != RG_OK) return st;
    if (!std::isfinite(scale * kLog2e)) return set_error(RG_ERR_ARG, "the scale must be finite, and below 2e38");
    if ((uint64_t)id_base + nb > 0xffffffffull) return set_error(RG_ERR_ARG, "row ids beyond 2^32 - 2");
    return RG_OK;
}
rg_status check_scratch(const void *work, uint64_t have, uint64_t need) {
    if (need == 0) return RG_OK;
    if (!work) return set_error(RG_ERR_ARG, "null argument");
    if ((uintptr_t)work & 255) return set_error(RG_ERR_ARG, "the scratch is not 256-byte aligned");
    if (have < need) return set_error(RG_ERR_ARG, "the scratch is smaller than rg_softmax_workspace() says");
    return RG_OK;
}

struct Call {      // the arguments of the entry points
    const void *base, *queries;
    uint64_t bstride, qstride;
    uint32_t nb, nq, dim, id_base;
    float scale;
    const uint32_t *targets;
    char *work;
    hipStream_t s;
};

template <int DT>
rg_status shard(const Call &c, float *rest, float *own, float *lse, float *loss, float *mean) {
    const int mode = mean ? kMean : kStats;
    const Plan p = plan_of(DT, mode, c.dim, c.nq, c.nb, direct_rows(c.base, c.bstride, c.dim, DT));
    const Layout L = layout_of(p, mode, DT, c.dim);
    PassArgs A{};
    A.x = c.queries; A.xstride = c.qstride; A.nx = c.nq;
    A.dim = A.ydim = c.dim;
    A.k = c.scale * kLog2e;
    A.opitch = opitch_of(c.dim);
    A.targets = c.targets; A.own2 = reinterpret_cast<float *>(c.work + L.aux);
    float4 *ml = reinterpret_cast<float4 *>(c.work + L.ml);
    float *o = reinterpret_cast<float *>(c.work + L.o);
    A.ml = ml; A.o = o;
    A.nsplit = p.nslots;
    for (uint64_t y = 0; y == 0 || y < c.nb; y += std::max(p.piece, 1u)) {
        const uint32_t n = (uint32_t)std::min<uint64_t>(p.piece, c.nb - y);
        A.y = static_cast<const char *>(c.base) + y * c.bstride * sizeof(typename Elem<DT>::T);
        A.ystride = c.bstride; A.ny = n;
        A.id_base = c.id_base + (uint32_t)y;
        A.rows_per_split = up32((uint32_t)(((uint64_t)n + p.nslots - 1) / p.nslots));
        A.resume = y != 0;
        if (p.planes && n) {
            float *info = reinterpret_cast<float *>(c.work + L.info);
            rg_status st = make_planes<DT>(A.y, c.bstride, n, c.dim, p.ks, c.work + L.planes, info, c.s);
            if (st != RG_OK) return st;
            A.y = c.work + L.planes; A.ystride = p.row_bytes / 2; A.ydim = 32 * p.ks; A.yinfo = info;
        }
        rg_status st = launch_pass(p, A, c.s);
        if (st != RG_OK) return st;
    }
    hipLaunchKernelGGL(rg_softmax_join_kernel, dim3(c.nq, mean ? std::clamp(4096u / c.nq, 1u, (c.dim + kJoinDims - 1) / kJoinDims) : 1), dim3(256), 0, c.s, ml, o, A.opitch, p.nslots, c.nq, c.dim, c.nb, c.id_base, A.own2, c.targets, rest, own, lse, loss, mean);
    RG_HIP(hipGetLastError());
    return RG_OK;
}

template <int DT>
rg_status grad(const Call &c, const float *lse, const float *loss, const float *rest, const float *mean, const float *weights, void *dq, uint64_t dqstride, void *db, uint64_t dbstride) {
    const uint32_t rows = db ? c.nb : 0;
    const Plan p = plan_of(DT, kRows, c.dim, rows, c.nq, direct_rows(c.queries, c.qstride, c.dim, DT));
    const Layout L = layout_of(p, kRows, DT, c.dim);
    float *info = rows ? reinterpret_cast<float *>(c.work + L.info) : nullptr;
    float *ytarget = rows ? reinterpret_cast<float *>(c.work + L.aux) : nullptr;
    uint16_t *planes = p.planes && rows && c.nq ? reinterpret_cast<uint16_t *>(c.work + L.planes) : nullptr;
    if (c.nq) {
        hipLaunchKernelGGL((rg_softmax_dq_kernel<DT>), dim3(rows ? up32(c.nq) : c.nq), dim3(64), 0, c.s, c.queries, c.qstride, c.base, c.bstride, c.nb, c.id_base, c.nq, c.dim, c.scale, c.targets, lse, loss, rest, mean, weights,
                           dq, dqstride, info, ytarget, planes, (uint32_t)p.ks);
        RG_HIP(hipGetLastError());
    }
    if (!rows) return RG_OK;
    const Plan::Cut cut = p.cut(c.nq);
    PassArgs A{};
    A.x = c.base; A.xstride = c.bstride; A.nx = rows;
    A.y = c.queries; A.ystride = c.qstride; A.ny = c.nq;
    A.dim = A.ydim = c.dim;
    A.k = c.scale * kLog2e;
    A.nsplit = cut.nsplit; A.rows_per_split = cut.rows; A.opitch = opitch_of(c.dim);
    A.ml = reinterpret_cast<float4 *>(c.work + L.ml);
    A.o = reinterpret_cast<float *>(c.work + L.o);
    A.yinfo = info; A.ytarget = ytarget;
    A.out = db; A.ostride = dbstride; A.oscale = c.scale;
    if (planes) {
        A.y = c.work + L.planes; A.ystride = p.row_bytes / 2; A.ydim = 32 * p.ks;
    }
    rg_status st = launch_pass(p, A, c.s);
    if (st != RG_OK || cut.nsplit == 1) return st;
    const uint64_t n = (uint64_t)rows * c.dim;
    hipLaunchKernelGGL((rg_softmax_db_kernel<DT>), dim3((uint32_t)std::min<uint64_t>((n + 255) / 256, 1u << 20)), dim3(256), 0, c.s, A.ml, A.o, A.opitch, cut.nsplit, rows, c.dim, c.scale, db, dbstride);
    RG_HIP(hipGetLastError());
    return RG_OK;
}

}  // namespace
}  // namespace rg

using namespace rg;

extern "C" {

rg_status rg_softmax_workspace(int what, uint32_t nb, uint32_t nq, uint32_t dim, int dtype, uint64_t *bytes) {
    if (!bytes) return set_error(RG_ERR_ARG, "null argument");
    if (what != RG_SOFTMAX_STATS && what != RG_SOFTMAX_MEAN && what != RG_SOFTMAX_GRAD) return set_error(RG_ERR_ARG, "unknown kind of call");
    rg_status st = check_shapes(nb, nq, dim, dtype);
    if (st != RG_OK) return st;
    *bytes = scratch_of(what, nb, nq, dim, dtype);
    return RG_OK;
}

rg_status rg_softmax_shard_dev(const void *d_base, uint32_t nb, uint64_t bstride, const void *d_queries, uint32_t nq, uint64_t qstride,
                               uint32_t dim, int dtype, float scale, const uint32_t *d_targets, uint32_t id_base, float *d_rest,
                               float *d_own, float *d_lse, float *d_loss, float *d_mean, void *d_work, uint64_t work_bytes, int device,
                               void *stream) {
    rg_status st = check_call(nb, d_base, bstride, nq, d_queries, qstride, dim, dtype, scale, id_base);
    if (st != RG_OK || nq == 0) return st;
    if (!d_targets || !d_rest || !d_own) return set_error(RG_ERR_ARG, "null argument");
    st = check_scratch(d_work, work_bytes, scratch_of(d_mean ? kMean : kStats, nb, nq, dim, dtype));
    if (st != RG_OK) return st;
    OnDevice on(device);
    if (on.st != RG_OK) return on.st;
    const Call c{d_base, d_queries, bstride, qstride, nb, nq, dim, id_base, scale, d_targets, static_cast<char *>(d_work), (hipStream_t)stream};
    auto run = dtype == RG_DTYPE_F32 ? shard<RG_DTYPE_F32> : dtype == RG_DTYPE_F16 ? shard<RG_DTYPE_F16> : shard<RG_DTYPE_BF16>;
    return run(c, d_rest, d_own, d_lse, d_loss, d_mean);
}

rg_status rg_softmax_merge_dev(const float *d_rest_in, const float *d_own_in, uint32_t nlists, uint32_t nq, const uint32_t *d_targets,
                               float *d_lse, float *d_loss, int device, void *stream) {
    if (nlists == 0) return set_error(RG_ERR_ARG, "nlists must be positive");
    if (nq > kMaxQueries) return set_error(RG_ERR_ARG, "softmax over a base: at most 2^24 - 1 queries");
    if (nq == 0) return RG_OK;
    if (!d_rest_in || !d_own_in || !d_targets || !d_lse || !d_loss) return set_error(RG_ERR_ARG, "null argument");
    OnDevice on(device);
    if (on.st != RG_OK) return on.st;
    hipLaunchKernelGGL(rg_softmax_merge_kernel, dim3((nq + 255) / 256), dim3(256), 0, (hipStream_t)stream, d_rest_in, d_own_in, nlists, nq, d_targets, d_lse, d_loss);
    RG_HIP(hipGetLastError());
    return RG_OK;
}

rg_status rg_softmax_grad_dev(const void *d_base, uint32_t nb, uint64_t bstride, const void *d_queries, uint32_t nq, uint64_t qstride,
                              uint32_t dim, int dtype, float scale, const uint32_t *d_targets, uint32_t id_base, const float *d_lse,
                              const float *d_loss, const float *d_rest, const float *d_mean, const float *d_weights, void *d_dq,
                              uint64_t dqstride, void *d_db, uint64_t dbstride, void *d_work, uint64_t work_bytes, int device,
                              void *stream) {
    rg_status st = check_call(nb, d_base, bstride, nq, d_queries, qstride, dim, dtype, scale, id_base);
    if (st == RG_OK && d_dq) st = check_rows(d_dq, nq, dqstride, dim, dtype, "gradient of the queries");
    if (st == RG_OK && d_db) st = check_rows(d_db, nb, dbstride, dim, dtype, "gradient of the base");
    if (st != RG_OK) return st;
    if (nq && (!d_targets || !d_lse || !d_loss || !d_weights || (d_dq && (!d_mean || !d_rest)))) return set_error(RG_ERR_ARG, "null argument");
    st = check_scratch(d_work, work_bytes, scratch_of(kRows, d_db ? nb : 0, nq, dim, dtype));
    if (st != RG_OK) return st;
    OnDevice on(device);
    if (on.st != RG_OK) return on.st;
    const Call c{d_base, d_queries, bstride, qstride, nb, nq, dim, id_base, scale, d_targets, static_cast<char *>(d_work), (hipStream_t)stream};
    auto run = dtype == RG_DTYPE_F32 ? grad<RG_DTYPE_F32> : dtype == RG_DTYPE_F16 ? grad<RG_DTYPE_F16> : grad<RG_DTYPE_BF16>;
    return run(c, d_lse, d_loss, d_rest, d_mean, d_weights, d_dq, dqstride, d_db, dbstride);
}

}  // extern "C"
