// rg_softmax.hip -- softmax cross entropy over all rows of a base, and its gradients, without storing the logits.
//
// With z_ij = scale <q_i, b_j> (kept in units of log 2: z2 = z log2 e, so that every exponential is one v_exp_f32):
//
//   statistics + mean   for each query i one pass over the rows j != target with a running reference M, sum l and sum O:
//                         P = 2^(z2 - M),  l += P,  O += P b_j          rest = ln 2 (M + log2 l),  mean = O / l
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

constexpr uint32_t kMaxDim = 1024;
constexpr uint32_t kCUs = 256;             // MI355X; the workspace query needs no device
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ bool target_here(uint32_t t, uint32_t id_base, uint32_t nb) { return t != kNoTarget && t >= id_base && t - id_base < nb; }

// log(1 + e^d) without overflow: loss of a target d below the others' log sum
__device__ __forceinline__ float softplus(float d) { return d > 15.0f ? d + log1pf(expf(-d)) : log1pf(expf(d)); }

// joins the slots of a query: rest, target logit, lse, loss, mean of the others.  One workgroup per query.
__global__ void __launch_bounds__(256) rg_softmax_join_kernel(const float4 *ml, const float *o, uint32_t opitch, uint32_t nslots, uint32_t nq, uint32_t dim, uint32_t nb, uint32_t id_base, const float *own2,
                                                              const uint32_t *targets, float *rest, float *own, float *lse, float *loss, float *mean) {
    const uint32_t i = blockIdx.x, tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    __shared__ float red[8];
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
    const bool none = M == kNothing;       // no other row than the target
    float l = 0.0f;
    for (uint32_t s = tid; s < nslots; s += 256) {
        const float4 v = ml[(size_t)s * nq + i];
        l += v.y * exp2f(v.x - M);
    }
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
    __syncthreads();
    if (lane == 0) red[wave] = l;
    __syncthreads();
    l = red[0] + red[1] + red[2] + red[3];
    if (tid == 0) {
        const uint32_t t = targets[i];
        const bool here = target_here(t, id_base, nb);
        const float r = none ? -INFINITY : (M + log2f(l)) * kLn2;
        const float z = here ? own2[i] * kLn2 : -INFINITY;
        const float v = here ? softplus(r - z) : t == kNoTarget ? 0.0f : INFINITY;
        rest[i] = r;
        own[i] = z;
        if (lse) lse[i] = here ? z + v : r;
        if (loss) loss[i] = v;
    }
    if (mean) {
        const float f = none ? 0.0f : exp2f(Mo - M) / l;
        for (uint32_t k = tid; k < dim; k += 256) {
            float s = 0.0f;
            for (uint32_t e = 0; e < nslots; ++e) s = fmaf(exp2f(ml[(size_t)e * nq + i].z - Mo), o[((size_t)e * nq + i) * opitch + k], s);
            mean[(size_t)i * dim + k] = s * f;
        }
    }
}

__global__ void __launch_bounds__(256) rg_softmax_merge_kernel(const float *rest_in, const float *own_in, uint32_t nlists, uint32_t nq, const uint32_t *targets, float *lse, float *loss) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= nq) return;
    float m = -INFINITY, own = -INFINITY;
    for (uint32_t s = 0; s < nlists; ++s) {
        m = fmaxf(m, rest_in[(size_t)s * nq + i]);
        own = fmaxf(own, own_in[(size_t)s * nq + i]);
    }
    float l = 0.0f;
    const float ref = m == -INFINITY ? 0.0f : m;
    for (uint32_t s = 0; s < nlists; ++s) l += expf(rest_in[(size_t)s * nq + i] - ref);
    const float r = m == -INFINITY ? -INFINITY : m + logf(l);
    const float v = targets[i] == kNoTarget ? 0.0f : own == -INFINITY ? INFINITY : softplus(r - own);
    lse[i] = targets[i] == kNoTarget || own == -INFINITY ? r : own + v;
    loss[i] = v;
}

// per query: what the pass over the rows needs of it, and dq.  One wave per query.
template <int DT>
__global__ void __launch_bounds__(64) rg_softmax_dq_kernel(const void *base, uint64_t bstride, uint32_t nb, uint32_t id_base, uint32_t nq, uint32_t dim, float scale,
                                                           const uint32_t *targets, const float *lse, const float *loss, const float *rest, const float *mean,
                                                           const float *weights, void *dq, uint64_t dqstride, float4 *yparam) {
    typedef typename Elem<DT>::T T;
    const uint32_t i = blockIdx.x, t = targets[i], row = t - id_base;
    const bool here = target_here(t, id_base, nb);
    const float w = t == kNoTarget ? 0.0f : weights[i], miss = here ? -expm1f(-loss[i]) : 0.0f;      // 1 - p_target
    if (yparam && threadIdx.x == 0) {
        const float lw = log2f(fabsf(w));
        yparam[i] = make_float4(t == kNoTarget ? -INFINITY : lw - lse[i] * kLog2e, lw + log2f(miss), w < 0.0f ? -1.0f : 1.0f, __uint_as_float(here ? row : kNoTarget));
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

// the instantiation a width runs in, as the smallest number of 32-element steps that holds it
constexpr int kSteps[] = {2, 4, 7, 8, 12, 16, 24, 32};
int steps_of(uint32_t dim) {
    if (dim > 192 && dim <= 208) return 7;              // (its output blocks end at 208)
    for (int ks : kSteps)
        if (ks != 7 && dim <= 32u * ks) return ks;
    return 32;
}
struct Shape {
    int ks;
    uint32_t xt, nslices, resident, lds;
};
template <int DT, int KS>
Shape shape_at(uint32_t dim) {
    typedef PassCfg<DT, KS> C;
    return Shape{KS, (uint32_t)C::XT, (dim + 16 * C::OB - 1) / (16 * C::OB), kCUs * std::min<uint32_t>(C::WPS, 160 * 1024 / C::LDS), (uint32_t)C::LDS};
}
template <int DT>
Shape shape_dt(uint32_t dim) {
    switch (steps_of(dim)) {
        case 2: return shape_at<DT, 2>(dim);
        case 4: return shape_at<DT, 4>(dim);
        case 7: return shape_at<DT, 7>(dim);
        case 8: return shape_at<DT, 8>(dim);
        case 12: return shape_at<DT, 12>(dim);
        case 16: return shape_at<DT, 16>(dim);
        case 24: return shape_at<DT, 24>(dim);
        default: return shape_at<DT, 32>(dim);
    }
}
Shape shape_of(int dtype, uint32_t dim, bool sums) {
    Shape s = dtype == RG_DTYPE_F32 ? shape_dt<RG_DTYPE_F32>(dim) : dtype == RG_DTYPE_F16 ? shape_dt<RG_DTYPE_F16>(dim) : shape_dt<RG_DTYPE_BF16>(dim);
    if (!sums) s.nslices = 1;
    return s;
}

// how a pass is cut: slots = pieces of y whose partial results are joined afterwards.  As many as give every workgroup place of the device
// the same work, of at least four tiles.
struct Plan {
    Shape shape;
    uint32_t nsplit, rows_per_split;
    uint64_t grid;
};
Plan plan_of(int dtype, uint32_t dim, uint32_t nx, uint32_t ny, bool sums) {
    Plan p;
    p.shape = shape_of(dtype, dim, sums);
    const uint64_t nt = std::max<uint64_t>(1, ((uint64_t)nx + p.shape.xt - 1) / p.shape.xt) * p.shape.nslices, places = p.shape.resident;
    const uint32_t most = std::max(1u, ny / 128);
    uint32_t best = 1;
    double best_use = 0;
    for (uint32_t n = 1; n <= most && n * nt <= 2 * places + nt; ++n) {
        const uint64_t rounds = (n * nt + places - 1) / places;
        const double use = (double)(n * nt) / (double)(rounds * places) - 0.01 * (double)(rounds > 1 ? rounds - 1 : 0);
        if (use > best_use + 0.02) { best_use = use; best = n; }
    }
    p.rows_per_split = ((std::max(ny, 1u) + best - 1) / best + 31) / 32 * 32;
    p.nsplit = std::max(1u, (ny + p.rows_per_split - 1) / p.rows_per_split);
    p.grid = nt * p.nsplit;
    return p;
}

uint32_t opitch_of(uint32_t dim) { return (dim + 15) / 16 * 16; }
uint64_t up256(uint64_t n) { return (n + 255) / 256 * 256; }

// the instantiations of a type and mode live in a unit of their own (rg_softmax_inst_*.hip)
rg_status launch_softmax_pass(int dtype, int mode, int ks, const PassArgs &A, uint64_t grid, uint32_t lds, hipStream_t s) {
    if (grid > 0xffffffull) return set_error(RG_ERR_ARG, "softmax over a base: too many rows for one launch");
    typedef const void *(*Pick)(int);
    static const Pick pick[3][3] = {{softmax_kernel_f32_stats, softmax_kernel_f32_mean, softmax_kernel_f32_rows},
                                    {softmax_kernel_f16_stats, softmax_kernel_f16_mean, softmax_kernel_f16_rows},
                                    {softmax_kernel_bf16_stats, softmax_kernel_bf16_mean, softmax_kernel_bf16_rows}};
    const void *kern = pick[dtype][mode](ks);
    RG_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    void *args[] = {const_cast<PassArgs *>(&A)};
    RG_HIP(hipLaunchKernel(kern, dim3((uint32_t)grid), dim3(256), args, lds, s));
    return RG_OK;
}

// bytes of the three parts of the scratch: M and l of the slots, sums of the slots, and per query the target's logit or the parameters
struct Scratch {
    uint64_t ml, o, y;
    uint64_t total() const { return ml + o + y; }
};
Scratch scratch_of(int what, uint32_t nb, uint32_t nq, uint32_t dim, int dtype) {
    const uint32_t nx = what == RG_SOFTMAX_GRAD ? nb : nq, ny = what == RG_SOFTMAX_GRAD ? nq : nb;
    const Plan p = plan_of(dtype, dim, nx, ny, what != RG_SOFTMAX_STATS);
    Scratch s;
    const bool pieces = what != RG_SOFTMAX_GRAD || p.nsplit > 1;
    s.ml = pieces ? up256((uint64_t)p.nsplit * nx * 16) : 0;
    s.o = pieces && what != RG_SOFTMAX_STATS ? up256((uint64_t)p.nsplit * nx * opitch_of(dim) * 4) : 0;
    s.y = up256((uint64_t)nq * (what == RG_SOFTMAX_GRAD ? 16 : 4));
    return s;
}

rg_status check_shapes(uint32_t nb, uint32_t nq, uint32_t dim, int dtype) {
    if (!known_dtype(dtype)) return set_error(RG_ERR_ARG, "unknown dtype");
    if (dim == 0 || dim > kMaxDim) return set_error(RG_ERR_ARG, "softmax over a base: dim must be in [1, 1024]");
    if (nb > 0x7fffffffu || nq > 0x7fffffffu) return set_error(RG_ERR_ARG, "softmax over a base: at most 2^31 - 1 rows and queries");
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
    if (!std::isfinite(scale)) return set_error(RG_ERR_ARG, "the scale must be finite");
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
    const Plan p = plan_of(DT, c.dim, c.nq, c.nb, mean != nullptr);
    const Scratch sc = scratch_of(mean ? RG_SOFTMAX_MEAN : RG_SOFTMAX_STATS, c.nb, c.nq, c.dim, DT);
    float *own2 = reinterpret_cast<float *>(c.work + sc.ml + sc.o);
    PassArgs A{c.queries, c.base, c.qstride, c.bstride, c.nq, c.nb, c.dim, c.scale * kLog2e, p.nsplit, p.rows_per_split, p.shape.nslices, opitch_of(c.dim),
               reinterpret_cast<float4 *>(c.work), reinterpret_cast<float *>(c.work + sc.ml), c.targets, c.id_base, own2, nullptr, nullptr, 0, 0.0f};
    rg_status st = launch_softmax_pass(DT, mean ? kMean : kStats, p.shape.ks, A, p.grid, p.shape.lds, c.s);
    if (st != RG_OK) return st;
    hipLaunchKernelGGL(rg_softmax_join_kernel, dim3(c.nq), dim3(256), 0, c.s, A.ml, A.o, A.opitch, p.nsplit, c.nq, c.dim, c.nb, c.id_base, own2, c.targets, rest, own, lse, loss, mean);
    RG_HIP(hipGetLastError());
    return RG_OK;
}

template <int DT>
rg_status grad(const Call &c, const float *lse, const float *loss, const float *rest, const float *mean, const float *weights, void *dq, uint64_t dqstride, void *db, uint64_t dbstride) {
    const Plan p = plan_of(DT, c.dim, c.nb, c.nq, true);
    const Scratch sc = scratch_of(RG_SOFTMAX_GRAD, c.nb, c.nq, c.dim, DT);
    float4 *yp = db ? reinterpret_cast<float4 *>(c.work + sc.ml + sc.o) : nullptr;
    if (c.nq) {
        hipLaunchKernelGGL((rg_softmax_dq_kernel<DT>), dim3(c.nq), dim3(64), 0, c.s, c.base, c.bstride, c.nb, c.id_base, c.nq, c.dim, c.scale, c.targets, lse, loss, rest, mean, weights, dq, dqstride, yp);
        RG_HIP(hipGetLastError());
    }
    if (!db || c.nb == 0) return RG_OK;
    PassArgs A{c.base, c.queries, c.bstride, c.qstride, c.nb, c.nq, c.dim, c.scale * kLog2e, p.nsplit, p.rows_per_split, p.shape.nslices, opitch_of(c.dim),
               reinterpret_cast<float4 *>(c.work), reinterpret_cast<float *>(c.work + sc.ml), nullptr, 0, nullptr, yp, db, dbstride, c.scale};
    rg_status st = launch_softmax_pass(DT, kRows, p.shape.ks, A, p.grid, p.shape.lds, c.s);
    if (st != RG_OK || p.nsplit == 1) return st;
    const uint64_t n = (uint64_t)c.nb * c.dim;
    hipLaunchKernelGGL((rg_softmax_db_kernel<DT>), dim3((uint32_t)std::min<uint64_t>((n + 255) / 256, 1u << 20)), dim3(256), 0, c.s, A.ml, A.o, A.opitch, p.nsplit, c.nb, c.dim, c.scale, db, dbstride);
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
    *bytes = scratch_of(what, nb, nq, dim, dtype).total();
    return RG_OK;
}

rg_status rg_softmax_shard_dev(const void *d_base, uint32_t nb, uint64_t bstride, const void *d_queries, uint32_t nq, uint64_t qstride,
                               uint32_t dim, int dtype, float scale, const uint32_t *d_targets, uint32_t id_base, float *d_rest,
                               float *d_own, float *d_lse, float *d_loss, float *d_mean, void *d_work, uint64_t work_bytes, int device,
                               void *stream) {
    rg_status st = check_call(nb, d_base, bstride, nq, d_queries, qstride, dim, dtype, scale, id_base);
    if (st != RG_OK || nq == 0) return st;
    if (!d_targets || !d_rest || !d_own) return set_error(RG_ERR_ARG, "null argument");
    st = check_scratch(d_work, work_bytes, scratch_of(d_mean ? RG_SOFTMAX_MEAN : RG_SOFTMAX_STATS, nb, nq, dim, dtype).total());
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
    st = check_scratch(d_work, work_bytes, scratch_of(RG_SOFTMAX_GRAD, d_db ? nb : 0, nq, dim, dtype).total());
    if (st != RG_OK) return st;
    OnDevice on(device);
    if (on.st != RG_OK) return on.st;
    const Call c{d_base, d_queries, bstride, qstride, nb, nq, dim, id_base, scale, d_targets, static_cast<char *>(d_work), (hipStream_t)stream};
    auto run = dtype == RG_DTYPE_F32 ? grad<RG_DTYPE_F32> : dtype == RG_DTYPE_F16 ? grad<RG_DTYPE_F16> : grad<RG_DTYPE_BF16>;
    return run(c, d_lse, d_loss, d_rest, d_mean, d_weights, d_dq, dqstride, d_db, dbstride);
}

}  // extern "C"
