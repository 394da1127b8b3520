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

// one wave per row and query
template <int DT>
__global__ void __launch_bounds__(256) rg_q4_score_kernel(const uint8_t *codes, uint64_t cstride, const uint16_t *scales, const uint16_t *mins, uint64_t sstride, uint32_t nb, uint32_t dim,
                                                          uint32_t group, const void *queries, uint32_t nq, uint64_t qstride, float *out, uint64_t ostride) {
    typedef typename Elem<DT>::T T;
    const uint32_t lane = threadIdx.x % 64;
    for (uint64_t j = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64; j < nb; j += (uint64_t)gridDim.x * 4)
        for (uint32_t i = 0; i < nq; ++i) {
            float acc = 0.0f;
            for (uint32_t k = lane; k < dim; k += 64) {
                const uint32_t c = codes[j * cstride + k / 2] >> (4 * (k & 1)) & 15u, g = k / group;
                const float s = half_bits(scales[j * sstride + g]);
                const float v = mins ? (float)c * s + half_bits(mins[j * sstride + g]) : (float)((int)c - 8) * s;
                acc = fmaf(v, (float)static_cast<const T *>(queries)[(size_t)i * qstride + k], acc);
            }
            for (int d = 1; d < 64; d <<= 1) acc += __shfl_xor(acc, d);
            if (lane == 0) out[(size_t)i * ostride + j] = acc;
        }
}

rg_status check_form(const void *codes, uint64_t cstride, const void *scales, const void *mins, uint64_t sstride, uint32_t nb, uint32_t dim, uint32_t group) {
    if (group != 32 && group != 64 && group != 128) return set_error(RG_ERR_ARG, "4-bit base: groups of 32, 64 or 128 elements");
    if (dim == 0 || dim > kMaxDim) return set_error(RG_ERR_ARG, "4-bit base: dim must be in [1, 4096]");
    if (nb > 0x7fffffffu) return set_error(RG_ERR_ARG, "4-bit base: at most 2^31 - 1 rows");
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
    auto kern = dtype == RG_DTYPE_F32 ? rg_q4_score_kernel<RG_DTYPE_F32> : dtype == RG_DTYPE_F16 ? rg_q4_score_kernel<RG_DTYPE_F16> : rg_q4_score_kernel<RG_DTYPE_BF16>;
    hipLaunchKernelGGL(kern, dim3(std::min<uint32_t>((nb + 3) / 4, 65536u)), dim3(256), 0, (hipStream_t)stream, d_codes, cstride, d_scales, d_mins, sstride, nb, dim, group, d_queries, nq, qstride,
                       d_out, ostride);
    RG_HIP(hipGetLastError());
    return RG_OK;
}

}  // extern "C"
