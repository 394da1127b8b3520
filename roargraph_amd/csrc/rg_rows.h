// rg_rows.h -- what the operators over typed rows (rg_softmax*.hip, rg_q4.hip) share: element types, the guard around the current device.
#pragma once
#include <hip/hip_runtime.h>

#include <string>

#include "rg.h"
#include "rg_internal.h"

#define RG_HIP(expr)                                                                                   \
    do {                                                                                               \
        hipError_t e_ = (expr);                                                                        \
        if (e_ != hipSuccess)                                                                          \
            return set_error(RG_ERR_DEVICE, std::string(#expr) + ": " + hipGetErrorString(e_));        \
    } while (0)

namespace rg {

template <int DT> struct Elem;
template <> struct Elem<RG_DTYPE_F32> { typedef float T; };
template <> struct Elem<RG_DTYPE_F16> { typedef _Float16 T; };
template <> struct Elem<RG_DTYPE_BF16> { typedef __bf16 T; };

inline bool known_dtype(int dtype) { return dtype == RG_DTYPE_F32 || dtype == RG_DTYPE_F16 || dtype == RG_DTYPE_BF16; }
inline uint32_t elem_bytes(int dtype) { return dtype == RG_DTYPE_F32 ? 4 : 2; }

// ---- fp32 rows as two fp16 halves, scaled by a power of two of their own
// exponent e of a row: 2^-e brings its largest value to [2^14, 2^15), the top of fp16's range, so that elements down to 2^-17 of it keep their
// 22 bits and none is off by more than 2^-39 of it (brought to [1, 2), the second halves of elements below 2^-3 of it were subnormal, off by 2^-25
// of it: two queries on 1630 x 177, elements of a gradient by 3e-5 of themselves).
// Rows below 2^-112 are brought as far as 2^126 does.
__device__ __forceinline__ int row_exponent(float top) {
    const uint32_t u = __float_as_uint(top) >> 23;
    return u >= 255 || top == 0.0f ? 0 : max((int)max(u, 1u) - 127 - 14, -126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

// a row that is not finite keeps the signs of its infinities (and its NaN) and nothing else; its logits are multiplied by infinity
__device__ __forceinline__ float row_factor(float top, int e) { return top < INFINITY ? pow2(e) : INFINITY; }

// makes `device` current for a call, and the caller's device current again afterwards
struct OnDevice {
    int before = -1;
    rg_status st = RG_OK;
    explicit OnDevice(int device) {
        int n = 0;
        if (hipGetDeviceCount(&n) != hipSuccess || n <= 0)
            st = set_error(RG_ERR_DEVICE, "no HIP device visible: the gfx950 path cannot run (there is no CPU fallback)");
        else if (device < 0 || device >= n)
            st = set_error(RG_ERR_ARG, "no such device");
        else if (hipGetDevice(&before) != hipSuccess || (before != device && hipSetDevice(device) != hipSuccess))
            st = set_error(RG_ERR_DEVICE, "cannot use the device");
        if (st != RG_OK || before == device) before = -1;
    }
    ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
};

}  // namespace rg
