// instantiations of the softmax pass: f32 rows, mode kMean
#include "rg_softmax_pass.h"

namespace rg {
const void *softmax_kernel_f32_mean(int ks) {
    switch (ks) {
#define RG_KS(K) case K: return reinterpret_cast<const void *>(rg_softmax_pass_kernel<RG_DTYPE_F32, K, kMean>);
        RG_KS(2) RG_KS(4) RG_KS(7) RG_KS(8) RG_KS(12) RG_KS(16) RG_KS(24)
#undef RG_KS
        default: return reinterpret_cast<const void *>(rg_softmax_pass_kernel<RG_DTYPE_F32, 32, kMean>);
    }
}
}  // namespace rg
