// instantiations of the softmax pass: f32 rows, gradient of the rows
#include "rg_softmax_wide.h"

namespace rg {

SoftmaxKernel softmax_wide_f32_rows(int ks) {
    switch (ks) {
#define RG_KS(K) case K: return {reinterpret_cast<const void *>(rg_softmax_wide_kernel<RG_DTYPE_F32, K, kRows>), (uint32_t)WideCfg<RG_DTYPE_F32, K, kRows>::XT, (uint32_t)WideCfg<RG_DTYPE_F32, K, kRows>::OB, (uint32_t)WideCfg<RG_DTYPE_F32, K, kRows>::LDS, (uint32_t)WideCfg<RG_DTYPE_F32, K, kRows>::WPS, (uint32_t)WideCfg<RG_DTYPE_F32, K, kRows>::NT};
        RG_KS(2) RG_KS(4) RG_KS(7) RG_KS(8) RG_KS(12) RG_KS(16) RG_KS(24) RG_KS(32)
#undef RG_KS
        default: return {};
    }
}

}  // namespace rg
