// instantiations of the softmax pass: f32 rows, statistics and mean rows
#include "rg_softmax_thin.h"
#include "rg_softmax_wide.h"

namespace rg {

SoftmaxKernel softmax_wide_f32_mean(int ks) {
    switch (ks) {
#define RG_KS(K) case K: return {reinterpret_cast<const void *>(rg_softmax_wide_kernel<RG_DTYPE_F32, K, kMean>), (uint32_t)WideCfg<RG_DTYPE_F32, K, kMean>::XT, (uint32_t)WideCfg<RG_DTYPE_F32, K, kMean>::OB, (uint32_t)WideCfg<RG_DTYPE_F32, K, kMean>::LDS, (uint32_t)WideCfg<RG_DTYPE_F32, K, kMean>::WPS, (uint32_t)WideCfg<RG_DTYPE_F32, K, kMean>::NT};
        RG_KS(2) RG_KS(4) RG_KS(7) RG_KS(8) RG_KS(12) RG_KS(16) RG_KS(24) RG_KS(32)
#undef RG_KS
        default: return {};
    }
}

SoftmaxKernel softmax_thin_f32_mean(int ks) {
    switch (ks) {
#define RG_KS(K) case K: return {reinterpret_cast<const void *>(rg_softmax_thin_kernel<RG_DTYPE_F32, K, kMean>), (uint32_t)ThinCfg<RG_DTYPE_F32, K>::XT, (uint32_t)ThinCfg<RG_DTYPE_F32, K>::OB, (uint32_t)ThinCfg<RG_DTYPE_F32, K>::LDS, (uint32_t)ThinCfg<RG_DTYPE_F32, K>::WPS, 256u};
        RG_KS(2) RG_KS(4) RG_KS(7) RG_KS(8) RG_KS(12) RG_KS(16)
#undef RG_KS
        default: return {};
    }
}

}  // namespace rg
