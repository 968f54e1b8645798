// RMSNorm of queries' and keys' heads with the rotation of one position a token
// (the kernels of mhc_qk.h); calls with several axes go on to qk_axes.hip.
#include "mhc_qk.h"

namespace mhc {

hipError_t launch_qk_norm_rope_fwd(int dt, int fmt, const QkArgs& a, hipStream_t s) {
    return a.axes > 1 ? launch_qk_axes_fwd(dt, fmt, a, s) : qk_fwd_launch<false>(dt, fmt, a, s);
}

int qk_norm_rope_bwd_rows(const QkArgs& a) {
    const dim3 g = qk_bwd_dims(a);
    return (int)(g.x * g.y);
}

hipError_t launch_qk_norm_rope_bwd(int dt, int fmt, const QkArgs& a, float* dw_part, hipStream_t s) {
    return a.axes > 1 ? launch_qk_axes_bwd(dt, fmt, a, dw_part, s) : qk_bwd_launch<false>(dt, fmt, a, dw_part, s);
}

}  // namespace mhc
