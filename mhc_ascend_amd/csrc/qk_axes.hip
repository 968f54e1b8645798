// RMSNorm of queries' and keys' heads with the rotation of positions on several
// axes: the kernels of mhc_qk.h with a table row an axis.  8192 tokens x 40 heads of
// 128 bf16 on three axes: forward 37 us (4.5 TB/s), backward 56 (4.5), as with one
// (37 and 55); with an int8 checkpoint 46 and 56 (45 and 54).
#include "mhc_qk.h"

namespace mhc {

// Whether the pairs of every lane's piece are of one axis.
static int qk_whole(const QkArgs& a) {
    const QkTiling t = qk_tiling(a.D, a.R, a.interleaved);
    if (t.v == 0 || a.interleaved || a.dealt) return 0;
    for (int s = 0; s + 1 < a.axes; ++s)
        if (a.part[s] % t.v != 0) return 0;
    return 1;
}

hipError_t launch_qk_axes_fwd(int dt, int fmt, QkArgs a, hipStream_t s) {
    a.whole = qk_whole(a);
    return qk_fwd_launch<true>(dt, fmt, a, s);
}

hipError_t launch_qk_axes_bwd(int dt, int fmt, QkArgs a, float* dw_part, hipStream_t s) {
    a.whole = qk_whole(a);
    return qk_bwd_launch<true>(dt, fmt, a, dw_part, s);
}

}  // namespace mhc
