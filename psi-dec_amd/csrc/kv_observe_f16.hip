// Instantiates the gfx950 observation kernels for f16 K.
#include "kv_observe_kernel.h"

namespace psi {
void launch_observe_f16(psi_hip_ctx* ctx, const ObserveArgs& a, uint32_t window_rows) {
    launch_observe<F16Tag>(ctx, a, window_rows);
}
}  // namespace psi
