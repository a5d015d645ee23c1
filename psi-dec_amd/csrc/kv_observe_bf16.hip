// Instantiates the gfx950 observation kernels for bf16 K.
#include "kv_observe_kernel.h"

namespace psi {
void launch_observe_bf16(psi_hip_ctx* ctx, const ObserveArgs& a, uint32_t window_rows) {
    launch_observe<BF16Tag>(ctx, a, window_rows);
}
}  // namespace psi
