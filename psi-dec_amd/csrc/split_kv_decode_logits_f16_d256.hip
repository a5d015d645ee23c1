// Instantiates the gfx950 decode map that stores its logits as well, for f16 K/V, head_dim 256 (all group sizes).
#include "split_kv_decode_kernel.h"

namespace psi {
int launch_decode_logits_f16_d256(psi_hip_ctx* ctx, const Geometry& g, const MapArgs& a) {
    return launch_decode_map_group<F16Tag, 256, true>(ctx, g, a);
}
}  // namespace psi
