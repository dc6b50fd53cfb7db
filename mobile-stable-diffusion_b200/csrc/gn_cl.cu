// Channels-last GroupNorm (+SiLU) and its gradient: choice of kernel.
#include "gn_cl_internal.h"

namespace sdfl {

size_t gn_cl_workspace_bytes(const GnClShape &s, bool backward) { return gn_cl_split_workspace_bytes(s, backward); }

cudaError_t gn_cl_forward_launch(const GnClShape &s, const GnClForward &a, void *ws, cudaStream_t stream) {
    if (a.codes) {
        // before the norm: out may be in
        const cudaError_t err = ckpt_pack_launch(a.in, a.codes, a.scales, s.batch * s.hw, s.channels, s.dtype, stream);
        if (err != cudaSuccess) return err;
    }
    return gn_cl_split_forward(s, a, ws, stream);
}

cudaError_t gn_cl_backward_launch(const GnClShape &s, const GnClBackward &a, void *ws, cudaStream_t stream) {
    return gn_cl_split_backward(s, a, ws, stream);
}

}  // namespace sdfl
