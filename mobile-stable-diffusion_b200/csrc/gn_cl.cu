// Channels-last GroupNorm (+SiLU) and its gradient: choice of kernel.
#include "common.cuh"
#include "gn_cl_internal.h"

#include <algorithm>

namespace sdfl {

namespace {

inline bool aligned(const void *p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

bool vectors_ok(const void *a, const void *b, const void *c) {
    return aligned(a, 16) && aligned(b, 16) && aligned(c, 16);
}


}  // namespace

// Which kernel a call takes also depends on its pointers, so the workspace holds the largest.
size_t gn_cl_workspace_bytes(const GnClShape &s, bool backward) {
    size_t bytes = gn_cl_split_workspace_bytes(s, backward);
    GnClTeamPlan p;
    for (int kept = 0; kept < 2; ++kept)
        if (gn_cl_team_plan(s, !backward && kept, backward, backward && kept, &p))
            bytes = std::max(bytes, gn_cl_team_workspace_bytes(s, p, backward));
    return bytes;
}

cudaError_t gn_cl_forward_launch(const GnClShape &s, const GnClForward &a, void *ws, cudaStream_t stream) {
    const bool vectors = vectors_ok(a.in, a.out, nullptr);
    GnClTeamPlan p;
    if (a.codes && vectors && aligned(a.codes, s.dtype == kF32 ? 4 : 8) && gn_cl_team_plan(s, true, false, false, &p))
        return gn_cl_team_forward(s, p, a, ws, stream);
    GnClForward norm = a;
    if (a.codes) {                                     // two steps, the checkpoint first: out may be in
        const cudaError_t err = ckpt_pack_launch(a.in, a.codes, a.scales, s.batch * s.hw, s.channels, s.dtype, stream);
        if (err != cudaSuccess) return err;
        norm.codes = nullptr;
        norm.scales = nullptr;
    }
    if (vectors && gn_cl_team_plan(s, false, false, false, &p)) return gn_cl_team_forward(s, p, norm, ws, stream);
    return gn_cl_split_forward(s, norm, ws, stream);
}

cudaError_t gn_cl_backward_launch(const GnClShape &s, const GnClBackward &a, void *ws, cudaStream_t stream) {
    GnClTeamPlan p;
    if (vectors_ok(a.in, a.grad_out, a.grad_in) && aligned(a.codes, 16) &&
        gn_cl_team_plan(s, false, true, a.codes != nullptr, &p))
        return gn_cl_team_backward(s, p, a, ws, stream);
    return gn_cl_split_backward(s, a, ws, stream);
}

}  // namespace sdfl
