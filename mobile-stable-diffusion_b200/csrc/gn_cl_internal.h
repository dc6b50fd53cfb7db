// Interfaces between the translation units of the channels-last GroupNorm (dispatch in gn_cl.cu).
#pragma once

#include "kernels.h"

namespace sdfl {

// ---- any shape and alignment, three or four launches (gn_cl_split.cu) ----------------------------
size_t gn_cl_split_workspace_bytes(const GnClShape &s, bool backward);
cudaError_t gn_cl_split_forward(const GnClShape &s, const GnClForward &a, void *ws, cudaStream_t stream);
cudaError_t gn_cl_split_backward(const GnClShape &s, const GnClBackward &a, void *ws, cudaStream_t stream);

}  // namespace sdfl
