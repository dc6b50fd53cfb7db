// Interfaces between the translation units of the channels-last GroupNorm (dispatch in gn_cl.cu).
#pragma once

#include "kernels.h"

namespace sdfl {

// ---- any shape and alignment, three or four launches (gn_cl_split.cu) ----------------------------
size_t gn_cl_split_workspace_bytes(const GnClShape &s, bool backward);
cudaError_t gn_cl_split_forward(const GnClShape &s, const GnClForward &a, void *ws, cudaStream_t stream);
cudaError_t gn_cl_split_backward(const GnClShape &s, const GnClBackward &a, void *ws, cudaStream_t stream);

// ---- one persistent launch for whole 16-byte vectors: channels a multiple of the vector, aligned buffers,
// ---- groups no wider than half a thread block's columns (gn_cl_team.cu) ----------------------------
struct GnClTeamPlan {
    int vec;               // elements per column: a 16-byte vector
    int cols, rows;        // columns of a slice; rows of threads in a block
    int rounds;            // rows per thread and chunk
    int slices;            // an image's channels / slice channels
    int slice_teams;       // teams side by side on the slices of an image
    int image_teams;       // teams side by side on images
    int members;           // thread blocks per team
    int slice_groups;      // groups of a slice
    int stagger;           // the odd one of two teams starts behind the even one's first pass
    int resident;          // one item per team, which fits the ring: read once
    int cluster;           // a team is a thread-block cluster, one item per team
};
// false: no plan for this shape.  pack: the forward pass also writes a checkpoint; ckpt: the
// backward pass reads one.
bool gn_cl_team_plan(const GnClShape &s, bool pack, bool backward, bool ckpt, GnClTeamPlan *p);
size_t gn_cl_team_shared_bytes(const GnClTeamPlan &p, bool backward, bool ckpt);    // dynamic, of a thread block
size_t gn_cl_team_workspace_bytes(const GnClShape &s, const GnClTeamPlan &p, bool backward);
cudaError_t gn_cl_team_forward(const GnClShape &s, const GnClTeamPlan &p, const GnClForward &a, void *ws, cudaStream_t stream);
cudaError_t gn_cl_team_backward(const GnClShape &s, const GnClTeamPlan &p, const GnClBackward &a, void *ws,
                                cudaStream_t stream);

}  // namespace sdfl
