// Channels-last GroupNorm (+SiLU) and its gradient: choice of kernel.
#include "common.cuh"
#include "gn_cl_internal.h"

#include <algorithm>
#include <initializer_list>

namespace sdfl {

namespace {

bool vectors_ok(const void *a, const void *b, const void *c) {
    return aligned(a, 16) && aligned(b, 16) && aligned(c, 16);
}

// Plans of recent shapes, per host thread: working one out takes 1-2 us, a tenth of a small call.
struct PlanKey {
    int64_t batch, channels, hw, groups;
    int dtype, flags, sms;                             // flags: 1 pack, 2 backward, 4 checkpoint as the source
    bool operator==(const PlanKey &o) const {
        return batch == o.batch && channels == o.channels && hw == o.hw && groups == o.groups && dtype == o.dtype &&
               flags == o.flags && sms == o.sms;
    }
};
struct PlanEntry {
    PlanKey key{};
    bool used = false, ok = false;
    GnClTeamPlan plan{};
};

bool find_plan(const GnClShape &s, bool pack, bool backward, bool ckpt, GnClTeamPlan *p) {
    thread_local PlanEntry memo[64];
    const PlanKey key{s.batch, s.channels, s.hw, s.groups, s.dtype, (pack ? 1 : 0) | (backward ? 2 : 0) | (ckpt ? 4 : 0),
                      sm_count()};
    uint64_t h = 0;
    for (const uint64_t v : {static_cast<uint64_t>(key.batch), static_cast<uint64_t>(key.channels), static_cast<uint64_t>(key.hw),
                             static_cast<uint64_t>(key.groups), static_cast<uint64_t>(key.dtype * 8 + key.flags)})
        h = (h ^ v) * 0x9E3779B97F4A7C15ull;
    PlanEntry &e = memo[h >> 58];
    if (!e.used || !(e.key == key)) {
        e.used = false;
        e.ok = gn_cl_team_plan(s, pack, backward, ckpt, &e.plan);
        e.key = key;
        e.used = true;
    }
    *p = e.plan;
    return e.ok;
}

}  // namespace

// Which kernel a call takes also depends on its pointers, so the workspace holds the largest.
size_t gn_cl_workspace_bytes(const GnClShape &s, bool backward) {
    size_t bytes = gn_cl_split_workspace_bytes(s, backward);
    GnClTeamPlan p;
    for (int kept = 0; kept < 2; ++kept)
        if (find_plan(s, !backward && kept, backward, backward && kept, &p))
            bytes = std::max(bytes, gn_cl_team_workspace_bytes(s, p, backward));
    return bytes;
}

// Teams need all of their blocks on the device at once; where it has no room for them, several launches do the same.
namespace {

bool no_room(cudaError_t err) {
    if (err != cudaErrorCooperativeLaunchTooLarge) return false;
    (void)cudaGetLastError();
    return true;
}

}  // namespace

cudaError_t gn_cl_forward_launch(const GnClShape &s, const GnClForward &a, void *ws, cudaStream_t stream) {
    const bool vectors = vectors_ok(a.in, a.out, nullptr);
    GnClTeamPlan p;
    if (a.codes && vectors && aligned(a.codes, s.dtype == kF32 ? 4 : 8) && find_plan(s, true, false, false, &p)) {
        const cudaError_t err = gn_cl_team_forward(s, p, a, ws, stream);
        if (!no_room(err)) return err;
    }
    GnClForward norm = a;
    if (a.codes) {                                     // two steps, the checkpoint first: out may be in
        const cudaError_t err = ckpt_pack_launch(a.in, a.codes, a.scales, s.batch * s.hw, s.channels, s.dtype, stream);
        if (err != cudaSuccess) return err;
        norm.codes = nullptr;
        norm.scales = nullptr;
    }
    if (vectors && find_plan(s, false, false, false, &p)) {
        const cudaError_t err = gn_cl_team_forward(s, p, norm, ws, stream);
        if (!no_room(err)) return err;
    }
    return gn_cl_split_forward(s, norm, ws, stream);
}

cudaError_t gn_cl_backward_launch(const GnClShape &s, const GnClBackward &a, void *ws, cudaStream_t stream) {
    GnClTeamPlan p;
    if (vectors_ok(a.in, a.grad_out, a.grad_in) && aligned(a.codes, 16) &&
        find_plan(s, false, true, a.codes != nullptr, &p)) {
        const cudaError_t err = gn_cl_team_backward(s, p, a, ws, stream);
        if (!no_room(err)) return err;
    }
    return gn_cl_split_backward(s, a, ws, stream);
}

}  // namespace sdfl
