// Plans of the channels-last GroupNorm over a sweep of shapes: the grid of a plan whose blocks wait for one another has
// to fit the device at once, and of a staggered plan, whose blocks number themselves by two on every SM, no third block may
// fit an SM, whatever the kernel's registers.  Needs no device (148 SMs are assumed without one).  Prints the plans that do not hold.
#include "../../mobile-stable-diffusion_b200/csrc/gn_cl_internal.h"

#include <algorithm>
#include <cstdio>

// An SM's shared memory, and what a block takes of it: its dynamic part, 128 bytes static (from the compiler's
// report), 1 KB reserved, in units of 128 bytes.
static int blocks_of_sm(size_t dynamic) {
    const size_t block = (dynamic + 128 + 127) / 128 * 128 + 1024;
    return static_cast<int>(228 * 1024 / block);
}

int main() {
    using namespace sdfl;
    const int64_t batches[] = {1, 2, 3, 4, 8, 16}, pixels[] = {64, 1000, 3001, 4096, 6000, 16384, 65536, 262144};
    const int64_t widths[] = {1, 2, 3, 4, 5, 8, 10, 16, 20, 25, 32, 40, 64, 80, 96, 120, 128, 160, 192, 200, 256, 320, 384, 400, 512, 640, 768, 1000, 1024, 1280};
    const int64_t groups[] = {1, 2, 3, 4, 8, 10, 16, 25, 32};
    long plans = 0, wrong = 0;
    for (int64_t b : batches) for (int64_t hw : pixels) for (int64_t w : widths) for (int64_t g : groups)
    for (int dtype = 0; dtype <= 2; ++dtype) for (int kind = 0; kind < 4; ++kind) {
        if (w * g > 5120 || b * hw * w * g > (1ll << 31)) continue;
        const bool backward = kind >= 2, pack = kind == 1, ckpt = kind == 3;
        GnClShape s{b, w * g, hw, g, dtype, 1e-5f, 1};
        GnClTeamPlan p;
        if (!gn_cl_team_plan(s, pack, backward, ckpt, &p)) continue;
        ++plans;
        if (p.cluster || p.members == 1) continue;
        const int fit = blocks_of_sm(gn_cl_team_shared_bytes(p, backward, ckpt));
        const int64_t grid = static_cast<int64_t>(p.slice_teams) * p.image_teams * p.members;
        if (grid > std::min(fit, 2) * 148 || (p.stagger && fit != 2)) {            // registers allow two blocks
            std::printf("[%lld, %lld, %lld] groups %lld dtype %d kind %d: %lld blocks, %d per SM\n", (long long)b, (long long)hw,
                        (long long)(w * g), (long long)g, dtype, kind, (long long)grid, fit);
            ++wrong;
        }
    }
    std::printf("%ld plans, %ld wrong\n", plans, wrong);
    return wrong != 0 || plans == 0;
}
