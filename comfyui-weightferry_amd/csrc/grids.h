// How long one-dimensional work is cut into launches. A grid dimension holds fewer than 2^32 work-items, so workgroups of 256
// threads end at 2^24 - 1 of them; longer work goes out in several launches. Plain host arithmetic.
#pragma once

#include <algorithm>
#include <cstdint>

namespace wf {

constexpr int64_t kGridMost = (1LL << 24) - 1;       // workgroups of 256 threads a launch

// f(first workgroup, workgroups) for each launch of wgs workgroups
template <typename F>
inline void over_grids(int64_t wgs, int64_t most, F&& f) {
    for (int64_t first = 0; first < wgs; first += most) f(first, (uint32_t)std::min(wgs - first, most));
}

// The launches of a call over `count` tensors of values(i) values, in blocks of `block` values, `wg_blocks` of them a workgroup:
// at most `tensors` parts and `most` workgroups a launch. part(slot, tensor, its first block, blocks, first workgroup) for each
// run of blocks of a tensor, launch(parts, workgroups) behind the last one of a launch. Every part but a tensor's last is
// whole workgroups.
template <typename V, typename P, typename L>
inline void over_tensors(int64_t count, int block, int wg_blocks, int tensors, int64_t most, V&& values, P&& part,
                         L&& launch) {
    int slot = 0;
    int64_t wgs = 0;
    for (int64_t i = 0; i < count; i++) {
        const int64_t blocks = (values(i) + block - 1) / block;
        for (int64_t done = 0; done < blocks;) {
            const int64_t n = std::min(blocks - done, (most - wgs) * wg_blocks);
            part(slot++, i, done, n, (uint32_t)wgs);
            wgs += (n + wg_blocks - 1) / wg_blocks;
            done += n;
            if (slot == tensors || wgs == most) {
                launch(slot, (uint32_t)wgs);
                slot = 0;
                wgs = 0;
            }
        }
    }
    if (slot) launch(slot, (uint32_t)wgs);
}

}  // namespace wf
