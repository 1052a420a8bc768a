// Shared by the window and shared-prefix attention and the split decode kernel:
// which keys a call sees, and the partials that its splits leave.
#pragma once

#include "locks_common.h"

namespace locks {

// The keys of a single-token decode over a range of the row's tokens:
// [lo, seq_len) and [0, min(sinks, lo)), lo = max(seq_len - window, 0) (0 without a
// window).
struct RangeSrc {
    int window, sinks;                      // window 0: none
};

// The prefix pages of request r's group (the same in every lane), or -1.  All loads
// of 64 groups go out together: a workgroup of a short row lives as long as its
// chain of dependent loads.
__device__ __forceinline__ int group_pages(const int* __restrict__ gstart, const int* __restrict__ gpages, int n_groups,
                                           int r) {
    const int lane = threadIdx.x & 63;
    for (int g0 = 0; g0 < n_groups; g0 += kWave) {
        const int g = min(g0 + lane, n_groups - 1);
        const int first = gstart[g], end = gstart[g + 1], pages = gpages[g];
        const unsigned long long m = __ballot(first <= r && r < end);
        if (m) return max(__builtin_amdgcn_readlane(pages, __ffsll(m) - 1), 0);
    }
    return -1;
}

// Partials of a call: per (token or request, kv head) row, split and query head
// of the group, m (the maximum, as a natural-log score) and l (the sum) and acc
// (D) in fp32.  A split without keys leaves m = -inf, l = 0 and no acc.
struct Partials {
    float* m; float* l; float* acc;
    int splits;                             // of a row
};

// The split decode over RangeSrc's keys (locks_decode.hip): n_req x n_kv x nsplit
// workgroups, each of at least min_steps 16-token steps.
int launch_decode_range(const uint16_t* q, long q_sr, long q_sh, const uint16_t* k, const long* ks, const uint16_t* v,
                        const long* vs, int num_blocks, const int* bt, long bt_sr, int bt_cols, const int* seq_lens,
                        const Partials& p, const RangeSrc& range, int nsplit, int min_steps, int n_req, int n_kv, int G,
                        int head_dim, int page, float scale, hipStream_t stream);

}  // namespace locks
