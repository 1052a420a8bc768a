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
// of the group, m (the maximum, as a natural-log score; base 2 where the cache has 4 bits),
// l (the sum) and acc
// (D) in fp32.  A split without keys leaves m = -inf and l = 0, and no acc that counts.
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

constexpr int AT_MAX_SPLITS = 128;          // of one row, all kinds together
constexpr int AT_ROWS = 128;                // query rows (token, head of the group) of a prompt's workgroup
constexpr float kLog2e = 1.44269504088896340736f;

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* lds_v4s;

__device__ __forceinline__ int wave_max_int(int v) { return (int)(wave_max_u32((uint32_t)v ^ 0x80000000u) ^ 0x80000000u); }
__device__ __forceinline__ int wave_min_int(int v) { return ~wave_max_int(~v); }

inline int clampi(long x, int lo, int hi) { return (int)(x < lo ? lo : x > hi ? hi : x); }
// Tiles of k non-empty requests (groups) of n tokens together: sum of ceil(c / TQ)
// <= floor((n - k) / TQ) + k, largest where all are non-empty.
inline long prefill_tiles(int n_tokens, int n_req, int G) {
    const int k = n_req < n_tokens ? n_req : n_tokens;
    return (long)(n_tokens - k) / (AT_ROWS / G) + k;
}
// The keys that a host-side bound leaves.
inline long bound_keys(int32_t max_seq_len, int32_t bt_cols, int32_t page) {
    const long cap = (long)bt_cols * page;
    return max_seq_len > 0 && max_seq_len < cap ? max_seq_len : cap;
}
// Splits of a row's keys in a call of many tokens: one once there are 256 workgroups, else
// about 512 workgroups of at least 4 tiles of key_tile keys.
inline int prefill_splits(long tiles, int n_kv, long max_keys, int key_tile) {
    const long wgs = tiles * n_kv;
    if (wgs >= 256) return 1;
    return clampi((512 + wgs - 1) / wgs, 1, clampi(max_keys / (4 * key_tile), 1, 64));
}

// Bytes of a call's partials, and where they stand in its workspace.
inline int64_t part_bytes(int64_t rows, int splits, int D) { return rows * splits * (D + 2) * 4; }
inline Partials part_layout(void* ws, int64_t rows, int splits, int D) {
    float* acc = static_cast<float*>(ws);   // first: 16-byte aligned
    return Partials{acc + rows * splits * D, acc + rows * splits * (D + 1), acc, splits};
}

// What every attention entry asks of its arguments, and of its workspace.
int32_t check_attn(const char* what, const uint16_t* q, int64_t q_st, int64_t q_sh, const uint16_t* k,
                   const int64_t* ks, const uint16_t* v, const int64_t* vs, int32_t num_blocks, const int32_t* bt,
                   int64_t bt_stride, int32_t bt_cols, const int32_t* seq_lens, int32_t window, int32_t sinks,
                   const uint16_t* out, int64_t o_st, int64_t o_sh, int32_t n_req, int32_t n_kv, int32_t G,
                   int32_t head_dim, int32_t page, int32_t max_keys, float scale);
int32_t check_ws(const char* what, const void* ws, int64_t have, int64_t need);
// And of a cache in 4 bits (locks_kv4.hip).
int32_t check_kv4(const char* what, const void* cache, int64_t sb, int64_t sh, int32_t num_blocks, int32_t n_kv,
                  int32_t head_dim, int32_t page);

// Workspace of a single-token call on one (locks_kv4.hip).
int64_t kv4_workspace(int n_req, int n_kv, int G, int head_dim);
constexpr int P4_KT = 64;                   // keys per tile of a call of many tokens on one

}  // namespace locks
