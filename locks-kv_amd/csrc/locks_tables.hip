// Block tables, lengths, positions and cache slots of a step, made on the GPU
// from the requests' lengths, with the blocks of a free list.
//
// Mathematics.  Request r of the batch is row w = rows[r] of the pool: c =
// lens[w] tokens in the cache, n = new_lens[r] new ones, page P.
//   have = ceil(c / P), all = ceil((c + n) / P), need = all - have
//   first[r] = sum of need over the requests before r
//   served   = need = 0, or first[r] + need <= the blocks that are free
//   block k of the call is free[head + k]; head advances by what is taken
//   start[r] = sum of n before r; token start[r] + i: position c + i, slot
//   table[position / P] * P + position % P
// Three prefix sums over at most TB_MAX requests; the rest is copying.
//
// One launch: every workgroup makes the sums again for itself (a few hundred
// bytes that stay in the cache) instead of waiting for another kernel, then
// takes its share of the page ids and of the tokens.  lens and head change in
// place, so the last workgroup to have read them writes them (an arrival count,
// left at zero).  Bound by latency: the rows are read three times, twice for the
// claims with a barrier behind each, then the lengths, three prefix sums of two
// barriers each, the arrival, and the copy of the page ids.  32 requests of up to 2048
// pages 6.2 us, 256 of up to 4096 with 16K tokens 11.4, the roll-back 4.4-4.7.
#include "locks_common.h"
#include "locks_hip.h"

namespace locks {

constexpr int TT_BLK = 256;
constexpr int TT_WAVES = TT_BLK / kWave;
constexpr int TT_MAX = LOCKS_TABLES_MAX_REQS;
constexpr int TT_BLOCKS = 1 << 22;          // blocks of a pool: TT_BLK needs sum within 31 bits
constexpr int TT_CHUNK = 4 * TT_BLK;        // page ids a workgroup copies at once (16 bytes per thread)

// Exclusive prefix sums of two values over the workgroup, and their totals.
__device__ __forceinline__ void scan2(int a, int b, int (*ws)[2], int* ea, int* eb, int* ta, int* tb) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int ia = wave_incl_scan_i(a), ib = wave_incl_scan_i(b);
    if (lane == 63) { ws[w][0] = ia; ws[w][1] = ib; }
    __syncthreads();
    int oa = 0, ob = 0, sa = 0, sb = 0;
#pragma unroll
    for (int i = 0; i < TT_WAVES; ++i) {
        const int x = ws[i][0], y = ws[i][1];
        oa += i < w ? x : 0; ob += i < w ? y : 0;
        sa += x; sb += y;
    }
    __syncthreads();
    *ea = oa + ia - a; *eb = ob + ib - b; *ta = sa; *tb = sb;
}

// The lowest request that names each row: dup[row] afterwards, for the rows named.
__device__ __forceinline__ void claim_rows(const int* __restrict__ rows, int n_req, int max_rows, int* dup) {
    for (int r = threadIdx.x; r < n_req; r += TT_BLK) {
        const int w = rows[r];
        if (w >= 0 && w < max_rows) dup[w] = 0x7fffffff;
    }
    __syncthreads();
    for (int r = threadIdx.x; r < n_req; r += TT_BLK) {
        const int w = rows[r];
        if (w >= 0 && w < max_rows) atomicMin(&dup[w], r);
    }
    __syncthreads();
}

// True in the last workgroup to arrive (after every one has read what the last
// one is about to change); leaves the count at zero.
__device__ __forceinline__ bool last_arrival(int* count, int* flag) {
    __syncthreads();
    if (threadIdx.x == 0) {
        const int old = __hip_atomic_fetch_add(count, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        *flag = old == (int)gridDim.x - 1;
        if (*flag) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return *flag;
}

__global__ __launch_bounds__(TT_BLK) void tables_step_kernel(
    const int* __restrict__ rows, const int* __restrict__ new_lens, int n_req, int n_tokens,
    int* lens, int* table, long tab_sr, int max_rows, int max_pages, const int* __restrict__ free_list,
    int num_blocks, int* state, int* __restrict__ bt, long bt_sr, int* __restrict__ seq_lens,
    int* __restrict__ qsl, int* __restrict__ positions, int64_t* __restrict__ slots, int page)
{
    __shared__ int start[TT_MAX + 1];       // first token of each request
    __shared__ int first[TT_MAX];           // its first fresh block among the call's
    __shared__ int had[TT_MAX];             // tokens it has in the cache; ~tokens when it is not served
    __shared__ int chunk0[TT_MAX + 1];      // first copy chunk of each request
    __shared__ int dup[TT_MAX], row[TT_MAX];
    __shared__ int ws[TT_WAVES][2];
    __shared__ int flag;
    const int tid = threadIdx.x;
    claim_rows(rows, n_req, max_rows, dup);
    const int head = min(max(state[0], 0), num_blocks), avail = num_blocks - head;
    int tok = 0, blocks = 0, chunks = 0, taken = 0, unserved = 0;
    for (int r0 = 0; r0 < n_req; r0 += TT_BLK) {
        const int r = r0 + tid;
        const int w = r < n_req ? rows[r] : -1;
        const int n = w >= 0 ? max(new_lens[r], 0) : 0;
        const bool mine = w >= 0 && w < max_rows && dup[w] == r;
        const int c = mine ? max(lens[w], 0) : 0;
        const long all_l = ((long)c + n + page - 1) / page;
        const bool fits = mine && all_l <= max_pages;
        const int have = (c + page - 1) / page, all = fits ? (int)all_l : have;
        const int need = min(all - have, avail + 1);        // past avail all needs are one: the sums stay small
        int et, eb, st, sb, ec, ez, sc, sz;
        scan2(n, need, ws, &et, &eb, &st, &sb);
        const bool served = fits && (need == 0 || blocks + eb + need <= avail);
        scan2(served ? (all + TT_CHUNK - 1) / TT_CHUNK : 0, served ? need : 0, ws, &ec, &ez, &sc, &sz);
        if (r < n_req) {
            start[r] = tok + et;
            first[r] = blocks + eb;
            row[r] = w;
            had[r] = served ? c : ~c;
            chunk0[r] = chunks + ec;
            if (blockIdx.x == 0) {
                seq_lens[r] = served ? c + n : 0;
                qsl[r] = tok + et;
            }
        }
        int x, y, lost;
        scan2(w >= 0 && !served ? 1 : 0, 0, ws, &x, &y, &lost, &y);
        tok += st; blocks = min(blocks + sb, TT_BLOCKS); chunks += sc; taken += sz; unserved += lost;
    }
    if (tid == 0) {
        start[n_req] = tok;
        chunk0[n_req] = chunks;
        if (blockIdx.x == 0) qsl[n_req] = tok;
    }
    const bool last = last_arrival(state + 2, &flag);
    if (last) {
        for (int r = tid; r < n_req; r += TT_BLK)
            if (had[r] >= 0) lens[row[r]] = had[r] + (start[r + 1] - start[r]);
        if (tid == 0) {
            state[0] = head + taken;
            state[1] = unserved;
        }
    }
    // the request of chunk / token x: the last r with at[r] <= x (x < at[n_req])
    auto owner = [&](const int* at, int x) {
        int lo = 0, hi = n_req - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (at[mid] <= x) lo = mid; else hi = mid - 1;
        }
        return lo;
    };
    // page ids: what the request owns from its row, then its fresh blocks
    for (int ch = blockIdx.x; ch < chunks; ch += gridDim.x) {
        const int r = owner(chunk0, ch);
        const int w = row[r], c = had[r], n = start[r + 1] - start[r];
        const int have = (c + page - 1) / page, all = (c + n + page - 1) / page;
        const int col = (ch - chunk0[r]) * TT_CHUNK + 4 * tid;
        int* src = table + (long)w * tab_sr;
        int* dst = bt + (long)r * bt_sr;
        if (col + 4 <= have) {
            *reinterpret_cast<int4*>(dst + col) = *reinterpret_cast<const int4*>(src + col);
        } else {
            for (int i = col; i < min(col + 4, all); ++i) {
                int id;
                if (i < have) id = src[i];
                else src[i] = id = free_list[head + first[r] + i - have];
                dst[i] = id;
            }
        }
    }
    for (int t = blockIdx.x * TT_BLK + tid; t < n_tokens; t += gridDim.x * TT_BLK) {
        int pos = 0;
        int64_t slot = -1;
        if (t < tok) {
            const int r = owner(start, t);
            const int h = had[r], c = h >= 0 ? h : ~h;
            pos = c + t - start[r];
            if (h >= 0) {
                const int pg = pos / page, have = (c + page - 1) / page;
                const int id = pg < have ? table[(long)row[r] * tab_sr + pg] : free_list[head + first[r] + pg - have];
                slot = (int64_t)id * page + pos % page;
            }
        }
        positions[t] = pos;
        slots[t] = slot;
    }
}

// Requests back to keep[r] tokens: the blocks past them return to the free list
// in the order in which a step takes them, so a step that is rolled back leaves
// the list as it was.
__global__ __launch_bounds__(TT_BLK) void tables_trim_kernel(
    const int* __restrict__ rows, const int* __restrict__ keep, int n_req, int* lens,
    const int* __restrict__ table, long tab_sr, int max_rows, int max_pages, int num_blocks, int* free_list,
    int* state, int page)
{
    __shared__ int first[TT_MAX + 1];       // first returned block of each request
    __shared__ int to[TT_MAX];              // tokens it keeps; -1: nothing changes
    __shared__ int dup[TT_MAX];
    __shared__ int ws[TT_WAVES][2];
    __shared__ int flag;
    const int tid = threadIdx.x;
    claim_rows(rows, n_req, max_rows, dup);
    const int head = min(max(state[0], 0), num_blocks);
    int total = 0;
    for (int r0 = 0; r0 < n_req; r0 += TT_BLK) {
        const int r = r0 + tid;
        const int w = r < n_req ? rows[r] : -1;
        const bool mine = w >= 0 && w < max_rows && dup[w] == r;
        const int c = mine ? min(max(lens[w], 0), max_pages * page) : 0;
        const int k = mine ? min(max(keep[r], 0), c) : 0;
        const int back = (c + page - 1) / page - (k + page - 1) / page;
        int eb, x, sb, y;
        scan2(back, 0, ws, &eb, &x, &sb, &y);
        if (r < n_req) {
            first[r] = total + eb;
            to[r] = mine ? k : -1;
        }
        total += sb;
    }
    if (tid == 0) first[n_req] = total;
    if (last_arrival(state + 2, &flag)) {
        for (int r = tid; r < n_req; r += TT_BLK)
            if (to[r] >= 0) lens[rows[r]] = to[r];
        if (tid == 0) state[0] = max(head - total, 0);
    }
    for (int i = blockIdx.x * TT_BLK + tid; i < total; i += gridDim.x * TT_BLK) {
        int lo = 0, hi = n_req - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= i) lo = mid; else hi = mid - 1;
        }
        const int at = head - total + i;
        if (at >= 0)
            free_list[at] = table[(long)rows[lo] * tab_sr + (to[lo] + page - 1) / page + i - first[lo]];
    }
}

}  // namespace locks

using namespace locks;

extern "C" int32_t locks_tables_step(
    const int32_t* rows, const int32_t* new_lens, int32_t n_req, int32_t n_tokens, int32_t* lens,
    int32_t* table, int64_t table_stride, int32_t max_reqs, int32_t max_pages, const int32_t* free_list,
    int32_t num_blocks, int32_t* state, int32_t* block_table, int64_t bt_stride, int32_t* seq_lens,
    int32_t* query_start_loc, int32_t* positions, int64_t* slot_mapping, int32_t page, void* stream)
{
    LOCKS_REQUIRE(page == 16 || page == 32 || page == 64, "locks_tables_step: page %d outside {16, 32, 64}", page);
    LOCKS_REQUIRE(max_reqs >= 1 && max_reqs <= TT_MAX, "locks_tables_step: max_reqs %d outside [1, %d]", max_reqs, TT_MAX);
    LOCKS_REQUIRE(n_req >= 0 && n_req <= max_reqs, "locks_tables_step: n_req %d outside [0, max_reqs %d]", n_req, max_reqs);
    LOCKS_REQUIRE(n_tokens >= 0, "locks_tables_step: n_tokens %d < 0", n_tokens);
    LOCKS_REQUIRE(max_pages >= 1 && (int64_t)max_pages * page <= 0x7fffffffLL - page,
                  "locks_tables_step: max_pages %d x page %d outside 32-bit lengths", max_pages, page);
    LOCKS_REQUIRE(num_blocks >= 1 && num_blocks <= TT_BLOCKS, "locks_tables_step: num_blocks %d outside [1, %d]",
                  num_blocks, TT_BLOCKS);
    LOCKS_REQUIRE(table_stride % 4 == 0 && bt_stride % 4 == 0 && table_stride >= max_pages && bt_stride >= max_pages &&
                  (uintptr_t)table % 16 == 0 && (uintptr_t)block_table % 16 == 0,
                  "locks_tables_step: table rows must hold max_pages ids, 16-byte aligned");
    LOCKS_REQUIRE(((rows && new_lens) || n_req == 0) && lens && table && free_list && state && block_table && seq_lens &&
                  query_start_loc && positions && slot_mapping, "locks_tables_step: null pointer argument");
    // a workgroup per 1024 page ids or tokens that the call can hold, at most 96 (256
    // requests, 16K tokens, step and roll-back: 64 17.1 us, 96 15.8, 256 20.1):
    // each repeats the sums over the requests and adds to the arrival count
    const long work = (long)n_req * cdiv(max_pages, TT_CHUNK) + cdiv(n_tokens, TT_CHUNK);
    const int grid = (int)(work < 1 ? 1 : work > 96 ? 96 : work);
    hipLaunchKernelGGL(tables_step_kernel, dim3(grid), dim3(TT_BLK), 0, (hipStream_t)stream, rows, new_lens, n_req,
                       n_tokens, lens, table, (long)table_stride, max_reqs, max_pages, free_list, num_blocks, state,
                       block_table, (long)bt_stride, seq_lens, query_start_loc, positions, slot_mapping, page);
    return check_launch("tables_step_kernel");
}

extern "C" int32_t locks_tables_trim(
    const int32_t* rows, const int32_t* keep_lens, int32_t n_req, int32_t* lens, const int32_t* table,
    int64_t table_stride, int32_t max_reqs, int32_t max_pages, int32_t* free_list, int32_t num_blocks,
    int32_t* state, int32_t page, void* stream)
{
    LOCKS_REQUIRE(page == 16 || page == 32 || page == 64, "locks_tables_trim: page %d outside {16, 32, 64}", page);
    LOCKS_REQUIRE(max_reqs >= 1 && max_reqs <= TT_MAX, "locks_tables_trim: max_reqs %d outside [1, %d]", max_reqs, TT_MAX);
    LOCKS_REQUIRE(n_req >= 0 && n_req <= max_reqs, "locks_tables_trim: n_req %d outside [0, max_reqs %d]", n_req, max_reqs);
    LOCKS_REQUIRE(max_pages >= 1 && (int64_t)max_pages * page <= 0x7fffffffLL - page && table_stride >= max_pages,
                  "locks_tables_trim: max_pages %d x page %d outside 32-bit lengths or the rows", max_pages, page);
    LOCKS_REQUIRE(num_blocks >= 1 && num_blocks <= TT_BLOCKS, "locks_tables_trim: num_blocks %d outside [1, %d]",
                  num_blocks, TT_BLOCKS);
    if (n_req == 0) return 0;
    LOCKS_REQUIRE(rows && keep_lens && lens && table && free_list && state, "locks_tables_trim: null pointer argument");
    const long work = (long)n_req * cdiv(max_pages, TT_CHUNK);
    const int grid = (int)(work > 64 ? 64 : work);
    hipLaunchKernelGGL(tables_trim_kernel, dim3(grid), dim3(TT_BLK), 0, (hipStream_t)stream, rows, keep_lens, n_req,
                       lens, table, (long)table_stride, max_reqs, max_pages, num_blocks, free_list, state, page);
    return check_launch("tables_trim_kernel");
}
