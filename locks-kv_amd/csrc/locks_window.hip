// Attention over the paged cache with a sliding window and first tokens that
// stay visible, for single tokens and for many, and single-token attention of
// requests that share a prefix.
//
// Mathematics.  Query i (position) sees key j when j <= i and (no window, or
// j > i - window, or j < sinks):
//   o = sum_j p_j v_j / l,  p_j = exp(scale q.k_j - m),  l = sum_j p_j,  lse = m + ln l
// with the running m and l of one pass over the keys (fp32).  Keys split over
// workgroups leave (m, l, acc) each; attn_merge_kernel joins them with weights
// exp(m_s - max m).  A shared prefix is one such split whose keys are read once
// for every member of the group, a request's own keys are the others.
//
// attn_tile_kernel: a workgroup of 4 waves holds 128 query rows (token, head of
// the group), 32 per wave, and walks over tiles of KT keys in LDS.
//   S^T = K Q^T (32x32x16 bf16 MFMA): a lane holds KT / 2 keys of ONE query, so
//     max and sum are in-lane plus one swap with lane ^ 32;
//   O^T += V^T P^T: the keys of an MFMA step are numbered so that a lane's P
//     values are the operand as they stand; V comes out of LDS transposed
//     (ds_read_b64_tr_b16: 4 keys x 16 columns per 16 lanes).
// K and V arrive by direct loads to LDS, one tile ahead (two at d 64 and 256).
// 16-byte chunks of a row are permuted by the row on the way in (an exclusive or),
// which keeps the reads of both operands free of bank conflicts.
// 8192 tokens, 32 / 8 heads, d 128, causal: 548 to 616 us over four cards, 1003 to 892
// TFLOP/s, the matrix cores 42-45 % busy: a wave does scores, softmax and V's
// products in turn, and only its SIMD's other wave fills the gaps (at d 64 the time
// is near the sum of products and softmax).  On a card of 556, copies for timing:
// without the softmax 496, without K and V reads from LDS too 440, without staging too
// 353.  64 keys a tile and 4 waves (577 on a third card): 32 keys with four tiles in
// LDS took 580 there, 8 waves on 256 rows 548 but 163 for 139 at d 64 and 96 for 77 on
// a prefix.
//
// Decode (one token): the split kernel of locks_decode.hip over a token range, or
// (with a shared prefix) the tiles above, of which a request fills one column block.
#include "locks_attn.h"
#include "locks_common.h"
#include "locks_hip.h"

#include <math.h>

#include <type_traits>

namespace locks {

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* lds_v4s;
typedef float v16f __attribute__((ext_vector_type(16)));
typedef unsigned short v2us __attribute__((ext_vector_type(2)));

constexpr int AT_WAVES = 4;
constexpr int AT_BLK = AT_WAVES * kWave;
constexpr int AT_ROWS = 32 * AT_WAVES;      // query rows per workgroup
constexpr int AT_MAX_SPLITS = 128;          // of one row, all kinds together
constexpr float kLog2e = 1.44269504088896340736f;

template <int D>
struct AtGeom {
    static constexpr int KT = D == 256 ? 32 : 64;        // keys per tile
    static constexpr int NST = D == 128 ? 2 : 3;        // tiles in LDS: one in use, the others on the way
    static constexpr int ROWB = 2 * D;                  // bytes of a K or V row
    static constexpr int TILEB = KT * ROWB;
    static constexpr int WROWS = KT / AT_WAVES;         // rows that a wave stages (of one cache page)
    static constexpr int NI = WROWS * ROWB / 1024;      // its 1 KB load instructions, K and V each
    // the chunk permutations: K is read 16 rows at one chunk, V 4 rows at 4 chunks
    static __device__ __forceinline__ int swz_k(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
    static __device__ __forceinline__ int swz_v(int row) { return D == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }
};

constexpr int vm_wait(int n) { return 0x0F70 | (n & 15) | ((n >> 4) << 14); }    // s_waitcnt vmcnt(n)

struct TileArgs {
    const uint16_t* q; long q_st, q_sh;
    const uint16_t* k; long k_sb, k_st, k_sh;
    const uint16_t* v; long v_sb, v_st, v_sh;
    const int* bt; long bt_sr;
    const int* seq_lens;
    const int* starts;                      // first token of each request, or first request of each group
    const int* gpages;                      // prefix pages of each group
    uint16_t* out; long o_st, o_sh;
    float* lse; long lse_st;
    Partials p;
    float c;                                // scale * log2(e)
    float scale;
    int NB, bt_cols, n_rows, n_seq, n_kv, G, pg_sh, window, sinks, nsplit;
    int own;                                // SHARED: splits of a request's own keys, behind the nsplit of its prefix
    int shared_units, own_units, chunk;     // and how the two kinds of work are dealt out (per kv head)
};

// 16 bytes per lane from its own address to 1 KB of LDS, in lane order
__device__ __forceinline__ void load_lds16(const uint8_t* src, uint8_t* dst) {
    __builtin_amdgcn_global_load_lds(src, (lds_ptr)dst, 16, 0, 0);
}
__device__ __forceinline__ int wave_max_int(int v) { return (int)(wave_max_u32((uint32_t)v ^ 0x80000000u) ^ 0x80000000u); }
__device__ __forceinline__ int wave_min_int(int v) { return ~wave_max_int(~v); }
// bit 0 / 1: the low / high bf16 of a word is infinite or NaN
__device__ __forceinline__ uint32_t nonfinite2(uint32_t w) {
    return ((w & 0x7F80u) == 0x7F80u ? 1u : 0u) | ((w & 0x7F800000u) == 0x7F800000u ? 2u : 0u);
}

// SHARED: rows are the members of a group and the keys its prefix, or (the other
// kind of work in the same launch) the heads of one request and its own keys;
// partials only.  The prefix is bound by the matrix cores, own keys by memory: dealt
// out in turns of one workgroup per CU, they overlap.
// PART: partials instead of the output.
template <int D, bool SHARED, bool PART>
__global__ __launch_bounds__(AT_BLK, D == 256 ? 1 : 2) void attn_tile_kernel(const TileArgs a)
{
    using GM = AtGeom<D>;
    constexpr int KT = GM::KT, ROWB = GM::ROWB, NB2 = KT / 32, ND = D / 32;
    constexpr int VPRE = D == 256 ? ND / 2 : ND;        // column blocks of V read before the softmax
    static_assert(!SHARED || PART, "a prefix is one part of a row");
    // one array per tile: the compiler can tell the DMA of one from the reads of
    // another, and waits for neither
    constexpr int NST = GM::NST, TB = GM::TILEB;
    __shared__ __attribute__((aligned(1024))) uint8_t k0[TB], k1[TB], k2[NST > 2 ? TB : 16];
    __shared__ __attribute__((aligned(1024))) uint8_t v0[TB], v1[TB], v2[NST > 2 ? TB : 16];
    static_assert(NST == 2 || NST == 3, "tiles in LDS");
    auto kbuf = [&](auto i) __attribute__((always_inline)) { return i() == 0 ? k0 : i() == 1 ? k1 : k2; };
    auto vbuf = [&](auto i) __attribute__((always_inline)) { return i() == 0 ? v0 : i() == 1 ? v1 : v2; };
    __shared__ int wlim[AT_WAVES][4];
    __shared__ int odd[2];                              // a value that is not finite is in the tile
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c32 = lane & 31, h = lane >> 5;
    const int G = a.G, TQ = AT_ROWS / G;                // tokens per tile
    const int kh = blockIdx.x % a.n_kv;
    const int unit = blockIdx.x / a.n_kv;
    int seq = -1, t_in = 0, first = 0, count = 0;
    int len = 0;                                        // tokens before the request's first row; pages of the prefix
    int sp = unit % a.nsplit, slot = sp, nsplit = a.nsplit, tile = unit / a.nsplit;
    bool own = false;
    if constexpr (SHARED) {
        // turns of `chunk` units of each kind while both last, then what is left
        const int turns = min(a.shared_units, a.own_units) / a.chunk;
        const int turn = unit / (2 * a.chunk), at = unit % (2 * a.chunk);
        int i;
        if (turn < turns) {
            own = at >= a.chunk;
            i = turn * a.chunk + (own ? at - a.chunk : at);
        } else {
            i = unit - turns * a.chunk;
            own = i >= a.shared_units;
            i = own ? unit - a.shared_units : i;
        }
        if (own) {
            seq = first = i / a.own;
            count = 1;
            sp = i % a.own; slot = a.nsplit + sp; nsplit = a.own;
        } else {
            // row tiles of one part of the prefix side by side: they read the same keys
            const int tiles = a.shared_units / a.nsplit;
            sp = slot = i / tiles; tile = i % tiles;
        }
    }
    // the request (group) that holds this tile
    for (int s0 = 0, done = 0; s0 < a.n_seq && seq < 0; s0 += kWave) {
        // (all loads together: a tile of few keys lives as long as its chain of them)
        const int s = min(s0 + lane, a.n_seq - 1);
        const int at = a.starts[s], end = a.starts[s + 1];
        const int len_s = SHARED ? max(a.gpages[s], 0) : a.seq_lens[s];
        const int f = max(at, 0), n = s0 + lane < a.n_seq ? max(min(end, a.n_rows) - f, 0) : 0;
        const int nt = (n + TQ - 1) / TQ;
        const int inc = wave_incl_scan_i(nt);
        const unsigned long long hit = __ballot(done + inc > tile);
        if (hit) {
            const int l = __ffsll(hit) - 1;
            seq = s0 + l;
            first = __builtin_amdgcn_readlane(f, l);
            count = __builtin_amdgcn_readlane(n, l);
            len = __builtin_amdgcn_readlane(SHARED ? len_s : len_s - (end - at), l);
            const int nt_l = __builtin_amdgcn_readlane(nt, l);
            // the tiles that see most first
            t_in = nt_l - 1 - (tile - done - (__builtin_amdgcn_readlane(inc, l) - nt_l));
        }
        done += __builtin_amdgcn_readlane(inc, 63);
    }
    if (seq < 0) return;

    // this lane's row and the keys [lo, hi) and [0, sinks) that it sees
    const long cap = (long)a.bt_cols << a.pg_sh;
    const int rho = 32 * wave + c32;
    const int j = t_in * TQ + rho / G, g = rho % G;
    const bool valid = rho < TQ * G && j < count;
    const int tok = first + (valid ? j : 0);
    int hi, lo = 0, sinks = 0, base = 0;                // base: where the key tiles start
    long bt_row;
    if constexpr (SHARED) {
        const int sl = a.seq_lens[tok];
        const int pages = own ? group_pages(a.starts, a.gpages, a.n_seq, seq) : len;
        const long pre = min((long)max(pages, 0), (long)a.bt_cols) << a.pg_sh;
        hi = (int)min(own ? cap : pre, (long)sl);
        if (own) {
            base = lo = (int)min(pre, (long)max(sl, 0));
            if (pages < 0 && sp == 0 && tid < G)        // a request in no group has no partials of a prefix
                for (int i = 0; i < a.nsplit; ++i) {
                    const long at = (((long)tok * a.n_kv + kh) * a.p.splits + i) * G + tid;
                    a.p.m[at] = -INFINITY;
                    a.p.l[at] = 0.f;
                }
        }
        bt_row = first;
        if (!own) {
            // The prefix's page ids: the row of the longest of the first 64 members (of
            // the next 64, and so on, until one is as long as the prefix).  A row that
            // ends sooner holds fewer pages, that of an unserved request an earlier
            // batch's.  No member sees further than the longest one's row.
            int best = 0, who = 0;
            for (int s0 = 0; s0 < count; s0 += kWave) {
                const int i = s0 + lane, sl_i = i < count ? a.seq_lens[first + i] : 0;
                who = sl_i > best ? i : who;
                best = max(best, sl_i);
                if (__any(best >= pre)) break;
            }
            const int top = wave_max_int(best);
            bt_row += __builtin_amdgcn_readfirstlane(wave_min_int(best == top ? who : count - 1));
        }
    } else {
        const int pos = len + j;
        hi = (int)min((long)pos + 1, cap);
        lo = a.window ? max(pos - a.window + 1, 0) : 0;
        sinks = a.sinks;
        bt_row = seq;
    }
    if (!valid) { hi = 0x7fffffff; lo = 0; }
    // of the wave's valid rows, then of the workgroup's
    const int w_min_hi = __builtin_amdgcn_readfirstlane(wave_min_int(hi));
    const int w_max_hi = __builtin_amdgcn_readfirstlane(wave_max_int(valid ? hi : 0));
    const int w_max_lo = __builtin_amdgcn_readfirstlane(wave_max_int(lo));
    const int w_min_lo = __builtin_amdgcn_readfirstlane(wave_min_int(valid ? lo : 0x7fffffff));
    if (tid < 2) odd[tid] = 0;
    int turn = 0;
    if (lane == 0) {
        wlim[wave][0] = w_min_hi; wlim[wave][1] = w_max_hi; wlim[wave][2] = w_max_lo; wlim[wave][3] = w_min_lo;
    }
    __syncthreads();
    int min_hi = wlim[0][0], max_hi = wlim[0][1], max_lo = wlim[0][2], min_lo = wlim[0][3];
#pragma unroll
    for (int w = 1; w < AT_WAVES; ++w) {
        min_hi = min(min_hi, wlim[w][0]); max_hi = max(max_hi, wlim[w][1]);
        max_lo = max(max_lo, wlim[w][2]); min_lo = min(min_lo, wlim[w][3]);
    }
    min_hi = __builtin_amdgcn_readfirstlane(min_hi); max_hi = __builtin_amdgcn_readfirstlane(max_hi);
    max_lo = __builtin_amdgcn_readfirstlane(max_lo); min_lo = __builtin_amdgcn_readfirstlane(min_lo);

    // key tiles: the first na, then [b0, b1); this split's share of them
    const int na = (min(min(sinks, min_lo), max(max_hi, 0)) + KT - 1) / KT;
    base = __builtin_amdgcn_readfirstlane(base);
    const int b0 = max((min_lo - base) / KT, na), b1 = (int)(((long)max_hi - base + KT - 1) / KT);
    const int nt = max_hi > base ? na + max(b1 - b0, 0) : 0;
    const int n0 = (int)((long)nt * sp / nsplit), n1 = (int)((long)nt * (sp + 1) / nsplit);
    auto key_of = [&](int n) __attribute__((always_inline)) { return base + (n < na ? n : b0 + n - na) * KT; };

    // Q: k-slots 8 h .. 8 h + 7 of MFMA step s are d = 16 s + 8 h ..
    v8bf qf[D / 16];
    {
        const uint16_t* qp = a.q + (long)tok * a.q_st + (long)(kh * G + g) * a.q_sh + 8 * h;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if (valid) w = *reinterpret_cast<const uint4*>(qp + 16 * s);
            qf[s] = __builtin_bit_cast(v8bf, w);
        }
    }

    // The block ids of 64 tiles are loaded at once, one per lane: no load waits
    // between a tile's DMA.  All rows that a wave stages lie on one page.
    const int last_page = max((int)(((long)max_hi + (1L << a.pg_sh) - 1) >> a.pg_sh) - 1, 0);
    int ids = 0, ids0 = n0;
    auto fetch_ids = [&](int n) __attribute__((always_inline)) {
        ids0 = n;
        const int key = key_of(min(n + lane, max(n1 - 1, n))) + wave * GM::WROWS;
        const int pg = min(min(key >> a.pg_sh, last_page), a.bt_cols - 1);
        ids = min(max(a.bt[bt_row * a.bt_sr + pg], 0), a.NB - 1);
    };
    // byte offsets of this lane's 16-byte chunks from the wave's first row
    uint32_t ko[GM::NI], vo[GM::NI];
#pragma unroll
    for (int i = 0; i < GM::NI; ++i) {
        const int at = i * 1024 + lane * 16, row = at / ROWB, slot = (at % ROWB) / 16;
        const int tr = wave * GM::WROWS + row;              // row of the tile
        ko[i] = (uint32_t)(row * a.k_st * 2) + 16 * (slot ^ GM::swz_k(tr));
        vo[i] = (uint32_t)(row * a.v_st * 2) + 16 * (slot ^ GM::swz_v(tr));
    }
    auto stage = [&](int n, uint8_t* kb, uint8_t* vb) __attribute__((always_inline)) {
        if (n - ids0 >= kWave) fetch_ids(n);
        const long blk = __builtin_amdgcn_readlane(ids, n - ids0);
        const int off = (key_of(n) + wave * GM::WROWS) & ((1 << a.pg_sh) - 1);
        const uint8_t* kp = reinterpret_cast<const uint8_t*>(a.k + blk * a.k_sb + (long)kh * a.k_sh + off * a.k_st);
        const uint8_t* vp = reinterpret_cast<const uint8_t*>(a.v + blk * a.v_sb + (long)kh * a.v_sh + off * a.v_st);
#pragma unroll
        for (int i = 0; i < GM::NI; ++i) {
            load_lds16(kp + ko[i], kb + wave * GM::WROWS * ROWB + i * 1024);
            load_lds16(vp + vo[i], vb + wave * GM::WROWS * ROWB + i * 1024);
        }
    };

    float m = -INFINITY, l = 0.f;                       // raw score units; this half-wave's keys
    v16f o[ND];
#pragma unroll
    for (int b = 0; b < ND; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] = 0.f;

    // K row c32 (+ 32 kb): chunk (2 s + h) ^ swz; V: rows 4 h + (i >> 2), i = lane & 15
    const int i16 = lane & 15;
    int ka[D / 16], va[ND];
#pragma unroll
    for (int s = 0; s < D / 16; ++s) ka[s] = c32 * ROWB + ((2 * s + h) ^ GM::swz_k(c32)) * 16;
#pragma unroll
    for (int b = 0; b < ND; ++b) {
        const int row = 4 * h + (i16 >> 2);
        const int chunk = 4 * b + 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
        va[b] = row * ROWB + (chunk ^ GM::swz_v(row)) * 16 + (i16 & 1) * 8;
    }

    // S^T of a tile: every K read first, then the products (left to itself the
    // compiler waits for each read before its product)
    auto scores = [&](const uint8_t* kb, v16f* s) __attribute__((always_inline)) {
        v8bf kf[NB2][D / 16];
#pragma unroll
        for (int kb2 = 0; kb2 < NB2; ++kb2)
#pragma unroll
            for (int st = 0; st < D / 16; ++st)
                kf[kb2][st] = *reinterpret_cast<const v8bf*>(kb + ka[st] + kb2 * 32 * ROWB);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kb2 = 0; kb2 < NB2; ++kb2)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb2][i] = 0.f;
#pragma unroll
        for (int st = 0; st < D / 16; ++st)
#pragma unroll
            for (int kb2 = 0; kb2 < NB2; ++kb2)
                s[kb2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kb2][st], qf[st], s[kb2], 0, 0, 0);
    };
    // The running maximum and sum, O^T rescaled where a maximum grew; P in bf16, PV's
    // operand: the product takes two operands of one type, and V in fp16 would lose
    // its range.  Half a step, 2^-8 of each weight; l keeps the unrounded ones.
    // (Outputs against 64 bits: 2.2e-3, with weights in fp32 1.6e-3.)
    auto weights = [&](const v16f* s, v8bf* pf) __attribute__((always_inline)) {
        float mx = s[0][0];
#pragma unroll
        for (int kb2 = 0; kb2 < NB2; ++kb2)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb2][i]);
        mx = xor32_max(mx);
        // m follows the maximum only when it has grown by 2^8 in weight: until then
        // the weights are at most 256, and o and l need no rescaling
        if (__any((mx - m) * a.c > 8.f)) {
            const float m_new = fmaxf(m, mx);
            // not below the smallest normal number: 0 x inf would turn an infinite
            // value's sum into NaN
            const float alpha = fmaxf(__builtin_amdgcn_exp2f((m - m_new) * a.c), 1.17549435e-38f);
            m = m_new;
            l *= alpha;
#pragma unroll
            for (int b = 0; b < ND; ++b) o[b] *= alpha;
        }
        const float mc = m == -INFINITY ? 0.f : m * a.c;
#pragma unroll
        for (int kb2 = 0; kb2 < NB2; ++kb2)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[kb2][i], a.c, -mc));
                l += p;
                pf[2 * kb2 + (i >> 3)][i & 7] = (__bf16)p;
            }
    };
    auto v_frag = [&](const uint8_t* vb, int b, int c) __attribute__((always_inline)) {
        const uint8_t* x = vb + va[b] + 16 * c * ROWB;
        const v4s x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(x));
        const v4s x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(x + 8 * ROWB));
        return __builtin_bit_cast(v8bf, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    // A tile that some row sees only part of: masked places of V must not reach the
    // sums (0 x NaN), whatever an unwritten page or a later token holds.  Values
    // that are not finite are added to the rows that see them (any weight leaves
    // them what they are) and count as zero in the product.
    auto make_finite = [&](int key0, bool live, uint8_t* vb) __attribute__((always_inline)) {
        uint4* mine = reinterpret_cast<uint4*>(vb) + tid;
        // the largest magnitude of each half word; infinite and NaN from 0x7F80 on
        v2us top = {0, 0};
#pragma unroll
        for (int i = 0; i < GM::TILEB / 16 / AT_BLK; ++i) {
            const uint4 x = mine[i * AT_BLK];
            for (uint32_t w : {x.x, x.y, x.z, x.w})
                top = __builtin_elementwise_max(top, __builtin_bit_cast(v2us, w & 0x7FFF7FFFu));
        }
        // two flags in turn: the one of the tile before is cleared behind this
        // tile's barrier, ahead of the next tile's
        if (__any(top[0] >= 0x7F80 || top[1] >= 0x7F80) && lane == 0) odd[turn] = 1;
        lds_barrier();
        const bool found = *static_cast<volatile int*>(&odd[turn]) != 0;
        turn ^= 1;
        if (tid == 0) odd[turn] = 0;
        if (!found) return;
        if (live) {
            for (int kk = 0; kk < KT; ++kk) {
                const int key = key0 + kk;
                const bool seen = valid && key < hi && (key >= lo || key < sinks);
#pragma unroll
                for (int b = 0; b < ND; ++b)
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4) {
                        const uint2 x = *reinterpret_cast<const uint2*>(
                            vb + kk * ROWB + ((4 * b + q4) ^ GM::swz_v(kk)) * 16 + 8 * h);
                        if (seen && (nonfinite2(x.x) | nonfinite2(x.y))) {
                            const float y[4] = {bf16lo(x.x), bf16hi(x.x), bf16lo(x.y), bf16hi(x.y)};
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[b][4 * q4 + e] += fabsf(y[e]) <= 3.4e38f ? 0.f : y[e];
                        }
                    }
            }
        }
        __syncthreads();
        for (int i = 0; i < GM::TILEB / 16 / AT_BLK; ++i) {
            uint32_t* x = reinterpret_cast<uint32_t*>(mine + i * AT_BLK);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t y = x[e];
                x[e] = y & ((nonfinite2(y) & 1 ? 0u : 0xFFFFu) | (nonfinite2(y) & 2 ? 0u : 0xFFFF0000u));
            }
        }
        __syncthreads();
    };
    auto compute = [&](int n, const uint8_t* kb, uint8_t* vb) __attribute__((always_inline)) {
        const int key0 = key_of(n);
        const bool live = key0 < w_max_hi && (key0 + KT > w_min_lo || key0 < sinks);
        if (key0 + KT > min_hi || (key0 < max_lo && key0 + KT > sinks)) make_finite(key0, live, vb);
        if (!live) return;                              // nothing for this wave's rows
        v16f s[NB2];
        scores(kb, s);
        __builtin_amdgcn_sched_barrier(0);
        // keys that a row does not see, each side by itself: a compare with a constant
        // and a select per key
        if (key0 + KT > w_min_hi) {
            const int top = hi - key0 - 4 * h;
#pragma unroll
            for (int kb2 = 0; kb2 < NB2; ++kb2)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[kb2][i] = 32 * kb2 + 8 * (i >> 2) + (i & 3) < top ? s[kb2][i] : -INFINITY;
        }
        if (key0 < w_max_lo && key0 + KT > sinks) {
            const int low = lo - key0 - 4 * h, sink = sinks - key0 - 4 * h;
            if (key0 >= sinks) {
#pragma unroll
                for (int kb2 = 0; kb2 < NB2; ++kb2)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        s[kb2][i] = 32 * kb2 + 8 * (i >> 2) + (i & 3) >= low ? s[kb2][i] : -INFINITY;
            } else {
#pragma unroll
                for (int kb2 = 0; kb2 < NB2; ++kb2)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int x = 32 * kb2 + 8 * (i >> 2) + (i & 3);
                        s[kb2][i] = x >= low || x < sink ? s[kb2][i] : -INFINITY;
                    }
            }
        }
        v8bf vf[ND][KT / 16], pf[KT / 16];
#pragma unroll
        for (int b = 0; b < VPRE; ++b)                  // on the way during the softmax
#pragma unroll
            for (int c = 0; c < KT / 16; ++c) vf[b][c] = v_frag(vb, b, c);
        __builtin_amdgcn_sched_barrier(0);
        weights(s, pf);
#pragma unroll
        for (int b = VPRE; b < ND; ++b)
#pragma unroll
            for (int c = 0; c < KT / 16; ++c) vf[b][c] = v_frag(vb, b, c);
#pragma unroll
        for (int c = 0; c < KT / 16; ++c)
#pragma unroll
            for (int b = 0; b < ND; ++b)
                o[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[b][c], pf[c], o[b], 0, 0, 0);
    };
    // Tile n is in LDS once at most the loads of the tiles behind it are under way,
    // and free for the next one once every wave has passed the barrier after it.
    auto tile_step = [&](int n, auto use, auto fill) __attribute__((always_inline)) {
        const int behind = min(n1 - 1 - n, NST - 2);
        if (behind == 0) __builtin_amdgcn_s_waitcnt(vm_wait(0));
        else __builtin_amdgcn_s_waitcnt(vm_wait(2 * GM::NI));
        lds_barrier();
        if (n + NST - 1 < n1) stage(n + NST - 1, kbuf(fill), vbuf(fill));
        compute(n, kbuf(use), vbuf(use));
    };
    using I0 = std::integral_constant<int, 0>; using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    if (n0 < n1) {
        fetch_ids(n0);
        stage(n0, k0, v0);
        if constexpr (NST > 2) { if (n0 + 1 < n1) stage(n0 + 1, k1, v1); }
    }
    for (int n = n0; n < n1; n += NST) {
        if constexpr (NST == 2) {
            tile_step(n, I0{}, I1{});
            if (n + 1 < n1) tile_step(n + 1, I1{}, I0{});
        } else {
            tile_step(n, I0{}, I2{});
            if (n + 1 < n1) tile_step(n + 1, I1{}, I0{});
            if (n + 2 < n1) tile_step(n + 2, I2{}, I1{});
        }
    }

    l = xor32_sum(l);
    if (!valid) return;
    if constexpr (PART) {
        const long at = (((long)tok * a.n_kv + kh) * a.p.splits + slot) * G + g;
        if (h == 0) {
            a.p.m[at] = l > 0.f || l != l ? m * a.scale : -INFINITY;
            a.p.l[at] = l;
        }
        float* ap = a.p.acc + at * D + 4 * h;
#pragma unroll
        for (int b = 0; b < ND; ++b)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                *reinterpret_cast<float4*>(ap + 32 * b + 8 * q4) =
                    make_float4(o[b][4 * q4], o[b][4 * q4 + 1], o[b][4 * q4 + 2], o[b][4 * q4 + 3]);
    } else {
        // no visible key: l = 0, the row is zero and its log-sum-exp -inf
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint16_t* op = a.out + (long)tok * a.o_st + (long)(kh * G + g) * a.o_sh + 4 * h;
#pragma unroll
        for (int b = 0; b < ND; ++b)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                uint2 w;
                w.x = (uint32_t)f32_to_bf16(o[b][4 * q4] * inv) | (uint32_t)f32_to_bf16(o[b][4 * q4 + 1] * inv) << 16;
                w.y = (uint32_t)f32_to_bf16(o[b][4 * q4 + 2] * inv) | (uint32_t)f32_to_bf16(o[b][4 * q4 + 3] * inv) << 16;
                *reinterpret_cast<uint2*>(op + 32 * b + 8 * q4) = w;
            }
        if (a.lse && h == 0)
            a.lse[(long)tok * a.lse_st + kh * G + g] = l == 0.f ? -INFINITY : m * a.scale + logf(l);
    }
}

// Joins the partials of a row's splits: one workgroup per (token, head), D / 4
// columns of four x 1024 / D streams over the splits.  Bound by its chain of loads
// for few rows (32 heads of 33 splits 4.0 us), by memory for many (2048 heads of 17
// splits 6.3 us, 2.8 TB/s).
constexpr int AM_BLK = 256;
constexpr int AM_PF = 4;                    // partials that a thread loads ahead
template <int D>
__global__ __launch_bounds__(AM_BLK) void attn_merge_kernel(const Partials p, uint16_t* __restrict__ out, long o_st,
                                                            long o_sh, float* __restrict__ lse, long lse_st, int n_kv,
                                                            int G, const int* __restrict__ starts, int n_seq)
{
    constexpr int COLS = D / 4, STREAMS = AM_BLK / COLS;
    __shared__ float w_s[AT_MAX_SPLITS];
    __shared__ float4 part[STREAMS][COLS];
    const int tid = threadIdx.x, lane = tid & 63;
    const int col = tid % COLS, strm = tid / COLS;
    const int H = n_kv * G, hd = blockIdx.x % H;
    const long t = blockIdx.x / H;
    // rows before the first request or after the last one have no partials
    if (starts && (t < starts[0] || t >= starts[n_seq])) return;
    const long row0 = (t * n_kv + hd / G) * p.splits * G + hd % G;     // of split 0; G apart
    // Every load goes out before anything waits: up to two splits' m and l per lane
    // (each wave the same), and this thread's first AM_PF partials, wanted or not (a
    // split without keys has no acc: what is there is left out by a select).
    const float* ap = p.acc + row0 * D + 4 * col;
    float4 pre[AM_PF];
#pragma unroll
    for (int k = 0; k < AM_PF; ++k)
        pre[k] = *reinterpret_cast<const float4*>(ap + (long)min(strm + k * STREAMS, p.splits - 1) * G * D);
    float ms[2], ls[2];
    float mm = -INFINITY;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int s = lane + 64 * k;
        ls[k] = s < p.splits ? p.l[row0 + (long)s * G] : 0.f;
        ms[k] = s < p.splits ? p.m[row0 + (long)s * G] : -INFINITY;
        if (ls[k] == 0.f) ms[k] = -INFINITY;
        mm = fmaxf(mm, ms[k]);
    }
    mm = wave_max(mm);
    float lt = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float w = ls[k] == 0.f ? 0.f : expf(ms[k] - mm);
        lt += ls[k] * w;
        if (tid < 64 && lane + 64 * k < p.splits) w_s[lane + 64 * k] = w;
    }
    lt = wave_sum(lt);
    __syncthreads();
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < AM_PF; ++k) {
        const int s = strm + k * STREAMS;
        const float w = s < p.splits ? w_s[s] : 0.f;
        acc.x = w != 0.f ? acc.x + w * pre[k].x : acc.x;
        acc.y = w != 0.f ? acc.y + w * pre[k].y : acc.y;
        acc.z = w != 0.f ? acc.z + w * pre[k].z : acc.z;
        acc.w = w != 0.f ? acc.w + w * pre[k].w : acc.w;
    }
    for (int s = strm + AM_PF * STREAMS; s < p.splits; s += STREAMS) {
        const float w = w_s[s];
        if (w != 0.f) {
            const float4 x = *reinterpret_cast<const float4*>(ap + (long)s * G * D);
            acc.x += w * x.x; acc.y += w * x.y; acc.z += w * x.z; acc.w += w * x.w;
        }
    }
    part[strm][col] = acc;
    __syncthreads();
    if (tid < COLS) {
#pragma unroll
        for (int k = 1; k < STREAMS; ++k) {
            const float4 x = part[k][tid];
            acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
        }
        const float inv = lt == 0.f ? 0.f : 1.f / lt;
        uint2 w;
        w.x = (uint32_t)f32_to_bf16(acc.x * inv) | (uint32_t)f32_to_bf16(acc.y * inv) << 16;
        w.y = (uint32_t)f32_to_bf16(acc.z * inv) | (uint32_t)f32_to_bf16(acc.w * inv) << 16;
        *reinterpret_cast<uint2*>(out + t * o_st + (long)hd * o_sh + 4 * tid) = w;
        if (lse && tid == 0) lse[t * lse_st + hd] = lt == 0.f ? -INFINITY : mm + logf(lt);
    }
}

// ---- launch shapes: host integers only, so that a captured call keeps them ----
static int clampi(long x, int lo, int hi) { return (int)(x < lo ? lo : x > hi ? hi : x); }

// A single-token call: about 512 workgroups (two per CU), each of at least 8
// 16-token steps (two per wave).  With `even`, a row's splits hold at most 64 steps:
// lengths differ, and the longest split is the call's time (32 ragged requests of a
// window of 8192, all on one card when the rule was set: 119 us at 2 splits, 96.5 at
// 9, 103 at 17; 93-94 now), up to 4096 workgroups.  64 splits at most: one row of 1M
// tokens at two kv heads has 128 workgroups on 256 CUs.
static int decode_splits(int n_req, int n_kv, long max_keys, bool even) {
    const long rows = (long)n_req * n_kv, steps = (max_keys + 15) / 16;
    const long fill = (512 + rows - 1) / rows, cap = (4096 + rows - 1) / rows;
    const long most = !even ? 1 : (steps + 63) / 64 < cap ? (steps + 63) / 64 : cap;
    return clampi(fill > most ? fill : most, 1, clampi((steps + 7) / 8, 1, 64));
}
// Tiles of k non-empty requests (groups) of n tokens together: sum of ceil(c / TQ)
// <= floor((n - k) / TQ) + k, largest where all are non-empty.
static long prefill_tiles(int n_tokens, int n_req, int G) {
    const int k = n_req < n_tokens ? n_req : n_tokens;
    return (long)(n_tokens - k) / (AT_ROWS / G) + k;
}
// Many tokens: one split once there are 256 workgroups, else about 512 of at
// least 4 key tiles.
static int prefill_splits(long tiles, int n_kv, long max_keys, int head_dim) {
    const long wgs = tiles * n_kv, kt = head_dim == 256 ? 32 : 64;
    if (wgs >= 256) return 1;
    return clampi((512 + wgs - 1) / wgs, 1, clampi(max_keys / (4 * kt), 1, 64));
}
// A prefix: one workgroup per CU, the other place on it is for the own keys (64
// requests on 32K tokens: 16 splits 82 us, 32 88, 8 106).
static int shared_splits(long tiles, int n_kv, long max_keys, int head_dim) {
    const long wgs = tiles * n_kv, kt = head_dim == 256 ? 32 : 64;
    return clampi((256 + wgs - 1) / wgs, 1, clampi(max_keys / (4 * kt), 1, 64));
}
static int64_t part_bytes(int64_t rows, int splits, int D) { return rows * splits * (D + 2) * 4; }
static Partials layout(void* ws, int64_t rows, int splits, int D) {
    float* acc = static_cast<float*>(ws);   // first: 16-byte aligned
    return Partials{acc + rows * splits * D, acc + rows * splits * (D + 1), acc, splits};
}

static int launch_merge(const Partials& p, uint16_t* out, long o_st, long o_sh, float* lse, long lse_st, int n_tok,
                        int n_kv, int G, int head_dim, const int* starts, int n_seq, hipStream_t st) {
#define LAUNCH_D(DV)                                                                                            \
    hipLaunchKernelGGL(attn_merge_kernel<DV>, dim3((unsigned)n_tok * n_kv * G), dim3(AM_BLK), 0, st, p, out, o_st, \
                       o_sh, lse, lse_st, n_kv, G, starts, n_seq)
    if (head_dim == 64) LAUNCH_D(64);
    else if (head_dim == 128) LAUNCH_D(128);
    else LAUNCH_D(256);
#undef LAUNCH_D
    return check_launch("attn_merge_kernel");
}

}  // namespace locks

using namespace locks;

// What every entry asks of its arguments.
static int32_t check_attn(const char* what, const uint16_t* q, int64_t q_st, int64_t q_sh, const uint16_t* k,
                          const int64_t* ks, const uint16_t* v, const int64_t* vs, int32_t num_blocks,
                          const int32_t* bt, int64_t bt_stride, int32_t bt_cols, const int32_t* seq_lens, int32_t window,
                          int32_t sinks, const uint16_t* out, int64_t o_st, int64_t o_sh, int32_t n_req, int32_t n_kv,
                          int32_t G, int32_t head_dim, int32_t page, int32_t max_keys, float scale)
{
    LOCKS_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "%s: head_dim %d outside {64, 128, 256}", what, head_dim);
    LOCKS_REQUIRE(page == 16 || page == 32 || page == 64, "%s: page %d outside {16, 32, 64}", what, page);
    LOCKS_REQUIRE(G >= 1 && G <= 16, "%s: G=%d outside [1, 16]", what, G);
    LOCKS_REQUIRE(n_kv >= 1 && n_kv <= 4096 && n_req >= 0 && n_req <= 65535, "%s: n_kv %d / n_req %d outside [1, 4096] / [0, 65535]", what, n_kv, n_req);
    LOCKS_REQUIRE(num_blocks >= 1 && bt_cols >= 1 && bt_stride >= 0, "%s: empty geometry", what);
    LOCKS_REQUIRE((int64_t)bt_cols * page <= 0x7fffffc0LL, "%s: %d columns of %d tokens pass 32-bit positions", what, bt_cols, page);
    LOCKS_REQUIRE(window >= 0 && sinks >= 0 && max_keys >= 0, "%s: window %d, sinks %d and max_seq_len %d must not be negative", what, window, sinks, max_keys);
    LOCKS_REQUIRE(scale > 0.f && scale <= 3.4e38f, "%s: scale must be positive and finite", what);
    LOCKS_REQUIRE(q && k && v && bt && seq_lens && out, "%s: null pointer argument", what);
    for (int64_t x : {q_st, q_sh, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2]})
        LOCKS_REQUIRE(x % 8 == 0, "%s: q/K/V strides must be multiples of 8 elements (16-byte loads)", what);
    for (int64_t x : {ks[1], vs[1]})
        LOCKS_REQUIRE(x >= 0 && x < (1 << 24), "%s: K/V token strides must be in [0, 2^24) elements", what);
    LOCKS_REQUIRE(o_st % 4 == 0 && o_sh % 4 == 0, "%s: out strides must be multiples of 4 elements", what);
    LOCKS_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (uintptr_t)out % 8 == 0,
                  "%s: q, K and V must be 16-byte aligned, out 8-byte", what);
    return 0;
}
static int32_t check_ws(const char* what, const void* ws, int64_t have, int64_t need)
{
    LOCKS_REQUIRE(need == 0 || (ws && (uintptr_t)ws % 16 == 0), "%s: the workspace is null or not 16-byte aligned", what);
    LOCKS_REQUIRE(have >= need, "%s: the workspace has %lld bytes, the call needs %lld (locks_attn_workspace_bytes)", what,
                  (long long)have, (long long)need);
    return 0;
}
static long bound_keys(int32_t max_seq_len, int32_t bt_cols, int32_t page) {
    const long cap = (long)bt_cols * page;
    return max_seq_len > 0 && max_seq_len < cap ? max_seq_len : cap;
}

extern "C" int64_t locks_attn_workspace_bytes(int32_t max_reqs, int32_t max_tokens, int32_t n_kv, int32_t G,
                                              int32_t head_dim)
{
    if (max_reqs < 0 || max_tokens < 0 || n_kv < 1 || G < 1 || G > 16 || head_dim < 1) return 0;
    const long long_row = 0x7fffffc0L;
    int64_t most = 0;
    // single-token calls of up to max_reqs requests, with a prefix (of one group:
    // more of them make fewer splits); calls of many tokens, of one request (ditto)
    for (int n = 1; n <= (max_reqs < 65535 ? max_reqs : 65535); ++n) {
        const int64_t alone = part_bytes((int64_t)n * n_kv * G, decode_splits(n, n_kv, long_row, true), head_dim);
        most = alone > most ? alone : most;
        const int own = decode_splits(n, n_kv, long_row, false);
        const int shr = shared_splits(prefill_tiles(n, 1, G), n_kv, long_row, head_dim);
        const int64_t b = part_bytes((int64_t)n * n_kv * G, own + shr, head_dim);
        most = b > most ? b : most;
    }
    for (int n = 1; n <= max_tokens && prefill_tiles(n, 1, G) * n_kv < 256; ++n) {
        const int64_t b = part_bytes((int64_t)n * n_kv * G, prefill_splits(prefill_tiles(n, 1, G), n_kv, long_row, head_dim), head_dim);
        most = b > most ? b : most;
    }
    return most;
}

extern "C" int32_t locks_window_decode(
    const uint16_t* q, int64_t q_stride_req, int64_t q_stride_head, const uint16_t* k_cache, int64_t k_stride_block,
    int64_t k_stride_tok, int64_t k_stride_head, const uint16_t* v_cache, int64_t v_stride_block, int64_t v_stride_tok,
    int64_t v_stride_head, int32_t num_blocks, const int32_t* block_table, int64_t bt_stride, int32_t bt_cols,
    const int32_t* seq_lens, int32_t window, int32_t sinks, uint16_t* out, int64_t out_stride_req,
    int64_t out_stride_head, float* lse, int64_t lse_stride_req, void* workspace, int64_t workspace_bytes,
    int32_t n_req, int32_t n_kv, int32_t G, int32_t head_dim, int32_t page, int32_t max_seq_len, float scale, void* stream)
{
    const char* what = "locks_window_decode";
    const int64_t ks64[3] = {k_stride_block, k_stride_tok, k_stride_head}, vs64[3] = {v_stride_block, v_stride_tok, v_stride_head};
    int rc = check_attn(what, q, q_stride_req, q_stride_head, k_cache, ks64, v_cache, vs64, num_blocks, block_table, bt_stride,
                        bt_cols, seq_lens, window, sinks, out, out_stride_req, out_stride_head, n_req, n_kv, G, head_dim,
                        page, max_seq_len, scale);
    if (rc) return rc;
    if (n_req == 0) return 0;
    long keys = bound_keys(max_seq_len, bt_cols, page);
    if (window && (long)window + sinks + 32 < keys) keys = (long)window + sinks + 32;
    const int ns = decode_splits(n_req, n_kv, keys, true);
    const int64_t rows = (int64_t)n_req * n_kv * G;
    rc = check_ws(what, workspace, workspace_bytes, part_bytes(rows, ns, head_dim));
    if (rc) return rc;
    const Partials p = layout(workspace, rows, ns, head_dim);
    const long ks[3] = {k_stride_block, k_stride_tok, k_stride_head}, vs[3] = {v_stride_block, v_stride_tok, v_stride_head};
    hipStream_t st = (hipStream_t)stream;
    rc = launch_decode_range(q, q_stride_req, q_stride_head, k_cache, ks, v_cache, vs, num_blocks, block_table, bt_stride,
                             bt_cols, seq_lens, p, RangeSrc{window, sinks}, ns, 4, n_req, n_kv, G,
                             head_dim, page, scale, st);
    if (rc) return rc;
    return launch_merge(p, out, out_stride_req, out_stride_head, lse, lse_stride_req, n_req, n_kv, G, head_dim, nullptr, 0, st);
}

#define AT_LAUNCH(SHARED, PART)                                                                                     \
    do {                                                                                                            \
        if (head_dim == 64) hipLaunchKernelGGL((attn_tile_kernel<64, SHARED, PART>), grid, dim3(AT_BLK), 0, st, a);  \
        else if (head_dim == 128) hipLaunchKernelGGL((attn_tile_kernel<128, SHARED, PART>), grid, dim3(AT_BLK), 0, st, a); \
        else hipLaunchKernelGGL((attn_tile_kernel<256, SHARED, PART>), grid, dim3(AT_BLK), 0, st, a);                \
    } while (0)

extern "C" int32_t locks_window_prefill(
    const uint16_t* q, int64_t q_stride_tok, int64_t q_stride_head, const uint16_t* k_cache, int64_t k_stride_block,
    int64_t k_stride_tok, int64_t k_stride_head, const uint16_t* v_cache, int64_t v_stride_block, int64_t v_stride_tok,
    int64_t v_stride_head, int32_t num_blocks, const int32_t* block_table, int64_t bt_stride, int32_t bt_cols,
    const int32_t* seq_lens, const int32_t* query_start_loc, int32_t window, int32_t sinks, uint16_t* out,
    int64_t out_stride_tok, int64_t out_stride_head, float* lse, int64_t lse_stride_tok, void* workspace,
    int64_t workspace_bytes, int32_t n_tokens, int32_t n_req, int32_t n_kv, int32_t G, int32_t head_dim, int32_t page,
    int32_t max_seq_len, float scale, void* stream)
{
    const char* what = "locks_window_prefill";
    const int64_t ks64[3] = {k_stride_block, k_stride_tok, k_stride_head}, vs64[3] = {v_stride_block, v_stride_tok, v_stride_head};
    int rc = check_attn(what, q, q_stride_tok, q_stride_head, k_cache, ks64, v_cache, vs64, num_blocks, block_table, bt_stride,
                        bt_cols, seq_lens, window, sinks, out, out_stride_tok, out_stride_head, n_req, n_kv, G, head_dim,
                        page, max_seq_len, scale);
    if (rc) return rc;
    LOCKS_REQUIRE(query_start_loc, "%s: null pointer argument", what);
    LOCKS_REQUIRE(n_tokens >= 0, "%s: n_tokens %d < 0", what, n_tokens);
    if (n_req == 0 || n_tokens == 0) return 0;
    const long keys = window ? (long)window + sinks + n_tokens : bound_keys(max_seq_len, bt_cols, page);
    const long tiles = prefill_tiles(n_tokens, n_req, G);
    int ns = prefill_splits(tiles, n_kv, keys < bound_keys(max_seq_len, bt_cols, page) ? keys : bound_keys(max_seq_len, bt_cols, page), head_dim);
    const int64_t rows = (int64_t)n_tokens * n_kv * G;
    LOCKS_REQUIRE(tiles * n_kv * ns <= 0x7fffffffL, "%s: too many tokens and heads for one launch", what);
    Partials p{};
    if (ns > 1) {
        rc = check_ws(what, workspace, workspace_bytes, part_bytes(rows, ns, head_dim));
        if (rc) return rc;
        p = layout(workspace, rows, ns, head_dim);
    }
    const TileArgs a{q, q_stride_tok, q_stride_head, k_cache, k_stride_block, k_stride_tok, k_stride_head, v_cache,
                     v_stride_block, v_stride_tok, v_stride_head, block_table, bt_stride, seq_lens, query_start_loc, nullptr,
                     out, out_stride_tok, out_stride_head, lse, lse_stride_tok, p, scale * kLog2e, scale, num_blocks, bt_cols,
                     n_tokens, n_req, n_kv, G, page == 16 ? 4 : page == 32 ? 5 : 6, window, sinks, ns, 0, 0, 0, 1};
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)(tiles * n_kv * ns));
    if (ns == 1) { AT_LAUNCH(false, false); return check_launch("attn_tile_kernel"); }
    AT_LAUNCH(false, true);
    rc = check_launch("attn_tile_kernel<part>");
    if (rc) return rc;
    return launch_merge(p, out, out_stride_tok, out_stride_head, lse, lse_stride_tok, n_tokens, n_kv, G, head_dim,
                        query_start_loc, n_req, st);
}

extern "C" int32_t locks_prefix_decode(
    const uint16_t* q, int64_t q_stride_req, int64_t q_stride_head, const uint16_t* k_cache, int64_t k_stride_block,
    int64_t k_stride_tok, int64_t k_stride_head, const uint16_t* v_cache, int64_t v_stride_block, int64_t v_stride_tok,
    int64_t v_stride_head, int32_t num_blocks, const int32_t* block_table, int64_t bt_stride, int32_t bt_cols,
    const int32_t* seq_lens, const int32_t* group_start, const int32_t* prefix_pages, int32_t n_groups, uint16_t* out,
    int64_t out_stride_req, int64_t out_stride_head, float* lse, int64_t lse_stride_req, void* workspace,
    int64_t workspace_bytes, int32_t n_req, int32_t n_kv, int32_t G, int32_t head_dim, int32_t page,
    int32_t max_prefix_pages, int32_t max_seq_len, float scale, void* stream)
{
    const char* what = "locks_prefix_decode";
    const int64_t ks64[3] = {k_stride_block, k_stride_tok, k_stride_head}, vs64[3] = {v_stride_block, v_stride_tok, v_stride_head};
    int rc = check_attn(what, q, q_stride_req, q_stride_head, k_cache, ks64, v_cache, vs64, num_blocks, block_table, bt_stride,
                        bt_cols, seq_lens, 0, 0, out, out_stride_req, out_stride_head, n_req, n_kv, G, head_dim, page,
                        max_seq_len, scale);
    if (rc) return rc;
    LOCKS_REQUIRE(group_start && prefix_pages, "%s: null pointer argument", what);
    LOCKS_REQUIRE(n_groups >= 1 && n_groups <= 65535, "%s: n_groups %d outside [1, 65535]", what, n_groups);
    LOCKS_REQUIRE(max_prefix_pages >= 0, "%s: max_prefix_pages %d < 0", what, max_prefix_pages);
    if (n_req == 0) return 0;
    const long keys = bound_keys(max_seq_len, bt_cols, page);
    const long pre = max_prefix_pages ? (long)max_prefix_pages * page : keys;
    const long tiles = prefill_tiles(n_req, n_groups, G);
    const int own = decode_splits(n_req, n_kv, keys, false), shr = shared_splits(tiles, n_kv, pre < keys ? pre : keys, head_dim);
    const int64_t rows = (int64_t)n_req * n_kv * G;
    LOCKS_REQUIRE((tiles * shr + (long)n_req * own) * n_kv <= 0x7fffffffL, "%s: too many requests and heads for one launch", what);
    rc = check_ws(what, workspace, workspace_bytes, part_bytes(rows, own + shr, head_dim));
    if (rc) return rc;
    const Partials p = layout(workspace, rows, own + shr, head_dim);
    const TileArgs a{q, q_stride_req, q_stride_head, k_cache, k_stride_block, k_stride_tok, k_stride_head, v_cache,
                     v_stride_block, v_stride_tok, v_stride_head, block_table, bt_stride, seq_lens, group_start, prefix_pages,
                     nullptr, 0, 0, nullptr, 0, p, scale * kLog2e, scale, num_blocks, bt_cols, n_req, n_groups, n_kv, G,
                     page == 16 ? 4 : page == 32 ? 5 : 6, 0, 0, shr, own, (int)(tiles * shr), n_req * own,
                     n_kv < 256 ? 256 / n_kv : 1};
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)((tiles * shr + (long)n_req * own) * n_kv));
    AT_LAUNCH(true, true);
    rc = check_launch("attn_tile_kernel<shared>");
    if (rc) return rc;
    return launch_merge(p, out, out_stride_req, out_stride_head, lse, lse_stride_req, n_req, n_kv, G, head_dim, nullptr, 0, st);
}
