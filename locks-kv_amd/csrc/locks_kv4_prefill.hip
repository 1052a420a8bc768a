// Attention of many tokens over a paged cache in 4 bits.
//
// Mathematics and visibility as in locks_window.hip, over the values that the codes
// stand for.  A workgroup of 4 waves holds 128 query rows (token, head of the group), 32
// per wave, and walks over tiles of 64 keys:
//   S^T = K Q^T (32x32x16 bf16 MFMA): a lane holds 32 keys of ONE query, so maximum and
//     sum are in the lane plus one swap with lane ^ 32;
//   O^T += V^T P^T: a lane's weights are the operand as they stand, V comes out of LDS
//     transposed (ds_read_b64_tr_b16).
// A tile is converted to bf16 once for its 128 rows: each wave takes 16 keys' codes to
// registers two tiles ahead, and writes their rows to LDS, K a tile before V.
//
// Matrix products and softmax are about as long as each other, and a wave that does
// them in turn leaves both units half idle.  So at d 128 and 256 they are skewed by a tile:
// the products K(n + 1) Q^T stand between the exponentials of tile n, and V(n) P(n) between
// the maximum of tile n + 1 and the conversion of the tiles behind it, issued alternately.
// 8192 tokens, 32 / 8 heads, d 128, causal: 500 to 533 us, 1030 to 1100 TFLOP/s (in turn,
// with the tiles of locks_window.hip, 555), by the card: its clock falls to 1.8 GHz under
// the call; d 256, 16 / 4 heads, 620 to 630 us (in turn 1080).  Two workgroups a CU at d
// 128, one at d 256 (registers).
// At d 64 a tile has half of the products of d 128 for the same softmax, too few to stand
// between it, and the skew's 215 registers leave a CU two workgroups, where in turn it holds
// three, whose products and softmax overlap.  8192 tokens, 64 / 8 heads: skewed 648 us, in
// turn 603 (with the tiles of locks_window.hip 620); 512 tokens on 16384 keys 98.3 and 96.6,
// ragged window 68.9 and 68.3, 300 tokens 10.4 and 10.5.
// What bounds it, by counters: at d 128 LDS (busy 72 % of the time), the vector units (55)
// and the matrix cores (49) together, and a timing copy without the exponentials took 6 %
// less, without LDS reads 7, without conversion and writes 13; at d 64 the vector units
// (76; LDS 63, matrix cores 40); at d 256 the one wave a SIMD, which waits 31 % of its time
// (LDS 49, vector units 35, matrix cores 35).
#include "locks_attn.h"
#include "locks_common.h"
#include "locks_hip.h"
#include "locks_kv4.h"

#include <math.h>

#include <type_traits>

namespace locks {

constexpr int P4_WAVES = 4;
constexpr int P4_BLK = P4_WAVES * kWave;
// (16 keys of a tile are a wave's to convert)
static_assert(AT_ROWS == 32 * P4_WAVES && P4_KT == 16 * P4_WAVES, "rows and keys of a workgroup");
// Whether a tile's products and softmax are skewed, and the workgroups that a CU has
// registers for.
constexpr bool p4_skewed(int head_dim) { return head_dim != 64; }
constexpr int p4_resident(int head_dim) { return head_dim == 256 ? 1 : p4_skewed(head_dim) ? 2 : 3; }

template <int D>
struct P4Geom {
    static constexpr int ROWB = 2 * D, TILEB = P4_KT * ROWB;       // bytes of a row, of a tile
    // 16-byte chunks of a row are permuted by the row (an exclusive or): K is read 16 rows
    // at one chunk, V 4 rows at 4 chunks, both free of bank conflicts
    static __device__ __forceinline__ int swz_k(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
    static __device__ __forceinline__ int swz_v(int row) { return D == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }
};

struct Kv4PrefillArgs {
    const uint16_t* q; long q_st, q_sh;
    const uint8_t* c; long c_sb, c_sh;      // bytes
    const int* bt; long bt_sr;
    const int* seq_lens;
    const int* starts;                      // first token of each request
    uint16_t* out; long o_st, o_sh;
    float* lse; long lse_st;
    Partials p;
    float scale_log2, scale;
    int NB, bt_cols, n_rows, n_seq, n_kv, G, pg_sh, window, sinks, nsplit;
};

// PART: partials instead of the output.
template <int D, bool PART>
__global__ __launch_bounds__(P4_BLK, p4_resident(D)) void kv4_prefill_kernel(const Kv4PrefillArgs a)
{
    using GM = P4Geom<D>;
    constexpr int KT = P4_KT, ROWB = GM::ROWB, ND = D / 32;
    // (an array for each buffer: the compiler can tell one's writes from another's reads)
    __shared__ __attribute__((aligned(1024))) uint8_t k0[GM::TILEB], k1[GM::TILEB], v0[GM::TILEB], v1[GM::TILEB];
    __shared__ int wlim[P4_WAVES][4];
    __shared__ int nan_s[2][P4_WAVES];                  // a block of V in the buffer is NaN ...
    __shared__ uint8_t nan_k[2][KT][D / 32];            // and which ones of a key
    auto kbuf = [&](auto i) __attribute__((always_inline)) { return i() == 0 ? k0 : k1; };
    auto vbuf = [&](auto i) __attribute__((always_inline)) { return i() == 0 ? v0 : v1; };
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c32 = lane & 31, h = lane >> 5;
    const int G = a.G, TQ = AT_ROWS / G;                // tokens per tile of rows
    const int kh = blockIdx.x % a.n_kv;
    const int unit = blockIdx.x / a.n_kv;
    const int sp = unit % a.nsplit, tile = unit / a.nsplit;

    // the request that holds this tile of rows
    int seq = -1, t_in = 0, first = 0, count = 0, len = 0;         // len: tokens before the first row
    for (int s0 = 0, done = 0; s0 < a.n_seq && seq < 0; s0 += kWave) {
        const int s = min(s0 + lane, a.n_seq - 1);
        const int at = a.starts[s], end = a.starts[s + 1], len_s = a.seq_lens[s];
        const int f = max(at, 0), n = s0 + lane < a.n_seq ? max(min(end, a.n_rows) - f, 0) : 0;
        const int nt = (n + TQ - 1) / TQ;
        const int inc = wave_incl_scan_i(nt);
        const unsigned long long hit = __ballot(done + inc > tile);
        if (hit) {
            const int l = __ffsll(hit) - 1;
            seq = s0 + l;
            first = __builtin_amdgcn_readlane(f, l);
            count = __builtin_amdgcn_readlane(n, l);
            len = __builtin_amdgcn_readlane(len_s - (end - at), l);
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
    const int pos = len + j, sinks = a.sinks;
    const int hi = valid ? (int)min((long)pos + 1, cap) : 0x7fffffff;
    const int lo = valid && a.window ? max(pos - a.window + 1, 0) : 0;
    // of the wave's valid rows, then of the workgroup's
    const int w_min_hi = __builtin_amdgcn_readfirstlane(wave_min_int(hi));
    const int w_max_lo = __builtin_amdgcn_readfirstlane(wave_max_int(lo));
    if (lane == 0) { wlim[wave][0] = w_min_hi; wlim[wave][2] = w_max_lo; }
    {
        const int w_max_hi = wave_max_int(valid ? hi : 0), w_min_lo = wave_min_int(valid ? lo : 0x7fffffff);
        if (lane == 0) { wlim[wave][1] = w_max_hi; wlim[wave][3] = w_min_lo; }
    }
    __syncthreads();
    int min_hi = wlim[0][0], max_hi = wlim[0][1], max_lo = wlim[0][2], min_lo = wlim[0][3];
#pragma unroll
    for (int w = 1; w < P4_WAVES; ++w) {
        min_hi = min(min_hi, wlim[w][0]); max_hi = max(max_hi, wlim[w][1]);
        max_lo = max(max_lo, wlim[w][2]); min_lo = min(min_lo, wlim[w][3]);
    }
    min_hi = __builtin_amdgcn_readfirstlane(min_hi); max_hi = __builtin_amdgcn_readfirstlane(max_hi);
    max_lo = __builtin_amdgcn_readfirstlane(max_lo); min_lo = __builtin_amdgcn_readfirstlane(min_lo);

    // key tiles: the first na, then [b0, b1); this split's share [n0, n1) of them
    const int na = (min(min(sinks, min_lo), max(max_hi, 0)) + KT - 1) / KT;
    const int b0 = max(min_lo / KT, na), b1 = (int)(((long)max_hi + KT - 1) / KT);
    const int nt = max_hi > 0 ? na + max(b1 - b0, 0) : 0;
    const int n0 = (int)((long)nt * sp / a.nsplit), n1 = (int)((long)nt * (sp + 1) / a.nsplit);
    auto key_of = [&](int n) __attribute__((always_inline)) { return (n < na ? n : b0 + n - na) * KT; };

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

    // This wave's 16 keys of a tile lie on one page: the addresses of 64 tiles' are made
    // at once, one per lane.
    const int last_page = max((int)(((long)max_hi + (1L << a.pg_sh) - 1) >> a.pg_sh) - 1, 0);
    uint32_t at_lo = 0, at_hi = 0;
    int n_of = 0;
    auto fetch = [&](int n) __attribute__((always_inline)) {
        n_of = n;
        const int key = key_of(min(n + lane, max(n1 - 1, n))) + 16 * wave;
        const int pg = min(min(key >> a.pg_sh, last_page), a.bt_cols - 1);
        const int id = min(max(a.bt[(long)seq * a.bt_sr + pg], 0), a.NB - 1);
        const uint64_t at = (uint64_t)a.c + (uint64_t)((long)id * a.c_sb + (long)kh * a.c_sh +
                                                       ((key >> 4) & ((1 << (a.pg_sh - 4)) - 1)) * Kv4<D>::TILE);
        at_lo = (uint32_t)at;
        at_hi = (uint32_t)(at >> 32);
    };
    auto tile_at = [&](int n) __attribute__((always_inline)) {
        return (kv4_ptr)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(at_lo, n - n_of) |
                         (uint64_t)(uint32_t)__builtin_amdgcn_readlane(at_hi, n - n_of) << 32);
    };
    // K of tile n and V of the one before it, whose addresses are kept that long
    Kv4Lane<D> ck{}, cv{};
    auto load_codes = [&](int nk, int nv) __attribute__((always_inline)) {
        if (nk - n_of >= kWave) fetch(nv);
        if (nk < n1) kv4_load_k<D, false>(tile_at(nk), lane, ck);
        if (nv < n1) kv4_load_v<D, false>(tile_at(nv), lane, cv);
    };
    const int r16 = lane & 15, kg = lane >> 4;
    auto put = [&](uint8_t* buf, int row, int chunk, int swz, const uint4& x) __attribute__((always_inline)) {
        *reinterpret_cast<uint4*>(buf + row * ROWB + ((chunk ^ swz) * 16)) = x;
    };
    // A tile's rows in items of one or two words of codes: K's, entries kg D / 4 .. of one
    // key, and V's, entries r16 D / 16 .. of four keys.
    constexpr int KI = D / 32, VI = D == 256 ? 8 : 4;
    auto write_k = [&](uint8_t* kb, const Kv4Lane<D>& ck, int st) __attribute__((always_inline)) {
        const int row = 16 * wave + r16;
        put(kb, row, kg * KI + st, GM::swz_k(row), kv4_eight(ck.w[st], kv4_scale(ck.s, D == 256 ? st >> 2 : 0)));
    };
    auto write_v = [&](uint8_t* vb, const Kv4Lane<D>& cv, int item) __attribute__((always_inline)) {
        const int i = D == 256 ? item >> 1 : item, row = 16 * wave + 4 * kg + i;
        const float sc = kv4_scale(cv.s, i);
        if constexpr (D == 64) {
            const uint32_t w = cv.w[i >> 1];
            const uint2 x = (i & 1) ? make_uint2(kv4_pair<2>(w, sc), kv4_pair<3>(w, sc))
                                    : make_uint2(kv4_pair<0>(w, sc), kv4_pair<1>(w, sc));
            *reinterpret_cast<uint2*>(vb + row * ROWB + (((r16 >> 1) ^ GM::swz_v(row)) * 16) + (r16 & 1) * 8) = x;
        } else {
            const int j = D == 256 ? item & 1 : 0;
            put(vb, row, r16 * (D / 128) + j, GM::swz_v(row), kv4_eight(cv.w[i * (D / 128) + j], sc));
        }
    };
    // A tile that some row sees only part of.
    auto part = [&](int n) __attribute__((always_inline)) {
        const int key0 = key_of(n);
        return key0 + KT > min_hi || (key0 < max_lo && key0 + KT > sinks);
    };
    // Blocks of V that are not finite must not reach the sums from masked places (0 x NaN):
    // NaN ones, and those of scales past a write's (bytes 253 and 254 in memory that nobody
    // wrote: 4 * 2^126 is infinite in bf16).  In such a tile they are written as zeros, and
    // noted: `nans` has a bit for each 32 columns that are so in a key that this lane's row
    // sees.
    auto clear_nan = [&](int n, Kv4Lane<D>& cv, int buf) __attribute__((always_inline)) {
        // a byte of 253 and more: 0x7D and more below its top bit, which is set
        const bool any = __any((((cv.s & 0x7F7F7F7Fu) + 0x03030303u) & cv.s & 0x80808080u) != 0);
        if (lane == 0) nan_s[buf][wave] = any;
        if (any && part(n)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool bad = (cv.s >> (8 * i) & 255u) >= 253u;
                if (r16 % (512 / D) == 0) nan_k[buf][16 * wave + 4 * kg + i][r16 / (512 / D)] = bad;
                cv.s &= bad ? ~(255u << (8 * i)) : ~0u;
                if constexpr (D == 64) cv.w[i >> 1] &= !bad ? ~0u : (i & 1) ? 0xFFFFu : 0xFFFF0000u;
                else
#pragma unroll
                    for (int x = 0; x < D / 128; ++x) cv.w[i * (D / 128) + x] &= bad ? 0u : ~0u;
            }
        }
    };
    uint32_t nans = 0;
    auto note_nan = [&](int n, int buf) __attribute__((always_inline)) {
        if (!part(n)) return;
        const volatile int* f = nan_s[buf];
        if (!(f[0] | f[1] | f[2] | f[3])) return;
        const int key0 = key_of(n);
#pragma unroll 1
        for (int kk = 0; kk < KT; ++kk) {
            if (!f[kk >> 4]) continue;
            const int key = key0 + kk;
            const bool seen = valid && key < hi && (key >= lo || key < sinks);
            for (int b = 0; b < ND; ++b) nans |= seen && nan_k[buf][kk][b] ? 1u << b : 0u;
        }
    };

    float m = -INFINITY, l = 0.f, l1 = 0.f;             // raw score units; this half-wave's keys, even and odd
    v16f o[ND];
#pragma unroll
    for (int b = 0; b < ND; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] = 0.f;

    // K row c32 (+ 32 kb): chunk (2 s + h) ^ swz, whose bits of s are one exclusive or
    // away; V: rows 4 h + (i >> 2), i = lane & 15, chunks of column block b ditto
    const int i16 = lane & 15;
    const int ka = c32 * ROWB + (h ^ GM::swz_k(c32)) * 16;
    const int va = (4 * h + (i16 >> 2)) * ROWB +
                   ((2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ GM::swz_v(4 * h + (i16 >> 2))) * 16 + (i16 & 1) * 8;
    auto k_frag = [&](const uint8_t* kb, int i) __attribute__((always_inline)) {
        return *reinterpret_cast<const v8bf*>(kb + (ka ^ (i >> 1) * 32) + (i & 1) * 32 * ROWB);
    };
    auto v_frag = [&](const uint8_t* vb, int i) __attribute__((always_inline)) {
        const uint8_t* x = vb + (va ^ (i % ND) * 64) + 16 * (i / ND) * ROWB;
        const v4s x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(x));
        const v4s x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(x + 8 * ROWB));
        return __builtin_bit_cast(v8bf, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    v16f zero;
#pragma unroll
    for (int i = 0; i < 16; ++i) zero[i] = 0.f;
    auto score = [&](const v8bf& kf, int i, v16f* s) __attribute__((always_inline)) {
        s[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[i >> 1], i < 2 ? zero : s[i & 1], 0, 0, 0);
    };
    auto maximum = [&](const v16f* s) __attribute__((always_inline)) {
        float mx = s[0][0];
#pragma unroll
        for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb2][i]);
        return mx;
    };
    // Keys that a row does not see; then m follows the tile's maximum, and what is summed
    // with it, where the maximum grew by 2^8 in weight (until then weights are at most
    // 256, and nothing needs rescaling).
    auto settle = [&](int n, v16f* s, float mx) __attribute__((always_inline)) {
        const int key0 = key_of(n);
        // each side by itself: a compare with a constant and a select per key
        const bool above = key0 + KT > w_min_hi, below = key0 < w_max_lo && key0 + KT > sinks;
        if (above || below) {
            if (above) {
                const int top = hi - key0 - 4 * h;
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    s[i >> 4][i & 15] = 32 * (i >> 4) + 8 * ((i & 15) >> 2) + (i & 3) < top ? s[i >> 4][i & 15] : -INFINITY;
            }
            if (below) {
                const int low = lo - key0 - 4 * h, sink = key0 < sinks ? sinks - key0 - 4 * h : -0x40000000;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const int x = 32 * (i >> 4) + 8 * ((i & 15) >> 2) + (i & 3);
                    s[i >> 4][i & 15] = x >= low || x < sink ? s[i >> 4][i & 15] : -INFINITY;
                }
            }
            mx = maximum(s);
        }
        mx = xor32_max(mx);
        if (__any((mx - m) * a.scale_log2 > 8.f)) {
            const float m_new = fmaxf(m, mx);
            const float al = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * a.scale_log2);
            m = m_new;
            l *= al;
            l1 *= al;
#pragma unroll
            for (int b = 0; b < ND; ++b) o[b] *= al;
        }
    };
    constexpr int NM = D / 8, AHEAD = 2;                // products of each kind of a tile; reads ahead of them
    // Weights in bf16, the product's other operand (half a step, 2^-8 of each); l keeps
    // the unrounded ones.
    auto weight = [&](const v16f* s, v8bf* pf, int i, float mc) __attribute__((always_inline)) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[i >> 4][i & 15], a.scale_log2, -mc));
        (i & 1 ? l1 : l) += p;
        pf[i >> 3][i & 7] = (__bf16)p;
    };
    auto value = [&](const v8bf& vf, const v8bf* pf, int i) __attribute__((always_inline)) {
        o[i % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[i / ND], o[i % ND], 0, 0, 0);
    };
    // Tile n and the scores of the next one: s are n's, settled; V(n) and K(n + 1) are
    // written, the codes of K(n + 2) and V(n + 1) on hand or on their way.
    auto step = [&](int n, v16f* s, v16f* next, auto use, auto fill) __attribute__((always_inline)) {
        lds_barrier();
        note_nan(n, use());
        const float mc = m == -INFINITY ? 0.f : m * a.scale_log2;
        v8bf pf[KT / 16], f[AHEAD];
        // each product with its share of the exponentials, in this order
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) f[i] = k_frag(kbuf(fill), i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            score(f[i % AHEAD], i, next);
            if (i + AHEAD < NM) f[i % AHEAD] = k_frag(kbuf(fill), i + AHEAD);
#pragma unroll
            for (int e = i * 32 / NM; e < (i + 1) * 32 / NM; ++e) {
                weight(s, pf, e, mc);
                // (made here: left to itself the compiler moves them behind the next branch)
                if ((e & 7) == 7) asm volatile("" : "+v"(pf[e >> 3]));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        clear_nan(n + 1, cv, fill());
        // each with its share of the next tile's maximum and of the rows to convert
        // (behind the share's end: of codes that no one reads)
        float mx = next[0][0];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) f[i] = v_frag(vbuf(use), i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            value(f[i % AHEAD], pf, i);
            if (i + AHEAD < NM) f[i % AHEAD] = v_frag(vbuf(use), i + AHEAD);
#pragma unroll
            for (int e = i * 32 / NM; e < (i + 1) * 32 / NM; ++e) mx = fmaxf(mx, next[e >> 4][e & 15]);
#pragma unroll
            for (int x = i * (KI + VI) / NM; x < (i + 1) * (KI + VI) / NM; ++x) {
                if (x < KI) write_k(kbuf(use), ck, x);
                else write_v(vbuf(fill), cv, x - KI);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("" : "+v"(mx));                // (here, not in the branch that reads it)
        load_codes(n + 3, n + 2);
        settle(n + 1, next, mx);
    };
    auto last = [&](int n, const v16f* s, auto use) __attribute__((always_inline)) {
        lds_barrier();
        note_nan(n, use());
        const float mc = m == -INFINITY ? 0.f : m * a.scale_log2;
        v8bf pf[KT / 16];
#pragma unroll
        for (int e = 0; e < 32; ++e) weight(s, pf, e, mc);
#pragma unroll
        for (int i = 0; i < NM; ++i) value(v_frag(vbuf(use), i), pf, i);
    };

    // In turn: K(n) and V(n) are written, the codes of both of n + 1 on hand or on their way.
    auto write_rows = [&](int n, auto buf) __attribute__((always_inline)) {
        clear_nan(n, cv, buf());
#pragma unroll
        for (int x = 0; x < KI; ++x) write_k(kbuf(buf), ck, x);
#pragma unroll
        for (int x = 0; x < VI; ++x) write_v(vbuf(buf), cv, x);
    };
    auto in_turn = [&](int n, auto use, auto fill) __attribute__((always_inline)) {
        lds_barrier();
        if (n + 1 < n1) {
            write_rows(n + 1, fill);
            load_codes(n + 2, n + 2);
        }
        note_nan(n, use());
        v16f s[2];
#pragma unroll
        for (int i = 0; i < NM; ++i) score(k_frag(kbuf(use), i), i, s);
        settle(n, s, maximum(s));
        const float mc = m == -INFINITY ? 0.f : m * a.scale_log2;
        v8bf pf[KT / 16];
#pragma unroll
        for (int e = 0; e < 32; ++e) weight(s, pf, e, mc);
#pragma unroll
        for (int i = 0; i < NM; ++i) value(v_frag(vbuf(use), i), pf, i);
    };

    using I0 = std::integral_constant<int, 0>; using I1 = std::integral_constant<int, 1>;
    if constexpr (!p4_skewed(D)) {
        if (n0 < n1) {
            fetch(n0);
            load_codes(n0, n0);
            write_rows(n0, I0{});
            load_codes(n0 + 1, n0 + 1);
            for (int n = n0; n < n1; n += 2) {
                in_turn(n, I0{}, I1{});
                if (n + 1 < n1) in_turn(n + 1, I1{}, I0{});
            }
        }
    } else if (n0 < n1) {
        v16f s0[2], s1[2];
        fetch(n0);
        load_codes(n0, n0);
        Kv4Lane<D> k_0 = ck, v_0 = cv;
        load_codes(n0 + 1, n0 + 1);                     // (with the first tile's: one wait for both)
#pragma unroll
        for (int x = 0; x < KI; ++x) write_k(k0, k_0, x);
        clear_nan(n0, v_0, 0);
#pragma unroll
        for (int x = 0; x < VI; ++x) write_v(v0, v_0, x);
#pragma unroll
        for (int x = 0; x < KI; ++x) write_k(k1, ck, x);
        if (n0 + 2 < n1) kv4_load_k<D, false>(tile_at(n0 + 2), lane, ck);
        lds_barrier();
#pragma unroll
        for (int i = 0; i < NM; ++i) score(k_frag(k0, i), i, s0);
        settle(n0, s0, maximum(s0));
        int n = n0;
        for (; n + 2 < n1; n += 2) {
            step(n, s0, s1, I0{}, I1{});
            step(n + 1, s1, s0, I1{}, I0{});
        }
        if (n + 1 < n1) {
            step(n, s0, s1, I0{}, I1{});
            last(n + 1, s1, I1{});
        } else {
            last(n, s0, I0{});
        }
    }

    l = xor32_sum(l + l1);
    if (!valid) return;
    if (nans)
#pragma unroll
        for (int b = 0; b < ND; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[b][i] = nans >> b & 1 ? __uint_as_float(0x7FC00000u) : o[b][i];
    if constexpr (PART) {
        const long at = (((long)tok * a.n_kv + kh) * a.p.splits + sp) * G + g;
        if (h == 0) {
            a.p.m[at] = l > 0.f || l != l ? m * a.scale_log2 : -INFINITY;
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

}  // namespace locks

using namespace locks;

extern "C" int32_t locks_kv4_prefill(
    const uint16_t* q, int64_t q_stride_tok, int64_t q_stride_head, const uint8_t* cache, int64_t c_stride_block,
    int64_t c_stride_head, int32_t num_blocks, const int32_t* block_table, int64_t bt_stride, int32_t bt_cols,
    const int32_t* seq_lens, const int32_t* query_start_loc, int32_t window, int32_t sinks, uint16_t* out,
    int64_t out_stride_tok, int64_t out_stride_head, float* lse, int64_t lse_stride_tok, void* workspace,
    int64_t workspace_bytes, int32_t n_tokens, int32_t n_req, int32_t n_kv, int32_t G, int32_t head_dim, int32_t page,
    int32_t max_seq_len, float scale, void* stream)
{
    const char* what = "locks_kv4_prefill";
    int rc = check_kv4(what, cache, c_stride_block, c_stride_head, num_blocks, n_kv, head_dim, page);
    if (rc) return rc;
    // q, out, the table and the lengths: what the bf16 cache's entries ask
    const int64_t none[3] = {0, 0, 0};
    const uint16_t* any = reinterpret_cast<const uint16_t*>(cache);
    rc = check_attn(what, q, q_stride_tok, q_stride_head, any, none, any, none, num_blocks, block_table, bt_stride, bt_cols,
                    seq_lens, window, sinks, out, out_stride_tok, out_stride_head, n_req, n_kv, G, head_dim, page,
                    max_seq_len, scale);
    if (rc) return rc;
    LOCKS_REQUIRE(query_start_loc, "%s: null pointer argument", what);
    LOCKS_REQUIRE(n_tokens >= 0, "%s: n_tokens %d < 0", what, n_tokens);
    if (n_req == 0 || n_tokens == 0) return 0;
    const long bound = bound_keys(max_seq_len, bt_cols, page), reach = (long)window + sinks + n_tokens;
    const long tiles = prefill_tiles(n_tokens, n_req, G);
    const int ns = prefill_splits(tiles, n_kv, window && reach < bound ? reach : bound, P4_KT);
    const int64_t rows = (int64_t)n_tokens * n_kv * G;
    LOCKS_REQUIRE(tiles * n_kv * ns <= 0x7fffffffL, "%s: too many tokens and heads for one launch", what);
    Kv4PrefillArgs a{q, q_stride_tok, q_stride_head, cache, c_stride_block, c_stride_head, block_table, bt_stride, seq_lens,
                     query_start_loc, out, out_stride_tok, out_stride_head, lse, lse_stride_tok, Partials{},
                     scale * kLog2e, scale, num_blocks, bt_cols, n_tokens, n_req, n_kv, G,
                     page == 16 ? 4 : page == 32 ? 5 : 6, window, sinks, ns};
    if (ns > 1) {
        rc = check_ws(what, workspace, workspace_bytes, part_bytes(rows, ns, head_dim));
        if (rc) return rc;
        a.p = part_layout(workspace, rows, ns, head_dim);
    }
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)(tiles * n_kv * ns));
#define P4_LAUNCH(PART)                                                                                                \
    do {                                                                                                               \
        if (head_dim == 64) hipLaunchKernelGGL((kv4_prefill_kernel<64, PART>), grid, dim3(P4_BLK), 0, st, a);           \
        else if (head_dim == 128) hipLaunchKernelGGL((kv4_prefill_kernel<128, PART>), grid, dim3(P4_BLK), 0, st, a);    \
        else hipLaunchKernelGGL((kv4_prefill_kernel<256, PART>), grid, dim3(P4_BLK), 0, st, a);                         \
    } while (0)
    if (ns == 1) P4_LAUNCH(false);
    else P4_LAUNCH(true);
#undef P4_LAUNCH
    rc = check_launch("kv4_prefill_kernel");
    if (rc || ns == 1) return rc;
    return launch_kv4_merge(Kv4MergeArgs{a.p.m, a.p.l, a.p.acc, nullptr, ns, query_start_loc, n_req, out, out_stride_tok,
                                         out_stride_head, lse, lse_stride_tok, n_kv, G}, n_tokens, head_dim, st);
}
