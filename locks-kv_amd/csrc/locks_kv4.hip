// Single-token attention over a paged cache in 4 bits, and its rows read back.
//
// Mathematics: as in locks_window.hip, over the values that the codes stand for.  One
// query per request, at the last position, sees the keys [lo, len) and [0, min(sinks,
// lo)), lo = max(len - window, 0):
//   o = sum_j p_j v_j / l,  p_j = exp(scale q.k_j - m),  l = sum_j p_j,  lse = m + ln l
//
// A wave takes two tiles of 16 keys a step, straight from memory to registers:
//   S^T = K Q^T  (16x16x32 bf16 MFMA, the group's heads in the columns): a lane's
//       codes are its operand, four converted pairs a word;
//   O^T += V^T P^T: a lane's weights are the operand as they stand; its V codes are
//       four keys of d / 16 entries, which pair up by one byte permutation a pair.
// Every wave keeps its own running maximum and sum; the waves of a workgroup join in
// LDS, and the workgroups of a row in kv4_merge_kernel.
//
// Work is dealt out in equal shares (bound by memory, a call is as long as its longest
// workgroup, and lengths are known to the GPU alone): the tiles of all (request, kv
// head) rows in order, K4_ROW tiles' worth more for each row's start, cut into one share
// a workgroup.  A share holds whole rows, whose outputs it writes, and at most an end of
// one row and a start of another, whose partials go to its two slots.
//
// Bound by memory: 17 d bytes for K and V of 16 keys and a head, read once, past the
// caches.  1M keys of 8 heads, d 128: 180 us, 6.3 TB/s; 131072 keys 33 us (28 and the
// merge: the chain of lengths, block ids and first tiles, and the join, are 10 of them); 32
// requests of 1 to 32768 keys 54 us, 5.3 TB/s.  Two workgroups a CU, two steps on their
// way: 70 KB a CU, more than latency x rate needs (three and four steps, and three
// workgroups, were slower).  At d 64 a step has 0.7 of d 128's vector instructions for half
// of the bytes: 1M keys 111 us, 5.1 TB/s, the vector units busy 55 % of the time (d 128 48,
// d 256 38) and waves waiting for half of theirs.
#include "locks_attn.h"
#include "locks_common.h"
#include "locks_hip.h"
#include "locks_kv4.h"

#include <math.h>

#include <type_traits>

namespace locks {

constexpr int K4_WAVES = 4;
constexpr int K4_BLK = K4_WAVES * kWave;
constexpr int K4_TILES = 2;                 // of a wave's step
constexpr int K4_ROW = 32;                  // a row's start (query, first loads, output) in tiles' time
constexpr int K4_SHARE = 24;                // tiles that a share has at least
// Workgroups that a CU has registers for: at d 64 128 of them do (300 requests of 1500 keys
// 56.1 us with three workgroups a CU, 51.3 with four).
constexpr int kv4_resident(int head_dim) { return head_dim == 64 ? 4 : 2; }
// Shares at most: two workgroups a CU, or three at d 64, whose waves have more to issue for
// their bytes (1M keys of 8 heads 122 -> 111 us, 64 requests of 4096 41.0 -> 37.5, of 1500
// 23.3 -> 21.9; four 110 and 37.1).  Calls between cost up to 3 % by it: with 4 heads 16
// requests of 3000 keys 13.0 -> 13.3, 32 of 2000 14.5 -> 14.9, 131072 keys 18.2 -> 18.7.
// Three cost more than they give at d 128 (131072 keys 33.2 -> 37.9 us) and where a group's
// partials are large (16 heads 19.7 -> 21.0).
static int kv4_grid(int head_dim, int G) { return head_dim == 64 && G <= 8 ? 768 : 512; }
constexpr float kLn2 = 0.69314718055994530942f;

struct Kv4DecodeArgs {
    const uint16_t* q; long q_sr, q_sh;
    const uint8_t* c; long c_sb, c_sh;              // bytes
    const int* bt; long bt_sr;
    const int* seq_lens;
    uint16_t* out; long o_sr, o_sh;
    float* lse; long lse_sr;
    // partials by slot (two a share) and head of the group, and the shares of each row
    float* m; float* l; float* acc; int2* shares;
    float scale_log2;
    double inv_grid;                                // 1 / workgroups
    int NB, bt_cols, n_req, n_kv, G, pg_sh, window, sinks;
    bool rows;                                      // a workgroup for each row: no shares, no partials
};

// The keys that a request's query sees, as tiles: the first na, then [b0, b0 + nt - na).
struct Kv4Row {
    int len, lo, sinks, na, b0, nt;
    __device__ __forceinline__ Kv4Row(const Kv4DecodeArgs& a, int seq_len) {
        const long cap = (long)a.bt_cols << a.pg_sh, full = max(seq_len, 0);
        len = (int)min(full, cap);
        // (a length past the table: the window still ends at it)
        lo = a.window ? (int)min(max(full - a.window, 0L), (long)len) : 0;
        sinks = min(a.sinks, lo);
        na = (sinks + 15) >> 4;
        b0 = max(lo >> 4, na);
        nt = na + max(((len + 15) >> 4) - b0, 0);
    }
    __device__ __forceinline__ int cost() const { return K4_ROW + max(nt, 1); }
};

// A value that every lane holds, in scalar registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long uniform(long x) {
    return (long)((uint64_t)(uint32_t)uniform((int)x) | (uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32);
}

// Inclusive prefix sums over the wave, as wave_incl_scan_i.
__device__ __forceinline__ double wave_incl_scan(double v) {
    auto shifted = [](double x, auto ctrl, auto rows) __attribute__((always_inline)) {
        const long u = __double_as_longlong(x);
        const int lo = __builtin_amdgcn_update_dpp(0, (int)u, ctrl(), rows(), 0xf, false);
        const int hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), ctrl(), rows(), 0xf, false);
        return __longlong_as_double((long)((uint64_t)(uint32_t)lo | (uint64_t)(uint32_t)hi << 32));
    };
    using All = std::integral_constant<int, 0xf>;
    v += shifted(v, std::integral_constant<int, 0x111>{}, All{});
    v += shifted(v, std::integral_constant<int, 0x112>{}, All{});
    v += shifted(v, std::integral_constant<int, 0x114>{}, All{});
    v += shifted(v, std::integral_constant<int, 0x118>{}, All{});
    v += shifted(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
    v += shifted(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
    return v;
}

// The low (high) halves of two words as one, a's below b's.
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// WV waves: 4, or 8 where a workgroup has a row and a CU to itself (a step is some 260
// instructions one after the other, 1 us for a wave alone on its SIMD).
template <int D, int WV>
__global__ __launch_bounds__(WV * kWave, WV == 4 ? kv4_resident(D) : 1) void kv4_decode_kernel(const Kv4DecodeArgs a)
{
    constexpr int BLK = WV * kWave;
    using L = Kv4<D>;
    constexpr int ND = D / 16, W = L::W, T = K4_TILES;
    __shared__ float m_s[WV][16], l_s[WV][16];
    __shared__ __attribute__((aligned(16))) float o_s[WV][16][D + 4];
    __shared__ double sum_s[WV];
    __shared__ long at_s[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15, kg = lane >> 4;
    const int G = a.G;

    // this workgroup's share [lo, hi) of all rows' cost, and the row that it starts in
    int r = 0, kh = 0;
    long start = 0, lo = 0, hi = 0, total = 0;      // start: of row (r, kh)
    long share = 0;
    if (a.rows) {
        r = blockIdx.x / a.n_kv;
        kh = blockIdx.x % a.n_kv;
        hi = 0x7fffffff;
    } else {
        // (sums as doubles: exact up to 2^53, and their quotients' whole parts too)
        const int sh = blockIdx.x;
        if (a.n_req <= kWave) {                     // every wave by itself
            const Kv4Row mine(a, a.seq_lens[min(lane, a.n_req - 1)]);
            const double cost = lane < a.n_req ? (double)mine.cost() * a.n_kv : 0.0, inc = wave_incl_scan(cost);
            total = uniform((long)__shfl(inc, 63));
            share = max((long)((double)total * a.inv_grid) + 1, (long)K4_SHARE);
            lo = sh * share;
            if (lo >= total) return;
            r = __ffsll(__ballot(inc > (double)lo)) - 1;
            start = uniform((long)__shfl(inc - cost, r));
        } else {
            const int per = (a.n_req + BLK - 1) / BLK;       // consecutive requests of a thread
            const int r0 = min(tid * per, a.n_req), r1 = min(r0 + per, a.n_req);
            double mine = 0.0;
            for (int i = r0; i < r1; ++i) mine += (double)Kv4Row(a, a.seq_lens[i]).cost() * a.n_kv;
            const double inc = wave_incl_scan(mine);
            if (lane == 63) sum_s[wave] = inc;
            __syncthreads();
            double before = inc - mine, all = 0.0;
            for (int w = 0; w < WV; ++w) {
                before += w < wave ? sum_s[w] : 0.0;
                all += sum_s[w];
            }
            total = uniform((long)all);
            share = max((long)((double)total * a.inv_grid) + 1, (long)K4_SHARE);
            lo = sh * share;
            if (lo >= total) return;
            if (before <= (double)lo && (double)lo < before + mine) {
                int i = r0;
                for (;; ++i) {
                    const double c = (double)Kv4Row(a, a.seq_lens[i]).cost() * a.n_kv;
                    if (i == r1 - 1 || (double)lo < before + c) break;
                    before += c;
                }
                at_s[0] = i;
                at_s[1] = (long)before;
            }
            __syncthreads();
            r = uniform((int)at_s[0]);
            start = uniform(at_s[1]);
        }
        hi = min(lo + share, total);
        const int c = Kv4Row(a, uniform(a.seq_lens[r])).cost();
        kh = uniform((int)((double)(lo - start) / (double)c));
        start += (long)kh * c;
    }

    for (;;) {
    // Q, asked for together with the row's length (one latency less: 500 keys 6.75 -> 6.61
    // us): k-slots 8 kg .. of step st are entries kg D / 4 + 8 st ..
    v8bf qf[W];
    {
        const uint16_t* qp = a.q + (long)r * a.q_sr + (long)(kh * G + c16) * a.q_sh + kg * (D / 4);
#pragma unroll
        for (int st = 0; st < W; ++st) {
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if (c16 < G) w = *reinterpret_cast<const uint4*>(qp + 8 * st);
            qf[st] = __builtin_bit_cast(v8bf, w);
        }
    }

    const Kv4Row row(a, uniform(a.seq_lens[r]));
    const int len = row.len, klo = row.lo, sinks = row.sinks, na = row.na, b0 = row.b0;
    const int units = max(row.nt, 1);
    // the row's tiles [n0, n1) are this share's
    const long first = start + K4_ROW;
    int n0 = __builtin_amdgcn_readfirstlane((int)min(max(lo - first, 0L), (long)units));
    int n1 = __builtin_amdgcn_readfirstlane((int)min(max(hi - first, 0L), (long)units));
    if (a.rows) { n0 = 0; n1 = units; }
    const bool whole = n0 == 0 && n1 == units;
    const bool work = n0 < n1;
    const long slot = 2L * blockIdx.x + (n0 == 0);
    if (!a.rows && work && n0 == 0 && tid == 0) {
        a.shares[(long)r * a.n_kv + kh] =
            whole ? make_int2(0, -1) : make_int2((int)blockIdx.x, (int)((double)(first + units - 1) / (double)share));
    }
    n1 = min(n1, row.nt);
    if (work) {
    // step `it` of this wave: tiles n0 + T (wave + WV it) .., T of them.  Addresses
    // and first keys of 64 tiles are made at once, one per lane.
    const int mine = n0 + T * wave;
    const int steps = n1 > mine ? (n1 - mine + T * WV - 1) / (T * WV) : 0;
    uint32_t at_lo = 0, at_hi = 0;
    int key_of = 0, it_of = 0;
    uint64_t edges = 0;
    auto fetch = [&](int it) __attribute__((always_inline)) {
        it_of = it;
        const int n = mine + T * (WV * (it + lane / T)) + lane % T, nc = min(n, n1 - 1);
        const int tile = nc < na ? nc : b0 + nc - na;
        const int id = a.bt[(long)r * a.bt_sr + min(tile >> (a.pg_sh - 4), a.bt_cols - 1)];
        const uint64_t at = (uint64_t)a.c + (uint64_t)((long)min(max(id, 0), a.NB - 1) * a.c_sb + (long)kh * a.c_sh +
                                                       (tile & ((1 << (a.pg_sh - 4)) - 1)) * L::TILE);
        at_lo = (uint32_t)at;
        at_hi = (uint32_t)(at >> 32);
        key_of = n < n1 ? tile << 4 : 0x7fffffc0;   // behind the share: keys that no query sees
        edges = __ballot(key_of + 15 >= len || !(key_of >= klo || key_of + 16 <= sinks));
    };
    struct Step { Kv4Lane<D> k[T], v[T]; int key0[T]; bool edge; };
    auto load = [&](int it, Step& x) __attribute__((always_inline)) {
        if (it - it_of >= kWave / T) fetch(it);
        const int l0 = T * (it - it_of);
        x.edge = (edges >> l0 & ((1u << T) - 1)) != 0;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const kv4_ptr p = (kv4_ptr)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(at_lo, l0 + t) |
                                        (uint64_t)(uint32_t)__builtin_amdgcn_readlane(at_hi, l0 + t) << 32);
            x.key0[t] = __builtin_amdgcn_readlane(key_of, l0 + t);
            kv4_load_k<D, true>(p, lane, x.k[t]);
            kv4_load_v<D, true>(p, lane, x.v[t]);
        }
    };

    float m = -INFINITY, l = 0.f;                   // of head c16, over this lane's keys
    v4f o[ND];                                      // o[b][i]: entry (4 kg + i) D / 16 + b
#pragma unroll
    for (int b = 0; b < ND; ++b) o[b] = v4f{0.f, 0.f, 0.f, 0.f};

    auto compute = [&](Step& x) __attribute__((always_inline)) {
        v4f s[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            s[t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < W; ++st) {
                const float sc = kv4_scale(x.k[t].s, D == 256 ? st >> 2 : 0);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, kv4_eight(x.k[t].w[st], sc)),
                                                               qf[st], s[t], 0, 0, 0);
            }
        }
        // keys that the query does not see: no weight, and no value (0 x NaN)
        if (x.edge) {
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = x.key0[t] + 4 * kg + i;
                    const bool seen = key < len && (key >= klo || key < sinks);
                    s[t][i] = seen ? s[t][i] : -INFINITY;
                    x.v[t].s &= seen ? ~0u : ~(255u << (8 * i));
                    if constexpr (D == 64) x.v[t].w[i >> 1] &= seen ? ~0u : (i & 1) ? 0xFFFFu : 0xFFFF0000u;
                    else
#pragma unroll
                        for (int j = 0; j < D / 128; ++j) x.v[t].w[i * (D / 128) + j] &= seen ? ~0u : 0u;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[t][i]);
        mx = xor32_max(xor16_max(mx));
        // m follows the maximum once it has grown by 2^8 in weight: until then weights
        // are at most 256, and o and l need no rescaling
        if (__any((mx - m) * a.scale_log2 > 8.f)) {
            const float m_new = fmaxf(m, mx);
            const float al = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * a.scale_log2);
            m = m_new;
            l *= al;
#pragma unroll
            for (int b = 0; b < ND; ++b) o[b] *= al;
        }
        const float mc = m == -INFINITY ? 0.f : m * a.scale_log2;
        // Weights in bf16, the product's other operand (half a step, 2^-8 of each);
        // l keeps the unrounded ones
        v8bf pf[T / 2];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[t][i], a.scale_log2, -mc));
                l += p;
                pf[t >> 1][4 * (t & 1) + i] = (__bf16)p;
            }
#pragma unroll
        for (int u = 0; u < T / 2; ++u) {
            const Kv4Lane<D>* v = x.v + 2 * u;
            float vs[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) vs[t][i] = kv4_scale(v[t].s, i);
            // two column blocks at once: the entries 2 j and 2 j + 1 of every lane's share
            auto pair = [&](auto byte, int b, int word) __attribute__((always_inline)) {
                constexpr int B = decltype(byte)::value;
                uint32_t y[2][4];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (D == 64)
                            y[t][i] = (i & 1) ? kv4_pair<(B + 2) & 3>(v[t].w[i >> 1], vs[t][i]) : kv4_pair<B>(v[t].w[i >> 1], vs[t][i]);
                        else
                            y[t][i] = kv4_pair<B>(v[t].w[(D / 128) * i + word], vs[t][i]);
                    }
                const uint4 even = make_uint4(lows(y[0][0], y[0][1]), lows(y[0][2], y[0][3]), lows(y[1][0], y[1][1]), lows(y[1][2], y[1][3]));
                const uint4 odd = make_uint4(highs(y[0][0], y[0][1]), highs(y[0][2], y[0][3]), highs(y[1][0], y[1][1]), highs(y[1][2], y[1][3]));
                o[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, even), pf[u], o[b], 0, 0, 0);
                o[b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, odd), pf[u], o[b + 1], 0, 0, 0);
            };
            using B0 = std::integral_constant<int, 0>; using B1 = std::integral_constant<int, 1>;
            using B2 = std::integral_constant<int, 2>; using B3 = std::integral_constant<int, 3>;
            if constexpr (D == 64) {
                pair(B0{}, 0, 0); pair(B1{}, 2, 0);
            } else {
#pragma unroll
                for (int w = 0; w < D / 128; ++w) {
                    pair(B0{}, 8 * w, w); pair(B1{}, 8 * w + 2, w);
                    pair(B2{}, 8 * w + 4, w); pair(B3{}, 8 * w + 6, w);
                }
            }
        }
    };

    if (steps > 0) {
        Step x0, x1;                                // the one in use and the one on its way
        fetch(0);
        load(0, x0);
        for (int it = 0; it < steps; it += 2) {
            if (it + 1 < steps) load(it + 1, x1);
            compute(x0);
            if (it + 1 < steps) {
                if (it + 2 < steps) load(it + 2, x0);
                compute(x1);
            }
        }
    }

    // the waves' shares of each head: (m, l, o) scaled to the largest m
    l = xor32_sum(xor16_sum(l));
    const bool any = l > 0.f || l != l;
    if (kg == 0) { m_s[wave][c16] = any ? m * a.scale_log2 : -INFINITY; l_s[wave][c16] = l; }
    if (c16 < G) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int b = 0; b < ND; b += 4)
                *reinterpret_cast<float4*>(&o_s[wave][c16][(4 * kg + i) * (D / 16) + b]) =
                    make_float4(o[b][i], o[b + 1][i], o[b + 2][i], o[b + 3][i]);
    }
    __syncthreads();
    for (int u = tid; u < G * (D / 4); u += BLK) {
        const int g = u / (D / 4), e = 4 * (u % (D / 4));
        float mm = -INFINITY, lt = 0.f;
#pragma unroll
        for (int w = 0; w < WV; ++w) mm = fmaxf(mm, m_s[w][g]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WV; ++w) {
            const float lw = l_s[w][g];
            if (lw == 0.f) continue;                // a wave without keys
            const float f = mm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_s[w][g] - mm);
            const float4 y = *reinterpret_cast<const float4*>(&o_s[w][g][e]);
            lt += lw * f;
            acc.x += f * y.x; acc.y += f * y.y; acc.z += f * y.z; acc.w += f * y.w;
        }
        if (!whole) {
            *reinterpret_cast<float4*>(a.acc + (slot * G + g) * D + e) = acc;
            if (e == 0) { a.m[slot * G + g] = mm; a.l[slot * G + g] = lt; }
        } else {
            const float inv = lt == 0.f ? 0.f : 1.f / lt;
            uint2 w;
            w.x = (uint32_t)f32_to_bf16(acc.x * inv) | (uint32_t)f32_to_bf16(acc.y * inv) << 16;
            w.y = (uint32_t)f32_to_bf16(acc.z * inv) | (uint32_t)f32_to_bf16(acc.w * inv) << 16;
            *reinterpret_cast<uint2*>(a.out + (long)r * a.o_sr + (long)(kh * G + g) * a.o_sh + e) = w;
            if (a.lse && e == 0) a.lse[(long)r * a.lse_sr + kh * G + g] = lt == 0.f ? -INFINITY : mm * kLn2 + logf(lt);
        }
    }
    __syncthreads();
    }
    // the next row
    start += row.cost();
    if (a.rows || start >= hi) break;
    if (++kh == a.n_kv) { kh = 0; ++r; }
    }
}

// Joins the partials of every row that has several: `hpw` heads of a row a workgroup (all
// that fit where there are many rows, one where there are few), D / 4 columns each, and
// what threads are left as streams over the partials.  A decode's row has those of its
// shares, the first one's in its second slot (it starts the row), the others' in their
// first; a prompt's row (SHARES false) one of each split.
template <int D, bool ONE, bool SHARES>
__global__ __launch_bounds__(K4_BLK) void kv4_merge_kernel(const Kv4MergeArgs a, int heads)
{
    const int hpw = ONE ? 1 : heads;
    constexpr int COLS = D / 4, PF = 8;
    __shared__ float4 acc_s[K4_BLK];
    __shared__ float2 ml_s[K4_BLK];
    const int tid = threadIdx.x, col = tid % COLS, n_heads = (a.G + hpw - 1) / hpw;
    const int hh = tid / COLS % hpw, strm = tid / (COLS * hpw), streams = K4_BLK / (COLS * hpw);
    const long row = blockIdx.x / n_heads;          // request, kv head
    const int g = blockIdx.x % n_heads * hpw + hh;
    int2 sh = make_int2(0, 0);
    int n = a.splits;
    if constexpr (SHARES) {
        sh = a.shares[row];
        n = sh.y - sh.x + 1;
        if (n <= 0) return;
    } else {
        // rows before the first request or after the last one have no partials
        const long t = row / a.n_kv;
        if (t < a.starts[0] || t >= a.starts[a.n_seq]) return;
    }
    const bool mine = strm < streams && g < a.G;
    // the running maximum, sum and columns over this stream's shares
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = strm; mine && i0 < n; i0 += PF * streams) {
        float4 x[PF];
        float mi[PF], li[PF];
#pragma unroll
        for (int k = 0; k < PF; ++k) {
            const int i = min(i0 + k * streams, n - 1);
            const long at = (SHARES ? 2L * (sh.x + i) + (i == 0) : row * n + i) * a.G + g;
            mi[k] = a.m[at];
            li[k] = i0 + k * streams < n ? a.l[at] : 0.f;
            x[k] = *reinterpret_cast<const float4*>(a.acc + at * D + 4 * col);
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < PF; ++k) top = fmaxf(top, li[k] == 0.f ? -INFINITY : mi[k]);
        // (a maximum of -inf: every weight so far is 0 or NaN, and stays what it is)
        const float old = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top);
        l *= old;
        acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
#pragma unroll
        for (int k = 0; k < PF; ++k)
            if (li[k] != 0.f) {                     // a share without keys has no columns
                const float w = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mi[k] - top);
                l += li[k] * w;
                acc.x += w * x[k].x; acc.y += w * x[k].y; acc.z += w * x[k].z; acc.w += w * x[k].w;
            }
        m = top;
    }
    if (streams > 1) {
        acc_s[tid] = acc;
        if (col == 0) ml_s[tid / COLS] = make_float2(m, l);
        __syncthreads();
        if (strm > 0 || !mine) return;
        float top = m;
#pragma unroll
        for (int k = 1; k < streams; ++k) top = fmaxf(top, ml_s[k * hpw + hh].x);
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
        l = 0.f;
#pragma unroll
        for (int k = 0; k < streams; ++k) {
            const float2 ml = ml_s[k * hpw + hh];
            const float4 x = acc_s[tid + k * COLS * hpw];
            if (ml.y == 0.f) continue;
            const float w = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - top);
            l += ml.y * w;
            acc.x += w * x.x; acc.y += w * x.y; acc.z += w * x.z; acc.w += w * x.w;
        }
        m = top;
    }
    if (!mine) return;
    const long r = row / a.n_kv;
    const int hd = (int)(row % a.n_kv) * a.G + g;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint2 w;
    w.x = (uint32_t)f32_to_bf16(acc.x * inv) | (uint32_t)f32_to_bf16(acc.y * inv) << 16;
    w.y = (uint32_t)f32_to_bf16(acc.z * inv) | (uint32_t)f32_to_bf16(acc.w * inv) << 16;
    *reinterpret_cast<uint2*>(a.out + r * a.o_sr + (long)hd * a.o_sh + 4 * col) = w;
    if (a.lse && col == 0) a.lse[r * a.lse_sr + hd] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
}

// ---- rows read back -------------------------------------------------------------
// A lane takes eight entries of a row: 4 bytes of codes and a scale, K and V, in; 16
// bytes each out.  Bound by the writes: 8272 rows of 8 heads 9.7 us, 4.4 TB/s.
struct Kv4ReadArgs {
    const uint8_t* c; long c_sb, c_sh;
    const int64_t* slots;
    uint16_t* k; long k_st, k_sh;
    uint16_t* v; long v_st, v_sh;
    long n_slots, units;                            // units: (token, kv head, word of eight entries)
    int n_kv, pg_sh;
};

// RD_UNITS units of a thread: their loads are in flight together.
template <int D, int RD_UNITS>
__global__ __launch_bounds__(256) void kv4_read_kernel(const Kv4ReadArgs a)
{
    using L = Kv4<D>;
    constexpr int LPH = D / 8;
    const long u0 = (long)blockIdx.x * (256 * RD_UNITS) + threadIdx.x;
    long slot[RD_UNITS], t[RD_UNITS];
    int kh[RD_UNITS];
    const int l = threadIdx.x % LPH;
#pragma unroll
    for (int k = 0; k < RD_UNITS; ++k) {
        const long u = u0 + 256 * k, row = (u < a.units ? u : 0) / LPH;
        t[k] = row / a.n_kv;
        kh[k] = (int)(row - t[k] * a.n_kv);
        slot[k] = u < a.units ? a.slots[t[k]] : -1;
    }
    uint32_t kw[RD_UNITS], vw[RD_UNITS], ks[RD_UNITS], vs[RD_UNITS];
#pragma unroll
    for (int k = 0; k < RD_UNITS; ++k) {
        const bool here = slot[k] >= 0 && slot[k] < a.n_slots;
        const long s = here ? slot[k] : 0;
        slot[k] = here ? s : -1;
        const int off = (int)(s & ((1 << a.pg_sh) - 1)), key = off & 15;
        const uint8_t* p = a.c + (s >> a.pg_sh) * a.c_sb + (long)kh[k] * a.c_sh + (off >> 4) * L::TILE;
        kw[k] = *reinterpret_cast<const uint32_t*>(p + L::k_code(key, l));
        if constexpr (D == 64)
            vw[k] = *reinterpret_cast<const uint16_t*>(p + L::v_code(key, l)) |
                    (uint32_t)*reinterpret_cast<const uint16_t*>(p + L::v_code(key, l) + 8) << 16;
        else
            vw[k] = *reinterpret_cast<const uint32_t*>(p + L::v_code(key, l));
        ks[k] = p[L::k_scale(key, l >> 2)];
        vs[k] = p[L::v_scale(key, l >> 2)];
    }
#pragma unroll
    for (int k = 0; k < RD_UNITS; ++k)
        if (slot[k] >= 0) {
            *reinterpret_cast<uint4*>(a.k + t[k] * a.k_st + (long)kh[k] * a.k_sh + 8 * l) = kv4_eight(kw[k], kv4_scale(ks[k], 0));
            *reinterpret_cast<uint4*>(a.v + t[k] * a.v_st + (long)kh[k] * a.v_sh + 8 * l) = kv4_eight(vw[k], kv4_scale(vs[k], 0));
        }
}

int launch_kv4_merge(const Kv4MergeArgs& a, int n_rows, int head_dim, hipStream_t st)
{
    // heads of a workgroup: with 256 rows or more they fill the card together
    const int64_t rows = (int64_t)n_rows * a.n_kv;
    int hpw = 1;
    while (rows >= 256 && hpw < a.G && 2 * hpw * (head_dim / 4) <= K4_BLK) hpw *= 2;
    const dim3 grid((unsigned)(rows * ((a.G + hpw - 1) / hpw)));
#define KV4_MERGE(D, SHARES)                                                                                          \
    do {                                                                                                              \
        if (hpw == 1) hipLaunchKernelGGL((kv4_merge_kernel<D, true, SHARES>), grid, dim3(K4_BLK), 0, st, a, 1);       \
        else hipLaunchKernelGGL((kv4_merge_kernel<D, false, SHARES>), grid, dim3(K4_BLK), 0, st, a, hpw);             \
    } while (0)
#define KV4_MERGE_D(D)                          \
    do {                                        \
        if (a.shares) KV4_MERGE(D, true);       \
        else KV4_MERGE(D, false);               \
    } while (0)
    if (head_dim == 64) KV4_MERGE_D(64);
    else if (head_dim == 128) KV4_MERGE_D(128);
    else KV4_MERGE_D(256);
#undef KV4_MERGE_D
#undef KV4_MERGE
    return check_launch("kv4_merge_kernel");
}

// Workgroups of a call: one for each row where rows are short, or else as many shares as
// the card holds at once.
// (a row of its own for each workgroup: 49 requests of up to 936 tokens 11.8 -> 9.4 us, 32 of 2000
// 22.0 -> 18.7, but one of 2000 10.8 -> 16.7)
static bool kv4_rows(int n_req, int n_kv, long max_keys) {
    return max_keys <= 1024 || (max_keys <= 2048 && (long)n_req * n_kv >= 256);
}
int64_t kv4_workspace(int n_req, int n_kv, int G, int head_dim) {
    return (int64_t)kv4_grid(head_dim, G) * 2 * G * (head_dim + 2) * 4 + (int64_t)n_req * n_kv * 8;
}

int32_t check_kv4(const char* what, const void* cache, int64_t sb, int64_t sh, int32_t num_blocks, int32_t n_kv,
                         int32_t head_dim, int32_t page)
{
    LOCKS_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "%s: head_dim %d outside {64, 128, 256}", what, head_dim);
    LOCKS_REQUIRE(page == 16 || page == 32 || page == 64, "%s: page %d outside {16, 32, 64}", what, page);
    LOCKS_REQUIRE(n_kv >= 1 && n_kv <= 4096 && num_blocks >= 1, "%s: n_kv %d outside [1, 4096] or no blocks", what, n_kv);
    LOCKS_REQUIRE(cache, "%s: null pointer argument", what);
    LOCKS_REQUIRE((uintptr_t)cache % 16 == 0 && sb % 16 == 0 && sh % 16 == 0 && sb >= 0 && sh >= 0,
                  "%s: the cache and its block and head strides must be multiples of 16 bytes", what);
    return 0;
}

}  // namespace locks

using namespace locks;

extern "C" int32_t locks_kv4_decode(
    const uint16_t* q, int64_t q_stride_req, int64_t q_stride_head, const uint8_t* cache, int64_t c_stride_block,
    int64_t c_stride_head, int32_t num_blocks, const int32_t* block_table, int64_t bt_stride, int32_t bt_cols,
    const int32_t* seq_lens, int32_t window, int32_t sinks, uint16_t* out, int64_t out_stride_req,
    int64_t out_stride_head, float* lse, int64_t lse_stride_req, void* workspace, int64_t workspace_bytes,
    int32_t n_req, int32_t n_kv, int32_t G, int32_t head_dim, int32_t page, int32_t max_seq_len, float scale, void* stream)
{
    const char* what = "locks_kv4_decode";
    int rc = check_kv4(what, cache, c_stride_block, c_stride_head, num_blocks, n_kv, head_dim, page);
    if (rc) return rc;
    // q, out, the table and the lengths: what the bf16 cache's entries ask
    const int64_t none[3] = {0, 0, 0};
    rc = check_attn(what, q, q_stride_req, q_stride_head, (const uint16_t*)cache, none, (const uint16_t*)cache, none,
                    num_blocks, block_table, bt_stride, bt_cols, seq_lens, window, sinks, out, out_stride_req,
                    out_stride_head, n_req, n_kv, G, head_dim, page, max_seq_len, scale);
    if (rc) return rc;
    if (n_req == 0) return 0;
    long keys = bound_keys(max_seq_len, bt_cols, page);
    if (window && (long)window + sinks + 32 < keys) keys = (long)window + sinks + 32;
    const int shares = kv4_grid(head_dim, G);
    Kv4DecodeArgs a{q, q_stride_req, q_stride_head, cache, c_stride_block, c_stride_head, block_table, bt_stride, seq_lens,
                    out, out_stride_req, out_stride_head, lse, lse_stride_req, nullptr, nullptr, nullptr, nullptr,
                    scale * kLog2e, 1.0 / shares, num_blocks, bt_cols, n_req, n_kv, G,
                    page == 16 ? 4 : page == 32 ? 5 : 6, window, sinks, kv4_rows(n_req, n_kv, keys)};
    int wgs = n_req * n_kv;
    if (!a.rows) {
        rc = check_ws(what, workspace, workspace_bytes, kv4_workspace(n_req, n_kv, G, head_dim));
        if (rc) return rc;
        wgs = shares;
        const int64_t slots = 2L * wgs * G;
        a.acc = static_cast<float*>(workspace);
        a.m = a.acc + slots * head_dim;
        a.l = a.m + slots;
        a.shares = reinterpret_cast<int2*>(a.l + slots);
    }
    hipStream_t st = (hipStream_t)stream;
    const bool wide = a.rows && wgs <= 256;
#define KV4_DECODE(D)                                                                                                    \
    do {                                                                                                                 \
        if (wide) hipLaunchKernelGGL((kv4_decode_kernel<D, 8>), dim3((unsigned)wgs), dim3(8 * kWave), 0, st, a);         \
        else hipLaunchKernelGGL((kv4_decode_kernel<D, K4_WAVES>), dim3((unsigned)wgs), dim3(K4_BLK), 0, st, a);          \
    } while (0)
    if (head_dim == 64) KV4_DECODE(64);
    else if (head_dim == 128) KV4_DECODE(128);
    else KV4_DECODE(256);
#undef KV4_DECODE
    rc = check_launch("kv4_decode_kernel");
    if (rc || a.rows) return rc;
    return launch_kv4_merge(Kv4MergeArgs{a.m, a.l, a.acc, a.shares, 0, nullptr, 0, out, out_stride_req, out_stride_head, lse,
                                         lse_stride_req, n_kv, G}, n_req, head_dim, st);
}

extern "C" int32_t locks_kv4_read(
    const uint8_t* cache, int64_t c_stride_block, int64_t c_stride_head, int32_t num_blocks, const int64_t* slots,
    uint16_t* k_out, int64_t k_stride_tok, int64_t k_stride_head, uint16_t* v_out, int64_t v_stride_tok,
    int64_t v_stride_head, int32_t n_tokens, int32_t n_kv, int32_t head_dim, int32_t page, void* stream)
{
    const char* what = "locks_kv4_read";
    const int rc = check_kv4(what, cache, c_stride_block, c_stride_head, num_blocks, n_kv, head_dim, page);
    if (rc) return rc;
    LOCKS_REQUIRE(n_tokens >= 0, "%s: n_tokens %d < 0", what, n_tokens);
    LOCKS_REQUIRE(slots && k_out && v_out, "%s: null pointer argument", what);
    for (int64_t x : {k_stride_tok, k_stride_head, v_stride_tok, v_stride_head})
        LOCKS_REQUIRE(x % 8 == 0, "%s: strides must be multiples of 8 elements (16-byte stores)", what);
    LOCKS_REQUIRE((uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0 && (uintptr_t)slots % 8 == 0,
                  "%s: the outputs must be 16-byte aligned, the slots 8-byte", what);
    if (n_tokens == 0) return 0;
    const long units = (long)n_tokens * n_kv * (head_dim / 8);
    // four units a thread where that leaves two workgroups a CU and more (8272 tokens of 8
    // heads 11.5 -> 9.7 us), or else one (112 tokens 2.7 us, with four 3.5)
    const int per = units >= 256 * 4 * 512 ? 4 : 1;
    const long wgs = (units + 256 * per - 1) / (256 * per);
    LOCKS_REQUIRE(wgs <= 0x7fffffffL, "%s: too many tokens and heads for one launch", what);
    const Kv4ReadArgs a{cache, c_stride_block, c_stride_head, slots, k_out, k_stride_tok, k_stride_head, v_out,
                        v_stride_tok, v_stride_head, (long)num_blocks * page, units, n_kv,
                        page == 16 ? 4 : page == 32 ? 5 : 6};
    const dim3 grid((unsigned)wgs);
    hipStream_t st = (hipStream_t)stream;
#define KV4_READ(D)                                                                             \
    do {                                                                                        \
        if (per == 4) hipLaunchKernelGGL((kv4_read_kernel<D, 4>), grid, dim3(256), 0, st, a);   \
        else hipLaunchKernelGGL((kv4_read_kernel<D, 1>), grid, dim3(256), 0, st, a);            \
    } while (0)
    if (head_dim == 64) KV4_READ(64);
    else if (head_dim == 128) KV4_READ(128);
    else KV4_READ(256);
#undef KV4_READ
    return check_launch("kv4_read_kernel");
}
