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
// LDS, the workgroups of a row in attn_merge_kernel.
#include "locks_attn.h"
#include "locks_common.h"
#include "locks_hip.h"
#include "locks_kv4.h"

#include <math.h>

namespace locks {

constexpr int K4_WAVES = 4;
constexpr int K4_BLK = K4_WAVES * kWave;
constexpr float kLog2e = 1.44269504088896340736f;

struct Kv4DecodeArgs {
    const uint16_t* q; long q_sr, q_sh;
    const uint8_t* c; long c_sb, c_sh;              // bytes
    const int* bt; long bt_sr;
    const int* seq_lens;
    uint16_t* out; long o_sr, o_sh;
    float* lse; long lse_sr;
    Partials p;                                     // splits 1: none, the output is written
    float scale_log2, scale;
    int NB, bt_cols, n_kv, G, pg_sh, window, sinks, chunk;      // chunk: tiles of a workgroup
};

// Bits 2 lo .. of two words as one: {low or high halves of a, of b}.
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

template <int D>
__global__ __launch_bounds__(K4_BLK, D == 256 ? 2 : 3) void kv4_decode_kernel(const Kv4DecodeArgs a)
{
    using L = Kv4<D>;
    constexpr int ND = D / 16, W = L::W;
    __shared__ float m_s[K4_WAVES][16], l_s[K4_WAVES][16];
    __shared__ __attribute__((aligned(16))) float o_s[K4_WAVES][16][D + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15, kg = lane >> 4;
    const int nsplit = a.p.splits, G = a.G;
    const int sp = blockIdx.x % nsplit, kh = blockIdx.x / nsplit % a.n_kv;
    const long r = blockIdx.x / nsplit / a.n_kv;

    const long cap = (long)a.bt_cols << a.pg_sh;
    const int len = (int)min((long)max(a.seq_lens[r], 0), cap);
    // a length past the table: the window still ends at it
    const long full = max(a.seq_lens[r], 0);
    const int lo = a.window ? (int)min(max(full - a.window, 0L), (long)len) : 0;
    const int sinks = min(a.sinks, lo);
    // tiles: the first na, then [b0, b1); this workgroup's [n0, n1) of them
    const int na = (sinks + 15) >> 4, b0 = max(lo >> 4, na), b1 = (len + 15) >> 4;
    const int nt = na + max(b1 - b0, 0);
    const int n0 = min(sp * a.chunk, nt), n1 = sp == nsplit - 1 ? nt : min(n0 + a.chunk, nt);
    const long row = (r * a.n_kv + kh) * nsplit + sp;
    if (n0 >= n1 && nsplit > 1) {
        if (tid < G) { a.p.m[row * G + tid] = -INFINITY; a.p.l[row * G + tid] = 0.f; }
        return;
    }

    // Q: k-slots 8 kg .. of step st are entries kg D / 4 + 8 st ..
    v8bf qf[W];
    {
        const uint16_t* qp = a.q + r * a.q_sr + (long)(kh * G + c16) * a.q_sh + kg * (D / 4);
#pragma unroll
        for (int st = 0; st < W; ++st) {
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if (c16 < G) w = *reinterpret_cast<const uint4*>(qp + 8 * st);
            qf[st] = __builtin_bit_cast(v8bf, w);
        }
    }

    auto tile_of = [&](int n) __attribute__((always_inline)) { return n < na ? n : b0 + n - na; };
    // step `it` of this wave: tiles n0 + 2 (wave + K4_WAVES it) and the next one; the
    // block ids of 32 steps are loaded at once
    const int mine = n0 + 2 * wave;
    const int steps = n1 > mine ? (n1 - mine + 2 * K4_WAVES - 1) / (2 * K4_WAVES) : 0;
    const int per = 1 << (a.pg_sh - 4);             // tiles of a page
    int ids = 0, ids0 = 0;
    auto fetch_ids = [&](int it) __attribute__((always_inline)) {
        ids0 = it;
        const int n = min(mine + 2 * K4_WAVES * (it + (lane >> 1)) + (lane & 1), n1 - 1);
        const int pg = min(tile_of(n) >> (a.pg_sh - 4), a.bt_cols - 1);
        ids = min(max(a.bt[r * a.bt_sr + pg], 0), a.NB - 1);
    };
    struct Step { Kv4Lane<D> k[2], v[2]; };
    auto load = [&](int it, Step& x) __attribute__((always_inline)) {
        if (it - ids0 >= 32) fetch_ids(it);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int n = min(mine + 2 * K4_WAVES * it + t, n1 - 1);
            const long blk = __builtin_amdgcn_readlane(ids, 2 * (it - ids0) + t);
            const uint8_t* p = a.c + blk * a.c_sb + (long)kh * a.c_sh + (tile_of(n) & (per - 1)) * L::TILE;
            kv4_load_k<D>(p, lane, x.k[t]);
            kv4_load_v<D>(p, lane, x.v[t]);
        }
    };

    float m = -INFINITY, l = 0.f;                   // of head c16, over this lane's keys
    v4f o[ND];                                      // o[b][i]: entry (4 kg + i) D / 16 + b
#pragma unroll
    for (int b = 0; b < ND; ++b) o[b] = v4f{0.f, 0.f, 0.f, 0.f};

    auto compute = [&](int it, Step& x) __attribute__((always_inline)) {
        v4f s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < W; ++st) {
                const float sc = kv4_scale(x.k[t].s, D == 256 ? st >> 2 : 0);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, kv4_eight(x.k[t].w[st], sc)),
                                                               qf[st], s[t], 0, 0, 0);
            }
        }
        // keys that the query does not see: no weight, and no value (0 x NaN)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int n = mine + 2 * K4_WAVES * it + t, key0 = tile_of(n) << 4;
            const bool whole = n < n1 && key0 + 16 <= len && (key0 >= lo || key0 + 16 <= sinks);
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 4 * kg + i;
                    const bool seen = n < n1 && key < len && (key >= lo || key < sinks);
                    s[t][i] = seen ? s[t][i] : -INFINITY;
                    if (!seen) {
                        x.v[t].s &= ~(255u << (8 * i));
                        if constexpr (D == 64) x.v[t].w[i >> 1] &= (i & 1) ? 0xFFFFu : 0xFFFF0000u;
                        else if constexpr (D == 128) x.v[t].w[i] = 0;
                        else { x.v[t].w[2 * i] = 0; x.v[t].w[2 * i + 1] = 0; }
                    }
                }
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[t][i]);
        mx = xor32_max(xor16_max(mx));
        // m follows the maximum once it has grown by 2^8 in weight: until then weights
        // are at most 256, and o and l need no rescaling
        if (__any((mx - m) * a.scale_log2 > 8.f)) {
            const float m_new = fmaxf(m, mx);
            const float alpha = __builtin_amdgcn_exp2f((m - m_new) * a.scale_log2);
            const float al = m_new == -INFINITY ? 1.f : alpha;
            m = m_new;
            l *= al;
#pragma unroll
            for (int b = 0; b < ND; ++b) o[b] *= al;
        }
        const float mc = m == -INFINITY ? 0.f : m * a.scale_log2;
        // Weights in bf16, the product's other operand (half a step, 2^-8 of each);
        // l keeps the unrounded ones
        v8bf pf;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[t][i], a.scale_log2, -mc));
                l += p;
                pf[4 * t + i] = (__bf16)p;
            }
        float vs[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) vs[t][i] = kv4_scale(x.v[t].s, i);
        // two column blocks at once: the entries 2 j and 2 j + 1 of every lane's share
        auto pair = [&](auto byte, int b, int word, int step) __attribute__((always_inline)) {
            constexpr int B = decltype(byte)::value;
            uint32_t y[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (D == 64) {
                        y[t][i] = (i & 1) ? kv4_pair<B + 2>(x.v[t].w[i >> 1], vs[t][i]) : kv4_pair<B>(x.v[t].w[i >> 1], vs[t][i]);
                    } else {
                        y[t][i] = kv4_pair<B>(x.v[t].w[step * i + word], vs[t][i]);
                    }
                }
            const uint4 even = make_uint4(lows(y[0][0], y[0][1]), lows(y[0][2], y[0][3]), lows(y[1][0], y[1][1]), lows(y[1][2], y[1][3]));
            const uint4 odd = make_uint4(highs(y[0][0], y[0][1]), highs(y[0][2], y[0][3]), highs(y[1][0], y[1][1]), highs(y[1][2], y[1][3]));
            o[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, even), pf, o[b], 0, 0, 0);
            o[b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, odd), pf, o[b + 1], 0, 0, 0);
        };
        using B0 = std::integral_constant<int, 0>; using B1 = std::integral_constant<int, 1>;
        using B2 = std::integral_constant<int, 2>; using B3 = std::integral_constant<int, 3>;
        if constexpr (D == 64) {
            pair(B0{}, 0, 0, 0); pair(B1{}, 2, 0, 0);
        } else {
#pragma unroll
            for (int w = 0; w < D / 128; ++w) {
                pair(B0{}, 8 * w, w, D / 128); pair(B1{}, 8 * w + 2, w, D / 128);
                pair(B2{}, 8 * w + 4, w, D / 128); pair(B3{}, 8 * w + 6, w, D / 128);
            }
        }
    };

    if (steps > 0) {
        Step x0, x1;
        fetch_ids(0);
        load(0, x0);
        for (int it = 0; it < steps; it += 2) {
            if (it + 1 < steps) load(it + 1, x1);
            compute(it, x0);
            if (it + 1 < steps) {
                if (it + 2 < steps) load(it + 2, x0);
                compute(it + 1, x1);
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
    for (int u = tid; u < G * (D / 4); u += K4_BLK) {
        const int g = u / (D / 4), e = 4 * (u % (D / 4));
        float mm = -INFINITY, lt = 0.f;
#pragma unroll
        for (int w = 0; w < K4_WAVES; ++w) mm = fmaxf(mm, m_s[w][g]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < K4_WAVES; ++w) {
            const float lw = l_s[w][g];
            if (lw == 0.f) continue;                // a wave without keys
            const float f = mm == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_s[w][g] - mm);
            const float4 y = *reinterpret_cast<const float4*>(&o_s[w][g][e]);
            lt += lw * f;
            acc.x += f * y.x; acc.y += f * y.y; acc.z += f * y.z; acc.w += f * y.w;
        }
        constexpr float kLn2 = 0.69314718055994530942f;
        if (nsplit > 1) {
            *reinterpret_cast<float4*>(a.p.acc + (row * G + g) * D + e) = acc;
            if (e == 0) { a.p.m[row * G + g] = mm * kLn2; a.p.l[row * G + g] = lt; }
        } else {
            const float inv = lt == 0.f ? 0.f : 1.f / lt;
            uint2 w;
            w.x = (uint32_t)f32_to_bf16(acc.x * inv) | (uint32_t)f32_to_bf16(acc.y * inv) << 16;
            w.y = (uint32_t)f32_to_bf16(acc.z * inv) | (uint32_t)f32_to_bf16(acc.w * inv) << 16;
            *reinterpret_cast<uint2*>(a.out + r * a.o_sr + (long)(kh * G + g) * a.o_sh + e) = w;
            if (a.lse && e == 0) a.lse[r * a.lse_sr + kh * G + g] = lt == 0.f ? -INFINITY : mm * kLn2 + logf(lt);
        }
    }
}

// ---- rows read back -------------------------------------------------------------
struct Kv4ReadArgs {
    const uint8_t* c; long c_sb, c_sh;
    const int64_t* slots;
    uint16_t* k; long k_st, k_sh;
    uint16_t* v; long v_st, v_sh;
    long n_slots, units;                            // units: (token, kv head, word of eight entries)
    int n_kv, pg_sh;
};

template <int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(const Kv4ReadArgs a)
{
    using L = Kv4<D>;
    constexpr int LPH = D / 8;
    const long u = (long)blockIdx.x * 256 + threadIdx.x;
    if (u >= a.units) return;
    const int l = (int)(u % LPH), kh = (int)(u / LPH % a.n_kv);
    const long t = u / LPH / a.n_kv;
    const long slot = a.slots[t];
    if (slot < 0 || slot >= a.n_slots) return;
    const long blk = slot >> a.pg_sh;
    const int off = (int)(slot & ((1 << a.pg_sh) - 1)), key = off & 15;
    const uint8_t* p = a.c + blk * a.c_sb + (long)kh * a.c_sh + (off >> 4) * L::TILE;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(p + L::k_code(key, l));
    uint32_t vw;
    if constexpr (D == 64)
        vw = *reinterpret_cast<const uint16_t*>(p + L::v_code(key, l)) |
             (uint32_t)*reinterpret_cast<const uint16_t*>(p + L::v_code(key, l) + 8) << 16;
    else
        vw = *reinterpret_cast<const uint32_t*>(p + L::v_code(key, l));
    const float ks = kv4_scale(p[L::k_scale(key, l >> 2)], 0), vs = kv4_scale(p[L::v_scale(key, l >> 2)], 0);
    *reinterpret_cast<uint4*>(a.k + t * a.k_st + (long)kh * a.k_sh + 8 * l) = kv4_eight(kw, ks);
    *reinterpret_cast<uint4*>(a.v + t * a.v_st + (long)kh * a.v_sh + 8 * l) = kv4_eight(vw, vs);
}

// Workgroups of a row: about 1024 in all, and each of at most 2048 keys up to 4096
// workgroups; at least 256 keys each (two steps a wave).
int kv4_decode_splits(int n_req, int n_kv, long max_keys) {
    const long rows = (long)n_req * n_kv;
    const long fill = (1024 + rows - 1) / rows, cap = (4096 + rows - 1) / rows;
    const long even = (max_keys + 2047) / 2048 < cap ? (max_keys + 2047) / 2048 : cap, least = (max_keys + 255) / 256;
    long n = fill > even ? fill : even;
    n = n < least ? n : least;
    return (int)(n < 1 ? 1 : n > AT_MAX_SPLITS ? AT_MAX_SPLITS : n);
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
    long keys = (long)bt_cols * page;
    if (max_seq_len > 0 && max_seq_len < keys) keys = max_seq_len;
    if (window && (long)window + sinks + 32 < keys) keys = (long)window + sinks + 32;
    const int ns = kv4_decode_splits(n_req, n_kv, keys);
    const int64_t rows = (int64_t)n_req * n_kv * G;
    Partials p{nullptr, nullptr, nullptr, 1};
    if (ns > 1) {
        rc = check_ws(what, workspace, workspace_bytes, part_bytes(rows, ns, head_dim));
        if (rc) return rc;
        p = part_layout(workspace, rows, ns, head_dim);
    }
    // tiles of a workgroup: a whole number of steps of its waves.  A window's and the
    // sinks' tiles stand at any offset, a tile more than their keys fill each.
    const long wg = 2 * K4_WAVES, tiles = (keys + 15) / 16 + (window ? 2 : 0);
    const long chunk = ((tiles + ns - 1) / ns + wg - 1) / wg * wg;
    const Kv4DecodeArgs a{q, q_stride_req, q_stride_head, cache, c_stride_block, c_stride_head, block_table, bt_stride,
                          seq_lens, out, out_stride_req, out_stride_head, lse, lse_stride_req, p, scale * kLog2e, scale,
                          num_blocks, bt_cols, n_kv, G, page == 16 ? 4 : page == 32 ? 5 : 6, window, sinks, (int)chunk};
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)((int64_t)n_req * n_kv * ns));
    if (head_dim == 64) hipLaunchKernelGGL(kv4_decode_kernel<64>, grid, dim3(K4_BLK), 0, st, a);
    else if (head_dim == 128) hipLaunchKernelGGL(kv4_decode_kernel<128>, grid, dim3(K4_BLK), 0, st, a);
    else hipLaunchKernelGGL(kv4_decode_kernel<256>, grid, dim3(K4_BLK), 0, st, a);
    rc = check_launch("kv4_decode_kernel");
    if (rc || ns == 1) return rc;
    return launch_merge(p, out, out_stride_req, out_stride_head, lse, lse_stride_req, n_req, n_kv, G, head_dim, nullptr, 0, st);
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
    LOCKS_REQUIRE((units + 255) / 256 <= 0x7fffffffL, "%s: too many tokens and heads for one launch", what);
    const Kv4ReadArgs a{cache, c_stride_block, c_stride_head, slots, k_out, k_stride_tok, k_stride_head, v_out,
                        v_stride_tok, v_stride_head, (long)num_blocks * page, units, n_kv,
                        page == 16 ? 4 : page == 32 ? 5 : 6};
    const dim3 grid((unsigned)((units + 255) / 256));
    hipStream_t st = (hipStream_t)stream;
    if (head_dim == 64) hipLaunchKernelGGL(kv4_read_kernel<64>, grid, dim3(256), 0, st, a);
    else if (head_dim == 128) hipLaunchKernelGGL(kv4_read_kernel<128>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(kv4_read_kernel<256>, grid, dim3(256), 0, st, a);
    return check_launch("kv4_read_kernel");
}
