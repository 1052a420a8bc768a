// Norm and rotation of the query and key heads, and the write of K and V into
// the paged cache, in one pass over the projection's output.
//
// Mathematics, per token t at position p and head x (d entries):
//   y = x * rsqrt(mean(x^2) + eps) * w          (q and k heads with a weight)
//   (a, b) -> (a cos - b sin, b cos + a sin)    for each pair of the first rot
//     entries, the angles of (p, pair) from the caller's fp32 table
//   q: to q_out; k and v: to the cache row of the token's slot.
// Everything in fp32; the one rounding is the store to bf16.
//
// Layout: eight consecutive entries (16 bytes) per lane, d / 8 lanes per head,
// so a wave takes 512 / d heads at once; the mean is a sum over d / 8 lanes (DPP
// row rotations and one permlane swap at most).  The partner of an adjacent pair
// is in the lane, that of a half-split pair rot / 16 lanes away (its raw bf16
// comes over with four permutes and is normed again here).  Bound by memory: every
// row is read and written once.  8192 tokens of 32 + 16 heads of 128: 41 us, 5.0 TB/s,
// a copy's rate; one token 3.8 us.
#include "locks_attn.h"
#include "locks_common.h"
#include "locks_hip.h"
#include "locks_kv4.h"

namespace locks {

constexpr int QK_WAVES = 4;
constexpr int QK_BLK = QK_WAVES * kWave;

struct QkvArgs {
    const uint16_t* q; long q_st, q_sh;
    const uint16_t* k; long k_st, k_sh;
    const uint16_t* v; long v_st, v_sh;
    const int* pos; const int64_t* slot;
    uint16_t* kc; long kc_sb, kc_st, kc_sh;
    uint16_t* vc; long vc_sb, vc_st, vc_sh;
    const float* cs;
    const void* qw; const void* kw;
    uint16_t* qo; long qo_st, qo_sh;
    uint16_t* ko; long ko_st, ko_sh;
    long slots;                             // num_blocks * page
    int max_pos, rot, n_tok, H, n_kv, pg_sh, groups;
    float eps;
    // staged: positions of n_axes axes, pos_ax apart, and each pair's axis in two bits
    int n_axes; long pos_ax;
    uint64_t axes[4];
    int w_f32;
    uint8_t* c4; long c_sb, c_sh;           // KV4: the cache, in place of kc and vc
};
constexpr int QK_AXES = 4;

__device__ __forceinline__ void unpack8(const uint4& w, float* x) {
    x[0] = bf16lo(w.x); x[1] = bf16hi(w.x); x[2] = bf16lo(w.y); x[3] = bf16hi(w.y);
    x[4] = bf16lo(w.z); x[5] = bf16hi(w.z); x[6] = bf16lo(w.w); x[7] = bf16hi(w.w);
}
__device__ __forceinline__ uint4 pack8(const float* x) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    v8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (__bf16)x[e];        // to nearest even, NaN kept
    return __builtin_bit_cast(uint4, y);
}
// Eight consecutive weights, as they stand in memory (bf16 or fp32).
template <bool F32>
struct Weights8 {
    uint4 a, b;
    __device__ __forceinline__ void load(const void* w, int e0) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(w) + (F32 ? 4 : 2) * e0);
        a = p[0];
        if constexpr (F32) b = p[1];
    }
    __device__ __forceinline__ void get(float* x) const {
        if constexpr (F32) {
            const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(u[e]);
        } else {
            unpack8(a, x);
        }
    }
};

// Sum over the D / 8 lanes of a head.
template <int D>
__device__ __forceinline__ float head_sum(float s) {
    if constexpr (D == 64) {                // 8 lanes: xor within the half row by lane swaps of 1, 2, 4
        s += __shfl_xor(s, 1);
        s += __shfl_xor(s, 2);
        s += __shfl_xor(s, 4);
    } else {
        s += row_ror<8>(s); s += row_ror<4>(s); s += row_ror<2>(s); s += row_ror<1>(s);
        if constexpr (D == 256) s = xor16_sum(s);
    }
    return s;
}

template <int D, int IT, bool INTER, bool WF32>
__global__ __launch_bounds__(QK_BLK) void qkv_write_kernel(const QkvArgs a)
{
    constexpr int LPH = D / 8, HPW = kWave / LPH;       // lanes per head, heads per wave
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // waves run over (token, IT groups of heads)
    const int chunks = (a.groups + IT - 1) / IT;
    const long unit = (long)blockIdx.x * QK_WAVES + wave;
    const int t = (int)(unit / chunks), g0 = (int)(unit % chunks) * IT;
    if (t >= a.n_tok) return;
    const int l = lane % LPH, e0 = 8 * l;
    const int NU = a.H + 2 * a.n_kv;

    // every load first
    int u[IT];
    uint4 raw[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        u[i] = (g0 + i) * HPW + lane / LPH;
        const int x = min(u[i], NU - 1);
        const uint16_t* p = x < a.H ? a.q + (long)t * a.q_st + (long)x * a.q_sh
                          : x < a.H + a.n_kv ? a.k + (long)t * a.k_st + (long)(x - a.H) * a.k_sh
                                             : a.v + (long)t * a.v_st + (long)(x - a.H - a.n_kv) * a.v_sh;
        // read once: not kept in the caches, where the outputs' next reader finds them
        // (8192 tokens 47.5 -> 45 us, with the attention behind it 133 -> 129; stores
        // past the caches too: 42.5 alone, but 134 with the attention)
        raw[i] = __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const v4i*>(p + e0)));
    }
    const int pos = a.pos[t];
    const long slot = a.slot[t];
    const bool placed = pos >= 0 && pos < a.max_pos;
    const int half = a.rot >> 1;
    const bool turned = e0 < a.rot;
    // angles of this lane's entries (8 pairs, or 4 adjacent ones); the partner lane of a half-split pair
    float c[8], s[8];
    const bool low = e0 < half;
    const int pl = (lane & ~(LPH - 1)) + (low ? l + half / 8 : l - half / 8);
    const float* row = a.cs + (long)(placed ? pos : 0) * a.rot;
    if (turned) {
        const int j = INTER ? e0 >> 1 : low ? e0 : e0 - half;
        constexpr int N = INTER ? 4 : 8;
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            const float4 x = *reinterpret_cast<const float4*>(row + j + e);
            const float4 y = *reinterpret_cast<const float4*>(row + half + j + e);
            c[e] = x.x; c[e + 1] = x.y; c[e + 2] = x.z; c[e + 3] = x.w;
            s[e] = y.x; s[e + 1] = y.y; s[e + 2] = y.z; s[e + 3] = y.w;
        }
    }
    // weights of this lane's entries and of its partner's, for q and for k
    Weights8<WF32> wq{}, wk{}, pq{}, pk{};
    const int ep = !INTER && turned ? (low ? e0 + half : e0 - half) : e0;
    if (a.qw) { wq.load(a.qw, e0); pq.load(a.qw, ep); }
    if (a.kw) { wk.load(a.kw, e0); pk.load(a.kw, ep); }
    const long blk = slot >> a.pg_sh;
    const int off = (int)(slot & ((1 << a.pg_sh) - 1));
    const bool cached = placed && slot >= 0 && slot < a.slots;

#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const bool is_q = u[i] < a.H, is_k = !is_q && u[i] < a.H + a.n_kv;
        const bool normed = is_q ? a.qw != nullptr : is_k && a.kw != nullptr;
        float x[8], y[8];
        unpack8(raw[i], x);
        uint4 pr = raw[i];
        if constexpr (!INTER) {             // the partner's raw entries
            pr.x = __shfl(raw[i].x, pl); pr.y = __shfl(raw[i].y, pl);
            pr.z = __shfl(raw[i].z, pl); pr.w = __shfl(raw[i].w, pl);
        }
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
        ss = head_sum<D>(ss);
        unpack8(pr, y);
        if (normed) {
            const float inv = rsqrtf(ss * (1.f / D) + a.eps);
            float gq[8], gk[8];
            wq.get(gq); wk.get(gk);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * (is_q ? gq[e] : gk[e]);
            if constexpr (!INTER) {
                pq.get(gq); pk.get(gk);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = y[e] * inv * (is_q ? gq[e] : gk[e]);
            }
        }
        if (turned && (is_q || is_k)) {
            if constexpr (INTER) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = x[2 * e], r = x[2 * e + 1];
                    x[2 * e] = p * c[e] - r * s[e];
                    x[2 * e + 1] = r * c[e] + p * s[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = low ? x[e] * c[e] - y[e] * s[e] : x[e] * c[e] + y[e] * s[e];
            }
        }
        uint4 out = pack8(x);
        if (!placed) out = make_uint4(0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u);
        if (u[i] < a.H) {
            *reinterpret_cast<uint4*>(a.qo + (long)t * a.qo_st + (long)u[i] * a.qo_sh + e0) = out;
        } else if (u[i] < a.H + a.n_kv) {
            const int h = u[i] - a.H;
            if (cached) *reinterpret_cast<uint4*>(a.kc + blk * a.kc_sb + (long)off * a.kc_st + (long)h * a.kc_sh + e0) = out;
            if (a.ko) *reinterpret_cast<uint4*>(a.ko + (long)t * a.ko_st + (long)h * a.ko_sh + e0) = out;
        } else if (u[i] < NU && cached) {
            const int h = u[i] - a.H - a.n_kv;
            *reinterpret_cast<uint4*>(a.vc + blk * a.vc_sb + (long)off * a.vc_st + (long)h * a.vc_sh + e0) = raw[i];
        }
    }
}

// ---- a cache in 4 bits ----------------------------------------------------------
// A code's steps are wide, and a value next to a border decides one: codes are those of
// norm and rotation in 64 bits.  In fp32 a value is off by at most 14 * 2^-24 of its
// pair's magnitude |a cos| + |b sin| (inverse root of the sum of squares 9, three products
// and the sum 4, the subtraction below 1); with twice that and more, 2^-19, on either side
// the code is mostly the same, and only the heads of a wave with a value in doubt (one
// wave of 50 to 100) go to 64 bits.  That holds where no product loses its bits below
// fp32's normal numbers: a value next to a border is 2^-104 at least (of a block whose
// largest is 2^-100, below which all is in doubt), and such a product is off by 2^-150,
// times the weight and the angle behind it: less than 2^-127 with weights below 2^16 and
// angles below 2^6, 2^-23 of the value.  Larger ones go to 64 bits.
// 8192 tokens of 48 heads: all in 64 bits 54.6 us, so 48.5 (three groups a wave; 43.1
// with six), without rounding keys at all 41.
template <int D>
__device__ __forceinline__ double head_sum(double s) {
#pragma unroll
    for (int x = D / 16; x >= 1; x >>= 1) s += __shfl_xor(s, x);
    return s;
}
// The largest word of the four lanes that share a scale.
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false));    // lane ^ 1
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false));  // lane ^ 2
}
__device__ __forceinline__ int kv4_exp(int e) { return min(max(e, -125), 125); }
__device__ __forceinline__ uint32_t codes8(const float* y) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], 1.f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.f, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.f, 3);
}
// The leading 32 bits of a double's magnitude, rounded up: not above 7 * 2^e, whose
// lower bits are zero, unless the double is.
__device__ __forceinline__ uint32_t top_bits(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x) & 0x7FFFFFFFFFFFFFFFull;
    return (uint32_t)(u >> 32) + ((uint32_t)u ? 1u : 0u);
}
// To fp32 with the last bit set where the value is not exact: what rounds to fewer
// bits from there, rounds as from 64.
__device__ __forceinline__ float to_odd(double y) {
    const float f = (float)y;
    const double d = y - (double)f;
    uint32_t u = __float_as_uint(f);
    if (d != 0.0 && !(u & 1)) u += (d > 0.0) != (bool)(u >> 31) ? 1u : -1u;
    return __uint_as_float(u);
}
// 2^-e and the scale's byte of a block whose largest magnitude has these top bits.
__device__ __forceinline__ double kv4_inverse(uint32_t top, uint32_t& byte) {
    // 1.75 = 7 / 4 is mantissa 0xC0000 of the leading 20 bits
    const int ex = kv4_exp((int)(top >> 20) - 1023 - 2 + ((top & 0xFFFFFu) > 0xC0000u ? 1 : 0));
    byte = top >= 0x7FF00000u ? 255u : (uint32_t)(ex + 127);
    return __longlong_as_double((long long)(1023 - ex) << 52);
}
// The codes of eight entries, each within 2^-19 mag of x, over their block's 2^e, and its
// byte; `doubt` where that does not tell a code.
__device__ __forceinline__ uint32_t to_codes(const float* x, const float* mag, uint32_t& byte, bool& doubt) {
    float lo[8], hi[8];
    uint32_t least = 0, most = 0;           // of the block's largest magnitude
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float d = mag[e] * 0x1p-19f;
        lo[e] = x[e] - d;
        hi[e] = x[e] + d;
        least = max(least, __float_as_uint(fmaxf(fabsf(x[e]) - d, 0.f)));
        most = max(most, __float_as_uint(fabsf(x[e]) + d));
    }
    least = block_max(least);
    most = block_max(most);
    const int ex = kv4_exp((int)(most >> 23) - 127 - 2 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0));
    const int ex_least = kv4_exp((int)(least >> 23) - 127 - 2 + ((least & 0x7FFFFFu) > 0x600000u ? 1 : 0));
    byte = (uint32_t)(ex + 127);
    const float inv = __uint_as_float((uint32_t)(127 - ex) << 23);
#pragma unroll
    for (int e = 0; e < 8; ++e) { lo[e] *= inv; hi[e] *= inv; }
    const uint32_t w = codes8(lo);
    doubt = doubt || ex != ex_least || w != codes8(hi) || most >= 0x7F800000u || most < 0x0D800000u;     // 2^-100
    return w;
}
// The same of bf16 entries, exact in fp32 (over 2^e too: the smallest is 2^-133 * 2^125).
__device__ __forceinline__ uint32_t to_codes(const uint4& raw, uint32_t& byte) {
    uint32_t top = 0;
    for (uint32_t w : {raw.x, raw.y, raw.z, raw.w}) top = max(top, max(w & 0x7FFFu, w >> 16 & 0x7FFFu));
    top = block_max(top);
    const int ex = kv4_exp((int)(top >> 7) - 127 - 2 + ((top & 0x7Fu) > 0x60u ? 1 : 0));
    byte = top >= 0x7F80u ? 255u : (uint32_t)(ex + 127);
    const float inv = __uint_as_float((uint32_t)(127 - ex) << 23);
    float y[8];
    unpack8(raw, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= inv;
    return codes8(y);
}

// Heads whose pairs turn by several axes' positions, or that go to a cache in 4 bits (KV4,
// with one axis or more).  As above, but what a token's heads share stands in LDS, in fp32:
// its angles, put together from every axis' row once, and the weights (8192 tokens along
// three axes: every lane its pairs' rows 54 us, so 44, with six groups of heads a wave
// 42.6, 4.8 TB/s).  A lane reads of them what it needs where it needs it, which leaves the
// registers to the rows on their way.  Bound by memory; into 4 bits 43.2 us, of which the
// keys' rounding is 2.
constexpr int QK_TOK = QK_WAVES;            // tokens that a workgroup's waves may stand in
template <int D, int IT, bool INTER, bool KV4>
__global__ __launch_bounds__(QK_BLK) void qkv_staged_kernel(const QkvArgs a)
{
    constexpr int LPH = D / 8, HPW = kWave / LPH;
    __shared__ __attribute__((aligned(16))) float ang_s[QK_TOK][D], w_s[2][D];
    __shared__ int wild_s[QK_WAVES];        // a weight or an angle past what to_codes' bound allows
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chunks = (a.groups + IT - 1) / IT;
    // KV4: 16 tokens share the lines of a tile.  Workgroups go round the 8 XCDs; of 128
    // of them, 16 consecutive ones' tokens go to one XCD, whose L2 puts the lines together
    int wg = blockIdx.x;
    if (KV4 && (wg | 127) < (int)gridDim.x) wg = (wg & ~127) | (wg & 7) << 4 | (wg >> 3 & 15);
    const long unit0 = (long)wg * QK_WAVES, unit = unit0 + wave;
    const int t0 = (int)(unit0 / chunks), t = min((int)(unit / chunks), a.n_tok - 1);
    const bool live = unit / chunks < a.n_tok;
    // KV4: a wave of K and V heads has several times the arithmetic of one of q heads;
    // turned by the token, they do not all come to the same SIMD of their CUs
    const int g0 = (int)((unit + (KV4 ? t : 0)) % chunks) * IT;
    const int l = lane % LPH, e0 = 8 * l;
    const int NU = a.H + 2 * a.n_kv;

    int u[IT];
    uint4 raw[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        u[i] = (g0 + i) * HPW + lane / LPH;
        const int x = min(u[i], NU - 1);
        const uint16_t* p = x < a.H ? a.q + (long)t * a.q_st + (long)x * a.q_sh
                          : x < a.H + a.n_kv ? a.k + (long)t * a.k_st + (long)(x - a.H) * a.k_sh
                                             : a.v + (long)t * a.v_st + (long)(x - a.H - a.n_kv) * a.v_sh;
        raw[i] = __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const v4i*>(p + e0)));
    }
    bool placed = true;
#pragma unroll
    for (int x = 0; x < QK_AXES; ++x) {
        const int pos = a.pos[t + min(x, a.n_axes - 1) * a.pos_ax];
        placed = placed && pos >= 0 && pos < a.max_pos;
    }
    const long slot = a.slot[t];
    const int half = a.rot >> 1;
    // the angles of this workgroup's tokens, and the weights
    bool big = false;
    const int t1 = min((int)((unit0 + QK_WAVES - 1) / chunks), a.n_tok - 1);
    for (int i = tid; i < (t1 - t0 + 1) * a.rot; i += QK_BLK) {
        const int tt = i / a.rot, j = i - tt * a.rot, pair = j < half ? j : j - half;
        const uint64_t w = pair < 32 ? a.axes[0] : pair < 64 ? a.axes[1] : pair < 96 ? a.axes[2] : a.axes[3];
        const int x = (int)(w >> (2 * (pair & 31)) & 3);
        const int pos = a.pos[t0 + tt + x * a.pos_ax];
        const float y = a.cs[(long)(pos >= 0 && pos < a.max_pos ? pos : 0) * a.rot + j];
        ang_s[tt][j] = y;
        big = big || !(fabsf(y) < 0x1p6f);
    }
    for (int i = tid; i < 2 * D; i += QK_BLK) {
        const void* w = i < D ? a.qw : a.kw;
        const int e = i % D;
        if (w) {
            const float x = a.w_f32 ? static_cast<const float*>(w)[e] : bf16_to_f32(static_cast<const uint16_t*>(w)[e]);
            w_s[i / D][e] = x;
            big = big || !(fabsf(x) < 0x1p16f);
        }
    }
    if (KV4) {
        const bool any = __any(big);
        if (lane == 0) wild_s[wave] = any;
    }
    lds_barrier();
    if (!live) return;

    const bool turned = e0 < a.rot, low = e0 < half;
    const int pl = (lane & ~(LPH - 1)) + (low ? l + half / 8 : l - half / 8);
    const float* ang = ang_s[t - t0];
    const int j = INTER ? e0 >> 1 : low ? e0 : e0 - half;
    const int ep = !INTER && turned ? (low ? e0 + half : e0 - half) : e0;
    const long blk = slot >> a.pg_sh;
    const int off = (int)(slot & ((1 << a.pg_sh) - 1));
    const bool cached = placed && slot >= 0 && slot < a.slots;
    bool wild = false;
    if constexpr (KV4)
        for (int w = 0; w < QK_WAVES; ++w) wild = wild || wild_s[w];
    auto read8 = [](const float* p, float* x) __attribute__((always_inline)) {
        const float4 y = *reinterpret_cast<const float4*>(p), z = *reinterpret_cast<const float4*>(p + 4);
        x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w; x[4] = z.x; x[5] = z.y; x[6] = z.z; x[7] = z.w;
    };

#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const bool is_q = u[i] < a.H, is_k = !is_q && u[i] < a.H + a.n_kv;
        const bool normed = is_q ? a.qw != nullptr : is_k && a.kw != nullptr;
        uint4 pr = raw[i];
        if constexpr (!INTER) {             // the partner's raw entries
            pr.x = __shfl(raw[i].x, pl); pr.y = __shfl(raw[i].y, pl);
            pr.z = __shfl(raw[i].z, pl); pr.w = __shfl(raw[i].w, pl);
        }
        uint32_t word = 0, byte = 0;        // KV4: the codes of a key's entries, and their scale
        bool doubt = false;
        if (is_q || is_k) {
            float x[8], y[8], g[8], mag[8];
            unpack8(raw[i], x);
            unpack8(pr, y);
            if (normed) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
                ss = head_sum<D>(ss) * (1.f / D) + a.eps;
                const float inv = rsqrtf(ss);
                if constexpr (KV4) doubt = !(ss > 0x1p-100f && ss < 0x1p100f);
                read8(w_s[is_q ? 0 : 1] + e0, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * g[e];
                if constexpr (!INTER) {
                    read8(w_s[is_q ? 0 : 1] + ep, g);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = y[e] * inv * g[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) mag[e] = fabsf(x[e]);
            if (turned) {
                float c[8], s[8];
                if constexpr (INTER) {
                    *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(ang + j);
                    *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(ang + half + j);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float p = x[2 * e], r = x[2 * e + 1];
                        x[2 * e] = p * c[e] - r * s[e];
                        x[2 * e + 1] = r * c[e] + p * s[e];
                        mag[2 * e] = fmaf(fabsf(p), fabsf(c[e]), fabsf(r * s[e]));
                        mag[2 * e + 1] = fmaf(fabsf(r), fabsf(c[e]), fabsf(p * s[e]));
                    }
                } else {
                    read8(ang + j, c);
                    read8(ang + half + j, s);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        mag[e] = fmaf(fabsf(x[e]), fabsf(c[e]), fabsf(y[e] * s[e]));
                        x[e] = low ? x[e] * c[e] - y[e] * s[e] : x[e] * c[e] + y[e] * s[e];
                    }
                }
            }
            if constexpr (KV4) {
                if (is_k) word = to_codes(x, mag, byte, doubt);
            }
            uint4 out = pack8(x);
            if (!placed) out = make_uint4(0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u);
            if (is_q) {
                *reinterpret_cast<uint4*>(a.qo + (long)t * a.qo_st + (long)u[i] * a.qo_sh + e0) = out;
            } else {
                const int h = u[i] - a.H;
                if (!KV4 && cached)
                    *reinterpret_cast<uint4*>(a.kc + blk * a.kc_sb + (long)off * a.kc_st + (long)h * a.kc_sh + e0) = out;
                if (a.ko) *reinterpret_cast<uint4*>(a.ko + (long)t * a.ko_st + (long)h * a.ko_sh + e0) = out;
            }
        }
        if constexpr (!KV4) {
            if (!is_q && !is_k && u[i] < NU && cached) {
                const int h = u[i] - a.H - a.n_kv;
                *reinterpret_cast<uint4*>(a.vc + blk * a.vc_sb + (long)off * a.vc_st + (long)h * a.vc_sh + e0) = raw[i];
            }
        } else if (!is_q && u[i] < NU && cached) {
            uint8_t* tile = a.c4 + blk * a.c_sb + (long)(u[i] - a.H - (is_k ? 0 : a.n_kv)) * a.c_sh + (off >> 4) * Kv4<D>::TILE;
            const int key = off & 15;
            if (is_k && __any(doubt || wild)) {
                // In 64 bits, four entries at a time, twice: rare, and eight doubles at once
                // would take registers from every wave of the kernel (104 in place of 82:
                // 8192 tokens 48.5 us, so 52.7); not where a wave's own time is the call's
                auto four = [](const uint4& x, int h, double* z) __attribute__((always_inline)) {
                    const uint32_t w0 = h ? x.z : x.x, w1 = h ? x.w : x.y;
                    z[0] = bf16lo(w0); z[1] = bf16hi(w0); z[2] = bf16lo(w1); z[3] = bf16hi(w1);
                };
                auto times = [](double* z, const float* p) __attribute__((always_inline)) {
                    const float4 g = *reinterpret_cast<const float4*>(p);
                    z[0] *= (double)g.x; z[1] *= (double)g.y; z[2] *= (double)g.z; z[3] *= (double)g.w;
                };
                double sum = 0.0, f = 1.0, z[4], p[4];
                if (normed) {
#pragma unroll IT == 1 ? 2 : 1
                    for (int h = 0; h < 2; ++h) {
                        four(raw[i], h, z);
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum = fma(z[e], z[e], sum);
                    }
                    f = 1.0 / sqrt(head_sum<D>(sum) * (1.0 / D) + (double)a.eps);
                }
                // the norm's factor comes last: entry x weight x angle is exact with bf16
                // weights (40 bits), and within 2^-53 of itself with fp32 ones (56)
                auto values = [&](int h) __attribute__((always_inline)) {
                    four(raw[i], h, z);
                    if (normed) times(z, w_s[1] + e0 + 4 * h);
                    if (turned) {
                        if constexpr (INTER) {
                            const float2 c = *reinterpret_cast<const float2*>(ang + j + 2 * h);
                            const float2 s = *reinterpret_cast<const float2*>(ang + half + j + 2 * h);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const double v = z[e ^ 1] * (double)(e < 2 ? s.x : s.y);
                                p[e] = fma(z[e], (double)(e < 2 ? c.x : c.y), (e & 1) ? v : -v);
                            }
#pragma unroll
                            for (int e = 0; e < 4; ++e) z[e] = p[e];
                        } else {
                            four(pr, h, p);
                            if (normed) times(p, w_s[1] + ep + 4 * h);
                            times(z, ang + j + 4 * h);
                            times(p, ang + half + j + 4 * h);
#pragma unroll
                            for (int e = 0; e < 4; ++e) z[e] += low ? -p[e] : p[e];
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[e] *= f;
                };
                uint32_t top = 0;
#pragma unroll IT == 1 ? 2 : 1
                for (int h = 0; h < 2; ++h) {
                    values(h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = max(top, top_bits(z[e]));
                }
                const double inv = kv4_inverse(block_max(top), byte);
                word = 0;
#pragma unroll IT == 1 ? 2 : 1
                for (int h = 0; h < 2; ++h) {
                    values(h);
                    uint32_t w = 0;
                    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, to_odd(z[0] * inv), to_odd(z[1] * inv), 1.f, 0);
                    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, to_odd(z[2] * inv), to_odd(z[3] * inv), 1.f, 1);
                    word |= w << (16 * h);
                }
            }
            if (is_k) {
                *reinterpret_cast<uint32_t*>(tile + Kv4<D>::k_code(key, l)) = word;
                if ((l & 3) == 0) tile[Kv4<D>::k_scale(key, l >> 2)] = (uint8_t)byte;
            } else {
                const uint32_t w = to_codes(raw[i], byte);
                uint8_t* p4 = tile + Kv4<D>::v_code(key, l);
                if constexpr (D == 64) {
                    *reinterpret_cast<uint16_t*>(p4) = (uint16_t)w;
                    *reinterpret_cast<uint16_t*>(p4 + 8) = (uint16_t)(w >> 16);
                } else {
                    *reinterpret_cast<uint32_t*>(p4) = w;
                }
                if ((l & 3) == 0) tile[Kv4<D>::v_scale(key, l >> 2)] = (uint8_t)byte;
            }
        }
    }
}

}  // namespace locks

using namespace locks;

namespace {

// The strides and pointers of a call, whatever its cache.
int32_t check_qkv(const char* what, const QkvArgs& a, int head_dim, int page, int num_blocks)
{
    LOCKS_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "%s: head_dim %d outside {64, 128, 256}", what, head_dim);
    LOCKS_REQUIRE(page == 16 || page == 32 || page == 64, "%s: page %d outside {16, 32, 64}", what, page);
    LOCKS_REQUIRE(a.rot >= 0 && a.rot <= head_dim && a.rot % 16 == 0,
                  "%s: rot %d is not a multiple of 16 in [0, head_dim %d]", what, a.rot, head_dim);
    LOCKS_REQUIRE(a.n_tok >= 0 && a.H >= 1 && a.n_kv >= 1 && num_blocks >= 1 && a.max_pos >= 1, "%s: empty geometry", what);
    LOCKS_REQUIRE(a.H <= 4096 && a.n_kv <= 4096, "%s: more than 4096 heads", what);
    LOCKS_REQUIRE(a.eps >= 0.f, "%s: eps must not be negative", what);
    LOCKS_REQUIRE(a.q && a.k && a.v && a.pos && a.slot && (a.c4 || (a.kc && a.vc)) && a.qo && (a.cs || a.rot == 0),
                  "%s: null pointer argument", what);
    for (int64_t x : {a.q_st, a.q_sh, a.k_st, a.k_sh, a.v_st, a.v_sh, a.kc_sb, a.kc_st, a.kc_sh, a.vc_sb, a.vc_st, a.vc_sh,
                      a.qo_st, a.qo_sh, a.ko_st, a.ko_sh})
        LOCKS_REQUIRE(x % 8 == 0, "%s: strides must be multiples of 8 elements (16-byte accesses)", what);
    for (const void* x : {(const void*)a.q, (const void*)a.k, (const void*)a.v, (const void*)a.kc, (const void*)a.vc,
                          (const void*)a.qo, (const void*)a.ko, (const void*)a.cs, a.qw, a.kw})
        LOCKS_REQUIRE((uintptr_t)x % 16 == 0, "%s: pointers must be 16-byte aligned", what);
    return 0;
}
int32_t check_axes(const char* what, QkvArgs& a, int32_t n_axes, int64_t pos_stride, const int64_t (&words)[4])
{
    LOCKS_REQUIRE(n_axes >= 0 && n_axes <= QK_AXES, "%s: n_axes %d outside [0, %d]", what, n_axes, QK_AXES);
    if (n_axes == 0) return 0;
    uint64_t axes[4];
    for (int i = 0; i < 4; ++i) axes[i] = (uint64_t)words[i];
    for (int j = 0; j < a.rot / 2; ++j)
        LOCKS_REQUIRE((int)(axes[j >> 5] >> (2 * (j & 31)) & 3) < n_axes, "%s: pair %d turns by an axis past the %d", what, j, n_axes);
    a.n_axes = n_axes;
    a.pos_ax = pos_stride;
    for (int i = 0; i < 4; ++i) a.axes[i] = axes[i];
    return 0;
}

int32_t launch_qkv(QkvArgs a, bool kv4, int head_dim, int interleaved, int weights_f32, hipStream_t st)
{
    if (a.n_tok == 0) return 0;
    a.groups = cdiv(a.H + 2 * a.n_kv, 512 / head_dim);
    // groups per wave: the angles and weights of a token are loaded once for them,
    // and their rows are in flight together (8192 tokens of 48 heads: 2 groups 50.5
    // us, 3 and 4 45)
    constexpr int IT = 3;
    auto grid_of = [&](int it) { return dim3((unsigned)(((long)a.n_tok * cdiv(a.groups, it) + QK_WAVES - 1) / QK_WAVES)); };
    const dim3 grid = grid_of(IT);
    a.w_f32 = weights_f32;
    // The staged kernel.  One group per wave up to two waves a SIMD, where a call is as
    // long as one wave (32 tokens of 12 groups, along three axes 4.7 -> 3.6 us; 512 tokens
    // 5.9 -> 6.6); six where many workgroups follow each other on a CU and their starts
    // (positions, angles, barrier) count (8192 tokens, into 4 bits 48.3 -> 43.1; 4097 of an
    // image encoder 13.6 -> 11.7; 512 tokens 5.9 -> 7.0).
    const long units = (long)a.n_tok * a.groups;
    const int it = units <= 2048 ? 1 : units < 16384 ? IT : 6;
    const dim3 grid_s = grid_of(it);
#define LAUNCH_S(DV, INTER, KV4)                                                                                   \
    if (it == 1) hipLaunchKernelGGL((qkv_staged_kernel<DV, 1, INTER, KV4>), grid_s, dim3(QK_BLK), 0, st, a);       \
    else if (it == IT) hipLaunchKernelGGL((qkv_staged_kernel<DV, IT, INTER, KV4>), grid_s, dim3(QK_BLK), 0, st, a); \
    else hipLaunchKernelGGL((qkv_staged_kernel<DV, 6, INTER, KV4>), grid_s, dim3(QK_BLK), 0, st, a)
#define LAUNCH_W(DV, INTER)                                                                                             \
    if (kv4) { LAUNCH_S(DV, INTER, true); }                                                                             \
    else if (a.n_axes) { LAUNCH_S(DV, INTER, false); }                                                                  \
    else if (weights_f32) hipLaunchKernelGGL((qkv_write_kernel<DV, IT, INTER, true>), grid, dim3(QK_BLK), 0, st, a);    \
    else hipLaunchKernelGGL((qkv_write_kernel<DV, IT, INTER, false>), grid, dim3(QK_BLK), 0, st, a)
#define LAUNCH(DV)                              \
    if (interleaved) { LAUNCH_W(DV, true); }    \
    else { LAUNCH_W(DV, false); }
    if (head_dim == 64) { LAUNCH(64); }
    else if (head_dim == 128) { LAUNCH(128); }
    else { LAUNCH(256); }
#undef LAUNCH
#undef LAUNCH_W
#undef LAUNCH_S
    return check_launch("qkv_write_kernel");
}

int page_shift(int page) { return page == 16 ? 4 : page == 32 ? 5 : 6; }

}  // namespace

extern "C" int32_t locks_qkv_write_axes(
    const uint16_t* q, int64_t q_stride_tok, int64_t q_stride_head, const uint16_t* k, int64_t k_stride_tok,
    int64_t k_stride_head, const uint16_t* v, int64_t v_stride_tok, int64_t v_stride_head, const int32_t* positions,
    int64_t pos_stride_axis, int32_t n_axes, int64_t axes0, int64_t axes1, int64_t axes2, int64_t axes3,
    const int64_t* slot_mapping, uint16_t* k_cache, int64_t kc_stride_block, int64_t kc_stride_tok,
    int64_t kc_stride_head, uint16_t* v_cache, int64_t vc_stride_block, int64_t vc_stride_tok, int64_t vc_stride_head,
    int32_t num_blocks, const float* cos_sin, int32_t max_pos, int32_t rot, int32_t interleaved, const void* q_weight,
    const void* k_weight, int32_t weights_f32, float eps, uint16_t* q_out, int64_t qo_stride_tok,
    int64_t qo_stride_head, uint16_t* k_out, int64_t ko_stride_tok, int64_t ko_stride_head, int32_t n_tokens,
    int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t page, void* stream)
{
    const char* what = "locks_qkv_write_axes";
    QkvArgs a{q, q_stride_tok, q_stride_head, k, k_stride_tok, k_stride_head, v, v_stride_tok, v_stride_head,
              positions, slot_mapping, k_cache, kc_stride_block, kc_stride_tok, kc_stride_head, v_cache,
              vc_stride_block, vc_stride_tok, vc_stride_head, cos_sin, q_weight, k_weight, q_out, qo_stride_tok,
              qo_stride_head, k_out, ko_stride_tok, ko_stride_head, (long)num_blocks * page, max_pos, rot,
              n_tokens, n_heads, n_kv, page_shift(page), 0, eps, 0, 0, {}, 0, nullptr, 0, 0};
    int rc = check_qkv(what, a, head_dim, page, num_blocks);
    if (rc) return rc;
    LOCKS_REQUIRE(n_axes >= 1, "%s: n_axes %d outside [1, %d]", what, n_axes, QK_AXES);
    rc = check_axes(what, a, n_axes, pos_stride_axis, {axes0, axes1, axes2, axes3});
    if (rc) return rc;
    return launch_qkv(a, false, head_dim, interleaved, weights_f32, (hipStream_t)stream);
}

extern "C" int32_t locks_kv4_write(
    const uint16_t* q, int64_t q_stride_tok, int64_t q_stride_head, const uint16_t* k, int64_t k_stride_tok,
    int64_t k_stride_head, const uint16_t* v, int64_t v_stride_tok, int64_t v_stride_head, const int32_t* positions,
    int64_t pos_stride_axis, int32_t n_axes, int64_t axes0, int64_t axes1, int64_t axes2, int64_t axes3,
    const int64_t* slot_mapping, uint8_t* cache, int64_t c_stride_block, int64_t c_stride_head, int32_t num_blocks,
    const float* cos_sin, int32_t max_pos, int32_t rot, int32_t interleaved, const void* q_weight, const void* k_weight,
    int32_t weights_f32, float eps, uint16_t* q_out, int64_t qo_stride_tok, int64_t qo_stride_head, uint16_t* k_out,
    int64_t ko_stride_tok, int64_t ko_stride_head, int32_t n_tokens, int32_t n_heads, int32_t n_kv, int32_t head_dim,
    int32_t page, void* stream)
{
    const char* what = "locks_kv4_write";
    QkvArgs a{q, q_stride_tok, q_stride_head, k, k_stride_tok, k_stride_head, v, v_stride_tok, v_stride_head,
              positions, slot_mapping, nullptr, 0, 0, 0, nullptr, 0, 0, 0, cos_sin, q_weight, k_weight, q_out,
              qo_stride_tok, qo_stride_head, k_out, ko_stride_tok, ko_stride_head, (long)num_blocks * page, max_pos, rot,
              n_tokens, n_heads, n_kv, page_shift(page), 0, eps, 0, 0, {}, 0, cache, c_stride_block, c_stride_head};
    int rc = check_kv4(what, cache, c_stride_block, c_stride_head, num_blocks, n_kv, head_dim, page);
    if (rc) return rc;
    rc = check_qkv(what, a, head_dim, page, num_blocks);
    if (rc) return rc;
    rc = check_axes(what, a, n_axes, pos_stride_axis, {axes0, axes1, axes2, axes3});
    if (rc) return rc;
    a.n_axes = n_axes ? n_axes : 1;         // one position: one axis, all words 0
    return launch_qkv(a, true, head_dim, interleaved, weights_f32, (hipStream_t)stream);
}

extern "C" int32_t locks_qkv_write(
    const uint16_t* q, int64_t q_stride_tok, int64_t q_stride_head, const uint16_t* k, int64_t k_stride_tok,
    int64_t k_stride_head, const uint16_t* v, int64_t v_stride_tok, int64_t v_stride_head, const int32_t* positions,
    const int64_t* slot_mapping, uint16_t* k_cache, int64_t kc_stride_block, int64_t kc_stride_tok,
    int64_t kc_stride_head, uint16_t* v_cache, int64_t vc_stride_block, int64_t vc_stride_tok, int64_t vc_stride_head,
    int32_t num_blocks, const float* cos_sin, int32_t max_pos, int32_t rot, int32_t interleaved, const void* q_weight,
    const void* k_weight, int32_t weights_f32, float eps, uint16_t* q_out, int64_t qo_stride_tok,
    int64_t qo_stride_head, uint16_t* k_out, int64_t ko_stride_tok, int64_t ko_stride_head, int32_t n_tokens,
    int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t page, void* stream)
{
    const QkvArgs a{q, q_stride_tok, q_stride_head, k, k_stride_tok, k_stride_head, v, v_stride_tok, v_stride_head,
                    positions, slot_mapping, k_cache, kc_stride_block, kc_stride_tok, kc_stride_head, v_cache,
                    vc_stride_block, vc_stride_tok, vc_stride_head, cos_sin, q_weight, k_weight, q_out, qo_stride_tok,
                    qo_stride_head, k_out, ko_stride_tok, ko_stride_head, (long)num_blocks * page, max_pos, rot,
                    n_tokens, n_heads, n_kv, page_shift(page), 0, eps, 0, 0, {}, 0, nullptr, 0, 0};
    const int rc = check_qkv("locks_qkv_write", a, head_dim, page, num_blocks);
    if (rc) return rc;
    return launch_qkv(a, false, head_dim, interleaved, weights_f32, (hipStream_t)stream);
}
