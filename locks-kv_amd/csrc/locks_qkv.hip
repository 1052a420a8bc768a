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
#include "locks_common.h"
#include "locks_hip.h"

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
};

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

}  // namespace locks

using namespace locks;

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
    LOCKS_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256,
                  "locks_qkv_write: head_dim %d outside {64, 128, 256}", head_dim);
    LOCKS_REQUIRE(page == 16 || page == 32 || page == 64, "locks_qkv_write: page %d outside {16, 32, 64}", page);
    LOCKS_REQUIRE(rot >= 0 && rot <= head_dim && rot % 16 == 0,
                  "locks_qkv_write: rot %d is not a multiple of 16 in [0, head_dim %d]", rot, head_dim);
    LOCKS_REQUIRE(n_tokens >= 0 && n_heads >= 1 && n_kv >= 1 && num_blocks >= 1 && max_pos >= 1,
                  "locks_qkv_write: empty geometry");
    LOCKS_REQUIRE(n_heads <= 4096 && n_kv <= 4096, "locks_qkv_write: more than 4096 heads");
    LOCKS_REQUIRE(eps >= 0.f, "locks_qkv_write: eps must not be negative");
    LOCKS_REQUIRE(q && k && v && positions && slot_mapping && k_cache && v_cache && q_out && (cos_sin || rot == 0),
                  "locks_qkv_write: null pointer argument");
    for (int64_t x : {q_stride_tok, q_stride_head, k_stride_tok, k_stride_head, v_stride_tok, v_stride_head,
                      kc_stride_block, kc_stride_tok, kc_stride_head, vc_stride_block, vc_stride_tok, vc_stride_head,
                      qo_stride_tok, qo_stride_head, ko_stride_tok, ko_stride_head})
        LOCKS_REQUIRE(x % 8 == 0, "locks_qkv_write: strides must be multiples of 8 elements (16-byte accesses)");
    for (const void* x : {(const void*)q, (const void*)k, (const void*)v, (const void*)k_cache, (const void*)v_cache,
                          (const void*)q_out, (const void*)k_out, (const void*)cos_sin, q_weight, k_weight})
        LOCKS_REQUIRE((uintptr_t)x % 16 == 0, "locks_qkv_write: pointers must be 16-byte aligned");
    if (n_tokens == 0) return 0;
    const int per_wave = 512 / head_dim;
    QkvArgs a{q, q_stride_tok, q_stride_head, k, k_stride_tok, k_stride_head, v, v_stride_tok, v_stride_head,
              positions, slot_mapping, k_cache, kc_stride_block, kc_stride_tok, kc_stride_head, v_cache,
              vc_stride_block, vc_stride_tok, vc_stride_head, cos_sin, q_weight, k_weight, q_out, qo_stride_tok,
              qo_stride_head, k_out, ko_stride_tok, ko_stride_head, (long)num_blocks * page, max_pos, rot,
              n_tokens, n_heads, n_kv, page == 16 ? 4 : page == 32 ? 5 : 6,
              cdiv(n_heads + 2 * n_kv, per_wave), eps};
    hipStream_t st = (hipStream_t)stream;
    // groups per wave: the angles and weights of a token are loaded once for them,
    // and their rows are in flight together (8192 tokens of 48 heads: 2 groups 50.5
    // us, 3 and 4 45)
    constexpr int IT = 3;
    const long waves = (long)n_tokens * cdiv(a.groups, IT);
    const dim3 grid((unsigned)((waves + QK_WAVES - 1) / QK_WAVES));
#define LAUNCH_W(DV, INTER)                                                                                     \
    if (weights_f32) hipLaunchKernelGGL((qkv_write_kernel<DV, IT, INTER, true>), grid, dim3(QK_BLK), 0, st, a); \
    else hipLaunchKernelGGL((qkv_write_kernel<DV, IT, INTER, false>), grid, dim3(QK_BLK), 0, st, a)
#define LAUNCH(DV)                              \
    if (interleaved) { LAUNCH_W(DV, true); }    \
    else { LAUNCH_W(DV, false); }
    if (head_dim == 64) { LAUNCH(64); }
    else if (head_dim == 128) { LAUNCH(128); }
    else { LAUNCH(256); }
#undef LAUNCH
#undef LAUNCH_W
    return check_launch("qkv_write_kernel");
}
