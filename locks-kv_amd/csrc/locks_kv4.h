// The paged cache in 4 bits: its layout and the conversions of its entries.
//
// 32 consecutive entries of one head of one token share a scale 2^e (one byte, e +
// 127); an entry is sign, two bits of exponent and one of mantissa: +-{0, 0.5, 1, 1.5,
// 2, 3, 4, 6} 2^e, the type that this card converts with the scale in one instruction
// for two entries (the 4-bit integers of other formats take a subtraction, a
// conversion and a product each).  e is the smallest whole number of [-125, 125] with
// max |x| <= 7 * 2^e: no entry is off by more than half a step (6 to 8 have 6 as their
// neighbour, 7 is off by 1 as 5 is); rms error of normal entries 0.112 of them, with
// 6 in place of 7 0.115, with 8 0.115.  The exponents' range keeps every value a normal
// number that bf16 holds.  A block with an infinite or NaN entry has scale byte 255
// and reads as NaN.
//
// 16 tokens of one (block, kv head) are one tile of 17 d consecutive bytes, laid out
// in the order in which a wave's lanes take them:
//   K codes   8 d   lane 16 kg + key: entries [kg d / 4, (kg + 1) d / 4) of token key
//   V codes   8 d   lane 16 kg + r: entries [r d / 16, (r + 1) d / 16) of tokens 4 kg ..
//   K scales  d/2   of lane 16 kg + key's entries
//   V scales  d/2   (kg, entry block, token & 3)
// d / 8 bytes a lane; at d 256 two planes of 16 bytes a lane.  These are the operands
// of 16x16x32 matrix products as they stand, with the sum over d of K's products, and
// over tokens of V's, in another order: no transpose, no pass through LDS.
#pragma once

#include "locks_common.h"

namespace locks {

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef int v2i __attribute__((ext_vector_type(2)));

template <int D>
struct Kv4 {
    static constexpr int TILE = 17 * D;             // bytes of 16 tokens, K and V
    static constexpr int VC = 8 * D, KS = 16 * D, VS = 16 * D + D / 2;
    static constexpr int W = D / 32;                // words of a lane's codes, K or V
    static constexpr int NBLK = D / 32;             // scales of a token

    // byte offset of the word of codes of K entries 8 l .. 8 l + 7 of a token
    static __device__ __forceinline__ int k_code(int key, int l) {
        const int kg = l / W, st = l % W;
        return D == 256 ? (st >> 2) * 1024 + (kg * 16 + key) * 16 + (st & 3) * 4 : (kg * 16 + key) * (D / 8) + st * 4;
    }
    // and of V's; at d 64 of the first half of it, the other one is 8 bytes on
    static __device__ __forceinline__ int v_code(int key, int l) {
        const int kg = key >> 2, i = key & 3;
        if constexpr (D == 64) return VC + (kg * 16 + 2 * l) * 8 + 2 * i;
        else if constexpr (D == 128) return VC + (kg * 16 + l) * 16 + 4 * i;
        else return VC + (i >> 1) * 1024 + (kg * 16 + (l >> 1)) * 16 + (i & 1) * 8 + (l & 1) * 4;
    }
    static __device__ __forceinline__ int k_scale(int key, int blk) {
        return KS + (D == 256 ? ((blk >> 1) * 16 + key) * 2 + (blk & 1) : blk * 16 + key);
    }
    static __device__ __forceinline__ int v_scale(int key, int blk) { return VS + ((key >> 2) * NBLK + blk) * 4 + (key & 3); }
};

// The codes and scales of a tile that one lane holds.
template <int D>
struct Kv4Lane {
    uint32_t w[D / 32];
    uint32_t s;                                     // K: one or two scale bytes; V: one of each token
};
// (by pointers of the global address space: an address put together from integers would
// be loaded from through the path that LDS shares)
typedef const __attribute__((address_space(1))) uint8_t* kv4_ptr;
// NT: read once (decode), so past the caches; a prompt's tiles are read by all its rows.
template <typename T, bool NT>
__device__ __forceinline__ T kv4_read(kv4_ptr p) {
    const __attribute__((address_space(1))) T* q = (const __attribute__((address_space(1))) T*)p;
    if constexpr (NT) return __builtin_nontemporal_load(q);
    else return *q;
}
template <int D, bool NT>
__device__ __forceinline__ void kv4_codes(kv4_ptr p, int lane, uint32_t* w) {
    if constexpr (D == 64) {
        const v2i x = kv4_read<v2i, NT>(p + lane * 8);
        w[0] = x[0]; w[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < D / 128; ++i) {
            const v4i x = kv4_read<v4i, NT>(p + i * 1024 + lane * 16);
            w[4 * i] = x[0]; w[4 * i + 1] = x[1]; w[4 * i + 2] = x[2]; w[4 * i + 3] = x[3];
        }
    }
}
template <int D, bool NT>
__device__ __forceinline__ void kv4_load_k(kv4_ptr tile, int lane, Kv4Lane<D>& x) {
    kv4_codes<D, NT>(tile, lane, x.w);
    if constexpr (D == 64) x.s = tile[Kv4<D>::KS + (lane >> 5) * 16 + (lane & 15)];
    else if constexpr (D == 128) x.s = tile[Kv4<D>::KS + lane];
    else x.s = *(const __attribute__((address_space(1))) uint16_t*)(tile + Kv4<D>::KS + 2 * lane);
}
template <int D, bool NT>
__device__ __forceinline__ void kv4_load_v(kv4_ptr tile, int lane, Kv4Lane<D>& x) {
    kv4_codes<D, NT>(tile + Kv4<D>::VC, lane, x.w);
    const int blk = (lane & 15) * (D / 16) / 32;
    x.s = *(const __attribute__((address_space(1))) uint32_t*)(tile + Kv4<D>::VS + ((lane >> 4) * Kv4<D>::NBLK + blk) * 4);
}

// The scale 2^e of a byte as the converters take it (255: infinite, whose entries
// they turn into NaN).
__device__ __forceinline__ float kv4_scale(uint32_t s, int byte) { return __uint_as_float(((s >> (8 * byte)) & 255u) << 23); }

// Entries 2 byte and 2 byte + 1 of a word of codes, as packed bf16: exact.
template <int BYTE>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, BYTE));
}
// The eight entries of a word, in order.
__device__ __forceinline__ uint4 kv4_eight(uint32_t w, float scale) {
    return make_uint4(kv4_pair<0>(w, scale), kv4_pair<1>(w, scale), kv4_pair<2>(w, scale), kv4_pair<3>(w, scale));
}

// What kv4_merge_kernel joins: partials m (the maximum, as a base-2 logarithm of the
// weight), l and acc, of a row's shares, or of its `splits`.
struct Kv4MergeArgs {
    const float* m; const float* l; const float* acc;
    const int2* shares;                     // or null: splits
    int splits;
    const int* starts; int n_seq;           // splits: the requests' first tokens
    uint16_t* out; long o_sr, o_sh;
    float* lse; long lse_sr;
    int n_kv, G;
};
int launch_kv4_merge(const Kv4MergeArgs& a, int n_rows, int head_dim, hipStream_t st);

}  // namespace locks
