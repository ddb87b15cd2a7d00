// Element types and dropout masks of the operators that take fp32, bf16 or fp16 activations: arithmetic is fp32, a
// value is rounded (to nearest even) once, where it is stored.
#pragma once
#include <type_traits>
#include "siv_common.h"

namespace siv {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// calls f with a null pointer of the element type `type` stands for
template <typename F>
static inline int with_type(int type, F f) {
    if (type == SIV_F32) return f((float*)nullptr);
    if (type == SIV_BF16) return f((bf16_t*)nullptr);
    return f((f16_t*)nullptr);
}
static inline bool known_type(int type) { return type == SIV_F32 || type == SIV_BF16 || type == SIV_F16; }
static inline int type_size(int type) { return type == SIV_F32 ? 4 : 2; }

// ---- 16 bytes of a row --------------------------------------------------------------------------------------------
template <typename T>
struct alignas(16) Pack {
    static constexpr int N = 16 / sizeof(T);
    T e[N];
};
// `have` elements of the row are left at p (<= 0: none, the pack is zero; >= N: a whole one).  AL: p is 16-byte
// aligned and have is a multiple of N.  Otherwise p has the element's alignment only: the hardware takes a 16-byte
// access at any address, so whole packs still are one instruction.
template <bool AL, typename T>
__device__ __forceinline__ Pack<T> load_pack(const T* p, long have) {
    constexpr int N = Pack<T>::N;
    Pack<T> v;
    if (AL) {
        if (have > 0) v = *reinterpret_cast<const Pack<T>*>(p);
        else
#pragma unroll
            for (int j = 0; j < N; ++j) v.e[j] = (T)0.f;
    } else if (have >= N) {
        __builtin_memcpy(v.e, p, 16);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v.e[j] = j < have ? p[j] : (T)0.f;
    }
    return v;
}
template <bool AL, typename T>
__device__ __forceinline__ void store_pack(T* p, long have, const Pack<T>& v) {
    constexpr int N = Pack<T>::N;
    if (AL) {
        if (have > 0) *reinterpret_cast<Pack<T>*>(p) = v;
    } else if (have >= N) {
        __builtin_memcpy(p, v.e, 16);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < have) p[j] = v.e[j];
    }
}
static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// ---- dropout as an operator's own step: the mask is a stored tensor, or drawn here, or absent ------------------------
struct Drop {
    const uint8_t* keep;              // stored mask, element order of the tensor
    uint64_t seed, sid;
    const unsigned long long* epoch;
    uint32_t thresh;                  // an element is kept when the top 24 bits of its word are >= thresh
    float scale;                      // 1 / (1 - p)
    int mode;                         // 0: keep everything, 1: draw, 2: read `keep`
};
// p in [0, 1): the smallest 24-bit integer t with t * 2^-24 >= p, so that the integer comparison is philox_keeps
static inline Drop make_drop(const uint8_t* keep, uint64_t seed, uint64_t sid, const uint64_t* epoch, float p) {
    Drop d;
    d.keep = keep;
    d.seed = seed;
    d.sid = sid;
    d.epoch = (const unsigned long long*)epoch;
    const double t = (double)p * 16777216.0;
    d.thresh = (uint32_t)t;
    if ((double)d.thresh < t) ++d.thresh;
    d.scale = 1.0f / (1.0f - p);
    d.mode = keep ? 2 : (p > 0.f ? 1 : 0);
    return d;
}
__device__ __forceinline__ uint64_t drop_sid(const Drop& d) {
    return (d.mode == 1 && d.epoch) ? d.sid + *d.epoch * SIV_EPOCH_STRIDE : d.sid;
}
// Bits 0 .. N-1: elements i .. i+N-1 are kept; of those, only the first `have` exist (others: unspecified).  QUAD: i is
// a multiple of 4, so the N elements are whole Philox calls; otherwise one call more and a shift.
template <int N, bool QUAD>
__device__ __forceinline__ uint32_t drop_bits(const Drop& d, uint64_t sid, long i, long have) {
    if (d.mode == 0) return ~0u;
    uint32_t bits = 0;
    if (d.mode == 2) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < have) bits |= (uint32_t)(d.keep[i + j] != 0) << j;
        return bits;
    }
    const uint64_t q = (uint64_t)i >> 2;
    constexpr int CALLS = N / 4 + (QUAD ? 0 : 1);
#pragma unroll
    for (int k = 0; k < CALLS; ++k) {
        const u4 r = philox4x32_10(q + k, sid, d.seed);
        bits |= (uint32_t)((r.x >> 8) >= d.thresh) << (4 * k);
        bits |= (uint32_t)((r.y >> 8) >= d.thresh) << (4 * k + 1);
        bits |= (uint32_t)((r.z >> 8) >= d.thresh) << (4 * k + 2);
        bits |= (uint32_t)((r.w >> 8) >= d.thresh) << (4 * k + 3);
    }
    return QUAD ? bits : bits >> ((uint32_t)i & 3);
}

}  // namespace siv
