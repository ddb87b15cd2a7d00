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
// A result that nothing in the call reads again: stored non-temporally, so that it leaves the L2 (which a kernel's end
// writes back anyway) to the operands.
template <typename T>
__device__ __forceinline__ void store_stream(T* p, const Pack<T>& v) {
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    words w;
    __builtin_memcpy(&w, v.e, 16);
    __builtin_nontemporal_store(w, reinterpret_cast<words*>(p));
}
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
        if (have > 0) store_stream(p, v);
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
    uint32_t least;                   // an element is kept when its word is >= least
    float scale;                      // 1 / (1 - p)
    int mode;                         // 0: keep everything, 1: draw, 2: read `keep`
};
// p in [0, 1).  A drawn element is kept when the top 24 bits of its word, as a fraction, are >= p (philox_keeps), i.e.
// when the word is >= ceil(p 2^24) 2^8, which is at most (2^24 - 1) 2^8 for p < 1.  A stored mask's words are 0 or ~0.
static inline Drop make_drop(const uint8_t* keep, uint64_t seed, uint64_t sid, const uint64_t* epoch, float p) {
    Drop d;
    d.keep = keep;
    d.seed = seed;
    d.sid = sid;
    d.epoch = (const unsigned long long*)epoch;
    d.mode = keep ? 2 : (p > 0.f ? 1 : 0);
    const double t = (double)p * 16777216.0;
    uint32_t k = (uint32_t)t;
    if ((double)k < t) ++k;
    d.least = d.mode == 1 ? k << 8 : 1;
    d.scale = 1.0f / (1.0f - p);
    return d;
}
__device__ __forceinline__ uint64_t drop_sid(const Drop& d) {
    return (d.mode == 1 && d.epoch) ? d.sid + *d.epoch * SIV_EPOCH_STRIDE : d.sid;
}
// Words of elements i .. i+N-1 of a stored mask, of which the first `have` exist.
template <int N>
__device__ __forceinline__ void stored_words(const Drop& d, uint64_t i, long have, uint32_t (&w)[N]) {
    if (have >= N) {
        uint8_t m[N];
        __builtin_memcpy(m, d.keep + i, N);
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = m[j] ? ~0u : 0u;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = (j < have && d.keep[i + j]) ? ~0u : 0u;
    }
}
// The same drawn.  QUAD: i is a multiple of 4, so the N elements are whole Philox calls; otherwise one call more and a
// shift by 0 to 3 words.
template <int N, bool QUAD>
__device__ __forceinline__ void drawn_words(const Drop& d, uint64_t sid, uint64_t i, uint32_t (&w)[N]) {
    const uint64_t q = i >> 2;
    constexpr int CALLS = N / 4 + (QUAD ? 0 : 1);
    uint32_t v[CALLS * 4];
#pragma unroll
    for (int k = 0; k < CALLS; ++k) {
        const u4 r = philox4x32_10(q + k, sid, d.seed);
        v[4 * k] = r.x;
        v[4 * k + 1] = r.y;
        v[4 * k + 2] = r.z;
        v[4 * k + 3] = r.w;
    }
    if (!QUAD) {
        // (values, not elements, are chosen between: a choice of elements becomes an array in LDS, and with it a read of
        // the launch packet by every wave)
        const bool one = i & 1, two = i & 2;
#pragma unroll
        for (int j = 0; j + 1 < CALLS * 4; ++j) {
            const uint32_t here = v[j], next = v[j + 1];
            v[j] = one ? next : here;
        }
#pragma unroll
        for (int j = 0; j + 2 < CALLS * 4; ++j) {
            const uint32_t here = v[j], next = v[j + 2];
            v[j] = two ? next : here;
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = v[j];
}
// modes 1 and 2
template <int N, bool QUAD>
__device__ __forceinline__ void drop_words(const Drop& d, uint64_t sid, uint64_t i, long have, uint32_t (&w)[N]) {
    if (d.mode == 2) stored_words<N>(d, i, have, w);
    else drawn_words<N, QUAD>(d, sid, i, w);
}

}  // namespace siv
