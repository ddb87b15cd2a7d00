// Element types of the operators that take fp32, bf16 or fp16 activations: arithmetic is fp32, a value is rounded
// (to nearest even) once, where it is stored.
#pragma once
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

// a weight vector of either type (the activations' own, or fp32), read one element at a time
template <typename T>
__device__ __forceinline__ float ld_param(const void* w, int f32, long i) {
    return f32 ? ((const float*)w)[i] : (float)((const T*)w)[i];
}

// Dropout as an operator's own step: the mask is a stored tensor, or drawn here, or absent.
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

}  // namespace siv
