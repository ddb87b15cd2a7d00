// Dropout whose mask is never stored (fp32, bf16, fp16): out = [residual +] keep * act(x) / (1 - p).
#include "elem_types.h"

namespace siv {

// One thread per quad of elements: one Philox call is four of them.
template <typename T>
__global__ __launch_bounds__(256) void dropout_fwd_k(const T* __restrict__ x, const T* __restrict__ res, Drop d,
                                                     float slope, T* __restrict__ out, long n) {
    const uint64_t sid = drop_sid(d);
    const long quads = (n + 3) / 4;
    for (long q = (long)blockIdx.x * 256 + threadIdx.x; q < quads; q += (long)gridDim.x * 256) {
        uint32_t w[4] = {~0u, ~0u, ~0u, ~0u};
        if (d.mode == 1) {
            const u4 r = philox4x32_10((uint64_t)q, sid, d.seed);
            w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
        }
        for (int j = 0; j < 4; ++j) {
            const long i = q * 4 + j;
            if (i >= n) break;
            float v = leaky((float)x[i], slope);
            if (d.mode) v = (d.mode == 1 ? (w[j] >> 8) >= d.thresh : d.keep[i] != 0) ? v * d.scale : 0.f;
            out[i] = (T)(res ? (float)res[i] + v : v);
        }
    }
}
template <typename T>
__global__ __launch_bounds__(256) void dropout_bwd_k(const T* __restrict__ dout, const T* __restrict__ x, Drop d,
                                                     float slope, T* __restrict__ dx, long n) {
    const uint64_t sid = drop_sid(d);
    const long quads = (n + 3) / 4;
    for (long q = (long)blockIdx.x * 256 + threadIdx.x; q < quads; q += (long)gridDim.x * 256) {
        uint32_t w[4] = {~0u, ~0u, ~0u, ~0u};
        if (d.mode == 1) {
            const u4 r = philox4x32_10((uint64_t)q, sid, d.seed);
            w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
        }
        for (int j = 0; j < 4; ++j) {
            const long i = q * 4 + j;
            if (i >= n) break;
            float g = (float)dout[i];
            if (d.mode) g = (d.mode == 1 ? (w[j] >> 8) >= d.thresh : d.keep[i] != 0) ? g * d.scale : 0.f;
            dx[i] = (T)(x ? g * leaky_grad((float)x[i], slope) : g);
        }
    }
}

}  // namespace siv

using namespace siv;

#define SIV_CHECK_DROP(what)                                                                              \
    SIV_CHECK_ARG(known_type(type), what ": unknown element type");                                       \
    SIV_CHECK_ARG(p >= 0.f && p < 1.f, what ": dropout p out of range")

extern "C" int siv_dropout_fwd(const void* x, const void* residual, const uint8_t* keep, uint64_t seed,
                               uint64_t stream_id, const uint64_t* epoch, float p, float slope, void* out,
                               int type, long n, siv_stream_t stream) {
    SIV_CHECK_ARG(x && out && n > 0, "dropout_fwd: bad argument");
    SIV_CHECK_DROP("dropout_fwd");
    const Drop d = make_drop(keep, seed, stream_id, epoch, p);
    return with_type(type, [&](auto* t) {
        typedef typename std::remove_reference<decltype(*t)>::type T;
        const long g = cdiv(cdiv(n, 4), 256);
        dropout_fwd_k<T><<<(unsigned)(g > 4096 ? 4096 : g), 256, 0, (hipStream_t)stream>>>(
            (const T*)x, (const T*)residual, d, slope, (T*)out, n);
        SIV_CHECK_LAUNCH("dropout_fwd");
        return SIV_OK;
    });
}
extern "C" int siv_dropout_bwd(const void* dout, const void* x, const uint8_t* keep, uint64_t seed,
                               uint64_t stream_id, const uint64_t* epoch, float p, float slope, void* dx, int type,
                               long n, siv_stream_t stream) {
    SIV_CHECK_ARG(dout && dx && n > 0, "dropout_bwd: bad argument");
    SIV_CHECK_ARG(x || slope == 1.f, "dropout_bwd: the activation's backward needs x");
    SIV_CHECK_DROP("dropout_bwd");
    const Drop d = make_drop(keep, seed, stream_id, epoch, p);
    return with_type(type, [&](auto* t) {
        typedef typename std::remove_reference<decltype(*t)>::type T;
        const long g = cdiv(cdiv(n, 4), 256);
        dropout_bwd_k<T><<<(unsigned)(g > 4096 ? 4096 : g), 256, 0, (hipStream_t)stream>>>(
            (const T*)dout, slope == 1.f ? nullptr : (const T*)x, d, slope, (T*)dx, n);
        SIV_CHECK_LAUNCH("dropout_bwd");
        return SIV_OK;
    });
}
