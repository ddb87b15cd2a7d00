// Dropout whose mask is never stored (fp32, bf16, fp16): out = [residual +] keep * act(x) / (1 - p).
// Element i of a call is component i % 4 of Philox(i / 4, stream id, seed): forward and backward draw it again instead
// of writing and reading a mask.
#include "elem_types.h"

namespace siv {

// 256 threads take a tile of 256 packs of 16 bytes at a time, one each.  The tile starts at a multiple of 2^8 Philox
// calls, so the upper counter word, like stream id and key, is the same for the whole block: a tenth of the products
// of the generator's first two rounds stay on the scalar unit.
template <typename T, bool AL, bool RES, bool BWD>
__global__ __launch_bounds__(256) void dropout_k(const T* __restrict__ in, const T* __restrict__ other, Drop d,
                                                 float slope, T* __restrict__ out, long n) {
    constexpr int N = Pack<T>::N;
    const uint64_t sid = drop_sid(d);
    const long tiles = (n + 256 * N - 1) / (256 * N);
    for (long t = blockIdx.x; t < tiles; t += gridDim.x) {
        const long i = t * (256 * N) + threadIdx.x * N, have = n - i;
        const bool whole = have >= N;
        const Pack<T> p = whole ? load_pack<AL>(in + i, N) : load_pack<false>(in + i, have);
        Pack<T> q;
        if (other) q = whole ? load_pack<AL>(other + i, N) : load_pack<false>(other + i, have);
        float v[N];
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = BWD ? (float)p.e[j] : leaky((float)p.e[j], slope);
        if (d.mode) {
            uint32_t w[N];
            if (d.mode == 1) {
                const uint64_t q0 = (uint64_t)t * (256 * N / 4);
#pragma unroll
                for (int k = 0; k < N / 4; ++k) {
                    const u4 r = philox4x32_10((q0 & ~0xffffffffull) | ((uint32_t)q0 + threadIdx.x * (N / 4) + k), sid, d.seed);
                    w[4 * k] = r.x;
                    w[4 * k + 1] = r.y;
                    w[4 * k + 2] = r.z;
                    w[4 * k + 3] = r.w;
                }
            } else {
                stored_words<N>(d, i, have, w);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = w[j] >= d.least ? v[j] * d.scale : 0.f;
        }
        Pack<T> o;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (BWD && other) v[j] *= leaky_grad((float)q.e[j], slope);
            if (RES) v[j] = (float)q.e[j] + v[j];
            o.e[j] = (T)v[j];
        }
        if (whole) store_pack<AL>(out + i, N, o);
        else store_pack<false>(out + i, have, o);
    }
}

// in / other: x and the residual (forward), dout and x (backward)
template <bool BWD>
static int dropout(const char* what, const void* in, const void* other, const Drop& d, float slope, void* out, int type,
                   long n, hipStream_t st) {
    const bool al = aligned16(in) && aligned16(other) && aligned16(out);
    return with_type(type, [&](auto* t) {
        typedef typename std::remove_reference<decltype(*t)>::type T;
        const long tiles = cdiv(n, 256 * Pack<T>::N);
        const unsigned g = (unsigned)(tiles < 4096 ? tiles : 4096);
        const T *a = (const T*)in, *b = (const T*)other;
        if (al && (BWD || !b)) dropout_k<T, true, false, BWD><<<g, 256, 0, st>>>(a, b, d, slope, (T*)out, n);
        else if (al) dropout_k<T, true, !BWD, BWD><<<g, 256, 0, st>>>(a, b, d, slope, (T*)out, n);
        else if (BWD || !b) dropout_k<T, false, false, BWD><<<g, 256, 0, st>>>(a, b, d, slope, (T*)out, n);
        else dropout_k<T, false, !BWD, BWD><<<g, 256, 0, st>>>(a, b, d, slope, (T*)out, n);
        SIV_CHECK_LAUNCH(what);
        return SIV_OK;
    });
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
    return dropout<false>("dropout_fwd", x, residual, make_drop(keep, seed, stream_id, epoch, p), slope, out, type, n,
                          (hipStream_t)stream);
}
extern "C" int siv_dropout_bwd(const void* dout, const void* x, const uint8_t* keep, uint64_t seed,
                               uint64_t stream_id, const uint64_t* epoch, float p, float slope, void* dx, int type,
                               long n, siv_stream_t stream) {
    SIV_CHECK_ARG(dout && dx && n > 0, "dropout_bwd: bad argument");
    SIV_CHECK_ARG(x || slope == 1.f, "dropout_bwd: the activation's backward needs x");
    SIV_CHECK_DROP("dropout_bwd");
    return dropout<true>("dropout_bwd", dout, slope == 1.f ? nullptr : x, make_drop(keep, seed, stream_id, epoch, p),
                         slope, dx, type, n, (hipStream_t)stream);
}
