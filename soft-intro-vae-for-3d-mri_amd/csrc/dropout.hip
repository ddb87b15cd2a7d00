// Dropout whose mask is never stored (fp32, bf16, fp16): out = [residual +] keep * act(x) / (1 - p).
// Element i of a call is component i % 4 of Philox(i / 4, stream id, seed): forward and backward draw it again instead
// of writing and reading a mask.  Bytes: one tensor read and one written (two read onto a residual).  Arithmetic: per
// four elements 18 products of 32 x 32 bits and 18 three-way xors; with 16-bit elements that takes about as long as
// the traffic.  315 M elements of bf16: 214-234 us = 5.4-5.9 TB/s (a device copy: 278 us); 78.6 M of fp32: 108 us = 5.8.
#include "elem_types.h"

namespace siv {

// What a call does beyond the product with the mask; OTHER is the residual (forward) or x (backward of an activation).
// (ACT_RES: siv_dropout_fwd and the backend's dropout_fwd with a slope and a residual; siv.ops calls one or the other.)
enum What { PLAIN, ACT, RES, ACT_RES, BWD_ACT };

// A block takes a tile of 256 x P packs of 16 bytes, P to a thread, all requested before the first is worked on.  A tile
// starts at a multiple of 2^8 Philox calls and holds fewer than 2^12, so the upper counter word, like stream id and key,
// is the same for the whole block: a tenth of the generator's products stay on the scalar unit.
template <typename T, int P, bool AL, int WHAT>
__global__ __launch_bounds__(256) void dropout_k(const T* __restrict__ in, const T* __restrict__ other, Drop d,
                                                 float slope, T* __restrict__ out, long n) {
    constexpr int N = Pack<T>::N;
    constexpr bool OTHER = WHAT == RES || WHAT == ACT_RES || WHAT == BWD_ACT;
    const uint64_t sid = drop_sid(d);
    const long tiles = (n + 256 * P * N - 1) / (256 * P * N);
    for (long t = blockIdx.x; t < tiles; t += gridDim.x) {
        const long i0 = t * (256 * P * N) + threadIdx.x * N;
        Pack<T> p[P], q[P];
#pragma unroll
        for (int k = 0; k < P; ++k) {
            const long i = i0 + k * 256 * N, have = n - i;
            p[k] = have >= N ? load_pack<AL>(in + i, N) : load_pack<false>(in + i, have);
            if (OTHER) q[k] = have >= N ? load_pack<AL>(other + i, N) : load_pack<false>(other + i, have);
        }
#pragma unroll
        for (int k = 0; k < P; ++k) {
            const long i = i0 + k * 256 * N, have = n - i;
            float v[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[j] = (float)p[k].e[j];
                if (WHAT == ACT || WHAT == ACT_RES) v[j] = leaky(v[j], slope);
            }
            if (d.mode) {
                uint32_t w[N];
                if (d.mode == 1) {
                    const uint64_t q0 = (uint64_t)t * (256 * P * N / 4);
#pragma unroll
                    for (int c = 0; c < N / 4; ++c) {
                        const u4 r = philox4x32_10(
                            (q0 & ~0xffffffffull) | ((uint32_t)q0 + (k * 256 + threadIdx.x) * (N / 4) + c), sid, d.seed);
                        w[4 * c] = r.x;
                        w[4 * c + 1] = r.y;
                        w[4 * c + 2] = r.z;
                        w[4 * c + 3] = r.w;
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
                if (WHAT == BWD_ACT) v[j] *= leaky_grad((float)q[k].e[j], slope);
                else if (OTHER) v[j] = (float)q[k].e[j] + v[j];
                o.e[j] = (T)v[j];
            }
            if (have >= N) store_pack<AL>(out + i, N, o);
            else store_pack<false>(out + i, have, o);
        }
    }
}

template <typename T, int P, bool AL>
static void dropout_launch(int what, const T* in, const T* other, const Drop& d, float slope, T* out, long n, long cap,
                           hipStream_t st) {
    constexpr int PO = P < 2 ? P : 2;          // packs in flight of two operands
    const bool two = what == RES || what == ACT_RES || what == BWD_ACT;
    const long tiles = cdiv(n, 256L * (two ? PO : P) * Pack<T>::N);
    const unsigned g = (unsigned)(tiles < cap ? tiles : cap);
    switch (what) {
        case PLAIN: dropout_k<T, P, AL, PLAIN><<<g, 256, 0, st>>>(in, other, d, slope, out, n); break;
        case ACT: dropout_k<T, P, AL, ACT><<<g, 256, 0, st>>>(in, other, d, slope, out, n); break;
        case RES: dropout_k<T, PO, AL, RES><<<g, 256, 0, st>>>(in, other, d, slope, out, n); break;
        case ACT_RES: dropout_k<T, PO, AL, ACT_RES><<<g, 256, 0, st>>>(in, other, d, slope, out, n); break;
        default: dropout_k<T, PO, AL, BWD_ACT><<<g, 256, 0, st>>>(in, other, d, slope, out, n); break;
    }
}
// Packs per thread and grid.  fp32 is bound by HBM: one pack a thread and a block per tile (78.6 M elements: 107 us =
// 5.9 TB/s; a grid of 4096 that walks the tensor 118, two packs 110).  Of 16-bit types a pack is two Philox calls, whose
// arithmetic is as long as their traffic: several packs a thread.  A call whose operands fit the Infinity Cache (256 MB)
// runs two packs over a grid of 2048, a larger one a block per tile, with four packs where there is one operand.  Measured
// on both sides in turn (us, bf16; grid of 2048 | block per tile): one operand 16.8 M elements 11.8 | 13.6, 50 M 32.5 | 34.3,
// 67 M (268 MB) 42.6 | 43.7, 101 M 74.3 | 70.3, 315 M 245 | 226; onto a residual 33.6 M (201 MB) 35.1 | 34.6, 50 M (302 MB)
// 62.9 | 54.8, 101 M 129 | 105, 315 M 410 | 323.
constexpr long BLOCKS_MAX = 1L << 20, CACHE = 256L << 20;
template <typename T, bool AL>
static void dropout_size(int what, const T* in, const T* other, const Drop& d, float slope, T* out, long n,
                         hipStream_t st) {
    const long bytes = n * (other ? 3 : 2) * (long)sizeof(T);
    if constexpr (sizeof(T) == 4) dropout_launch<T, 1, AL>(what, in, other, d, slope, out, n, BLOCKS_MAX, st);
    else if (bytes > CACHE) dropout_launch<T, 4, AL>(what, in, other, d, slope, out, n, BLOCKS_MAX, st);
    else dropout_launch<T, 2, AL>(what, in, other, d, slope, out, n, 2048, st);
}
static int dropout(const char* name, int what, const void* in, const void* other, const Drop& d, float slope, void* out,
                   int type, long n, hipStream_t st) {
    const bool al = aligned16(in) && aligned16(other) && aligned16(out);
    return with_type(type, [&](auto* t) {
        typedef typename std::remove_reference<decltype(*t)>::type T;
        if (al) dropout_size<T, true>(what, (const T*)in, (const T*)other, d, slope, (T*)out, n, st);
        else dropout_size<T, false>(what, (const T*)in, (const T*)other, d, slope, (T*)out, n, st);
        SIV_CHECK_LAUNCH(name);
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
    return dropout("dropout_fwd", slope == 1.f ? (residual ? RES : PLAIN) : (residual ? ACT_RES : ACT), x, residual,
                   make_drop(keep, seed, stream_id, epoch, p), slope, out, type, n, (hipStream_t)stream);
}
extern "C" int siv_dropout_bwd(const void* dout, const void* x, const uint8_t* keep, uint64_t seed,
                               uint64_t stream_id, const uint64_t* epoch, float p, float slope, void* dx, int type,
                               long n, siv_stream_t stream) {
    SIV_CHECK_ARG(dout && dx && n > 0, "dropout_bwd: bad argument");
    SIV_CHECK_ARG(x || slope == 1.f, "dropout_bwd: the activation's backward needs x");
    SIV_CHECK_DROP("dropout_bwd");
    return dropout("dropout_bwd", slope == 1.f ? PLAIN : BWD_ACT, dout, slope == 1.f ? nullptr : x,
                   make_drop(keep, seed, stream_id, epoch, p), slope, dx, type, n, (hipStream_t)stream);
}
