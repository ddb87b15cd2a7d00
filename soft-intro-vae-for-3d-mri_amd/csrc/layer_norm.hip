// Layer normalisation over the elements of a row, alone or behind residual + dropout, forward and backward
// (fp32, bf16, fp16; arithmetic fp32).
//   mean = sum x / C, var = sum (x - mean)^2 / C, r = 1 / sqrt(var + eps), h = (x - mean) r, y = h w + b
//   g = dy w;  dx = r (g - sum g / C - h sum(g h) / C);  dw = sum_rows dy h;  db = sum_rows dy
// The backward pass forms the statistics again from the row it reads anyway, so forward leaves nothing behind.
#include "elem_types.h"

namespace siv {

struct NormArgs {
    const void* x;          // [rows] at ldx: the input, or (backward of the residual form) the sum
    const void* res;        // [rows][C] residual or NULL
    const void* dy;         // [rows] at lddy
    const void* ds;         // [rows][C] gradient of the sum or NULL
    const void* weight;     // [C] or NULL
    const void* bias;
    void* s;                // [rows][C] the sum
    void* y;
    void* dx;               // gradient of x
    void* dres;             // gradient of residual
    long rows, C, ldx, lddy;
    float eps;
    int wf32;               // weight / bias are fp32 (else the activations' type)
};

template <typename T>
__device__ __forceinline__ bool drop_keeps(const Drop& d, uint64_t sid, long i) {
    if (d.mode == 0) return true;
    if (d.mode == 2) return d.keep[i] != 0;
    const u4 r = philox4x32_10((uint64_t)(i >> 2), sid, d.seed);
    const int j = (int)(i & 3);
    return ((j == 0 ? r.x : j == 1 ? r.y : j == 2 ? r.z : r.w) >> 8) >= d.thresh;
}

// One block per row.  RES: x is residual + dropout(x), written to s first.
template <typename T, bool RES>
__global__ __launch_bounds__(256) void ln_fwd_k(NormArgs a, Drop d) {
    __shared__ float sh[4];
    const uint64_t sid = drop_sid(d);
    const float invC = 1.0f / (float)a.C;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = (const T*)a.x + row * a.ldx;
        T* s = (T*)a.s + row * a.C;
        if (RES)
            for (long c = threadIdx.x; c < a.C; c += 256) {
                const long i = row * a.C + c;
                float v = (float)x[c];
                if (d.mode) v = drop_keeps<T>(d, sid, i) ? v * d.scale : 0.f;
                s[c] = (T)((float)((const T*)a.res)[i] + v);
            }
        const T* src = RES ? (const T*)s : x;
        float sum = 0.f;
        for (long c = threadIdx.x; c < a.C; c += 256) sum += (float)src[c];
        const float m0 = block_sum_256(sum, sh) * invC;
        float s1 = 0.f, s2 = 0.f;
        for (long c = threadIdx.x; c < a.C; c += 256) {
            const float t = (float)src[c] - m0;
            s1 += t;
            s2 += t * t;
        }
        const float delta = block_sum_256(s1, sh) * invC;
        const float var = fmaxf(block_sum_256(s2, sh) * invC - delta * delta, 0.f);
        const float r = rsqrtf(var + a.eps);
        for (long c = threadIdx.x; c < a.C; c += 256) {
            float h = (((float)src[c] - m0) - delta) * r;
            if (a.weight) h *= ld_param<T>(a.weight, a.wf32, c);
            if (a.bias) h += ld_param<T>(a.bias, a.wf32, c);
            ((T*)a.y)[row * a.C + c] = (T)h;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_k(NormArgs a, Drop d, float* __restrict__ stats) {
    __shared__ float sh[4];
    const uint64_t sid = drop_sid(d);
    const float invC = 1.0f / (float)a.C;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = (const T*)a.x + row * a.ldx;
        const T* dy = (const T*)a.dy + row * a.lddy;
        float sum = 0.f;
        for (long c = threadIdx.x; c < a.C; c += 256) sum += (float)x[c];
        const float m0 = block_sum_256(sum, sh) * invC;
        float s1 = 0.f, s2 = 0.f, g1 = 0.f, g2 = 0.f;
        for (long c = threadIdx.x; c < a.C; c += 256) {
            const float t = (float)x[c] - m0;
            const float g = (float)dy[c] * (a.weight ? ld_param<T>(a.weight, a.wf32, c) : 1.f);
            s1 += t;
            s2 += t * t;
            g1 += g;
            g2 += g * t;
        }
        const float delta = block_sum_256(s1, sh) * invC;
        const float var = fmaxf(block_sum_256(s2, sh) * invC - delta * delta, 0.f);
        const float r = rsqrtf(var + a.eps);
        const float gs = block_sum_256(g1, sh);
        const float c1 = gs * invC;
        const float c2 = (block_sum_256(g2, sh) - delta * gs) * r * invC;
        if (threadIdx.x == 0) {
            stats[3 * row] = m0;             // the mean is m0 + delta; their sum in one float would lose delta where
            stats[3 * row + 1] = delta;      // the row sits far off zero
            stats[3 * row + 2] = r;
        }
        for (long c = threadIdx.x; c < a.C; c += 256) {
            const long i = row * a.C + c;
            const float h = (((float)x[c] - m0) - delta) * r;
            const float g = (float)dy[c] * (a.weight ? ld_param<T>(a.weight, a.wf32, c) : 1.f);
            float v = r * (g - c1 - h * c2);
            if (a.ds) v += (float)((const T*)a.ds)[i];
            if (a.dres) ((T*)a.dres)[i] = (T)v;
            if (a.dx) {
                if (d.mode) v = drop_keeps<T>(d, sid, i) ? v * d.scale : 0.f;
                ((T*)a.dx)[i] = (T)v;
            }
        }
    }
}
// dw[c] = sum_rows dy h, db[c] = sum_rows dy in two steps, both in a fixed order: block (64 columns, part) sums its
// share of the rows, its four waves taking every fourth; then the parts are added.
template <typename T>
__global__ __launch_bounds__(256) void ln_param_grad_k(NormArgs a, const float* __restrict__ stats,
                                                       float* __restrict__ part) {
    __shared__ float sh[2][4][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const long c = (long)blockIdx.x * 64 + lane;
    const long lo = a.rows * blockIdx.y / gridDim.y, hi = a.rows * (blockIdx.y + 1) / gridDim.y;
    float gw = 0.f, gb = 0.f;
    if (c < a.C)
        for (long row = lo + wv; row < hi; row += 4) {
            const float v = (float)((const T*)a.dy)[row * a.lddy + c];
            const float xc = ((float)((const T*)a.x)[row * a.ldx + c] - stats[3 * row]) - stats[3 * row + 1];
            gw += v * (xc * stats[3 * row + 2]);
            gb += v;
        }
    sh[0][wv][lane] = gw;
    sh[1][wv][lane] = gb;
    __syncthreads();
    if (wv < 2 && c < a.C)
        part[((long)blockIdx.y * 2 + wv) * a.C + c] =
            (sh[wv][0][lane] + sh[wv][1][lane]) + (sh[wv][2][lane] + sh[wv][3][lane]);
}
template <typename T>
__global__ __launch_bounds__(256) void ln_param_sum_k(const float* __restrict__ part, int parts, long C, void* dw,
                                                      void* db, int wf32, int accumulate) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= 2 * C) return;
    void* out = i < C ? dw : db;
    const long c = i < C ? i : i - C;
    if (!out) return;
    float v = 0.f;
    for (int k = 0; k < parts; ++k) v += part[(long)k * 2 * C + i];
    if (wf32) ((float*)out)[c] = accumulate ? ((float*)out)[c] + v : v;
    else ((T*)out)[c] = (T)(accumulate ? (float)((T*)out)[c] + v : v);
}

static int ln_check(const char* what, const NormArgs& a, int type, int wtype) {
    SIV_CHECK_ARG(a.rows > 0 && a.C > 0 && a.C < (1L << 31) && a.rows < (1L << 40), "%s: rows and C must be positive (C < 2^31)", what);
    SIV_CHECK_ARG(a.ldx >= a.C && a.lddy >= a.C, "%s: a row stride is shorter than the row", what);
    SIV_CHECK_ARG(known_type(type), "%s: unknown element type", what);
    SIV_CHECK_ARG(wtype == SIV_F32 || wtype == type, "%s: weights must be fp32 or of the activations' type", what);
    SIV_CHECK_ARG(a.eps >= 0.f, "%s: eps must not be negative", what);
    return SIV_OK;
}
static long ln_parts(long rows) { return rows > 256 * 64 ? 256 : cdiv(rows, 64); }
static size_t ln_ws_bytes(long rows, long C, int, int backward) {
    return backward ? align256((size_t)rows * 12) + (size_t)ln_parts(rows) * 2 * C * 4 : 0;
}

static int ln_fwd(const char* what, const NormArgs& a, const Drop& d, bool res, int type, void*, size_t, hipStream_t st) {
    return with_type(type, [&](auto* t) {
        typedef typename std::remove_reference<decltype(*t)>::type T;
        const unsigned g = (unsigned)(a.rows > 8192 ? 8192 : a.rows);
        if (res) ln_fwd_k<T, true><<<g, 256, 0, st>>>(a, d);
        else ln_fwd_k<T, false><<<g, 256, 0, st>>>(a, d);
        SIV_CHECK_LAUNCH(what);
        return SIV_OK;
    });
}
static int ln_bwd(const char* what, const NormArgs& a, const Drop& d, void* dw, void* db, int accumulate, int type,
                  void* ws, size_t ws_bytes, hipStream_t st) {
    SIV_CHECK_ARG(ws || ws_bytes == 0, "%s: null workspace", what);
    SIV_CHECK_WS(ln_ws_bytes(a.rows, a.C, type, 1), ws_bytes, what);
    return with_type(type, [&](auto* t) {
        typedef typename std::remove_reference<decltype(*t)>::type T;
        const unsigned g = (unsigned)(a.rows > 8192 ? 8192 : a.rows);
        ln_bwd_k<T><<<g, 256, 0, st>>>(a, d, (float*)ws);
        SIV_CHECK_LAUNCH(what);
        if (dw || db) {
            float* part = (float*)((char*)ws + align256((size_t)a.rows * 12));
            const int parts = (int)ln_parts(a.rows);
            ln_param_grad_k<T><<<dim3((unsigned)cdiv(a.C, 64), parts), 256, 0, st>>>(a, (const float*)ws, part);
            SIV_CHECK_LAUNCH(what);
            ln_param_sum_k<T><<<(unsigned)cdiv(2 * a.C, 256), 256, 0, st>>>(part, parts, a.C, dw, db, a.wf32, accumulate);
            SIV_CHECK_LAUNCH(what);
        }
        return SIV_OK;
    });
}

}  // namespace siv

using namespace siv;

extern "C" int siv_layer_norm_workspace(long rows, long C, int type, int backward, size_t* bytes) {
    SIV_CHECK_ARG(bytes && rows > 0 && C > 0 && known_type(type), "layer_norm_workspace: bad argument");
    *bytes = ln_ws_bytes(rows, C, type, backward);
    return SIV_OK;
}
extern "C" int siv_layer_norm_fwd(const void* x, long ldx, const void* weight, const void* bias, int wtype, float eps,
                                  void* y, int type, long rows, long C, void* ws, size_t ws_bytes,
                                  siv_stream_t stream) {
    SIV_CHECK_ARG(x && y, "layer_norm_fwd: null pointer");
    NormArgs a = {};
    a.x = x; a.weight = weight; a.bias = bias; a.y = y;
    a.rows = rows; a.C = C; a.ldx = ldx; a.lddy = C; a.eps = eps; a.wf32 = wtype == SIV_F32;
    if (int rc = ln_check("layer_norm_fwd", a, type, wtype)) return rc;
    return ln_fwd("layer_norm_fwd", a, make_drop(nullptr, 0, 0, nullptr, 0.f), false, type, ws, ws_bytes,
                  (hipStream_t)stream);
}
extern "C" int siv_layer_norm_bwd(const void* dy, long lddy, const void* x, long ldx, const void* weight, int wtype,
                                  float eps, void* dx, void* dweight, void* dbias, int accumulate, int type, long rows,
                                  long C, void* ws, size_t ws_bytes, siv_stream_t stream) {
    SIV_CHECK_ARG(dy && x && (dx || dweight || dbias), "layer_norm_bwd: null pointer");
    NormArgs a = {};
    a.x = x; a.dy = dy; a.weight = weight; a.dx = dx;
    a.rows = rows; a.C = C; a.ldx = ldx; a.lddy = lddy; a.eps = eps; a.wf32 = wtype == SIV_F32;
    if (int rc = ln_check("layer_norm_bwd", a, type, wtype)) return rc;
    return ln_bwd("layer_norm_bwd", a, make_drop(nullptr, 0, 0, nullptr, 0.f), dweight, dbias, accumulate, type, ws,
                  ws_bytes, (hipStream_t)stream);
}
extern "C" int siv_add_layer_norm_fwd(const void* x, const void* residual, const uint8_t* keep, uint64_t seed,
                                      uint64_t stream_id, const uint64_t* epoch, float p, const void* weight,
                                      const void* bias, int wtype, float eps, void* s, void* y, int type, long rows,
                                      long C, void* ws, size_t ws_bytes, siv_stream_t stream) {
    SIV_CHECK_ARG(x && residual && s && y, "add_layer_norm_fwd: null pointer");
    SIV_CHECK_ARG(p >= 0.f && p < 1.f, "add_layer_norm_fwd: dropout p out of range");
    NormArgs a = {};
    a.x = x; a.res = residual; a.weight = weight; a.bias = bias; a.s = s; a.y = y;
    a.rows = rows; a.C = C; a.ldx = C; a.lddy = C; a.eps = eps; a.wf32 = wtype == SIV_F32;
    if (int rc = ln_check("add_layer_norm_fwd", a, type, wtype)) return rc;
    return ln_fwd("add_layer_norm_fwd", a, make_drop(keep, seed, stream_id, epoch, p), true, type, ws, ws_bytes,
                  (hipStream_t)stream);
}
extern "C" int siv_add_layer_norm_bwd(const void* dy, const void* ds, const void* s, const uint8_t* keep, uint64_t seed,
                                      uint64_t stream_id, const uint64_t* epoch, float p, const void* weight, int wtype,
                                      float eps, void* dx, void* dresidual, void* dweight, void* dbias, int accumulate,
                                      int type, long rows, long C, void* ws, size_t ws_bytes, siv_stream_t stream) {
    SIV_CHECK_ARG(dy && s && (dx || dresidual || dweight || dbias), "add_layer_norm_bwd: null pointer");
    SIV_CHECK_ARG(p >= 0.f && p < 1.f, "add_layer_norm_bwd: dropout p out of range");
    NormArgs a = {};
    a.x = s; a.dy = dy; a.ds = ds; a.weight = weight; a.dx = dx; a.dres = dresidual;
    a.rows = rows; a.C = C; a.ldx = C; a.lddy = C; a.eps = eps; a.wf32 = wtype == SIV_F32;
    if (int rc = ln_check("add_layer_norm_bwd", a, type, wtype)) return rc;
    return ln_bwd("add_layer_norm_bwd", a, make_drop(keep, seed, stream_id, epoch, p), dweight, dbias, accumulate, type,
                  ws, ws_bytes, (hipStream_t)stream);
}
