// Layer normalisation over the elements of a row, alone or behind residual + dropout, forward and backward
// (fp32, bf16, fp16; arithmetic fp32).
//   mean = sum x / C, var = sum (x - mean)^2 / C, r = 1 / sqrt(var + eps), h = (x - mean) r, y = h w + b
//   g = dy w;  dx = r (g - sum g / C - h sum(g h) / C);  dw = sum_rows dy h;  db = sum_rows dy
// The mean is summed twice: m0 = sum x / C, then d = x - m0, delta = sum d / C, var = sum d^2 / C - delta^2.  x - m0
// is exact or nearly so, and delta takes back the rounding of m0, so rows far off zero keep their deviations.
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
    void* dw;               // [C] gradients of the parameters, or NULL
    void* db;
    float* part;            // [blocks][2][C] their partial sums
    long rows, C, ldx, lddy;
    float eps;
    int wf32;               // weight / bias are fp32 (else the activations' type)
    int accumulate;
    int lg;                 // a row is spread over 2^lg lanes of a wave (wave form)
};

// ---- sums over a group of lanes ------------------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp_mov(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// sum over 2^lg neighbouring lanes (lg wave-uniform), the same bits in every lane: each step adds two values that are
// already equal within their halves, in either order
template <int N>
__device__ __forceinline__ void lanes_sum(float (&v)[N], int lg) {
#define SIV_STEP(n, expr)                                                       \
    if (lg >= n) {                                                              \
        _Pragma("unroll") for (int k = 0; k < N; ++k) { expr; }                 \
    }
    SIV_STEP(1, v[k] += dpp_mov<0xB1>(v[k]))       // quad_perm [1,0,3,2]
    SIV_STEP(2, v[k] += dpp_mov<0x4E>(v[k]))       // quad_perm [2,3,0,1]
    SIV_STEP(3, v[k] += dpp_mov<0x141>(v[k]))      // mirror of 8 lanes
    SIV_STEP(4, v[k] += dpp_mov<0x140>(v[k]))      // mirror of 16 lanes
    SIV_STEP(5, const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[k]), __float_as_uint(v[k]), false, false);
             v[k] = __uint_as_float(t[0]) + __uint_as_float(t[1]))
    SIV_STEP(6, const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[k]), __float_as_uint(v[k]), false, false);
             v[k] = __uint_as_float(t[0]) + __uint_as_float(t[1]))
#undef SIV_STEP
}
// Sums over the lanes that share a row: part of a wave, or (BLK) a block of 256.  Two LDS buffers in turn: the barrier
// of one sum also separates the readers of the sum before it from the writers of the next.
template <bool BLK>
struct RowSum {
    float (*sh)[4][4];
    int lg, turn;
    template <int N>
    __device__ __forceinline__ void operator()(float (&v)[N]) {
        if (!BLK) {
            lanes_sum(v, lg);
            return;
        }
        lanes_sum(v, 6);
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) sh[turn][w][k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = (sh[turn][0][k] + sh[turn][1][k]) + (sh[turn][2][k] + sh[turn][3][k]);
        turn ^= 1;
    }
};

// N consecutive parameters from column c on (have of them exist; the rest 0)
template <bool AL, typename T, int N>
__device__ __forceinline__ void load_params(const void* w, int f32, long c, long have, float dflt, float (&out)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = dflt;
    if (!w) return;
    if (f32) {
        const float* p = (const float*)w + c;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (AL ? have > 0 : j < have) out[j] = p[j];
    } else {
        const T* p = (const T*)w + c;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (AL ? have > 0 : j < have) out[j] = (float)p[j];
    }
}
template <typename T>
__device__ __forceinline__ void put_param(void* out, int f32, long c, float v, int accumulate) {
    if (f32) ((float*)out)[c] = accumulate ? ((float*)out)[c] + v : v;
    else ((T*)out)[c] = (T)(accumulate ? (float)((T*)out)[c] + v : v);
}

// residual + dropout(x) of one pack, as it is held
template <typename T, bool AL>
__device__ __forceinline__ Pack<T> add_drop(const Pack<T>& x, const Pack<T>& res, const Drop& d, uint64_t sid, long i,
                                            long have) {
    constexpr int N = Pack<T>::N;
    Pack<T> s;
    if (d.mode == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) s.e[j] = (T)((float)res.e[j] + (float)x.e[j]);
        return s;
    }
    uint32_t w[N];
    drop_words<N, AL>(d, sid, i, have, w);
#pragma unroll
    for (int j = 0; j < N; ++j) s.e[j] = (T)((float)res.e[j] + (w[j] >= d.least ? (float)x.e[j] * d.scale : 0.f));
    return s;
}

// ---- rows held in registers -----------------------------------------------------------------------------------------
// A row is spread over 2^lg lanes of a wave, 64 >> lg rows to a wave (wave form), or over the 256 threads of a block
// (BLK); a lane holds NV packs of 16 bytes.  One pass over the data; blocks walk the rows in strides of the grid, so
// that weights and the parameters' gradients stay in registers.
template <typename T, int NV, bool BLK, bool AL, bool RES>
__global__ __launch_bounds__(256) void ln_fwd_k(NormArgs a, Drop d) {
    constexpr int N = Pack<T>::N;
    __shared__ float sh[2][4][4];
    RowSum<BLK> row_sum{sh, a.lg, 0};
    const int lane = threadIdx.x & 63;
    const int G = BLK ? 256 : 1 << a.lg;
    const int sub = BLK ? threadIdx.x : lane & (G - 1);
    const long per = BLK ? 1 : 256 >> a.lg;                           // rows of one block step
    const long first = BLK ? 0 : threadIdx.x >> a.lg;
    const uint64_t sid = RES ? drop_sid(d) : 0;
    const float invC = 1.0f / (float)a.C;
    long have[NV];
    float w[NV][N], b[NV][N];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const long c = (long)(k * G + sub) * N;
        have[k] = a.C - c;
        load_params<AL, T>(a.weight, a.wf32, c, have[k], 1.f, w[k]);
        load_params<AL, T>(a.bias, a.wf32, c, have[k], 0.f, b[k]);
    }
    for (long row0 = (long)blockIdx.x * per; row0 < a.rows; row0 += (long)gridDim.x * per) {
        const long row = row0 + first;
        const bool ok = row < a.rows;
        float v[NV][N];
        float s1[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const long c = (long)(k * G + sub) * N;
            const long hv = ok ? have[k] : 0;
            Pack<T> p = load_pack<AL>((const T*)a.x + row * a.ldx + c, hv);
            if (RES) {
                const long i = row * a.C + c;
                const Pack<T> q = load_pack<AL>((const T*)a.res + i, hv);
                if (hv > 0) p = add_drop<T, AL>(p, q, d, sid, i, hv);
                store_pack<AL>((T*)a.s + i, hv, p);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[k][j] = (AL || j < hv) ? (float)p.e[j] : 0.f;
                s1[0] += v[k][j];
            }
        }
        row_sum(s1);
        const float m0 = s1[0] * invC;
        float m[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[k][j] = (AL ? have[k] > 0 : j < have[k]) ? v[k][j] - m0 : 0.f;
                m[0] += v[k][j];
                m[1] += v[k][j] * v[k][j];
            }
        row_sum(m);
        const float delta = m[0] * invC;
        const float r = rsqrtf(fmaxf(m[1] * invC - delta * delta, 0.f) + a.eps);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            Pack<T> p;
#pragma unroll
            for (int j = 0; j < N; ++j) p.e[j] = (T)((v[k][j] - delta) * r * w[k][j] + b[k][j]);
            store_pack<AL>((T*)a.y + row * a.C + (long)(k * G + sub) * N, ok ? have[k] : 0, p);
        }
    }
}

// The same rows backward.  Each lane sums dy h and dy of its columns over the rows it sees; a block's sums go to
// a.part, or straight to the results where there is one block.
template <typename T, int NV, bool BLK, bool AL>
__global__ __launch_bounds__(256) void ln_bwd_k(NormArgs a, Drop d) {
    constexpr int N = Pack<T>::N;
    __shared__ float sh[2][4][4];
    __shared__ float fold[BLK ? 1 : 4 * 64 * NV * N];
    RowSum<BLK> row_sum{sh, a.lg, 0};
    const int lane = threadIdx.x & 63;
    const int G = BLK ? 256 : 1 << a.lg;
    const int sub = BLK ? threadIdx.x : lane & (G - 1);
    const long per = BLK ? 1 : 256 >> a.lg;
    const long first = BLK ? 0 : threadIdx.x >> a.lg;
    const uint64_t sid = drop_sid(d);
    const float invC = 1.0f / (float)a.C;
    long have[NV];
    float w[NV][N], gw[NV][N], gb[NV][N];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const long c = (long)(k * G + sub) * N;
        have[k] = a.C - c;
        load_params<AL, T>(a.weight, a.wf32, c, have[k], 1.f, w[k]);
#pragma unroll
        for (int j = 0; j < N; ++j) gw[k][j] = gb[k][j] = 0.f;
    }
    for (long row0 = (long)blockIdx.x * per; row0 < a.rows; row0 += (long)gridDim.x * per) {
        const long row = row0 + first;
        const bool ok = row < a.rows;
        float v[NV][N];
        Pack<T> gy[NV], ds[NV];
        float s1[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const long c = (long)(k * G + sub) * N;
            const long hv = ok ? have[k] : 0;
            const Pack<T> p = load_pack<AL>((const T*)a.x + row * a.ldx + c, hv);
            gy[k] = load_pack<AL>((const T*)a.dy + row * a.lddy + c, hv);
            if (a.ds) ds[k] = load_pack<AL>((const T*)a.ds + row * a.C + c, hv);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[k][j] = (float)p.e[j];
                s1[0] += v[k][j];
            }
        }
        row_sum(s1);
        const float m0 = s1[0] * invC;
        float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[k][j] = (AL ? have[k] > 0 : j < have[k]) ? v[k][j] - m0 : 0.f;
                const float g = (float)gy[k].e[j] * w[k][j];
                m[0] += v[k][j];
                m[1] += v[k][j] * v[k][j];
                m[2] += g;
                m[3] += g * v[k][j];
            }
        row_sum(m);
        const float delta = m[0] * invC;
        float r = rsqrtf(fmaxf(m[1] * invC - delta * delta, 0.f) + a.eps);
        if (!ok) r = 0.f;                    // lanes without a row add nothing, whatever eps is
        const float c1 = m[2] * invC, c2 = (m[3] - delta * m[2]) * r * invC;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const long hv = ok ? have[k] : 0;
            const long i = row * a.C + (long)(k * G + sub) * N;
            float g[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float dy = (float)gy[k].e[j];
                const float h = (v[k][j] - delta) * r;
                gw[k][j] += dy * h;
                gb[k][j] += dy;
                g[j] = r * (dy * w[k][j] - c1 - h * c2);
            }
            if (a.ds)
#pragma unroll
                for (int j = 0; j < N; ++j) g[j] += (float)ds[k].e[j];
            Pack<T> p;
            if (a.dres) {
#pragma unroll
                for (int j = 0; j < N; ++j) p.e[j] = (T)g[j];
                store_pack<AL>((T*)a.dres + i, hv, p);
            }
            if (a.dx) {
                if (d.mode && hv > 0) {
                    uint32_t u[N];
                    drop_words<N, AL>(d, sid, i, hv, u);
#pragma unroll
                    for (int j = 0; j < N; ++j) g[j] = u[j] >= d.least ? g[j] * d.scale : 0.f;
                }
#pragma unroll
                for (int j = 0; j < N; ++j) p.e[j] = (T)g[j];
                store_pack<AL>((T*)a.dx + i, hv, p);
            }
        }
    }
    if (!a.dw && !a.db) return;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* out = a.part + ((long)blockIdx.x * 2 + which) * a.C;
        void* res = which ? a.db : a.dw;
        if (BLK) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const long c = (long)(k * G + sub) * N + j;
                    const float t = which ? gb[k][j] : gw[k][j];
                    if (c < a.C) {
                        if (gridDim.x > 1) out[c] = t;
                        else if (res) put_param<T>(res, a.wf32, c, t, a.accumulate);
                    }
                }
        } else {
            // rows of one wave that share columns, then the four waves
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    float t = which ? gb[k][j] : gw[k][j];
                    for (int o = G; o < 64; o <<= 1) t += __shfl_xor(t, o, 64);
                    if (lane < G) fold[((threadIdx.x >> 6) * NV + k) * 64 * N + lane * N + j] = t;
                }
            __syncthreads();
            for (long c = threadIdx.x; c < a.C; c += 256) {
                const int k = (int)(c / (G * N)), o = (int)(c - (long)k * G * N);
                const float t = (fold[(0 * NV + k) * 64 * N + o] + fold[(1 * NV + k) * 64 * N + o]) +
                                (fold[(2 * NV + k) * 64 * N + o] + fold[(3 * NV + k) * 64 * N + o]);
                if (gridDim.x > 1) out[c] = t;
                else if (res) put_param<T>(res, a.wf32, c, t, a.accumulate);
            }
            __syncthreads();
        }
    }
}

// ---- rows too long for registers: a row is cut into chunks ------------------------------------------------------------
// Two launches: statistics of every chunk (a block each, 256 threads x SPLIT_NV packs at a time), then blocks that join
// the chunks of a row and go over the data again.  What a chunk leaves: its mean (double: a float could not hold the
// mean of a row far off zero to within its deviations), M2 = sum (x - mean)^2, and backward G = sum g and
// H = sum g (x - mean), all about the chunk's own mean; joined about the row's mean,
//   M2 = sum M2_c + n_c (mean_c - mean)^2,   H = sum H_c + G_c (mean_c - mean).
constexpr int SPLIT_NV = 2;
constexpr int SPLIT_MAX = 256;            // chunks of a row; beyond, a chunk is several tiles
struct Chunk {
    double mean;
    float m2, g, h, pad;
};
struct SplitPlan {
    long tile, tiles, per, chunks;        // elements of a tile, tiles of a row, tiles of a chunk, chunks of a row
};
__host__ __device__ static inline SplitPlan split_plan(long C, int size) {
    SplitPlan s;
    s.tile = 256L * SPLIT_NV * (16 / size);
    s.tiles = (C + s.tile - 1) / s.tile;
    s.per = (s.tiles + SPLIT_MAX - 1) / SPLIT_MAX;
    s.chunks = (s.tiles + s.per - 1) / s.per;
    return s;
}

template <typename T, bool AL, bool RES, bool BWD>
__global__ __launch_bounds__(256) void ln_split_stats_k(NormArgs a, Drop d, Chunk* __restrict__ st) {
    constexpr int N = Pack<T>::N;
    __shared__ float sh[2][4][4];
    RowSum<true> row_sum{sh, 6, 0};
    const SplitPlan sp = split_plan(a.C, sizeof(T));
    const uint64_t sid = RES ? drop_sid(d) : 0;
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        double n = 0, mean = 0, m2 = 0, G = 0, H = 0;
        for (long t = blockIdx.x * sp.per; t < (blockIdx.x + 1) * sp.per && t < sp.tiles; ++t) {
            float v[SPLIT_NV][N], g[SPLIT_NV][N];
            float s1[1] = {0.f};
#pragma unroll
            for (int k = 0; k < SPLIT_NV; ++k) {
                const long c = t * sp.tile + (long)(k * 256 + threadIdx.x) * N;
                const long hv = a.C - c;
                Pack<T> p = load_pack<AL>((const T*)a.x + row * a.ldx + c, hv);
                if (RES) {
                    const long i = row * a.C + c;
                    const Pack<T> q = load_pack<AL>((const T*)a.res + i, hv);
                    if (hv > 0) p = add_drop<T, AL>(p, q, d, sid, i, hv);
                    store_pack<AL>((T*)a.s + i, hv, p);
                }
                if (BWD) {
                    const Pack<T> q = load_pack<AL>((const T*)a.dy + row * a.lddy + c, hv);
                    load_params<AL, T>(a.weight, a.wf32, c, hv, 1.f, g[k]);
#pragma unroll
                    for (int j = 0; j < N; ++j) g[k][j] *= (float)q.e[j];
                }
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    v[k][j] = (AL || j < hv) ? (float)p.e[j] : 0.f;
                    s1[0] += v[k][j];
                }
            }
            row_sum(s1);
            const long nt = a.C - t * sp.tile < sp.tile ? a.C - t * sp.tile : sp.tile;
            const float m0 = s1[0] / (float)nt;
            float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < SPLIT_NV; ++k)
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const long hv = a.C - (t * sp.tile + (long)(k * 256 + threadIdx.x) * N);
                    const float x = (AL ? hv > 0 : j < hv) ? v[k][j] - m0 : 0.f;
                    m[0] += x;
                    m[1] += x * x;
                    if (BWD) {
                        m[2] += g[k][j];
                        m[3] += g[k][j] * x;
                    }
                }
            row_sum(m);
            // this tile about its own mean, then joined to the tiles before it
            const float delta = m[0] / (float)nt;
            const double tm = (double)m0 + (double)delta;
            const double tm2 = fmaxf(m[1] - delta * m[0], 0.f), tg = m[2], th = m[3] - delta * m[2];
            const double all = n + (double)nt, e = tm - mean, step = e * ((double)nt / all);
            if (BWD) {
                H = (H - G * step) + (th + tg * (e - step));
                G += tg;
            }
            m2 += tm2 + e * step * n;
            mean += step;
            n = all;
        }
        if (threadIdx.x == 0) {
            Chunk c;
            c.mean = mean;
            c.m2 = (float)m2;
            c.g = (float)G;
            c.h = (float)H;
            c.pad = 0.f;
            st[row * sp.chunks + blockIdx.x] = c;
        }
    }
}
// Every wave joins all chunks of the row by itself: the same operations in the same order, no barrier.
struct RowStats {
    float hi, lo, r, c1, c2;              // mean = hi + lo
};
template <bool BWD>
__device__ __forceinline__ RowStats join_chunks(const Chunk* __restrict__ st, const SplitPlan& sp, long C, float eps) {
    const int lane = threadIdx.x & 63;
    const long whole = sp.per * sp.tile;
    double sum = 0;
    for (long k = lane; k < sp.chunks; k += 64) sum += st[k].mean * (double)(k + 1 < sp.chunks ? whole : C - k * whole);
    const double mean = wave_sum_d(sum) / (double)C;
    double m2 = 0, G = 0, H = 0;
    for (long k = lane; k < sp.chunks; k += 64) {
        const Chunk c = st[k];
        const double e = c.mean - mean;
        m2 += (double)c.m2 + e * e * (double)(k + 1 < sp.chunks ? whole : C - k * whole);
        if (BWD) {
            G += c.g;
            H += (double)c.h + (double)c.g * e;
        }
    }
    m2 = wave_sum_d(m2);
    RowStats s;
    s.hi = (float)mean;
    s.lo = (float)(mean - (double)s.hi);
    s.r = rsqrtf((float)(m2 / (double)C) + eps);
    if (BWD) {
        s.c1 = (float)(wave_sum_d(G) / (double)C);
        s.c2 = (float)(wave_sum_d(H) / (double)C) * s.r;
    }
    return s;
}
template <typename T, bool AL>
__global__ __launch_bounds__(256) void ln_split_fwd_k(NormArgs a, const Chunk* __restrict__ st) {
    constexpr int N = Pack<T>::N;
    const SplitPlan sp = split_plan(a.C, sizeof(T));
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const RowStats s = join_chunks<false>(st + row * sp.chunks, sp, a.C, a.eps);
#pragma unroll
        for (int k = 0; k < SPLIT_NV; ++k) {
            const long c = blockIdx.x * sp.tile + (long)(k * 256 + threadIdx.x) * N;
            const long hv = a.C - c;
            float w[N], b[N];
            load_params<AL, T>(a.weight, a.wf32, c, hv, 1.f, w);
            load_params<AL, T>(a.bias, a.wf32, c, hv, 0.f, b);
            const Pack<T> p = a.s ? load_pack<AL>((const T*)a.s + row * a.C + c, hv)
                                  : load_pack<AL>((const T*)a.x + row * a.ldx + c, hv);
            Pack<T> o;
#pragma unroll
            for (int j = 0; j < N; ++j) o.e[j] = (T)((((float)p.e[j] - s.hi) - s.lo) * s.r * w[j] + b[j]);
            store_pack<AL>((T*)a.y + row * a.C + c, hv, o);
        }
    }
}
// Backward: block (tile, part of the rows) keeps the parameter gradients of its columns in registers.
template <typename T, bool AL>
__global__ __launch_bounds__(256) void ln_split_bwd_k(NormArgs a, Drop d, const Chunk* __restrict__ st) {
    constexpr int N = Pack<T>::N;
    const SplitPlan sp = split_plan(a.C, sizeof(T));
    const uint64_t sid = drop_sid(d);
    float w[SPLIT_NV][N], gw[SPLIT_NV][N], gb[SPLIT_NV][N];
#pragma unroll
    for (int k = 0; k < SPLIT_NV; ++k) {
        const long c = blockIdx.x * sp.tile + (long)(k * 256 + threadIdx.x) * N;
        load_params<AL, T>(a.weight, a.wf32, c, a.C - c, 1.f, w[k]);
#pragma unroll
        for (int j = 0; j < N; ++j) gw[k][j] = gb[k][j] = 0.f;
    }
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const RowStats s = join_chunks<true>(st + row * sp.chunks, sp, a.C, a.eps);
#pragma unroll
        for (int k = 0; k < SPLIT_NV; ++k) {
            const long c = blockIdx.x * sp.tile + (long)(k * 256 + threadIdx.x) * N;
            const long hv = a.C - c, i = row * a.C + c;
            const Pack<T> p = load_pack<AL>((const T*)a.x + row * a.ldx + c, hv);
            const Pack<T> q = load_pack<AL>((const T*)a.dy + row * a.lddy + c, hv);
            float g[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float dy = (float)q.e[j];
                const float h = (((float)p.e[j] - s.hi) - s.lo) * s.r;
                gw[k][j] += dy * h;
                gb[k][j] += dy;
                g[j] = s.r * (dy * w[k][j] - s.c1 - h * s.c2);
            }
            if (a.ds) {
                const Pack<T> e = load_pack<AL>((const T*)a.ds + i, hv);
#pragma unroll
                for (int j = 0; j < N; ++j) g[j] += (float)e.e[j];
            }
            Pack<T> o;
            if (a.dres) {
#pragma unroll
                for (int j = 0; j < N; ++j) o.e[j] = (T)g[j];
                store_pack<AL>((T*)a.dres + i, hv, o);
            }
            if (a.dx) {
                if (d.mode && hv > 0) {
                    uint32_t u[N];
                    drop_words<N, AL>(d, sid, i, hv, u);
#pragma unroll
                    for (int j = 0; j < N; ++j) g[j] = u[j] >= d.least ? g[j] * d.scale : 0.f;
                }
#pragma unroll
                for (int j = 0; j < N; ++j) o.e[j] = (T)g[j];
                store_pack<AL>((T*)a.dx + i, hv, o);
            }
        }
    }
    if (!a.dw && !a.db) return;
#pragma unroll
    for (int k = 0; k < SPLIT_NV; ++k)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const long c = blockIdx.x * sp.tile + (long)(k * 256 + threadIdx.x) * N + j;
            if (c >= a.C) continue;
            if (gridDim.y > 1) {
                a.part[((long)blockIdx.y * 2 + 0) * a.C + c] = gw[k][j];
                a.part[((long)blockIdx.y * 2 + 1) * a.C + c] = gb[k][j];
            } else {
                if (a.dw) put_param<T>(a.dw, a.wf32, c, gw[k][j], a.accumulate);
                if (a.db) put_param<T>(a.db, a.wf32, c, gb[k][j], a.accumulate);
            }
        }
}

// the blocks' partial sums joined: 16 columns to a block, 64 threads down each, in a fixed order
template <typename T>
__global__ __launch_bounds__(1024) void ln_param_sum_k(const float* __restrict__ part, long parts, NormArgs a) {
    __shared__ float sh[64][17];
    const int col = threadIdx.x & 15, down = threadIdx.x >> 4;
    const long i = (long)blockIdx.x * 16 + col, C2 = 2 * a.C;
    float t = 0.f;
    if (i < C2)
        for (long k = down; k < parts; k += 64) t += part[k * C2 + i];
    sh[down][col] = t;
    for (int o = 32; o > 0; o >>= 1) {
        __syncthreads();
        if (down < o) sh[down][col] += sh[down + o][col];
    }
    if (down || i >= C2) return;
    void* out = i < a.C ? a.dw : a.db;
    if (out) put_param<T>(out, a.wf32, i < a.C ? i : i - a.C, sh[0][col], a.accumulate);
}

// ---- host -------------------------------------------------------------------------------------------------------------
// Which kernel: a function of the row length and the type alone, so that a row's result does not depend on what is
// computed beside it.
enum Form { WAVE1, WAVE2, BLOCK1, BLOCK2, BLOCK4, SPLIT };
static Form ln_form(long C, int type, int* lg) {
    const long n = 16 / type_size(type), packs = cdiv(C, n);
    *lg = 0;
    if (packs <= 64) {
        while ((1L << *lg) < packs) ++*lg;
        return WAVE1;
    }
    *lg = 6;
    return packs <= 128 ? WAVE2 : packs <= 256 ? BLOCK1 : packs <= 512 ? BLOCK2 : packs <= 1024 ? BLOCK4 : SPLIT;
}
static long ln_blocks(long rows, Form f, int lg, bool bwd) {
    const long per = f <= WAVE2 ? 256 >> lg : 1;
    const long steps = cdiv(rows, per);
    const long cap = bwd ? 1024 : 2048;
    if (bwd && steps <= 2) return 1;                 // the parameters' gradients in one launch
    return steps < cap ? steps : cap;
}
// parts of the rows in the second launch of the split form: enough blocks for the chip, eight rows each at least
static long ln_split_parts(long rows, const SplitPlan& sp) {
    long p = cdiv(1024, sp.tiles);
    if (p > rows / 8) p = rows / 8;
    return p < 1 ? 1 : p;
}
static size_t ln_ws_bytes(long rows, long C, int type, int bwd) {
    int lg;
    const Form f = ln_form(C, type, &lg);
    if (f == SPLIT) {
        const SplitPlan sp = split_plan(C, type_size(type));
        const long parts = bwd ? ln_split_parts(rows, sp) : 1;
        return align256((size_t)rows * sp.chunks * sizeof(Chunk)) + (parts > 1 ? (size_t)parts * 2 * C * 4 : 0);
    }
    const long blocks = bwd ? ln_blocks(rows, f, lg, true) : 1;
    return blocks > 1 ? (size_t)blocks * 2 * C * 4 : 0;
}
static int ln_check(const char* what, const NormArgs& a, int type, int wtype) {
    SIV_CHECK_ARG(a.rows > 0 && a.C > 0 && a.C < (1L << 31) && a.rows < (1L << 40), "%s: rows and C must be positive (C < 2^31)", what);
    SIV_CHECK_ARG(a.ldx >= a.C && a.lddy >= a.C, "%s: a row stride is shorter than the row", what);
    SIV_CHECK_ARG(known_type(type), "%s: unknown element type", what);
    SIV_CHECK_ARG(wtype == SIV_F32 || wtype == type, "%s: weights must be fp32 or of the activations' type", what);
    SIV_CHECK_ARG(a.eps >= 0.f, "%s: eps must not be negative", what);
    return SIV_OK;
}
static int ln_check_ws(const char* what, size_t need, const void* ws, size_t have) {
    SIV_CHECK_ARG(ws || need == 0 || have == 0, "%s: null workspace", what);
    SIV_CHECK_WS(need, have, what);
    SIV_CHECK_ARG(need == 0 || ((uintptr_t)ws & 15) == 0, "%s: the workspace must be 16-byte aligned", what);
    return SIV_OK;
}
static bool ln_aligned(const NormArgs& a, int type) {
    const long n = 16 / type_size(type);
    return a.C % n == 0 && a.ldx % n == 0 && a.lddy % n == 0 && aligned16(a.x) && aligned16(a.res) && aligned16(a.dy) &&
           aligned16(a.ds) && aligned16(a.s) && aligned16(a.y) && aligned16(a.dx) && aligned16(a.dres);
}

template <typename T, bool AL, bool RES>
static void ln_fwd_launch(const NormArgs& a, const Drop& d, Form f, unsigned g, hipStream_t st) {
    switch (f) {
        case WAVE1: ln_fwd_k<T, 1, false, AL, RES><<<g, 256, 0, st>>>(a, d); break;
        case WAVE2: ln_fwd_k<T, 2, false, AL, RES><<<g, 256, 0, st>>>(a, d); break;
        case BLOCK1: ln_fwd_k<T, 1, true, AL, RES><<<g, 256, 0, st>>>(a, d); break;
        case BLOCK2: ln_fwd_k<T, 2, true, AL, RES><<<g, 256, 0, st>>>(a, d); break;
        default: ln_fwd_k<T, 4, true, AL, RES><<<g, 256, 0, st>>>(a, d); break;
    }
}
template <typename T, bool AL>
static void ln_bwd_launch(const NormArgs& a, const Drop& d, Form f, unsigned g, hipStream_t st) {
    switch (f) {
        case WAVE1: ln_bwd_k<T, 1, false, AL><<<g, 256, 0, st>>>(a, d); break;
        case WAVE2: ln_bwd_k<T, 2, false, AL><<<g, 256, 0, st>>>(a, d); break;
        case BLOCK1: ln_bwd_k<T, 1, true, AL><<<g, 256, 0, st>>>(a, d); break;
        case BLOCK2: ln_bwd_k<T, 2, true, AL><<<g, 256, 0, st>>>(a, d); break;
        default: ln_bwd_k<T, 4, true, AL><<<g, 256, 0, st>>>(a, d); break;
    }
}
static unsigned grid_y(long n) { return (unsigned)(n < 65535 ? n : 65535); }

static int ln_fwd(const char* what, NormArgs a, const Drop& d, bool res, int type, void* ws, size_t ws_bytes, hipStream_t st) {
    if (int rc = ln_check_ws(what, ln_ws_bytes(a.rows, a.C, type, 0), ws, ws_bytes)) return rc;
    const Form f = ln_form(a.C, type, &a.lg);
    const bool al = ln_aligned(a, type);
    const unsigned g = (unsigned)ln_blocks(a.rows, f, a.lg, false);
    return with_type(type, [&](auto* t) {
        typedef typename std::remove_reference<decltype(*t)>::type T;
        if (f != SPLIT) {
            if (al && res) ln_fwd_launch<T, true, true>(a, d, f, g, st);
            else if (al) ln_fwd_launch<T, true, false>(a, d, f, g, st);
            else if (res) ln_fwd_launch<T, false, true>(a, d, f, g, st);
            else ln_fwd_launch<T, false, false>(a, d, f, g, st);
            SIV_CHECK_LAUNCH(what);
            return SIV_OK;
        }
        const SplitPlan sp = split_plan(a.C, sizeof(T));
        const dim3 gs((unsigned)sp.chunks, grid_y(a.rows)), ga((unsigned)sp.tiles, grid_y(a.rows));
        Chunk* c = (Chunk*)ws;
        if (al && res) ln_split_stats_k<T, true, true, false><<<gs, 256, 0, st>>>(a, d, c);
        else if (al) ln_split_stats_k<T, true, false, false><<<gs, 256, 0, st>>>(a, d, c);
        else if (res) ln_split_stats_k<T, false, true, false><<<gs, 256, 0, st>>>(a, d, c);
        else ln_split_stats_k<T, false, false, false><<<gs, 256, 0, st>>>(a, d, c);
        SIV_CHECK_LAUNCH(what);
        if (al) ln_split_fwd_k<T, true><<<ga, 256, 0, st>>>(a, c);
        else ln_split_fwd_k<T, false><<<ga, 256, 0, st>>>(a, c);
        SIV_CHECK_LAUNCH(what);
        return SIV_OK;
    });
}
static int ln_bwd(const char* what, NormArgs a, const Drop& d, int type, void* ws, size_t ws_bytes, hipStream_t st) {
    if (int rc = ln_check_ws(what, ln_ws_bytes(a.rows, a.C, type, 1), ws, ws_bytes)) return rc;
    const Form f = ln_form(a.C, type, &a.lg);
    const bool al = ln_aligned(a, type);
    return with_type(type, [&](auto* t) {
        typedef typename std::remove_reference<decltype(*t)>::type T;
        long parts;
        if (f != SPLIT) {
            parts = ln_blocks(a.rows, f, a.lg, true);
            a.part = (float*)ws;
            if (al) ln_bwd_launch<T, true>(a, d, f, (unsigned)parts, st);
            else ln_bwd_launch<T, false>(a, d, f, (unsigned)parts, st);
        } else {
            const SplitPlan sp = split_plan(a.C, sizeof(T));
            Chunk* c = (Chunk*)ws;
            a.part = (float*)((char*)ws + align256((size_t)a.rows * sp.chunks * sizeof(Chunk)));
            parts = ln_split_parts(a.rows, sp);
            const dim3 gs((unsigned)sp.chunks, grid_y(a.rows)), ga((unsigned)sp.tiles, (unsigned)parts);
            if (al) ln_split_stats_k<T, true, false, true><<<gs, 256, 0, st>>>(a, d, c);
            else ln_split_stats_k<T, false, false, true><<<gs, 256, 0, st>>>(a, d, c);
            SIV_CHECK_LAUNCH(what);
            if (al) ln_split_bwd_k<T, true><<<ga, 256, 0, st>>>(a, d, c);
            else ln_split_bwd_k<T, false><<<ga, 256, 0, st>>>(a, d, c);
        }
        SIV_CHECK_LAUNCH(what);
        if ((a.dw || a.db) && parts > 1) {
            ln_param_sum_k<T><<<(unsigned)cdiv(2 * a.C, 16), 1024, 0, st>>>(a.part, parts, a);
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
    a.x = x; a.dy = dy; a.weight = weight; a.dx = dx; a.dw = dweight; a.db = dbias; a.accumulate = accumulate;
    a.rows = rows; a.C = C; a.ldx = ldx; a.lddy = lddy; a.eps = eps; a.wf32 = wtype == SIV_F32;
    if (int rc = ln_check("layer_norm_bwd", a, type, wtype)) return rc;
    return ln_bwd("layer_norm_bwd", a, make_drop(nullptr, 0, 0, nullptr, 0.f), type, ws, ws_bytes, (hipStream_t)stream);
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
    a.x = s; a.dy = dy; a.ds = ds; a.weight = weight; a.dx = dx; a.dres = dresidual; a.dw = dweight; a.db = dbias;
    a.accumulate = accumulate;
    a.rows = rows; a.C = C; a.ldx = C; a.lddy = C; a.eps = eps; a.wf32 = wtype == SIV_F32;
    if (int rc = ln_check("add_layer_norm_bwd", a, type, wtype)) return rc;
    return ln_bwd("add_layer_norm_bwd", a, make_drop(keep, seed, stream_id, epoch, p), type, ws, ws_bytes,
                  (hipStream_t)stream);
}
