// Layer normalisation over the elements of a row, alone or behind residual + dropout, forward and backward
// (fp32, bf16, fp16; arithmetic fp32).
//   mean = sum x / C, var = sum (x - mean)^2 / C, r = 1 / sqrt(var + eps), h = (x - mean) r, y = h w + b
//   g = dy w;  dx = r (g - sum g / C - h sum(g h) / C);  dw = sum_rows dy h;  db = sum_rows dy
// The mean is summed twice: m0 = sum x / C, then d = x - m0, delta = sum d / C, var = sum d^2 / C - delta^2.  x - m0
// is exact or nearly so, and delta takes back the rounding of m0, so rows far off zero keep their deviations.
// The backward pass forms the statistics again from the row it reads anyway, so forward leaves nothing behind.
//
// Bound by HBM: forward reads and writes the tensor once, backward reads two and writes one (residual form: two and two,
// three and two).  What the kernels move is that: WRITE_SIZE of a 4915200 x 64 fp32 call (1.26 GB tensors) is the tensor
// to 0.04 %.  Back-to-back calls of this build on one MI355X (profiles/norm_dropout_shapes.txt), TB/s of those bytes, where a
// device copy of that size runs at 4.5-5.2: 4915200 x 64 fp32 forward 437 us (5.8), backward 667 us (5.7); residual form
// 614400 x 128 fp32 228 (5.5) and 305 us (5.2).  With 16-bit elements the arithmetic of the backward pass (about 16
// operations an element on a lane that holds eight) is close behind: 614400 x 128 bf16 forward 61 us (5.2), backward 92 us
// (5.2); 100000 x 601, where 52 of 128 lanes have no column, 110 us (3.3).  Where a comment below gives two times for a
// choice, they are of one series on the build of that day: the difference is meant, not the level.
#include <algorithm>
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
// Sums over the lanes that share a row: part of a wave (NT = 64), or NT threads of a block of NT x R.  Two LDS buffers
// in turn: the barrier of one sum also separates the readers of the sum before it from the writers of the next.
template <int NT, int R>
struct RowSum {
    float4 (*sh)[R * NT / 64];
    int lg, turn;
    template <int N>
    __device__ __forceinline__ void operator()(float (&v)[N]) {
        if (NT == 64) {
            lanes_sum(v, lg);
            return;
        }
        lanes_sum(v, 6);
        float4* buf = sh[turn] + (R > 1 ? threadIdx.x / NT * (NT / 64) : 0);
        if ((threadIdx.x & 63) == 0)
            sh[turn][threadIdx.x >> 6] = make_float4(v[0], N > 1 ? v[N > 1 ? 1 : 0] : 0.f, N > 2 ? v[N > 2 ? 2 : 0] : 0.f,
                                                N > 3 ? v[N > 3 ? 3 : 0] : 0.f);
        __syncthreads();
        float4 s = buf[0];
#pragma unroll
        for (int w = 1; w < NT / 64; ++w) {
            const float4 o = buf[w];
            s.x += o.x;
            if (N > 1) s.y += o.y;
            if (N > 2) s.z += o.z;
            if (N > 3) s.w += o.w;
        }
        v[0] = s.x;
        if (N > 1) v[N > 1 ? 1 : 0] = s.y;
        if (N > 2) v[N > 2 ? 2 : 0] = s.z;
        if (N > 3) v[N > 3 ? 3 : 0] = s.w;
        turn ^= 1;
    }
};

// ---- the columns of a lane's pack ------------------------------------------------------------------------------------
// ALIGNED: rows start on 16 bytes and hold whole packs.  OVERLAP: they need not; the last pack of a row is moved back so
// that it ends with the row, the columns it shares with the pack before it count there only (both store the same
// value).  Every access is one 16-byte instruction either way.  SHORT: rows of less than a pack, element by element.
enum Cols { SHORT, OVERLAP, ALIGNED };
// Lanes without a column or a row are not branched around: a conditional store in a loop makes the compiler wait for
// every store of a step before it uses what was loaded a step ahead.  They go to an offset that the buffer descriptor
// turns away (loads give zero, stores nothing).
constexpr uint32_t NOWHERE = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00020000);
}
template <typename T, int COLS>
struct Span {
    static constexpr int N = Pack<T>::N;
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    uint32_t c;             // first column accessed
    int lo, hi;             // elements lo .. hi-1 of the pack are this lane's
    __device__ __forceinline__ Span() {}
    __device__ __forceinline__ Span(long pack, long C) {
        const long have = C - pack * N;
        lo = 0;
        hi = have >= N ? N : have > 0 ? (int)have : 0;
        c = (uint32_t)(pack * N);
        if (COLS == OVERLAP && have < N) {
            lo = have > 0 ? N - (int)have : N;
            hi = N;
            c = (uint32_t)(C - N);
        }
    }
    __device__ __forceinline__ bool any() const { return lo < hi; }
    // whether some lane of the wave holds part of a pack: only there do sums look at single elements
    __device__ __forceinline__ bool ragged() const { return COLS != ALIGNED && __any(any() && hi - lo < N); }
    __device__ __forceinline__ bool mine(int j) const {
        return COLS == ALIGNED ? hi > 0 : COLS == OVERLAP ? j >= lo : j < hi;
    }
    // byte offset of the pack in a tensor whose rows are ld apart, from `row` rows behind the base (and `from` columns
    // into it) on
    __device__ __forceinline__ uint32_t at(long row, long ld, uint32_t from = 0) const {
        return any() ? (uint32_t)((row * ld + c - from) * (long)sizeof(T)) : NOWHERE;
    }
    // base: the same for the whole wave.  LAST: nothing is expected to read the tensor again soon.
    template <bool LAST = false>
    __device__ __forceinline__ Pack<T> load(const void* base, uint32_t off) const {
        Pack<T> v;
        if (COLS == SHORT) {
            const T* p = (const T*)((const char*)base + off);
#pragma unroll
            for (int j = 0; j < N; ++j) v.e[j] = off != NOWHERE && j < hi ? p[j] : (T)0.f;
        } else {
            const words w = __builtin_amdgcn_raw_buffer_load_b128(rows_rsrc(base), off, 0, LAST ? 2 : 0);
            __builtin_memcpy(v.e, &w, 16);
        }
        return v;
    }
    __device__ __forceinline__ void store(void* base, uint32_t off, const Pack<T>& v) const {
        if (COLS == SHORT) {
            T* p = (T*)((char*)base + off);
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (off != NOWHERE && j < hi) p[j] = v.e[j];
        } else {
            words w;
            __builtin_memcpy(&w, v.e, 16);
            // non-temporal: the L2, which a kernel's end writes back anyway, is left to the operands
            __builtin_amdgcn_raw_buffer_store_b128(w, rows_rsrc(base), off, 0, 2);
        }
    }
    // this pack's columns of a parameter vector, in as few loads as the type allows
    __device__ __forceinline__ void params(const void* w, int f32, float dflt, float (&out)[N]) const {
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = dflt;
        if (!w || !any()) return;
        if (f32) {
            const float* p = (const float*)w + c;
            if (COLS == SHORT) {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (j < hi) out[j] = p[j];
            } else {
                __builtin_memcpy(out, p, 4 * N);
            }
        } else {
            const T* p = (const T*)w + c;
            Pack<T> v;
            if (COLS == SHORT) {
#pragma unroll
                for (int j = 0; j < N; ++j) v.e[j] = j < hi ? p[j] : (T)0.f;
            } else {
                __builtin_memcpy(v.e, p, 16);
            }
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (COLS != SHORT || j < hi) out[j] = (float)v.e[j];
        }
    }
};
template <typename T>
__device__ __forceinline__ void put_param(void* out, int f32, long c, float v, int accumulate) {
    if (f32) ((float*)out)[c] = accumulate ? ((float*)out)[c] + v : v;
    else ((T*)out)[c] = (T)(accumulate ? (float)((T*)out)[c] + v : v);
}

// What one pack adds to a row's sums: sum x; or, of d = x - m0 and g = dy w, sum d, sum d^2, sum g, sum g d.
template <typename T, int COLS>
__device__ __forceinline__ float pack_sum(const Span<T, COLS>& sp, bool ragged, const Pack<T>& x) {
    float s = 0.f;
    if (ragged) {
#pragma unroll
        for (int j = 0; j < Pack<T>::N; ++j) s += sp.mine(j) ? (float)x.e[j] : 0.f;
    } else {
#pragma unroll
        for (int j = 0; j < Pack<T>::N; ++j) s += (float)x.e[j];
    }
    return sp.any() ? s : 0.f;
}
template <typename T, int COLS, bool BWD>
__device__ __forceinline__ void pack_sums(const Span<T, COLS>& sp, bool ragged, const float* d, const float* g,
                                          float (&m)[4]) {
    constexpr int N = Pack<T>::N;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float dj = !ragged || sp.mine(j) ? d[j] : 0.f;
        s[0] += dj;
        s[1] += dj * dj;
        if (BWD) {
            const float gj = !ragged || sp.mine(j) ? g[j] : 0.f;
            s[2] += gj;
            s[3] += gj * dj;
        }
    }
#pragma unroll
    for (int i = 0; i < (BWD ? 4 : 2); ++i) m[i] += sp.any() ? s[i] : 0.f;
}

// residual + dropout(x) of one pack from element i on, as it is held
template <typename T, int COLS>
__device__ __forceinline__ Pack<T> add_drop(const Pack<T>& x, const Pack<T>& res, const Drop& d, uint64_t sid, long i,
                                            int hi) {
    constexpr int N = Pack<T>::N;
    Pack<T> s;
    if (d.mode == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) s.e[j] = (T)((float)res.e[j] + (float)x.e[j]);
        return s;
    }
    uint32_t w[N];
    drop_words<N, COLS == ALIGNED>(d, sid, i, hi, w);
#pragma unroll
    for (int j = 0; j < N; ++j) s.e[j] = (T)((float)res.e[j] + (w[j] >= d.least ? (float)x.e[j] * d.scale : 0.f));
    return s;
}

// ---- rows held in registers -----------------------------------------------------------------------------------------
// A row is spread over 2^lg lanes of a wave, 64 >> lg rows to a wave and four waves to a block (NT = 64), or over NT
// threads, R rows to a block; a lane holds NV packs of 16 bytes.  One pass over the data.  Blocks walk the rows in
// strides of the grid, so that weights and the parameters' gradients stay in registers; the next row is requested before
// the present one is worked on (not in the forward wave form, whose blocks take one step: 4915200 x 64 fp32 483 us with a
// grid of 2048 that walks, 441 us with a block per step).
template <typename T, int NV, int NT, int R, int COLS, bool RES>
__global__ __launch_bounds__(NT == 64 ? 256 : NT * R) void ln_fwd_k(NormArgs a, Drop d) {
    constexpr int N = Pack<T>::N;
    constexpr bool AHEAD = NV > 1 || NT > 64;
    __shared__ float4 sh[2][R * NT / 64];
    RowSum<NT, R> row_sum{sh, a.lg, 0};
    const int lane = threadIdx.x & 63;
    const int G = NT == 64 ? 1 << a.lg : NT;
    const int sub = NT == 64 ? lane & (G - 1) : threadIdx.x % NT;
    const long per = NT == 64 ? 256 >> a.lg : R;                      // rows of one block step
    const long step = (long)gridDim.x * per;
    const uint64_t sid = RES ? drop_sid(d) : 0;
    const float invC = 1.0f / (float)a.C;
    const int rin = NT == 64 ? threadIdx.x >> a.lg : threadIdx.x / NT;   // this lane's row within the step
    Span<T, COLS> sp[NV];
    float w[NV][N], b[NV][N];
    uint32_t ox[NV], od[NV];                                          // offsets in x, and in the dense tensors
    bool ragged[NV];
    long lead = (long)blockIdx.x * per;                               // first row of the step
    bool ok = rin < a.rows - lead;
    Pack<T> x[NV], q[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        sp[k] = Span<T, COLS>(k * G + sub, a.C);
        ragged[k] = sp[k].ragged();
        ox[k] = sp[k].at(rin, a.ldx);
        od[k] = sp[k].at(rin, a.C);
        x[k] = sp[k].load((const T*)a.x + lead * a.ldx, ok ? ox[k] : NOWHERE);
        if (RES) q[k] = sp[k].load((const T*)a.res + lead * a.C, ok ? od[k] : NOWHERE);
        sp[k].params(a.weight, a.wf32, 1.f, w[k]);
        sp[k].params(a.bias, a.wf32, 0.f, b[k]);
    }
    for (; lead < a.rows; lead += step) {
        const bool more = rin < a.rows - (lead + step);
        Pack<T> xn[NV], qn[NV];
        if (AHEAD)
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                xn[k] = sp[k].load((const T*)a.x + (lead + step) * a.ldx, more ? ox[k] : NOWHERE);
                if (RES) qn[k] = sp[k].load((const T*)a.res + (lead + step) * a.C, more ? od[k] : NOWHERE);
            }
        float v[NV][N];
        float s1[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (RES) {
                x[k] = add_drop<T, COLS>(x[k], q[k], d, sid, (lead + rin) * a.C + sp[k].c, ok ? sp[k].hi : 0);
                sp[k].store((T*)a.s + lead * a.C, ok ? od[k] : NOWHERE, x[k]);
            }
            s1[0] += pack_sum(sp[k], ragged[k], x[k]);
        }
        row_sum(s1);
        const float m0 = s1[0] * invC;
        float m4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int j = 0; j < N; ++j) v[k][j] = (float)x[k].e[j] - m0;
            pack_sums<T, COLS, false>(sp[k], ragged[k], v[k], nullptr, m4);
        }
        float m[2] = {m4[0], m4[1]};
        row_sum(m);
        const float delta = m[0] * invC;
        const float r = rsqrtf(fmaxf(m[1] * invC - delta * delta, 0.f) + a.eps), dr = -delta * r;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            Pack<T> p;
#pragma unroll
            for (int j = 0; j < N; ++j) p.e[j] = (T)((v[k][j] * r + dr) * w[k][j] + b[k][j]);
            sp[k].store((T*)a.y + lead * a.C, ok ? od[k] : NOWHERE, p);
            if (AHEAD) {
                x[k] = xn[k];
                if (RES) q[k] = qn[k];
            }
        }
        ok = more;
        if (AHEAD) continue;
        if (lead + step >= a.rows) break;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            x[k] = sp[k].load((const T*)a.x + (lead + step) * a.ldx, more ? ox[k] : NOWHERE);
            if (RES) q[k] = sp[k].load((const T*)a.res + (lead + step) * a.C, more ? od[k] : NOWHERE);
        }
    }
}

// The same rows backward.  Each lane sums dy h and dy of its columns over the rows it sees; a block's sums go to
// a.part, or straight to the results where there is one block.  x and dy of the wave form, which nothing is expected to
// read after this, are loaded non-temporally.  That pays where a call moves more than the Infinity Cache holds and costs where
// it moves less (us, plain | non-temporal, profiles/norm_dropout_rules.txt): 4915200 x 64 fp32 706 | 684, 614400 x 128 bf16
// 92.8 | 84.7, 153600 x 256 bf16 (236 MB) 48.5 | 45.6; 76800 x 256 bf16 (118 MB) 25.0 | 26.5, 200000 x 33 fp32 (79 MB)
// 20.3 | 22.8.  One hint for all sizes: the large tensors are where the time is.
template <typename T, int NV, int NT, int R, int COLS, bool RES>
__global__ __launch_bounds__(NT == 64 ? 256 : NT * R) void ln_bwd_k(NormArgs a, Drop d) {
    constexpr int N = Pack<T>::N;
    constexpr bool LAST = NT == 64;
    __shared__ float4 sh[2][R * NT / 64];
    constexpr int ROWS = NT == 64 ? 4 : R, WIDE = NT * NV * N;    // sums to join at the end, columns of one
    __shared__ float fold[ROWS * WIDE];
    RowSum<NT, R> row_sum{sh, a.lg, 0};
    const int lane = threadIdx.x & 63;
    const int G = NT == 64 ? 1 << a.lg : NT;
    const int sub = NT == 64 ? lane & (G - 1) : threadIdx.x % NT;
    const long per = NT == 64 ? 256 >> a.lg : R;
    const long step = (long)gridDim.x * per;
    const uint64_t sid = RES ? drop_sid(d) : 0;
    const float invC = 1.0f / (float)a.C;
    const int rin = NT == 64 ? threadIdx.x >> a.lg : threadIdx.x / NT;
    Span<T, COLS> sp[NV];
    float w[NV][N], gw[NV][N], gb[NV][N];
    uint32_t ox[NV], oy[NV], od[NV];
    bool ragged[NV];
    long lead = (long)blockIdx.x * per;
    bool ok = rin < a.rows - lead;
    Pack<T> x[NV], gy[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        sp[k] = Span<T, COLS>(k * G + sub, a.C);
        ragged[k] = sp[k].ragged();
        ox[k] = sp[k].at(rin, a.ldx);
        oy[k] = sp[k].at(rin, a.lddy);
        od[k] = sp[k].at(rin, a.C);
        x[k] = sp[k].template load<LAST>((const T*)a.x + lead * a.ldx, ok ? ox[k] : NOWHERE);
        gy[k] = sp[k].template load<LAST>((const T*)a.dy + lead * a.lddy, ok ? oy[k] : NOWHERE);
        sp[k].params(a.weight, a.wf32, 1.f, w[k]);
#pragma unroll
        for (int j = 0; j < N; ++j) gw[k][j] = gb[k][j] = 0.f;
    }
    for (; lead < a.rows; lead += step) {
        const bool more = rin < a.rows - (lead + step);
        Pack<T> xn[NV], gn[NV], ds[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (RES) ds[k] = sp[k].template load<LAST>((const T*)a.ds + lead * a.C, ok && a.ds ? od[k] : NOWHERE);
            xn[k] = sp[k].template load<LAST>((const T*)a.x + (lead + step) * a.ldx, more ? ox[k] : NOWHERE);
            gn[k] = sp[k].template load<LAST>((const T*)a.dy + (lead + step) * a.lddy, more ? oy[k] : NOWHERE);
        }
        float s1[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) s1[0] += pack_sum(sp[k], ragged[k], x[k]);
        row_sum(s1);
        const float m0 = s1[0] * invC;
        float m[4] = {0.f, 0.f, 0.f, 0.f};
        float v[NV][N], g[NV][N];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[k][j] = (float)x[k].e[j] - m0;
                g[k][j] = (float)gy[k].e[j] * w[k][j];
            }
            pack_sums<T, COLS, true>(sp[k], ragged[k], v[k], g[k], m);
        }
        row_sum(m);
        const float delta = m[0] * invC;
        float r = rsqrtf(fmaxf(m[1] * invC - delta * delta, 0.f) + a.eps);
        if (!ok) r = 0.f;                    // lanes without a row add nothing, whatever eps is
        // h = v r + dr;  dx = g r - c1 r - h c2 r
        const float dr = -delta * r, k1 = -m[2] * invC * r, k2 = -(m[3] - delta * m[2]) * r * invC * r;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float dy = (float)gy[k].e[j], h = v[k][j] * r + dr;
                gw[k][j] += dy * h;
                gb[k][j] += dy;
                g[k][j] = h * k2 + (g[k][j] * r + k1);
                if (RES) g[k][j] += (float)ds[k].e[j];
            }
            Pack<T> p;
#pragma unroll
            for (int j = 0; j < N; ++j) p.e[j] = (T)g[k][j];
            if (RES) {
                sp[k].store((T*)a.dres + lead * a.C, ok && a.dres ? od[k] : NOWHERE, p);
                if (d.mode) {
                    uint32_t u[N];
                    drop_words<N, COLS == ALIGNED>(d, sid, (lead + rin) * a.C + sp[k].c, ok ? sp[k].hi : 0, u);
#pragma unroll
                    for (int j = 0; j < N; ++j) p.e[j] = (T)(u[j] >= d.least ? g[k][j] * d.scale : 0.f);
                }
            }
            sp[k].store((T*)a.dx + lead * a.C, ok && a.dx ? od[k] : NOWHERE, p);
            x[k] = xn[k];
            gy[k] = gn[k];
        }
        ok = more;
    }
    if (!a.dw && !a.db) return;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* out = a.part + ((long)blockIdx.x * 2 + which) * a.C;
        void* res = which ? a.db : a.dw;
        const int mine = NT == 64 ? threadIdx.x >> 6 : rin;
        // wave form: rows of one wave that share columns; then the waves or rows of the block
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float t = which ? gb[k][j] : gw[k][j];
                if (NT == 64)
                    for (int o = G; o < 64; o <<= 1) t += __shfl_xor(t, o, 64);
                if ((NT > 64 || lane < G) && sp[k].mine(j)) fold[mine * WIDE + (int)sp[k].c + j] = t;
            }
        __syncthreads();
        for (int c = threadIdx.x; c < (int)a.C; c += blockDim.x) {
            float t = fold[c];
#pragma unroll
            for (int i = 1; i < ROWS; ++i) t += fold[i * WIDE + c];
            if (gridDim.x > 1) out[c] = t;
            else if (res) put_param<T>(res, a.wf32, c, t, a.accumulate);
        }
        __syncthreads();
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

// first column that a tile's packs may touch (the last pack of a row may reach back into the tile before it)
template <typename T>
__device__ __forceinline__ long split_from(const SplitPlan& sp, long tile) {
    return tile ? tile * sp.tile - Pack<T>::N : 0;
}

template <typename T, int COLS, bool RES, bool BWD>
__global__ __launch_bounds__(256) void ln_split_stats_k(NormArgs a, Drop d, Chunk* __restrict__ st) {
    constexpr int N = Pack<T>::N;
    __shared__ float4 sh[2][4];
    RowSum<256, 1> row_sum{sh, 6, 0};
    const SplitPlan sp = split_plan(a.C, sizeof(T));
    const uint64_t sid = RES ? drop_sid(d) : 0;
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        double n = 0, mean = 0, m2 = 0, G = 0, H = 0;
        for (long t = blockIdx.x * sp.per; t < (blockIdx.x + 1) * sp.per && t < sp.tiles; ++t) {
            const long from = split_from<T>(sp, t);
            Pack<T> x[SPLIT_NV];
            float g[SPLIT_NV][N];
            Span<T, COLS> c[SPLIT_NV];
            float s1[1] = {0.f};
#pragma unroll
            for (int k = 0; k < SPLIT_NV; ++k) {
                c[k] = Span<T, COLS>((t * SPLIT_NV + k) * 256 + threadIdx.x, a.C);
                const uint32_t off = c[k].at(0, 0, (uint32_t)from);
                x[k] = c[k].load((const T*)a.x + row * a.ldx + from, off);
                if (RES) {
                    const Pack<T> q = c[k].load((const T*)a.res + row * a.C + from, off);
                    x[k] = add_drop<T, COLS>(x[k], q, d, sid, row * a.C + c[k].c, c[k].hi);
                    c[k].store((T*)a.s + row * a.C + from, off, x[k]);
                }
                if (BWD) {
                    const Pack<T> q = c[k].load((const T*)a.dy + row * a.lddy + from, off);
                    c[k].params(a.weight, a.wf32, 1.f, g[k]);
#pragma unroll
                    for (int j = 0; j < N; ++j) g[k][j] = c[k].mine(j) ? g[k][j] * (float)q.e[j] : 0.f;
                }
#pragma unroll
                for (int j = 0; j < N; ++j) s1[0] += c[k].mine(j) ? (float)x[k].e[j] : 0.f;
            }
            row_sum(s1);
            const long nt = a.C - t * sp.tile < sp.tile ? a.C - t * sp.tile : sp.tile;
            const float m0 = s1[0] / (float)nt;
            float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < SPLIT_NV; ++k)
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float v = c[k].mine(j) ? (float)x[k].e[j] - m0 : 0.f;
                    m[0] += v;
                    m[1] += v * v;
                    if (BWD) {
                        m[2] += g[k][j];
                        m[3] += g[k][j] * v;
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
// Every wave joins all chunks of the row by itself: the same operations in the same order, no barrier.  Means are taken
// relative to the first chunk's, which leaves numbers of the size of the deviations: floats hold those.
struct RowStats {
    float hi, lo, r, c1, c2;              // mean = hi + lo
};
template <bool BWD>
__device__ __forceinline__ RowStats join_chunks(const Chunk* __restrict__ st, const SplitPlan& sp, long C, float eps) {
    constexpr int PER = SPLIT_MAX / 64;
    const int lane = threadIdx.x & 63;
    const long whole = sp.per * sp.tile;
    const float invC = 1.0f / (float)C;
    const double base = st[0].mean;
    float e[PER], n[PER], s1[1] = {0.f};
    Chunk c[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const long k = lane + 64 * i;
        const bool in = k < sp.chunks;
        if (in) c[i] = st[k];
        n[i] = in ? (float)(k + 1 < sp.chunks ? whole : C - k * whole) : 0.f;
        e[i] = in ? (float)(c[i].mean - base) : 0.f;
        s1[0] += n[i] * e[i];
    }
    lanes_sum(s1, 6);
    const float off = s1[0] * invC;
    float m[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (n[i] == 0.f) continue;
        const float x = e[i] - off;
        m[0] += c[i].m2 + n[i] * x * x;
        m[1] += c[i].g;
        m[2] += c[i].h + c[i].g * x;
    }
    lanes_sum(m, 6);
    const double mean = base + (double)off;
    RowStats s;
    s.hi = (float)mean;
    s.lo = (float)(mean - (double)s.hi);
    s.r = rsqrtf(m[0] * invC + eps);
    s.c1 = BWD ? m[1] * invC : 0.f;
    s.c2 = BWD ? m[2] * invC * s.r : 0.f;
    return s;
}
template <typename T, int COLS>
__global__ __launch_bounds__(256) void ln_split_fwd_k(NormArgs a, const Chunk* __restrict__ st) {
    constexpr int N = Pack<T>::N;
    const SplitPlan sp = split_plan(a.C, sizeof(T));
    const long from = split_from<T>(sp, blockIdx.x);
    Span<T, COLS> c[SPLIT_NV];
    uint32_t off[SPLIT_NV];
#pragma unroll
    for (int k = 0; k < SPLIT_NV; ++k) {
        c[k] = Span<T, COLS>((blockIdx.x * (long)SPLIT_NV + k) * 256 + threadIdx.x, a.C);
        off[k] = c[k].at(0, 0, (uint32_t)from);
    }
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const T* src = (a.s ? (const T*)a.s + row * a.C : (const T*)a.x + row * a.ldx) + from;
        Pack<T> x[SPLIT_NV];
#pragma unroll
        for (int k = 0; k < SPLIT_NV; ++k) x[k] = c[k].load(src, off[k]);
        const RowStats s = join_chunks<false>(st + row * sp.chunks, sp, a.C, a.eps);
#pragma unroll
        for (int k = 0; k < SPLIT_NV; ++k) {
            float w[N], b[N];
            c[k].params(a.weight, a.wf32, 1.f, w);
            c[k].params(a.bias, a.wf32, 0.f, b);
            Pack<T> o;
#pragma unroll
            for (int j = 0; j < N; ++j) o.e[j] = (T)((((float)x[k].e[j] - s.hi) * s.r - s.lo * s.r) * w[j] + b[j]);
            c[k].store((T*)a.y + row * a.C + from, off[k], o);
        }
    }
}
// Backward: block (tile, part of the rows) keeps the parameter gradients of its columns in registers.  Its waves first
// join the chunks of a batch of rows, four rows at a time, so that the rows behind are one stream of loads.
constexpr int SPLIT_BATCH = 16;
template <typename T, int COLS>
__global__ __launch_bounds__(256) void ln_split_bwd_k(NormArgs a, Drop d, const Chunk* __restrict__ st) {
    constexpr int N = Pack<T>::N;
    __shared__ RowStats stats[SPLIT_BATCH];
    const SplitPlan sp = split_plan(a.C, sizeof(T));
    const uint64_t sid = drop_sid(d);
    const int wave = threadIdx.x >> 6;
    float w[SPLIT_NV][N], gw[SPLIT_NV][N], gb[SPLIT_NV][N];
    Span<T, COLS> c[SPLIT_NV];
    Pack<T> x[SPLIT_NV], gy[SPLIT_NV];
    const long from = split_from<T>(sp, blockIdx.x);
    uint32_t off[SPLIT_NV];
    long row = blockIdx.y;
#pragma unroll
    for (int k = 0; k < SPLIT_NV; ++k) {
        c[k] = Span<T, COLS>((blockIdx.x * (long)SPLIT_NV + k) * 256 + threadIdx.x, a.C);
        off[k] = c[k].at(0, 0, (uint32_t)from);
        x[k] = c[k].load((const T*)a.x + row * a.ldx + from, off[k]);
        gy[k] = c[k].load((const T*)a.dy + row * a.lddy + from, off[k]);
        c[k].params(a.weight, a.wf32, 1.f, w[k]);
#pragma unroll
        for (int j = 0; j < N; ++j) gw[k][j] = gb[k][j] = 0.f;
    }
    for (int at = 0; row < a.rows; row += gridDim.y, at = (at + 1) % SPLIT_BATCH) {
        if (at == 0) {
            __syncthreads();                                     // the last batch has been read
            for (int i = wave; i < SPLIT_BATCH; i += 4) {
                const long r = row + (long)i * gridDim.y;
                if (r >= a.rows) break;
                const RowStats s = join_chunks<true>(st + r * sp.chunks, sp, a.C, a.eps);
                if ((threadIdx.x & 63) == 0) stats[i] = s;
            }
            __syncthreads();
        }
        const RowStats s = stats[at];
        const float dr = -s.lo * s.r, k1 = -s.c1 * s.r, k2 = -s.c2 * s.r;
        const long next = row + gridDim.y;
        const bool more = next < a.rows;
        Pack<T> xn[SPLIT_NV], gn[SPLIT_NV], ds[SPLIT_NV];
#pragma unroll
        for (int k = 0; k < SPLIT_NV; ++k) {
            ds[k] = c[k].load((const T*)a.ds + row * a.C + from, a.ds ? off[k] : NOWHERE);
            xn[k] = c[k].load((const T*)a.x + next * a.ldx + from, more ? off[k] : NOWHERE);
            gn[k] = c[k].load((const T*)a.dy + next * a.lddy + from, more ? off[k] : NOWHERE);
        }
#pragma unroll
        for (int k = 0; k < SPLIT_NV; ++k) {
            float g[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float dy = (float)gy[k].e[j];
                const float h = ((float)x[k].e[j] - s.hi) * s.r + dr;
                gw[k][j] += dy * h;
                gb[k][j] += dy;
                g[j] = h * k2 + (dy * w[k][j] * s.r + k1) + (float)ds[k].e[j];
            }
            Pack<T> o;
#pragma unroll
            for (int j = 0; j < N; ++j) o.e[j] = (T)g[j];
            c[k].store((T*)a.dres + row * a.C + from, a.dres ? off[k] : NOWHERE, o);
            if (d.mode) {
                uint32_t u[N];
                drop_words<N, COLS == ALIGNED>(d, sid, row * a.C + c[k].c, c[k].hi, u);
#pragma unroll
                for (int j = 0; j < N; ++j) o.e[j] = (T)(u[j] >= d.least ? g[j] * d.scale : 0.f);
            }
            c[k].store((T*)a.dx + row * a.C + from, a.dx ? off[k] : NOWHERE, o);
            x[k] = xn[k];
            gy[k] = gn[k];
        }
    }
    if (!a.dw && !a.db) return;
#pragma unroll
    for (int k = 0; k < SPLIT_NV; ++k)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (!c[k].mine(j)) continue;
            const long i = (long)c[k].c + j;
            if (gridDim.y > 1) {
                a.part[((long)blockIdx.y * 2 + 0) * a.C + i] = gw[k][j];
                a.part[((long)blockIdx.y * 2 + 1) * a.C + i] = gb[k][j];
            } else {
                if (a.dw) put_param<T>(a.dw, a.wf32, i, gw[k][j], a.accumulate);
                if (a.db) put_param<T>(a.db, a.wf32, i, gb[k][j], a.accumulate);
            }
        }
}

// the blocks' partial sums joined: 1024 / DOWN columns to a block, DOWN threads down each, in a fixed order
template <typename T, int DOWN>
__global__ __launch_bounds__(1024) void ln_param_sum_k(const float* __restrict__ part, long parts, NormArgs a) {
    constexpr int ACROSS = 1024 / DOWN;
    __shared__ float sh[DOWN][ACROSS + 1];
    const int col = threadIdx.x % ACROSS, down = threadIdx.x / ACROSS;
    const long i = (long)blockIdx.x * ACROSS + col, C2 = 2 * a.C;
    float t = 0.f;
    if (i < C2) {
        long k = down;
        for (; k + 3 * DOWN < parts; k += 4 * DOWN)          // four loads at a time
            t += (part[k * C2 + i] + part[(k + DOWN) * C2 + i]) +
                 (part[(k + 2 * DOWN) * C2 + i] + part[(k + 3 * DOWN) * C2 + i]);
        for (; k < parts; k += DOWN) t += part[k * C2 + i];
    }
    sh[down][col] = t;
    for (int o = DOWN / 2; o > 0; o >>= 1) {
        __syncthreads();
        if (down < o) sh[down][col] += sh[down + o][col];
    }
    if (down || i >= C2) return;
    void* out = i < a.C ? a.dw : a.db;
    if (out) put_param<T>(out, a.wf32, i < a.C ? i : i - a.C, sh[0][col], a.accumulate);
}

// ---- host -------------------------------------------------------------------------------------------------------------
// The forms, by packs of 16 bytes in a row (fp32: 4 elements, 16-bit: 8).  Up to 64: lanes of one wave.  Up to 128: forward
// two packs to a lane (100000 x 601 bf16: 47 us; 56 against 64 with a pack to each of 128 threads), backward 128 threads,
// since two packs' sums and gradients need 168 registers.  Then a thread per pack up to 1024, four, two or one rows to a block so
// that a block's partial sums stand for several rows (20000 x 1024 bf16 backward: 25 us; one row to a block 39, four 28).
// Up to 2048: two packs a thread, except 16-bit backward, which spills.  Longer rows: chunks, whose second read costs half as
// much again (300 x 100000 fp32: forward 59 us = 6.1 TB/s of three passes, backward 110 us = 5.5 of five).
// Which kernel: a function of the row length and stride, the type and the direction alone, so that a row's result does
// not depend on what is computed beside it.
struct Form {
    int nt, nv, lg;         // nt 0: split
    int rows() const { return nt == 64 ? 256 >> lg : nt == 128 ? 4 : nt == 256 ? 2 : 1; }      // of one block step
    int threads() const { return nt == 64 ? 256 : nt * rows(); }
};
static Form ln_form(long C, long ld, int type, bool bwd) {
    const long packs = cdiv(C, 16 / type_size(type));
    Form f = {0, 0, 0};
    if (packs <= 64) {
        f = {64, 1, 0};
        while ((1L << f.lg) < packs) ++f.lg;
    } else if (packs <= 128) {
        f = bwd ? Form{128, 1, 6} : Form{64, 2, 6};
    } else if (packs <= 256) {
        f = {256, 1, 6};
    } else if (packs <= 512) {
        f = {512, 1, 6};
    } else if (packs <= 1024) {
        f = {1024, 1, 6};
    } else if (packs <= 2048 && (!bwd || type == SIV_F32)) {
        f = {1024, 2, 6};
    }
    // the rows of a step are reached with 31-bit offsets: rows very far apart go one to a step
    if (f.nt && f.rows() > 1 && ld >= (1L << 31) / (f.rows() * 4L)) f = {512, 1, 6};
    return f;
}
static long ln_blocks(long rows, const Form& f, bool bwd) {
    const long steps = cdiv(rows, f.rows());
    if (!bwd) {
        // (block forms walk: 2000 x 16384 bf16 28 us, with a block per row 35)
        const long cap = f.nt > 64 ? 2048 * 256L / f.threads() : f.nv == 2 ? 8192 : 1L << 20;
        return steps < cap ? steps : cap;
    }
    if (steps <= 4) return 1;                        // the parameters' gradients in one launch
    // Blocks that stay: 768 x 256 threads in the wave form (4915200 x 64 fp32: 664 us; 640: 697, 896: 712, 1024: 704;
    // with plain loads and stores 768: 688, 512: 816, 1024: 738), 1024 x 256 with the barriers of the block forms (8192 x
    // 4096 fp32: 92 us; 768: 112, 1280: 130).  Four steps each at least, where that leaves a block per CU.
    const long cap = (f.nt == 64 ? 768 : 1024) * 256L / f.threads();
    const long b = steps / 4 > 256 ? steps / 4 : 256;
    return std::min(std::min(b, cap), steps);
}
// parts of the rows in the second launch of the split form: enough blocks for the chip, eight rows each at least
static long ln_split_parts(long rows, const SplitPlan& sp) {
    long p = cdiv(1024, sp.tiles);
    if (p > rows / 8) p = rows / 8;
    return p < 1 ? 1 : p;
}
static size_t ln_ws_bytes(long rows, long C, long ld, int type, int bwd) {
    const Form f = ln_form(C, ld, type, bwd);
    if (f.nt == 0) {
        const SplitPlan sp = split_plan(C, type_size(type));
        const long parts = bwd ? ln_split_parts(rows, sp) : 1;
        return align256((size_t)rows * sp.chunks * sizeof(Chunk)) + (parts > 1 ? (size_t)parts * 2 * C * 4 : 0);
    }
    const long blocks = bwd ? ln_blocks(rows, f, true) : 1;
    return blocks > 1 ? (size_t)blocks * 2 * C * 4 : 0;
}
static int ln_check(const char* what, const NormArgs& a, int type, int wtype) {
    SIV_CHECK_ARG(a.rows > 0 && a.C > 0 && a.C < (1L << 31) && a.rows < (1L << 40),
                  "%s: rows and C must be positive (C < 2^31)", what);
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
static Cols ln_cols(const NormArgs& a, int type) {
    const long n = 16 / type_size(type);
    if (a.C < n) return SHORT;
    return a.C % n == 0 && a.ldx % n == 0 && a.lddy % n == 0 && aligned16(a.x) && aligned16(a.res) && aligned16(a.dy) &&
                   aligned16(a.ds) && aligned16(a.s) && aligned16(a.y) && aligned16(a.dx) && aligned16(a.dres)
               ? ALIGNED
               : OVERLAP;
}
// calls f with std::integral_constant of the column kind
template <typename F>
static int with_cols(Cols c, F f) {
    if (c == ALIGNED) return f(std::integral_constant<int, ALIGNED>());
    if (c == OVERLAP) return f(std::integral_constant<int, OVERLAP>());
    return f(std::integral_constant<int, SHORT>());
}
template <typename T, int COLS, bool RES>
static void ln_fwd_launch(const NormArgs& a, const Drop& d, const Form& f, unsigned g, hipStream_t st) {
    if (f.nt == 64 && f.nv == 1) ln_fwd_k<T, 1, 64, 1, COLS, RES><<<g, 256, 0, st>>>(a, d);
    else if (f.nt == 512) ln_fwd_k<T, 1, 512, 1, COLS, RES><<<g, 512, 0, st>>>(a, d);
    else if constexpr (COLS != SHORT) {              // (a row of less than a pack takes one of the two above)
        if (f.nt == 64) ln_fwd_k<T, 2, 64, 1, COLS, RES><<<g, 256, 0, st>>>(a, d);
        else if (f.nt == 256) ln_fwd_k<T, 1, 256, 2, COLS, RES><<<g, 512, 0, st>>>(a, d);
        else if (f.nv == 1) ln_fwd_k<T, 1, 1024, 1, COLS, RES><<<g, 1024, 0, st>>>(a, d);
        else ln_fwd_k<T, 2, 1024, 1, COLS, RES><<<g, 1024, 0, st>>>(a, d);
    }
}
template <typename T, int COLS, bool RES>
static void ln_bwd_launch(const NormArgs& a, const Drop& d, const Form& f, unsigned g, hipStream_t st) {
    if (f.nt == 64 && f.nv == 1) ln_bwd_k<T, 1, 64, 1, COLS, RES><<<g, 256, 0, st>>>(a, d);
    else if (f.nt == 512) ln_bwd_k<T, 1, 512, 1, COLS, RES><<<g, 512, 0, st>>>(a, d);
    else if constexpr (COLS != SHORT) {
        if (f.nt == 128) ln_bwd_k<T, 1, 128, 4, COLS, RES><<<g, 512, 0, st>>>(a, d);
        else if (f.nt == 256) ln_bwd_k<T, 1, 256, 2, COLS, RES><<<g, 512, 0, st>>>(a, d);
        else if (f.nv == 1) ln_bwd_k<T, 1, 1024, 1, COLS, RES><<<g, 1024, 0, st>>>(a, d);
        else if constexpr (sizeof(T) == 4) ln_bwd_k<T, 2, 1024, 1, COLS, RES><<<g, 1024, 0, st>>>(a, d);
    }
}
static unsigned grid_y(long n) { return (unsigned)(n < 65535 ? n : 65535); }

static int ln_fwd(const char* what, NormArgs a, const Drop& d, bool res, int type, void* ws, size_t ws_bytes,
                  hipStream_t st) {
    if (int rc = ln_check_ws(what, ln_ws_bytes(a.rows, a.C, a.ldx, type, 0), ws, ws_bytes)) return rc;
    const Form f = ln_form(a.C, a.ldx, type, false);
    a.lg = f.lg;
    return with_type(type, [&](auto* t) {
        typedef typename std::remove_reference<decltype(*t)>::type T;
        return with_cols(ln_cols(a, type), [&](auto kind) {
            constexpr int COLS = decltype(kind)::value;
            if (f.nt) {
                const unsigned g = (unsigned)ln_blocks(a.rows, f, false);
                if (res) ln_fwd_launch<T, COLS, true>(a, d, f, g, st);
                else ln_fwd_launch<T, COLS, false>(a, d, f, g, st);
            } else if constexpr (COLS != SHORT) {
                const SplitPlan sp = split_plan(a.C, sizeof(T));
                const dim3 gs((unsigned)sp.chunks, grid_y(a.rows)), ga((unsigned)sp.tiles, grid_y(a.rows));
                Chunk* c = (Chunk*)ws;
                if (res) ln_split_stats_k<T, COLS, true, false><<<gs, 256, 0, st>>>(a, d, c);
                else ln_split_stats_k<T, COLS, false, false><<<gs, 256, 0, st>>>(a, d, c);
                SIV_CHECK_LAUNCH(what);
                ln_split_fwd_k<T, COLS><<<ga, 256, 0, st>>>(a, c);
            }
            SIV_CHECK_LAUNCH(what);
            return SIV_OK;
        });
    });
}
static int ln_bwd(const char* what, NormArgs a, const Drop& d, bool res, int type, void* ws, size_t ws_bytes,
                  hipStream_t st) {
    if (int rc = ln_check_ws(what, ln_ws_bytes(a.rows, a.C, std::max(a.ldx, a.lddy), type, 1), ws, ws_bytes)) return rc;
    const Form f = ln_form(a.C, std::max(a.ldx, a.lddy), type, true);
    a.lg = f.lg;
    return with_type(type, [&](auto* t) {
        typedef typename std::remove_reference<decltype(*t)>::type T;
        return with_cols(ln_cols(a, type), [&](auto kind) {
            constexpr int COLS = decltype(kind)::value;
            long parts = 1;
            if (f.nt) {
                parts = ln_blocks(a.rows, f, true);
                a.part = (float*)ws;
                if (res) ln_bwd_launch<T, COLS, true>(a, d, f, (unsigned)parts, st);
                else ln_bwd_launch<T, COLS, false>(a, d, f, (unsigned)parts, st);
            } else if constexpr (COLS != SHORT) {
                const SplitPlan sp = split_plan(a.C, sizeof(T));
                Chunk* c = (Chunk*)ws;
                a.part = (float*)((char*)ws + align256((size_t)a.rows * sp.chunks * sizeof(Chunk)));
                parts = ln_split_parts(a.rows, sp);
                const dim3 gs((unsigned)sp.chunks, grid_y(a.rows)), ga((unsigned)sp.tiles, (unsigned)parts);
                ln_split_stats_k<T, COLS, false, true><<<gs, 256, 0, st>>>(a, d, c);
                SIV_CHECK_LAUNCH(what);
                ln_split_bwd_k<T, COLS><<<ga, 256, 0, st>>>(a, d, c);
            }
            SIV_CHECK_LAUNCH(what);
            if ((a.dw || a.db) && parts > 1) {
                // threads down a column: a few additions each, but enough blocks (768 x 128 sums: 4.9 us with 64; 21 x
                // 200000: 6 us with 4, 30 with 64)
                const float* p = a.part;
                const int down = parts <= 32 ? 4 : parts <= 256 || a.C >= 4096 ? 16 : 64;
                const unsigned g = (unsigned)cdiv(2 * a.C * down, 1024);
                if (down == 4) ln_param_sum_k<T, 4><<<g, 1024, 0, st>>>(p, parts, a);
                else if (down == 16) ln_param_sum_k<T, 16><<<g, 1024, 0, st>>>(p, parts, a);
                else ln_param_sum_k<T, 64><<<g, 1024, 0, st>>>(p, parts, a);
                SIV_CHECK_LAUNCH(what);
            }
            return SIV_OK;
        });
    });
}

}  // namespace siv

using namespace siv;

extern "C" int siv_layer_norm_workspace(long rows, long C, int type, int backward, size_t* bytes) {
    SIV_CHECK_ARG(bytes && rows > 0 && C > 0 && known_type(type), "layer_norm_workspace: bad argument");
    // (rows far apart take another kernel: enough for both)
    *bytes = std::max(ln_ws_bytes(rows, C, C, type, backward), ln_ws_bytes(rows, C, 1L << 40, type, backward));
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
    return ln_bwd("layer_norm_bwd", a, make_drop(nullptr, 0, 0, nullptr, 0.f), false, type, ws, ws_bytes,
                  (hipStream_t)stream);
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
    return ln_bwd("add_layer_norm_bwd", a, make_drop(keep, seed, stream_id, epoch, p), true, type, ws, ws_bytes,
                  (hipStream_t)stream);
}
