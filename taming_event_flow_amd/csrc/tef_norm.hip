// tef_norm.hip — layer normalisation over one axis, fused with what follows it in a normalised layer:
//
//   mean = sum_c x / C,  rstd = 1 / sqrt(sum_c (x - mean)^2 / C + eps),  u = (x - mean) * rstd
//   z = u * weight[c] + bias[c] (+ residual),  y = act(z)
//
// and the gradients, with g = dy * act'(z), h = g * weight:
//
//   dx = rstd * (h - sum_c h / C - u * sum_c (h * u) / C),  dresidual = g
//   dweight[c] = sum_rows g * u,  dbias[c] = sum_rows g
//
// x is [outer][C][inner], normalised over C: inner = 1 are rows (tokens, channels-last maps), inner > 1 the feature maps of
// this package's networks.  Bound by memory: the forward pass reads x (and residual) once and writes y once, the backward
// pass reads x, dy (and residual where the activation needs z) once and writes dx (and dresidual) once; a row's values stay
// in registers between its sums and its results.  Sums and statistics are fp32: a lane adds its own elements, then lanes
// and waves are joined in a fixed order.  The variance is taken of d = x - mean, not as a difference of large moments, and the mean of d,
// the mean's own rounding, is taken off d (its sum rides on the join of the variance's): a constant row gives exactly the bias, and a mean far
// larger than the spread costs the forward pass nothing.  The mean that the backward pass gets is that one rounded to fp32.  z is
// formed again in the backward pass instead of being derived from the rounded y: 1 - y^2 of a half-precision y near 1 has
// no correct digit.  The sums over rows (dweight, dbias) go through one partial row per workgroup and a second launch that
// adds those in a fixed order: bit-for-bit reproducible, no atomics.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tef.h"
#include "tef_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 1024;       // persistent workgroups of a backward pass = partial rows of dweight / dbias

template <typename T> __device__ inline float to_f(T v);
template <> __device__ inline float to_f<float>(float v) { return v; }
template <> __device__ inline float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ inline float to_f<__hip_bfloat16>(__hip_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ inline T from_f(float v);
template <> __device__ inline float from_f<float>(float v) { return v; }
template <> __device__ inline __half from_f<__half>(float v) { return __float2half(v); }                          // nearest even
template <> __device__ inline __hip_bfloat16 from_f<__hip_bfloat16>(float v) { return __float2bfloat16(v); }      // nearest even

// V consecutive elements; the address is a multiple of the ELEMENT's size only (views, odd row lengths): gfx950's global
// loads take that, in one instruction.
template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[V]; };
template <typename T, int V> __device__ inline Pack<T, V> raw(const T *p) { return *reinterpret_cast<const Pack<T, V> *>(p); }
template <typename T, int V> __device__ inline void store(T *p, const float (&f)[V])
{
    Pack<T, V> q;
#pragma unroll
    for (int k = 0; k < V; ++k) q.v[k] = from_f<T>(f[k]);
    *reinterpret_cast<Pack<T, V> *>(p) = q;
}
// Elements c .. c + V - 1 of a row of C: no branch around the load, so that all packs of a row are in flight together — what
// lies past the row's end is read at its last element and set to 0 by the caller.  EVEN: C is a multiple of V.
template <typename T, int V, bool EVEN> __device__ inline Pack<T, V> raw_row(const T *row, int c, int C)
{
    if (EVEN) return raw<T, V>(row + (c < C ? c : C - V));
    Pack<T, V> q;
#pragma unroll
    for (int k = 0; k < V; ++k) q.v[k] = row[c + k < C ? c + k : C - 1];
    return q;
}
template <typename T, int V, bool EVEN> __device__ inline void store_row(T *row, int c, int C, const float (&f)[V])
{
    if (EVEN) {
        if (c < C) store<T, V>(row + c, f);
        return;
    }
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (c + k < C) row[c + k] = from_f<T>(f[k]);
}

struct Vecs {            // weight and bias (either may be missing) in one of the three types
    const void *w, *b;
    int dtype;
};
__device__ inline float vec_at(const void *p, int dtype, int c, float missing)
{
    if (!p) return missing;
    if (dtype == TEF_F32) return reinterpret_cast<const float *>(p)[c];
    if (dtype == TEF_F16) return __half2float(reinterpret_cast<const __half *>(p)[c]);
    return __bfloat162float(reinterpret_cast<const __hip_bfloat16 *>(p)[c]);
}
__device__ inline void vec_put(void *p, int dtype, int c, float v)
{
    if (dtype == TEF_F32) reinterpret_cast<float *>(p)[c] = v;
    else if (dtype == TEF_F16) reinterpret_cast<__half *>(p)[c] = __float2half(v);
    else reinterpret_cast<__hip_bfloat16 *>(p)[c] = __float2bfloat16(v);
}

__device__ inline float act(int a, float z)
{
    if (a == TEF_ACT_NONE) return z;
    if (a == TEF_ACT_RELU) return z > 0.0f || z != z ? z : 0.0f;      // (NaN stays NaN)
    if (a == TEF_ACT_TANH) return tanhf(z);
    return 1.0f / (1.0f + expf(-z));
}
__device__ inline float act_slope(int a, float z)
{
    if (a == TEF_ACT_NONE) return 1.0f;
    if (a == TEF_ACT_RELU) return z > 0.0f ? 1.0f : z != z ? z : 0.0f;
    if (a == TEF_ACT_TANH) { const float y = tanhf(z); return 1.0f - y * y; }
    const float y = 1.0f / (1.0f + expf(-z));
    return y * (1.0f - y);
}

struct Args {
    const void *x, *res, *dy;
    void *y, *dx, *dres;
    float *mean, *rstd, *part;       // part: [workgroups][2][C] partial sums of dweight, dbias
    Vecs v;
    long rows;                       // outer * inner
    long inner;
    int C, act;
    float eps;
};

// ---- rows: C contiguous --------------------------------------------------------------------------------------------------
// A row belongs to L lanes (a power of two, at most one wave: no barrier, several short rows a wave) or, WG, to the whole
// workgroup.  Lane l holds the elements V * (l + L * i) .. + V - 1, i < NV, in registers, and keeps the weights of its
// columns over all rows that it takes.  4096 x 4096 bf16: 30 us forward, 42 backward (2.2, 2.4 TB/s; one row a workgroup at a time,
// two joins of its waves each: latency, hidden by eight workgroups a CU).  Rows that are no multiple of 4 are loaded by the element: 8192 x 8191
// f32 592 us forward and backward (x 8188: 347; 19 of the backward pass's registers do not fit), in the form below, x 8193, 1092.
constexpr int V = 4;

template <bool WG> __device__ inline float row_sum(float s, int L, float *red)
{
    for (int o = (WG ? 64 : L) >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (WG) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
        __syncthreads();
        s = (red[0] + red[1]) + (red[2] + red[3]);
    }
    return s;
}

// the same of two sums at once
template <bool WG> __device__ inline void row_sums(float &s, float &q, int L, float *red)
{
    for (int o = (WG ? 64 : L) >> 1; o > 0; o >>= 1) {
        s += __shfl_xor(s, o, 64);
        q += __shfl_xor(q, o, 64);
    }
    if (WG) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = s; red[4 + (threadIdx.x >> 6)] = q; }
        __syncthreads();
        s = (red[0] + red[1]) + (red[2] + red[3]);
        q = (red[4] + red[5]) + (red[6] + red[7]);
    }
}
// 1 / sqrt(v), within a unit of its last bit: the error of the two roundings of 1.0f / sqrtf(v), r, taken off once.  (0, inf and NaN as they come.)
__device__ inline float inverse_root(float v)
{
    const float r = 1.0f / sqrtf(v), h = v * r, low = fmaf(v, r, -h), off = fmaf(-h, r, 1.0f) - low * r;      // 1 - v r^2
    return fabsf(off) < 1.0f ? fmaf(0.5f * r, off, r) : r;
}
// sums of d and d^2 -> 1 / sqrt(variance + eps), the correction of the mean times that (and the mean corrected): u = d rstd - by in one rounding
// (inv = 1 / C: products, not divisions, which cost the widest maps a tenth of their time; what a product adds to the first mean is
// corrected here with the rest of it)
__device__ inline float correct(float &mean, float sd, float sq, float inv, float eps, float &rstd)
{
    const float by = sd * inv, var = (sq - sd * by) * inv;
    rstd = inverse_root((var < 0.0f ? 0.0f : var) + eps);      // (NaN stays NaN)
    mean += by;
    return by * rstd;
}

template <int NV> __device__ inline void row_vec(const void *p, int dtype, int l, int L, int C, float missing, float (&f)[NV][V])
{
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = V * (l + L * i) + k;
            f[i][k] = vec_at(p, dtype, c < C ? c : C - 1, missing);
        }
}

template <typename T, int NV, bool WG, bool EVEN> __global__ __launch_bounds__(kThreads) void rows_fwd(Args a, int L)
{
    __shared__ float red[2 * kThreads / 64];
    const int l = WG ? threadIdx.x : threadIdx.x & (L - 1), per = WG ? 1 : kThreads / L, C = a.C;
    const float inv = 1.0f / (float)C;
    float w[NV][V], b[NV][V];
    row_vec<NV>(a.v.w, a.v.dtype, l, L, C, 1.0f, w);
    row_vec<NV>(a.v.b, a.v.dtype, l, L, C, 0.0f, b);
    for (long r0 = (long)blockIdx.x * per; r0 < a.rows; r0 += (long)gridDim.x * per) {
        const long r = WG ? r0 : r0 + threadIdx.x / L;
        const bool live = r < a.rows;
        const long at = (live ? r : a.rows - 1) * C;
        Pack<T, V> q[NV], e[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) q[i] = raw_row<T, V, EVEN>(reinterpret_cast<const T *>(a.x) + at, V * (l + L * i), C);
        if (a.res)
#pragma unroll
            for (int i = 0; i < NV; ++i) e[i] = raw_row<T, V, EVEN>(reinterpret_cast<const T *>(a.res) + at, V * (l + L * i), C);
        float f[NV][V], s = 0.0f, v = 0.0f, d = 0.0f, rstd;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int k = 0; k < V; ++k) f[i][k] = V * (l + L * i) + k < C ? to_f<T>(q[i].v[k]) : 0.0f;
            s += (f[i][0] + f[i][1]) + (f[i][2] + f[i][3]);
        }
        float mean = row_sum<WG>(s, L, red) * inv;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const bool in = V * (l + L * i) + k < C;
                f[i][k] -= mean;
                d += in ? f[i][k] : 0.0f;
                v += in ? f[i][k] * f[i][k] : 0.0f;
            }
        row_sums<WG>(d, v, L, red);
        const float by = correct(mean, d, v, inv, a.eps, rstd);
        if (!live) continue;
        if (l == 0 && a.mean) { a.mean[r] = mean; a.rstd[r] = rstd; }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int k = 0; k < V; ++k)
                f[i][k] = act(a.act, fmaf(fmaf(f[i][k], rstd, -by), w[i][k], b[i][k]) + (a.res ? to_f<T>(e[i].v[k]) : 0.0f));
            store_row<T, V, EVEN>(reinterpret_cast<T *>(a.y) + at, V * (l + L * i), C, f[i]);
        }
    }
}

template <typename T, int NV, bool WG, bool EVEN> __global__ __launch_bounds__(kThreads) void rows_bwd(Args a, int L)
{
    __shared__ float red[kThreads / 64];
    __shared__ float cols[WG ? 1 : kThreads * V];
    const int l = WG ? threadIdx.x : threadIdx.x & (L - 1), per = WG ? 1 : kThreads / L, C = a.C;
    const float inv = 1.0f / (float)C;
    const bool need_z = a.act != TEF_ACT_NONE, need_e = need_z && a.res;
    float w[NV][V], b[NV][V], dw[NV][V], db[NV][V];
    row_vec<NV>(a.v.w, a.v.dtype, l, L, C, 1.0f, w);
    row_vec<NV>(need_z ? a.v.b : nullptr, a.v.dtype, l, L, C, 0.0f, b);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) dw[i][k] = db[i][k] = 0.0f;
    for (long r0 = (long)blockIdx.x * per; r0 < a.rows; r0 += (long)gridDim.x * per) {
        const long r = WG ? r0 : r0 + threadIdx.x / L;
        const bool live = r < a.rows;
        const long row = live ? r : a.rows - 1, at = row * C;
        Pack<T, V> qx[NV], qd[NV], qe[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            qx[i] = raw_row<T, V, EVEN>(reinterpret_cast<const T *>(a.x) + at, V * (l + L * i), C);
            qd[i] = raw_row<T, V, EVEN>(reinterpret_cast<const T *>(a.dy) + at, V * (l + L * i), C);
        }
        if (need_e)
#pragma unroll
            for (int i = 0; i < NV; ++i) qe[i] = raw_row<T, V, EVEN>(reinterpret_cast<const T *>(a.res) + at, V * (l + L * i), C);
        const float mean = a.mean[row], rstd = a.rstd[row];
        float u[NV][V], h[NV][V], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float e[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const bool in = live && V * (l + L * i) + k < C;
                u[i][k] = in ? (to_f<T>(qx[i].v[k]) - mean) * rstd : 0.0f;
                float g = in ? to_f<T>(qd[i].v[k]) : 0.0f;
                if (need_z && in) g *= act_slope(a.act, fmaf(u[i][k], w[i][k], b[i][k]) + (need_e ? to_f<T>(qe[i].v[k]) : 0.0f));
                e[k] = g;
                dw[i][k] += g * u[i][k];
                db[i][k] += g;
                h[i][k] = g * w[i][k];
                s1 += h[i][k];
                s2 += h[i][k] * u[i][k];
            }
            if (a.dres && live) store_row<T, V, EVEN>(reinterpret_cast<T *>(a.dres) + at, V * (l + L * i), C, e);
        }
        if (!a.dx) continue;
        s1 = row_sum<WG>(s1, L, red) * inv;
        s2 = row_sum<WG>(s2, L, red) * inv;
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float e[V];
#pragma unroll
            for (int k = 0; k < V; ++k) e[k] = rstd * fmaf(-u[i][k], s2, h[i][k] - s1);
            store_row<T, V, EVEN>(reinterpret_cast<T *>(a.dx) + at, V * (l + L * i), C, e);
        }
    }
    if (!a.part) return;
    float *part = a.part + (long)blockIdx.x * 2 * C;
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = V * (l + L * i);
            if (WG) {
#pragma unroll
                for (int k = 0; k < V; ++k)
                    if (c + k < C) part[which * C + c + k] = which ? db[i][k] : dw[i][k];
            } else {      // the row groups of the workgroup, in order
                __syncthreads();
#pragma unroll
                for (int k = 0; k < V; ++k) cols[threadIdx.x * V + k] = which ? db[i][k] : dw[i][k];
                __syncthreads();
                if ((int)threadIdx.x < L)
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        float s = 0.0f;
                        for (int g = 0; g < per; ++g) s += cols[(g * L + l) * V + k];
                        if (c + k < C) part[which * C + c + k] = s;
                    }
            }
        }
}

// ---- maps: the channels of a position lie `inner` elements apart --------------------------------------------------------
// A workgroup takes LX * P neighbouring positions (P per lane: 4 when inner is a multiple of 4, so that a lane's positions
// are one load; else 1) and all channels: lane group g of G = 256 / LX holds the channels g, g + G, ... in registers.
// 80 x 32 x 128 x 128 f32 with tanh: 81 us forward, 110 backward (4.1, 4.6 TB/s of a copy's 4.9).
// A thread holds up to 64 values, one position at a time up to 16: 64 channels do not fit the register file (the backward pass spilled 789
// registers), and 32 leave one wave a SIMD: 32 x 256 x 61 x 63 f32 takes 927 us forward and backward with up to 64, 396 with up to 32, 268 with
// up to 16 (x 257: 1280, 578, 416).  Past 4096 channels, where a workgroup has one position, up to 32 are better than 16 with a
// second read of everything (20 x 4097 x 15 x 15: 792 against 1600); past 8192 they are read again (8 x 16000 x 9 x 9: 891, with 64 of them 750).
template <int P> __device__ inline void map_sum(float (&s)[P], int LX, float *red)      // over the lane groups
{
    const int lx = threadIdx.x & (LX - 1), wave = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < P; ++k)
        for (int o = 32; o >= LX; o >>= 1) s[k] += __shfl_xor(s[k], o, 64);
    __syncthreads();
    if ((int)(threadIdx.x & 63) < LX)
#pragma unroll
        for (int k = 0; k < P; ++k) red[(wave * LX + lx) * P + k] = s[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < P; ++k)
        s[k] = (red[lx * P + k] + red[(LX + lx) * P + k]) + (red[(2 * LX + lx) * P + k] + red[(3 * LX + lx) * P + k]);
}

// Second sums of a tile's positions, of d = x - mean and d^2: by[k] what the mean is corrected by, times rstd[k]; position j of the tile is
// finished by thread j alone (all threads for themselves: 103 us instead of 81 for the map above) and, if asked for, stored.
// red: the partial sums that the mean was made of, then room for 3 * 256.
template <int P>
__device__ inline void map_stats(const float (&d)[P], const float (&q)[P], float (&by)[P], float (&rstd)[P], int LX, float *red, float inv,
                                 float eps, float *mean_out, float *rstd_out, long at, long rows)
{
    const int lx = threadIdx.x & (LX - 1), wave = threadIdx.x >> 6, j = threadIdx.x, n = LX * P;
    float *rd = red + 256, *rq = red + 512, *out = red + 768;
    float sd[P], sq[P];
#pragma unroll
    for (int k = 0; k < P; ++k) {
        sd[k] = d[k];
        sq[k] = q[k];
        for (int o = 32; o >= LX; o >>= 1) {
            sd[k] += __shfl_xor(sd[k], o, 64);
            sq[k] += __shfl_xor(sq[k], o, 64);
        }
    }
    if ((int)(threadIdx.x & 63) < LX)
#pragma unroll
        for (int k = 0; k < P; ++k) {
            rd[wave * n + lx * P + k] = sd[k];
            rq[wave * n + lx * P + k] = sq[k];
        }
    __syncthreads();
    if (j < n) {
        float mean = ((red[j] + red[n + j]) + (red[2 * n + j] + red[3 * n + j])) * inv, r;
        out[j] = correct(mean, (rd[j] + rd[n + j]) + (rd[2 * n + j] + rd[3 * n + j]), (rq[j] + rq[n + j]) + (rq[2 * n + j] + rq[3 * n + j]), inv, eps, r);
        out[64 + j] = r;
        if (mean_out && at + j < rows) { mean_out[at + j] = mean; rstd_out[at + j] = r; }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < P; ++k) { by[k] = out[lx * P + k]; rstd[k] = out[64 + lx * P + k]; }
}

template <typename T, int NC, int P> __global__ __launch_bounds__(kThreads) void maps_fwd(Args a, int LX)
{
    __shared__ __attribute__((aligned(16))) float red[3 * 256 + 128];      // (a tile has at most 64 positions)
    const int lx = threadIdx.x & (LX - 1), g = threadIdx.x / LX, G = kThreads / LX, C = a.C;
    const float inv = 1.0f / (float)C;
    const long tile = (long)LX * P;
    float w[NC], b[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = g + G * i < C ? g + G * i : C - 1;
        w[i] = vec_at(a.v.w, a.v.dtype, c, 1.0f);
        b[i] = vec_at(a.v.b, a.v.dtype, c, 0.0f);
    }
    for (long t = blockIdx.x; t * tile < a.rows; t += gridDim.x) {
        const bool live = t * tile + (long)lx * P < a.rows;
        const long pos = live ? t * tile + (long)lx * P : a.rows - P;
        const long o = pos / a.inner, at = o * C * a.inner + (pos - o * a.inner);
        Pack<T, P> q[NC], e[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) q[i] = raw<T, P>(reinterpret_cast<const T *>(a.x) + at + (g + G * i < C ? g + G * i : C - 1) * a.inner);
        if (a.res)
#pragma unroll
            for (int i = 0; i < NC; ++i) e[i] = raw<T, P>(reinterpret_cast<const T *>(a.res) + at + (g + G * i < C ? g + G * i : C - 1) * a.inner);
        float f[NC][P], s[P], v[P], d[P], by[P], rstd[P];
#pragma unroll
        for (int k = 0; k < P; ++k) s[k] = v[k] = d[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int k = 0; k < P; ++k) {
                f[i][k] = to_f<T>(q[i].v[k]);
                s[k] += g + G * i < C ? f[i][k] : 0.0f;
            }
        map_sum<P>(s, LX, red);
#pragma unroll
        for (int k = 0; k < P; ++k) s[k] *= inv;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int k = 0; k < P; ++k) {
                f[i][k] -= s[k];
                d[k] += g + G * i < C ? f[i][k] : 0.0f;
                v[k] += g + G * i < C ? f[i][k] * f[i][k] : 0.0f;
            }
        map_stats<P>(d, v, by, rstd, LX, red, inv, a.eps, a.mean, a.rstd, t * tile, a.rows);
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = g + G * i;
            if (c >= C) continue;
#pragma unroll
            for (int k = 0; k < P; ++k) f[i][k] = act(a.act, fmaf(fmaf(f[i][k], rstd[k], -by[k]), w[i], b[i]) + (a.res ? to_f<T>(e[i].v[k]) : 0.0f));
            store<T, P>(reinterpret_cast<T *>(a.y) + at + c * a.inner, f[i]);
        }
    }
}

template <typename T, int NC, int P> __global__ __launch_bounds__(kThreads) void maps_bwd(Args a, int LX)
{
    __shared__ float red[256];
    const int lx = threadIdx.x & (LX - 1), g = threadIdx.x / LX, G = kThreads / LX, C = a.C;
    const float inv = 1.0f / (float)C;
    const bool need_z = a.act != TEF_ACT_NONE, need_e = need_z && a.res;
    const long tile = (long)LX * P;
    float w[NC], b[NC], dw[NC], db[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = g + G * i < C ? g + G * i : C - 1;
        w[i] = vec_at(a.v.w, a.v.dtype, c, 1.0f);
        b[i] = need_z ? vec_at(a.v.b, a.v.dtype, c, 0.0f) : 0.0f;
        dw[i] = db[i] = 0.0f;
    }
    for (long t = blockIdx.x; t * tile < a.rows; t += gridDim.x) {
        const bool live = t * tile + (long)lx * P < a.rows;
        const long pos = live ? t * tile + (long)lx * P : a.rows - P;
        const long o = pos / a.inner, at = o * C * a.inner + (pos - o * a.inner);
        Pack<T, P> qx[NC], qd[NC], qe[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const long off = at + (g + G * i < C ? g + G * i : C - 1) * a.inner;
            qx[i] = raw<T, P>(reinterpret_cast<const T *>(a.x) + off);
            qd[i] = raw<T, P>(reinterpret_cast<const T *>(a.dy) + off);
        }
        if (need_e)
#pragma unroll
            for (int i = 0; i < NC; ++i) qe[i] = raw<T, P>(reinterpret_cast<const T *>(a.res) + at + (g + G * i < C ? g + G * i : C - 1) * a.inner);
        const Pack<float, P> mean = raw<float, P>(a.mean + pos), rstd = raw<float, P>(a.rstd + pos);
        float u[NC][P], h[NC][P], s1[P], s2[P];
#pragma unroll
        for (int k = 0; k < P; ++k) s1[k] = s2[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const bool in = live && g + G * i < C;
#pragma unroll
            for (int k = 0; k < P; ++k) {
                u[i][k] = in ? (to_f<T>(qx[i].v[k]) - mean.v[k]) * rstd.v[k] : 0.0f;
                h[i][k] = in ? to_f<T>(qd[i].v[k]) : 0.0f;
                if (need_z && in) h[i][k] *= act_slope(a.act, fmaf(u[i][k], w[i], b[i]) + (need_e ? to_f<T>(qe[i].v[k]) : 0.0f));
            }
            if (a.dres && in) store<T, P>(reinterpret_cast<T *>(a.dres) + at + (g + G * i) * a.inner, h[i]);
#pragma unroll
            for (int k = 0; k < P; ++k) {
                dw[i] += h[i][k] * u[i][k];
                db[i] += h[i][k];
                h[i][k] *= w[i];
                s1[k] += h[i][k];
                s2[k] += h[i][k] * u[i][k];
            }
        }
        if (!a.dx) continue;
        map_sum<P>(s1, LX, red);
        map_sum<P>(s2, LX, red);
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = g + G * i;
            if (c >= C) continue;
            float e[P];
#pragma unroll
            for (int k = 0; k < P; ++k) e[k] = rstd.v[k] * fmaf(-u[i][k], s2[k] * inv, fmaf(-inv, s1[k], h[i][k]));
            store<T, P>(reinterpret_cast<T *>(a.dx) + at + c * a.inner, e);
        }
    }
    if (!a.part) return;
    float *part = a.part + (long)blockIdx.x * 2 * C;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        for (int o2 = LX >> 1; o2 > 0; o2 >>= 1) {
            dw[i] += __shfl_xor(dw[i], o2, 64);
            db[i] += __shfl_xor(db[i], o2, 64);
        }
        const int c = g + G * i;
        if (lx == 0 && c < C) { part[c] = dw[i]; part[C + c] = db[i]; }
    }
}

// ---- any C: one workgroup per position, the row read again for every sum ------------------------------------------------
// For rows and channel counts that do not fit into the registers of a workgroup.
// Sums are 64 bits: a thread alone adds up to 2^22 values, of which fp32 would drop the last ones' lower half.
__device__ inline double long_sum(double s, double *red)
{
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

template <typename T> __global__ __launch_bounds__(kThreads) void long_fwd(Args a)
{
    __shared__ double red[kThreads / 64];
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const long o = r / a.inner, at = o * a.C * a.inner + (r - o * a.inner);
        const T *x = reinterpret_cast<const T *>(a.x) + at;
        double s = 0.0, q = 0.0;
        for (int c = threadIdx.x; c < a.C; c += kThreads) s += to_f<T>(x[(long)c * a.inner]);
        const double mean = long_sum(s, red) / a.C;
        for (int c = threadIdx.x; c < a.C; c += kThreads) {
            const double d = to_f<T>(x[(long)c * a.inner]) - mean;
            q += d * d;
        }
        const float rstd = (float)(1.0 / sqrt(long_sum(q, red) / a.C + (double)a.eps));
        if (threadIdx.x == 0 && a.mean) { a.mean[r] = (float)mean; a.rstd[r] = rstd; }
        for (int c = threadIdx.x; c < a.C; c += kThreads) {
            const long off = at + (long)c * a.inner;
            const float e = a.res ? to_f<T>(reinterpret_cast<const T *>(a.res)[off]) : 0.0f;
            const float u = (float)(to_f<T>(reinterpret_cast<const T *>(a.x)[off]) - mean) * rstd;
            const float z = fmaf(u, vec_at(a.v.w, a.v.dtype, c, 1.0f), vec_at(a.v.b, a.v.dtype, c, 0.0f)) + e;
            reinterpret_cast<T *>(a.y)[off] = from_f<T>(act(a.act, z));
        }
    }
}

template <typename T> __device__ inline float long_g(const Args &a, long off, int c, float mean, float rstd, float *u)
{
    *u = (to_f<T>(reinterpret_cast<const T *>(a.x)[off]) - mean) * rstd;
    float g = to_f<T>(reinterpret_cast<const T *>(a.dy)[off]);
    if (a.act != TEF_ACT_NONE) {
        const float e = a.res ? to_f<T>(reinterpret_cast<const T *>(a.res)[off]) : 0.0f;
        g *= act_slope(a.act, fmaf(*u, vec_at(a.v.w, a.v.dtype, c, 1.0f), vec_at(a.v.b, a.v.dtype, c, 0.0f)) + e);
    }
    return g;
}

template <typename T> __global__ __launch_bounds__(kThreads) void long_bwd(Args a)
{
    __shared__ double red[kThreads / 64];
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const long o = r / a.inner, at = o * a.C * a.inner + (r - o * a.inner);
        const float mean = a.mean[r], rstd = a.rstd[r];
        double t1 = 0.0, t2 = 0.0;
        float u;
        for (int c = threadIdx.x; c < a.C; c += kThreads) {
            const long off = at + (long)c * a.inner;
            const float g = long_g<T>(a, off, c, mean, rstd, &u), h = g * vec_at(a.v.w, a.v.dtype, c, 1.0f);
            t1 += h;
            t2 += h * u;
            if (a.dres) reinterpret_cast<T *>(a.dres)[off] = from_f<T>(g);
            if (a.part) {      // this thread is the only one of the workgroup at channel c
                float *p = a.part + (long)blockIdx.x * 2 * a.C + c;
                const bool first = r == (long)blockIdx.x;
                p[0] = (first ? 0.0f : p[0]) + g * u;
                p[a.C] = (first ? 0.0f : p[a.C]) + g;
            }
        }
        if (!a.dx) continue;
        const float s1 = (float)(long_sum(t1, red) / a.C), s2 = (float)(long_sum(t2, red) / a.C);
        for (int c = threadIdx.x; c < a.C; c += kThreads) {
            const long off = at + (long)c * a.inner;
            const float h = long_g<T>(a, off, c, mean, rstd, &u) * vec_at(a.v.w, a.v.dtype, c, 1.0f);
            reinterpret_cast<T *>(a.dx)[off] = from_f<T>(rstd * fmaf(-u, s2, h - s1));
        }
    }
}

// dweight / dbias = the sum of the workgroups' partial rows: 64 columns a workgroup of 16 waves, wave k takes the rows k, k + 16,
// ..., eight of them in flight (a partial row comes from another XCD's L2: latency is all there is), joined in a fixed order.
constexpr int kJoinWaves = 16;
__global__ __launch_bounds__(64 * kJoinWaves) void norm_join(const float *__restrict__ part, int parts, int C, void *dw, void *db, int dtype)
{
    __shared__ float red[kJoinWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long cols = 2l * C;
    for (long c0 = blockIdx.x * 64l; c0 < cols; c0 += gridDim.x * 64l) {      // (one round, unless the columns outnumber a launch's threads)
        const long col = c0 + lane;
        float s[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = 0.0f;
        if (col < cols)
            for (int k = wave; k < parts; k += 8 * kJoinWaves) {
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = part[(k + kJoinWaves * j < parts ? k + kJoinWaves * j : parts - 1) * cols + col];
#pragma unroll
                for (int j = 0; j < 8; ++j) s[j] += k + kJoinWaves * j < parts ? f[j] : 0.0f;
            }
        __syncthreads();
        red[wave][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
        __syncthreads();
        if (wave == 0 && col < cols) {
            float v = 0.0f;
            for (int k = 0; k < kJoinWaves; ++k) v += red[k][lane];
            if (col < C) { if (dw) vec_put(dw, dtype, (int)col, v); }
            else if (db) vec_put(db, dtype, (int)(col - C), v);
        }
    }
}

__global__ __launch_bounds__(kThreads) void norm_zero(void *dw, void *db, int C, int dtype)
{
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= C) return;
    if (dw) vec_put(dw, dtype, c, 0.0f);
    if (db) vec_put(db, dtype, c, 0.0f);
}

// How a description is cut: which kernel, its register blocking, its grid.
struct Plan {
    int kind;          // 0 rows (lanes of a wave), 1 rows (workgroup), 2 maps, 3 long
    int n;             // NV or NC
    int lanes;         // L or LX
    int per;           // P (maps)
    long tiles;
};

inline int pow2_at_least(long v)
{
    int p = 1;
    while (p < v) p <<= 1;
    return p;
}

Plan make_plan(const tef_norm_desc &d)
{
    Plan p{};
    const long rows = (long)d.outer * d.inner;
    if (d.inner == 1) {
        const long packs = (d.channels + V - 1) / V;
        if (packs <= 64 * 8) {
            p.kind = 0;
            p.lanes = packs < 64 ? pow2_at_least(packs) : 64;
            p.n = pow2_at_least((packs + p.lanes - 1) / p.lanes);
            p.tiles = (rows + kThreads / p.lanes - 1) / (kThreads / p.lanes);
            return p;
        }
        if (packs <= kThreads * 8) {
            p.kind = 1;
            p.lanes = kThreads;
            p.n = pow2_at_least((packs + kThreads - 1) / kThreads);
            p.tiles = rows;
            return p;
        }
    } else {
        p.per = d.inner % 4 == 0 ? 4 : 1;
        // as many lanes along the positions as leave a thread at most 16 channels (long runs of memory per channel), then
        // fewer while the grid does not cover the 256 CUs and a thread still has more than one channel
        const int most = 16, last = p.per == 4 ? 16 : 32;      // ... with one lane along the positions: what the registers hold
        int lx = p.per == 4 ? 16 : 64;
        while (lx > 1 && (d.channels + kThreads / lx - 1) / (kThreads / lx) > most) lx >>= 1;
        while (lx > 1 && (rows + lx * p.per - 1) / (lx * p.per) < 256 && (long)d.channels * lx > kThreads) lx >>= 1;
        const int nc = (d.channels + kThreads / lx - 1) / (kThreads / lx);
        if (nc <= last) {
            p.kind = 2;
            p.lanes = lx;
            p.n = pow2_at_least(nc);
            p.tiles = (rows + (long)lx * p.per - 1) / ((long)lx * p.per);
            return p;
        }
    }
    p.kind = 3;
    p.tiles = rows;
    return p;
}

template <typename T, int N, bool WG> void go_rows(const Plan &p, bool bwd, dim3 grid, hipStream_t st, const Args &a)
{
    const dim3 block(kThreads);
    if (a.C % V == 0) {
        if (bwd) hipLaunchKernelGGL((rows_bwd<T, N, WG, true>), grid, block, 0, st, a, p.lanes);
        else hipLaunchKernelGGL((rows_fwd<T, N, WG, true>), grid, block, 0, st, a, p.lanes);
    } else {
        if (bwd) hipLaunchKernelGGL((rows_bwd<T, N, WG, false>), grid, block, 0, st, a, p.lanes);
        else hipLaunchKernelGGL((rows_fwd<T, N, WG, false>), grid, block, 0, st, a, p.lanes);
    }
}
template <typename T, int N, int P> void go_maps(const Plan &p, bool bwd, dim3 grid, hipStream_t st, const Args &a)
{
    if (bwd) hipLaunchKernelGGL((maps_bwd<T, N, P>), grid, dim3(kThreads), 0, st, a, p.lanes);
    else hipLaunchKernelGGL((maps_fwd<T, N, P>), grid, dim3(kThreads), 0, st, a, p.lanes);
}
template <typename T, int N> void go_n(const Plan &p, bool bwd, dim3 grid, hipStream_t st, const Args &a)
{
    if constexpr (N <= 8) {
        if (p.kind == 0) return go_rows<T, N, false>(p, bwd, grid, st, a);
        if constexpr (N > 2)      // (the workgroup form starts at 513 packs, three a thread)
            if (p.kind == 1) return go_rows<T, N, true>(p, bwd, grid, st, a);
    }
    if constexpr (N <= 16)
        if (p.kind == 2 && p.per == 4) return go_maps<T, N, 4>(p, bwd, grid, st, a);
    if (p.kind == 2 && p.per == 1) go_maps<T, N, 1>(p, bwd, grid, st, a);
}

template <typename T> void go(const Plan &p, bool bwd, dim3 grid, hipStream_t st, const Args &a)
{
    if (p.kind == 3) {
        if (bwd) hipLaunchKernelGGL(long_bwd<T>, grid, dim3(kThreads), 0, st, a);
        else hipLaunchKernelGGL(long_fwd<T>, grid, dim3(kThreads), 0, st, a);
        return;
    }
    switch (p.n) {
    case 1: go_n<T, 1>(p, bwd, grid, st, a); break;
    case 2: go_n<T, 2>(p, bwd, grid, st, a); break;
    case 4: go_n<T, 4>(p, bwd, grid, st, a); break;
    case 8: go_n<T, 8>(p, bwd, grid, st, a); break;
    case 16: go_n<T, 16>(p, bwd, grid, st, a); break;
    default: go_n<T, 32>(p, bwd, grid, st, a); break;
    }
}

void launch(const tef_norm_desc &d, const Plan &p, bool bwd, unsigned blocks, hipStream_t st, const Args &a)
{
    const dim3 grid(blocks);
    if (d.dtype == TEF_F32) go<float>(p, bwd, grid, st, a);
    else if (d.dtype == TEF_F16) go<__half>(p, bwd, grid, st, a);
    else go<__hip_bfloat16>(p, bwd, grid, st, a);
}

// (rows too long for the registers: fewer workgroups, since each has a partial row of that length in the workspace)
unsigned bwd_blocks(const Plan &p, int channels)
{
    long most = kMaxBlocks;
    if (p.kind == 3) {
        most = (1l << 23) / channels;
        most = most < 64 ? 64 : most > kMaxBlocks ? kMaxBlocks : most;
    }
    return (unsigned)(p.tiles < most ? p.tiles : most);
}

bool valid(const tef_norm_desc *d)
{
    if (!d) return tef::fail("layer norm: null description");
    // (a thread's channel number goes up to 256 past the last one: 32 bits)
    const bool ok = d->channels >= 1 && d->channels <= (1 << 30) && d->outer >= 0 && d->inner >= 1 && d->dtype >= TEF_F32 && d->dtype <= TEF_BF16 &&
                    (d->wdtype == TEF_F32 || d->wdtype == d->dtype) && d->act >= TEF_ACT_NONE && d->act <= TEF_ACT_SIGMOID &&
                    d->eps >= 0.0f && d->eps < 1e30f;
    if (!ok) return tef::fail("layer norm: invalid description (sizes, types, activation or eps)");
    const double n = (double)d->outer * (double)d->inner * (double)d->channels;
    if (n > 4e18) return tef::fail("layer norm: more elements than 64-bit offsets can address");
    return true;
}

}  // namespace

extern "C" {

int tef_layer_norm_forward(const tef_norm_desc *d, const void *x, const void *weight, const void *bias, const void *residual,
                           void *y, float *mean, float *rstd, void *stream)
{
    if (!valid(d)) return TEF_ERR_INVALID;
    if (d->outer == 0) return 0;
    if (!x || !y || (!mean != !rstd)) return tef::fail("tef_layer_norm_forward: null pointer"), TEF_ERR_INVALID;
    const Plan p = make_plan(*d);
    Args a{};
    a.x = x; a.res = residual; a.y = y; a.mean = mean; a.rstd = rstd;
    a.v = Vecs{weight, bias, d->wdtype};
    a.rows = (long)d->outer * d->inner; a.inner = d->inner; a.C = d->channels; a.act = d->act; a.eps = d->eps;
    const long most = p.kind <= 1 ? 2048 : 1l << 20;      // rows: a workgroup keeps the weights of its columns over several rows
    launch(*d, p, false, (unsigned)(p.tiles < most ? p.tiles : most), (hipStream_t)stream, a);
    return tef::check_launch("layer norm forward");
}

size_t tef_layer_norm_workspace_bytes(const tef_norm_desc *d)
{
    if (!valid(d)) return 0;
    if (d->outer == 0) return 16;
    return (size_t)bwd_blocks(make_plan(*d), d->channels) * 2 * (size_t)d->channels * sizeof(float);
}

int tef_layer_norm_backward(const tef_norm_desc *d, const void *x, const void *weight, const void *bias, const void *residual,
                            const float *mean, const float *rstd, const void *dy, void *dx, void *dresidual, void *dweight,
                            void *dbias, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!valid(d)) return TEF_ERR_INVALID;
    hipStream_t st = (hipStream_t)stream;
    if (d->outer == 0) {      // no rows: the sums over rows are zero
        if (dweight || dbias)
            hipLaunchKernelGGL(norm_zero, dim3((unsigned)((d->channels + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, dweight, dbias, d->channels, d->wdtype);
        return tef::check_launch("layer norm backward");
    }
    if (!x || !mean || !rstd || !dy) return tef::fail("tef_layer_norm_backward: null pointer"), TEF_ERR_INVALID;
    const bool sums = dweight || dbias;
    if (!dx && !dresidual && !sums) return 0;
    if (sums && (!workspace || workspace_bytes < tef_layer_norm_workspace_bytes(d)))
        return tef::fail("tef_layer_norm_backward: workspace too small"), TEF_ERR_WORKSPACE;
    const Plan p = make_plan(*d);
    Args a{};
    a.x = x; a.res = residual; a.dy = dy; a.dx = dx; a.dres = dresidual;
    a.mean = const_cast<float *>(mean); a.rstd = const_cast<float *>(rstd);
    a.part = sums ? (float *)workspace : nullptr;
    a.v = Vecs{weight, bias, d->wdtype};
    a.rows = (long)d->outer * d->inner; a.inner = d->inner; a.C = d->channels; a.act = d->act; a.eps = d->eps;
    const unsigned blocks = bwd_blocks(p, d->channels);
    launch(*d, p, true, blocks, st, a);
    if (sums) {
        const long joins = (2l * d->channels + 63) / 64, most = 1l << 21;      // (a launch holds less than 2^32 threads)
        hipLaunchKernelGGL(norm_join, dim3((unsigned)(joins < most ? joins : most)), dim3(64 * kJoinWaves), 0, st, (const float *)workspace, (int)blocks,
                           d->channels, dweight, dbias, d->wdtype);
    }
    return tef::check_launch("layer norm backward");
}

}  // extern "C"
