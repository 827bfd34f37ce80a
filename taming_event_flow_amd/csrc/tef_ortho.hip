// tef_ortho.hip — orthogonalised updates: Newton-Schulz orthogonalisation of matrices, and the optimiser step built on it
// (clip, momentum, orthogonalise, apply; Adam for the vectors).
//
// Orthogonalisation.  For U [m][n] (m <= n; a tall matrix is taken transposed) and X_0 = U / max(|U|_F, eps) the iteration
//
//   A = X X^T,  P = a I + b A + c A A,  X <- P X            (the singular values go through  a s + b s^3 + c s^5)
//
// can be run on the small side: P is a polynomial of A, so A' = X' X'^T = P A P and X_k = Q_k X_0 with Q' = P Q, and a segment of
// steps needs ONE Gram matrix of X and ONE product Q X; in between all matrices are m x m, symmetric, and commute (products of
// them are symmetric: half of the tiles are computed, the other half mirrored).  Every matrix close to a multiple of the identity is kept as its
// difference from it — P = a (I + B), B = (b/a) A + (c/a) A A, and Q = q (I + R), q = a^k — so that nothing small is rounded at the size of
// a diagonal:
//
//   W = A (I + B),  A' = a^2 W (I + B),  R' = R (I + B) + B,  X' = q (I + R) X
//
// where what the I brings is added to a product's fp32 sums unrounded.  The recurrence
// for A multiplies its rounding errors by up to a^2 = 12 a step along small singular values, the direct iteration by a; against the plain
// iteration in fp32, on gradients of rank m / 4 to m, segments of 2, 1, 1, 1 steps are 1.05 to 1.2 times as far from 64 bits
// (1.4 below 64 rows), 3 + 2 steps 1.5 to 3.5 times.  orthogonalize() takes the former: 6 m^2 n + 4 m^3
// multiply-adds (symmetric products at half) where the plain iteration takes 10 m^2 n + 5 m^3.  Small matrices take the same segments in
// one workgroup; those of up to 8 rows are iterated on the small side alone, in 64 bits, without planes.  The optimiser
// takes the latter, 3 m^2 n + 7 m^3: on momenta as networks have them (rank m / 4 to m over noise, 9 to 512 rows) the rms distance of a step's
// parameters from 64 bits is 0.97 to 1.21 times that of the plain iteration, the largest element's 0.7 to 1.7 times; segments of 2, 1, 1, 1
// would make that 0.81 to 1.09 and 0.6 to 1.7 and the default network's step 1.25 ms instead of 0.92.
//
// Arithmetic.  fp32 matrix instructions run at 1/16 of the fp16 rate, so every operand is held as two fp16 planes, v = hi + lo
// with hi = fp16(v), lo = fp16(v - hi) — 22 bits — and a product is hi hi + hi lo + lo hi with fp32 accumulation; the dropped lo lo
// is 2^-22 of the product.  All matrices have bounded entries (|X|, |A|, |B|, |R| of the order of 1), so a fixed power of two
// per matrix kind puts them into fp16's normal range.  Nothing is rounded to a single fp16 anywhere.
//
// Layout.  A split matrix is [rows][cols / 32][hi 32 | lo 32]: a row's 32 columns are one 128-byte line with both planes, so a
// step of 32 along k loads whole lines.  Rows and columns are padded to multiples of 32 with zeros.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "tef.h"
#include "tef_common.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kGroup = 64;             // matrices (with their batches) a set of launches takes
constexpr int kChunk = 16;             // of them per kernel argument
constexpr int kMaxParts = 512;         // partial sums of a matrix's squares
constexpr int kExpX = 12, kExpA = 12, kExpB = 12;      // powers of two that X, that A and W, that B and R are scaled by

// What the kernels know of a matrix (a batch of equal ones): lives in the workspace, written by the first launch.
struct Mat {
    const void *src;                   // [rows][cols], row stride src_ld, batch stride src_stride (elements)
    void *dst;
    long src_ld, dst_ld, src_stride, dst_stride;
    long ws;                           // bytes from the workspace's start to this matrix's area
    long area;                         // ... of one batch element
    long part;                         // bytes to the sums of products that are cut along k
    int m, n, mp, np;                  // short and long side, padded
    int tall;                          // src is [n][m]
    int batch;
    int parts;                         // partial sums of squares per batch element
    int splits;                        // pieces of the Gram product's k (lists of matrices)
    float scale;                       // of the applied update (optimiser)
    int first[6];                      // first work item in the launch of each phase (below)
};
enum { PH_SQ = 0, PH_PACK, PH_GRAM, PH_JOIN, PH_CHAIN, PH_APPLY, PHASES };

// One batch element's area: doubles parts[kMaxParts], int exponents[kMaxSteps + 1], then the split matrices.
// Bytes from a row to the next: an odd number of lines, so that a column of lines (the rows of a tile) lies in all the memory channels
// and not, as with 4096 columns, 16 KB apart in one of them.
__host__ __device__ inline long pitch(int cols) { return ((cols / 32) | 1) * 128l; }
__host__ __device__ inline long split_bytes(int rows, int cols) { return rows * pitch(cols); }
enum { BUF_X0 = 0, BUF_X1, BUF_A, BUF_W, BUF_B0, BUF_B1, BUF_R0, BUF_R1, BUF_END };
constexpr int kMaxSteps = 32;
constexpr long kHead = kMaxParts * 8 + 256;      // (a multiple of 256, at least 4 * (kMaxSteps + 1) past the sums)
__host__ __device__ inline long buf_at(int which, int mp, int np)
{
    const long x = split_bytes(mp, np), s = split_bytes(mp, mp);
    return which <= BUF_X1 ? kHead + which * x : kHead + 2 * x + (which - BUF_A) * s;
}

struct Table { const Mat *mats; int count; };

// The work item of a workgroup: consecutive ones — tiles that read the same rows — go to ONE of the 8 XCDs (workgroups are dealt to
// them in turn), so that a matrix is read into one L2 instead of all eight.  The first `whole` items (a multiple of 8) are
// dealt on their own: they take longer than the rest.
__device__ inline int work_item(int whole = 0)
{
    const int id = blockIdx.x, from = id < whole ? 0 : whole, total = id < whole ? whole : gridDim.x - whole;
    const int lin = id - from, xcd = lin & 7, each = total >> 3, more = total & 7;
    return from + xcd * each + (xcd < more ? xcd : more) + (lin >> 3);
}
// Which matrix an item of a phase belongs to: `first` is ascending, the wave looks at up to 64 of them at once.
__device__ inline int find(const Table &t, int phase, int item, int products = 1)
{
    if (t.count == 1) return 0;
    const int lane = threadIdx.x & 63;
    const int f = lane < t.count ? t.mats[lane].first[phase] * products : 0x7fffffff;
    return __popcll(__ballot(f <= item)) - 1;
}

template <typename T> __device__ inline float to_f(T v);
template <> __device__ inline float to_f<float>(float v) { return v; }
template <> __device__ inline float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ inline float to_f<__hip_bfloat16>(__hip_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ inline T from_f(float v);
template <> __device__ inline float from_f<float>(float v) { return v; }
template <> __device__ inline __half from_f<__half>(float v) { return __float2half(v); }
template <> __device__ inline __hip_bfloat16 from_f<__hip_bfloat16>(float v) { return __float2bfloat16(v); }
template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[V]; };

__device__ inline void split(float v, _Float16 &hi, _Float16 &lo)
{
    // v as ONE rounded number: without this the compiler forms a product's hi in one instruction from the unrounded product where hi is
    // stored, and from the rounded one where it is subtracted; near a tie the two differ by a unit of hi and lo belongs to the other
    asm("" : "+v"(v));
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);      // (infinite hi: NaN, as an overflow should show)
}

// eight neighbouring values of a split matrix's row
__device__ inline _Float16 *split_at(char *base, int cols, long row, int col)
{
    return reinterpret_cast<_Float16 *>(base + row * pitch(cols) + (col >> 5) * 128) + (col & 31);
}
__device__ inline void put_split(char *base, int cols, long row, int col, const float (&f)[8])
{
    _Float16 *p = split_at(base, cols, row, col);
    half8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        _Float16 h, l;
        split(f[k], h, l);
        hi[k] = h;
        lo[k] = l;
    }
    *reinterpret_cast<half8 *>(p) = hi;
    *reinterpret_cast<half8 *>(p + 32) = lo;
}

__device__ inline double block_sum(double s, double *red)
{
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- the matrices' values ---------------------------------------------------------------------------------------------------
// Orthogonalisation: the caller's matrix.  Optimiser step: the look-ahead of the momentum, u = g + mu (m' - g) (Nesterov) or m',
// g the clipped gradient, m' = m + (1 - mu) (g - m); the first sweep writes m', the second one clears g.  u is formed as mu m' + (1 - mu) g:
// while the momentum is young g and mu (m' - g) nearly cancel (a tenth is left on the first step), and their roundings would be ten times u's own.
struct Step {
    float *g, *m, *p;                  // flat buffers; a Mat's src / dst are element offsets into them
    const float *norm;
    const double *hp;                  // lr, momentum, weight_decay, max_norm
    int nesterov;
};
__device__ inline float clip_scale(const float *norm, double max_norm)
{
    if (!(max_norm > 0.0)) return 1.0f;
    const float s = (float)max_norm / (norm[0] + 1e-6f);      // (a NaN norm poisons the step: loud, like clip_grad_norm_)
    return s < 1.0f || s != s ? s : 1.0f;
}

// ---- phase 0: sums of squares (double: no overflow or underflow of a square for any fp32 input) -----------------------------
// Bound by memory: 31 million parameters, momentum updated on the way (g, m read, m written), 65 us = 5.8 TB/s.
struct Chunk { Mat m[kChunk]; int n, at; };

template <typename T, bool STEP> __global__ __launch_bounds__(kThreads) void ortho_squares(Chunk ch, Mat *table, char *ws, Step st)
{
    __shared__ double red[4];
    int k = 0;
    const int base = ch.m[0].first[PH_SQ];
    const int wg = blockIdx.x + base;
    while (k + 1 < ch.n && ch.m[k + 1].first[PH_SQ] <= wg) ++k;
    if (blockIdx.x == 0 && (int)threadIdx.x < ch.n) table[ch.at + threadIdx.x] = ch.m[threadIdx.x];
    const Mat &M = ch.m[k];
    const int part = (wg - M.first[PH_SQ]) % M.parts, bi = (wg - M.first[PH_SQ]) / M.parts;
    const long total = (long)M.m * M.n, per = ((total + M.parts - 1) / M.parts + 3) & ~3l;
    const long lo = part * per, hi = lo + per < total ? lo + per : total;
    double s = 0.0;
    if (STEP) {
        const float mu = (float)st.hp[1], clip = clip_scale(st.norm, st.hp[3]), w = (float)(1.0 - st.hp[1]);
        const long off = (long)M.src;
        auto one = [&](long i) {
            const float g = st.g[off + i] * clip;
            float mm = st.m[off + i];
            mm = mm + w * (g - mm);
            st.m[off + i] = mm;
            const float u = st.nesterov ? mu * mm + w * g : mm;
            s += (double)u * u;
        };
        long i = lo + 4l * threadIdx.x;
        for (; i + 4 <= hi; i += 4l * kThreads) {
            Pack<float, 4> g = *reinterpret_cast<const Pack<float, 4> *>(st.g + off + i), mm = *reinterpret_cast<const Pack<float, 4> *>(st.m + off + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float gc = g.v[j] * clip;
                mm.v[j] = mm.v[j] + w * (gc - mm.v[j]);
                const float u = st.nesterov ? mu * mm.v[j] + w * gc : mm.v[j];
                s += (double)u * u;
            }
            *reinterpret_cast<Pack<float, 4> *>(st.m + off + i) = mm;
        }
        for (; i < hi; ++i) one(i);
    } else {
        const int cols = M.tall ? M.m : M.n;
        const T *src = reinterpret_cast<const T *>(M.src) + bi * M.src_stride;
        if (M.src_ld == cols) {
            long i = lo + 4l * threadIdx.x;
            for (; i + 4 <= hi; i += 4l * kThreads) {
                const Pack<T, 4> q = *reinterpret_cast<const Pack<T, 4> *>(src + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) s += (double)to_f<T>(q.v[j]) * to_f<T>(q.v[j]);
            }
            for (; i < hi; ++i) s += (double)to_f<T>(src[i]) * to_f<T>(src[i]);
        } else {
            for (long i = lo + threadIdx.x; i < hi; i += kThreads) {
                const float v = to_f<T>(src[(i / cols) * M.src_ld + i % cols]);
                s += (double)v * v;
            }
        }
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) reinterpret_cast<double *>(ws + M.ws + bi * M.area)[part] = s;
}

// ---- phase 1: normalise and split ---------------------------------------------------------------------------------------------
// A workgroup writes 32 rows x 64 columns of the padded X (8 values a thread); bound by memory: g, m read, X written and g cleared for 31
// million parameters in 100 us = 5 TB/s.  The scale is kExpX plus, where |U| < eps leaves
// X small, the power of two that brings it back up: what is multiplied later always has 22 good bits.
template <typename T, bool STEP> __global__ __launch_bounds__(kThreads) void ortho_pack(Table t, char *ws, double eps, int grow_first, int grow_rest, Step st)
{
    __shared__ double red[4];
    __shared__ float turn[64][33];
    const Mat &M = t.mats[find(t, PH_PACK, (int)blockIdx.x)];
    const int tiles_n = (M.np + 63) / 64, tiles = (M.mp / 32) * tiles_n;
    const int wg = blockIdx.x - M.first[PH_PACK], bi = wg / tiles, ti = wg % tiles / tiles_n, tj = wg % tiles % tiles_n;
    char *area = ws + M.ws + bi * M.area;
    const double *parts = reinterpret_cast<const double *>(area);
    double s = 0.0;
    for (int k = threadIdx.x; k < M.parts; k += kThreads) s += parts[k];
    s = sqrt(block_sum(s, red));
    const double div = s < eps ? eps : s, rho = s / div;      // (a NaN norm: NaN everywhere)
    int up = 0;
    if (rho < 1.0 && rho > 0.0) {
        up = -ilogb(rho);
        up = up > 100 ? 100 : up;
    }
    if (wg % tiles == 0 && threadIdx.x == 0) {
        int *e = reinterpret_cast<int *>(area + kMaxParts * 8);
        e[0] = kExpX + up;
        for (int k = 1; k <= kMaxSteps; ++k) {      // a segment multiplies X by at most 2^grow
            up -= k == 1 ? grow_first : grow_rest;
            up = up > 0 ? up : 0;
            e[k] = kExpX + up;
        }
        up = e[0] - kExpX;
    }
    const double mul = ldexp(1.0 / div, kExpX + up);
    const float clip = STEP ? clip_scale(st.norm, st.hp[3]) : 1.0f, mu = STEP ? (float)st.hp[1] : 0.0f, w = STEP ? (float)(1.0 - st.hp[1]) : 0.0f;
    const T *src = reinterpret_cast<const T *>(M.src) + bi * M.src_stride;
    auto value = [&](long off) -> float {      // element `off` of the source
        if constexpr (STEP) {
            const long i = (long)M.src + off;
            const float g = st.g[i] * clip, mm = st.m[i];
            st.g[i] = 0.0f;
            return st.nesterov ? mu * mm + w * g : mm;
        } else {
            return to_f<T>(src[off]);
        }
    };
    float f[8];
    const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 8;      // row of the tile, first of 8 columns
    const int i0 = ti * 32, j0 = tj * 64;
    if (M.tall) {      // X[i][j] = src[j][i]: read along i, turn in LDS
        const int i = threadIdx.x & 31;
        for (int j = threadIdx.x >> 5; j < 64; j += 8)
            turn[j][i] = i0 + i < M.m && j0 + j < M.n ? value((long)(j0 + j) * M.src_ld + i0 + i) : 0.0f;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = turn[c + k][r];
    } else {
        const int i = i0 + r, j = j0 + c;
        const long off = (long)i * M.src_ld + j;
        if (i < M.m && j + 8 <= M.n) {
            if constexpr (STEP) {
                const long at = (long)M.src + off;
                const Pack<float, 8> g = *reinterpret_cast<const Pack<float, 8> *>(st.g + at), mm = *reinterpret_cast<const Pack<float, 8> *>(st.m + at);
                Pack<float, 8> zero;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float gc = g.v[k] * clip;
                    f[k] = st.nesterov ? mu * mm.v[k] + w * gc : mm.v[k];
                    zero.v[k] = 0.0f;
                }
                *reinterpret_cast<Pack<float, 8> *>(st.g + at) = zero;
            } else {
                const Pack<T, 8> q = *reinterpret_cast<const Pack<T, 8> *>(src + off);
#pragma unroll
                for (int k = 0; k < 8; ++k) f[k] = to_f<T>(q.v[k]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = i < M.m && j + k < M.n ? value(off + k) : 0.0f;
        }
    }
    if (j0 + c >= M.np) return;
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = (float)((double)f[k] * mul);
    put_split(area + buf_at(BUF_X0, M.mp, M.np), M.np, i0 + r, j0 + c, f);
}

// ---- the products -----------------------------------------------------------------------------------------------------------
// A workgroup of four waves computes TS x TS values (TS = 128 or 64), each wave a quarter of them in 32 x 32 blocks.  k advances
// by one line of 32 a stage, from global memory through registers (AHEAD stages in flight) into LDS while the previous stage is
// multiplied: two buffers, one barrier a stage.  The 16-byte chunks of a row are permuted by the row, chunk ^ (row / 2 & 7):
// sixteen lanes that read the same chunk of sixteen neighbouring rows (128 bytes each) meet all 64 banks once.
//
// What bounds them: large tiles (128) the way from L2 into the CU, 32 KB a line and workgroup, at 8 to 11 TB/s over the chip — 1.0 to 1.05
// PFLOP/s of fp16 products on 4096 x 4096, the matrix pipes 0.56 of the time busy; deeper prefetch, priorities and other instruction orders change
// nothing.  Small ones (64: 32 KB for a quarter of the work) the same on many CUs, latency on few.  A line's three plane products
// share its loads, which is why a line of 128 x 128 costs two thirds of the traffic per product that plain fp16 operands would.
template <int TS> struct Geo {
    static constexpr int FR = TS / 64;                       // 32 x 32 blocks of a wave along each side
    static constexpr int STAGE = TS * 128;                   // bytes of an operand's stage
    static constexpr int LOADS = STAGE / 16 / kThreads;      // 16-byte chunks of it per thread
    static constexpr int PITCH = TS + 4;                     // floats; the finished tile
    static constexpr int LDS = 4 * STAGE > TS * PITCH * 4 ? 4 * STAGE : TS * PITCH * 4;
};

// operand whose rows run along k: a row's 8 chunks side by side
template <int TS> __device__ inline void load_rows(uint4v (&r)[Geo<TS>::LOADS], const char *base, long ld, int row0, int rows, int kb)
{
    constexpr int per = 8;
#pragma unroll
    for (int i = 0; i < Geo<TS>::LOADS; ++i) {
        const int q = threadIdx.x + i * kThreads, row = row0 + q / per;
        r[i] = *reinterpret_cast<const uint4v *>(base + (long)(row < rows ? row : rows - 1) * ld + (long)kb * 128 + (q % per) * 16);
    }
}
template <int TS> __device__ inline void put_rows(char *lds, const uint4v (&r)[Geo<TS>::LOADS])
{
    constexpr int per = 8;
#pragma unroll
    for (int i = 0; i < Geo<TS>::LOADS; ++i) {
        const int q = threadIdx.x + i * kThreads, row = q / per;
        *reinterpret_cast<uint4v *>(lds + row * (per * 16) + (((q % per) ^ (row >> 1 & 7)) << 4)) = r[i];
    }
}
// rows `row` (this lane's), k = 16 * s + 8 * (lane >> 5) ..: plane 0 hi, 1 lo
__device__ inline half8 frag_rows(const char *lds, int row, int s, int plane)
{
    const int chunk = plane * 4 + s * 2 + ((threadIdx.x & 63) >> 5);
    return *reinterpret_cast<const half8 *>(lds + row * 128 + ((chunk ^ (row >> 1 & 7)) << 4));
}
// operand whose COLUMNS are the tile's (X in Q X): a stage is 32 rows of TS / 32 lines.  64-byte slots (one plane of one line)
// are permuted by the row; ds_read_b64_tr_b16 hands every lane four consecutive k of its column.
template <int TS> __device__ inline void load_cols(uint4v (&r)[Geo<TS>::LOADS], const char *base, long ld, int blk0, int blks, int kb)
{
    constexpr int per = TS / 4;      // chunks of a row
#pragma unroll
    for (int i = 0; i < Geo<TS>::LOADS; ++i) {
        const int q = threadIdx.x + i * kThreads, row = kb * 32 + q / per, c = q % per, blk = blk0 + (c >> 3);
        r[i] = *reinterpret_cast<const uint4v *>(base + (long)row * ld + (long)(blk < blks ? blk : blks - 1) * 128 + (c & 7) * 16);
    }
}
template <int TS> __device__ inline void put_cols(char *lds, const uint4v (&r)[Geo<TS>::LOADS])
{
    constexpr int per = TS / 4, slots = TS / 16;
#pragma unroll
    for (int i = 0; i < Geo<TS>::LOADS; ++i) {
        const int q = threadIdx.x + i * kThreads, row = q / per, c = q % per, slot = (c >> 2) ^ (row & (slots - 1));
        *reinterpret_cast<uint4v *>(lds + row * (TS * 4) + slot * 64 + (c & 3) * 16) = r[i];
    }
}
template <int TS> __device__ inline half8 frag_cols(const char *lds, int col0, int s, int plane)
{
    constexpr int slots = TS / 16;
    const int lane = threadIdx.x & 63, g = lane >> 4, src = lane & 15;
    const int slot = (col0 >> 5) * 2 + plane, within = ((g & 1) * 16 + (src & 3) * 4) * 2;
    half8 v;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = s * 16 + (g >> 1) * 8 + h * 4 + (src >> 2);
        const char *p = lds + row * (TS * 4) + (slot ^ (row & (slots - 1))) * 64 + within;
        const short4v q = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v *)p);
        const half4 f = __builtin_bit_cast(half4, q);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[h * 4 + k] = f[k];
    }
    return v;
}

template <int TS> struct Acc { float16v v[Geo<TS>::FR][Geo<TS>::FR]; };

// the identity's 32 x 16 block s (rows or columns this lane's, k = 16 s + 8 (lane >> 5) ..), times v
__device__ inline half8 identity(int s, _Float16 v)
{
    const int lane = threadIdx.x & 63, at = (lane & 31) - s * 16 - (lane >> 5) * 8;
    half8 f;
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = at == k ? v : (_Float16)0.0f;
    return f;
}

// acc = L (rows li0 ..) times R (rows rj0 .. as columns, or, COLS, the 32-column blocks rj0 / 32 ..), k lines k0 .. k1
template <int TS, int AHEAD, bool COLS>
__device__ inline void product(Acc<TS> &acc, char *lds, const char *L, long ldL, int li0, int rowsL, const char *R, long ldR, int rj0, int limR, int k0, int k1)
{
    using G = Geo<TS>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = (wave >> 1) * (TS / 2), wj = (wave & 1) * (TS / 2);
#pragma unroll
    for (int i = 0; i < G::FR; ++i)
#pragma unroll
        for (int j = 0; j < G::FR; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc.v[i][j][e] = 0.0f;
    uint4v a[AHEAD][G::LOADS], b[AHEAD][G::LOADS];
    // (past the end the last line is fetched again: no branch around the loads)
#define TEF_FETCH(slot, line)                                                              \
    do {                                                                                   \
        const int at_ = (line) < k1 ? (line) : k1 - 1;                                     \
        load_rows<TS>(a[slot], L, ldL, li0, rowsL, at_);                                   \
        if (COLS) load_cols<TS>(b[slot], R, ldR, rj0 >> 5, limR, at_);                     \
        else load_rows<TS>(b[slot], R, ldR, rj0, limR, at_);                               \
    } while (0)
#define TEF_PUT(slot, buf)                                                                 \
    do {                                                                                   \
        put_rows<TS>(lds + (buf) * 2 * G::STAGE, a[slot]);                                 \
        if (COLS) put_cols<TS>(lds + (buf) * 2 * G::STAGE + G::STAGE, b[slot]);            \
        else put_rows<TS>(lds + (buf) * 2 * G::STAGE + G::STAGE, b[slot]);                 \
    } while (0)
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) TEF_FETCH(d, k0 + d);
    __syncthreads();      // (whoever used this LDS before is done with it)
    TEF_PUT(0, 0);
    __syncthreads();
    auto multiply = [&](int d) {      // the line in LDS buffer d & 1
        const char *la = lds + (d & 1) * 2 * G::STAGE, *lb = la + G::STAGE;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            half8 fa[G::FR][2], fb[G::FR][2];
#pragma unroll
            for (int i = 0; i < G::FR; ++i)
#pragma unroll
                for (int pl = 0; pl < 2; ++pl) {
                    fa[i][pl] = frag_rows(la, wi + i * 32 + (lane & 31), s, pl);
                    fb[i][pl] = COLS ? frag_cols<TS>(lb, wj + i * 32, s, pl) : frag_rows(lb, wj + i * 32 + (lane & 31), s, pl);
                }
#pragma unroll
            for (int t = 0; t < 3; ++t)      // lo hi, hi lo, hi hi
#pragma unroll
                for (int i = 0; i < G::FR; ++i)
#pragma unroll
                    for (int j = 0; j < G::FR; ++j)
                        acc.v[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[i][t == 0], fb[j][t == 1], acc.v[i][j], 0, 0, 0);
        }
    };
    int kb = k0;
    for (; kb + AHEAD <= k1; kb += AHEAD) {      // (no way out in between: a wait would have to cover loads of both paths)
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {        // line kb + d lies in LDS buffer d & 1, the following AHEAD - 1 on their way in registers
            TEF_FETCH(d, kb + d + AHEAD);
            multiply(d);
            TEF_PUT((d + 1) % AHEAD, (d + 1) & 1);
            __syncthreads();
        }
    }
#pragma unroll
    for (int d = 0; d + 1 < AHEAD; ++d)
        if (kb + d < k1) {
            multiply(d);
            TEF_PUT(d + 1, (d + 1) & 1);
            __syncthreads();
        }
#undef TEF_FETCH
#undef TEF_PUT
}

// acc += one * M, the tile (i0, j0) of a split matrix, straight from memory: M's rows times an identity, exact (one: a power of two)
template <int TS> __device__ inline void add_tile(Acc<TS> &acc, const char *M, int rows, int cols, int i0, int j0, float one)
{
    using G = Geo<TS>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = (wave >> 1) * (TS / 2), wj = (wave & 1) * (TS / 2);
#pragma unroll
    for (int i = 0; i < G::FR; ++i)
#pragma unroll
        for (int j = 0; j < G::FR; ++j) {
            const int row = i0 + wi + i * 32 + (lane & 31), line = ((j0 + wj) >> 5) + j, lines = cols / 32;
            const char *p = M + (row < rows ? row : rows - 1) * pitch(cols) + (line < lines ? line : lines - 1) * 128 + (lane >> 5) * 16;
            half8 f[2][2];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int pl = 0; pl < 2; ++pl) f[s][pl] = *reinterpret_cast<const half8 *>(p + pl * 64 + s * 32);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int pl = 0; pl < 2; ++pl) acc.v[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[s][pl], identity(s, (_Float16)one), acc.v[i][j], 0, 0, 0);
        }
}

// The finished tile in LDS, row-major or, TURN, transposed (a lane of a 32 x 32 block holds column lane & 31 and the rows
// 8 (e / 4) + 4 (lane >> 5) + e % 4: four neighbours of a row of the transposed tile, one 16-byte write); either way free of
// bank conflicts, and read back in rows.
template <int TS, bool TURN> __device__ inline float *to_tile(const Acc<TS> &acc, char *lds)
{
    using G = Geo<TS>;
    typedef float float4v __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = (wave >> 1) * (TS / 2), wj = (wave & 1) * (TS / 2);
    float *tile = reinterpret_cast<float *>(lds);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < G::FR; ++i)
#pragma unroll
        for (int j = 0; j < G::FR; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = wi + i * 32 + 8 * e + 4 * (lane >> 5), col = wj + j * 32 + (lane & 31);
                if (TURN) {
                    *reinterpret_cast<float4v *>(tile + col * G::PITCH + row) = float4v{acc.v[i][j][4 * e], acc.v[i][j][4 * e + 1], acc.v[i][j][4 * e + 2], acc.v[i][j][4 * e + 3]};
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) tile[(row + k) * G::PITCH + col] = acc.v[i][j][4 * e + k];
                }
            }
    __syncthreads();
    return tile;
}

// a diagonal tile: its upper triangle, and that mirrored
template <int TS> __device__ inline float *to_tile_upper(const Acc<TS> &acc, char *lds)
{
    using G = Geo<TS>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = (wave >> 1) * (TS / 2), wj = (wave & 1) * (TS / 2);
    float *tile = reinterpret_cast<float *>(lds);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < G::FR; ++i)
#pragma unroll
        for (int j = 0; j < G::FR; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = wi + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3), col = wj + j * 32 + (lane & 31);
                if (row <= col) {
                    tile[row * G::PITCH + col] = acc.v[i][j][e];
                    tile[col * G::PITCH + row] = acc.v[i][j][e];
                }
            }
    __syncthreads();
    return tile;
}

// Writes rows row0 .. of the tile in LDS to the split matrix `out`, from column col0 on: mul * value (+ PLUS: plus * A).
template <int TS, bool PLUS>
__device__ inline void put_tile(const float *tile, char *out, int rows, int cols, int row0, int col0, float mul, char *A, float plus)
{
    constexpr int per = TS / 8, ROUNDS = TS * per / kThreads, BATCH = ROUNDS < 4 ? ROUNDS : 4;
    for (int at = 0; at < ROUNDS; at += BATCH) {
        half8 hi[BATCH], lo[BATCH];
        if (PLUS)
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {      // (on their way before the first value is needed)
                const int q = threadIdx.x + (at + i) * kThreads, row = row0 + q / per, col = col0 + q % per * 8;
                const _Float16 *p = split_at(A, cols, row < rows ? row : rows - 1, col < cols ? col : cols - 8);
                hi[i] = *reinterpret_cast<const half8 *>(p);
                lo[i] = *reinterpret_cast<const half8 *>(p + 32);
            }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int q = threadIdx.x + (at + i) * kThreads, r = q / per, c = q % per * 8, row = row0 + r, col = col0 + c;
            float f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                f[k] = mul * tile[r * Geo<TS>::PITCH + c + k];
                if (PLUS) f[k] += plus * ((float)hi[i][k] + (float)lo[i][k]);
            }
            if (row < rows && col < cols) put_split(out, cols, row, col, f);
        }
    }
}

// ... of a symmetric matrix: the tile (i0, j0) and its mirror image.  A diagonal tile holds both triangles, the same products added
// up in another order: the upper one is taken for both.  (The iteration relies on it: an asymmetry of one rounding grows with every step and
// cost a factor of twelve in the result of a 40 x 300 matrix of rank one.)
template <int TS, bool PLUS>
__device__ inline void put_symmetric(const Acc<TS> &acc, char *lds, char *out, int mp, int i0, int j0, float mul, char *A, float plus)
{
    put_tile<TS, PLUS>(i0 == j0 ? to_tile_upper<TS>(acc, lds) : to_tile<TS, false>(acc, lds), out, mp, mp, i0, j0, mul, A, plus);
    if (i0 != j0) put_tile<TS, PLUS>(to_tile<TS, true>(acc, lds), out, mp, mp, j0, i0, mul, A, plus);
}

// tile number -> (i, j), j >= i, of a symmetric matrix of T x T tiles: eight columns at a time, so that 64 consecutive tiles, which run
// side by side on one XCD, read 8 + 8 blocks of rows
__device__ inline void triangle(int t, int T, int &i, int &j)
{
    int j0 = 0;
    for (;;) {
        const int w = T - j0 < 8 ? T - j0 : 8, n = w * j0 + w * (w + 1) / 2;
        if (t < n) {
            if (t < w * j0) { i = t / w; j = j0 + t % w; return; }
            t -= w * j0;
            i = 0;
            while (t >= w - i) { t -= w - i; ++i; }
            j = j0 + i + t;
            i += j0;
            return;
        }
        t -= n;
        j0 += 8;
    }
}

// ---- phases 2 and 3: the symmetric products A = X X^T (k the long side) and those of the m x m matrices ------------------------------
// A launch computes one or two of them (`products`, of every matrix).  Where their tiles do not fill the machine evenly some are
// cut along k: `splits` pieces of every tile from number `whole` on (0 splits: the matrix's own number of pieces, all tiles); a
// piece's fp32 sums go to the workspace as the threads hold them and ortho_join adds them up in order.
struct Sym {
    int l[2], r[2], out[2];            // buffers
    float mul[2];                      // of the values
    int plus_l[2], plus_r[2];          // add L, add R to the product (at the scale of B: the other factor is I + ..)
    int products;
    int poly;                          // product 0 is A A, its result B
    float plus;
    int gram, seg;                     // product 0 is X X^T of this segment's X
    int whole, splits;
};
struct Piece { int w, bi, ti, tj, slot, piece, pieces; };
template <int TS> __device__ inline Piece piece_of(const Mat &M, const Sym &c, int local, bool join)
{
    const int T = (M.mp + TS - 1) / TS, tiles = T * (T + 1) / 2, total = tiles * M.batch * c.products;
    Piece p;
    const int cut = c.splits ? c.splits : M.splits;
    int tile;
    if (join) {
        p.slot = local; tile = c.whole + local; p.piece = 0; p.pieces = cut;
    } else if (local < c.whole) {
        p.slot = 0; tile = local; p.piece = 0; p.pieces = 1;
    } else {
        const int n = total - c.whole;      // (the tiles of one piece of k next to each other: they read the same lines)
        p.slot = (local - c.whole) % n; tile = c.whole + p.slot; p.piece = (local - c.whole) / n; p.pieces = cut;
    }
    p.w = tile / (tiles * M.batch);
    tile %= tiles * M.batch;
    p.bi = tile / tiles;
    triangle(tile % tiles, T, p.ti, p.tj);
    return p;
}
template <int TS> __device__ inline void finish(const Acc<TS> &acc, char *lds, const Mat &M, char *area, const Sym &c, const Piece &p)
{
    char *out = area + buf_at(c.out[p.w], M.mp, M.np);
    if (c.poly) {
        put_symmetric<TS, true>(acc, lds, out, M.mp, p.ti * TS, p.tj * TS, c.mul[p.w], area + buf_at(c.l[p.w], M.mp, M.np), c.plus);
    } else {
        const float mul = c.gram ? ldexpf(1.0f, kExpA - 2 * reinterpret_cast<const int *>(area + kMaxParts * 8)[c.seg]) : c.mul[p.w];
        put_symmetric<TS, false>(acc, lds, out, M.mp, p.ti * TS, p.tj * TS, mul, nullptr, 0.0f);
    }
}
// DEEP: at most one workgroup a CU, which then has the registers for twice the lines in flight.
template <int TS, bool DEEP> __global__ __launch_bounds__(kThreads, DEEP ? 1 : 2) void ortho_symmetric(Table t, char *ws, Sym c)
{
    __shared__ __attribute__((aligned(16))) char lds[Geo<TS>::LDS];
    const int item = work_item(c.splits > 1 ? c.whole : 0), phase = c.gram ? PH_GRAM : PH_CHAIN;
    const Mat &M = t.mats[find(t, phase, item, c.products)];
    const Piece p = piece_of<TS>(M, c, item - M.first[phase] * c.products, false);
    char *area = ws + M.ws + p.bi * M.area;
    const char *L = area + buf_at(c.l[p.w], M.mp, M.np), *R = area + buf_at(c.r[p.w], M.mp, M.np);
    const int side = c.gram ? M.np : M.mp, lines = side / 32;
    const int k0 = (int)((long)lines * p.piece / p.pieces), k1 = (int)((long)lines * (p.piece + 1) / p.pieces);
    Acc<TS> acc;
    product<TS, (TS == 64 ? 4 : 2) * (DEEP ? 2 : 1), false>(acc, lds, L, pitch(side), p.ti * TS, M.mp, R, pitch(side), p.tj * TS, M.mp, k0, k1);
    if (p.piece == 0) {
        if (c.plus_l[p.w]) add_tile<TS>(acc, L, M.mp, M.mp, p.ti * TS, p.tj * TS, (float)(1 << kExpB));
        if (c.plus_r[p.w]) add_tile<TS>(acc, R, M.mp, M.mp, p.ti * TS, p.tj * TS, (float)(1 << kExpB));
    }
    if (p.pieces == 1) return finish<TS>(acc, lds, M, area, c, p);
    float *part = reinterpret_cast<float *>(ws + M.part) + ((long)p.slot * p.pieces + p.piece) * TS * TS;
#pragma unroll
    for (int i = 0; i < Geo<TS>::FR; ++i)
#pragma unroll
        for (int j = 0; j < Geo<TS>::FR; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) part[((i * Geo<TS>::FR + j) * 16 + e) * kThreads + threadIdx.x] = acc.v[i][j][e];
}

template <int TS> __global__ __launch_bounds__(kThreads) void ortho_join(Table t, char *ws, Sym c)
{
    __shared__ __attribute__((aligned(16))) char lds[Geo<TS>::LDS];
    const int item = work_item();
    const Mat &M = t.mats[find(t, PH_JOIN, item)];
    const Piece p = piece_of<TS>(M, c, item - (t.count == 1 ? 0 : M.first[PH_JOIN]), true);
    if (p.pieces == 1) return;
    const float *part = reinterpret_cast<const float *>(ws + M.part) + (long)p.slot * p.pieces * TS * TS;
    Acc<TS> acc;
#pragma unroll
    for (int i = 0; i < Geo<TS>::FR; ++i)
#pragma unroll
        for (int j = 0; j < Geo<TS>::FR; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc.v[i][j][e] = 0.0f;
    for (int s = 0; s < p.pieces; s += 2) {      // two pieces' sums in flight
        constexpr int N = Geo<TS>::FR * Geo<TS>::FR * 16;
        const float *q = part + (long)s * TS * TS + threadIdx.x;
        const bool two = s + 1 < p.pieces;
        float f[2][N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            f[0][k] = q[k * kThreads];
            f[1][k] = q[(two ? TS * TS : 0) + k * kThreads];
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            auto &v = acc.v[k / 16 / Geo<TS>::FR][k / 16 % Geo<TS>::FR];
            v[k % 16] += f[0][k];
            v[k % 16] += two ? f[1][k] : 0.0f;
        }
    }
    finish<TS>(acc, lds, M, ws + M.ws + p.bi * M.area, c, p);
}

// The same for m x m products of few and short tiles, where a launch is latency (385 x 385: 8.4 us with 64 x 64 tiles, 6.9 with these; past some
// 500 tiles the operands' re-reading costs more: 27 us against 15 for nine matrices of 512): 32 x 32 tiles, k dealt line by line to the four waves,
// fragments straight from memory (no LDS, no barrier; four lines of a wave in flight), the waves' sums joined in order in LDS.
__global__ __launch_bounds__(kThreads) void ortho_symmetric32(Table t, char *ws, Sym c)
{
    constexpr int TS = 32, PITCH = 36, BATCH = 4;
    typedef float float4v __attribute__((ext_vector_type(4)));
    __shared__ __attribute__((aligned(16))) float sums[4][TS * PITCH];
    __shared__ float done[TS * (TS + 1)];
    const int item = work_item();
    const Mat &M = t.mats[find(t, PH_CHAIN, item, c.products)];
    const int T = M.mp / TS, tiles = T * (T + 1) / 2;
    int tile = item - M.first[PH_CHAIN] * c.products, ti, tj;
    const int w = tile / (tiles * M.batch), bi = tile % (tiles * M.batch) / tiles;
    triangle(tile % tiles, T, ti, tj);
    char *area = ws + M.ws + bi * M.area;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lines = M.mp / 32;
    const long ld = pitch(M.mp), at = (lane >> 5) * 16;
    const char *L = area + buf_at(c.l[w], M.mp, M.np) + (ti * TS + (lane & 31)) * ld + at, *R = area + buf_at(c.r[w], M.mp, M.np) + (tj * TS + (lane & 31)) * ld + at;
    const int r = threadIdx.x >> 3, q = (threadIdx.x & 7) * 4, row = ti * TS + r, col = tj * TS + q;
    half4 hi[2], lo[2];      // this thread's part of L and R, where they are added
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (k ? c.plus_r[w] : c.plus_l[w] | c.poly) {
            const _Float16 *p = split_at(area + buf_at(k ? c.r[w] : c.l[w], M.mp, M.np), M.mp, row, col);
            hi[k] = *reinterpret_cast<const half4 *>(p);
            lo[k] = *reinterpret_cast<const half4 *>(p + 32);
        }
    float16v acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
    for (int l0 = wave; l0 < lines; l0 += 4 * BATCH) {
        half8 a[BATCH][2][2], b[BATCH][2][2];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int l = l0 + 4 * k < lines ? l0 + 4 * k : lines - 1;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int pl = 0; pl < 2; ++pl) {
                    a[k][s][pl] = *reinterpret_cast<const half8 *>(L + l * 128l + pl * 64 + s * 32);
                    b[k][s][pl] = *reinterpret_cast<const half8 *>(R + l * 128l + pl * 64 + s * 32);
                }
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
            if (l0 + 4 * k < lines)
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int x = 0; x < 3; ++x) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[k][s][x == 0], b[k][s][x == 1], acc, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) sums[wave][(8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * PITCH + (lane & 31)] = acc[e];
    __syncthreads();
    float4v f = *reinterpret_cast<const float4v *>(&sums[0][r * PITCH + q]);
#pragma unroll
    for (int k = 1; k < 4; ++k) f += *reinterpret_cast<const float4v *>(&sums[k][r * PITCH + q]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (c.plus_l[w]) f[k] += (float)(1 << kExpB) * ((float)hi[0][k] + (float)lo[0][k]);
        if (c.plus_r[w]) f[k] += (float)(1 << kExpB) * ((float)hi[1][k] + (float)lo[1][k]);
        f[k] *= c.mul[w];
        if (c.poly) f[k] += c.plus * ((float)hi[0][k] + (float)lo[0][k]);
        done[r * (TS + 1) + q + k] = f[k];
    }
    __syncthreads();
    char *out = area + buf_at(c.out[w], M.mp, M.np);
    for (int mirror = 0; mirror < (ti == tj ? 1 : 2); ++mirror) {
        half4 vhi, vlo;
#pragma unroll
        for (int k = 0; k < 4; ++k) {      // (the diagonal tile: its upper triangle for both, see put_symmetric)
            const bool turn = mirror || (ti == tj && r > q + k);
            _Float16 h, lw;
            split(turn ? done[(q + k) * (TS + 1) + r] : f[k], h, lw);
            vhi[k] = h;
            vlo[k] = lw;
        }
        _Float16 *p = split_at(out, M.mp, mirror ? tj * TS + r : row, mirror ? ti * TS + q : col);
        *reinterpret_cast<half4 *>(p) = vhi;
        *reinterpret_cast<half4 *>(p + 32) = vlo;
    }
}

// ---- phase 4: X' = q (I + R) X, into the other X, the caller's matrix, or the parameters -------------------------------------------------
// 4096 x 4096: 410 us = 1.0 PFLOP/s of fp16 products; the default network's matrices: 141 us into X, 168 into the parameters (0.6 PFLOP/s, 16
// lines a tile: a third of the time is the tile's way out).
enum { TO_X = 0, TO_DST, TO_PARAM };
template <int TS, typename T, int DEST> __global__ __launch_bounds__(kThreads, 2) void ortho_apply(Table t, char *ws, int seg, int r_buf, float q, Step st)
{
    __shared__ __attribute__((aligned(16))) char lds[Geo<TS>::LDS];
    const int item = work_item();
    const Mat M = t.mats[find(t, PH_APPLY, item)];      // (a copy: the stores below could be to the table, as far as the compiler knows)
    const int Ti = (M.mp + TS - 1) / TS, Tj = (M.np + TS - 1) / TS;
    const int wg = item - M.first[PH_APPLY], bi = wg / (Ti * Tj), r = wg % (Ti * Tj);
    const int j8 = r / (8 * Ti) * 8, w8 = Tj - j8 < 8 ? Tj - j8 : 8, ti = (r - j8 * Ti) / w8, tj = j8 + (r - j8 * Ti) % w8;      // (as in triangle())
    char *area = ws + M.ws + bi * M.area;
    const char *X = area + buf_at(seg & 1 ? BUF_X1 : BUF_X0, M.mp, M.np);
    const int *ex = reinterpret_cast<const int *>(area + kMaxParts * 8);
    const int e0 = ex[seg], e1 = ex[seg + 1];
    Acc<TS> acc;
    product<TS, TS == 64 ? 4 : 2, true>(acc, lds, area + buf_at(r_buf, M.mp, M.np), pitch(M.mp), ti * TS, M.mp, X, pitch(M.np), tj * TS, M.np / 32, 0, M.mp / 32);
    add_tile<TS>(acc, X, M.mp, M.np, ti * TS, tj * TS, (float)(1 << kExpB));
    if constexpr (DEST == TO_X) {
        put_tile<TS, false>(to_tile<TS, false>(acc, lds), area + buf_at(seg & 1 ? BUF_X0 : BUF_X1, M.mp, M.np), M.mp, M.np, ti * TS, tj * TS, ldexpf(q, e1 - e0 - kExpB), nullptr, 0.0f);
        return;
    }
    // the result, in the caller's orientation: row r of the output tile, four neighbours of it
    const float mul = ldexpf(q, -(e0 + kExpB));
    float keep = 1.0f, step = 1.0f;
    if constexpr (DEST == TO_PARAM) {
        keep = (float)(1.0 - st.hp[0] * st.hp[2]);
        step = (float)(st.hp[0] * (double)M.scale);
    }
    constexpr int quads = TS / 4;
    const float *tile = M.tall ? to_tile<TS, true>(acc, lds) : to_tile<TS, false>(acc, lds);
    const int R = M.tall ? M.n : M.m, C = M.tall ? M.m : M.n, r0 = (M.tall ? tj : ti) * TS, c0 = (M.tall ? ti : tj) * TS;
    for (int k = threadIdx.x; k < TS * quads; k += kThreads) {
        const int r = k / quads, c = k % quads * 4, row = r0 + r, col = c0 + c;
        if (row >= R || col >= C) continue;
        float f[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) f[x] = mul * tile[r * Geo<TS>::PITCH + c + x];
        if constexpr (DEST == TO_PARAM) {
            float *p = st.p + (long)M.dst + (long)row * M.dst_ld + col;
            if (col + 4 <= C) {
                Pack<float, 4> o = *reinterpret_cast<const Pack<float, 4> *>(p);
#pragma unroll
                for (int x = 0; x < 4; ++x) o.v[x] = o.v[x] * keep - step * f[x];
                *reinterpret_cast<Pack<float, 4> *>(p) = o;
            } else {
                for (int x = 0; x < 4 && col + x < C; ++x) p[x] = p[x] * keep - step * f[x];
            }
        } else {
            T *p = reinterpret_cast<T *>(M.dst) + bi * M.dst_stride + (long)row * M.dst_ld + col;
            if (col + 4 <= C) {
                Pack<T, 4> o;
#pragma unroll
                for (int x = 0; x < 4; ++x) o.v[x] = from_f<T>(f[x]);
                *reinterpret_cast<Pack<T, 4> *>(p) = o;
            } else {
                for (int x = 0; x < 4 && col + x < C; ++x) p[x] = from_f<T>(f[x]);
            }
        }
    }
}

// ---- small matrices: the whole iteration in one workgroup --------------------------------------------------------------------------
// m <= 64 and at most 32 LINES columns: X, A, B and R stay in LDS as split matrices (line l: 64 rows of 128 bytes, permuted as the
// stages above) and one launch does what the general path spreads over twenty, each a few microseconds of latency whatever the
// size.  X <- q (I + R) X goes to X's own place (a tile's values are in registers when its columns have been read), and so does every
// other product to one of its operands'.
__device__ inline char *line_at(char *m, int line) { return m + line * (64 * 128); }
// acc = L R^T over `lines` lines (this wave's 32 x 32 block); hi lo and lo hi have a sum of their own, 2^-11 of the other's size: a third of
// the additions round at the size of the result
__device__ inline void small_rows(Acc<64> &acc, const char *L, const char *R, int lines)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
    float16v cross;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc.v[0][0][e] = cross[e] = 0.0f;
    for (int l = 0; l < lines; ++l)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            half8 a[2], b[2];
#pragma unroll
            for (int pl = 0; pl < 2; ++pl) {
                a[pl] = frag_rows(L + l * 8192, wi + (lane & 31), s, pl);
                b[pl] = frag_rows(R + l * 8192, wj + (lane & 31), s, pl);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[t == 0], b[t == 1], cross, 0, 0, 0);
            acc.v[0][0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[0], acc.v[0][0], 0, 0, 0);
        }
#pragma unroll
    for (int e = 0; e < 16; ++e) acc.v[0][0][e] += cross[e];
}
// acc = (B + one I) X over `lines` lines of B, for the two lines of X from `X` on (64 columns; X's rows are k)
__device__ inline void small_cols(Acc<64> &acc, const char *B, const char *X, int lines, _Float16 one)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = (wave >> 1) * 32, g = lane >> 4, src = lane & 15;
    const char *x = X + (wave & 1) * 8192;
    float16v cross;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc.v[0][0][e] = cross[e] = 0.0f;
    for (int l = 0; l < lines; ++l)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            half8 a[2], b[2];
#pragma unroll
            for (int pl = 0; pl < 2; ++pl) {
                a[pl] = frag_rows(B + l * 8192, wi + (lane & 31), s, pl);
#pragma unroll
                for (int h = 0; h < 2; ++h) {      // four k of this lane's column: see frag_cols
                    const int row = l * 32 + s * 16 + (g >> 1) * 8 + h * 4 + (src >> 2), col = (g & 1) * 16 + (src & 3) * 4;
                    const char *p = x + row * 128 + (((pl * 4 + (col >> 3)) ^ (row >> 1 & 7)) << 4) + (col & 4) * 2;
                    const half4 f = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v *)p));
#pragma unroll
                    for (int k = 0; k < 4; ++k) b[pl][h * 4 + k] = f[k];
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[t == 0], b[t == 1], cross, 0, 0, 0);
            acc.v[0][0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[0], acc.v[0][0], 0, 0, 0);
            if (l * 32 == wi)
#pragma unroll
                for (int pl = 0; pl < 2; ++pl) acc.v[0][0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(identity(s, one), b[pl], acc.v[0][0], 0, 0, 0);
        }
#pragma unroll
    for (int e = 0; e < 16; ++e) acc.v[0][0][e] += cross[e];
}
__device__ inline char *small_at(char *m, int row, int col, int plane)      // 16 bytes: eight columns from `col` on
{
    return line_at(m, col >> 5) + row * 128 + (((plane * 4 + ((col & 31) >> 3)) ^ (row >> 1 & 7)) << 4);
}
// mul times the 64 x 64 values of the tile, plus (ADD 1) plus * A, plus (ADD 2) B too — this thread's 16 values of them as they were
// before they were split: B's linear term would otherwise carry A's rounding, the largest one in small matrices — to the split matrix
// `out` of two lines and, unsplit, back
struct Kept { float v[16]; };
template <int ADD> __device__ inline Kept small_put(const float *tile, char *out, float mul, const Kept &A, float plus, const Kept &B)
{
    Kept kept;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int q = threadIdx.x + i * kThreads, r = q >> 3, c = (q & 7) * 8;
        half8 hi, lo;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float f = mul * tile[r * Geo<64>::PITCH + c + k];
            if (ADD > 0) f += plus * A.v[i * 8 + k];
            if (ADD > 1) f += B.v[i * 8 + k];
            kept.v[i * 8 + k] = f;
            _Float16 h, l;
            split(f, h, l);
            hi[k] = h;
            lo[k] = l;
        }
        *reinterpret_cast<half8 *>(small_at(out, r, c, 0)) = hi;
        *reinterpret_cast<half8 *>(small_at(out, r, c, 1)) = lo;
    }
    __syncthreads();
    return kept;
}

struct Small { Mat m[kChunk]; int first[kChunk]; int n; };
struct SmallPoly { float a, b, c; int steps, first, grow_first, grow_rest; double eps; };      // b, c: over a
template <typename T, int LINES> __global__ __launch_bounds__(kThreads) void ortho_small(Small list, SmallPoly p)
{
    __shared__ __attribute__((aligned(16))) char mats[3 * 16384];
    __shared__ __attribute__((aligned(16))) char X[LINES * 8192];
    __shared__ __attribute__((aligned(16))) char scratch[64 * Geo<64>::PITCH * 4];
    __shared__ double red[4];
    int k = 0;
    while (k + 1 < list.n && list.first[k + 1] <= (int)blockIdx.x) ++k;
    const Mat &M = list.m[k];
    const int bi = blockIdx.x - list.first[k], cols = M.tall ? M.m : M.n, m = M.m, n = M.n, klines = m > 32 ? 2 : 1;
    const T *src = reinterpret_cast<const T *>(M.src) + bi * M.src_stride;
    double s = 0.0;
    for (int i = threadIdx.x; i < m * n; i += kThreads) {
        const float v = to_f<T>(src[(long)(i / cols) * M.src_ld + i % cols]);
        s += (double)v * v;
    }
    s = sqrt(block_sum(s, red));
    const double div = s < p.eps ? p.eps : s, rho = s / div;
    int up = 0;
    if (rho < 1.0 && rho > 0.0) {
        up = -ilogb(rho);
        up = up > 100 ? 100 : up;
    }
    const double mul = ldexp(1.0 / div, kExpX + up);
    const int xlines = 2 * ((n + 63) / 64);      // (whole 64-column tiles; LINES is even)
    for (int q = threadIdx.x; q < xlines * 256; q += kThreads) {      // eight columns of a row; a wave along the source's rows
        const int per = xlines * 4, r = M.tall ? q & 63 : q / per, c = (M.tall ? q >> 6 : q % per) * 8;
        half8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = r < m && c + e < n;
            const long off = M.tall ? (long)(c + e) * M.src_ld + r : (long)r * M.src_ld + c + e;
            const float v = in ? (float)((double)to_f<T>(src[in ? off : 0]) * mul) : 0.0f;
            _Float16 h, l;
            split(v, h, l);
            hi[e] = h;
            lo[e] = l;
        }
        *reinterpret_cast<half8 *>(small_at(X, r, c, 0)) = hi;
        *reinterpret_cast<half8 *>(small_at(X, r, c, 1)) = lo;
    }
    __syncthreads();
    Acc<64> acc;
    for (int done = 0; done < p.steps;) {
        const bool two = done == 0 && p.first == 2 && p.steps > 1;      // the first segment; the rest goes step by step
        char *A = mats, *B = mats + 16384, *R = B;
        const float b1 = ldexpf(p.b, kExpB - kExpA), c1 = ldexpf(p.c, kExpB - 2 * kExpA), unit = ldexpf(1.0f, -kExpB);
        const Kept none{};
        small_rows(acc, X, X, xlines);
        Kept a = small_put<0>(to_tile_upper<64>(acc, scratch), A, ldexpf(1.0f, kExpA - 2 * (kExpX + up)), none, 0.0f, none);
        small_rows(acc, A, A, klines);
        const Kept b = small_put<1>(to_tile_upper<64>(acc, scratch), B, c1, a, b1, none);
        if (two) {
            small_rows(acc, A, B, klines);      // W = A + A B, in A's place
            a = small_put<1>(to_tile_upper<64>(acc, scratch), A, unit, a, 1.0f, none);
            small_rows(acc, A, B, klines);      // A' = a^2 (W + W B)
            a = small_put<1>(to_tile_upper<64>(acc, scratch), A, p.a * p.a * unit, a, p.a * p.a, none);
            B = mats + 32768;
            small_rows(acc, A, A, klines);
            const Kept b2 = small_put<1>(to_tile_upper<64>(acc, scratch), B, c1, a, b1, none);
            small_rows(acc, R, B, klines);      // R' = R + B + R B
            small_put<2>(to_tile_upper<64>(acc, scratch), R, unit, b, 1.0f, b2);
        }
        done += two ? 2 : 1;
        const int e0 = kExpX + up;
        up -= two || done == 1 ? p.grow_first : p.grow_rest;
        up = up > 0 ? up : 0;
        const float q = two ? p.a * p.a : p.a;
        for (int x = 0; x < xlines; x += 2) {
            small_cols(acc, R, line_at(X, x), klines, (_Float16)(float)(1 << kExpB));
            if (done < p.steps) {
                small_put<0>(to_tile<64, false>(acc, scratch), line_at(X, x), ldexpf(q, kExpX + up - e0 - kExpB), Kept{}, 0.0f, Kept{});
                continue;
            }
            const float *tile = M.tall ? to_tile<64, true>(acc, scratch) : to_tile<64, false>(acc, scratch);
            const float out = ldexpf(q, -(e0 + kExpB));
            T *dst = reinterpret_cast<T *>(M.dst) + bi * M.dst_stride;
            const int c0 = x * 32;      // columns of X: rows of a tall result
            for (int q = threadIdx.x; q < 64 * 64; q += kThreads) {
                const int r = q >> 6, c = q & 63, row = M.tall ? c0 + r : r, col = M.tall ? c : c0 + c;
                if (row < (M.tall ? n : m) && col < cols) dst[(long)row * M.dst_ld + col] = from_f<T>(out * tile[r * Geo<64>::PITCH + c]);
            }
        }
    }
}

// ---- tiny matrices: m <= 8, sums and the iteration in 64 bits ------------------------------------------------------------------------
// A matrix instruction would be idle for the most part, and with so few terms the planes' 22 bits show.  One pass over the matrix sums
// A = X X^T (m (m + 1) / 2 sums a thread), the iteration runs on the small side alone (P = a I + b A + c A A, A' = P A P, Q' = P Q, 64 lanes
// an 8 x 8 matrix), a second pass writes Q X: everything in 64 bits, rounded once at the end.  A' multiplies A's rounding by up to max|P|^2 a
// step, so more steps than `run` (10^6 between them: 5 with the usual coefficients) are cut into segments of as many: X <- Q X is kept in
// 64 bits, in LDS or the workspace, and A summed again.  Distance from an iteration in 64 bits on gradients of 2 x 3 to 8 x 8192: half a
// step of fp32, where the plain fp32 iteration is 0.4 to 4.8e-6 off.
// Up to kTinyOne columns a matrix is one workgroup's, in one launch (TINY); longer ones take a launch for each sum and one for the
// result, in workgroups of kTinyPer columns and more, whose sums go through the workspace and are added up in order by every workgroup
// of the next launch (THIN): 8 x 960 takes 18.8 us in one launch and 20.4 in two, 8 x 1500 23.8 and 20.8, 512 of 8 x 1000 31.5 and 33.  2 x 3: 17
// us a call, kernel 6.0; 8 x 8192: 20, kernels 7.3 + 9.0; 8 x 200000: 43 (planes: 605).  Bound by the call and by latency, the long ones by
// 64-bit multiply-adds.
constexpr int kTinySide = 8, kTinyPairs = kTinySide * (kTinySide + 1) / 2;
constexpr long kTinyOne = 1024, kTinyPer = 512, kTinyParts = 128;
enum { TINY_ALL = 0, TINY_ALL_SEGMENTS, TINY_SUMS, TINY_APPLY };
struct TinyPoly { double a, b, c, eps; int steps, run, seg; };

// a column of the matrix.  The optimiser's: the first pass moves the momentum.
template <typename T, bool STEP, bool FIRST> __device__ inline void tiny_column(double (&x)[kTinySide], const Mat &M, const T *src, const Step &st, float clip, double mu, long c)
{
#pragma unroll
    for (int r = 0; r < kTinySide; ++r) {
        x[r] = 0.0;
        if (r >= M.m) continue;
        const long off = M.tall ? c * M.src_ld + r : r * M.src_ld + c;
        if constexpr (STEP) {
            const long at = (long)M.src + off;
            const float g = st.g[at] * clip;
            float mm = st.m[at];
            if (FIRST) {
                mm = mm + (float)(1.0 - mu) * (g - mm);
                st.m[at] = mm;
            }
            x[r] = st.nesterov ? mu * mm + (1.0 - mu) * g : mm;
        } else {
            x[r] = to_f<T>(src[off]);
        }
    }
}

// NT: threads of a workgroup; with at most 64 columns one wave has all of them, and the same sums.
template <typename T, bool STEP, int WHAT, int NT = kThreads> __global__ __launch_bounds__(NT) void ortho_tiny(Small list, TinyPoly p, char *ws, Step st)
{
    constexpr int S = kTinySide, WAVES = NT / 64;
    constexpr bool ONE = WHAT == TINY_ALL || WHAT == TINY_ALL_SEGMENTS;
    __shared__ double red[WAVES][kTinyPairs], A[S * S], W[S * S], V[S * S], Q[2][S * S], held[WHAT == TINY_ALL_SEGMENTS ? S * kTinyOne : 1];
    int k = 0;
    while (k + 1 < list.n && list.first[k + 1] <= (int)blockIdx.x) ++k;
    const Mat &M = list.m[k];
    const int item = blockIdx.x - list.first[k], bi = item / M.parts, part = item % M.parts, m = M.m, pairs = m * (m + 1) / 2;
    const int per = ((M.n + M.parts - 1) / M.parts + NT - 1) & ~(NT - 1), c0 = part * per, c1 = c0 + per < M.n ? c0 + per : M.n;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, e = lane;
    const int r = e >> 3, c = e & 7, lo = r < c ? r : c, hi = r < c ? c : r, pair = hi * (hi + 1) / 2 + lo;
    const double mu = STEP ? st.hp[1] : 0.0;
    const float clip = STEP ? clip_scale(st.norm, st.hp[3]) : 1.0f;
    const T *src = STEP ? nullptr : reinterpret_cast<const T *>(M.src) + bi * M.src_stride;
    // the workspace of a batch element (THIN): two sets of the parts' sums, by the parity of the segment that they belong to, then X
    double *sums = nullptr, *X = held;
    if (!ONE) {
        sums = reinterpret_cast<double *>(ws + M.part) + bi * (2l * M.parts * pairs + (long)m * M.n);
        X = sums + 2l * M.parts * pairs;
    }
    auto column = [&](double (&x)[S], long col, bool source) {      // (what a thread reads of X it wrote itself)
        if (source) return tiny_column<T, STEP, false>(x, M, src, st, clip, mu, col);
#pragma unroll
        for (int i = 0; i < S; ++i) x[i] = i < m ? X[(long)i * M.n + col] : 0.0;
    };
    double *q = Q[0], *spare = Q[1];
    // this workgroup's sums of the products of X's rows, X <- Q X first (seg > 0)
    auto sum = [&](int seg) {
        double s[kTinyPairs];
#pragma unroll
        for (int i = 0; i < kTinyPairs; ++i) s[i] = 0.0;
        for (int col = c0 + tid; col < c1; col += NT) {
            double x[S];
            if (seg == 0) {
                tiny_column<T, STEP, true>(x, M, src, st, clip, mu, col);
            } else {
                double u[S];
                column(u, col, seg == 1);
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    x[i] = 0.0;
                    if (i >= m) continue;
#pragma unroll
                    for (int j = 0; j < S; ++j) x[i] = fma(q[i * S + j], u[j], x[i]);
                    X[(long)i * M.n + col] = x[i];
                }
            }
#pragma unroll
            for (int i = 0; i < S; ++i)
                if (i < m)
#pragma unroll
                    for (int j = 0; j <= i; ++j) s[i * (i + 1) / 2 + j] = fma(x[i], x[j], s[i * (i + 1) / 2 + j]);
        }
        __syncthreads();
        if (c0 + wave * 64 >= c1) {      // (no column for this wave)
            if (lane < pairs) red[wave][lane] = 0.0;
        } else if (m <= 4) {
#pragma unroll
            for (int i = 0; i < 10; ++i)
                if (i < pairs) {
                    for (int o = 32; o > 0; o >>= 1) s[i] += __shfl_xor(s[i], o, 64);
                    if (lane == 0) red[wave][i] = s[i];
                }
        } else {      // halving: a lane sends the half of its sums that it does not keep (63 exchanges instead of 216), lane i ends with sum i
            double v[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) v[i] = i < kTinyPairs ? s[i] : 0.0;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const bool upper = lane & o;
#pragma unroll
                for (int i = 0; i < o; ++i) v[i] = (upper ? v[i + o] : v[i]) + __shfl_xor(upper ? v[i] : v[i + o], o, 64);
            }
            if (lane < pairs) red[wave][lane] = v[0];
        }
        __syncthreads();
    };
    auto joined = [&](int i) {
        if constexpr (WAVES == 1) return red[0][i];
        else return (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
    };
    auto times = [&](const double *L, const double *R) {      // (of matrices that commute: symmetric, so the upper triangle's value for both)
        double f = 0.0;
#pragma unroll
        for (int x = 0; x < S; ++x) f = fma(L[lo * S + x], R[x * S + hi], f);
        return f;
    };
    // the steps of segment `seg` on the sums in `red`, into q: one wave's work, whose LDS accesses are done in the order that they are written in
    auto in_order = [] { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); };
    auto iterate = [&](int seg) {
        const int begin = seg * p.run, end = begin + p.run < p.steps ? begin + p.run : p.steps;
        if (wave == 0) {
            A[e] = hi < m ? joined(pair) : 0.0;
            double mul = 1.0;
            if (seg == 0) {
                in_order();
                double norm = 0.0;
                for (int i = 0; i < m; ++i) norm += A[i * S + i];
                norm = sqrt(norm);
                mul = 1.0 / (norm < p.eps ? p.eps : norm);      // (a NaN norm: NaN everywhere)
                in_order();
                A[e] = A[e] * mul * mul;
            }
            q[e] = r == c ? mul : 0.0;
            in_order();
            double *from = q, *to = spare;
            for (int step = begin; step < end; ++step) {
                W[e] = fma(p.c, times(A, A), fma(p.b, A[e], r == c ? p.a : 0.0));      // P
                in_order();
                to[e] = times(W, from);
                if (step + 1 < end) {
                    V[e] = times(A, W);
                    in_order();
                    A[e] = times(W, V);
                }
                in_order();
                double *const was = from;
                from = to;
                to = was;
            }
        }
        if ((end - begin) & 1) {
            double *const was = q;
            q = spare;
            spare = was;
        }
        __syncthreads();
    };
    const int segments = (p.steps + p.run - 1) / p.run;
    if (ONE) {
        for (int seg = 0; seg < (WHAT == TINY_ALL ? 1 : segments); ++seg) {
            sum(seg);
            iterate(seg);
        }
    } else {
        if (p.seg > 0) {      // the segment before this launch's: its parts' sums, a quarter of them a wave
            const int was = (p.seg - 1) & 1;
            if (e < pairs) {
                double s = 0.0;
                for (int k = wave; k < M.parts; k += WAVES) s += sums[((long)was * M.parts + k) * pairs + e];
                red[wave][e] = s;
            }
            __syncthreads();
            iterate(p.seg - 1);
        }
        if (WHAT == TINY_SUMS) {
            const int now = p.seg & 1;
            sum(p.seg);
            if (tid < pairs) sums[((long)now * M.parts + part) * pairs + tid] = joined(tid);
            return;
        }
    }
    const float keep = STEP ? (float)(1.0 - st.hp[0] * st.hp[2]) : 1.0f, go = STEP ? (float)(st.hp[0] * (double)M.scale) : 1.0f;
    T *dst = STEP ? nullptr : reinterpret_cast<T *>(M.dst) + bi * M.dst_stride;
    for (int col = c0 + tid; col < c1; col += NT) {
        double x[S];
        column(x, col, segments == 1);
#pragma unroll
        for (int i = 0; i < S; ++i) {
            if (i >= m) continue;
            double f = 0.0;
#pragma unroll
            for (int j = 0; j < S; ++j) f = fma(q[i * S + j], x[j], f);
            const long off = M.tall ? (long)col * M.dst_ld + i : i * M.dst_ld + col;
            if constexpr (STEP) {
                st.g[(long)M.src + off] = 0.0f;      // (the optimiser's rows are as far apart in both)
                float *o = st.p + (long)M.dst + off;
                *o = *o * keep - go * (float)f;
            } else {
                dst[off] = from_f<T>((float)f);
            }
        }
    }
}

constexpr int kSmallSide = 64, kSmallLong = 320;      // (10 lines of X: 148 KB of LDS with A, B, R and the tile)

// ---- Adam for the vectors (the same arithmetic as tef_adam_clip_step, over a list of ranges of the flat buffers) --------------------
constexpr int kRanges = 96;
struct Ranges { long off[kRanges]; int first[kRanges + 1]; int v0; int n; };
__global__ __launch_bounds__(kThreads) void muon_vectors(Ranges rg, float *p, float *g, float *m, float *v, const float *norm, const double *hp, const float *step)
{
    const float clip = clip_scale(norm, hp[3]);
    const double b1 = hp[5], b2d = hp[6], t = (double)step[0];
    const double bc1 = 1.0 - pow(b1, t), bc2 = 1.0 - pow(b2d, t);
    const float step_size = (float)(hp[4] / bc1), bc2_sqrt = (float)sqrt(bc2), w1 = (float)(1.0 - b1), b2 = (float)b2d, w2 = (float)(1.0 - b2d), eps = (float)hp[7];
    const int total = rg.first[rg.n];
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < total; i += gridDim.x * kThreads) {
        int lo = 0, hi = rg.n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (rg.first[mid] <= i) lo = mid;
            else hi = mid - 1;
        }
        const long at = rg.off[lo] + (i - rg.first[lo]);
        const float gr = g[at] * clip;
        const float mm = m[at] + w1 * (gr - m[at]), vv = v[rg.v0 + i] * b2 + (w2 * gr) * gr;
        m[at] = mm;
        v[rg.v0 + i] = vv;
        p[at] = p[at] - step_size * (mm / (sqrtf(vv) / bc2_sqrt + eps));
        g[at] = 0.0f;
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
struct Poly { double a, b, c; int steps, first, rest, grow_first, grow_rest; double most; };      // most: max|P| on the way; steps of the first segment and of the following ones; the powers of two X grows by in them

// The bounds that the fixed scales rely on, for singular values that start anywhere in [0, 1]: X and A stay below 2^2 (s < 4 would
// square to 16: 2^12 * 16 = 65536 overflows fp16), B and R below 15, and a segment's q below 2^6 (the exponents of X).
bool bounded(Poly &p)
{
    if (!(isfinite(p.a) && isfinite(p.b) && isfinite(p.c)) || fabs(p.a) < 1e-3) return tef::fail("orthogonalisation: the coefficients have to be finite, the first one not 0");
    // 513 values s (0 among them: its q is 1); W at once, no branches between them: the host does this on every call
    constexpr int W = 8;
    const double a = p.a, b = p.b / p.a, c = p.c / p.a;
    double first = 1.0, rest = 1.0, least[W], largest[W];
    for (int w = 0; w < W; ++w) least[w] = largest[w] = 1.0;
    for (int g = 1; g <= 512; g += W) {
        double s[W], q[W], top[W], far[W], size = 1.0;
        for (int w = 0; w < W; ++w) s[w] = (g + w) / 512.0, q[w] = 1.0;
        for (int k = 0, left = p.first; k < p.steps; ++k, --left) {
            if (left == 0) {
                left = p.rest;
                size = 1.0;
                for (int w = 0; w < W; ++w) q[w] = 1.0;
            }
            size *= a;
            for (int w = 0; w < W; ++w) {
                const double l = s[w] * s[w], poly = 1.0 + (b + c * l) * l;
                q[w] *= poly;
                s[w] *= a * poly;
                least[w] = poly < least[w] ? poly : least[w];
                largest[w] = poly > largest[w] ? poly : largest[w];
                top[w] = fabs(s[w]);
                far[w] = fabs(q[w] - 1.0);
            }
            double grown = 1.0;
            int held = 1;
            for (int w = 0; w < W; ++w) {
                held &= (int)(top[w] < 3.9) & (int)(far[w] < 15.0);      // (not for NaN)
                grown = fabs(q[w]) > grown ? fabs(q[w]) : grown;
            }
            grown *= fabs(size);
            if (!held || !(grown < 64.0))
                return tef::fail("orthogonalisation: these coefficients let the iteration grow past what it can hold (singular values below 3.9, their polynomial below 64 in two steps)");
            double &most = k < p.first ? first : rest;
            most = grown > most ? grown : most;
        }
    }
    double low = 1.0, high = 1.0;
    for (int w = 0; w < W; ++w) {
        low = least[w] < low ? least[w] : low;
        high = largest[w] > high ? largest[w] : high;
    }
    if (high - 1.0 >= 15.0 || 1.0 - low >= 15.0) return tef::fail("orthogonalisation: these coefficients let the iteration grow past what it can hold (singular values below 3.9, their polynomial below 64 in two steps)");
    p.most = fabs(a) * (high > -low ? high : -low);
    p.grow_first = (int)ceil(log2(first));
    p.grow_rest = (int)ceil(log2(rest));
    return true;
}

enum Form { TINY, THIN, SMALL, TILED, FORMS };
struct Cut { int whole, splits; long items, joins; };
struct Group {
    Mat m[kGroup];
    int n;
    long bytes;                        // workspace
    int grid[PHASES];
    int ts_gram, ts_chain, ts_apply;
    Cut gram, chain[2];                // one, two products
};

inline int round32(long v) { return (int)((v + 31) & ~31l); }

inline long triangle_tiles(int mp, int ts)
{
    const long T = (mp + ts - 1) / ts;
    return T * (T + 1) / 2;
}

// How the tiles of ONE matrix's product are dealt to 256 CUs: as many as are a multiple of 256 whole, the rest cut along k so that the
// pieces, too, are about 256 (512 of the large tiles when there is nothing else to run beside them), of at least 8 lines: a piece's sums have to be
// written and read again, and joining takes a launch of its own (about 10 us), so products of fewer than 32 lines are left alone.
// 4096 x 4096: 528 tiles take 280 us whole — two on every CU, then the last 16 — and 180 us with those 16 in pieces.
Cut cut_one(long tiles, long lines, int ts)
{
    Cut c{(int)tiles, 1, tiles, 0};
    const long rest = tiles % 256;
    if (lines < 32 || tiles > (1l << 24) || !rest) return c;
    long s = tiles < 256 ? (ts == 128 ? 512 : 256) / tiles : 256 / rest;
    if (s > lines / 8) s = lines / 8;
    if (s < 2) return c;
    if (s > 64) s = 64;
    c.whole = (int)(tiles - rest);
    c.splits = (int)s;
    c.items = c.whole + rest * s;
    c.joins = rest;
    return c;
}

// Tile sizes: 128 where the launch then still covers the 256 CUs, else 64 (a quarter of the work each, so that four times as many
// workgroups share it).
bool plan(Group &g)
{
    long chain128 = 0, apply128 = 0, steps128 = 0;
    for (int k = 0; k < g.n; ++k) {
        const Mat &M = g.m[k];
        const long T = (M.mp + 127) / 128;
        chain128 += (long)M.batch * triangle_tiles(M.mp, 128);
        apply128 += (long)M.batch * T * ((M.np + 127) / 128);
        steps128 += (long)M.batch * triangle_tiles(M.mp, 128) * (M.np / 32);
    }
    g.ts_chain = chain128 >= 256 || (g.n == 1 && chain128 >= 64 && g.m[0].mp >= 1024) ? 128 : 64;
    long chain32 = 0;
    for (int k = 0; k < g.n; ++k) chain32 += (long)g.m[k].batch * triangle_tiles(g.m[k].mp, 32);
    if (g.ts_chain == 64 && chain32 <= 512) g.ts_chain = 32;
    g.ts_gram = steps128 >= 256 * 16 ? 128 : 64;
    g.ts_apply = apply128 >= 192 ? 128 : 64;
    // a list: every tile of the Gram products in pieces of one length, the shortest that gives no more pieces than run at once
    long piece = 8, slots = g.ts_gram == 128 ? 512 : 1024;
    if (g.n > 1)
        for (;; piece += piece / 8) {
            long items = 0, longest = 0;
            for (int k = 0; k < g.n; ++k) {
                const long lines = g.m[k].np / 32;
                items += (long)g.m[k].batch * triangle_tiles(g.m[k].mp, g.ts_gram) * ((lines + piece - 1) / piece);
                longest = longest > lines ? longest : lines;
            }
            if (items <= slots || piece >= longest) break;
        }
    long first[PHASES] = {};
    long at = (long)((sizeof(Mat) * kGroup + 255) & ~255ul);
    g.gram = Cut{0, 0, 0, 0};
    for (int k = 0; k < g.n; ++k) {
        Mat &M = g.m[k];
        const long tiles = triangle_tiles(M.mp, g.ts_gram), lines = M.np / 32;
        long splits = (lines + piece - 1) / piece, parts = 0;
        if (g.n == 1) {
            g.gram = cut_one(tiles * M.batch, lines, g.ts_gram);
            parts = g.gram.joins * g.gram.splits * g.ts_gram * g.ts_gram;
            splits = 1;
            for (int w = 0; w < 2; ++w) {
                const long all = triangle_tiles(M.mp, g.ts_chain) * M.batch * (w + 1);
                g.chain[w] = g.ts_chain == 32 ? Cut{(int)all, 1, all, 0} : cut_one(all, M.mp / 32, g.ts_chain);
                const long p = g.chain[w].joins * g.chain[w].splits * g.ts_chain * g.ts_chain;
                parts = parts > p ? parts : p;
            }
        } else {
            splits = splits > 64 ? 64 : splits;
            if (splits > 1) {
                parts = tiles * M.batch * splits * g.ts_gram * g.ts_gram;
                g.gram.joins = 1;
            }
        }
        M.splits = (int)splits;
        const long total = (long)M.m * M.n;
        long sums = (total + 16383) / 16384;
        M.parts = (int)(sums < 1 ? 1 : sums > kMaxParts ? kMaxParts : sums);
        M.area = (buf_at(BUF_END, M.mp, M.np) + 255) & ~255l;
        M.ws = at;
        M.part = at + M.area * M.batch;
        at = M.part + ((parts * 4 + 255) & ~255l);
        const long Ta = (M.mp + g.ts_apply - 1) / g.ts_apply, Tb = (M.np + g.ts_apply - 1) / g.ts_apply;
        const long per[PHASES] = {M.parts, (M.mp / 32) * ((M.np + 63l) / 64), tiles * splits, tiles, triangle_tiles(M.mp, g.ts_chain), Ta * Tb};
        for (int f = 0; f < PHASES; ++f) {
            M.first[f] = (int)first[f];
            first[f] += per[f] * M.batch;
        }
    }
    if (g.n > 1) {
        g.gram.items = first[PH_GRAM];
        if (g.gram.joins) g.gram.joins = first[PH_JOIN];
        for (int w = 0; w < 2; ++w) g.chain[w] = Cut{0, 1, first[PH_CHAIN] * (w + 1), 0};
    }
    // (a launch holds less than 2^32 threads: 2^24 workgroups of 256, and a launch of two products has twice the items)
    g.bytes = at;
    for (int f = 0; f < PHASES; ++f) {
        if (first[f] > 0x7fffff) return tef::fail("orthogonalisation: too many tiles for one launch");
        g.grid[f] = (int)first[f];
    }
    return true;
}

bool describe(Mat &M, long rows, long cols, long batch)
{
    if (rows < 1 || cols < 1 || batch < 1) return tef::fail("orthogonalisation: empty matrix");
    const long m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    if (n > (1l << 24) || m > (1l << 15) || batch > (1l << 20)) return tef::fail("orthogonalisation: matrix sides up to 2^15 x 2^24, batches up to 2^20");
    memset(&M, 0, sizeof(M));
    M.m = (int)m; M.n = (int)n; M.mp = round32(m); M.np = round32(n);
    M.tall = rows > cols;
    M.batch = (int)batch;
    return true;
}

#define TS_LAUNCH(ts, call128, call64) do { if ((ts) == 128) { call128; } else { call64; } } while (0)

template <typename T, bool STEP>
int iterate(Group &g, const Poly &p, double eps, char *ws, const Step &st, hipStream_t stream)
{
    Mat *table = reinterpret_cast<Mat *>(ws);
    const dim3 block(kThreads);
    for (int at = 0; at < g.n; at += kChunk) {
        Chunk ch;
        ch.at = at;
        ch.n = g.n - at < kChunk ? g.n - at : kChunk;
        memcpy(ch.m, g.m + at, sizeof(Mat) * ch.n);
        const int end = at + ch.n < g.n ? g.m[at + ch.n].first[PH_SQ] : g.grid[PH_SQ];
        hipLaunchKernelGGL((ortho_squares<T, STEP>), dim3((unsigned)(end - ch.m[0].first[PH_SQ])), block, 0, stream, ch, table, ws, st);
    }
    const Table t{table, g.n};
    hipLaunchKernelGGL((ortho_pack<T, STEP>), dim3((unsigned)g.grid[PH_PACK]), block, 0, stream, t, ws, eps, p.grow_first, p.grow_rest, st);
    const dim3 apply((unsigned)g.grid[PH_APPLY]);
    auto symmetric = [&](Sym c, int products, int ts, const Cut &cut) {
        c.products = products;
        c.whole = cut.whole;
        c.splits = cut.splits;
        const dim3 grid((unsigned)cut.items);
        const bool deep = cut.items <= 256;
        if (ts == 32) {
            hipLaunchKernelGGL(ortho_symmetric32, grid, block, 0, stream, t, ws, c);
            return;
        }
        if (ts == 128) {
            if (deep) hipLaunchKernelGGL((ortho_symmetric<128, true>), grid, block, 0, stream, t, ws, c);
            else hipLaunchKernelGGL((ortho_symmetric<128, false>), grid, block, 0, stream, t, ws, c);
        } else {
            if (deep) hipLaunchKernelGGL((ortho_symmetric<64, true>), grid, block, 0, stream, t, ws, c);
            else hipLaunchKernelGGL((ortho_symmetric<64, false>), grid, block, 0, stream, t, ws, c);
        }
        if (cut.joins)
            TS_LAUNCH(ts, hipLaunchKernelGGL(ortho_join<128>, dim3((unsigned)cut.joins), block, 0, stream, t, ws, c),
                      hipLaunchKernelGGL(ortho_join<64>, dim3((unsigned)cut.joins), block, 0, stream, t, ws, c));
    };
    for (int s = 0, done = 0; done < p.steps; ++s) {
        int len = s ? p.rest : p.first;
        if (len > p.steps - done) len = p.steps - done;
        Sym x{};
        x.gram = 1; x.seg = s;
        x.l[0] = x.r[0] = s & 1 ? BUF_X1 : BUF_X0; x.out[0] = BUF_A;
        symmetric(x, 1, g.ts_gram, g.gram);
        int R = -1;
        double q = 1.0;
        for (int k = 0; k < len; ++k) {
            const int B = k & 1 ? BUF_B1 : BUF_B0;
            Sym c{};      // B = (b/a) A + (c/a) A A
            c.l[0] = c.r[0] = BUF_A; c.out[0] = B; c.poly = 1;
            c.mul[0] = (float)ldexp(p.c / p.a, kExpB - 2 * kExpA); c.plus = (float)ldexp(p.b / p.a, kExpB - kExpA);
            symmetric(c, 1, g.ts_chain, g.chain[0]);
            // W = A (I + B) and R' = R (I + B) + B
            Sym d{};
            int products = 0;
            if (k + 1 < len) {
                d.l[0] = BUF_A; d.r[0] = B; d.out[0] = BUF_W; d.mul[0] = ldexpf(1.0f, -kExpB); d.plus_l[0] = 1;
                products = 1;
            }
            if (k > 0) {
                const int out = R == BUF_R0 ? BUF_R1 : BUF_R0;
                d.l[products] = R; d.r[products] = B; d.out[products] = out; d.mul[products] = ldexpf(1.0f, -kExpB);
                d.plus_l[products] = d.plus_r[products] = 1;
                ++products;
                R = out;
            } else {
                R = B;
            }
            if (products) symmetric(d, products, g.ts_chain, g.chain[products - 1]);
            if (k + 1 < len) {
                Sym e{};      // A' = a^2 W (I + B)
                e.l[0] = BUF_W; e.r[0] = B; e.out[0] = BUF_A; e.mul[0] = (float)ldexp(p.a * p.a, -kExpB); e.plus_l[0] = 1;
                symmetric(e, 1, g.ts_chain, g.chain[0]);
            }
            q *= p.a;
        }
        done += len;
        const float qf = (float)q;
        if (done < p.steps) {
            TS_LAUNCH(g.ts_apply, hipLaunchKernelGGL((ortho_apply<128, float, TO_X>), apply, block, 0, stream, t, ws, s, R, qf, st),
                      hipLaunchKernelGGL((ortho_apply<64, float, TO_X>), apply, block, 0, stream, t, ws, s, R, qf, st));
        } else {
            constexpr int D = STEP ? TO_PARAM : TO_DST;
            TS_LAUNCH(g.ts_apply, hipLaunchKernelGGL((ortho_apply<128, T, D>), apply, block, 0, stream, t, ws, s, R, qf, st),
                      hipLaunchKernelGGL((ortho_apply<64, T, D>), apply, block, 0, stream, t, ws, s, R, qf, st));
        }
    }
    return tef::check_launch("orthogonalisation");
}

// The launches of up to kChunk matrices each: items(matrix) workgroups a matrix.  (Batches hold up to 2^20 matrices and a matrix's items are at
// most 2^22, a launch holds up to 2^24 workgroups.)
template <typename Items, typename Launch> void in_chunks(const Group &g, Items items, Launch launch)
{
    for (int at = 0; at < g.n;) {
        Small list;
        int total = 0, longest = 0;
        for (list.n = 0; list.n < kChunk && at < g.n && total <= 0x700000; ++list.n, ++at) {
            list.m[list.n] = g.m[at];
            list.first[list.n] = total;
            total += (int)items(g.m[at]);
            longest = longest > g.m[at].n ? longest : g.m[at].n;
        }
        launch(list, dim3((unsigned)total), longest);
    }
}

// One workgroup a matrix for small ones: 27 us against the tiled launches' 71 for a single 64 x 18 one,
// 81 against 94 at the limit of 64 x 320, 63 against 185 for 512 of 64 x 64.
template <typename T> int small(const Group &g, const Poly &p, double eps, hipStream_t stream)
{
    const SmallPoly sp{(float)p.a, (float)(p.b / p.a), (float)(p.c / p.a), p.steps, p.first, p.grow_first, p.grow_rest, eps};
    in_chunks(g, [](const Mat &M) { return M.batch; }, [&](const Small &list, dim3 grid, int longest) {
        const dim3 block(kThreads);
        if (longest <= 64) hipLaunchKernelGGL((ortho_small<T, 2>), grid, block, 0, stream, list, sp);
        else if (longest <= 128) hipLaunchKernelGGL((ortho_small<T, 4>), grid, block, 0, stream, list, sp);
        else hipLaunchKernelGGL((ortho_small<T, 10>), grid, block, 0, stream, list, sp);
    });
    return tef::check_launch("orthogonalisation");
}

void plan_thin(Group &g)
{
    long at = 0;
    for (int k = 0; k < g.n; ++k) {
        Mat &M = g.m[k];
        const long most = (1l << 22) / M.batch;
        long parts = (M.n + kTinyPer - 1) / kTinyPer;
        parts = parts > kTinyParts ? kTinyParts : parts;
        parts = parts > most ? most : parts;
        M.parts = (int)parts;
        M.part = at;
        at += (M.batch * (parts * M.m * (M.m + 1) + (long)M.m * M.n) * 8 + 255) & ~255l;      // two sets of m (m + 1) / 2 sums; X
    }
    g.bytes = at;
}
template <typename T, bool STEP> int tiny(const Group &g, Form form, const Poly &p, double eps, char *ws, const Step &st, hipStream_t stream)
{
    // (rounding of 10^-16 stays below 10^-9 of A through a run: A' takes max|P|^2 of it a step)
    const double most = p.most > 1.0 ? log(p.most) : 0.0;
    const int run = most > 0.0 && 2.0 * most * p.steps > log(1e6) ? (int)fmax(1.0, floor(log(1e6) / (2.0 * most))) : p.steps;
    TinyPoly tp{p.a, p.b, p.c, eps, p.steps, run, 0};
    const dim3 block(kThreads);
    const auto items = [](const Mat &M) { return M.batch * M.parts; };
    if (form == TINY) {
        in_chunks(g, items, [&](const Small &list, dim3 grid, int longest) {
            if (run >= p.steps && longest <= 64) hipLaunchKernelGGL((ortho_tiny<T, STEP, TINY_ALL, 64>), grid, dim3(64), 0, stream, list, tp, ws, st);
            else if (run >= p.steps) hipLaunchKernelGGL((ortho_tiny<T, STEP, TINY_ALL>), grid, block, 0, stream, list, tp, ws, st);
            else hipLaunchKernelGGL((ortho_tiny<T, STEP, TINY_ALL_SEGMENTS>), grid, block, 0, stream, list, tp, ws, st);
        });
    } else {
        for (; tp.seg * run < p.steps; ++tp.seg)
            in_chunks(g, items, [&](const Small &list, dim3 grid, int) { hipLaunchKernelGGL((ortho_tiny<T, STEP, TINY_SUMS>), grid, block, 0, stream, list, tp, ws, st); });
        in_chunks(g, items, [&](const Small &list, dim3 grid, int) { hipLaunchKernelGGL((ortho_tiny<T, STEP, TINY_APPLY>), grid, block, 0, stream, list, tp, ws, st); });
    }
    return tef::check_launch("orthogonalisation");
}

bool polynomial(Poly &p, int steps, double a, double b, double c, double eps, int first, int rest)
{
    if (steps < 1 || steps > kMaxSteps) return tef::fail("orthogonalisation: 1 to 32 steps");
    if (!(eps >= 1e-200 && eps < 1e30)) return tef::fail("orthogonalisation: eps must be positive (1e-200 at least: 1 / eps is formed)");
    p = Poly{a, b, c, steps, first, rest, 0, 0, 0.0};
    return bounded(p);
}

// What a matrix goes through, by its own size alone: its bits do not depend on the other matrices of the call.  (Tiles are planned for a
// group, though: where a product is cut along k, and with it the order of its sums, depends on the tiled matrices beside it.)
template <typename D> Form form_of(const D &d, bool step)
{
    const long m = d.rows < d.cols ? d.rows : d.cols, n = d.rows < d.cols ? d.cols : d.rows;
    if (m <= kTinySide) return n <= kTinyOne ? TINY : THIN;
    return !step && m <= kSmallSide && n <= kSmallLong ? SMALL : TILED;      // (the optimiser's momentum and parameters: tiny or tiles)
}

bool take(Mat &M, const tef_ortho_matrix &d)
{
    if (!describe(M, d.rows, d.cols, d.batch)) return false;
    if (d.src_ld < d.cols || d.dst_ld < d.cols) return tef::fail("orthogonalisation: row stride shorter than a row");
    M.src = d.src; M.dst = d.dst;
    M.src_ld = d.src_ld; M.dst_ld = d.dst_ld;
    M.src_stride = d.src_stride; M.dst_stride = d.dst_stride;
    return true;
}
bool take(Mat &M, const tef_muon_matrix &d)
{
    if (!describe(M, d.rows, d.cols, 1)) return false;
    if (d.offset < 0) return tef::fail("tef_muon_step: negative offset");
    M.src = reinterpret_cast<const void *>(d.offset); M.dst = reinterpret_cast<void *>(d.offset);
    M.src_ld = M.dst_ld = d.cols;
    M.scale = d.scale;
    return true;
}

// the list's next matrices of one form, from number `at` on (g.n = 0: no more)
template <typename D> bool next_group(Group &g, const D *m, int &at, int count, Form form, bool step)
{
    g.n = 0;
    g.bytes = 0;
    for (; at < count && g.n < kGroup; ++at)
        if (form_of(m[at], step) == form && !take(g.m[g.n++], m[at])) return false;
    if (g.n && form == TILED && !plan(g)) return false;
    if (form == THIN) plan_thin(g);
    if (form == TINY)
        for (int k = 0; k < g.n; ++k) g.m[k].parts = 1;
    return true;
}

template <typename T> int run(Group &g, Form form, const Poly &p, double eps, char *ws, hipStream_t stream)
{
    return form == TILED ? iterate<T, false>(g, p, eps, ws, Step{}, stream) : form == SMALL ? small<T>(g, p, eps, stream) : tiny<T, false>(g, form, p, eps, ws, Step{}, stream);
}

template <typename D> size_t workspace_of(const D *m, int count, bool step)
{
    if (count < 0 || (count && !m)) return tef::fail("orthogonalisation: null matrix list"), 0;
    size_t most = 256;
    Group g;
    for (int form = 0; form < FORMS; ++form)
        for (int at = 0; at < count;) {
            if (!next_group(g, m, at, count, (Form)form, step)) return 0;
            if ((size_t)g.bytes > most) most = (size_t)g.bytes;
        }
    return most;
}

}  // namespace

extern "C" {

int tef_orthogonalize_check(int steps, double a, double b, double c, double eps)
{
    Poly p;
    return polynomial(p, steps, a, b, c, eps, 2, 1) ? 0 : TEF_ERR_INVALID;
}

size_t tef_orthogonalize_workspace_bytes(const tef_ortho_matrix *matrices, int count) { return workspace_of(matrices, count, false); }

int tef_orthogonalize(const tef_ortho_matrix *matrices, int count, int dtype, int steps, double a, double b, double c, double eps,
                      void *workspace, size_t workspace_bytes, void *stream)
{
    Poly p;
    if (!polynomial(p, steps, a, b, c, eps, 2, 1)) return TEF_ERR_INVALID;
    if (dtype < TEF_F32 || dtype > TEF_BF16) return tef::fail("tef_orthogonalize: type"), TEF_ERR_INVALID;
    const size_t need = workspace_of(matrices, count, false);
    if (!need) return TEF_ERR_INVALID;
    if (count == 0) return 0;
    for (int k = 0; k < count; ++k)
        if (!matrices[k].src || !matrices[k].dst) return tef::fail("tef_orthogonalize: null pointer"), TEF_ERR_INVALID;
    if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < need)
        return tef::fail("tef_orthogonalize: workspace too small or not 256-byte aligned"), TEF_ERR_WORKSPACE;
    Group g;
    for (int f = 0; f < FORMS; ++f)
        for (int at = 0; at < count;) {
            const Form form = (Form)f;
            if (!next_group(g, matrices, at, count, form, false)) return TEF_ERR_INVALID;
            if (!g.n) break;
            const int rc = dtype == TEF_F32 ? run<float>(g, form, p, eps, (char *)workspace, (hipStream_t)stream)
                         : dtype == TEF_F16 ? run<__half>(g, form, p, eps, (char *)workspace, (hipStream_t)stream)
                                            : run<__hip_bfloat16>(g, form, p, eps, (char *)workspace, (hipStream_t)stream);
            if (rc) return rc;
        }
    return 0;
}

int tef_orthogonalize_plan(const tef_ortho_matrix *matrices, int count, int index, int optimiser, tef_ortho_plan *out)
{
    if (!out || index < 0 || index >= count) return tef::fail("tef_orthogonalize_plan: no such matrix"), TEF_ERR_INVALID;
    if (!workspace_of(matrices, count, optimiser != 0)) return TEF_ERR_INVALID;
    memset(out, 0, sizeof(*out));
    const Form form = form_of(matrices[index], optimiser != 0);
    out->form = form;
    if (form != TILED) return 0;
    Group g;
    for (int at = 0; at <= index;)
        if (!next_group(g, matrices, at, count, form, optimiser != 0)) return TEF_ERR_INVALID;
    out->gram_tile = g.ts_gram; out->gram_items = (int)g.gram.items; out->gram_joins = (int)g.gram.joins;
    out->chain_tile = g.ts_chain;
    for (int k = 0; k < 2; ++k) { out->chain_items[k] = (int)g.chain[k].items; out->chain_joins[k] = (int)g.chain[k].joins; }
    out->apply_tile = g.ts_apply;
    return 0;
}

size_t tef_muon_workspace_bytes(const tef_muon_matrix *matrices, int count) { return workspace_of(matrices, count, true); }

int tef_muon_step(float *p, float *g, float *m, float *v, const tef_muon_matrix *matrices, int nmatrices, const tef_muon_vector *vectors,
                  int nvectors, const float *norm, const double *hp, const float *step, int nesterov, int steps, double a, double b,
                  double c, double eps, void *workspace, size_t workspace_bytes, void *stream)
{
    Poly poly;
    // (segments of three steps where their q stays below 2^6: a below 4; else as orthogonalize, with the same refusals)
    if (!polynomial(poly, steps, a, b, c, eps, steps % 3 == 1 && steps > 1 ? 2 : 3, 3) && !polynomial(poly, steps, a, b, c, eps, 2, 1)) return TEF_ERR_INVALID;
    if (!p || !g || !m || !norm || !hp || !step || nvectors < 0 || (nvectors && (!vectors || !v)))
        return tef::fail("tef_muon_step: null pointer"), TEF_ERR_INVALID;
    long total = 0;
    for (int k = 0; k < nvectors; ++k) {
        if (vectors[k].offset < 0 || vectors[k].size < 1) return tef::fail("tef_muon_step: empty or misplaced vector"), TEF_ERR_INVALID;
        total += vectors[k].size;
    }
    if (total > 0x3fffffff) return tef::fail("tef_muon_step: more than 2^30 vector elements"), TEF_ERR_INVALID;
    const size_t need = workspace_of(matrices, nmatrices, true);
    if (!need) return TEF_ERR_INVALID;
    if (nmatrices && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < need))
        return tef::fail("tef_muon_step: workspace too small or not 256-byte aligned"), TEF_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    const Step s{g, m, p, norm, hp, nesterov != 0};
    Group gr;
    for (int f = 0; f < FORMS; ++f)
        for (int at = 0; at < nmatrices;) {
            const Form form = (Form)f;
            if (!next_group(gr, matrices, at, nmatrices, form, true)) return TEF_ERR_INVALID;
            if (!gr.n) break;
            const int rc = form == TILED ? iterate<float, true>(gr, poly, eps, (char *)workspace, s, st)
                                         : tiny<float, true>(gr, form, poly, eps, (char *)workspace, s, st);
            if (rc) return rc;
        }
    long v0 = 0;
    for (int at = 0; at < nvectors; at += kRanges) {
        Ranges rg;
        rg.n = nvectors - at < kRanges ? nvectors - at : kRanges;
        rg.v0 = (int)v0;
        rg.first[0] = 0;
        for (int k = 0; k < rg.n; ++k) {
            rg.off[k] = vectors[at + k].offset;
            rg.first[k + 1] = rg.first[k] + (int)vectors[at + k].size;
        }
        const int n = rg.first[rg.n];
        v0 += n;
        const int blocks = (n + kThreads - 1) / kThreads;
        hipLaunchKernelGGL(muon_vectors, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(kThreads), 0, st, rg, p, g, m, v, norm, hp, step);
    }
    return tef::check_launch("muon step");
}

}  // extern "C"
