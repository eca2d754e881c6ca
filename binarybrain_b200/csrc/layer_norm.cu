// Layer norm over the nodes of a frame, forward and backward, on fp32 and bf16 frame buffers.  (The reference normalises over the frames of a node,
// include/bb/StochasticBatchNormalization.h:521-617; it has no counterpart of this.)
//
//   forward    m = mean_n x,  v = mean_n (x - m)^2,  r = 1 / sqrt(v + eps),  y = (x - m) r gamma_n + beta_n
//   backward   xh = (x - m) r,  c1 = mean_n gamma_n dy,  c2 = mean_n gamma_n dy xh,  dx = r (gamma_n dy - c1 - xh c2),
//              dgamma_n = sum_f dy xh,  dbeta_n = sum_f dy
//
// Statistics and sums are 32 bits or more throughout; bf16 frames are widened when they are read and rounded once when they are written.  A frame of one value
// has that value for a mean and a variance of 0 in both forms below, and single nodes far from all others cost neither of them digits.
//
// The work is some ten operations a value, so memory bounds it: 8 bytes a value of fp32 forward, 12 backward, at the 6.5 TB/s of a copy.  A frame's values lie
// a row apart, but 64 or 128 bytes of every row are enough: copies in columns of such pieces run at 5.5 to 6.4 TB/s.  What costs is that a frame is needed
// whole before its first output: up to 4096 nodes (backward 4096) a cluster holds the columns and everything is read once, at two thirds to half of a copy's
// rate, bound by the phases of a CTA (three or four CTAs an SM overlap them; issue slots 30 to 45 % used); beyond, two passes at 85 to 95 % of it move
// half as much again (two thirds, backward).
#include <algorithm>

#include "frame_columns.cuh"
#include "packed_pairs.cuh"

namespace bb200 {

constexpr int kMostNodes = 1 << 20;                    // 32 rows a CTA are 32768 CTAs at most
constexpr int kNormThreads = 256;                      // of the kernels that stream over chunks of rows

// ---- two passes: statistics of the frames, then what is made of them.  The second one finds what L2 (126 MB) still holds of the first.
// (8192 x 16384 fp32: statistics 95 us, y 153; backward of 65536 x 1024: sums 103, dx and the weights' parts 119, their sums 4.)

__device__ __forceinline__ float middle(float a, float b, float c) { return fmaxf(fminf(a, b), fminf(fmaxf(a, b), c)); }

// rows first, first + step, ... below N
__device__ __forceinline__ int n_rows(int N, int first, int step) { return first < N ? (N - first + step - 1) / step : 0; }

// A cluster has the columns of 128 (few frames: 32) bytes of a row; its CTAs take turns at the rows.  Each thread adds up d = x - level and d^2 of its rows
// in 32 bits, with a level of its own: the middle one of its first three values, moved to the mean of all its rows so far after 1, 2, 4, 8, 16, 32, 48 ...
// batches, when d^2 goes to a sum of its own.  A move subtracts (sum d)^2 / count, which after the first one is at most half of what the rows since the last
// one have added to sum d^2: neither a level of the frame nor single nodes far from all others, wherever they are, cost digits (one level for all threads,
// the frame's first value, left rstd of 65536 nodes off by 7e-4 where that value was 1000 standard deviations away).  Threads of a warp move to a level in
// common, and warps and CTAs join relative to the first value in 64 bits.  A frame of one value has d = 0 at every step: its mean is that value and its
// variance 0.  Where d^2 is beyond the largest number (a node at the type's lowest one, say) the level stays, so that the mean is a number, the variance
// infinite and rstd 0.
// (64 bits in the threads, too: 8192 x 16384 bf16 76 us instead of 62.  One level for all threads, an operation a value and the moves less: 60.)
constexpr int kFoldBatches = 16;
template <typename T, int LPR, bool ALIGNED>
__global__ void __launch_bounds__(kNormThreads, 4)
k_layer_norm_stats(const T *x, float *mean_out, float *rstd_out, float eps, int N, int F, long long xs)
{
    grid_dependency();
    constexpr int kBatch = sizeof(T) == 4 ? 8 : 4;
    using Col = Column<T, LPR>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    __shared__ float red[8][3][kCols];                                    // level, mean from there, sum of squares about the mean
    __shared__ int red_rows[8];
    __shared__ double2 part[kCols];
    const Col c;
    const uint32_t cl = cluster_size(), rank = cluster_rank();
    const int f0 = (int)(blockIdx.x / cl) * kCols, f = f0 + c.col, step = c.step * (int)cl, first = (int)rank * c.step + c.row;
    float s1[kVec] = {}, s2[kVec] = {}, folded[kVec] = {}, level[kVec] = {};
    for (int n = first, k = 0; n < N; n += step * kBatch, ++k) {
        if (k > 0 && ((k & (k - 1)) == 0 || k % kFoldBatches == 0)) {
            const float count = (float)(k * kBatch), inv = 1.0f / count;
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const float to = fmaf(s1[j], inv, level[j]), d = to - level[j], moved = count * d;
                if (folded[j] + s2[j] < INFINITY) {
                    folded[j] += fmaf(d, moved - 2.0f * s1[j], s2[j]);
                    s1[j] -= moved;
                    s2[j] = 0.0f;
                    level[j] = to;
                }
            }
        }
        uint4 raw[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * step;
            if (m < N) raw[i] = load_frames<T, ALIGNED>(x + (long long)m * xs, f, F);
        }
        if (k == 0) {
            unpack<T>(raw[0], level);
            if (n + 2 * step < N) {
                float u[kVec], v[kVec];
                unpack<T>(raw[1], u);
                unpack<T>(raw[2], v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) level[j] = middle(level[j], u[j], v[j]);
            }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (n + i * step < N) {
                float v[kVec];
                unpack<T>(raw[i], v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    const float d = v[j] - level[j];
                    s1[j] += d;
                    s2[j] = fmaf(d, d, s2[j]);
                }
            }
        }
    }
    // a warp's lanes of a column take the mean of their means for a level
    const int rows = n_rows(N, first, step), warp_rows = __reduce_add_sync(0xffffffffu, rows) / LPR;
    const float count = (float)rows, inv = rows ? 1.0f / count : 0.0f, inv_warp = warp_rows ? 1.0f / (float)warp_rows : 0.0f;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        const float mean = fmaf(s1[j], inv, level[j]), start = __shfl_sync(0xffffffffu, mean, c.lane % LPR);
        float to = (mean - start) * (count * inv_warp);
#pragma unroll
        for (int m = LPR; m < 32; m <<= 1) to += __shfl_xor_sync(0xffffffffu, to, m);
        to += start;
        const float d = to - level[j], moved = count * d;
        const float squares = folded[j] + s2[j];
        s2[j] = !rows ? 0.0f : squares < INFINITY ? fmaf(d, moved - 2.0f * s1[j], squares) : squares;
        s1[j] = rows ? s1[j] - moved : 0.0f;
        level[j] = to;
#pragma unroll
        for (int m = LPR; m < 32; m <<= 1) {
            s1[j] += __shfl_xor_sync(0xffffffffu, s1[j], m);
            s2[j] += __shfl_xor_sync(0xffffffffu, s2[j], m);
        }
    }
    if (c.lane < LPR) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            const float off = s1[j] * inv_warp;
            red[c.warp][0][c.col + j] = level[j];
            red[c.warp][1][c.col + j] = off;
            red[c.warp][2][c.col + j] = s2[j] < INFINITY ? fmaf(-s1[j], off, s2[j]) : s2[j];
        }
        if (c.lane == 0) red_rows[c.warp] = warp_rows;
    }
    __syncthreads();
    const bool has = threadIdx.x < kCols && f0 + (int)threadIdx.x < F;
    const double start = has ? (double)to_float(x[f0 + threadIdx.x]) : 0.0;
    if (threadIdx.x < kCols) {
        double2 t = make_double2(0.0, 0.0);
        for (int w = 0; w < c.warps; ++w) {
            const double n = (double)red_rows[w], d = (double)red[w][0][threadIdx.x] - start + (double)red[w][1][threadIdx.x];
            if (n > 0.0) { t.x += n * d; t.y += (double)red[w][2][threadIdx.x] + n * d * d; }
        }
        part[threadIdx.x] = t;
    }
    if (cl > 1) { cluster_arrive(); cluster_wait(); }
    if (rank == 0 && has) {
        double2 t = part[threadIdx.x];
        for (uint32_t r = 1; r < cl; ++r) {
            const double2 p = peer_load_double2(&part[threadIdx.x], r);
            t.x += p.x;
            t.y += p.y;
        }
        t.x /= (double)N;
        double var = t.y / (double)N - t.x * t.x;
        if (var < 0.0) var = 0.0;                                         // (and a NaN stays one)
        mean_out[f0 + threadIdx.x] = (float)(start + t.x);
        rstd_out[f0 + threadIdx.x] = 1.0f / sqrtf((float)var + eps);
    }
    if (cl > 1) { cluster_arrive(); cluster_wait(); }                     // nobody leaves while its sums may still be read
}

// Along the rows: a warp takes 512 bytes of a row, a CTA 8 x kApplyRows rows, which share the frames' statistics.
constexpr int kApplyRows = 8;
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kNormThreads)
k_layer_norm_apply(const T *x, T *y, const float *__restrict__ gamma, const float *__restrict__ beta, const float *__restrict__ mean_in,
                   const float *__restrict__ rstd_in, int N, int F, long long xs, long long ys)
{
    grid_dependency();
    constexpr int kVec = kFramesPerVec<T>;
    const Line<T, ALIGNED> line((int)blockIdx.x * 32 * kVec, (int)(threadIdx.x & 31), F);
    const int n0 = ((int)blockIdx.y * 8 + (int)(threadIdx.x >> 5)) * kApplyRows;
    if (line.empty()) return;
    uint4 raw[kApplyRows];
#pragma unroll
    for (int i = 0; i < kApplyRows; ++i)
        if (n0 + i < N) raw[i] = line.load(x + (long long)(n0 + i) * xs);
    float mean[kVec], rstd[kVec];
    line.load_columns(mean_in, mean);
    line.load_columns(rstd_in, rstd);
#pragma unroll
    for (int i = 0; i < kApplyRows; ++i) {
        if (n0 + i < N) {
            const float g = gamma ? gamma[n0 + i] : 1.0f, b = beta ? beta[n0 + i] : 0.0f;
            float v[kVec];
            unpack<T>(raw[i], v);
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[j] = fmaf((v[j] - mean[j]) * rstd[j], g, b);
            line.store(y + (long long)(n0 + i) * ys, v);
        }
    }
}

// backward: sums[frame] = mean_n gamma dy, sums[padded + frame] = mean_n gamma dy xh
template <typename T, int LPR, bool ALIGNED>
__global__ void __launch_bounds__(kNormThreads, 4)
k_layer_norm_grad_stats(const T *x, const T *dy, const float *__restrict__ gamma, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                        float *sums_out, int padded, int N, int F, long long xs, long long dys)
{
    grid_dependency();
    constexpr int kBatch = sizeof(T) == 4 ? 4 : 2;
    using Col = Column<T, LPR>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    __shared__ float red[8][2 * kCols];
    __shared__ float part[2 * kCols];
    const Col c;
    const uint32_t cl = cluster_size(), rank = cluster_rank();
    const int f0 = (int)(blockIdx.x / cl) * kCols, f = f0 + c.col, step = c.step * (int)cl;
    float mean[kVec], s[2][kVec] = {};
    load_columns(mean_in, f, F, mean);
    for (int n = (int)rank * c.step + c.row; n < N; n += step * kBatch) {
        uint4 xr[kBatch], gr[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * step;
            if (m < N) {
                xr[i] = load_frames<T, ALIGNED>(x + (long long)m * xs, f, F);
                gr[i] = load_frames<T, ALIGNED>(dy + (long long)m * dys, f, F);
            }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * step;
            if (m < N) {
                const float gm = gamma ? gamma[m] : 1.0f;
                float xv[kVec], gv[kVec];
                unpack<T>(xr[i], xv);
                unpack<T>(gr[i], gv);
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    const float g = gm * gv[j];
                    s[0][j] += g;
                    s[1][j] = fmaf(g, xv[j] - mean[j], s[1][j]);          // times rstd at the end
                }
            }
        }
    }
#pragma unroll
    for (int m = LPR; m < 32; m <<= 1)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int j = 0; j < kVec; ++j) s[q][j] += __shfl_xor_sync(0xffffffffu, s[q][j], m);
    if (c.lane < LPR) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int j = 0; j < kVec; ++j) red[c.warp][q * kCols + c.col + j] = s[q][j];
    }
    __syncthreads();
    if (threadIdx.x < 2 * kCols) {
        float t = red[0][threadIdx.x];
        for (int w = 1; w < c.warps; ++w) t += red[w][threadIdx.x];
        part[threadIdx.x] = t;
    }
    if (cl > 1) { cluster_arrive(); cluster_wait(); } else __syncthreads();
    if (rank == 0 && threadIdx.x < kCols && f0 + (int)threadIdx.x < F) {
        float a = 0.0f, b = 0.0f;
        for (uint32_t r = 0; r < cl; ++r) { a += peer_load(&part[threadIdx.x], r); b += peer_load(&part[kCols + threadIdx.x], r); }
        sums_out[f0 + threadIdx.x] = a / (float)N;
        // (where rstd is 0 every xh is, though x - mean may have been too much for a sum)
        const float rstd = rstd_in[f0 + threadIdx.x];
        sums_out[padded + f0 + threadIdx.x] = rstd == 0.0f ? 0.0f : b * rstd / (float)N;
    }
    if (cl > 1) { cluster_arrive(); cluster_wait(); }
}

// Along the rows again: a CTA has 8 x R rows and every gridDim.x-th piece of 512 bytes of them, and adds up their sums over the frames on the way:
// grad_part[blockIdx.x][node] = (sum dy xh, sum dy)
template <typename T, int R, bool ALIGNED>
__global__ void __launch_bounds__(kNormThreads, 2)
k_layer_norm_grad_apply(const T *x, const T *dy, T *dx, const float *__restrict__ sums, int padded, const float *__restrict__ gamma, const float *__restrict__ mean_in,
                        const float *__restrict__ rstd_in, float2 *grad_part, int N, int F, long long xs, long long dys, long long dxs)
{
    grid_dependency();
    constexpr int kVec = kFramesPerVec<T>;
    const int lane = threadIdx.x & 31, n0 = ((int)blockIdx.y * 8 + (int)(threadIdx.x >> 5)) * R;
    float ag[R] = {}, ab[R] = {}, gm[R];
#pragma unroll
    for (int i = 0; i < R; ++i) gm[i] = gamma && n0 + i < N ? gamma[n0 + i] : 1.0f;
    for (int f0 = (int)blockIdx.x * 32 * kVec; f0 < F; f0 += (int)gridDim.x * 32 * kVec) {
        const Line<T, ALIGNED> line(f0, lane, F);
        if (line.empty()) break;
        uint4 xr[R], gr[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (n0 + i < N) {
                xr[i] = line.load(x + (long long)(n0 + i) * xs);
                gr[i] = line.load(dy + (long long)(n0 + i) * dys);
            }
        }
        float mean[kVec], rstd[kVec], k1[kVec], k2[kVec];                 // dx = (gamma rstd) dy + k1 + k2 xh
        line.load_columns(mean_in, mean);
        line.load_columns(rstd_in, rstd);
        line.load_columns(sums, k1);
        line.load_columns(sums + padded, k2);
#pragma unroll
        for (int j = 0; j < kVec; ++j) { k1[j] *= -rstd[j]; k2[j] *= -rstd[j]; }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (n0 + i < N) {
                float xv[kVec], gv[kVec];
                unpack<T>(xr[i], xv);
                unpack<T>(gr[i], gv);
                if (line.frame(kVec - 1) >= F) {                          // what lies beyond the frames may be anything
#pragma unroll
                    for (int j = 0; j < kVec; ++j)
                        if (line.frame(j) >= F) xv[j] = gv[j] = 0.0f;
                }
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    const float xh = (xv[j] - mean[j]) * rstd[j];
                    ag[i] = fmaf(gv[j], xh, ag[i]);
                    ab[i] += gv[j];
                    gv[j] = fmaf(gv[j], gm[i] * rstd[j], fmaf(xh, k2[j], k1[j]));
                }
                line.store(dx + (long long)(n0 + i) * dxs, gv);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) {
            ag[i] += __shfl_xor_sync(0xffffffffu, ag[i], m);
            ab[i] += __shfl_xor_sync(0xffffffffu, ab[i], m);
        }
        if (lane == i && n0 + i < N) grad_part[(long long)blockIdx.x * N + n0 + i] = make_float2(ag[i], ab[i]);
    }
}

// ---- layers whose columns a cluster holds in shared memory: everything is read once.  The clusters walk over the column tiles; each thread brings its
// own 16-byte pieces, reads them back for the statistics and for the output, and sends for those of the next tile.  The CTAs of an SM are in different
// phases of this, so that the memory system does not wait for an exchange of sums.  Rows on 16-byte boundaries.
template <typename T>
__device__ __forceinline__ void fetch_rows(uint8_t *to, int piece, const T *from, long long distance, int rows)
{
    to += threadIdx.x * 16;
#pragma unroll 4
    for (int i = 0; i < rows; ++i, to += piece, from += distance) cp_async16(to, from, true);
}

// (A sum over all rows times 1 / N, one operation a value less, is off by a rounding for equal values: y by 0.02 at a level of 1000.  The operations in pairs
// pay for it: 4096 x 8192 fp32 61.5 us with that sum, 58 now; a single frame of 1024, in a graph, 4.85 and 5.05.)
// Means of rows joined to their mean with weights that are the shares of the rows, each part as its distance from the first one: means that are equal stay
// what they are, so that a frame of one value has that value for a mean and nothing but zeros about it.
template <typename T, int LPR> struct MeanWeights {
    float mine, lane;                                                     // 1 / rows of the thread; their share of the warp's
    float (&shared)[2][8];                                                // the shares of the CTA's warps and of the cluster's CTAs

    // rows: of this thread, cta_rows: of a CTA at most; a barrier stands between this and the first use
    __device__ __forceinline__ MeanWeights(const Column<T, LPR> &c, const Cluster &cl, float (&shared)[2][8], int rows, int cta_rows, int N) : shared(shared)
    {
        const int count = max(rows, 0), warp = __reduce_add_sync(0xffffffffu, count) / LPR;
        auto of_cta = [&](uint32_t r) { return (float)min(max(N - (int)r * cta_rows, 0), cta_rows); };
        mine = count ? __fdividef(1.0f, (float)count) : 0.0f;
        lane = count ? __fdividef((float)count, (float)warp) : 0.0f;
        if (c.lane == 0) shared[0][c.warp] = warp ? __fdividef((float)warp, of_cta(cl.rank)) : 0.0f;
        if (threadIdx.x < cl.size) shared[1][threadIdx.x] = __fdividef(of_cta(threadIdx.x), (float)N);
    }
    template <int WHAT> __device__ __forceinline__ float join_parts(const float *from, int distance, int count) const      // up to eight, all of them on their way first
    {
        const float4 lower = *reinterpret_cast<const float4 *>(shared[WHAT]), upper = *reinterpret_cast<const float4 *>(shared[WHAT] + 4);
        const float w[8] = {lower.x, lower.y, lower.z, lower.w, upper.x, upper.y, upper.z, upper.w};
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < count ? from[i * distance] : 0.0f;
        float s = 0.0f;
#pragma unroll
        for (int i = 1; i < 8; ++i)
            if (i < count) s = fmaf(v[i] - v[0], w[i], s);
        return v[0] + s;
    }
    // v: of this thread's rows, then of all rows of the tile
    __device__ __forceinline__ void join(float (&v)[1][kFramesPerVec<T>], const Column<T, LPR> &c, Exchange<1, LPR * kFramesPerVec<T>> &e, const Cluster &cl, uint32_t phase) const
    {
#pragma unroll
        for (int j = 0; j < kFramesPerVec<T>; ++j) {
            const float start = __shfl_sync(0xffffffffu, v[0][j], c.lane % LPR);
            float off = (v[0][j] - start) * lane;
#pragma unroll
            for (int m = LPR; m < 32; m <<= 1) off += __shfl_xor_sync(0xffffffffu, off, m);
            v[0][j] = start + off;
        }
        exchange_columns<1, T, LPR>(v, c, e, cl, phase, [&](const float *from, int distance, int count) { return join_parts<0>(from, distance, count); },
                                    [&](const float *from, int distance, int count) { return join_parts<1>(from, distance, count); }, [](int, float m) { return m; });
    }
};

template <typename T, int LPR>
__global__ void __launch_bounds__(kColumnThreads, 4)
k_layer_norm_once(const T *x, T *y, const float *__restrict__ gamma, const float *__restrict__ beta, float *mean_out, float *rstd_out, float eps, int N, int F,
                  long long xs, long long ys, int rows, int tiles, int *fault)
{
    grid_dependency();
    using Col = Column<T, LPR>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    extern __shared__ __align__(16) uint8_t buffer[];
    __shared__ Exchange<1, kCols> sums[2];
    __shared__ __align__(16) float shares[2][8];
    __shared__ int gave_up;
    const Col c;
    Cluster cl(&gave_up);
    const int clusters = (int)(gridDim.x / cl.size), cta_first = (int)cl.rank * c.step * rows, first = cta_first + c.row, piece = blockDim.x * 16;
    const int mine = min(rows, (N - first + c.step - 1) / c.step);         // rows of this thread that exist (none: 0 or less)
    float2 *const gain = reinterpret_cast<float2 *>(buffer + rows * piece);
    const uint8_t *const at = buffer + threadIdx.x * 16;
    const long long x_step = c.step * xs, y_step = c.step * ys;
    const T *const x_first = x + first * xs;
    int tile = (int)(blockIdx.x / cl.size), f = tile * kCols + c.col;
    uint32_t phase = 0;
    if (f < F) fetch_rows(buffer, piece, x_first + f, x_step, mine);
    auto gain_at = [&](int i) { return cta_first + i < N ? make_float2(gamma ? gamma[cta_first + i] : 1.0f, beta ? beta[cta_first + i] : 0.0f) : make_float2(0.0f, 0.0f); };
    const float2 first_gain = gain_at(threadIdx.x);                       // on its way beside the shares of the rows
    const MeanWeights<T, LPR> weights(c, cl, shares, mine, c.step * rows, N);
    if ((int)threadIdx.x < c.step * rows) gain[threadIdx.x] = first_gain;
    for (int i = threadIdx.x + blockDim.x; i < c.step * rows; i += blockDim.x) gain[i] = gain_at(i);
    cl.meet(sums, gain + c.step * rows);
    const float inv = 1.0f / (float)N;
    for (; tile < tiles; tile += clusters, f += clusters * kCols, phase ^= 1) {
        cp_async_commit();
        cp_async_wait<0>();
        float mean[1][kVec] = {}, rstd[1][kVec] = {};
        if (mine > 0) {                                                   // about one of the first two values, the smaller one: far nodes stay out of it
            float level[kVec], v[kVec];
            unpack<T>(*reinterpret_cast<const uint4 *>(at), level);
            unpack<T>(*reinterpret_cast<const uint4 *>(at + (mine > 1 ? piece : 0)), v);
#pragma unroll
            for (int j = 0; j < kVec; ++j) level[j] = fabsf(v[j]) < fabsf(level[j]) ? v[j] : level[j];
            f32x2 sum[kVec / 2], from[kVec / 2];
#pragma unroll
            for (int j = 0; j < kVec / 2; ++j) { sum[j] = pack2(0.0f, 0.0f); from[j] = pack2(level[2 * j], level[2 * j + 1]); }
            const uint8_t *p = at;
#pragma unroll 2
            for (int i = 0; i < mine; ++i, p += piece) {
                float v[kVec];
                unpack<T>(*reinterpret_cast<const uint4 *>(p), v);
#pragma unroll
                for (int j = 0; j < kVec / 2; ++j) sum[j] = add2(sum[j], sub2(pack2(v[2 * j], v[2 * j + 1]), from[j]));
            }
#pragma unroll
            for (int j = 0; j < kVec / 2; ++j) unpack2(fma2(sum[j], pack2(weights.mine, weights.mine), from[j]), mean[0][2 * j], mean[0][2 * j + 1]);
        }
        weights.join(mean, c, sums[0], cl, phase);
        {
            const uint8_t *p = at;
#pragma unroll 4
            for (int i = 0; i < mine; ++i, p += piece) {
                float v[kVec];
                unpack<T>(*reinterpret_cast<const uint4 *>(p), v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) { v[j] -= mean[0][j]; rstd[0][j] = fmaf(v[j], v[j], rstd[0][j]); }
            }
        }
        join_columns<ColumnSum, 1, T, LPR>(rstd, c, sums[1], cl, phase, [&](int, float s) { return 1.0f / sqrtf(fmaf(s, inv, eps)); });
        if (cl.rank == 0 && c.row == 0) {
#pragma unroll
            for (int j = 0; j < kVec; ++j)
                if (f + j < F) { mean_out[f + j] = mean[0][j]; rstd_out[f + j] = rstd[0][j]; }
        }
        const uint8_t *p = at;
        const float2 *g = gain + c.row;
        T *out = y + first * ys;
#pragma unroll 4
        for (int i = 0; i < mine; ++i, p += piece, g += c.step, out += y_step) {
            const float2 gb = *g;
            float v[kVec];
            unpack<T>(*reinterpret_cast<const uint4 *>(p), v);
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[j] = fmaf((v[j] - mean[0][j]) * rstd[0][j], gb.x, gb.y);
            store_frames<T, true>(out, f, F, v);
        }
        if (f + clusters * kCols < F) fetch_rows(buffer, piece, x_first + f + clusters * kCols, x_step, mine);
    }
    cl.leave(fault);
}

// R rows a thread at most; the sums over the frames of a node stay in registers on the way: grad_part[cluster][node] = (sum dy xh, sum dy)
template <typename T, int LPR, int R>
__global__ void __launch_bounds__(kColumnThreads, 3)
k_layer_norm_grad_once(const T *x, const T *dy, T *dx, const float *__restrict__ gamma, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                       float2 *grad_part, int N, int F, long long xs, long long dys, long long dxs, int rows, int tiles, int *fault)
{
    grid_dependency();
    using Col = Column<T, LPR>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    extern __shared__ __align__(16) uint8_t buffer[];
    __shared__ Exchange<2, kCols> sums[2];
    __shared__ int gave_up;
    const Col c;
    Cluster cl(&gave_up);
    const int cluster = (int)(blockIdx.x / cl.size), clusters = (int)(gridDim.x / cl.size), first = (int)cl.rank * c.step * rows + c.row, piece = blockDim.x * 16;
    const int mine = min(rows, (N - first + c.step - 1) / c.step), half = rows * piece;
    float *const gain = reinterpret_cast<float *>(buffer + 2 * half);
    const uint8_t *const at = buffer + threadIdx.x * 16;
    const float inv = 1.0f / (float)N;
    const long long x_step = c.step * xs, dy_step = c.step * dys, dx_step = c.step * dxs;
    const T *const x_first = x + first * xs, *const dy_first = dy + first * dys;
    int tile = cluster, f = tile * kCols + c.col;
    if (f < F) {
        fetch_rows(buffer, piece, x_first + f, x_step, mine);
        fetch_rows(buffer + half, piece, dy_first + f, dy_step, mine);
    }
    for (int i = threadIdx.x; i < c.step * rows; i += blockDim.x) gain[i] = gamma && first - c.row + i < N ? gamma[first - c.row + i] : 1.0f;
    float ag[R] = {}, ab[R] = {};
    __syncthreads();
    cl.meet(sums, gain + (c.step * rows + 3) / 4 * 4);
    uint32_t turn = 0;                                                    // the exchange is its lowest bit, the phase the next
    for (; tile < tiles; tile += clusters, f += clusters * kCols, ++turn) {
        cp_async_commit();
        float mean[kVec], rstd[kVec], s[2][kVec] = {};
        load_columns(mean_in, f, F, mean);
        load_columns(rstd_in, f, F, rstd);
        cp_async_wait<0>();
        if (f < F && f + kVec > F) {                                      // what lies beyond the frames may be anything
            for (int i = 0; i < mine; ++i)
#pragma unroll
                for (int j = 0; j < kVec; ++j)
                    if (f + j >= F) {
                        reinterpret_cast<T *>(buffer + threadIdx.x * 16 + i * piece)[j] = from_float<T>(0.0f);
                        reinterpret_cast<T *>(buffer + threadIdx.x * 16 + half + i * piece)[j] = from_float<T>(0.0f);
                    }
        }
        if (f < F) {
            const uint8_t *p = at;
            const float *g = gain + c.row;
#pragma unroll
            for (int i = 0; i < R; ++i, p += piece, g += c.step) {
                if (i >= mine) break;
                const float gm = *g;
                float xv[kVec], gv[kVec];
                unpack<T>(*reinterpret_cast<const uint4 *>(p), xv);
                unpack<T>(*reinterpret_cast<const uint4 *>(p + half), gv);
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    const float xh = (xv[j] - mean[j]) * rstd[j], t = gm * gv[j];
                    ag[i] = fmaf(gv[j], xh, ag[i]);
                    ab[i] += gv[j];
                    s[0][j] += t;
                    s[1][j] = fmaf(t, xh, s[1][j]);
                }
            }
        }
        join_columns<ColumnSum, 2, T, LPR>(s, c, sums[turn & 1], cl, turn >> 1 & 1, [&](int, float v) { return v * inv; });
        // dx = rstd (gamma dy - c1 - (c2 rstd) (x - mean)): no power of rstd, which is 1e18 for spreads of 1e-18 and the reverse
#pragma unroll
        for (int j = 0; j < kVec; ++j) s[1][j] *= rstd[j];
        if (f < F) {
            const uint8_t *p = at;
            const float *g = gain + c.row;
            T *out = dx + first * dxs;
#pragma unroll
            for (int i = 0; i < R; ++i, p += piece, g += c.step, out += dx_step) {
                if (i >= mine) break;
                const float gm = *g;
                float xv[kVec], gv[kVec];
                unpack<T>(*reinterpret_cast<const uint4 *>(p), xv);
                unpack<T>(*reinterpret_cast<const uint4 *>(p + half), gv);
#pragma unroll
                for (int j = 0; j < kVec; ++j) gv[j] = rstd[j] * fmaf(gv[j], gm, -fmaf(xv[j] - mean[j], s[1][j], s[0][j]));
                store_frames<T, true>(out, f, F, gv);
            }
        }
        if (f + clusters * kCols < F) {
            fetch_rows(buffer, piece, x_first + f + clusters * kCols, x_step, mine);
            fetch_rows(buffer + half, piece, dy_first + f + clusters * kCols, dy_step, mine);
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int n = first + i * c.step;
#pragma unroll
        for (int m = 1; m < LPR; m <<= 1) {
            ag[i] += __shfl_xor_sync(0xffffffffu, ag[i], m);
            ab[i] += __shfl_xor_sync(0xffffffffu, ab[i], m);
        }
        if (i < mine && c.lane % LPR == 0) grad_part[(long long)cluster * N + n] = make_float2(ag[i], ab[i]);
    }
    cl.leave(fault);
}

// dgamma, dbeta (either may be absent) = or += the sums of the parts, 8 parts side by side and in a fixed order
__global__ void __launch_bounds__(256)
k_layer_norm_grad_weights(const float2 *__restrict__ grad_part, float *dgamma, float *dbeta, int N, int parts, int accumulate)
{
    grid_dependency();
    __shared__ float2 s[8][32];
    const int n = (int)blockIdx.x * 32 + (threadIdx.x & 31);
    float2 a = make_float2(0.0f, 0.0f);
    if (n < N)
        for (int k = threadIdx.x >> 5; k < parts; k += 8) {
            const float2 p = grad_part[(long long)k * N + n];
            a.x += p.x;
            a.y += p.y;
        }
    s[threadIdx.x >> 5][threadIdx.x & 31] = a;
    __syncthreads();
    if (threadIdx.x < 32 && n < N) {
        for (int k = 1; k < 8; ++k) {
            a.x += s[k][threadIdx.x].x;
            a.y += s[k][threadIdx.x].y;
        }
        if (dgamma) dgamma[n] = accumulate ? dgamma[n] + a.x : a.x;
        if (dbeta) dbeta[n] = accumulate ? dbeta[n] + a.y : a.y;
    }
}

// dgamma = dbeta = 0 of a batch without frames
__global__ void __launch_bounds__(256) k_layer_norm_no_frames(float *dgamma, float *dbeta, int N)
{
    grid_dependency();
    const int n = (int)blockIdx.x * 256 + threadIdx.x;
    if (n < N && dgamma) dgamma[n] = 0.0f;
    if (n < N && dbeta) dbeta[n] = 0.0f;
}

constexpr int kNormRows = 16, kNormGradRows = 8;         // rows a thread where everything is read once, at most
constexpr int kNormSmem = 120 * 1024;                    // more than either direction's tile, weights and parts take

template <typename T, int LPR>
static int layer_norm_once(const T *x, T *y, const float *gamma, const float *beta, float *mean, float *rstd, float eps, int N, int F, long long xs,
                           long long ys, const ColumnPlan &p, cudaStream_t st)
{
    constexpr int kCols = Column<T, LPR>::kCols;
    int *fault = fault_word();
    BB200_REQUIRE(fault != nullptr, BBCU_ERR_NO_DEVICE);
    auto kernel = k_layer_norm_once<T, LPR>;
    const int threads = 32 * p.warps, smem = p.rows * threads * 16 + p.rows * p.warps * (32 / LPR) * (int)sizeof(float2) + exchange_bytes<1, kCols>(p.cluster),
              tiles = (F + kCols - 1) / kCols;
    BB200_REQUIRE(allow_big_smem(kernel, kNormSmem), (int)cudaErrorInvalidValue);
    const int clusters = std::min(tiles, resident_clusters(reinterpret_cast<const void *>(kernel), p.cluster, threads, smem));
    return launch_cluster(kernel, (unsigned)p.cluster, (unsigned)(clusters * p.cluster), threads, smem, st, x, y, gamma, beta, mean, rstd, eps, N, F, xs, ys, p.rows,
                          tiles, fault);
}

template <typename T, int LPR, int R>
static int layer_norm_grad_once(const T *x, const T *dy, T *dx, const float *gamma, const float *mean, const float *rstd, float *dgamma, float *dbeta,
                                int accumulate, int N, int F, long long xs, long long dys, long long dxs, const ColumnPlan &p, cudaStream_t st)
{
    constexpr int kCols = Column<T, LPR>::kCols;
    int *fault = fault_word();
    BB200_REQUIRE(fault != nullptr, BBCU_ERR_NO_DEVICE);
    auto kernel = k_layer_norm_grad_once<T, LPR, R>;
    const int threads = 32 * p.warps, smem = 2 * p.rows * threads * 16 + (p.rows * p.warps * (32 / LPR) + 3) / 4 * 4 * (int)sizeof(float) +
              exchange_bytes<2, kCols>(p.cluster), tiles = (F + kCols - 1) / kCols;
    BB200_REQUIRE(allow_big_smem(kernel, kNormSmem), (int)cudaErrorInvalidValue);
    const int clusters = std::min(tiles, resident_clusters(reinterpret_cast<const void *>(kernel), p.cluster, threads, smem));
    HeldScratch held;
    float2 *part = static_cast<float2 *>(held.get(st, (size_t)clusters * N * sizeof(float2)));
    BB200_REQUIRE(part != nullptr, BBCU_ERR_NO_MEMORY);
    const int e = launch_cluster(kernel, (unsigned)p.cluster, (unsigned)(clusters * p.cluster), threads, smem, st, x, dy, dx, gamma, mean, rstd, part, N, F, xs, dys,
                                 dxs, p.rows, tiles, fault);
    if (e != BBCU_OK) return e;
    if (dgamma || dbeta) launch(k_layer_norm_grad_weights, (unsigned)((N + 31) / 32), 256, 0, st, part, dgamma, dbeta, N, clusters, accumulate);
    return launch_status();
}

template <typename T>
static int layer_norm_forward(const T *x, T *y, const float *gamma, const float *beta, float *mean, float *rstd, float eps, int N, int F, long long xs,
                              long long ys, cudaStream_t st)
{
    const bool aligned = frames_aligned<T>(x, xs) && frames_aligned<T>(y, ys);
    BB200_REQUIRE(F <= (1 << 30), BBCU_ERR_TOO_LARGE);
    // us a pass, once / two passes: 4096 x 8192 fp32 58 / 68, 3000 x 5001 31 / 34; backward 4096 x 16384 bf16 123 / 137, fp32 189 / 224.  Larger clusters than
    // these lose to the two passes, larger ones of the backward than 8, too (8192 x 16384 fp32 251 / 253, bf16 158 / 140; backward 8192 x 8192 fp32 225 / 223).
    if (const ColumnPlan p = plan_columns<T>(N, F, sizeof(T) == 4 ? 8 : 4, kNormRows, sizeof(T) == 4 ? 8 : 4); aligned && p.cluster)
        return (p.lanes == 2 ? layer_norm_once<T, 2> : layer_norm_once<T, sizeof(T) == 4 ? 8 : 4>)(x, y, gamma, beta, mean, rstd, eps, N, F, xs, ys, p, st);
    constexpr int kWide = 32 * kFramesPerVec<T>;
    const long long bands = ((long long)N + 8 * kApplyRows - 1) / (8 * kApplyRows);
    BB200_REQUIRE(bands <= 65535, BBCU_ERR_TOO_LARGE);
    const StreamingPlan s = plan_streaming<T>(N, F);
    auto stats = s.lanes == 2 ? (aligned ? k_layer_norm_stats<T, 2, true> : k_layer_norm_stats<T, 2, false>)
                              : (aligned ? k_layer_norm_stats<T, 8, true> : k_layer_norm_stats<T, 8, false>);
    if (const int e = launch_cluster(stats, s.cluster, s.ctas, kNormThreads, 0, st, x, mean, rstd, eps, N, F, xs)) return e;
    launch(aligned ? k_layer_norm_apply<T, true> : k_layer_norm_apply<T, false>, dim3((unsigned)((F + kWide - 1) / kWide), (unsigned)bands), kNormThreads, 0, st, x, y, gamma,
           beta, mean, rstd, N, F, xs, ys);
    return launch_status();
}

template <typename T>
static int layer_norm_backward(const T *x, const T *dy, T *dx, const float *gamma, const float *mean, const float *rstd, float *dgamma, float *dbeta,
                               int accumulate, int N, int F, long long xs, long long dys, long long dxs, cudaStream_t st)
{
    const bool aligned = frames_aligned<T>(x, xs) && frames_aligned<T>(dy, dys) && frames_aligned<T>(dx, dxs);
    BB200_REQUIRE(F <= (1 << 30), BBCU_ERR_TOO_LARGE);
    const bool wide = N <= 8 * kColumnThreads / 8 * 4;                    // 128 bytes of a row and four rows a thread in clusters of up to 8, or 64 and eight
    if (const ColumnPlan p = plan_columns<T>(N, F, wide ? 8 : 4, wide ? 4 : kNormGradRows, 8); aligned && p.cluster) {
#define BB200_ONCE(L) (p.rows <= 4 ? layer_norm_grad_once<T, L, 4> : layer_norm_grad_once<T, L, kNormGradRows>)
        return (p.lanes == 2 ? BB200_ONCE(2) : p.lanes == 4 ? BB200_ONCE(4) : layer_norm_grad_once<T, 8, 4>)(x, dy, dx, gamma, mean, rstd, dgamma, dbeta, accumulate, N,
                                                                                                        F, xs, dys, dxs, p, st);
#undef BB200_ONCE
    }
    constexpr int kWide = 32 * kFramesPerVec<T>, kRows = 4;
    const long long bands = ((long long)N + 8 * kRows - 1) / (8 * kRows), pieces = ((long long)F + kWide - 1) / kWide;
    BB200_REQUIRE(bands <= 65535, BBCU_ERR_TOO_LARGE);
    long long sweeps = std::min(pieces, std::max(1LL, (8LL * device_info().sm_count + bands - 1) / bands));
    const int padded = (F + 3) / 4 * 4;
    const size_t sums_bytes = (size_t)padded * sizeof(float2);
    HeldScratch held;
    char *scratch = static_cast<char *>(held.get(st, sums_bytes + (size_t)sweeps * N * sizeof(float2)));
    BB200_REQUIRE(scratch != nullptr, BBCU_ERR_NO_MEMORY);
    float *sums = reinterpret_cast<float *>(scratch);
    float2 *grad_part = reinterpret_cast<float2 *>(scratch + sums_bytes);
    const StreamingPlan s = plan_streaming<T>(N, F);
    auto stats = s.lanes == 2 ? (aligned ? k_layer_norm_grad_stats<T, 2, true> : k_layer_norm_grad_stats<T, 2, false>)
                              : (aligned ? k_layer_norm_grad_stats<T, 8, true> : k_layer_norm_grad_stats<T, 8, false>);
    if (const int e = launch_cluster(stats, s.cluster, s.ctas, kNormThreads, 0, st, x, dy, gamma, mean, rstd, sums, padded, N, F, xs, dys)) return e;
    launch(aligned ? k_layer_norm_grad_apply<T, kRows, true> : k_layer_norm_grad_apply<T, kRows, false>, dim3((unsigned)sweeps, (unsigned)bands), kNormThreads, 0, st, x, dy,
           dx, sums, padded, gamma, mean, rstd, grad_part, N, F, xs, dys, dxs);
    BB200_CUDA(cudaPeekAtLastError());
    if (dgamma || dbeta) launch(k_layer_norm_grad_weights, (unsigned)((N + 31) / 32), 256, 0, st, grad_part, dgamma, dbeta, N, (int)sweeps, accumulate);
    return launch_status();
}

template <typename T>
static int layer_norm_forward_checked(const T *x, T *y, const float *gamma, const float *beta, float *mean, float *rstd, float eps, int N, int F, int xs,
                                      int ys, bbcu_stream_t stream)
{
    BB200_REQUIRE(N > 0 && F >= 0 && eps >= 0.0f, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(N <= kMostNodes, BBCU_ERR_TOO_LARGE);
    BB200_REQUIRE(xs >= F && ys >= F, BBCU_ERR_BAD_STRIDE);
    if (F == 0) return BBCU_OK;
    BB200_REQUIRE_PTR(x); BB200_REQUIRE_PTR(y); BB200_REQUIRE_PTR(mean); BB200_REQUIRE_PTR(rstd);
    return layer_norm_forward<T>(x, y, gamma, beta, mean, rstd, eps, N, F, xs, ys, as_stream(stream));
}

template <typename T>
static int layer_norm_backward_checked(const T *x, const T *dy, T *dx, const float *gamma, const float *mean, const float *rstd, float *dgamma, float *dbeta,
                                       int accumulate, int N, int F, int xs, int dys, int dxs, bbcu_stream_t stream)
{
    BB200_REQUIRE(N > 0 && F >= 0, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(N <= kMostNodes, BBCU_ERR_TOO_LARGE);
    BB200_REQUIRE(xs >= F && dys >= F && dxs >= F, BBCU_ERR_BAD_STRIDE);
    if (F == 0) {
        if (!accumulate && (dgamma || dbeta)) launch(k_layer_norm_no_frames, (unsigned)((N + 255) / 256), 256, 0, as_stream(stream), dgamma, dbeta, N);
        return launch_status();
    }
    BB200_REQUIRE_PTR(x); BB200_REQUIRE_PTR(dy); BB200_REQUIRE_PTR(dx); BB200_REQUIRE_PTR(mean); BB200_REQUIRE_PTR(rstd);
    return layer_norm_backward<T>(x, dy, dx, gamma, mean, rstd, dgamma, dbeta, accumulate, N, F, xs, dys, dxs, as_stream(stream));
}

}   // namespace bb200

using namespace bb200;

extern "C" int bbcu_fp32_LayerNormalization_Forward(const float *x, float *y, const float *gamma, const float *beta, float *mean, float *rstd, float eps,
                                                    int node_size, int frame_size, int x_frame_stride, int y_frame_stride, bbcu_stream_t stream)
{
    return layer_norm_forward_checked<float>(x, y, gamma, beta, mean, rstd, eps, node_size, frame_size, x_frame_stride, y_frame_stride, stream);
}

extern "C" int bbcu_bf16_LayerNormalization_Forward(const bbcu_bf16_t *x, bbcu_bf16_t *y, const float *gamma, const float *beta, float *mean, float *rstd,
                                                    float eps, int node_size, int frame_size, int x_frame_stride, int y_frame_stride,
                                                    bbcu_stream_t stream)
{
    return layer_norm_forward_checked<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16 *>(x), reinterpret_cast<__nv_bfloat16 *>(y), gamma, beta, mean, rstd,
                                                     eps, node_size, frame_size, x_frame_stride, y_frame_stride, stream);
}

extern "C" int bbcu_fp32_LayerNormalization_Backward(const float *x, const float *dy, float *dx, const float *gamma, const float *mean, const float *rstd,
                                                     float *dgamma, float *dbeta, int accumulate, int node_size, int frame_size, int x_frame_stride,
                                                     int dy_frame_stride, int dx_frame_stride, bbcu_stream_t stream)
{
    return layer_norm_backward_checked<float>(x, dy, dx, gamma, mean, rstd, dgamma, dbeta, accumulate, node_size, frame_size, x_frame_stride, dy_frame_stride,
                                              dx_frame_stride, stream);
}

extern "C" int bbcu_bf16_LayerNormalization_Backward(const bbcu_bf16_t *x, const bbcu_bf16_t *dy, bbcu_bf16_t *dx, const float *gamma, const float *mean,
                                                     const float *rstd, float *dgamma, float *dbeta, int accumulate, int node_size, int frame_size,
                                                     int x_frame_stride, int dy_frame_stride, int dx_frame_stride, bbcu_stream_t stream)
{
    return layer_norm_backward_checked<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16 *>(x), reinterpret_cast<const __nv_bfloat16 *>(dy),
                                                      reinterpret_cast<__nv_bfloat16 *>(dx), gamma, mean, rstd, dgamma, dbeta, accumulate, node_size, frame_size,
                                                      x_frame_stride, dy_frame_stride, dx_frame_stride, stream);
}
