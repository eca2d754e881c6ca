// Layer norm over the nodes of a frame, forward and backward, on fp32 and bf16 frame buffers.  (The reference normalises over the frames of a node,
// include/bb/StochasticBatchNormalization.h:521-617; it has no counterpart of this.)
//
//   forward    m = mean_n x,  v = mean_n (x - m)^2,  r = 1 / sqrt(v + eps),  y = (x - m) r gamma_n + beta_n
//   backward   xh = (x - m) r,  c1 = mean_n gamma_n dy,  c2 = mean_n gamma_n dy xh,  dx = r (gamma_n dy - c1 - xh c2),
//              dgamma_n = sum_f dy xh,  dbeta_n = sum_f dy
//
// Statistics and sums are 32 bits throughout; bf16 frames are widened when they are read and rounded once when they are written.
#include "frame_columns.cuh"

namespace bb200 {

constexpr int kMostNodes = 1 << 24;                    // row numbers and their distances stay far from 2^31
constexpr int kNormThreads = 256;                      // of the kernels that stream over chunks of rows

// ---- sums of a chunk of rows: part[chunk][column] = (sum d, sum d^2), d = x minus the column's first value, which takes a large level out.  Eight
// rows are added up in 32 bits and joined with the rest in 64, so that a long column costs no digits either.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kNormThreads)
k_layer_norm_stats(const T *x, double2 *part, int N, int F, long long xs, int chunk_rows, int columns)
{
    grid_dependency();
    constexpr int kLpr = 8, kBatch = 8;
    using Col = Column<T, kLpr>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    __shared__ double2 red[8][kCols];
    const Col c;
    const int f = (int)blockIdx.x * kCols + c.col;
    const int n0 = (int)blockIdx.y * chunk_rows, n1 = min(N, n0 + chunk_rows);
    double s1[kVec] = {}, s2[kVec] = {};
    float level[kVec];
    unpack<T>(load_frames<T, ALIGNED>(x, f, F), level);
    for (int n = n0 + c.row; n < n1; n += c.step * kBatch) {
        uint4 raw[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * c.step;
            if (m < n1) raw[i] = load_frames<T, ALIGNED>(x + (long long)m * xs, f, F);
        }
        float b1[kVec] = {}, b2[kVec] = {};
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (n + i * c.step < n1) {
                float v[kVec];
                unpack<T>(raw[i], v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    const float d = v[j] - level[j];
                    b1[j] += d;
                    b2[j] = fmaf(d, d, b2[j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j) { s1[j] += (double)b1[j]; s2[j] += (double)b2[j]; }
    }
#pragma unroll
    for (int m = kLpr; m < 32; m <<= 1)
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            s1[j] += __shfl_xor_sync(0xffffffffu, s1[j], m);
            s2[j] += __shfl_xor_sync(0xffffffffu, s2[j], m);
        }
    if (c.lane < kLpr) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) red[c.warp][c.col + j] = make_double2(s1[j], s2[j]);
    }
    __syncthreads();
    if (threadIdx.x < kCols) {
        double2 t = red[0][threadIdx.x];
        for (int w = 1; w < c.warps; ++w) { t.x += red[w][threadIdx.x].x; t.y += red[w][threadIdx.x].y; }
        part[(long long)blockIdx.y * columns + (long long)blockIdx.x * kCols + threadIdx.x] = t;
    }
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kNormThreads)
k_layer_norm_apply(const T *x, T *y, const double2 *__restrict__ part, const float *__restrict__ gamma, const float *__restrict__ beta, float *mean_out,
                   float *rstd_out, float eps, int N, int F, long long xs, long long ys, int chunk_rows, int chunks, int columns)
{
    grid_dependency();
    constexpr int kLpr = 8, kBatch = 8;
    using Col = Column<T, kLpr>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    __shared__ float s_mean[kCols], s_rstd[kCols];
    const Col c;
    const int f0 = (int)blockIdx.x * kCols, f = f0 + c.col;
    if (threadIdx.x < kCols) {
        double s1 = 0.0, s2 = 0.0;
        for (int k = 0; k < chunks; ++k) {
            const double2 p = part[(long long)k * columns + f0 + threadIdx.x];
            s1 += p.x;
            s2 += p.y;
        }
        const bool live = f0 + (int)threadIdx.x < F;
        s1 /= (double)N;
        double var = s2 / (double)N - s1 * s1;
        if (var < 0.0) var = 0.0;                                        // (and a NaN stays one)
        const float mean = (float)((live ? (double)to_float(x[f0 + threadIdx.x]) : 0.0) + s1), rstd = 1.0f / sqrtf((float)var + eps);
        s_mean[threadIdx.x] = mean;
        s_rstd[threadIdx.x] = rstd;
        if (blockIdx.y == 0 && live) {
            mean_out[f0 + threadIdx.x] = mean;
            rstd_out[f0 + threadIdx.x] = rstd;
        }
    }
    __syncthreads();
    float mean[kVec], rstd[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) { mean[j] = s_mean[c.col + j]; rstd[j] = s_rstd[c.col + j]; }
    const int n0 = (int)blockIdx.y * chunk_rows, n1 = min(N, n0 + chunk_rows);
    for (int n = n0 + c.row; n < n1; n += c.step * kBatch) {
        uint4 raw[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * c.step;
            if (m < n1) raw[i] = load_frames<T, ALIGNED>(x + (long long)m * xs, f, F);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * c.step;
            if (m < n1) {
                const float g = gamma ? gamma[m] : 1.0f, b = beta ? beta[m] : 0.0f;
                float v[kVec];
                unpack<T>(raw[i], v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) v[j] = fmaf((v[j] - mean[j]) * rstd[j], g, b);
                store_frames<T, ALIGNED>(y + (long long)m * ys, f, F, v);
            }
        }
    }
}

// ---- backward: the two sums over the nodes of a chunk
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kNormThreads)
k_layer_norm_grad_stats(const T *x, const T *dy, const float *__restrict__ gamma, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                        float2 *part, int N, int F, long long xs, long long dys, int chunk_rows, int columns)
{
    grid_dependency();
    constexpr int kLpr = 8, kBatch = 4;
    using Col = Column<T, kLpr>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    __shared__ float red[8 * 2 * kCols];
    const Col c;
    const int f0 = (int)blockIdx.x * kCols, f = f0 + c.col;
    const int n0 = (int)blockIdx.y * chunk_rows, n1 = min(N, n0 + chunk_rows);
    float mean[kVec], rstd[kVec], s[2][kVec] = {};
#pragma unroll
    for (int j = 0; j < kVec; ++j) { mean[j] = f + j < F ? mean_in[f + j] : 0.0f; rstd[j] = f + j < F ? rstd_in[f + j] : 0.0f; }
    for (int n = n0 + c.row; n < n1; n += c.step * kBatch) {
        uint4 xr[kBatch], gr[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * c.step;
            xr[i] = m < n1 ? load_frames<T, ALIGNED>(x + (long long)m * xs, f, F) : make_uint4(0, 0, 0, 0);
            gr[i] = m < n1 ? load_frames<T, ALIGNED>(dy + (long long)m * dys, f, F) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * c.step;
            if (m < n1) {
                const float gm = gamma ? gamma[m] : 1.0f;
                float xv[kVec], gv[kVec];
                unpack<T>(xr[i], xv);
                unpack<T>(gr[i], gv);
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    const float g = gm * gv[j], xh = (xv[j] - mean[j]) * rstd[j];
                    s[0][j] += g;
                    s[1][j] = fmaf(g, xh, s[1][j]);
                }
            }
        }
    }
    join_columns<ColumnSum, 2, T, kLpr>(s, c, red, nullptr, 1);
    if (c.warp == 0 && c.lane < kLpr) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) part[(long long)blockIdx.y * columns + f + j] = make_float2(s[0][j], s[1][j]);
    }
}

// dx of R rows a thread over every gridDim.x-th column tile, with the sums over those frames kept in registers on the way:
// grad_part[blockIdx.x][node] = (sum dy xh, sum dy)
template <typename T, int R, bool ALIGNED>
__global__ void __launch_bounds__(kNormThreads)
k_layer_norm_grad_apply(const T *x, const T *dy, T *dx, const float2 *__restrict__ part, const float *__restrict__ gamma, const float *__restrict__ mean_in,
                        const float *__restrict__ rstd_in, float2 *grad_part, int N, int F, long long xs, long long dys, long long dxs, int chunks,
                        int columns)
{
    grid_dependency();
    constexpr int kLpr = 8;
    using Col = Column<T, kLpr>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    __shared__ float s_c[2][kCols];
    const Col c;
    const long long first = (long long)blockIdx.y * c.step * R + c.row;
    const float inv = 1.0f / (float)N;
    float gm[R], ag[R], ab[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const long long n = first + i * c.step;
        gm[i] = n < N ? (gamma ? gamma[n] : 1.0f) : 0.0f;
        ag[i] = ab[i] = 0.0f;
    }
    for (int tile = blockIdx.x; tile < columns / kCols; tile += gridDim.x) {
        const int f0 = tile * kCols, f = f0 + c.col;
        uint4 xr[R], gr[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const long long n = first + i * c.step;
            xr[i] = n < N ? load_frames<T, ALIGNED>(x + n * xs, f, F) : make_uint4(0, 0, 0, 0);
            gr[i] = n < N ? load_frames<T, ALIGNED>(dy + n * dys, f, F) : make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
        if (threadIdx.x < kCols) {
            float a = 0.0f, b = 0.0f;
            for (int k = 0; k < chunks; ++k) {
                const float2 p = part[(long long)k * columns + f0 + threadIdx.x];
                a += p.x;
                b += p.y;
            }
            s_c[0][threadIdx.x] = a * inv;
            s_c[1][threadIdx.x] = b * inv;
        }
        __syncthreads();
        float mean[kVec], rstd[kVec];
#pragma unroll
        for (int j = 0; j < kVec; ++j) { mean[j] = f + j < F ? mean_in[f + j] : 0.0f; rstd[j] = f + j < F ? rstd_in[f + j] : 0.0f; }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const long long n = first + i * c.step;
            float xv[kVec], gv[kVec];
            unpack<T>(xr[i], xv);
            unpack<T>(gr[i], gv);
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const bool live = f + j < F;
                const float g = live ? gv[j] : 0.0f, xh = live ? (xv[j] - mean[j]) * rstd[j] : 0.0f;
                ag[i] = fmaf(g, xh, ag[i]);
                ab[i] += g;
                gv[j] = rstd[j] * (gm[i] * g - s_c[0][c.col + j] - xh * s_c[1][c.col + j]);
            }
            if (n < N) store_frames<T, ALIGNED>(dx + n * dxs, f, F, gv);
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const long long n = first + i * c.step;
#pragma unroll
        for (int m = 1; m < kLpr; m <<= 1) {
            ag[i] += __shfl_xor_sync(0xffffffffu, ag[i], m);
            ab[i] += __shfl_xor_sync(0xffffffffu, ab[i], m);
        }
        if (c.lane % kLpr == 0 && n < N) grad_part[(long long)blockIdx.x * N + n] = make_float2(ag[i], ab[i]);
    }
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

// rows of a chunk so that about four CTAs an SM are there, a multiple of 64
static int chunk_of(int N, long long tiles)
{
    const long long want = 4LL * device_info().sm_count;
    long long chunks = (want + tiles - 1) / tiles;
    long long rows = ((N + chunks - 1) / chunks + 63) / 64 * 64;
    if (rows < 64) rows = 64;
    while ((N + rows - 1) / rows > 65535) rows *= 2;
    return (int)rows;
}

template <typename T>
static int layer_norm_forward(const T *x, T *y, const float *gamma, const float *beta, float *mean, float *rstd, float eps, int N, int F, long long xs,
                              long long ys, cudaStream_t st)
{
    const bool aligned = frames_aligned<T>(x, xs) && frames_aligned<T>(y, ys);
    constexpr int kCols = Column<T, 8>::kCols;
    const long long tiles = ((long long)F + kCols - 1) / kCols;
    BB200_REQUIRE(tiles * kCols < (1LL << 31), BBCU_ERR_TOO_LARGE);
    const int columns = (int)(tiles * kCols), rows = chunk_of(N, tiles), chunks = (N + rows - 1) / rows;
    double2 *part = static_cast<double2 *>(stream_scratch(st, (size_t)chunks * columns * sizeof(double2), kFrameOpSlot));
    BB200_REQUIRE(part != nullptr, BBCU_ERR_NO_MEMORY);
    const dim3 grid((unsigned)tiles, (unsigned)chunks);
    launch(aligned ? k_layer_norm_stats<T, true> : k_layer_norm_stats<T, false>, grid, kNormThreads, 0, st, x, part, N, F, xs, rows, columns);
    BB200_CUDA(cudaPeekAtLastError());
    launch(aligned ? k_layer_norm_apply<T, true> : k_layer_norm_apply<T, false>, grid, kNormThreads, 0, st, x, y, part, gamma, beta, mean, rstd, eps, N, F,
           xs, ys, rows, chunks, columns);
    return launch_status();
}

template <typename T>
static int layer_norm_backward(const T *x, const T *dy, T *dx, const float *gamma, const float *mean, const float *rstd, float *dgamma, float *dbeta,
                               int accumulate, int N, int F, long long xs, long long dys, long long dxs, cudaStream_t st)
{
    const bool aligned = frames_aligned<T>(x, xs) && frames_aligned<T>(dy, dys) && frames_aligned<T>(dx, dxs);
    constexpr int kCols = Column<T, 8>::kCols, kRows = 4, kPerCta = kNormThreads / 32 * 4 * kRows;
    const long long tiles = ((long long)F + kCols - 1) / kCols;
    BB200_REQUIRE(tiles * kCols < (1LL << 31), BBCU_ERR_TOO_LARGE);
    const int columns = (int)(tiles * kCols), rows = chunk_of(N, tiles), chunks = (N + rows - 1) / rows;
    const int row_ctas = (N + kPerCta - 1) / kPerCta;
    BB200_REQUIRE(row_ctas <= 65535, BBCU_ERR_TOO_LARGE);
    long long sweeps = (4LL * device_info().sm_count + row_ctas - 1) / row_ctas;
    if (sweeps > tiles) sweeps = tiles;
    const size_t part_bytes = (size_t)chunks * columns * sizeof(float2);
    char *scratch = static_cast<char *>(stream_scratch(st, part_bytes + (size_t)sweeps * N * sizeof(float2), kFrameOpSlot));
    BB200_REQUIRE(scratch != nullptr, BBCU_ERR_NO_MEMORY);
    float2 *part = reinterpret_cast<float2 *>(scratch), *grad_part = reinterpret_cast<float2 *>(scratch + part_bytes);
    launch(aligned ? k_layer_norm_grad_stats<T, true> : k_layer_norm_grad_stats<T, false>, dim3((unsigned)tiles, (unsigned)chunks), kNormThreads, 0, st, x, dy,
           gamma, mean, rstd, part, N, F, xs, dys, rows, columns);
    BB200_CUDA(cudaPeekAtLastError());
    launch(aligned ? k_layer_norm_grad_apply<T, kRows, true> : k_layer_norm_grad_apply<T, kRows, false>, dim3((unsigned)sweeps, (unsigned)row_ctas), kNormThreads,
           0, st, x, dy, dx, part, gamma, mean, rstd, grad_part, N, F, xs, dys, dxs, chunks, columns);
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

bool allow_cluster_16_once(const void *kernel)
{
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
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
