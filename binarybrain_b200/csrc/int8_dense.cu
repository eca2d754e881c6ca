// Dense layer in 8-bit integers with a scale per frame and per output node, and the quantisers that make its operands.  (The reference's dense layers
// are fp32 through cuBLAS, include/bb/DenseAffine.h, and DepthwiseDenseAffineQuantize.h; it has no integer product.)
//
//   quantiser   per frame f of a frame buffer x[node][frame]: s = max_n |x| / 127,  q = rint(x / s) in [-127, 127], both in 32 bits, ties to even;
//               a frame of zeros has s = 0, one with a NaN or an infinity s = NaN, both q = 0.  The frames become rows, q[frame][node], 16-byte
//               pieces along the nodes, which is how the product reads both of its operands.  The channel form does the same to the rows of W[out][in].
//   product     y[o][f] = s_w[o] s_x[f] sum_k Wq[o][k] q[f][k] + bias[o],  the sum exact in 32-bit integers (at most 131071 inputs), y fp32 or bf16
#include "frame_columns.cuh"

namespace bb200 {

constexpr int kQuantThreads = 256, kQuantRows = 128;      // rows of x that a CTA turns over at a time
constexpr int kMostInputs = 131071;                       // times 128 x 128 is below 2^31

__device__ __forceinline__ float quant_scale(uint32_t abs_bits)
{
    return abs_bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __fdiv_rn(__uint_as_float(abs_bits), 127.0f);
}

__device__ __forceinline__ int quantize(float x, float scale)
{
    if (!(scale > 0.0f)) return 0;                        // zeros, or not finite
    return max(-127, min(127, __float2int_rn(__fdiv_rn(x, scale))));
}

// part[chunk][column] = bits of the largest |x| (as integers they order like the numbers, with infinities and NaN on top)
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kQuantThreads)
k_quantize_max(const T *x, uint32_t *part, int N, int F, long long xs, int chunk_rows, int columns)
{
    grid_dependency();
    constexpr int kLpr = 8, kBatch = 8;
    using Col = Column<T, kLpr>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    __shared__ uint32_t s[8][kCols];
    const Col c;
    const int f = (int)blockIdx.x * kCols + c.col;
    const int n0 = (int)blockIdx.y * chunk_rows, n1 = min(N, n0 + chunk_rows);
    uint32_t top[kVec] = {};
    for (int n = n0 + c.row; n < n1; n += c.step * kBatch) {
        uint4 raw[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * c.step;
            raw[i] = m < n1 ? load_frames<T, ALIGNED>(x + (long long)m * xs, f, F) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            float v[kVec];
            unpack<T>(raw[i], v);
#pragma unroll
            for (int j = 0; j < kVec; ++j) top[j] = max(top[j], __float_as_uint(fabsf(v[j])));
        }
    }
#pragma unroll
    for (int m = kLpr; m < 32; m <<= 1)
#pragma unroll
        for (int j = 0; j < kVec; ++j) top[j] = max(top[j], __shfl_xor_sync(0xffffffffu, top[j], m));
    if (c.lane < kLpr) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) s[c.warp][c.col + j] = top[j];
    }
    __syncthreads();
    if (threadIdx.x < kCols) {
        uint32_t t = 0;
        for (int w = 0; w < c.warps; ++w) t = max(t, s[w][threadIdx.x]);
        part[(long long)blockIdx.y * columns + (long long)blockIdx.x * kCols + threadIdx.x] = t;
    }
}

// 128 rows of x at a time: a thread reads four neighbouring rows of its columns, so that its four values of a frame are a word of q; the words cross
// through shared memory and leave as 16 bytes of a frame's row.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kQuantThreads)
k_quantize_apply(const T *x, int8_t *q, const uint32_t *__restrict__ part, float *scale_out, int N, int F, long long xs, long long qs, int chunk_rows,
                 int chunks, int columns)
{
    grid_dependency();
    constexpr int kLpr = 8;
    using Col = Column<T, kLpr>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols, kWords = kQuantRows / 4;
    __shared__ float s_scale[kCols];
    __shared__ __align__(16) uint32_t tile[kCols][kWords + 4];
    const Col c;
    const int f0 = (int)blockIdx.x * kCols, f = f0 + c.col;
    if (threadIdx.x < kCols) {
        uint32_t t = 0;
        for (int k = 0; k < chunks; ++k) t = max(t, part[(long long)k * columns + f0 + threadIdx.x]);
        const float s = quant_scale(t);
        s_scale[threadIdx.x] = s;
        if (blockIdx.y == 0 && f0 + (int)threadIdx.x < F) scale_out[f0 + threadIdx.x] = s;
    }
    __syncthreads();
    float scale[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) scale[j] = s_scale[c.col + j];
    const int n0 = (int)blockIdx.y * chunk_rows, n1 = min(N, n0 + chunk_rows);
    for (int base = n0; base < n1; base += kQuantRows) {
        uint32_t word[kVec] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = base + 4 * c.row + i;
            float v[kVec];
            unpack<T>(n < n1 ? load_frames<T, ALIGNED>(x + (long long)n * xs, f, F) : make_uint4(0, 0, 0, 0), v);
#pragma unroll
            for (int j = 0; j < kVec; ++j) word[j] |= (uint32_t)(quantize(v[j], scale[j]) & 0xff) << (8 * i);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kVec; ++j) tile[c.col + j][c.row] = word[j];
        __syncthreads();
        for (int e = threadIdx.x; e < kCols * (kQuantRows / 16); e += kQuantThreads) {
            const int col = e / (kQuantRows / 16), piece = e % (kQuantRows / 16), n = base + 16 * piece;
            if (f0 + col < F && n < n1) *reinterpret_cast<uint4 *>(q + (long long)(f0 + col) * qs + n) = *reinterpret_cast<const uint4 *>(&tile[col][4 * piece]);
        }
    }
}

// a row of W a CTA
__global__ void __launch_bounds__(256)
k_quantize_channels(const float *__restrict__ W, int8_t *q, float *scale_out, int N, long long ws, long long qs)
{
    grid_dependency();
    __shared__ uint32_t red[8];
    const float *row = W + (long long)blockIdx.x * ws;
    uint32_t top = 0;
    for (int n = threadIdx.x; n < N; n += 256) top = max(top, __float_as_uint(fabsf(row[n])));
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int w = 0; w < 8; ++w) top = max(top, red[w]);
    const float scale = quant_scale(top);
    if (threadIdx.x == 0) scale_out[blockIdx.x] = scale;
    const int padded = (N + 15) / 16 * 16;
    for (int n = threadIdx.x; n < padded; n += 256) q[(long long)blockIdx.x * qs + n] = n < N ? (int8_t)quantize(row[n], scale) : (int8_t)0;
}

// The 16 bytes at k of a frame's row, with what lies beyond the inputs cleared: the padding of W may then hold anything.
__device__ __forceinline__ int4 load_q(const int8_t *row, int k, int K)
{
    int4 v = *reinterpret_cast<const int4 *>(row + k);
    if (k + 16 > K) {
        int *w = reinterpret_cast<int *>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int left = K - k - 4 * i;
            w[i] = left >= 4 ? w[i] : left <= 0 ? 0 : (int)((uint32_t)w[i] & ((1u << (8 * left)) - 1u));
        }
    }
    return v;
}

// NF frames and ROWS output nodes a warp, 512 bytes of every row a step
template <typename T, int NF, int ROWS>
__global__ void __launch_bounds__(256)
k_int8_dense_rows(const int8_t *__restrict__ q, const float *__restrict__ q_scale, const int8_t *__restrict__ W, const float *__restrict__ w_scale,
                  const float *__restrict__ bias, T *y, int K, int O, int F, long long qs, long long ws, long long ys)
{
    grid_dependency();
    const int lane = threadIdx.x & 31;
    const int o0 = ((int)blockIdx.x * 8 + (int)(threadIdx.x >> 5)) * ROWS;
    const int f0 = (int)blockIdx.y * NF;
    if (o0 >= O) return;
    int acc[ROWS][NF] = {};
    for (int k = lane * 16; k < K; k += 512) {
        int4 w[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) w[r] = *reinterpret_cast<const int4 *>(W + (long long)min(o0 + r, O - 1) * ws + k);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int4 v = load_q(q + (long long)min(f0 + f, F - 1) * qs, k, K);
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                acc[r][f] = __dp4a(w[r].w, v.w, __dp4a(w[r].z, v.z, __dp4a(w[r].y, v.y, __dp4a(w[r].x, v.x, acc[r][f]))));
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int s = __reduce_add_sync(0xffffffffu, acc[r][f]);
            if (lane == (r * NF + f) % 32 && o0 + r < O && f0 + f < F)
                y[(long long)(o0 + r) * ys + f0 + f] = from_float<T>(fmaf((float)s, w_scale[o0 + r] * q_scale[f0 + f], bias ? bias[o0 + r] : 0.0f));
        }
}

template <typename T>
static int quantize_frames(const T *x, int8_t *q, float *scale, int N, int F, int xs, int qs, bbcu_stream_t stream)
{
    BB200_REQUIRE(N > 0 && F >= 0, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(N <= (1 << 24), BBCU_ERR_TOO_LARGE);
    BB200_REQUIRE(xs >= F && qs >= (N + 15) / 16 * 16 && qs % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0, BBCU_ERR_BAD_STRIDE);
    if (F == 0) return BBCU_OK;
    BB200_REQUIRE_PTR(x); BB200_REQUIRE_PTR(q); BB200_REQUIRE_PTR(scale);
    cudaStream_t st = as_stream(stream);
    const bool aligned = frames_aligned<T>(x, xs);
    constexpr int kCols = Column<T, 8>::kCols;
    const long long tiles = ((long long)F + kCols - 1) / kCols;
    BB200_REQUIRE(tiles * kCols < (1LL << 31), BBCU_ERR_TOO_LARGE);
    const long long want = 4LL * device_info().sm_count, per = (want + tiles - 1) / tiles;
    int rows = (int)(((N + per - 1) / per + kQuantRows - 1) / kQuantRows * kQuantRows);
    while ((N + rows - 1) / rows > 65535) rows *= 2;
    const int columns = (int)(tiles * kCols), chunks = (N + rows - 1) / rows;
    uint32_t *part = static_cast<uint32_t *>(stream_scratch(st, (size_t)chunks * columns * sizeof(uint32_t), kFrameOpSlot));
    BB200_REQUIRE(part != nullptr, BBCU_ERR_NO_MEMORY);
    const dim3 grid((unsigned)tiles, (unsigned)chunks);
    launch(aligned ? k_quantize_max<T, true> : k_quantize_max<T, false>, grid, kQuantThreads, 0, st, x, part, N, F, xs, rows, columns);
    BB200_CUDA(cudaPeekAtLastError());
    launch(aligned ? k_quantize_apply<T, true> : k_quantize_apply<T, false>, grid, kQuantThreads, 0, st, x, q, part, scale, N, F, xs, qs, rows, chunks, columns);
    return launch_status();
}

template <typename T>
static int int8_dense(const int8_t *q, const float *q_scale, const int8_t *W, const float *w_scale, const float *bias, T *y, int K, int O, int F, int qs,
                      int ws, int ys, bbcu_stream_t stream)
{
    BB200_REQUIRE(K > 0 && O >= 0 && F >= 0, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(K <= kMostInputs, BBCU_ERR_TOO_LARGE);
    const int least = (K + 15) / 16 * 16;
    BB200_REQUIRE(qs >= least && ws >= least && qs % 16 == 0 && ws % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(W) % 16 == 0 && ys >= F, BBCU_ERR_BAD_STRIDE);
    if (F == 0 || O == 0) return BBCU_OK;
    BB200_REQUIRE_PTR(q); BB200_REQUIRE_PTR(q_scale); BB200_REQUIRE_PTR(W); BB200_REQUIRE_PTR(w_scale); BB200_REQUIRE_PTR(y);
    constexpr int kFrames = 8, kRows = 4;
    const long long frame_ctas = ((long long)F + kFrames - 1) / kFrames, row_ctas = ((long long)O + 8 * kRows - 1) / (8 * kRows);
    BB200_REQUIRE(frame_ctas <= 65535, BBCU_ERR_TOO_LARGE);
    launch(k_int8_dense_rows<T, kFrames, kRows>, dim3((unsigned)row_ctas, (unsigned)frame_ctas), 256, 0, as_stream(stream), q, q_scale, W, w_scale, bias, y, K, O, F,
           qs, ws, ys);
    return launch_status();
}

}   // namespace bb200

using namespace bb200;

extern "C" int bbcu_fp32_QuantizeInt8_Frames(const float *x, signed char *q, float *scale, int node_size, int frame_size, int x_frame_stride,
                                             int q_node_stride, bbcu_stream_t stream)
{
    return quantize_frames<float>(x, q, scale, node_size, frame_size, x_frame_stride, q_node_stride, stream);
}

extern "C" int bbcu_bf16_QuantizeInt8_Frames(const bbcu_bf16_t *x, signed char *q, float *scale, int node_size, int frame_size, int x_frame_stride,
                                             int q_node_stride, bbcu_stream_t stream)
{
    return quantize_frames<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16 *>(x), q, scale, node_size, frame_size, x_frame_stride, q_node_stride, stream);
}

extern "C" int bbcu_fp32_QuantizeInt8_Channels(const float *W, signed char *q, float *scale, int input_node_size, int output_node_size, int w_node_stride,
                                               int q_node_stride, bbcu_stream_t stream)
{
    BB200_REQUIRE(input_node_size > 0 && output_node_size >= 0, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(input_node_size <= (1 << 24), BBCU_ERR_TOO_LARGE);
    BB200_REQUIRE(w_node_stride >= input_node_size && q_node_stride >= (input_node_size + 15) / 16 * 16, BBCU_ERR_BAD_STRIDE);
    if (output_node_size == 0) return BBCU_OK;
    BB200_REQUIRE_PTR(W); BB200_REQUIRE_PTR(q); BB200_REQUIRE_PTR(scale);
    launch(k_quantize_channels, (unsigned)output_node_size, 256, 0, as_stream(stream), W, q, scale, input_node_size, w_node_stride, q_node_stride);
    return launch_status();
}

extern "C" int bbcu_int8_fp32_DenseAffine_Forward(const signed char *q, const float *q_scale, const signed char *W, const float *w_scale, const float *bias,
                                                  float *y, int input_node_size, int output_node_size, int frame_size, int q_node_stride,
                                                  int w_node_stride, int y_frame_stride, bbcu_stream_t stream)
{
    return int8_dense<float>(q, q_scale, W, w_scale, bias, y, input_node_size, output_node_size, frame_size, q_node_stride, w_node_stride, y_frame_stride, stream);
}

extern "C" int bbcu_int8_bf16_DenseAffine_Forward(const signed char *q, const float *q_scale, const signed char *W, const float *w_scale, const float *bias,
                                                  bbcu_bf16_t *y, int input_node_size, int output_node_size, int frame_size, int q_node_stride,
                                                  int w_node_stride, int y_frame_stride, bbcu_stream_t stream)
{
    return int8_dense<__nv_bfloat16>(q, q_scale, W, w_scale, bias, reinterpret_cast<__nv_bfloat16 *>(y), input_node_size, output_node_size, frame_size,
                                     q_node_stride, w_node_stride, y_frame_stride, stream);
}
