// Root-mean-square norm over the nodes of a frame with the residual's addition, forward (fp32, bf16, or 8-bit rows with a scale, as the int8 product reads
// them) and backward, on fp32 and bf16 frame buffers.  (The reference normalises over the frames of a node, include/bb/StochasticBatchNormalization.h:521-617;
// it has no counterpart of this.)
//
//   forward    s = x + r, kept in the frames' type (without a residual: s = x),  rstd = 1 / sqrt(mean_n s^2 + eps),  y = (s rstd) gamma_n
//   8 bits     t = s gamma_n,  u = max_n |t| / 127,  q = rint(t / u),  scale = u rstd: q does not depend on rstd, and so not on the order of its sum
//   backward   xh = s rstd,  c = mean_n gamma_n dy xh,  ds = rstd (gamma_n dy - xh c) + dr,  dgamma_n = sum_f dy xh
//
// Sums are 32 bits; bf16 frames are widened when they are read and rounded once when they are written.  What is normalised is the sum as it is kept, so that
// the backward pass, which is given that, sees the numbers that the statistics are of.
//
// Memory bounds it (16 bytes a value of fp32 forward with a residual, 16 backward).  A frame is needed whole before its first output: a cluster of CTAs has
// the columns of 32 to 128 bytes of a row and goes over the rows twice.  Up to kHeldRows rows a thread stay in registers in between; the others are read
// again, out of L2, which holds them since they were written, or read, some microseconds before.
#include <algorithm>

#include "frame_columns.cuh"
#include "quantize.cuh"

namespace bb200 {

constexpr int kMostRmsNodes = 1 << 20;
constexpr int kHeldRows = 8;

template <typename T> struct RmsForward {
    const T *x, *r;
    T *s, *y;
    int8_t *q;
    const float *gamma;
    float *rstd, *scale, eps;
    int N, F, rounds;                                    // rounds of rows of a cluster
    long long xs, rs, ss, ys, qs;
    int *fault;
};

// a vector of s = x + r as it is kept
template <typename T> __device__ __forceinline__ uint4 add_frames(const uint4 &x, const uint4 &r)
{
    float a[kFramesPerVec<T>], b[kFramesPerVec<T>];
    unpack<T>(x, a);
    unpack<T>(r, b);
#pragma unroll
    for (int j = 0; j < kFramesPerVec<T>; ++j) a[j] += b[j];
    return pack<T>(a);
}

// A thread takes kRows neighbouring rows a round (8 bits: four, which are a word of q), the rounds of a cluster's CTAs in turn.
template <typename T, int LPR, bool ALIGNED, bool INT8, bool HELD>
__global__ void __launch_bounds__(kColumnThreads, 4)
k_rms_forward(const RmsForward<T> a)
{
    grid_dependency();
    using Col = Column<T, LPR>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols, kRows = 4, kQ = INT8 ? 2 : 1, kRounds = HELD ? kHeldRows / kRows : 1, kWords = kColumnThreads / LPR;
    extern __shared__ __align__(16) uint8_t parts[];
    __shared__ Exchange<kQ, kCols> sums[2];
    __shared__ __align__(16) uint32_t tile[INT8 ? kCols : 1][INT8 ? kWords : 4];
    __shared__ int gave_up;
    const Col c;
    Cluster cl(&gave_up);
    const int f0 = (int)(blockIdx.x / cl.size) * kCols, f = f0 + c.col, round_rows = c.step * kRows;
    const T *const in = a.r ? a.s : a.x;                                   // what a second reading finds
    const long long in_stride = a.r ? a.ss : a.xs;
    uint4 held[kRounds][kRows];
    float v[kQ][kVec] = {};
    for (int round = 0; round < a.rounds; ++round) {
        const int n = (round * (int)cl.size + (int)cl.rank) * round_rows + c.row * kRows;
        uint4 raw[kRows], more[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) raw[i] = n + i < a.N ? load_frames<T, ALIGNED>(a.x + (long long)(n + i) * a.xs, f, a.F) : make_uint4(0, 0, 0, 0);
        if (a.r) {
#pragma unroll
            for (int i = 0; i < kRows; ++i) more[i] = n + i < a.N ? load_frames<T, ALIGNED>(a.r + (long long)(n + i) * a.rs, f, a.F) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                raw[i] = add_frames<T>(raw[i], more[i]);
                float w[kVec];
                unpack<T>(raw[i], w);
                if (n + i < a.N) store_frames<T, ALIGNED>(a.s + (long long)(n + i) * a.ss, f, a.F, w);
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            float w[kVec];
            unpack<T>(raw[i], w);
            const float g = INT8 && a.gamma && n + i < a.N ? a.gamma[n + i] : 1.0f;
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                v[0][j] = fmaf(w[j], w[j], v[0][j]);
                if constexpr (INT8) v[1][j] = __uint_as_float(max(__float_as_uint(v[1][j]), __float_as_uint(fabsf(w[j] * g))));
            }
            if constexpr (HELD) {
#pragma unroll
                for (int k = 0; k < kRounds; ++k)
                    if (k == round) held[k][i] = raw[i];
            }
        }
    }
    cl.meet(sums, parts);
#pragma unroll
    for (int m = LPR; m < 32; m <<= 1)
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            v[0][j] += __shfl_xor_sync(0xffffffffu, v[0][j], m);
            if constexpr (INT8) v[1][j] = __uint_as_float(max(__float_as_uint(v[1][j]), __float_as_uint(__shfl_xor_sync(0xffffffffu, v[1][j], m))));
        }
    struct BitsMax { __device__ static float join(float p, float q) { return __uint_as_float(max(__float_as_uint(p), __float_as_uint(q))); } };
    const float inv = 1.0f / (float)a.N;
    Exchange<kQ, kCols> &e = sums[0];
    exchange_columns<kQ, T, LPR>(v, c, e, cl, 0,
        [&](const float *from, int distance, int count) { return from - &e.red[0][0] < kCols ? join_parts<ColumnSum>(from, distance, count) : join_parts<BitsMax>(from, distance, count); },
        [&](const float *from, int distance, int count) { return from - &e.part[0][0] < kCols ? join_parts<ColumnSum>(from, distance, count) : join_parts<BitsMax>(from, distance, count); },
        [&](int q, float t) { return q == 0 ? 1.0f / sqrtf(fmaf(t, inv, a.eps)) : quant_scale(__float_as_uint(t)); });
    if (cl.rank == 0 && threadIdx.x < kCols && f0 + (int)threadIdx.x < a.F) {
        if constexpr (INT8) a.scale[f0 + threadIdx.x] = e.out[threadIdx.x] * e.out[kCols + threadIdx.x];
        if (a.rstd) a.rstd[f0 + threadIdx.x] = e.out[threadIdx.x];
    }
    for (int round = 0; round < a.rounds; ++round) {
        const int first = (round * (int)cl.size + (int)cl.rank) * round_rows, n = first + c.row * kRows;
        uint4 raw[kRows];
        if constexpr (HELD) {
#pragma unroll
            for (int k = 0; k < kRounds; ++k)
                if (k == round) {
#pragma unroll
                    for (int i = 0; i < kRows; ++i) raw[i] = held[k][i];
                }
        } else {
#pragma unroll
            for (int i = 0; i < kRows; ++i) raw[i] = n + i < a.N ? load_frames<T, ALIGNED>(in + (long long)(n + i) * in_stride, f, a.F) : make_uint4(0, 0, 0, 0);
        }
        float w[kRows][kVec];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            unpack<T>(raw[i], w[i]);
            const float g = a.gamma && n + i < a.N ? a.gamma[n + i] : 1.0f;
#pragma unroll
            for (int j = 0; j < kVec; ++j) w[i][j] = INT8 ? w[i][j] * g : (w[i][j] * v[0][j]) * g;
            if constexpr (!INT8) {
                if (n + i < a.N) store_frames<T, ALIGNED>(a.y + (long long)(n + i) * a.ys, f, a.F, w[i]);
            }
        }
        if constexpr (INT8) {
            // the words cross shared memory, in 16-byte pieces whose order differs from column to column so that no banks collide, and leave as lines of the frames' rows
            if (round > 0) __syncthreads();
#pragma unroll
            for (int j = 0; j < kVec; ++j)
                tile[c.col + j][(c.row / 4 ^ c.lane % LPR) * 4 + c.row % 4] = Quantizer(v[kQ - 1][j])(w[0][j], w[1][j], w[2][j], w[3][j]);
            __syncthreads();
            const int pieces = c.step / 4;
            for (int e = threadIdx.x; e < kCols * pieces; e += blockDim.x) {
                const int col = e / pieces, piece = e % pieces, m = first + 16 * piece;
                if (f0 + col < a.F && m < a.N)
                    *reinterpret_cast<uint4 *>(a.q + (long long)(f0 + col) * a.qs + m) = *reinterpret_cast<const uint4 *>(&tile[col][(piece ^ col / kVec) * 4]);
            }
        }
    }
    cl.leave(a.fault);
}

template <typename T> struct RmsBackward {
    const T *s, *dy, *dr;
    T *ds;
    const float *gamma, *rstd;
    float *gamma_part;                                   // [tile][node]
    int N, F, rounds;
    long long ss, dys, drs, dss;
    int *fault;
};

template <typename T, int LPR, bool ALIGNED, bool HELD>
__global__ void __launch_bounds__(kColumnThreads, 3)
k_rms_backward(const RmsBackward<T> a)
{
    grid_dependency();
    using Col = Column<T, LPR>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols, kRows = 4;
    extern __shared__ __align__(16) uint8_t parts[];
    __shared__ Exchange<1, kCols> sums[2];
    __shared__ int gave_up;
    const Col c;
    Cluster cl(&gave_up);
    const int tile = (int)(blockIdx.x / cl.size), f0 = tile * kCols, f = f0 + c.col, round_rows = c.step * kRows;
    float rstd[kVec], v[1][kVec] = {};
    load_columns(a.rstd, f, a.F, rstd);
    uint4 s_raw[kRows], g_raw[kRows];
    auto load = [&](int n) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            s_raw[i] = n + i < a.N ? load_frames<T, ALIGNED>(a.s + (long long)(n + i) * a.ss, f, a.F) : make_uint4(0, 0, 0, 0);
            g_raw[i] = n + i < a.N ? load_frames<T, ALIGNED>(a.dy + (long long)(n + i) * a.dys, f, a.F) : make_uint4(0, 0, 0, 0);
        }
    };
    for (int round = 0; round < a.rounds; ++round) {
        const int n = (round * (int)cl.size + (int)cl.rank) * round_rows + c.row * kRows;
        load(n);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const float g = a.gamma && n + i < a.N ? a.gamma[n + i] : 1.0f;
            float s[kVec], d[kVec];
            unpack<T>(s_raw[i], s);
            unpack<T>(g_raw[i], d);
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[0][j] = fmaf(g * d[j], s[j] * rstd[j], v[0][j]);
        }
    }
    cl.meet(sums, parts);
    const float inv = 1.0f / (float)a.N;
    join_columns<ColumnSum, 1, T, LPR>(v, c, sums[0], cl, 0, [&](int, float t) { return t * inv; });
    for (int round = 0; round < a.rounds; ++round) {
        const int n = (round * (int)cl.size + (int)cl.rank) * round_rows + c.row * kRows;
        uint4 r_raw[kRows];
        if (a.dr) {
#pragma unroll
            for (int i = 0; i < kRows; ++i) r_raw[i] = n + i < a.N ? load_frames<T, ALIGNED>(a.dr + (long long)(n + i) * a.drs, f, a.F) : make_uint4(0, 0, 0, 0);
        }
        if constexpr (!HELD) load(n);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const float g = a.gamma && n + i < a.N ? a.gamma[n + i] : 1.0f;
            float s[kVec], d[kVec], along = 0.0f;
            unpack<T>(s_raw[i], s);
            unpack<T>(g_raw[i], d);
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const float xh = s[j] * rstd[j];
                if (f + j < a.F) along = fmaf(d[j], xh, along);            // what lies beyond the frames may be anything
                d[j] = rstd[j] * fmaf(-xh, v[0][j], g * d[j]);
            }
            if (a.dr) {
                float r[kVec];
                unpack<T>(r_raw[i], r);
#pragma unroll
                for (int j = 0; j < kVec; ++j) d[j] += r[j];
            }
            if (n + i < a.N) store_frames<T, ALIGNED>(a.ds + (long long)(n + i) * a.dss, f, a.F, d);
#pragma unroll
            for (int m = 1; m < LPR; m <<= 1) along += __shfl_xor_sync(0xffffffffu, along, m);
            if (a.gamma_part && c.lane % LPR == 0 && n + i < a.N) a.gamma_part[(long long)tile * a.N + n + i] = along;
        }
    }
    cl.leave(a.fault);
}

// dgamma = or += the sums of the parts, 8 parts side by side and in a fixed order
__global__ void __launch_bounds__(256)
k_rms_gamma(const float *__restrict__ part, float *dgamma, int N, int parts, int accumulate)
{
    grid_dependency();
    __shared__ float s[8][32];
    const int n = (int)blockIdx.x * 32 + (threadIdx.x & 31);
    float t = 0.0f;
    if (n < N)
        for (int k = threadIdx.x >> 5; k < parts; k += 8) t += part[(long long)k * N + n];
    s[threadIdx.x >> 5][threadIdx.x & 31] = t;
    __syncthreads();
    if (threadIdx.x < 32 && n < N) {
        for (int k = 1; k < 8; ++k) t += s[k][threadIdx.x];
        dgamma[n] = accumulate ? dgamma[n] + t : t;
    }
}

__global__ void __launch_bounds__(256) k_rms_no_frames(float *dgamma, int N)
{
    grid_dependency();
    const int n = (int)blockIdx.x * 256 + threadIdx.x;
    if (n < N) dgamma[n] = 0.0f;
}

// Lanes along a row (8, or 2 where frames are few), CTAs of a cluster, and rounds of four rows a thread.
struct RmsPlan { int lanes, cluster, rounds; unsigned ctas; };
template <typename T> static RmsPlan plan_rms(int N, int F)
{
    const long long sms = device_info().sm_count;
    auto tiles = [&](int lanes) { return ((long long)F + lanes * kFramesPerVec<T> - 1) / (lanes * kFramesPerVec<T>); };
    const int lanes = tiles(8) * 8 < sms ? 2 : 8, round_rows = kColumnThreads / lanes * 4;
    int cl = 1;
    while (cl < 8 && (tiles(lanes) * cl <= 2 * sms || (N + round_rows * cl - 1) / (round_rows * cl) > 8) && N > round_rows * cl) cl *= 2;
    return {lanes, cl, (N + round_rows * cl - 1) / (round_rows * cl), (unsigned)(tiles(lanes) * cl)};
}

template <typename T, bool INT8> static int rms_forward(RmsForward<T> &a, bool aligned, cudaStream_t st)
{
    const RmsPlan p = plan_rms<T>(a.N, a.F);
    a.rounds = p.rounds;
    a.fault = fault_word();
    BB200_REQUIRE(a.fault != nullptr, BBCU_ERR_NO_DEVICE);
    const bool held = p.rounds <= kHeldRows / 4;
#define BB200_RMS(L) (aligned ? (held ? k_rms_forward<T, L, true, INT8, true> : k_rms_forward<T, L, true, INT8, false>)  \
                              : (held ? k_rms_forward<T, L, false, INT8, true> : k_rms_forward<T, L, false, INT8, false>))
    auto kernel = p.lanes == 2 ? BB200_RMS(2) : BB200_RMS(8);
#undef BB200_RMS
    const int smem = p.lanes == 2 ? exchange_bytes<INT8 ? 2 : 1, Column<T, 2>::kCols>(p.cluster) : exchange_bytes<INT8 ? 2 : 1, Column<T, 8>::kCols>(p.cluster);
    return launch_cluster(kernel, (unsigned)p.cluster, p.ctas, kColumnThreads, smem, st, a);
}

template <typename T>
static int rms_forward_checked(const T *x, const T *r, T *s, T *y, int8_t *q, const float *gamma, float *rstd, float *scale, float eps, int N, int F, int xs, int rs,
                               int ss, int ys, int qs, bool int8, bbcu_stream_t stream)
{
    BB200_REQUIRE(N > 0 && F >= 0 && eps >= 0.0f, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(N <= kMostRmsNodes && F <= (1 << 27), BBCU_ERR_TOO_LARGE);
    BB200_REQUIRE(xs >= F && (!r || (rs >= F && ss >= F)), BBCU_ERR_BAD_STRIDE);
    if (int8) BB200_REQUIRE(qs >= (N + 15) / 16 * 16 && qs % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0, BBCU_ERR_BAD_STRIDE);
    else BB200_REQUIRE(ys >= F, BBCU_ERR_BAD_STRIDE);
    if (F == 0) return BBCU_OK;
    BB200_REQUIRE_PTR(x);
    if (r) BB200_REQUIRE_PTR(s);
    if (int8) { BB200_REQUIRE_PTR(q); BB200_REQUIRE_PTR(scale); }
    else { BB200_REQUIRE_PTR(y); BB200_REQUIRE_PTR(rstd); }
    RmsForward<T> a{x, r, s, y, q, gamma, rstd, scale, eps, N, F, 0, xs, rs, ss, ys, qs, nullptr};
    const bool aligned = frames_aligned<T>(x, xs) && (!r || (frames_aligned<T>(r, rs) && frames_aligned<T>(s, ss))) && (int8 || frames_aligned<T>(y, ys));
    return int8 ? rms_forward<T, true>(a, aligned, as_stream(stream)) : rms_forward<T, false>(a, aligned, as_stream(stream));
}

template <typename T>
static int rms_backward_checked(const T *s, const T *dy, const T *dr, T *ds, const float *gamma, const float *rstd, float *dgamma, int accumulate, int N, int F, int ss,
                                int dys, int drs, int dss, bbcu_stream_t stream)
{
    BB200_REQUIRE(N > 0 && F >= 0, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(N <= kMostRmsNodes && F <= (1 << 27), BBCU_ERR_TOO_LARGE);
    BB200_REQUIRE(ss >= F && dys >= F && dss >= F && (!dr || drs >= F), BBCU_ERR_BAD_STRIDE);
    cudaStream_t st = as_stream(stream);
    if (F == 0) {
        if (!accumulate && dgamma) launch(k_rms_no_frames, (unsigned)((N + 255) / 256), 256, 0, st, dgamma, N);
        return launch_status();
    }
    BB200_REQUIRE_PTR(s); BB200_REQUIRE_PTR(dy); BB200_REQUIRE_PTR(ds); BB200_REQUIRE_PTR(rstd);
    RmsBackward<T> a{s, dy, dr, ds, gamma, rstd, nullptr, N, F, 0, ss, dys, drs, dss, fault_word()};
    BB200_REQUIRE(a.fault != nullptr, BBCU_ERR_NO_DEVICE);
    const bool aligned = frames_aligned<T>(s, ss) && frames_aligned<T>(dy, dys) && frames_aligned<T>(ds, dss) && (!dr || frames_aligned<T>(dr, drs));
    const RmsPlan p = plan_rms<T>(N, F);
    a.rounds = p.rounds;
    const int tiles = (int)(p.ctas / p.cluster);
    HeldScratch held_scratch;
    if (dgamma) {
        a.gamma_part = static_cast<float *>(held_scratch.get(st, (size_t)tiles * N * sizeof(float)));
        BB200_REQUIRE(a.gamma_part != nullptr, BBCU_ERR_NO_MEMORY);
    }
    const bool held = p.rounds == 1;
#define BB200_RMS(L) (aligned ? (held ? k_rms_backward<T, L, true, true> : k_rms_backward<T, L, true, false>)  \
                              : (held ? k_rms_backward<T, L, false, true> : k_rms_backward<T, L, false, false>))
    auto kernel = p.lanes == 2 ? BB200_RMS(2) : BB200_RMS(8);
#undef BB200_RMS
    const int smem = p.lanes == 2 ? exchange_bytes<1, Column<T, 2>::kCols>(p.cluster) : exchange_bytes<1, Column<T, 8>::kCols>(p.cluster);
    if (const int e = launch_cluster(kernel, (unsigned)p.cluster, p.ctas, kColumnThreads, smem, st, a)) return e;
    if (dgamma) launch(k_rms_gamma, (unsigned)((N + 31) / 32), 256, 0, st, a.gamma_part, dgamma, N, tiles, accumulate);
    return launch_status();
}

}   // namespace bb200

using namespace bb200;

#define BB200_RMS_ENTRIES(name, T, B)                                                                                                                            \
    extern "C" int bbcu_##name##_RmsNormalization_Forward(const B *x, const B *residual, B *s, B *y, const float *gamma, float *rstd, float eps, int node_size,   \
                                                          int frame_size, int x_frame_stride, int residual_frame_stride, int s_frame_stride, int y_frame_stride, \
                                                          bbcu_stream_t stream)                                                                                  \
    {                                                                                                                                                            \
        return rms_forward_checked<T>(reinterpret_cast<const T *>(x), reinterpret_cast<const T *>(residual), reinterpret_cast<T *>(s), reinterpret_cast<T *>(y), \
                                      nullptr, gamma, rstd, nullptr, eps, node_size, frame_size, x_frame_stride, residual_frame_stride, s_frame_stride,           \
                                      y_frame_stride, 0, false, stream);                                                                                         \
    }                                                                                                                                                            \
    extern "C" int bbcu_##name##_RmsNormalization_QuantizeInt8(const B *x, const B *residual, B *s, signed char *q, float *scale, const float *gamma, float *rstd, \
                                                               float eps, int node_size, int frame_size, int x_frame_stride, int residual_frame_stride,          \
                                                               int s_frame_stride, int q_node_stride, bbcu_stream_t stream)                                      \
    {                                                                                                                                                            \
        return rms_forward_checked<T>(reinterpret_cast<const T *>(x), reinterpret_cast<const T *>(residual), reinterpret_cast<T *>(s), nullptr, q, gamma, rstd,   \
                                      scale, eps, node_size, frame_size, x_frame_stride, residual_frame_stride, s_frame_stride, 0, q_node_stride, true, stream);  \
    }                                                                                                                                                            \
    extern "C" int bbcu_##name##_RmsNormalization_Backward(const B *s, const B *dy, const B *dresidual, B *ds, const float *gamma, const float *rstd,            \
                                                           float *dgamma, int accumulate, int node_size, int frame_size, int s_frame_stride, int dy_frame_stride, \
                                                           int dresidual_frame_stride, int ds_frame_stride, bbcu_stream_t stream)                                \
    {                                                                                                                                                            \
        return rms_backward_checked<T>(reinterpret_cast<const T *>(s), reinterpret_cast<const T *>(dy), reinterpret_cast<const T *>(dresidual),                  \
                                       reinterpret_cast<T *>(ds), gamma, rstd, dgamma, accumulate, node_size, frame_size, s_frame_stride, dy_frame_stride,       \
                                       dresidual_frame_stride, ds_frame_stride, stream);                                                                         \
    }
BB200_RMS_ENTRIES(fp32, float, float)
BB200_RMS_ENTRIES(bf16, __nv_bfloat16, bbcu_bf16_t)
