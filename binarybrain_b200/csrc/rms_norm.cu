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
// Memory bounds it (16 bytes a value of fp32 forward with a residual, 16 backward).  A frame is needed whole before its first output.  Small calls take one launch: a
// cluster of CTAs has the columns of 32 or 128 bytes of a row and goes over the rows twice, or once where they stay in registers; 16 bytes of a row or less are taken
// frame by frame by lanes that hold their rows.  Large calls go along the rows
// in two passes at 5.9 to 6.9 TB/s, which move a quarter more forward with a residual (its sum is written by the first and read by the second: five rows instead of
// four), half more forward without one (three instead of two) and, with the second gradient, backward (six instead of four: s and dy are read twice).
#include <algorithm>

#include "frame_columns.cuh"
#include "quantize.cuh"

namespace bb200 {

constexpr int kMostRmsNodes = 1 << 20;
constexpr int kHeldRows = 4;

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

// a vector of s = x + r as it is kept.  (bf16: rounded once by the packed addition, which is what the sum of 32 bits rounded again gives: it is inexact only
// where the smaller term is below half of the last place.)
template <typename T> __device__ __forceinline__ uint4 add_frames(const uint4 &x, const uint4 &r)
{
    if constexpr (sizeof(T) == 2) {
        const uint32_t p[4] = {x.x, x.y, x.z, x.w}, q[4] = {r.x, r.y, r.z, r.w};
        uint32_t s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 v = __hadd2(reinterpret_cast<const __nv_bfloat162 &>(p[j]), reinterpret_cast<const __nv_bfloat162 &>(q[j]));
            s[j] = reinterpret_cast<const uint32_t &>(v);
        }
        return make_uint4(s[0], s[1], s[2], s[3]);
    } else {
        float a[4], b[4];
        unpack<T>(x, a);
        unpack<T>(r, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] += b[j];
        return pack<T>(a);
    }
}

// The end of a row: four, two and one of eight numbers.  (Apart, since it is rare and would slow the rest; one by one it took twice the time of a call whose tiles
// are few, 16384 x 100 bf16.)
__device__ __noinline__ void store_end(__nv_bfloat16 *at, uint4 v, int left)
{
    if (left & 4) *reinterpret_cast<uint2 *>(at) = make_uint2(v.x, v.y);
    if (left & 2) *reinterpret_cast<uint32_t *>(at + (left & 4)) = left & 4 ? v.z : v.x;
    if (left & 1) {
        const uint32_t word = left < 2 ? v.x : left < 4 ? v.y : left < 6 ? v.z : v.w;
        at[left & 6] = __ushort_as_bfloat16((unsigned short)word);
    }
}

template <typename T, bool ALIGNED> __device__ __forceinline__ void store_vector(T *row, int f, int F, const uint4 &v)
{
    if (ALIGNED && f + kFramesPerVec<T> <= F) {
        *reinterpret_cast<uint4 *>(row + f) = v;
    } else if constexpr (ALIGNED && sizeof(T) == 2) {
        if (f < F) store_end(row + f, v, F - f);
    } else {
        const T *const one = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int j = 0; j < kFramesPerVec<T>; ++j)
            if (f + j < F) row[f + j] = one[j];
    }
}

// The same and a load for what is read or written once: it leaves L2 first, so that what is read again stays.  (3000 x 5001 fp32 with a residual in two passes 51.4
// and 44.7 us, 1024 x 16384 bf16 in one 26.8 and 22.9.)
template <typename T, bool ONCE, bool ALIGNED> __device__ __forceinline__ uint4 load_frames_once(const T *row, int f, int F)
{
    if constexpr (ONCE) return f < F ? __ldcs(reinterpret_cast<const uint4 *>(row + f)) : make_uint4(0, 0, 0, 0);
    return load_frames<T, ALIGNED>(row, f, F);
}
template <typename T, bool ALIGNED> __device__ __forceinline__ void store_frames_once(T *row, int f, int F, const float (&v)[kFramesPerVec<T>])
{
    if (ALIGNED && f + kFramesPerVec<T> <= F) __stcs(reinterpret_cast<uint4 *>(row + f), pack<T>(v));
    else store_vector<T, ALIGNED>(row, f, F, pack<T>(v));
}
template <typename T, bool ALIGNED> __device__ __forceinline__ uint4 load_once(const Line<T, ALIGNED> &line, const T *row)
{
    if constexpr (ALIGNED) return load_frames_once<T, true, true>(row, line.first, line.F);
    return line.load(row);
}
template <typename T, bool ALIGNED> __device__ __forceinline__ void store_once(const Line<T, ALIGNED> &line, T *row, const float (&v)[kFramesPerVec<T>])
{
    if constexpr (ALIGNED) store_frames_once<T, true>(row, line.first, line.F, v);
    else line.store(row, v);
}

// the larger one, and NaN where either is
__device__ __forceinline__ float max_or_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
struct MaxOrNan { __device__ static float join(float a, float b) { return max_or_nan(a, b); } };

// A thread takes kRows neighbouring rows a round (8 bits: four, which are a word of q), the rounds of a cluster's CTAs in turn.
template <typename T, int LPR, bool ALIGNED, bool INT8, bool HELD>
__global__ void __launch_bounds__(kColumnThreads, HELD ? 2 : 4)
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
        for (int i = 0; i < kRows; ++i) raw[i] = n + i < a.N ? load_frames_once<T, ALIGNED && HELD, ALIGNED>(a.x + (long long)(n + i) * a.xs, f, a.F) : make_uint4(0, 0, 0, 0);
        if (a.r) {
#pragma unroll
            for (int i = 0; i < kRows; ++i) more[i] = n + i < a.N ? load_frames_once<T, ALIGNED, ALIGNED>(a.r + (long long)(n + i) * a.rs, f, a.F) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                raw[i] = add_frames<T>(raw[i], more[i]);
                if (n + i < a.N) store_vector<T, ALIGNED>(a.s + (long long)(n + i) * a.ss, f, a.F, raw[i]);
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
                if constexpr (INT8) v[1][j] = max_or_nan(v[1][j], fabsf(w[j] * g));
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
            if constexpr (INT8) v[1][j] = max_or_nan(v[1][j], __shfl_xor_sync(0xffffffffu, v[1][j], m));
        }
    const float inv = 1.0f / (float)a.N;
    Exchange<kQ, kCols> &e = sums[0];
    exchange_columns<kQ, T, LPR>(v, c, e, cl, 0,
        [&](const float *from, int distance, int count) { return from - &e.red[0][0] < kCols ? join_parts<ColumnSum>(from, distance, count) : join_parts<MaxOrNan>(from, distance, count); },
        [&](const float *from, int distance, int count) { return from - &e.part[0][0] < kCols ? join_parts<ColumnSum>(from, distance, count) : join_parts<MaxOrNan>(from, distance, count); },
        [&](int q, float t) { return q == 0 ? 1.0f / sqrtf(fmaf(t, inv, a.eps)) : quant_scale(__float_as_uint(t) & 0x7fffffffu); });
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
                if (n + i < a.N) store_frames_once<T, ALIGNED>(a.y + (long long)(n + i) * a.ys, f, a.F, w[i]);
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
    float *gamma_part;                                   // [tile or sweep][node]
    int N, F, rounds;
    long long ss, dys, drs, dss;
    int *fault;
};

template <typename T, int LPR, bool ALIGNED, bool HELD>
__global__ void __launch_bounds__(kColumnThreads, HELD ? 2 : 3)
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
        float along[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const float g = a.gamma && n + i < a.N ? a.gamma[n + i] : 1.0f;
            float s[kVec], d[kVec], r[kVec] = {};
            unpack<T>(s_raw[i], s);
            unpack<T>(g_raw[i], d);
            if (a.dr) unpack<T>(r_raw[i], r);
            if (f + kVec > a.F) {                                         // what lies beyond the frames may be anything
#pragma unroll
                for (int j = 0; j < kVec; ++j)
                    if (f + j >= a.F) s[j] = d[j] = 0.0f;
            }
            along[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const float xh = s[j] * rstd[j];
                along[i] = fmaf(d[j], xh, along[i]);
                d[j] = fmaf(rstd[j], fmaf(-xh, v[0][j], g * d[j]), r[j]);
            }
            if (n + i < a.N) store_vector<T, ALIGNED>(a.ds + (long long)(n + i) * a.dss, f, a.F, pack<T>(d));
        }
        if (!a.gamma_part) continue;
        // four rows over the lanes of a row: half of the rows change places for half of the lanes at each step
        static_assert(kRows == 4 && (LPR == 2 || LPR == 8));
        const bool odd = c.lane & 1;
        float p = odd ? along[2] : along[0], q = odd ? along[3] : along[1];
        p += __shfl_xor_sync(0xffffffffu, odd ? along[0] : along[2], 1);
        q += __shfl_xor_sync(0xffffffffu, odd ? along[1] : along[3], 1);
        float *const part = a.gamma_part + (long long)tile * a.N + n + (odd ? 2 : 0);
        if constexpr (LPR == 2) {
            if (n + (odd ? 2 : 0) < a.N) part[0] = p;
            if (n + (odd ? 3 : 1) < a.N) part[1] = q;
        } else {
            const bool second = c.lane & 2;
            float one = second ? q : p;
            one += __shfl_xor_sync(0xffffffffu, second ? p : q, 2);
            one += __shfl_xor_sync(0xffffffffu, one, 4);
            if (!(c.lane & 4) && n + (odd ? 2 : 0) + (second ? 1 : 0) < a.N) part[second ? 1 : 0] = one;
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
#pragma unroll 4
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

// ---- few frames: a lane has four neighbouring rows of one frame (a word of q), in up to kRounds rounds of a cluster's threads, and keeps them.  Nothing but the
// latencies of one load, one exchange and one store counts, so a lane has numbers of its own only, and what a vector of 16 bytes would bring along is not touched.
// The gradient of gamma needs no second launch, as a row's frames are neighbouring lanes.
constexpr int kFewFrames = 8, kFewRounds = 4;

template <int Q> struct FewExchange {
    float warps[32][Q * kFewFrames], ctas[8][Q * kFewFrames];
    uint64_t bar;
    int gave_up;
};

template <int Q> __device__ __forceinline__ void few_meet(FewExchange<Q> &e, const Cluster &cl)
{
    if (cl.size == 1) return;
    if (threadIdx.x == 0) {
        e.gave_up = 0;
        mbar_init(&e.bar, 1);
        mbar_init_fence();
    }
    cluster_arrive();
}

// v of all rows of a lane's frame: of the warp's lanes, the CTA's warps and the cluster's CTAs, in a fixed order.  lanes: a power of two that the frames fit in.
template <int Q, typename JOIN> __device__ __forceinline__ void few_join(float (&v)[Q], int lanes, FewExchange<Q> &e, const Cluster &cl, JOIN join)
{
    const int lane = threadIdx.x & 31, warp = (int)threadIdx.x >> 5, warps = (int)blockDim.x >> 5, f = lane & (lanes - 1);
    for (int m = lanes; m < 32; m <<= 1)
#pragma unroll
        for (int q = 0; q < Q; ++q) v[q] = join(q, v[q], __shfl_xor_sync(0xffffffffu, v[q], m));
    if (lane < lanes) {
#pragma unroll
        for (int q = 0; q < Q; ++q) e.warps[warp][q * kFewFrames + f] = v[q];
    }
    if (cl.size > 1) {
        cluster_wait();                                                   // all CTAs have their barriers
        if (threadIdx.x == 0) mbar_arrive_expect_tx(&e.bar, cl.size * Q * lanes * (uint32_t)sizeof(float));
    }
    __syncthreads();
    for (int i = warp; i < Q * lanes; i += warps) {
        const int q = i >= lanes, at = q * kFewFrames + (i & (lanes - 1));
        float s = lane < warps ? e.warps[lane][at] : 0.0f;                // 0: for a sum and for a maximum of magnitudes
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) s = join(q, s, __shfl_xor_sync(0xffffffffu, s, m));
        if (cl.size == 1) {
            if (lane == 0) e.ctas[0][at] = s;
        } else if (lane < (int)cl.size) {
            peer_send(peer_addr(&e.ctas[cl.rank][at], (uint32_t)lane), s, peer_addr(&e.bar, (uint32_t)lane));
        }
    }
    if (cl.size == 1) {
        __syncthreads();
    } else {
        int spins = 0;
        while (!mbar_try_wait(&e.bar, 0))
            if (++spins == kWaitSpins) { *(volatile int *)&e.gave_up = 1; break; }
        __syncwarp();
        cluster_arrive();
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        v[q] = e.ctas[0][q * kFewFrames + f];
        for (uint32_t r = 1; r < cl.size; ++r) v[q] = join(q, v[q], e.ctas[r][q * kFewFrames + f]);
    }
}

template <int Q> __device__ __forceinline__ void few_leave(FewExchange<Q> &e, const Cluster &cl, int *fault)
{
    if (cl.size == 1) return;
    if (*(volatile int *)&e.gave_up) atomicCAS(fault, 0, kFaultBarrierTimeout);
    cluster_wait();
}

template <typename T, bool INT8, int ROUNDS>
__global__ void __launch_bounds__(1024)
k_rms_few(const RmsForward<T> a, int lanes)
{
    constexpr int kQ = INT8 ? 2 : 1;
    __shared__ FewExchange<kQ> e;
    const Cluster cl(&e.gave_up);
    few_meet(e, cl);
    grid_dependency();
    const int f = (int)threadIdx.x & (lanes - 1), shift = __ffs(lanes) - 1;
    auto row = [&](int k) { return ((k * (int)cl.size + (int)cl.rank) * (int)blockDim.x + (int)threadIdx.x >> shift) * 4; };
    auto has = [&](int n) { return n < a.N && f < a.F; };
    float s[ROUNDS][4], g[ROUNDS][4], v[kQ] = {};
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = row(k) + i;
            s[k][i] = has(n) ? to_float(a.x[(long long)n * a.xs + f]) : 0.0f;
            g[k][i] = a.gamma && n < a.N ? a.gamma[n] : 1.0f;
        }
    if (a.r) {
        float r[ROUNDS][4];
#pragma unroll
        for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) r[k][i] = has(row(k) + i) ? to_float(a.r[(long long)(row(k) + i) * a.rs + f]) : 0.0f;
#pragma unroll
        for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const T sum = from_float<T>(s[k][i] + r[k][i]);
                s[k][i] = to_float(sum);
                if (has(row(k) + i)) a.s[(long long)(row(k) + i) * a.ss + f] = sum;
            }
    }
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[0] = fmaf(s[k][i], s[k][i], v[0]);
            if constexpr (INT8) {
                s[k][i] *= g[k][i];
                v[1] = max_or_nan(v[1], fabsf(s[k][i]));
            }
        }
    few_join(v, lanes, e, cl, [](int q, float p, float o) { return q == 0 ? p + o : max_or_nan(p, o); });
    const float rstd = 1.0f / sqrtf(fmaf(v[0], 1.0f / (float)a.N, a.eps));
    if constexpr (INT8) {
        const float unit = quant_scale(__float_as_uint(v[1]) & 0x7fffffffu);
        if (cl.rank == 0 && (int)threadIdx.x < a.F) {
            a.scale[f] = unit * rstd;
            if (a.rstd) a.rstd[f] = rstd;
        }
        const Quantizer quantizer(unit);
        const int end = (a.N + 15) / 16 * 16;                             // zeros as far as the row's last 16 bytes
#pragma unroll
        for (int k = 0; k < ROUNDS; ++k)
            if (row(k) < end && f < a.F) *reinterpret_cast<uint32_t *>(a.q + (long long)f * a.qs + row(k)) = quantizer(s[k][0], s[k][1], s[k][2], s[k][3]);
    } else {
        if (cl.rank == 0 && (int)threadIdx.x < a.F) a.rstd[f] = rstd;
#pragma unroll
        for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (has(row(k) + i)) a.y[(long long)(row(k) + i) * a.ys + f] = from_float<T>((s[k][i] * rstd) * g[k][i]);
    }
    few_leave(e, cl, a.fault);
}

template <typename T, int ROUNDS>
__global__ void __launch_bounds__(1024)
k_rms_grad_few(const RmsBackward<T> a, float *dgamma, int accumulate, int lanes)
{
    __shared__ FewExchange<1> e;
    const Cluster cl(&e.gave_up);
    few_meet(e, cl);
    grid_dependency();
    const int f = (int)threadIdx.x & (lanes - 1), shift = __ffs(lanes) - 1;
    auto row = [&](int k) { return ((k * (int)cl.size + (int)cl.rank) * (int)blockDim.x + (int)threadIdx.x >> shift) * 4; };
    auto has = [&](int n) { return n < a.N && f < a.F; };
    const float rstd = f < a.F ? a.rstd[f] : 0.0f;
    float xh[ROUNDS][4], d[ROUNDS][4], v[1] = {};
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = row(k) + i;
            xh[k][i] = has(n) ? to_float(a.s[(long long)n * a.ss + f]) : 0.0f;
            d[k][i] = has(n) ? to_float(a.dy[(long long)n * a.dys + f]) : 0.0f;
        }
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = row(k) + i;
            const float g = a.gamma && n < a.N ? a.gamma[n] : 1.0f;
            xh[k][i] *= rstd;
            float along = d[k][i] * xh[k][i];
            v[0] = fmaf(g * d[k][i], xh[k][i], v[0]);
            d[k][i] *= g;
            if (dgamma) {
                for (int m = 1; m < lanes; m <<= 1) along += __shfl_xor_sync(0xffffffffu, along, m);
                if (f == 0 && n < a.N) dgamma[n] = accumulate ? dgamma[n] + along : along;
            }
        }
    few_join(v, lanes, e, cl, [](int, float p, float o) { return p + o; });
    const float c = v[0] / (float)a.N;
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
        float r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = a.dr && has(row(k) + i) ? to_float(a.dr[(long long)(row(k) + i) * a.drs + f]) : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (has(row(k) + i)) a.ds[(long long)(row(k) + i) * a.dss + f] = from_float<T>(fmaf(rstd, fmaf(-xh[k][i], c, d[k][i]), r[i]));
    }
    few_leave(e, cl, a.fault);
}

// ---- large layers in two passes along the rows: a CTA has 512 bytes of the rows of a band, a warp every eighth of them, and the bands are as many as the device
// holds at a time.  The first pass adds up the columns of its band (part[band][frame], for 8 bits the largest numbers as well), the second one makes the output,
// and goes through the rows of its band from the end, where L2 still holds what the first one left there.  (Held by clusters in shared memory and read once,
// in columns of 64 and 128 bytes, these layers ran at 4.6 to 5.0 TB/s, with or without the exchange of sums; along the rows a copy runs at 6.5.)
constexpr int kBandWarps = 8, kBandBatch = 4;

// sums of the warps' columns, in the order of the warps; the first warp of the CTA has them
template <typename T, bool ALIGNED, int Q, typename JOIN>
__device__ __forceinline__ void store_band(float (&v)[Q][kFramesPerVec<T>], float *part, int bands, int band, int padded, const Line<T, ALIGNED> &line, JOIN join)
{
    constexpr int kVec = kFramesPerVec<T>;
    __shared__ float red[kBandWarps][Q][kVec][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int j = 0; j < kVec; ++j) red[warp][q][j][lane] = v[q][j];
    __syncthreads();
    // a warp joins some of the values
    for (int e = warp; e < Q * kVec; e += kBandWarps) {
        const int q = e / kVec, j = e % kVec;
        float s = red[0][q][j][lane];
        for (int w = 1; w < kBandWarps; ++w) s = join(q, s, red[w][q][j][lane]);
        if (line.frame(j) < line.F) part[((long long)q * bands + band) * padded + line.frame(j)] = s;
    }
}

template <typename T, bool ALIGNED, bool RESIDUAL, bool INT8>
__global__ void __launch_bounds__(32 * kBandWarps, 4)
k_rms_sums(const RmsForward<T> a, float *part, int rows, int padded)
{
    grid_dependency();
    constexpr int kVec = kFramesPerVec<T>, kQ = INT8 ? 2 : 1;
    const Line<T, ALIGNED> line((int)blockIdx.x * 32 * kVec, (int)(threadIdx.x & 31), a.F);
    const int first = (int)blockIdx.y * rows, end = min(first + rows, a.N);
    float v[kQ][kVec] = {};
    for (int n = first + (int)(threadIdx.x >> 5); n < end; n += kBandWarps * kBandBatch) {
        uint4 raw[kBandBatch], more[kBandBatch];
#pragma unroll
        for (int i = 0; i < kBandBatch; ++i)
            if (n + i * kBandWarps < end) raw[i] = RESIDUAL && !INT8 ? load_once(line, a.x + (n + i * kBandWarps) * a.xs) : line.load(a.x + (n + i * kBandWarps) * a.xs);
        if (RESIDUAL) {
#pragma unroll
            for (int i = 0; i < kBandBatch; ++i)
                if (n + i * kBandWarps < end) more[i] = INT8 ? line.load(a.r + (n + i * kBandWarps) * a.rs) : load_once(line, a.r + (n + i * kBandWarps) * a.rs);
        }
#pragma unroll
        for (int i = 0; i < kBandBatch; ++i) {
            const int m = n + i * kBandWarps;
            if (m >= end) break;
            float w[kVec];
            if (RESIDUAL) {
                raw[i] = add_frames<T>(raw[i], more[i]);
                unpack<T>(raw[i], w);
                line.store(a.s + m * a.ss, w);
            } else {
                unpack<T>(raw[i], w);
            }
            const float g = INT8 && a.gamma ? a.gamma[m] : 1.0f;
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                v[0][j] = fmaf(w[j], w[j], v[0][j]);
                if constexpr (INT8) v[1][j] = max_or_nan(v[1][j], fabsf(w[j] * g));
            }
        }
    }
    store_band<T, ALIGNED, kQ>(v, part, (int)gridDim.y, (int)blockIdx.y, padded, line, [](int q, float p, float o) { return q == 0 ? p + o : max_or_nan(p, o); });
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(32 * kBandWarps, 4)
k_rms_apply(const RmsForward<T> a, const float *__restrict__ part, int rows, int padded)
{
    grid_dependency();
    constexpr int kVec = kFramesPerVec<T>;
    __shared__ float red[kBandWarps][kVec][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Line<T, ALIGNED> line((int)blockIdx.x * 32 * kVec, lane, a.F);
    const int first = (int)blockIdx.y * rows, end = min(first + rows, a.N);
    const T *const in = a.r ? a.s : a.x;
    const long long stride = a.r ? a.ss : a.xs;
    int n = end - 1 - warp;
    uint4 raw[kBandBatch];
    auto load = [&] {
#pragma unroll
        for (int i = 0; i < kBandBatch; ++i)
            if (n - i * kBandWarps >= first && !line.empty()) raw[i] = line.load(in + (n - i * kBandWarps) * stride);
    };
    load();                                                               // on their way beside the parts of the sums, of which each warp adds up some
    float rstd[kVec] = {};
#pragma unroll 4
    for (int b = warp; b < (int)gridDim.y; b += kBandWarps) {
        float p[kVec];
        line.load_columns(part + (long long)b * padded, p);
#pragma unroll
        for (int j = 0; j < kVec; ++j) rstd[j] += p[j];
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) red[warp][j][lane] = rstd[j];
    __syncthreads();
    if (line.empty()) return;
    const float inv = 1.0f / (float)a.N;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        float s = red[0][j][lane];
#pragma unroll
        for (int w = 1; w < kBandWarps; ++w) s += red[w][j][lane];
        rstd[j] = 1.0f / sqrtf(fmaf(s, inv, a.eps));
        if (blockIdx.y == 0 && warp == 0 && line.frame(j) < a.F) a.rstd[line.frame(j)] = rstd[j];
    }
    while (n >= first) {
#pragma unroll
        for (int i = 0; i < kBandBatch; ++i) {
            const int m = n - i * kBandWarps;
            if (m < first) break;
            const float g = a.gamma ? a.gamma[m] : 1.0f;
            float w[kVec];
            unpack<T>(raw[i], w);
#pragma unroll
            for (int j = 0; j < kVec; ++j) w[j] = (w[j] * rstd[j]) * g;
            store_once(line, a.y + m * a.ys, w);
        }
        n -= kBandWarps * kBandBatch;
        load();
    }
}

// The parts of the bands joined over a frame: eight threads take some of them each, and one adds up what they have in a fixed order.
template <int Q, typename JOIN> __device__ __forceinline__ bool join_bands(const float *__restrict__ part, int bands, int padded, int F, int &f, float (&v)[Q], JOIN join)
{
    __shared__ float s[8][Q][32];
    const int lane = threadIdx.x & 31, some = threadIdx.x >> 5;
    f = (int)blockIdx.x * 32 + lane;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        v[q] = 0.0f;
#pragma unroll 4
        for (int b = some; b < bands; b += 8)
            if (f < F) v[q] = join(q, v[q], part[((long long)q * bands + b) * padded + f]);
        s[some][q][lane] = v[q];
    }
    __syncthreads();
    if (some || f >= F) return false;
#pragma unroll
    for (int q = 0; q < Q; ++q)
        for (int i = 1; i < 8; ++i) v[q] = join(q, v[q], s[i][q][lane]);
    return true;
}

// unit[frame] for k_rms_quantize, scale and rstd
__global__ void __launch_bounds__(256)
k_rms_scales(const float *__restrict__ part, int bands, int padded, float *unit_out, float *scale_out, float *rstd_out, float eps, int N, int F)
{
    grid_dependency();
    int f;
    float v[2];
    if (!join_bands<2>(part, bands, padded, F, f, v, [](int q, float a, float b) { return q == 0 ? a + b : max_or_nan(a, b); })) return;
    const float rstd = 1.0f / sqrtf(fmaf(v[0], 1.0f / (float)N, eps)), unit = quant_scale(__float_as_uint(v[1]) & 0x7fffffffu);
    unit_out[f] = unit;
    scale_out[f] = unit * rstd;
    if (rstd_out) rstd_out[f] = rstd;
}

// 256 rows x 128 bytes of s turned over into rows of q, as by k_quantize_apply of the quantisers, from the last rows on
constexpr int kRmsQuantRows = 256;
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256)
k_rms_quantize(const T *s, int8_t *q, const float *__restrict__ gamma, const float *__restrict__ unit_in, int N, int F, long long ss, long long qs)
{
    grid_dependency();
    constexpr int kLpr = 8, kPieces = kRmsQuantRows / 16;
    using Col = Column<T, kLpr>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    __shared__ __align__(16) uint32_t tile[kCols][kRmsQuantRows / 4];
    const Col c;
    const int f0 = (int)blockIdx.x * kCols, f = f0 + c.col, n0 = (int)(gridDim.y - 1 - blockIdx.y) * kRmsQuantRows, n = n0 + 4 * c.row;
    uint4 raw[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = n + 128 * h + i;
            raw[h][i] = m < N ? load_frames<T, ALIGNED>(s + m * ss, f, F) : make_uint4(0, 0, 0, 0);
        }
    float unit[kVec];
    load_columns(unit_in, f, F, unit);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float v[4][kVec];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unpack<T>(raw[h][i], v[i]);
            const float g = gamma && n + 128 * h + i < N ? gamma[n + 128 * h + i] : 1.0f;
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[i][j] *= g;
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j)
            tile[c.col + j][h * 32 + (c.row / 4 ^ c.lane % kLpr) * 4 + c.row % 4] = Quantizer(unit[j])(v[0][j], v[1][j], v[2][j], v[3][j]);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < kCols * kPieces; e += 256) {
        const int col = e / kPieces, piece = e % kPieces, m = n0 + 16 * piece;
        if (f0 + col < F && m < N)
            *reinterpret_cast<uint4 *>(q + (long long)(f0 + col) * qs + m) = *reinterpret_cast<const uint4 *>(&tile[col][(piece ^ col / kVec) * 4]);
    }
}

// backward: part[band][frame] = the band's sum of gamma dy xh
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(32 * kBandWarps, 4)
k_rms_grad_sums(const RmsBackward<T> a, float *part, int rows, int padded)
{
    grid_dependency();
    constexpr int kVec = kFramesPerVec<T>;
    const Line<T, ALIGNED> line((int)blockIdx.x * 32 * kVec, (int)(threadIdx.x & 31), a.F);
    const int first = (int)blockIdx.y * rows, end = min(first + rows, a.N);
    float v[1][kVec] = {}, rstd[kVec];
    line.load_columns(a.rstd, rstd);
    for (int n = first + (int)(threadIdx.x >> 5); n < end; n += kBandWarps * kBandBatch) {
        uint4 s_raw[kBandBatch], d_raw[kBandBatch];
#pragma unroll
        for (int i = 0; i < kBandBatch; ++i)
            if (n + i * kBandWarps < end) {
                s_raw[i] = line.load(a.s + (n + i * kBandWarps) * a.ss);
                d_raw[i] = line.load(a.dy + (n + i * kBandWarps) * a.dys);
            }
#pragma unroll
        for (int i = 0; i < kBandBatch; ++i) {
            const int m = n + i * kBandWarps;
            if (m >= end) break;
            const float g = a.gamma ? a.gamma[m] : 1.0f;
            float s[kVec], d[kVec];
            unpack<T>(s_raw[i], s);
            unpack<T>(d_raw[i], d);
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[0][j] = fmaf(g * d[j], s[j] * rstd[j], v[0][j]);
        }
    }
    store_band<T, ALIGNED, 1>(v, part, (int)gridDim.y, (int)blockIdx.y, padded, line, [](int, float p, float o) { return p + o; });
}

// mean[frame] = the mean over all rows
__global__ void __launch_bounds__(256) k_rms_grad_means(const float *__restrict__ part, int bands, int padded, float *mean, int N, int F)
{
    grid_dependency();
    int f;
    float v[1];
    if (join_bands<1>(part, bands, padded, F, f, v, [](int, float a, float b) { return a + b; })) mean[f] = v[0] / (float)N;
}

// A CTA has 8 x kGradRows rows and every gridDim.x-th piece of 512 bytes of them, and adds up their sums over the frames on the way: gamma_part[blockIdx.x][node].
// The rows are those of the bands' ends first.
constexpr int kGradRows = 4;
template <typename T, bool ALIGNED, bool RESIDUAL>
__global__ void __launch_bounds__(32 * kBandWarps, 2)
k_rms_grad_apply(const RmsBackward<T> a, const float *__restrict__ mean_in, int rows, int bands)
{
    grid_dependency();
    constexpr int kVec = kFramesPerVec<T>, R = kGradRows;
    const int lane = threadIdx.x & 31, band = (int)blockIdx.y % bands, back = (int)blockIdx.y / bands;
    const int end = min((band + 1) * rows, a.N), top = end - (back * kBandWarps + (int)(threadIdx.x >> 5)) * R, n0 = max(top - R, band * rows);
    const int mine = top - n0;                                            // rows of the warp, below 1: none
    float along[R] = {}, gm[R];
#pragma unroll
    for (int i = 0; i < R; ++i) gm[i] = a.gamma && i < mine ? a.gamma[n0 + i] : 1.0f;
    if (mine > 0)
        for (int f0 = (int)blockIdx.x * 32 * kVec; f0 < a.F; f0 += (int)gridDim.x * 32 * kVec) {
            const Line<T, ALIGNED> line(f0, lane, a.F);
            if (line.empty()) break;
            uint4 s_raw[R], d_raw[R], r_raw[R];
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (i < mine) {
                    s_raw[i] = line.load(a.s + (n0 + i) * a.ss);
                    d_raw[i] = line.load(a.dy + (n0 + i) * a.dys);
                    if (RESIDUAL) r_raw[i] = load_once(line, a.dr + (n0 + i) * a.drs);
                }
            float rstd[kVec], mean[kVec];
            line.load_columns(a.rstd, rstd);
            line.load_columns(mean_in, mean);
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (i < mine) {
                    float s[kVec], d[kVec], r[kVec] = {};
                    unpack<T>(s_raw[i], s);
                    unpack<T>(d_raw[i], d);
                    if (RESIDUAL) unpack<T>(r_raw[i], r);
                    if (line.frame(kVec - 1) >= a.F) {                    // what lies beyond the frames may be anything
#pragma unroll
                        for (int j = 0; j < kVec; ++j)
                            if (line.frame(j) >= a.F) s[j] = d[j] = 0.0f;
                    }
#pragma unroll
                    for (int j = 0; j < kVec; ++j) {
                        const float xh = s[j] * rstd[j];
                        along[i] = fmaf(d[j], xh, along[i]);
                        d[j] = fmaf(rstd[j], fmaf(-xh, mean[j], gm[i] * d[j]), r[j]);
                    }
                    store_once(line, a.ds + (n0 + i) * a.dss, d);
                }
        }
    if (!a.gamma_part) return;
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) along[i] += __shfl_xor_sync(0xffffffffu, along[i], m);
        if (lane == i && i < mine) a.gamma_part[(long long)blockIdx.x * a.N + n0 + i] = along[i];
    }
}

// Pieces of 512 bytes along the frames, bands that make one round of CTAs, four an SM, with whole batches of rows
constexpr long long kRmsInL2 = 104 << 20, kRmsFew = 1 << 21;              // bytes, values
// Backward: us, one launch and two passes: 4096 x 1024 fp32 15.0 / 19.0, 1024 x 4096 20.6 / 16.7, 5000 x 1000 bf16 33 / 20.6, 16384 x 100 fp32 15.1 / 30.8.
constexpr long long kRmsGradSmall = 1 << 22;             // values
struct BandPlan { int pieces, bands, rows, padded; };
template <typename T> static BandPlan plan_bands(int N, int F)
{
    constexpr int kWide = 32 * kFramesPerVec<T>, kUnit = kBandWarps * kBandBatch;
    const int pieces = (F + kWide - 1) / kWide, slots = 4 * device_info().sm_count;
    const int bands = std::max(1, std::min({slots / pieces, (N + kUnit - 1) / kUnit, 65535}));
    const int rows = ((N + bands - 1) / bands + kUnit - 1) / kUnit * kUnit;
    return {pieces, (N + rows - 1) / rows, rows, (F + 3) / 4 * 4};
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

// Lanes of a row, CTAs of the cluster (with 256 threads or more each), their threads and rounds; 0 rounds where this is not for the size.  (Device times in a graph, with
// a residual, by vectors and by lanes, us: 8 bits of 4096 x 1 bf16 7.9 and 5.2, backward 7.7 and 6.8, 16384 x 1 19.4 and 10.1, 30000 x 3 fp32 27.3 and 18.2, 65536 x 1
// 60.5 and 29.1; 4096 x 8 bf16 8.0 and 5.2, 7.5 and 7.0; beyond 16 bytes of a row vectors win, backward of 4096 x 12 fp32 6.6 and 9.7, 4096 x 16 bf16 7.1 and 9.6.)
struct FewPlan { int lanes, cluster, threads, rounds; };
template <typename T> static FewPlan plan_few(int N, int F)
{
    static_assert(kFramesPerVec<T> <= kFewFrames, "a frame a lane");
    if (F > kFramesPerVec<T>) return {};
    int lanes = 1, cl = 1, rounds = 1;
    while (lanes < F) lanes *= 2;
    const long long units = ((long long)N + 15) / 16 * 4 * lanes;         // of four rows
    while (cl < 8 && cl * 256 < units) cl *= 2;
    while (rounds <= kFewRounds && cl * 1024ll * rounds < units) rounds *= 2;
    if (rounds > kFewRounds) return {};
    return {lanes, cl, (int)((units + 32ll * cl * rounds - 1) / (32ll * cl * rounds)) * 32, rounds};
}

template <typename T, bool INT8> static int rms_forward(RmsForward<T> &a, bool aligned, cudaStream_t st)
{
    // The cluster's second reading finds L2 as the first one left it where everything fits there, and costs a latency a round where columns are few and long.  (us, one
    // launch and two passes: 1024 x 16384 bf16 with a residual 21.1 / 26.4, fp32 55.9 / 49.7; 4096 x 1024 fp32 12.3 / 13.6; 5000 x 1000 bf16 20.4 / 16.4; 16384 x 100 fp32
    // 13.5 / 27.2.)
    a.fault = fault_word();
    BB200_REQUIRE(a.fault != nullptr, BBCU_ERR_NO_DEVICE);
    if (const FewPlan few = plan_few<T>(a.N, a.F); few.rounds) {
        auto kernel = few.rounds == 1 ? k_rms_few<T, INT8, 1> : few.rounds == 2 ? k_rms_few<T, INT8, 2> : k_rms_few<T, INT8, kFewRounds>;
        return launch_cluster(kernel, (unsigned)few.cluster, (unsigned)few.cluster, (unsigned)few.threads, 0, st, a, few.lanes);
    }
    const RmsPlan p = plan_rms<T>(a.N, a.F);
    const bool held = p.rounds <= kHeldRows / 4;
    const long long values = (long long)a.N * a.F, bytes = values * (long long)sizeof(T) * (a.r ? 3 : 1);
    if (!held && (bytes > kRmsInL2 || (p.rounds > 4 && values > kRmsFew))) {
        const BandPlan b = plan_bands<T>(a.N, a.F);
        HeldScratch held;
        float *part = static_cast<float *>(held.get(st, ((size_t)b.bands * (INT8 ? 2 : 1) + 1) * b.padded * sizeof(float)));
        BB200_REQUIRE(part != nullptr, BBCU_ERR_NO_MEMORY);
        const dim3 grid((unsigned)b.pieces, (unsigned)b.bands);
        auto sums = aligned ? (a.r ? k_rms_sums<T, true, true, INT8> : k_rms_sums<T, true, false, INT8>) : (a.r ? k_rms_sums<T, false, true, INT8> : k_rms_sums<T, false, false, INT8>);
        launch(sums, grid, 32 * kBandWarps, 0, st, a, part, b.rows, b.padded);
        BB200_CUDA(cudaPeekAtLastError());
        if constexpr (INT8) {
            float *const unit = part + 2LL * b.bands * b.padded;
            constexpr int kCols = Column<T, 8>::kCols;
            const int bands = (a.N + kRmsQuantRows - 1) / kRmsQuantRows;
            launch(k_rms_scales, (unsigned)((a.F + 31) / 32), 256, 0, st, part, b.bands, b.padded, unit, a.scale, a.rstd, a.eps, a.N, a.F);
            launch(aligned ? k_rms_quantize<T, true> : k_rms_quantize<T, false>, dim3((unsigned)((a.F + kCols - 1) / kCols), (unsigned)bands), 256, 0, st, a.r ? a.s : a.x, a.q, a.gamma,
                   unit, a.N, a.F, a.r ? a.ss : a.xs, a.qs);
        } else {
            launch(aligned ? k_rms_apply<T, true> : k_rms_apply<T, false>, grid, 32 * kBandWarps, 0, st, a, part, b.rows, b.padded);
        }
        return launch_status();
    }
    a.rounds = p.rounds;
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
    if (const FewPlan few = plan_few<T>(N, F); few.rounds) {
        auto kernel = few.rounds == 1 ? k_rms_grad_few<T, 1> : few.rounds == 2 ? k_rms_grad_few<T, 2> : k_rms_grad_few<T, kFewRounds>;
        return launch_cluster(kernel, (unsigned)few.cluster, (unsigned)few.cluster, (unsigned)few.threads, 0, st, a, dgamma, accumulate, few.lanes);
    }
    HeldScratch held_scratch;
    if ((long long)N * F > kRmsGradSmall) {
        const BandPlan b = plan_bands<T>(N, F);
        const int backs = (b.rows + kBandWarps * kGradRows - 1) / (kBandWarps * kGradRows);
        const long long groups = (long long)b.bands * backs;
        BB200_REQUIRE(groups <= 65535, BBCU_ERR_TOO_LARGE);
        const int sweeps = (int)std::min<long long>(b.pieces, std::max(1LL, (8LL * device_info().sm_count + groups - 1) / groups));
        const size_t sums = ((size_t)b.bands + 1) * b.padded;
        float *part = static_cast<float *>(held_scratch.get(st, (sums + (dgamma ? (size_t)sweeps * N : 0)) * sizeof(float)));
        BB200_REQUIRE(part != nullptr, BBCU_ERR_NO_MEMORY);
        float *const mean = part + (size_t)b.bands * b.padded;
        if (dgamma) a.gamma_part = part + sums;
        launch(aligned ? k_rms_grad_sums<T, true> : k_rms_grad_sums<T, false>, dim3((unsigned)b.pieces, (unsigned)b.bands), 32 * kBandWarps, 0, st, a, part, b.rows, b.padded);
        BB200_CUDA(cudaPeekAtLastError());
        launch(k_rms_grad_means, (unsigned)((F + 31) / 32), 256, 0, st, part, b.bands, b.padded, mean, N, F);
        auto apply = aligned ? (dr ? k_rms_grad_apply<T, true, true> : k_rms_grad_apply<T, true, false>) : (dr ? k_rms_grad_apply<T, false, true> : k_rms_grad_apply<T, false, false>);
        launch(apply, dim3((unsigned)sweeps, (unsigned)groups), 32 * kBandWarps, 0, st, a, mean, b.rows, b.bands);
        if (dgamma) launch(k_rms_gamma, (unsigned)((N + 31) / 32), 256, 0, st, a.gamma_part, dgamma, N, sweeps, accumulate);
        return launch_status();
    }
    const RmsPlan p = plan_rms<T>(N, F);
    a.rounds = p.rounds;
    const int tiles = (int)(p.ctas / p.cluster);
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
