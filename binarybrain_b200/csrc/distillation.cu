// Distillation from a teacher's top logits: loss and gradient of the student's logits in one call, on node-major frame buffers (class = node).
// (The reference's losses are LossSoftmaxCrossEntropy and LossMeanSquaredError, include/bb/LossSoftmaxCrossEntropy.h:151-205; it has no counterpart.)
//
// Per frame, with temperature T, student logits z_c and up to K teacher slots (class i_k, logit t_k; a slot whose class lies outside or whose logit is -inf is empty):
//
//   p_k = exp(t_k / T - L),  L = log sum_k exp(t_k / T) over the slots, or the caller's log sum over all of the teacher's classes
//   q_c = exp(z_c / T) / sum_c exp(z_c / T)
//   loss = T^2 sum_k p_k (log p_k - log q_{i_k}),      dz_c = T (P q_c - sum_{k: i_k = c} p_k),  P = sum_k p_k
//
// both times the frame's weight; a slot with p_k = 0 adds nothing, whatever its class's log q is, and a class that is named twice gets both.  A frame
// without a slot, or of weight 0, has loss 0 and gradient 0 whatever its logits are.  exp(z / T) is evaluated as exp2((z - max z) log2(e) / T).
#include "frame_columns.cuh"

namespace bb200 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kDistillThreads = 256;

// maximum and sum of exponentials relative to it, of two sets joined; an empty set, and one of -inf alone, is (-inf, 0)
struct SoftSum { float top, sum; };
__device__ __forceinline__ SoftSum join_soft(const SoftSum &a, const SoftSum &b, float scale)
{
    const float top = fmaxf(a.top, b.top);
    if (top == -INFINITY) return {top, a.sum + b.sum};                    // (a NaN among them stays)
    return {top, a.sum * exp2f((a.top - top) * scale) + b.sum * exp2f((b.top - top) * scale)};
}

// part[chunk][column] of the student's logits
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kDistillThreads)
k_distill_stats(const T *z, SoftSum *part, float scale, int C, int F, long long zs, int chunk_rows, int columns)
{
    grid_dependency();
    constexpr int kLpr = 8, kBatch = 8;
    using Col = Column<T, kLpr>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    __shared__ SoftSum s[8][kCols];
    const Col c;
    const int f = (int)blockIdx.x * kCols + c.col;
    const int n0 = (int)blockIdx.y * chunk_rows, n1 = min(C, n0 + chunk_rows);
    SoftSum a[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) a[j] = {-INFINITY, 0.0f};
    for (int n = n0 + c.row; n < n1; n += c.step * kBatch) {
        uint4 raw[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * c.step;
            if (m < n1) raw[i] = load_frames<T, ALIGNED>(z + (long long)m * zs, f, F);
        }
        float top[kVec];
#pragma unroll
        for (int j = 0; j < kVec; ++j) top[j] = a[j].top;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (n + i * c.step < n1) {
                float v[kVec];
                unpack<T>(raw[i], v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) top[j] = fmaxf(top[j], v[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            a[j].sum *= a[j].top == -INFINITY ? 1.0f : exp2f((a[j].top - top[j]) * scale);
            a[j].top = top[j];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (n + i * c.step < n1) {
                float v[kVec];
                unpack<T>(raw[i], v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) a[j].sum += v[j] == -INFINITY ? 0.0f : exp2f((v[j] - top[j]) * scale);
            }
        }
    }
#pragma unroll
    for (int m = kLpr; m < 32; m <<= 1)
#pragma unroll
        for (int j = 0; j < kVec; ++j)
            a[j] = join_soft(a[j], {__shfl_xor_sync(0xffffffffu, a[j].top, m), __shfl_xor_sync(0xffffffffu, a[j].sum, m)}, scale);
    if (c.lane < kLpr) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) s[c.warp][c.col + j] = a[j];
    }
    __syncthreads();
    if (threadIdx.x < kCols) {
        SoftSum t = s[0][threadIdx.x];
        for (int w = 1; w < c.warps; ++w) t = join_soft(t, s[w][threadIdx.x], scale);
        part[(long long)blockIdx.y * columns + (long long)blockIdx.x * kCols + threadIdx.x] = t;
    }
}

// One thread a frame, its slots one after the other: coef[0] = max z, coef[1] = factor of exp2 in dz, loss_buf; and the slots' classes, -1 where the
// slot is empty or its class has been named by an earlier one, with the probabilities of a class added up, in slot_index / slot_p [K][columns].
template <typename T>
__global__ void __launch_bounds__(kDistillThreads)
k_distill_teacher(const T *z, const T *__restrict__ t, const int *__restrict__ index, const float *__restrict__ t_lse, const float *__restrict__ weight,
                  const SoftSum *__restrict__ part, float *coef, int *slot_index, float *slot_p, float *loss_buf, double *loss_part, float temperature,
                  float grad_reduction, double loss_reduction, int C, int K, int F, long long zs, long long ts, long long is, int chunks, int columns)
{
    grid_dependency();
    __shared__ double red[kDistillThreads / 32];
    const float inv_t = 1.0f / temperature, scale = kLog2e * inv_t;
    const int f = (int)blockIdx.x * kDistillThreads + threadIdx.x;
    double loss = 0.0;
    if (f < F) {
        SoftSum s = part[f];
        for (int k = 1; k < chunks; ++k) s = join_soft(s, part[(long long)k * columns + f], scale);
        const float w = weight ? weight[f] : 1.0f;
        float top = -INFINITY;
        int slots = 0;
        for (int k = 0; k < K; ++k) {
            const int i = index[k * is + f];
            const float tk = to_float(t[k * ts + f]);
            if (i >= 0 && i < C && tk != -INFINITY) { top = fmaxf(top, tk); ++slots; }
        }
        const bool live = slots > 0 && w != 0.0f;
        float lse = 0.0f;
        if (live) {
            if (t_lse) {
                lse = t_lse[f];
            } else {
                float sum = 0.0f;
                for (int k = 0; k < K; ++k) {
                    const int i = index[k * is + f];
                    const float tk = to_float(t[k * ts + f]);
                    if (i >= 0 && i < C && tk != -INFINITY) sum += exp2f((tk - top) * scale);
                }
                lse = top * inv_t + logf(sum);
            }
        }
        const float log_sum = logf(s.sum);
        float P = 0.0f, l = 0.0f;
        for (int k = 0; k < K; ++k) {
            const int i = index[k * is + f];
            const float tk = to_float(t[k * ts + f]);
            const bool has = live && i >= 0 && i < C && tk != -INFINITY;
            float p = 0.0f;
            if (has) {
                const float log_p = tk * inv_t - lse;
                p = exp2f(log_p * kLog2e);
                const float zi = to_float(z[i * zs + f]);
                const float log_q = zi == -INFINITY ? -INFINITY : (zi - s.top) * inv_t - log_sum;
                if (p != 0.0f) l += p * (log_p - log_q);
                P += p;
            }
            int owner = has ? i : -1;
            for (int e = 0; e < k && owner >= 0; ++e)
                if (slot_index[(long long)e * columns + f] == i) {
                    slot_p[(long long)e * columns + f] += p;
                    owner = -1;
                }
            slot_index[(long long)k * columns + f] = owner;
            slot_p[(long long)k * columns + f] = p;
        }
        const float g = live ? grad_reduction * w * temperature : 0.0f;
        coef[f] = s.top;
        coef[columns + f] = live ? g * P / s.sum : 0.0f;
        coef[2 * columns + f] = g;
        l = live ? w * temperature * temperature * l : 0.0f;
        loss_buf[f] = l;
        loss = (double)l;
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = loss;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < kDistillThreads / 32; ++k) loss += red[k];
        loss_part[blockIdx.x] = loss * loss_reduction;
    }
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kDistillThreads)
k_distill_apply(const T *z, T *dz, const float *__restrict__ coef, const int *__restrict__ slot_index, const float *__restrict__ slot_p,
                const double *__restrict__ loss_part, int loss_parts, float *loss, float scale, int C, int K, int F, long long zs, long long dzs, int chunk_rows,
                int columns)
{
    grid_dependency();
    constexpr int kLpr = 8, kBatch = 8;
    using Col = Column<T, kLpr>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    const Col c;
    const int f0 = (int)blockIdx.x * kCols, f = f0 + c.col;
    const int n0 = (int)blockIdx.y * chunk_rows, n1 = min(C, n0 + chunk_rows);
    float top[kVec], fac[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) { top[j] = f + j < F ? coef[f + j] : 0.0f; fac[j] = f + j < F ? coef[columns + f + j] : 0.0f; }
    for (int n = n0 + c.row; n < n1; n += c.step * kBatch) {
        uint4 raw[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * c.step;
            if (m < n1) raw[i] = load_frames<T, ALIGNED>(z + (long long)m * zs, f, F);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * c.step;
            if (m < n1) {
                float v[kVec];
                unpack<T>(raw[i], v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) v[j] = fac[j] == 0.0f || v[j] == -INFINITY ? 0.0f : fac[j] * exp2f((v[j] - top[j]) * scale);
                store_frames<T, ALIGNED>(dz + (long long)m * dzs, f, F, v);
            }
        }
    }
    __syncthreads();                                                     // the block's own values of dz stand before the named classes are written again
    for (int e = threadIdx.x; e < K * kCols; e += kDistillThreads) {
        const int g = f0 + e % kCols;
        const long long at = (long long)(e / kCols) * columns + g;
        if (g >= F) continue;
        const int i = slot_index[at];
        if (i < n0 || i >= n1) continue;
        const float v = to_float(z[i * zs + g]), fc = coef[columns + g];
        const float q = fc == 0.0f || v == -INFINITY ? 0.0f : fc * exp2f((v - coef[g]) * scale);
        dz[i * dzs + g] = from_float<T>(q - coef[2 * columns + g] * slot_p[at]);
    }
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 32) {
        double s = 0.0;
        for (int k = threadIdx.x; k < loss_parts; k += 32) s += loss_part[k];
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        if (threadIdx.x == 0) *loss = (float)s;
    }
}

template <typename T>
static int distillation(const T *z, T *dz, const T *t, const int *index, const float *t_lse, const float *weight, float *loss_buf, float *loss,
                        float temperature, float grad_reduction, double loss_reduction, int C, int K, int F, long long zs, long long dzs, long long ts,
                        long long is, cudaStream_t st)
{
    const bool aligned = frames_aligned<T>(z, zs) && frames_aligned<T>(dz, dzs);
    constexpr int kCols = Column<T, 8>::kCols;
    const long long tiles = ((long long)F + kCols - 1) / kCols;
    BB200_REQUIRE(tiles * kCols < (1LL << 31) && K <= (1 << 20) , BBCU_ERR_TOO_LARGE);
    const int columns = (int)(tiles * kCols);
    const long long want = 4LL * device_info().sm_count, per = (want + tiles - 1) / tiles;
    int rows = (int)(((C + per - 1) / per + 63) / 64 * 64);
    while ((C + rows - 1) / rows > 65535) rows *= 2;
    const int chunks = (C + rows - 1) / rows;
    const unsigned teacher_ctas = (unsigned)((F + kDistillThreads - 1) / kDistillThreads);
    const size_t part_b = (size_t)chunks * columns * sizeof(SoftSum), coef_b = (size_t)columns * 3 * 4, slot_b = (size_t)K * columns * 4;
    char *scratch = static_cast<char *>(stream_scratch(st, part_b + coef_b + 2 * slot_b + teacher_ctas * sizeof(double), kFrameOpSlot));
    BB200_REQUIRE(scratch != nullptr, BBCU_ERR_NO_MEMORY);
    SoftSum *part = reinterpret_cast<SoftSum *>(scratch);
    double *loss_part = reinterpret_cast<double *>(scratch + part_b);
    float *coef = reinterpret_cast<float *>(scratch + part_b + teacher_ctas * sizeof(double)), *slot_p = coef + 3 * (size_t)columns;
    int *slot_index = reinterpret_cast<int *>(slot_p + (size_t)K * columns);
    const float scale = kLog2e / temperature;
    const dim3 grid((unsigned)tiles, (unsigned)chunks);
    launch(aligned ? k_distill_stats<T, true> : k_distill_stats<T, false>, grid, kDistillThreads, 0, st, z, part, scale, C, F, zs, rows, columns);
    BB200_CUDA(cudaPeekAtLastError());
    launch(k_distill_teacher<T>, teacher_ctas, kDistillThreads, 0, st, z, t, index, t_lse, weight, part, coef, slot_index, slot_p, loss_buf, loss_part, temperature,
           grad_reduction, loss_reduction, C, K, F, zs, ts, is, chunks, columns);
    BB200_CUDA(cudaPeekAtLastError());
    launch(aligned ? k_distill_apply<T, true> : k_distill_apply<T, false>, grid, kDistillThreads, 0, st, z, dz, coef, slot_index, slot_p, loss_part,
           (int)teacher_ctas, loss, scale, C, K, F, zs, dzs, rows, columns);
    return launch_status();
}

template <typename T>
static int distillation_checked(const T *z, T *dz, const T *t, const int *index, const float *t_lse, const float *weight, float *loss_buf, float *loss,
                                float temperature, float grad_reduction, double loss_reduction, int C, int K, int F, int zs, int dzs, int ts, int is,
                                bbcu_stream_t stream)
{
    BB200_REQUIRE(C > 0 && K >= 0 && F >= 0 && temperature > 0.0f && temperature < INFINITY, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(C <= (1 << 24), BBCU_ERR_TOO_LARGE);
    BB200_REQUIRE(zs >= F && dzs >= F && (K == 0 || (ts >= F && is >= F)), BBCU_ERR_BAD_STRIDE);
    BB200_REQUIRE_PTR(loss);
    cudaStream_t st = as_stream(stream);
    if (F == 0) {
        BB200_CUDA(cudaMemsetAsync(loss, 0, sizeof(float), st));
        return BBCU_OK;
    }
    BB200_REQUIRE_PTR(z); BB200_REQUIRE_PTR(dz); BB200_REQUIRE_PTR(loss_buf);
    if (K > 0) { BB200_REQUIRE_PTR(t); BB200_REQUIRE_PTR(index); }
    return distillation<T>(z, dz, t, index, t_lse, weight, loss_buf, loss, temperature, grad_reduction, loss_reduction, C, K, F, zs, dzs, ts, is, st);
}

}   // namespace bb200

using namespace bb200;

extern "C" int bbcu_fp32_LossDistillation(const float *z, float *dz, const float *t, const int *index, const float *t_lse, const float *weight,
                                          float *loss_buf, float *loss, float temperature, float grad_reduction, double loss_reduction, int class_size,
                                          int top_size, int frame_size, int z_frame_stride, int dz_frame_stride, int t_frame_stride, int index_frame_stride,
                                          bbcu_stream_t stream)
{
    return distillation_checked<float>(z, dz, t, index, t_lse, weight, loss_buf, loss, temperature, grad_reduction, loss_reduction, class_size, top_size,
                                       frame_size, z_frame_stride, dz_frame_stride, t_frame_stride, index_frame_stride, stream);
}

extern "C" int bbcu_bf16_LossDistillation(const bbcu_bf16_t *z, bbcu_bf16_t *dz, const bbcu_bf16_t *t, const int *index, const float *t_lse,
                                          const float *weight, float *loss_buf, float *loss, float temperature, float grad_reduction, double loss_reduction,
                                          int class_size, int top_size, int frame_size, int z_frame_stride, int dz_frame_stride, int t_frame_stride,
                                          int index_frame_stride, bbcu_stream_t stream)
{
    return distillation_checked<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16 *>(z), reinterpret_cast<__nv_bfloat16 *>(dz),
                                               reinterpret_cast<const __nv_bfloat16 *>(t), index, t_lse, weight, loss_buf, loss, temperature, grad_reduction,
                                               loss_reduction, class_size, top_size, frame_size, z_frame_stride, dz_frame_stride, t_frame_stride,
                                               index_frame_stride, stream);
}
