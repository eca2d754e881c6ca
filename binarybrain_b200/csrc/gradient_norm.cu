// The global norm of many gradients, clipping by it, and Adam's step on gradients that are clipped on the way.  (The reference has no clipping; its Adam is
// cuda/OptimizerAdam.cu:12-48.)
//
//   norm = sqrt(sum over all tensors and elements g^2),   factor = max_norm / norm where that is below 1, else 1,   g <- factor g
//
// Squares are added up in 64 bits, so that neither large nor small gradients leave the range of the sum, in an order that the sizes alone decide.
//
// Memory bounds it: a gradient is read for the norm and again for what follows it.  The second kernel goes through the tensors and their elements from the
// end, where L2 still holds what the first one has read last, and marks everything else as read and written once.
#include "adam.cuh"
#include "common.cuh"

namespace bb200 {

constexpr int kNormThreads = 512, kNormCtasPerSm = 2, kNormBatch = 4;

__device__ __forceinline__ double block_total(double v, double *smem)      // in every thread
{
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
    __syncthreads();
    v = smem[threadIdx.x & (kNormThreads / 32 - 1)];
#pragma unroll
    for (int m = kNormThreads / 64; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// part[CTA] = the sum of the squares of its pieces of all tensors
__global__ void __launch_bounds__(kNormThreads, kNormCtasPerSm)
k_gradient_squares(int size, const int *__restrict__ size_table, float *const *__restrict__ grads, double *part)
{
    grid_dependency();
    __shared__ double red[kNormThreads / 32];
    const int threads = gridDim.x * kNormThreads, id = blockIdx.x * kNormThreads + threadIdx.x;
    double sum = 0.0;
    auto add = [&](float g) { sum = fma((double)g, (double)g, sum); };
    for (int t = 0; t < size; ++t) {
        const float *g = grads[t];
        const int n = size_table[t], quads = (reinterpret_cast<uintptr_t>(g) & 15) == 0 ? n / 4 : 0;
        for (long long i = id; i < quads; i += (long long)kNormBatch * threads) {
            float4 q[kNormBatch];
#pragma unroll
            for (int b = 0; b < kNormBatch; ++b) q[b] = i + (long long)b * threads < quads ? reinterpret_cast<const float4 *>(g)[i + (long long)b * threads] : make_float4(0, 0, 0, 0);
#pragma unroll
            for (int b = 0; b < kNormBatch; ++b) { add(q[b].x); add(q[b].y); add(q[b].z); add(q[b].w); }
        }
        for (long long i = 4LL * quads + id; i < n; i += threads) add(g[i]);
    }
    sum = block_total(sum, red);
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

// the norm from the parts, in every thread of every CTA alike
__device__ __forceinline__ double norm_of(const double *part, int parts)
{
    __shared__ double red[kNormThreads / 32];
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += kNormThreads) sum += part[i];
    return sqrt(block_total(sum, red));
}

__device__ __forceinline__ float clip_factor(double norm, float max_norm) { return norm > (double)max_norm ? (float)((double)max_norm / norm) : 1.0f; }

__global__ void __launch_bounds__(kNormThreads) k_gradient_norm(const double *part, int parts, float *norm_out)
{
    grid_dependency();
    const double norm = norm_of(part, parts);
    if (threadIdx.x == 0) *norm_out = (float)norm;
}

__global__ void __launch_bounds__(kNormThreads, kNormCtasPerSm)
k_gradient_clip(int size, const int *__restrict__ size_table, float *const *__restrict__ grads, const double *part, int parts, float max_norm, float *norm_out)
{
    grid_dependency();
    const double norm = norm_of(part, parts);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const float factor = clip_factor(norm, max_norm);
    if (factor == 1.0f) return;                                           // nothing changes
    const int threads = gridDim.x * kNormThreads, id = blockIdx.x * kNormThreads + threadIdx.x;
    for (int t = size - 1; t >= 0; --t) {
        float *g = grads[t];
        const int n = size_table[t], quads = (reinterpret_cast<uintptr_t>(g) & 15) == 0 ? n / 4 : 0;
        for (long long k = id; k < quads; k += threads) {
            float4 *at = reinterpret_cast<float4 *>(g) + (quads - 1 - k);
            float4 q = *at;
            q.x *= factor; q.y *= factor; q.z *= factor; q.w *= factor;
            __stcs(at, q);
        }
        for (long long i = 4LL * quads + id; i < n; i += threads) g[i] *= factor;
    }
}

template <bool CLEAR>
__global__ void __launch_bounds__(kNormThreads, kNormCtasPerSm)
k_adam_clipped(int size, const int *__restrict__ size_table, float *const *__restrict__ params, float *const *__restrict__ grads, float *const *__restrict__ m_tab,
               float *const *__restrict__ v_tab, float lr_t, float beta1, float beta2, const double *part, int parts, float max_norm, float *norm_out)
{
    grid_dependency();
    const double norm = norm_of(part, parts);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const float factor = clip_factor(norm, max_norm);
    const int threads = gridDim.x * kNormThreads, id = blockIdx.x * kNormThreads + threadIdx.x;
    for (int t = size - 1; t >= 0; --t) {
        float *p = params[t], *m = m_tab[t], *v = v_tab[t], *g = grads[t];
        const int n = size_table[t];
        const bool vec = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(g)) & 15) == 0;
        const int quads = vec ? n / 4 : 0;
        for (long long k = id; k < quads; k += threads) {
            const long long i = quads - 1 - k;
            float4 gq = reinterpret_cast<float4 *>(g)[i], pq = __ldcs(reinterpret_cast<float4 *>(p) + i), mq = __ldcs(reinterpret_cast<float4 *>(m) + i),
                   vq = __ldcs(reinterpret_cast<float4 *>(v) + i);
            adam_step(pq.x, gq.x * factor, mq.x, vq.x, lr_t, beta1, beta2);
            adam_step(pq.y, gq.y * factor, mq.y, vq.y, lr_t, beta1, beta2);
            adam_step(pq.z, gq.z * factor, mq.z, vq.z, lr_t, beta1, beta2);
            adam_step(pq.w, gq.w * factor, mq.w, vq.w, lr_t, beta1, beta2);
            __stcs(reinterpret_cast<float4 *>(p) + i, pq);
            __stcs(reinterpret_cast<float4 *>(m) + i, mq);
            __stcs(reinterpret_cast<float4 *>(v) + i, vq);
            if (CLEAR) __stcs(reinterpret_cast<float4 *>(g) + i, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        }
        for (long long i = 4LL * quads + id; i < n; i += threads) {
            float pi = p[i], mi = m[i], vi = v[i];
            adam_step(pi, g[i] * factor, mi, vi, lr_t, beta1, beta2);
            p[i] = pi;
            m[i] = mi;
            v[i] = vi;
            if (CLEAR) g[i] = 0.0f;
        }
    }
}

// the squares of all gradients as `parts` partial sums; null with a status set where there is no scratch
static double *gradient_squares(int size, const int *size_table, float *const *grads, HeldScratch &held, int &parts, cudaStream_t st)
{
    parts = device_info().sm_count * kNormCtasPerSm;
    double *part = static_cast<double *>(held.get(st, (size_t)parts * sizeof(double)));
    if (part) launch(k_gradient_squares, (unsigned)parts, kNormThreads, 0, st, size, size_table, grads, part);
    return part;
}

}   // namespace bb200

using namespace bb200;

extern "C" int bbcu_fp32_GradientNorm(int size, const int *size_table, float *const *grads, float *norm, bbcu_stream_t stream)
{
    BB200_REQUIRE(size >= 0, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE_PTR(norm);
    if (size > 0) { BB200_REQUIRE_PTR(size_table); BB200_REQUIRE_PTR(grads); }
    cudaStream_t st = as_stream(stream);
    HeldScratch held;
    int parts;
    const double *part = gradient_squares(size, size_table, grads, held, parts, st);
    BB200_REQUIRE(part != nullptr, BBCU_ERR_NO_MEMORY);
    launch(k_gradient_norm, 1, kNormThreads, 0, st, part, parts, norm);
    return launch_status();
}

extern "C" int bbcu_fp32_GradientClip(int size, const int *size_table, float *const *grads, float max_norm, float *norm, bbcu_stream_t stream)
{
    BB200_REQUIRE(size >= 0 && max_norm >= 0.0f, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE_PTR(norm);
    if (size > 0) { BB200_REQUIRE_PTR(size_table); BB200_REQUIRE_PTR(grads); }
    cudaStream_t st = as_stream(stream);
    HeldScratch held;
    int parts;
    const double *part = gradient_squares(size, size_table, grads, held, parts, st);
    BB200_REQUIRE(part != nullptr, BBCU_ERR_NO_MEMORY);
    launch(k_gradient_clip, (unsigned)parts, kNormThreads, 0, st, size, size_table, grads, part, parts, max_norm, norm);
    return launch_status();
}

extern "C" int bbcu_fp32_OptimizerAdamClipped(int size, const int *size_table, float *const *params, float *const *grads, float *const *m_tab, float *const *v_tab,
                                              float lr_t, float beta1, float beta2, float max_norm, float *norm, int clear_grads, bbcu_stream_t stream)
{
    BB200_REQUIRE(size >= 0 && max_norm >= 0.0f, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE_PTR(norm);
    if (size > 0) { BB200_REQUIRE_PTR(size_table); BB200_REQUIRE_PTR(params); BB200_REQUIRE_PTR(grads); BB200_REQUIRE_PTR(m_tab); BB200_REQUIRE_PTR(v_tab); }
    cudaStream_t st = as_stream(stream);
    HeldScratch held;
    int parts;
    const double *part = gradient_squares(size, size_table, grads, held, parts, st);
    BB200_REQUIRE(part != nullptr, BBCU_ERR_NO_MEMORY);
    launch(clear_grads ? k_adam_clipped<true> : k_adam_clipped<false>, (unsigned)parts, kNormThreads, 0, st, size, size_table, params, grads, m_tab, v_tab, lr_t, beta1,
           beta2, part, parts, max_norm, norm);
    return launch_status();
}
