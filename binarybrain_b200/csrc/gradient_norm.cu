// The global norm of many gradients, clipping by it, and Adam's step on gradients that are clipped on the way.  (The reference has no clipping; its Adam is
// cuda/OptimizerAdam.cu:12-48.)
//
//   norm = sqrt(sum over all tensors and elements g^2),   factor = max_norm / norm where that is below 1, else 1,   g <- factor g
//
// Squares are added up in 64 bits, so that neither large nor small gradients leave the range of the sum, in an order that the sizes alone decide.
//
// Memory bounds it: a gradient is read for the norm and again for what follows it.  The second kernel goes through the pieces of the tensors from the end, each by
// the CTA that had it before, since L2 still holds what has been read last, and marks everything else as read and written once.  (Clipped Adam of 6 x 65536 x 64: 126 us,
// from the end by other CTAs 129; the plain step 112, the norm alone 15.)
#include "adam.cuh"
#include "common.cuh"

namespace bb200 {

constexpr int kNormThreads = 512, kNormCtasPerSm = 2;

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

// The tensors in pieces of kPieceSize elements (kSmallPiece where three quarters of the CTAs would have none), numbered through for 512 tensors at a time; the CTAs take
// turns at them, from the first or, BACK, from the last one.  f(tensor, first element, count) is called by the whole CTA.  (Tensor by tensor, each over all
// threads, 200 tensors of 1000 took 250 us, now 8.  Pieces of 4096: 6 x 65536 x 64 130 us, of 8192 126; four small tensors then 7.8 and 9.5; numbered
// by all warps, in one size after the other, and their sizes asked for behind the norm, those took 7.6, now 6.2.)
constexpr int kPieceSize = 8192, kSmallPiece = 2048;
__host__ __device__ constexpr int pieces_of(int size, int piece) { return size > 0 ? (size - 1) / piece + 1 : 0; }
static_assert(pieces_of(0x7fffffff, kPieceSize) == 1 << 18 && pieces_of(0x7fffffff, kSmallPiece) == 1 << 20 && pieces_of(kPieceSize, kPieceSize) == 1 &&
              pieces_of(kPieceSize + 1, kPieceSize) == 2 && pieces_of(0, kPieceSize) == 0, "pieces of the largest and the smallest tensors");
// start[t + 1] = the pieces of the tensors up to t.  Only the warps that have a tensor number theirs.
__device__ __forceinline__ void number_pieces(int count, int size, int *start, int2 *warp_sum, int &piece)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int warps = (count + 31) / 32;
    const bool both = count <= (int)gridDim.x / 4;                        // too few pieces are possible
    int2 n;                                                               // by either size of pieces
    __syncthreads();                                                      // the numbers before are done with
    if (warp < warps) {
        n = make_int2(pieces_of(size, kPieceSize), pieces_of(size, kSmallPiece));
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int2 before = make_int2(__shfl_up_sync(0xffffffffu, n.x, d), both ? __shfl_up_sync(0xffffffffu, n.y, d) : 0);
            if (lane >= d) { n.x += before.x; n.y += before.y; }
        }
        if (lane == 31) warp_sum[warp] = n;
    }
    if (warps > 1) __syncthreads();
    else __syncwarp();
    if (warp < warps) {
        int whole = 0;
        for (int w = 0; w < (both ? warps : warp); ++w) {
            const int2 s = warp_sum[w];
            whole += s.x;
            if (w < warp) { n.x += s.x; n.y += s.y; }
        }
        const bool small = both && whole <= (int)gridDim.x / 4;
        start[threadIdx.x + 1] = small ? n.y : n.x;
        if (threadIdx.x == 0) {
            start[0] = 0;
            piece = small ? kSmallPiece : kPieceSize;
        }
    }
    __syncthreads();
}

template <bool BACK> __device__ __forceinline__ int first_size(int size, const int *__restrict__ size_table)
{
    const int t = (BACK ? (size - 1) / kNormThreads * kNormThreads : 0) + (int)threadIdx.x;
    return t < size ? size_table[t] : 0;
}
template <bool BACK, typename F> __device__ __forceinline__ void for_pieces(int size, const int *__restrict__ size_table, int size_here, F f)
{
    __shared__ int start[kNormThreads + 1], piece_size;
    __shared__ int2 warp_sum[kNormThreads / 32];
    const int tables = (size + kNormThreads - 1) / kNormThreads;
    for (int k = 0; k < tables; ++k) {
        const int t0 = (BACK ? tables - 1 - k : k) * kNormThreads, count = min(kNormThreads, size - t0);
        if (k > 0) size_here = (int)threadIdx.x < count ? size_table[t0 + threadIdx.x] : 0;
        number_pieces(count, size_here, start, warp_sum, piece_size);
        const int piece = piece_size;
        const int total = start[count], step = (int)gridDim.x;
        int t = 0;
        for (int c = BACK ? (total - 1 - (int)blockIdx.x) / step * step + (int)blockIdx.x : (int)blockIdx.x; c >= (int)blockIdx.x && c < total; c += BACK ? -step : step) {
            if (c < start[t] || c >= start[t + 1]) {                      // the last tensor that starts at or before the piece and is not empty
                int lo = 0, hi = count - 1;
                while (lo < hi) {
                    const int mid = (lo + hi + 1) / 2;
                    if (start[mid] <= c) lo = mid; else hi = mid - 1;
                }
                t = lo;
            }
            const int first = (c - start[t]) * piece;
            f(t0 + t, first, min(piece, size_table[t0 + t] - first));
        }
    }
}

// part[CTA] = the sum of the squares of its pieces
__global__ void __launch_bounds__(kNormThreads, kNormCtasPerSm)
k_gradient_squares(int size, const int *__restrict__ size_table, float *const *__restrict__ grads, double *part)
{
    grid_dependency();
    __shared__ double red[kNormThreads / 32];
    double sum = 0.0;
    auto add = [&](float g) { sum = fma((double)g, (double)g, sum); };
    for_pieces<false>(size, size_table, first_size<false>(size, size_table), [&](int t, int first, int count) {
        const float *g = grads[t] + first;
        const int quads = (reinterpret_cast<uintptr_t>(g) & 15) == 0 ? count / 4 : 0;
        float4 q[kPieceSize / 4 / kNormThreads];
#pragma unroll
        for (int i = 0; i < kPieceSize / 4 / kNormThreads; ++i) {
            const int k = threadIdx.x + i * kNormThreads;
            q[i] = k < quads ? reinterpret_cast<const float4 *>(g)[k] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int i = 0; i < kPieceSize / 4 / kNormThreads; ++i) { add(q[i].x); add(q[i].y); add(q[i].z); add(q[i].w); }
#pragma unroll 4
        for (int i = 4 * quads + threadIdx.x; i < count; i += kNormThreads) add(g[i]);
    });
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
    const int size_here = first_size<true>(size, size_table);             // on its way beside the parts
    const double norm = norm_of(part, parts);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const float factor = clip_factor(norm, max_norm);
    if (factor == 1.0f) return;                                           // nothing changes
    for_pieces<true>(size, size_table, size_here, [&](int t, int first, int count) {
        float *g = grads[t] + first;
        const int quads = (reinterpret_cast<uintptr_t>(g) & 15) == 0 ? count / 4 : 0;
#pragma unroll 2
        for (int i = threadIdx.x; i < quads; i += kNormThreads) {
            float4 q = reinterpret_cast<float4 *>(g)[i];
            q.x *= factor; q.y *= factor; q.z *= factor; q.w *= factor;
            __stcs(reinterpret_cast<float4 *>(g) + i, q);
        }
        for (int i = 4 * quads + threadIdx.x; i < count; i += kNormThreads) g[i] *= factor;
    });
}

template <bool CLEAR>
__global__ void __launch_bounds__(kNormThreads, kNormCtasPerSm)
k_adam_clipped(int size, const int *__restrict__ size_table, float *const *__restrict__ params, float *const *__restrict__ grads, float *const *__restrict__ m_tab,
               float *const *__restrict__ v_tab, float lr_t, float beta1, float beta2, const double *part, int parts, float max_norm, float *norm_out)
{
    grid_dependency();
    const int size_here = first_size<true>(size, size_table);             // on its way beside the parts
    const double norm = norm_of(part, parts);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const float factor = clip_factor(norm, max_norm);
    for_pieces<true>(size, size_table, size_here, [&](int t, int first, int count) {
        float *p = params[t] + first, *m = m_tab[t] + first, *v = v_tab[t] + first, *g = grads[t] + first;
        const bool vec = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(g)) & 15) == 0;
        const int quads = vec ? count / 4 : 0;
#pragma unroll 2
        for (int i = threadIdx.x; i < quads; i += kNormThreads) {
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
        for (int i = 4 * quads + threadIdx.x; i < count; i += kNormThreads) {
            float pi = p[i], mi = m[i], vi = v[i];
            adam_step(pi, g[i] * factor, mi, vi, lr_t, beta1, beta2);
            p[i] = pi;
            m[i] = mi;
            v[i] = vi;
            if (CLEAR) g[i] = 0.0f;
        }
    });
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
