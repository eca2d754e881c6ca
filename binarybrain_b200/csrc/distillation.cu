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
// without a slot, or of weight 0, has loss 0 and gradient 0 whatever its logits are.
// exp(z / T) is evaluated as exp2((z - max z) log2(e) / T), and by expf() in the sums of up to kFewClasses classes: there a small loss comes out of large
// terms, times T^2, and the teacher's sums, which are expf()'s, have the same errors.
#include <type_traits>

#include "frame_columns.cuh"

namespace bb200 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kFewClasses = 256;                         // (10 classes, T = 4: the mean loss is off by 5e-7 of it with exp2, by 2e-7 with expf)
constexpr int kMostSlots = 512;                          // of the teacher, a column of them in shared memory
constexpr int kDistillRows = 16, kDistillCluster = 4;    // rows a thread and CTAs a cluster where everything is read once, at most

template <typename T> struct Distill {
    const T *z, *t;
    T *dz;
    const int *index;
    const float *t_lse, *weight;
    float *loss_buf;
    double *loss_part;                                   // [column tile]
    float temperature, inv_t, scale, grad_reduction;     // scale = log2(e) / T
    int C, K, F;
    long long zs, dzs, ts, is;
};

// 2^x to 2^-22 of it, 0 below the normal numbers
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// maximum and sum of exponentials relative to it, of two sets joined; an empty set, and one of -inf alone, is (-inf, 0)
struct SoftSum { float top, sum; };
__device__ __forceinline__ SoftSum join_soft(const SoftSum &a, const SoftSum &b, float scale)
{
    const float top = fmaxf(a.top, b.top);
    if (top == -INFINITY) return {top, a.sum + b.sum};                    // (a NaN among them stays)
    return {top, a.sum * exp2_fast((a.top - top) * scale) + b.sum * exp2_fast((b.top - top) * scale)};
}
// what exponents are taken relative to: with no class left, anything finite
__device__ __forceinline__ float reference(float top) { return top == -INFINITY ? 0.0f : top; }

// How a frame's softmax becomes its gradient: dz = factor * min(exp2((z - top) scale), cap), minus `slope` times the teacher's probability where the
// class is named.  A frame that takes no part has factor, cap and slope 0, and min() gives the cap for a NaN; elsewhere the cap is infinite, and a NaN
// among the logits has made the factor one.
struct FrameGrad { float top, factor, cap, slope; };
__device__ __forceinline__ float soft_part(const FrameGrad &g, float z, float scale) { return g.factor * fminf(exp2_fast((z - g.top) * scale), g.cap); }

// the larger of each pair of 16 bytes of logits, a NaN being the smaller
template <typename T> __device__ __forceinline__ uint4 packed_max(const uint4 &a, const uint4 &b);
template <> __device__ __forceinline__ uint4 packed_max<float>(const uint4 &a, const uint4 &b)
{
    return make_uint4(__float_as_uint(fmaxf(__uint_as_float(a.x), __uint_as_float(b.x))), __float_as_uint(fmaxf(__uint_as_float(a.y), __uint_as_float(b.y))),
                      __float_as_uint(fmaxf(__uint_as_float(a.z), __uint_as_float(b.z))), __float_as_uint(fmaxf(__uint_as_float(a.w), __uint_as_float(b.w))));
}
template <> __device__ __forceinline__ uint4 packed_max<__nv_bfloat16>(const uint4 &a, const uint4 &b)
{
    uint4 r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r.x) : "r"(a.x), "r"(b.x));
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r.y) : "r"(a.y), "r"(b.y));
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r.z) : "r"(a.z), "r"(b.z));
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r.w) : "r"(a.w), "r"(b.w));
    return r;
}

// ---- the teacher's side of COLS frames from f0 on, by a CTA of a multiple of COLS threads: thread t has column t % COLS and every (threads / COLS)-th
// slot of it.  index[slot][column] (-1: empty) and log_p[slot][column] (-inf: p = 0) go to shared memory, and to each thread, for its column, P = sum p and the
// weight (0: the frame takes no part).  A barrier stands behind the last write of the two; red[0] may still be read.
struct TeacherColumn { float P, weight; };

// a value of each column joined over the lanes of a warp that have it
template <int COLS, typename JOIN> __device__ __forceinline__ float column_of_warp(float v, JOIN join)
{
#pragma unroll
    for (int m = COLS; m < 32; m <<= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}

template <typename T, int COLS>
__device__ __forceinline__ TeacherColumn teacher_columns(const Distill<T> &a, int f0, int *index, float *log_p, float (&red)[3][kColumnThreads / 32 * COLS])
{
    const int col = threadIdx.x % COLS, group = threadIdx.x / COLS, groups = blockDim.x / COLS, f = f0 + col;
    const float w = f < a.F ? (a.weight ? a.weight[f] : 1.0f) : 0.0f;
    float top = -INFINITY, slots = 0.0f;
    for (int k = group; k < a.K; k += groups) {
        int i = -1;
        float t = -INFINITY;
        if (f < a.F) {
            i = a.index[k * a.is + f];
            t = to_float(a.t[k * a.ts + f]);
            if (i < 0 || i >= a.C || t == -INFINITY) i = -1;
        }
        index[k * COLS + col] = i;
        log_p[k * COLS + col] = t;
        if (i >= 0) { top = fmaxf(top, t); slots += 1.0f; }
    }
    const int warps = blockDim.x / 32, own = threadIdx.x / 32 * COLS + threadIdx.x % 32;
    top = column_of_warp<COLS>(top, [](float a, float b) { return fmaxf(a, b); });
    slots = column_of_warp<COLS>(slots, [](float a, float b) { return a + b; });
    if (threadIdx.x % 32 < COLS) {
        red[0][own] = top;
        red[1][own] = slots;
    }
    __syncthreads();
    top = join_parts<ColumnMax>(&red[0][col], COLS, warps);
    slots = join_parts<ColumnSum>(&red[1][col], COLS, warps);
    const bool live = slots > 0.0f && w != 0.0f;
    // log p = (t - base) / T - lse: with the slots' own sum the level of the logits leaves before anything is rounded
    float lse = 0.0f, base = 0.0f;
    if (a.t_lse) {
        if (live) lse = a.t_lse[f];
        __syncthreads();                                                  // (the two sums are read before the next two take their place)
    } else {
        float sum = 0.0f;
        for (int k = group; k < a.K; k += groups)
            if (index[k * COLS + col] >= 0) sum += expf((log_p[k * COLS + col] - top) * a.inv_t);
        sum = column_of_warp<COLS>(sum, [](float a, float b) { return a + b; });
        if (threadIdx.x % 32 < COLS) red[2][own] = sum;
        __syncthreads();
        sum = join_parts<ColumnSum>(&red[2][col], COLS, warps);
        lse = logf(sum);
        base = top;
    }
    float P = 0.0f;
    for (int k = group; k < a.K; k += groups) {
        float lp = -INFINITY;
        if (live && index[k * COLS + col] >= 0) {
            lp = (log_p[k * COLS + col] - base) * a.inv_t - lse;
            P += expf(lp);
        }
        log_p[k * COLS + col] = lp;
    }
    P = column_of_warp<COLS>(P, [](float a, float b) { return a + b; });
    if (threadIdx.x % 32 < COLS) red[0][own] = P;
    __syncthreads();
    return {join_parts<ColumnSum>(&red[0][col], COLS, warps), live ? w : 0.0f};
}

// The probabilities of all slots of the column that name the class of slot k, in the order of the slots; `first`: k is the first of them.
template <int COLS> __device__ __forceinline__ float named_slots(const int *index, const float *log_p, int K, int k, int col, bool &first)
{
    const int i = index[k * COLS + col];
    float sum = 0.0f;
    first = true;
    for (int e = 0; e < K; ++e)
        if (index[e * COLS + col] == i) {
            first = first && e >= k;
            sum += expf(log_p[e * COLS + col]);
        }
    return sum;
}

// From a frame's joined sums its gradient's factors.  No class left: q = 0.
template <typename T> __device__ __forceinline__ FrameGrad finish_frame(const Distill<T> &a, float P, float weight, const SoftSum &s)
{
    if (weight == 0.0f) return {0.0f, 0.0f, 0.0f, 0.0f};
    const float slope = a.grad_reduction * weight * a.temperature;
    return {reference(s.top), s.top == -INFINITY && s.sum == 0.0f ? 0.0f : slope * P / s.sum, INFINITY, slope};
}

// loss_buf of the first warp's columns, and their sum
template <typename T> __device__ __forceinline__ void write_losses(const Distill<T> &a, int tile, int f, bool has, float loss)
{
    if (has) a.loss_buf[f] = loss;
    double sum = has ? (double)loss : 0.0;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    if (threadIdx.x == 0) a.loss_part[tile] = sum;
}

// ---- everything read once, as far as a cluster holds the classes of a column tile in shared memory (see layer_norm.cu for the walk over the tiles).  Each
// CTA reduces its classes to four numbers a frame, relative to its own largest logit m: m, sum exp((z - m) / T), and sum p (log p - (z - m) / T) and sum p over
// the slots that name one of its classes; one exchange joins them.
template <typename T, int LPR>
__global__ void __launch_bounds__(kColumnThreads, 3)
k_distill_once(const Distill<T> a, int rows, int tiles, int *fault)
{
    grid_dependency();
    using Col = Column<T, LPR>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    static_assert(kCols <= 32, "a warp finishes the columns");
    extern __shared__ __align__(16) uint8_t buffer[];
    __shared__ float red[3][kColumnThreads / 32 * kCols], red_soft[kColumnThreads / 32][kCols], s_top[kCols], s_log_sum[kCols];
    __shared__ FrameGrad s_grad[kCols];
    __shared__ uint64_t bar[2];
    __shared__ int gave_up;
    const Col c;
    const uint32_t cl = cluster_size(), rank = cluster_rank();
    const int clusters = (int)(gridDim.x / cl), cta_first = (int)rank * c.step * rows, first = cta_first + c.row, piece = blockDim.x * 16;
    const int mine = min(rows, (a.C - first + c.step - 1) / c.step), cta_rows = min(c.step * rows, a.C - cta_first);
    const uint8_t *const at = buffer + threadIdx.x * 16;
    const int shift = 31 - __clz(c.step);                                 // the warps are a power of two
    int *const index = reinterpret_cast<int *>(buffer + rows * piece);
    float *const log_p = reinterpret_cast<float *>(index + a.K * kCols);
    unsigned *const seen = reinterpret_cast<unsigned *>(log_p + a.K * kCols);   // a bit for each of the CTA's classes and columns: has a slot named it?
    const int seen_words = (c.step * rows + 31) / 32 * kCols;
    float (*const part)[4][kCols] = reinterpret_cast<float (*)[4][kCols]>(seen + seen_words);      // [two exchanges of the cluster's CTAs]
    for (int i = threadIdx.x; i < seen_words; i += blockDim.x) seen[i] = 0u;
    const long long z_step = c.step * a.zs, dz_step = c.step * a.dzs;
    const T *const z_first = a.z + first * a.zs;
    // the logit of a class of this CTA in a column of the tile
    auto logit = [&](int i, int col) {
        const int local = i - cta_first, in = local & (c.step - 1);
        return to_float(reinterpret_cast<const T *>(buffer + (local >> shift) * piece + (in * LPR + col / kVec) * 16)[col % kVec]);
    };
    auto fetch = [&](int f) {
        if (f >= a.F) return;
        uint8_t *to = buffer + threadIdx.x * 16;
        const T *from = z_first + f;
#pragma unroll 4
        for (int i = 0; i < mine; ++i, to += piece, from += z_step) cp_async16(to, from, true);
    };
    int tile = (int)(blockIdx.x / cl), f = tile * kCols + c.col;
    fetch(f);
    if (cl > 1) {
        if (threadIdx.x == 0) {
            gave_up = 0;
            mbar_init(&bar[0], 1);
            mbar_init(&bar[1], 1);
            mbar_init_fence();
        }
        cluster_arrive();
        cluster_wait();
    }
    const int my_col = threadIdx.x % kCols, group = threadIdx.x / kCols, groups = blockDim.x / kCols;
    const bool few = a.C <= kFewClasses;
    for (uint32_t turn = 0; tile < tiles; tile += clusters, f += clusters * kCols, ++turn) {
        cp_async_commit();
        const TeacherColumn teacher = teacher_columns<T, kCols>(a, tile * kCols, index, log_p, red);
        cp_async_wait<0>();
        float v[kVec], m[kVec], sum[kVec] = {};
#pragma unroll
        for (int j = 0; j < kVec; ++j) m[j] = -INFINITY;
        {
            const uint8_t *q = at;
#pragma unroll 4
            for (int i = 0; i < mine; ++i, q += piece) {
                unpack<T>(*reinterpret_cast<const uint4 *>(q), v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) m[j] = fmaxf(m[j], v[j]);
            }
        }
#pragma unroll
        for (int d = LPR; d < 32; d <<= 1)
#pragma unroll
            for (int j = 0; j < kVec; ++j) m[j] = fmaxf(m[j], __shfl_xor_sync(0xffffffffu, m[j], d));
        if (c.lane < LPR) {
#pragma unroll
            for (int j = 0; j < kVec; ++j) red_soft[c.warp][c.col + j] = m[j];
        }
        __syncthreads();                                                  // (the logits of the other threads are there, too)
        if (threadIdx.x < kCols) {
            s_top[threadIdx.x] = join_parts<ColumnMax>(&red_soft[0][threadIdx.x], kCols, c.warps);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kVec; ++j) m[j] = reference(s_top[c.col + j]);
        {
            const uint8_t *q = at;
#pragma unroll 4
            for (int i = 0; i < mine; ++i, q += piece) {
                unpack<T>(*reinterpret_cast<const uint4 *>(q), v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) sum[j] += few ? expf((v[j] - m[j]) * a.inv_t) : exp2_fast((v[j] - m[j]) * a.scale);
            }
        }
#pragma unroll
        for (int d = LPR; d < 32; d <<= 1)
#pragma unroll
            for (int j = 0; j < kVec; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], d);
        if (c.lane < LPR) {
#pragma unroll
            for (int j = 0; j < kVec; ++j) red_soft[c.warp][c.col + j] = sum[j];
        }
        const float own_top = reference(s_top[my_col]);
        float spread = 0.0f, own_p = 0.0f;
        int twice = 0;
        for (int k = group; k < a.K; k += groups) {
            const int i = index[k * kCols + my_col], local = i - cta_first;
            if (local >= 0 && local < cta_rows) {
                const unsigned bit = 1u << (local & 31);
                twice |= (int)(atomicOr(&seen[(local >> 5) * kCols + my_col], bit) & bit);
                if (cl > 1) {
                    const float lp = log_p[k * kCols + my_col], p = expf(lp);
                    if (p != 0.0f) {
                        spread += p * (lp - (logit(i, my_col) - own_top) * a.inv_t);
                        own_p += p;
                    }
                }
            }
        }
        if (cl > 1) {
            spread = column_of_warp<kCols>(spread, [](float a, float b) { return a + b; });
            own_p = column_of_warp<kCols>(own_p, [](float a, float b) { return a + b; });
            if (c.lane < kCols) {
                red[0][c.warp * kCols + c.lane] = spread;
                red[1][c.warp * kCols + c.lane] = own_p;
            }
            if (threadIdx.x == 0) mbar_arrive_expect_tx(&bar[turn & 1], cl * 4 * kCols * (uint32_t)sizeof(float));
        }
        twice = __syncthreads_or(twice);
        if (threadIdx.x < kCols) {                                        // all of them in the first warp
            SoftSum joined = {s_top[threadIdx.x], join_parts<ColumnSum>(&red_soft[0][threadIdx.x], kCols, c.warps)};
            if (cl > 1) {
                spread = join_parts<ColumnSum>(&red[0][threadIdx.x], kCols, c.warps);
                own_p = join_parts<ColumnSum>(&red[1][threadIdx.x], kCols, c.warps);
                float (*const from)[4][kCols] = part + (turn & 1) * cl, (*const to)[kCols] = from[rank];
                for (uint32_t r = 0; r < cl; ++r) {
                    const uint32_t b = peer_addr(&bar[turn & 1], r);
                    peer_send(peer_addr(&to[0][threadIdx.x], r), joined.top, b);
                    peer_send(peer_addr(&to[1][threadIdx.x], r), joined.sum, b);
                    peer_send(peer_addr(&to[2][threadIdx.x], r), spread, b);
                    peer_send(peer_addr(&to[3][threadIdx.x], r), own_p, b);
                }
                bool ok = *(volatile int *)&gave_up == 0;
                for (int i = 0; i < kWaitSpins && ok; ++i) {
                    if (mbar_try_wait(&bar[turn & 1], turn >> 1 & 1)) break;
                    if (i == kWaitSpins - 1) { *(volatile int *)&gave_up = 1; ok = false; }
                }
                joined = {from[0][0][threadIdx.x], from[0][1][threadIdx.x]};
                for (uint32_t r = 1; r < cl; ++r) joined = join_soft(joined, {from[r][0][threadIdx.x], from[r][1][threadIdx.x]}, a.scale);
                spread = 0.0f;
                for (uint32_t r = 0; r < cl; ++r) {
                    const float p = from[r][3][threadIdx.x];
                    spread += from[r][2][threadIdx.x];
                    if (p != 0.0f) spread -= p * ((reference(from[r][0][threadIdx.x]) - reference(joined.top)) * a.inv_t);
                }
            }
            s_grad[threadIdx.x] = finish_frame(a, teacher.P, teacher.weight, joined);
            const float log_sum = joined.sum == 0.0f ? 0.0f : logf(joined.sum);     // (no class left: the spread is infinite, as the loss is)
            s_log_sum[threadIdx.x] = log_sum;
            red[0][threadIdx.x] = teacher.weight == 0.0f ? 0.0f : teacher.weight * a.temperature * a.temperature * (spread + teacher.P * log_sum);
        }
        __syncthreads();
        if (cl > 1 && rank == 0 && c.warp == 0)
            write_losses(a, tile, tile * kCols + c.lane, c.lane < kCols && tile * kCols + c.lane < a.F, c.lane < kCols ? red[0][c.lane] : 0.0f);
        if (f < a.F) {
            FrameGrad g[kVec];
#pragma unroll
            for (int j = 0; j < kVec; ++j) g[j] = s_grad[c.col + j];
            const uint8_t *q = at;
            T *out = a.dz + first * a.dzs;
#pragma unroll 4
            for (int i = 0; i < mine; ++i, q += piece, out += dz_step) {
                unpack<T>(*reinterpret_cast<const uint4 *>(q), v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) v[j] = soft_part(g[j], v[j], a.scale);
                store_frames<T, true>(out, f, a.F, v);
            }
        }
        __syncthreads();                                                  // the CTA's values of dz stand before those of the named classes are written again
        float divergence = 0.0f;                                          // of a CTA by itself: term by term, which keeps the digits of a small one
        if (tile * kCols + my_col < a.F) {
            const FrameGrad g = s_grad[my_col];
            const float log_sum = s_log_sum[my_col];
            for (int k = group; k < a.K; k += groups) {
                const int i = index[k * kCols + my_col], local = i - cta_first;
                if (local < 0 || local >= cta_rows) continue;
                seen[(local >> 5) * kCols + my_col] = 0u;
                bool leads = true;
                const float lp = log_p[k * kCols + my_col], p = expf(lp);
                if (cl == 1 && p != 0.0f) divergence += p * (lp - ((logit(i, my_col) - g.top) * a.inv_t - log_sum));
                const float q = twice ? named_slots<kCols>(index, log_p, a.K, k, my_col, leads) : p;
                if (leads) a.dz[i * a.dzs + tile * kCols + my_col] = from_float<T>(soft_part(g, logit(i, my_col), a.scale) - g.slope * q);
            }
        }
        if (cl == 1) {
            divergence = column_of_warp<kCols>(divergence, [](float a, float b) { return a + b; });
            if (c.lane < kCols) red[2][c.warp * kCols + c.lane] = divergence;
        }
        __syncthreads();                                                  // nobody needs the logits and the slots any more
        fetch(f + clusters * kCols);
        if (cl == 1 && c.warp == 0) {                                     // (red[2] is written again behind a barrier of this warp)
            const bool has = c.lane < kCols && tile * kCols + c.lane < a.F;
            write_losses(a, tile, tile * kCols + c.lane, has,
                         has && teacher.weight != 0.0f ? teacher.weight * a.temperature * a.temperature * join_parts<ColumnSum>(&red[2][c.lane], kCols, c.warps) : 0.0f);
        }
    }
    if (cl > 1) {
        if (threadIdx.x == 0 && gave_up) atomicCAS(fault, 0, kFaultBarrierTimeout);
        __syncwarp();
        cluster_arrive();                                                 // nobody leaves while something may still be sent to it
        cluster_wait();
    }
}

// ---- more classes than that: the teacher's side beside the softmax's sums, what follows from both for a frame, dz of all classes, dz of the named ones.
// The teacher's CTAs have eight frames, 32 threads for each, and leave P and weight as teacher[2][columns], and of every slot its class i (~1 - i where an
// earlier slot names it, too, and -1 where the slot is empty), log p, and the probabilities of its class added up.
struct Slots { int *index; float *log_p, *p; };
constexpr int kFinishCols = 8, kFinishGroups = kColumnThreads / kFinishCols;

// Does a frame name a class twice?  Its slots mark a bit each of 2^slot_hash_bits(K), some 32 to 64 for a slot, and one that finds its bit marked looks
// through all of them; only a frame where that finds a class twice adds up all of its slots by K searches.  (500 slots of 6000 classes x 3000 frames
// bf16, with the searches for every frame: 343 us a call.)
__host__ __device__ inline int slot_hash_bits(int K)
{
    int bits = 5;
    while (bits < 14 && (1 << bits) < 32 * K) ++bits;
    return bits;
}
template <typename T>
__device__ __forceinline__ void teacher_slots(const Distill<T> &a, int cta, float *teacher, const Slots &slots, int columns)
{
    extern __shared__ __align__(16) uint8_t buffer[];
    __shared__ float red[3][kColumnThreads / 32 * kFinishCols];
    __shared__ int twice[kFinishCols];
    int *const index = reinterpret_cast<int *>(buffer);
    float *const log_p = reinterpret_cast<float *>(index + a.K * kFinishCols);
    const int col = threadIdx.x % kFinishCols, group = threadIdx.x / kFinishCols, f = cta * kFinishCols + col;
    unsigned *const hit = reinterpret_cast<unsigned *>(log_p + a.K * kFinishCols);
    const int hit_bits = slot_hash_bits(a.K);
    for (int i = threadIdx.x; i < (kFinishCols << hit_bits) / 32; i += kColumnThreads) hit[i] = 0u;
    if (threadIdx.x < kFinishCols) twice[threadIdx.x] = 0;
    const TeacherColumn c = teacher_columns<T, kFinishCols>(a, cta * kFinishCols, index, log_p, red);
    for (int k = group; k < a.K; k += kFinishGroups) {
        const int i = index[k * kFinishCols + col];
        if (i < 0) continue;
        const unsigned h = (unsigned)i * 2654435769u >> (32 - hit_bits), bit = 1u << (h & 31);
        if (atomicOr(&hit[(h >> 5) * kFinishCols + col], bit) & bit) {
            int named = 0;
            for (int e = 0; e < a.K; ++e) named += index[e * kFinishCols + col] == i;
            if (named > 1) twice[col] = 1;
        }
    }
    __syncthreads();
    const bool search = twice[col] != 0;
    for (int k = group; k < a.K; k += kFinishGroups) {
        const int i = index[k * kFinishCols + col];
        bool leads = true;
        float q = 0.0f;
        if (i >= 0) q = search ? named_slots<kFinishCols>(index, log_p, a.K, k, col, leads) : expf(log_p[k * kFinishCols + col]);
        const long long at = (long long)k * columns + f;
        slots.index[at] = i < 0 || leads ? i : ~1 - i;
        slots.log_p[at] = log_p[k * kFinishCols + col];
        slots.p[at] = q;
    }
    if (group == 0) {
        teacher[f] = c.P;
        teacher[columns + f] = c.weight;
    }
}

template <typename T> constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;       // logits of -inf, which add nothing

// part[chunk of classes][column], by the CTAs before the teacher's.  A thread's sum is relative to a logit not much below its largest one: it changes
// only where one is 2^32 to 2^64 times as much, so that the rows cost little more than their exponentials.  Rows on 16-byte boundaries come through a ring in
// shared memory, in which each thread has the rows that it will read itself: two batches are on their way while the exponentials of a third are taken.
constexpr int kSumBatch = 4, kSumRing = 3, kSumSmem = kSumBatch * kSumRing * kColumnThreads * 16;
template <typename T, int LPR, bool ALIGNED>
__global__ void __launch_bounds__(kColumnThreads, 4)
k_distill_sums(const Distill<T> a, SoftSum *part, int chunk_rows, int tiles, float *teacher, const Slots slots, int teacher_ctas)
{
    grid_dependency();
    extern __shared__ __align__(16) uint8_t buffer[];
    using Col = Column<T, LPR>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    __shared__ SoftSum red[kColumnThreads / 32][kCols];
    const int columns = tiles * kCols;
    const int cta = (int)blockIdx.x, first_teacher = (int)gridDim.x - teacher_ctas;
    if (cta >= first_teacher) {
        teacher_slots(a, cta - first_teacher, teacher, slots, columns);
        return;
    }
    const Col c;
    const int tile = cta % tiles, chunk = cta / tiles;
    const int f = tile * kCols + c.col, step = c.step, n0 = chunk * chunk_rows, n1 = min(a.C, n0 + chunk_rows);
    const float most_above = 32.0f / a.scale;                             // (as a limit in T up to twice that: 2^64)
    float ref[kVec], sum[kVec];                                           // a sum of 0: nothing above -inf yet
    uint4 limit = make_uint4(kNone<T>, kNone<T>, kNone<T>, kNone<T>);     // what a logit has to exceed to become the reference, in T
#pragma unroll
    for (int j = 0; j < kVec; ++j) ref[j] = sum[j] = 0.0f;
    const T *from = a.z + (long long)(n0 + c.row) * a.zs + f;
    const long long z_step = step * a.zs;
    uint8_t *const mine = buffer + threadIdx.x * 16;
    const bool has = f < a.F;
    auto fetch = [&](int slot, int n) {
#pragma unroll
        for (int i = 0; i < kSumBatch; ++i, from += z_step)
            if (has && n + i * step < n1) cp_async16(mine + (slot * kSumBatch + i) * (kColumnThreads * 16), from, true);
        cp_async_commit();
    };
    int n = n0 + c.row, ahead = n, slot = 0, to = 0;
    if constexpr (ALIGNED) {
        for (; to < kSumRing - 1; ++to, ahead += kSumBatch * step) fetch(to, ahead);
    }
    for (; n < n1; n += kSumBatch * step) {
        uint4 raw[kSumBatch], most;
        if constexpr (ALIGNED) {
            fetch(to, ahead);
            ahead += kSumBatch * step;
            to = to == kSumRing - 1 ? 0 : to + 1;
            cp_async_wait<kSumRing - 1>();
        }
        if (ALIGNED && has && n + (kSumBatch - 1) * step < n1) {
#pragma unroll
            for (int i = 0; i < kSumBatch; ++i) raw[i] = *reinterpret_cast<const uint4 *>(mine + (slot * kSumBatch + i) * (kColumnThreads * 16));
        } else {
#pragma unroll
            for (int i = 0; i < kSumBatch; ++i) {
                raw[i] = make_uint4(kNone<T>, kNone<T>, kNone<T>, kNone<T>);
                if (has && n + i * step < n1) {
                    if constexpr (ALIGNED) raw[i] = *reinterpret_cast<const uint4 *>(mine + (slot * kSumBatch + i) * (kColumnThreads * 16));
                    else raw[i] = load_frames<T, false>(a.z + (long long)(n + i * step) * a.zs, f, a.F);
                }
            }
        }
        slot = slot == kSumRing - 1 ? 0 : slot + 1;
        // their largest logits first, then the exponentials
        most = raw[0];
#pragma unroll
        for (int i = 1; i < kSumBatch; ++i) most = packed_max<T>(most, raw[i]);
        const uint4 reach = packed_max<T>(most, limit);
        if (reach.x != limit.x || reach.y != limit.y || reach.z != limit.z || reach.w != limit.w) {
            float top[kVec], l[kVec];
            unpack<T>(most, top);
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const bool first = sum[j] == 0.0f;
                if (first ? top[j] > -INFINITY : top[j] > ref[j]) {
                    if (!first) sum[j] *= exp2_fast((ref[j] - top[j]) * a.scale);
                    ref[j] = top[j];
                }
                l[j] = first && !(top[j] > -INFINITY) ? -INFINITY : ref[j] + most_above;
            }
            limit = pack<T>(l);
        }
#pragma unroll
        for (int i = 0; i < kSumBatch; ++i) {
            float v[kVec];
            unpack<T>(raw[i], v);
#pragma unroll
            for (int j = 0; j < kVec; ++j) sum[j] += exp2_fast((v[j] - ref[j]) * a.scale);
        }
    }
    SoftSum s[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) s[j] = {sum[j] == 0.0f ? -INFINITY : ref[j], sum[j]};
#pragma unroll
    for (int m = LPR; m < 32; m <<= 1)
#pragma unroll
        for (int j = 0; j < kVec; ++j)
            s[j] = join_soft(s[j], {__shfl_xor_sync(0xffffffffu, s[j].top, m), __shfl_xor_sync(0xffffffffu, s[j].sum, m)}, a.scale);
    if (c.lane < LPR) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) red[c.warp][c.col + j] = s[j];
    }
    __syncthreads();
    if (threadIdx.x < kCols) {
        SoftSum t = red[0][threadIdx.x];
        for (int w = 1; w < c.warps; ++w) t = join_soft(t, red[w][threadIdx.x], a.scale);
        part[(long long)chunk * columns + tile * kCols + threadIdx.x] = t;
    }
}

// The numbers of FrameGrad but the slope as grad[3][columns], the frames' losses, and in the place of the named classes' probabilities their dz.  A thread's
// first slots, and the logits that they name, are on their way before the sums are joined.
template <typename T>
__global__ void __launch_bounds__(kColumnThreads)
k_distill_finish(const Distill<T> a, const SoftSum *__restrict__ part, int chunks, const float *__restrict__ teacher, const Slots slots, float *grad, int columns)
{
    grid_dependency();
    __shared__ SoftSum sums[kColumnThreads / 32][kFinishCols];
    __shared__ float red[kColumnThreads / 32][kFinishCols], s_top[kFinishCols], s_log_sum[kFinishCols];
    __shared__ FrameGrad s_grad[kFinishCols];
    const int col = threadIdx.x % kFinishCols, group = threadIdx.x / kFinishCols, warp = threadIdx.x / 32, f = (int)blockIdx.x * kFinishCols + col;
    constexpr int kAhead = 2;
    int code[kAhead];
    float lp[kAhead], p_all[kAhead], z[kAhead];
    auto load = [&](int k0) {
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            const int k = k0 + e * kFinishGroups;
            const long long at = (long long)k * columns + f;
            code[e] = k < a.K ? slots.index[at] : -1;
            lp[e] = k < a.K ? slots.log_p[at] : -INFINITY;
            p_all[e] = k < a.K ? slots.p[at] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            const int i = code[e] < -1 ? ~1 - code[e] : code[e];
            z[e] = i >= 0 ? to_float(a.z[i * a.zs + f]) : 0.0f;
        }
    };
    load(group);
    SoftSum s = {-INFINITY, 0.0f};
    for (int k = group; k < chunks; k += kFinishGroups) s = join_soft(s, part[(long long)k * columns + f], a.scale);
#pragma unroll
    for (int m = kFinishCols; m < 32; m <<= 1) s = join_soft(s, {__shfl_xor_sync(0xffffffffu, s.top, m), __shfl_xor_sync(0xffffffffu, s.sum, m)}, a.scale);
    if (threadIdx.x % 32 < kFinishCols) sums[warp][col] = s;
    __syncthreads();
    if (threadIdx.x < kFinishCols) {
        for (int w = 1; w < kColumnThreads / 32; ++w) s = join_soft(s, sums[w][col], a.scale);
        s_top[col] = reference(s.top);
        s_log_sum[col] = s.sum == 0.0f ? 0.0f : logf(s.sum);
        s_grad[col] = finish_frame(a, teacher[f], teacher[columns + f], s);
    }
    __syncthreads();
    const float top = s_top[col], log_sum = s_log_sum[col];
    const FrameGrad g = s_grad[col];
    float divergence = 0.0f;
    for (int k = group; k < a.K; k += kAhead * kFinishGroups) {
        if (k > group) load(k);
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            const float p = expf(lp[e]);                                  // (0 of an empty slot, and beyond the last one)
            if (p != 0.0f) divergence += p * (lp[e] - ((z[e] - top) * a.inv_t - log_sum));
            if (code[e] >= 0) slots.p[(long long)(k + e * kFinishGroups) * columns + f] = soft_part(g, z[e], a.scale) - g.slope * p_all[e];
        }
    }
    divergence = column_of_warp<kFinishCols>(divergence, [](float x, float y) { return x + y; });
    if (threadIdx.x % 32 < kFinishCols) red[warp][col] = divergence;
    __syncthreads();
    if (threadIdx.x < 32) {
        float loss = 0.0f;
        if (group == 0) {
            const float weight = teacher[columns + f];
            if (weight != 0.0f) loss = weight * a.temperature * a.temperature * join_parts<ColumnSum>(&red[0][col], kFinishCols, kColumnThreads / 32);
            grad[f] = g.top;
            grad[columns + f] = g.factor;
            grad[2LL * columns + f] = g.cap;
        }
        write_losses(a, (int)blockIdx.x, f, group == 0 && f < a.F, loss);
    }
}

// Along the rows, as the layer norm's: what the softmax contributes to dz
constexpr int kDistillBand = 8;
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kColumnThreads)
k_distill_apply(const Distill<T> a, const float *__restrict__ grad, int columns)
{
    grid_dependency();
    constexpr int kVec = kFramesPerVec<T>;
    const Line<T, ALIGNED> line((int)blockIdx.x * 32 * kVec, (int)(threadIdx.x & 31), a.F);
    const int n0 = ((int)blockIdx.y * 8 + (int)(threadIdx.x >> 5)) * kDistillBand;
    if (line.empty()) return;
    uint4 raw[kDistillBand];
#pragma unroll
    for (int i = 0; i < kDistillBand; ++i)
        if (n0 + i < a.C) raw[i] = line.load(a.z + (long long)(n0 + i) * a.zs);
    float top[kVec], factor[kVec], cap[kVec];
    line.load_columns(grad, top);
    line.load_columns(grad + columns, factor);
    line.load_columns(grad + 2LL * columns, cap);
#pragma unroll
    for (int i = 0; i < kDistillBand; ++i) {
        if (n0 + i < a.C) {
            float v[kVec];
            unpack<T>(raw[i], v);
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[j] = soft_part({top[j], factor[j], cap[j], 0.0f}, v[j], a.scale);
            line.store(a.dz + (long long)(n0 + i) * a.dzs, v);
        }
    }
}

// the named classes, a frame and slot a thread
template <typename T>
__global__ void __launch_bounds__(kColumnThreads)
k_distill_named(const Distill<T> a, const Slots slots, int columns)
{
    grid_dependency();
    const int f = (int)blockIdx.x * kColumnThreads + threadIdx.x, k = blockIdx.y;
    if (f >= a.F) return;
    const int i = slots.index[(long long)k * columns + f];
    const float dz = slots.p[(long long)k * columns + f];
    if (i >= 0) a.dz[i * a.dzs + f] = from_float<T>(dz);
}

__global__ void __launch_bounds__(1024) k_distill_loss(const double *__restrict__ part, int parts, double loss_reduction, float *loss)
{
    grid_dependency();
    __shared__ double red[32];
    double s = 0.0;
    for (int k = threadIdx.x; k < parts; k += 1024) s += part[k];
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = red[threadIdx.x];
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        if (threadIdx.x == 0) *loss = (float)(s * loss_reduction);
    }
}

constexpr int kDistillSmem = 200 * 1024;                 // more than any call needs: 64 KB of logits, 128 KB of slots, 4 KB of bits

template <typename T, int LPR>
static int distillation_once(const Distill<T> &a, const ColumnPlan &p, int tiles, cudaStream_t st)
{
    int *fault = fault_word();
    BB200_REQUIRE(fault != nullptr, BBCU_ERR_NO_DEVICE);
    auto kernel = k_distill_once<T, LPR>;
    constexpr int kCols = Column<T, LPR>::kCols;
    const int threads = 32 * p.warps, smem = p.rows * threads * 16 + a.K * kCols * 8 + (p.warps * 32 / LPR * p.rows + 31) / 32 * kCols * 4 +
              (p.cluster > 1 ? 2 * p.cluster * 4 * kCols * 4 : 0);
    BB200_REQUIRE(allow_big_smem(kernel, kDistillSmem), (int)cudaErrorInvalidValue);
    const int clusters = std::min(tiles, resident_clusters(reinterpret_cast<const void *>(kernel), p.cluster, threads, smem));
    return launch_cluster(kernel, (unsigned)p.cluster, (unsigned)(clusters * p.cluster), threads, smem, st, a, p.rows, tiles, fault);
}

// Chunks of rows that a streaming kernel is cut into beside its column tiles: of up to `most`, the number whose CTAs fill their last round on the
// device best.
static int best_chunks(long long tiles, long long resident, int most)
{
    int best = 1;
    double filled = 0.0;
    for (int n = 1; n <= most; ++n) {
        const long long ctas = tiles * n, rounds = (ctas + resident - 1) / resident;
        if (rounds > 4 && n > 1) break;
        const double share = (double)ctas / (double)(rounds * resident);
        if (share > filled + 0.02) { filled = share; best = n; }
    }
    return best;
}

template <typename T, int LPR>
static int distillation_passes(Distill<T> &a, int &loss_parts, bool aligned, HeldScratch &held, cudaStream_t st)
{
    constexpr int kCols = Column<T, LPR>::kCols, kWide = 32 * kFramesPerVec<T>;
    const int tiles = (a.F + kCols - 1) / kCols, columns = tiles * kCols;
    const long long bands = ((long long)a.C + 8 * kDistillBand - 1) / (8 * kDistillBand);
    BB200_REQUIRE(bands <= 65535, BBCU_ERR_TOO_LARGE);
    auto sums = aligned ? k_distill_sums<T, LPR, true> : k_distill_sums<T, LPR, false>;
    const size_t sum_smem = std::max(aligned ? (size_t)kSumSmem : (size_t)0, (size_t)a.K * kFinishCols * 8 + ((size_t)kFinishCols << slot_hash_bits(a.K)) / 8);
    BB200_REQUIRE(allow_big_smem(sums, (int)sum_smem), (int)cudaErrorInvalidValue);
    // (chunks of 1024 rows at least, or 256 where there are few tiles: 8192 classes x 8192 frames bf16, 64 slots, 107 us by two chunks, 120 by nine)
    const int chunks = best_chunks(tiles, resident_clusters(reinterpret_cast<const void *>(sums), 1, kColumnThreads, sum_smem), std::min(64, std::max(1, a.C / (tiles >= device_info().sm_count / 2 ? 1024 : 256))));
    const int rows = (a.C + chunks - 1) / chunks;
    loss_parts = columns / kFinishCols;
    const size_t part_b = (size_t)chunks * columns * sizeof(SoftSum), loss_b = (size_t)loss_parts * sizeof(double), slots = (size_t)a.K * columns;
    char *scratch = static_cast<char *>(held.get(st, loss_b + part_b + ((size_t)5 * columns + 3 * slots) * 4));
    BB200_REQUIRE(scratch != nullptr, BBCU_ERR_NO_MEMORY);
    a.loss_part = reinterpret_cast<double *>(scratch);
    SoftSum *part = reinterpret_cast<SoftSum *>(scratch + loss_b);
    float *grad = reinterpret_cast<float *>(scratch + loss_b + part_b), *teacher = grad + (size_t)3 * columns, *slot_p = teacher + (size_t)2 * columns;
    const Slots kept = {reinterpret_cast<int *>(slot_p + 2 * slots), slot_p + slots, slot_p};
    BB200_REQUIRE((long long)tiles * chunks + loss_parts < (1LL << 31), BBCU_ERR_TOO_LARGE);
    launch(sums, (unsigned)(tiles * chunks + loss_parts), kColumnThreads, sum_smem, st, a, part, rows, tiles, teacher, kept, loss_parts);
    BB200_CUDA(cudaPeekAtLastError());
    launch(k_distill_finish<T>, (unsigned)loss_parts, kColumnThreads, 0, st, a, part, chunks, teacher, kept, grad, columns);
    BB200_CUDA(cudaPeekAtLastError());
    launch(aligned ? k_distill_apply<T, true> : k_distill_apply<T, false>, dim3((unsigned)((a.F + kWide - 1) / kWide), (unsigned)bands), kColumnThreads, 0, st, a, grad,
           columns);
    BB200_CUDA(cudaPeekAtLastError());
    if (a.K > 0)
        launch(k_distill_named<T>, dim3((unsigned)((a.F + kColumnThreads - 1) / kColumnThreads), (unsigned)a.K), kColumnThreads, 0, st, a, kept, columns);
    return launch_status();
}

template <typename T>
static int distillation(Distill<T> a, float *loss, double loss_reduction, cudaStream_t st)
{
    constexpr int kLanes = 4;                                              // 64 bytes of a row: up to 1024 classes a CTA
    const bool aligned = frames_aligned<T>(a.z, a.zs) && frames_aligned<T>(a.dz, a.dzs);
    ColumnPlan p = plan_columns<T>(a.C, a.F, kLanes, kDistillRows, kDistillCluster);
    if (!aligned) p.cluster = 0;
    if (p.cluster) {
        // a power of two of warps; where there are many tiles, few of them with more rows a thread, since all warps of a CTA take part in the teacher's side
        // and its barriers (100 classes x 65536 frames: eight warps 51 us, two 28)
        const int cols = p.lanes * kFramesPerVec<T>, per_warp = 32 / p.lanes, cta_rows = (a.C + p.cluster - 1) / p.cluster;
        while (p.warps & (p.warps - 1)) ++p.warps;
        if ((long long)(a.F / cols) * p.cluster >= 4LL * device_info().sm_count)
            while (p.warps > 2 && cta_rows <= per_warp * (p.warps / 2) * kDistillRows / 2) p.warps /= 2;
        p.rows = (cta_rows + per_warp * p.warps - 1) / (per_warp * p.warps);
    }
    HeldScratch held;                                                     // until the loss is on its way
    int parts = 0, e;
    if (p.cluster) {
        const int cols = p.lanes * kFramesPerVec<T>;
        parts = (a.F + cols - 1) / cols;
        a.loss_part = static_cast<double *>(held.get(st, (size_t)parts * sizeof(double)));
        BB200_REQUIRE(a.loss_part != nullptr, BBCU_ERR_NO_MEMORY);
        e = p.lanes == 2 ? distillation_once<T, 2>(a, p, parts, st) : distillation_once<T, kLanes>(a, p, parts, st);
    } else {
        e = distillation_passes<T, sizeof(T) == 4 ? 8 : 4>(a, parts, aligned, held, st);
    }
    if (e != BBCU_OK) return e;
    launch(k_distill_loss, 1, 1024, 0, st, a.loss_part, parts, loss_reduction, loss);
    return launch_status();
}

template <typename T>
static int distillation_checked(const T *z, T *dz, const T *t, const int *index, const float *t_lse, const float *weight, float *loss_buf, float *loss,
                                float temperature, float grad_reduction, double loss_reduction, int C, int K, int F, int zs, int dzs, int ts, int is,
                                bbcu_stream_t stream)
{
    BB200_REQUIRE(C > 0 && K >= 0 && F >= 0 && temperature > 0.0f && temperature < INFINITY &&
                  kLog2e / temperature < INFINITY, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(C <= (1 << 20) && K <= kMostSlots && F <= (1 << 30), BBCU_ERR_TOO_LARGE);
    BB200_REQUIRE(zs >= F && dzs >= F && (K == 0 || (ts >= F && is >= F)), BBCU_ERR_BAD_STRIDE);
    BB200_REQUIRE_PTR(loss);
    cudaStream_t st = as_stream(stream);
    if (F == 0) {
        BB200_CUDA(cudaMemsetAsync(loss, 0, sizeof(float), st));
        return BBCU_OK;
    }
    BB200_REQUIRE_PTR(z); BB200_REQUIRE_PTR(dz); BB200_REQUIRE_PTR(loss_buf);
    if (K > 0) { BB200_REQUIRE_PTR(t); BB200_REQUIRE_PTR(index); }
    return distillation<T>({z, t, dz, index, t_lse, weight, loss_buf, nullptr, temperature, 1.0f / temperature, kLog2e / temperature, grad_reduction, C, K, F, zs, dzs, ts, is},
                           loss, loss_reduction, st);
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
