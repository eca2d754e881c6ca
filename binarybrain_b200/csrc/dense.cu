// Dense layers in bf16 on the tensor cores, with what follows a product done before its sums leave the chip, and their gradients.  (The reference's dense
// layers are fp32 through cuBLAS, include/bb/DenseAffine.h; it has no gated block.)
//
//   forward          z[o][f] = sum_k W[o][k] x[k][f] + b[o],   y = act(z) + r
//   gated            g = (W x)[h],  u = (W x)[H + h]  (+ bias),   y[h][f] = act(g) u           both products on one read of x
//   input gradient   dx[i][f] = sum_o W[o][i] dy[o][f],  times act'(z[i][f]) where the input was an activation of z,  or, where it was a gated block's
//                    output, the gradients of both of its products: dg = dx u act'(g), du = dx act(g)
//   weight gradient  dW[o][i] += sum_f dy[o][f] x[i][f],  db[o] += sum_f dy[o][f]
//
// x, W, dy and the kept z are bf16; the sums are 32 bits, bias, activation, residual and gate are applied to them in 32 bits, and each output is rounded once.
// Frame buffers are read as they lie, frames next to each other: where the product sums over nodes, its operand is "across" (rows of shared memory along
// the frames), which the tensor cores take from TMA's 128-byte swizzled boxes as well as rows along k; the gradients read W and x the other way round, and nothing is transposed.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include <cuda.h>

#include "async_copy.cuh"
#include "frame_columns.cuh"
#include "tensor_core.cuh"

namespace bb200 {

enum DenseKind { kForward, kGated, kInputGrad, kWeightGrad };

constexpr int kTileM = 128, kTileK = 64;                 // output rows of a CTA; k of a stage (128 bytes)
constexpr int kMostSplits = 8;
constexpr int kTileGroup = 8;                            // tiles of output rows that are walked together, so that their operands stay in L2

struct DenseArgs {
    const float *bias;
    const void *extra;                                   // residual (forward), z (input gradient)
    void *out, *z_out;
    int act, gated, accumulate, vec;                     // vec: the rows of extra, out and z_out start on 16-byte boundaries; 2: on 32-byte ones
    int M, N, K, half;                                   // half: rows of a gated block's output, the distance between its two products
    int splits, chunk;                                   // chunk: stages of k between two additions in registers, for fp32 outputs (see sums_chunk)
    long long extra_stride, out_stride, z_stride;
    int *fault;
};

// ---- activations, in 32 bits: value and slope, of which the compiler keeps what is used.  FAST, for outputs of 16 bits: exp(x) by the special function unit,
// whose argument is rounded, so that it is off by |x| + 2 half-units in the last place of 32 bits; 88 at most.
struct Curve { float value, slope; };

template <bool FAST> __device__ __forceinline__ float exp_of(float x) { return FAST ? __expf(x) : expf(x); }

template <bool FAST> __device__ __forceinline__ Curve silu(float z)
{
    // (the divisor is between 1 and 2)
    const float e = exp_of<FAST>(-fabsf(z)), inv = __fdividef(1.0f, 1.0f + e), rest = e * inv, p = z < 0.0f ? rest : inv;
    return {z * p, fmaf(z, rest * inv, p)};
}

// gelu = z Phi(z), slope = Phi(z) + z phi(z).  Phi(-|z|) exp(z^2 / 2) is t times a polynomial in t = 1 / (1 + 0.35 |z|), fitted to 0.5 erfcx(|z| / sqrt 2) / t over
// |z| <= 14 by weighted least squares to 3.2e-8 of its value, so that the digits stay where Phi is small; gelu is off by 11 half-units in the last place for |z| < 3,
// and by those of the exponent's rounding beyond.  (erfcf takes three times the operations, which were half of the time of a product of 1024 inputs.)
template <bool FAST> __device__ __forceinline__ Curve gelu(float z)
{
    const float a = fabsf(z), t = __fdividef(1.0f, fmaf(0.35f, a, 1.0f)), e = FAST ? __expf(-0.5f * z * z) : exp2f(-0.72134752f * z * z);
    float p = -0.029145934f;
    p = fmaf(p, t, 0.14397171f);
    p = fmaf(p, t, -0.25571427f);
    p = fmaf(p, t, 0.15917419f);
    p = fmaf(p, t, -0.02310985f);
    p = fmaf(p, t, 0.10550801f);
    p = fmaf(p, t, 0.119832866f);
    p = fmaf(p, t, 0.13986187f);
    p = fmaf(p, t, 0.1396214f);
    const float q = t * p * e, phi = z < 0.0f ? q : 1.0f - q;
    return {z * phi, fmaf(z * 0.39894228f, e, phi)};
}

template <int ACT, bool FAST> __device__ __forceinline__ Curve curve(float z)
{
    if constexpr (ACT == BBCU_ACTIVATION_RELU) return {z < 0.0f ? 0.0f : z, z > 0.0f ? 1.0f : z != z ? z : 0.0f};
    if constexpr (ACT == BBCU_ACTIVATION_GELU) return gelu<FAST>(z);
    if constexpr (ACT == BBCU_ACTIVATION_SILU) return silu<FAST>(z);
    return {z, 1.0f};
}

// f(std::integral_constant<int, act>): the activation is one for all of a call
template <typename F> __device__ __forceinline__ void with_activation(int act, F f)
{
    switch (act) {
    case BBCU_ACTIVATION_RELU: f(std::integral_constant<int, BBCU_ACTIVATION_RELU>()); break;
    case BBCU_ACTIVATION_GELU: f(std::integral_constant<int, BBCU_ACTIVATION_GELU>()); break;
    case BBCU_ACTIVATION_SILU: f(std::integral_constant<int, BBCU_ACTIVATION_SILU>()); break;
    default: f(std::integral_constant<int, BBCU_ACTIVATION_NONE>()); break;
    }
}

// ---- what is made of eight (or, at the end of a row or at odd addresses, one) neighbouring sums of a row
template <typename T> __device__ __forceinline__ void load_8(const T *p, float (&v)[8])
{
    if constexpr (sizeof(T) == 4) {
        float a[4], b[4];
        unpack<float>(*reinterpret_cast<const uint4 *>(p), a);
        unpack<float>(*reinterpret_cast<const uint4 *>(p + 4), b);
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    } else {
        unpack<T>(*reinterpret_cast<const uint4 *>(p), v);
    }
}
template <typename T> __device__ __forceinline__ void store_8(T *p, const float (&v)[8])
{
    if constexpr (sizeof(T) == 4) {
        const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
        *reinterpret_cast<uint4 *>(p) = pack<float>(a);
        *reinterpret_cast<uint4 *>(p + 4) = pack<float>(b);
    } else {
        *reinterpret_cast<uint4 *>(p) = pack<T>(v);
    }
}
template <typename T, int V> __device__ __forceinline__ void load_some(const T *p, float (&v)[V])
{
    if constexpr (V == 8) load_8<T>(p, v);
    else v[0] = to_float(*p);
}
template <typename T, int V> __device__ __forceinline__ void store_some(T *p, const float (&v)[V])
{
    if constexpr (V == 8) store_8<T>(p, v);
    else *p = from_float<T>(v[0]);
}

// v: sums of row m, columns n on; w: those of a gated block's second product
template <int KIND, typename T, int V> __device__ __forceinline__ void finish(const DenseArgs &a, int m, int n, float (&v)[V], float (&w)[V])
{
    using B = __nv_bfloat16;
    T *const out = static_cast<T *>(a.out) + (long long)m * a.out_stride + n;
    if constexpr (KIND == kForward) {
        float r[V];
        if (a.extra) load_some<T, V>(static_cast<const T *>(a.extra) + (long long)m * a.extra_stride + n, r);
        const float b = a.bias ? a.bias[m] : 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += b;
        if (a.z_out) store_some<B, V>(static_cast<B *>(a.z_out) + (long long)m * a.z_stride + n, v);
        with_activation(a.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = curve<decltype(act)::value, sizeof(T) == 2>(v[j]).value;
        });
        if (a.extra) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] += r[j];
        }
        store_some<T, V>(out, v);
    } else if constexpr (KIND == kGated) {
        const float b = a.bias ? a.bias[m] : 0.0f, c = a.bias ? a.bias[a.half + m] : 0.0f;
        float y[V];
#pragma unroll
        for (int j = 0; j < V; ++j) { v[j] += b; w[j] += c; }
        with_activation(a.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < V; ++j) y[j] = curve<decltype(act)::value, sizeof(T) == 2>(v[j]).value * w[j];
        });
        store_some<T, V>(out, y);
        if (a.z_out) {
            store_some<B, V>(static_cast<B *>(a.z_out) + (long long)m * a.z_stride + n, v);
            store_some<B, V>(static_cast<B *>(a.z_out) + (long long)(a.half + m) * a.z_stride + n, w);
        }
    } else if constexpr (KIND == kInputGrad) {
        const B *const z = static_cast<const B *>(a.extra) + (long long)m * a.extra_stride + n;
        if (a.gated) {
            float g[V], u[V], d[V];
            load_some<B, V>(z, g);
            load_some<B, V>(z + (long long)a.half * a.extra_stride, u);
            with_activation(a.act, [&](auto act) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const Curve k = curve<decltype(act)::value, sizeof(T) == 2>(g[j]);
                    d[j] = v[j] * k.value;
                    v[j] *= u[j] * k.slope;
                }
            });
            store_some<T, V>(out, v);
            store_some<T, V>(out + (long long)a.half * a.out_stride, d);
        } else {
            if (a.extra) {
                float g[V];
                load_some<B, V>(z, g);
                with_activation(a.act, [&](auto act) {
#pragma unroll
                    for (int j = 0; j < V; ++j) v[j] *= curve<decltype(act)::value, sizeof(T) == 2>(g[j]).slope;
                });
            }
            store_some<T, V>(out, v);
        }
    } else {
        if (a.accumulate) {
            float r[V];
            load_some<T, V>(out, r);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] += r[j];
        }
        store_some<T, V>(out, v);
    }
}

// as many of eight columns as there are
template <int KIND, typename T> __device__ __forceinline__ void finish_8(const DenseArgs &a, int m, int n, float (&v)[8], float (&w)[8])
{
    if (a.vec && n + 8 <= a.N) {
        finish<KIND, T, 8>(a, m, n, v, w);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (n + j < a.N) {
                float p[1] = {v[j]}, q[1] = {w[j]};
                finish<KIND, T, 1>(a, m, n + j, p, q);
            }
    }
}

// ---- up to eight frames: what counts is to have W on its way, once.  A CTA has its share of the rows, whatever their number; a warp takes up to 16 rows and a part of the
// inputs, and each lane has its pieces of W, 16 bytes of two rows a block of 32 inputs, asked for two batches ahead, in registers, from where they go into products of
// 16 rows x 8 frames (the k of a product may be any, as long as W and the frames have the same: a lane's 16 bytes are two pairs of pairs).  The frames come
// out of shared memory, where the CTA has turned them over; the parts' sums meet there, in the order of the warps.
// (Multiplied out by each lane, a single frame took 27 instructions for 16 bytes of W: 4096 -> 2 x 8192 31 us.)
constexpr int kFewThreads = 512, kFewFrames = 8, kFewInputs = 32768;           // inputs x frames that a CTA holds at a time
constexpr int few_chunk(int frames) { return kFewInputs / (frames > 4 ? 8 : frames > 2 ? 4 : frames); }
template <int KIND, typename T>
__global__ void __launch_bounds__(kFewThreads, 1)
k_dense_few(const __nv_bfloat16 *__restrict__ x, const __nv_bfloat16 *__restrict__ W, long long xs, long long ws, const DenseArgs a, int groups, int chunk)
{
    grid_dependency();
    constexpr int kParts = KIND == kGated ? 2 : 1, kBatch = 4 / kParts, kWarps = kFewThreads / 32, kBlock = 32;
    extern __shared__ __align__(16) uint8_t smem_few[];
    __nv_bfloat16 *const frames = reinterpret_cast<__nv_bfloat16 *>(smem_few);     // [frame][chunk + 8]
    __shared__ float sums[kWarps][kParts][16][kFewFrames];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, pitch = chunk + 8;
    const int first = (int)((long long)a.M * blockIdx.x / gridDim.x), last = (int)((long long)a.M * (blockIdx.x + 1) / gridDim.x);
    const int group = warp % groups, part = warp / groups, parts = kWarps / groups;
    for (int m0 = first; m0 < last; m0 += groups * 16) {
        const int rows = min(groups * 16, last - m0), per_group = (rows + groups - 1) / groups;
        const int r0 = group * per_group + g, here = min(per_group, rows - group * per_group);      // rows of the group that exist
        float acc[kParts][4] = {}, total[kParts][4] = {};
        int done = 0;                                                     // blocks in acc, of whichever pieces of the inputs
        for (int k0 = 0; k0 < a.K; k0 += chunk) {
            const int inputs = min(chunk, a.K - k0), blocks = (inputs + kBlock - 1) / kBlock, begin = blocks * part / parts, end = blocks * (part + 1) / parts;
            const __nv_bfloat16 *const base = W + (long long)(m0 + r0) * ws + k0 + 8 * t;
            uint4 w[kBatch][kParts][2], next[kBatch][kParts][2];
            auto fetch = [&](int b, uint4 (&w)[kBatch][kParts][2]) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
#pragma unroll
                    for (int p = 0; p < kParts; ++p)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int k = (b + i) * kBlock;
                            w[i][p][h] = b + i < end && k + 8 * t < inputs && g + 8 * h < here
                                             ? __ldg(reinterpret_cast<const uint4 *>(base + (long long)(8 * h + p * a.half) * ws + k)) : make_uint4(0, 0, 0, 0);
                        }
            };
            fetch(begin, w);
            if (m0 == first || a.K > chunk) {
                __syncthreads();
#pragma unroll 4
                for (int k = threadIdx.x; k < blocks * kBlock; k += kFewThreads) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (k < inputs) v = *reinterpret_cast<const uint4 *>(x + (long long)(k0 + k) * xs);
                    const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int f = 0; f < kFewFrames; ++f)
                        if (f < a.N) reinterpret_cast<uint16_t *>(frames)[f * pitch + k] = (uint16_t)(word[f / 2] >> (16 * (f % 2)));
                }
                __syncthreads();
            }
            for (int b = begin; b < end; b += kBatch) {
                fetch(b + kBatch, next);
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    if (b + i >= end) break;
                    const int k = (b + i) * kBlock + 8 * t;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (g < a.N) v = *reinterpret_cast<const uint4 *>(frames + g * pitch + k);
                    if (k + 8 > inputs) {                                 // the padding of W may hold anything
                        const int left = inputs - k;
#pragma unroll
                        for (int p = 0; p < kParts; ++p)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                uint32_t *const word = reinterpret_cast<uint32_t *>(&w[i][p][h]);
#pragma unroll
                                for (int q = 0; q < 4; ++q) word[q] = left >= 2 * q + 2 ? word[q] : left == 2 * q + 1 ? word[q] & 0xffffu : 0u;
                            }
                    }
#pragma unroll
                    for (int p = 0; p < kParts; ++p) {
                        mma_rows_bf16(acc[p], w[i][p][0].x, w[i][p][1].x, w[i][p][0].y, w[i][p][1].y, v.x, v.y);
                        mma_rows_bf16(acc[p], w[i][p][0].z, w[i][p][1].z, w[i][p][0].w, w[i][p][1].w, v.z, v.w);
                    }
                }
                done += kBatch;
                if (sizeof(T) == 4 && done >= a.chunk * (kTileK / kBlock)) {  // the tensor cores cut what does not fit their running sum
                    done = 0;
#pragma unroll
                    for (int p = 0; p < kParts; ++p)
#pragma unroll
                        for (int j = 0; j < 4; ++j) { total[p][j] += acc[p][j]; acc[p][j] = 0.0f; }
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
#pragma unroll
                    for (int p = 0; p < kParts; ++p)
#pragma unroll
                        for (int h = 0; h < 2; ++h) w[i][p][h] = next[i][p][h];
            }
        }
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums[warp][p][g + (j >= 2 ? 8 : 0)][2 * t + j % 2] = total[p][j] + acc[p][j];
        __syncthreads();
        if ((int)threadIdx.x < rows) {
            const int from = threadIdx.x / per_group, row = threadIdx.x % per_group;
            float v[2][8] = {};
            for (int i = 0; i < parts; ++i)
#pragma unroll
                for (int p = 0; p < kParts; ++p)
#pragma unroll
                    for (int f = 0; f < kFewFrames; ++f) v[p][f] += sums[i * groups + from][p][row][f];
            finish_8<KIND, T>(a, m0 + threadIdx.x, 0, v[0], v[kParts - 1]);
        }
        __syncthreads();
    }
}

// ---- tiles of 128 output rows x TN columns in TMEM (lane = row), by one CTA; or, PAIR, of 256 rows by a pair of CTAs (cta_group::2), each of which brings its
// 128 rows of A and half of the columns of B and gets the sums of its rows.  64 of k a stage.  The accumulator is double: the sums of a tile leave beside the
// products of the next.  Where there are fewer tiles than SMs, a cluster of CTAs shares the k of one: their sums cross through distributed shared memory and
// are added in the order of the CTAs.
//
// Both products of a gated block: a CTA brings both operands' rows and has two accumulators, so that a lane has both sums of its row; a pair would bring 40 KB a stage
// that way, and 50 bytes a clock are what an SM gets.  A pair's tile is 128 rows x 256 columns of the output instead, 64 rows of either product in the 128
// lanes of a CTA, and the warps of the lower lanes get the second product's sums from those of the upper ones through shared memory.
//
// fp32 outputs: the sums are taken out every a.chunk stages and added up in registers, see sums_chunk().
template <int KIND, typename T, int TN, bool PAIR> struct DenseShape {
    static constexpr bool kAAcross = KIND == kInputGrad, kBAcross = KIND != kWeightGrad, kPromote = sizeof(T) == 4;
    static constexpr bool kStacked = KIND == kGated && PAIR;
    static constexpr int kRows = PAIR && !kStacked ? 2 * kTileM : kTileM, kOwnRows = kStacked ? kTileM / 2 : kTileM;      // output rows of a tile, of a CTA
    static constexpr int kParts = KIND == kGated && !PAIR ? 2 : 1, kOwnN = PAIR ? TN / 2 : TN, kBRows = kBAcross && kOwnN < 64 ? 64 : kOwnN;
    static constexpr int kABytes = kTileM * kTileK * 2, kStageBytes = kParts * kABytes + kBRows * kTileK * 2;
    static constexpr int kWarps = 16, kThreads = 64 + 32 * kWarps;        // warp 0 copies, warp 1 issues the products, the others take the sums out of TMEM
    static constexpr int kPiece = 16;                                     // columns that a warp takes at a time: a sector of bf16 (32: registers, gelu's gradient 91 -> 84 us)
    static constexpr int kOutBytes = 32 * kPiece * (int)sizeof(T);
    static constexpr int kCross = kStacked ? kWarps / 2 : 0, kCrossBytes = 2 * 32 * kPiece * 4;        // pairs of warps that exchange sums, two buffers each
    static constexpr int kRoom = 225 * 1024 - kWarps * kOutBytes - kCross * kCrossBytes, kStages = kRoom / kStageBytes > 8 ? 8 : kRoom / kStageBytes;
    static constexpr int kSmem = kStages * kStageBytes + kWarps * kOutBytes + kCross * kCrossBytes + 1024;
    static constexpr int kAccColumns = kParts * TN, kColumns = 2 * kAccColumns < 32 ? 32 : 2 * kAccColumns;
    static constexpr int kWarpColumns = TN * 4 / kWarps < kPiece ? kPiece : TN * 4 / kWarps;  // a warp's share of a tile's columns
};

// A warp's 32 rows, a row a lane, of P pieces of eight columns (fp32: of four) to memory (`base`: the first row at the first column, `rows` and `left` columns of it
// exist): they cross shared memory, where the order of a row's pieces differs from row to row so that no banks collide, and leave as P * 16 bytes of a row; at odd
// addresses a column a lane.
template <int P> __device__ __forceinline__ int staged_piece(int row, int q) { return row * P + (q ^ (P == 8 ? row & 7 : P == 4 ? row >> 1 & 3 : row >> 2 & 1)); }
template <int P> __device__ __forceinline__ void store_rows(uint4 *stage, const uint4 (&v)[P], __nv_bfloat16 *base, long long stride, int rows, int left, int vec)
{
    const int lane = threadIdx.x & 31;
    if (vec == 2) {
        // whole sectors of the lane's own row: nothing crosses shared memory, whose bandwidth the products live on
        if (lane >= rows) return;
        __nv_bfloat16 *const to = base + lane * stride;
#pragma unroll
        for (int q = 0; q < P; q += 2) {
            if (8 * q + 16 <= left) {
                store_32_bytes(to + 8 * q, v[q], v[q + 1]);
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const uint32_t word = reinterpret_cast<const uint32_t *>(&v[q + j / 8])[j % 8 / 2];
                    if (8 * q + j < left) to[8 * q + j] = __ushort_as_bfloat16((unsigned short)(j % 2 ? word >> 16 : word));
                }
            }
        }
        return;
    }
#pragma unroll
    for (int q = 0; q < P; ++q) stage[staged_piece<P>(lane, q)] = v[q];
    __syncwarp();
    if (vec) {
        const int q = lane % P;
#pragma unroll
        for (int it = 0; it < P; ++it) {
            const int r = it * (32 / P) + lane / P;
            const uint4 piece = stage[staged_piece<P>(r, q)];
            __nv_bfloat16 *const to = base + r * stride + 8 * q;
            if (r >= rows) continue;
            if (8 * q + 8 <= left) {
                *reinterpret_cast<uint4 *>(to) = piece;
            } else {
                const __nv_bfloat16 *const one = reinterpret_cast<const __nv_bfloat16 *>(&piece);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (8 * q + j < left) to[j] = one[j];
            }
        }
    } else if (lane < left && lane < 8 * P) {
#pragma unroll 8
        for (int r = 0; r < min(32, rows); ++r) base[r * stride + lane] = reinterpret_cast<const __nv_bfloat16 *>(&stage[staged_piece<P>(r, lane / 8)])[lane % 8];
    }
    __syncwarp();
}

// The way back: 32 rows of P pieces of eight columns of an input of the epilogue.  Rows on 32-byte boundaries come as whole sectors of the lane's own row.  Others are
// asked for as they lie, P * 16 bytes of a row by P lanes side by side, and change places through the same shared memory when they are needed.  (A lane asking for
// 16 bytes of its own row brings every sector twice.)
template <int P> __device__ __forceinline__ void load_rows(uint4 (&e)[P], const __nv_bfloat16 *base, long long stride, int rows, int left, int vec)
{
    const int lane = threadIdx.x & 31, q = lane % P;
    if (vec == 2) {
#pragma unroll
        for (int i = 0; i < P; i += 2) {
            e[i] = e[i + 1] = make_uint4(0, 0, 0, 0);
            if (lane < rows && 8 * i < left) load_32_bytes(base + lane * stride + 8 * i, e[i], e[i + 1]);
        }
        return;
    }
#pragma unroll
    for (int it = 0; it < P; ++it) {
        const int r = it * (32 / P) + lane / P;
        const __nv_bfloat16 *const p = base + r * stride + 8 * q;
        e[it] = make_uint4(0, 0, 0, 0);
        if (r >= rows || 8 * q >= left) continue;
        if (vec) {
            e[it] = *reinterpret_cast<const uint4 *>(p);
        } else {
            __nv_bfloat16 *const one = reinterpret_cast<__nv_bfloat16 *>(&e[it]);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (8 * q + j < left) one[j] = p[j];
        }
    }
}
template <int P> __device__ __forceinline__ void spread_rows(uint4 *stage, uint4 (&e)[P], int vec)
{
    const int lane = threadIdx.x & 31;
    if (vec == 2) return;
#pragma unroll
    for (int it = 0; it < P; ++it) stage[staged_piece<P>(it * (32 / P) + lane / P, lane % P)] = e[it];
    __syncwarp();
#pragma unroll
    for (int q = 0; q < P; ++q) e[q] = stage[staged_piece<P>(lane, q)];
    __syncwarp();
}

// fp32, with `extra` (null: nothing) added on the way, or added to what is there (one addition an element, so that its order does not matter)
template <int C> __device__ __forceinline__ void store_rows(uint4 *stage, const float (&v)[C], float *base, long long stride, const float *extra, long long extra_stride,
                                                            bool accumulate, int rows, int left, bool vec)
{
    constexpr int P = C / 4;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int q = 0; q < P; ++q) {
        const float p[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        stage[staged_piece<P>(lane, q)] = pack<float>(p);
    }
    __syncwarp();
    if (vec) {
        const int q = lane % P;
#pragma unroll
        for (int it = 0; it < P; ++it) {
            const int r = it * (32 / P) + lane / P;
            float p[4];
            unpack<float>(stage[staged_piece<P>(r, q)], p);
            float *const to = base + r * stride + 4 * q;
            if (r >= rows || 4 * q >= left) continue;
            if (4 * q + 4 <= left) {
                if (extra) {
                    float e[4];
                    unpack<float>(*reinterpret_cast<const uint4 *>(extra + r * extra_stride + 4 * q), e);
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[j] += e[j];
                }
                if (accumulate) red_add_v4(to, p[0], p[1], p[2], p[3]);
                else *reinterpret_cast<uint4 *>(to) = pack<float>(p);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (4 * q + j < left) to[j] = accumulate ? to[j] + p[j] : extra ? p[j] + extra[r * extra_stride + 4 * q + j] : p[j];
            }
        }
    } else if (lane < left && lane < C) {
#pragma unroll 4
        for (int r = 0; r < min(32, rows); ++r) {
            const float p = reinterpret_cast<const float *>(&stage[staged_piece<P>(r, lane / 4)])[lane % 4];
            float *const to = base + r * stride + lane;
            *to = accumulate ? *to + p : extra ? p + extra[r * extra_stride + lane] : p;
        }
    }
    __syncwarp();
}

template <int KIND, typename T, int TN, bool PAIR>
__global__ void __launch_bounds__(DenseShape<KIND, T, TN, PAIR>::kThreads, 1)
k_dense_tiles(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const DenseArgs a)
{
    using S = DenseShape<KIND, T, TN, PAIR>;
    constexpr int kStages = S::kStages, kAcc = 2, kParts = S::kParts, kPiece = S::kPiece;
    static_assert(S::kColumns <= 512 && (S::kColumns & (S::kColumns - 1)) == 0, "TMEM");
    static_assert(kStages >= 4 && kParts * kTileM * (TN + 4) * 4 <= kStages * S::kStageBytes, "shared memory");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[kStages], empty[kStages], acc_full[kAcc], acc_empty[kAcc], drained, cross_full[S::kStacked ? S::kCross : 1][2], cross_empty[S::kStacked ? S::kCross : 1][2];
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR || a.splits > 1 ? cluster_rank() : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int s = 0; s < kAcc; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], PAIR ? 2 * S::kWarps : S::kWarps); }
        mbar_init(&drained, 1);
        if (S::kStacked)
            for (int i = 0; i < 2 * S::kCross; ++i) { mbar_init(&cross_full[i / 2][i % 2], 1); mbar_init(&cross_empty[i / 2][i % 2], 1); }
        gave_up = 0;
        mbar_init_fence();
        tma_prefetch(&map_a);
        tma_prefetch(&map_b);
    }
    __syncwarp();
    if (warp == 1) {
        if constexpr (PAIR) tmem_alloc_pair(&tmem_base, S::kColumns);
        else tmem_alloc(&tmem_base, S::kColumns);
    }
    tcgen05_fence_before();
    __syncthreads();
    if constexpr (PAIR) { cluster_arrive(); cluster_wait(); }
    tcgen05_fence_after();
    const uint32_t tmem = tmem_base;
    grid_dependency();

    constexpr int kRows = S::kRows;
    const int tiles_m = (a.M + kRows - 1) / kRows, tiles_n = (a.N + TN - 1) / TN, tiles = tiles_m * tiles_n;
    const int blocks_k = (a.K + kTileK - 1) / kTileK, splits = PAIR ? 1 : a.splits;
    const int k0 = PAIR ? 0 : (int)((long long)blocks_k * rank / splits), k1 = PAIR ? blocks_k : (int)((long long)blocks_k * (rank + 1) / splits);
    const int first = (int)blockIdx.x / (PAIR ? 2 : splits), step = (int)gridDim.x / (PAIR ? 2 : splits);
    auto place = [&](int tile, int &m0, int &n0) {
        const int group = tile / (kTileGroup * tiles_n), in = tile % (kTileGroup * tiles_n), rows = min(kTileGroup, tiles_m - group * kTileGroup);
        m0 = (group * kTileGroup + in % rows) * kRows + (PAIR ? (int)rank * S::kOwnRows : 0);
        n0 = in / rows * TN;
    };

    if (warp == 0 && lane == 0) {
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
            int m0, n0;
            place(tile, m0, n0);
            if (PAIR) n0 += (int)rank * S::kOwnN;
            for (int kb = k0; kb < k1; ++kb) {
                ok = mbar_wait_one(&empty[stage], phase ^ 1, &gave_up);
                if (!ok) break;
                uint8_t *const at = smem + stage * S::kStageBytes;
                if (!PAIR || rank == 0) mbar_arrive_expect_tx(&full[stage], (PAIR ? 2 : 1) * S::kStageBytes);
                const uint32_t bar = PAIR ? peer_addr(&full[stage], 0) : 0;
                auto load = [&](uint8_t *to, const CUtensorMap *map, int x, int row) {
                    if constexpr (PAIR) tma_load_2d_pair(to, map, x, row, bar);
                    else tma_load_2d(to, map, x, row, &full[stage]);
                };
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
                    if constexpr (S::kStacked) {
                        load(at, &map_a, kb * kTileK, m0);
                        load(at + S::kABytes / 2, &map_a, kb * kTileK, m0 + a.half);
                    } else if constexpr (S::kAAcross) {
                        load(at, &map_a, m0, kb * kTileK);
                        load(at + S::kABytes / 2, &map_a, m0 + 64, kb * kTileK);
                    } else {
                        load(at + p * S::kABytes, &map_a, kb * kTileK, m0 + p * a.half);
                    }
                }
                if constexpr (S::kBAcross) {
#pragma unroll
                    for (int j = 0; j < S::kBRows; j += 64) load(at + kParts * S::kABytes + j * kTileK * 2, &map_b, n0 + j, kb * kTileK);
                } else {
                    load(at + S::kABytes, &map_b, kb * kTileK, n0);
                }
                ++issued;
                if (++stage == kStages) { stage = 0; phase ^= 1; }
            }
        }
        // what is under way, for either CTA of a pair, lands before they leave, also where a wait has run out
        if (!PAIR || rank == 0)
            for (int b = issued > kStages ? issued - kStages : 0; b < issued; ++b)
                mbar_wait_some(&full[b % kStages], (uint32_t)(b / kStages) & 1u, kDrainSpins);
    } else if (warp == 1 && lane == 0 && (!PAIR || rank == 0)) {
        constexpr uint32_t kInstr = mma_bf16_instruction(PAIR ? 2 * kTileM : kTileM, TN, S::kAAcross, S::kBAcross);
        constexpr uint32_t kHalfBox = 64 * kTileK * 2;                    // 64 rows along m or n of a stage
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
            for (int c = k0; c < k1 && ok;) {
                const int end = S::kPromote ? min(c + a.chunk, k1) : k1, begin = c;
                ok = mbar_wait_one(&acc_empty[acc], acc_phase ^ 1, &gave_up);
                if (!ok) break;
                tcgen05_fence_after();
                for (; c < end; ++c) {
                    ok = mbar_wait_one(&full[stage], phase, &gave_up);
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint32_t at = smem_addr(smem + stage * S::kStageBytes), bt = at + kParts * S::kABytes;
                    const uint64_t db = S::kBAcross ? smem_descriptor_128b_across(bt, kHalfBox) : smem_descriptor_128b(bt);
#pragma unroll
                    for (int p = 0; p < kParts; ++p) {
                        const uint64_t da = S::kAAcross ? smem_descriptor_128b_across(at, kHalfBox) : smem_descriptor_128b(at + p * S::kABytes);
#pragma unroll
                        for (int k = 0; k < kTileK / 16; ++k)
                            mma_bf16<PAIR>(tmem + acc * S::kAccColumns + p * TN, da + k * (S::kAAcross ? 128 : 2), db + k * (S::kBAcross ? 128 : 2), kInstr, c > begin || k > 0);
                    }
                    if constexpr (PAIR) tcgen05_commit_pair(&empty[stage]);
                    else tcgen05_commit(&empty[stage]);
                    if (++stage == kStages) { stage = 0; phase ^= 1; }
                }
                if (!ok) break;
                if constexpr (PAIR) tcgen05_commit_pair(&acc_full[acc]);
                else tcgen05_commit(&acc_full[acc]);
                if (++acc == kAcc) { acc = 0; acc_phase ^= 1; }
            }
        }
        // no product is under way when the TMEM goes back
        if constexpr (PAIR) tcgen05_commit_pair_own(&drained);
        else tcgen05_commit(&drained);
        mbar_wait_some(&drained, 0, kDrainSpins);
    } else if (warp >= 2) {
        const int part = warp & 3, c0 = (warp - 2) / 4 * S::kWarpColumns;  // the lanes of TMEM that this warp may read, its first column
        uint4 *const stage_out = reinterpret_cast<uint4 *>(smem + kStages * S::kStageBytes + (warp - 2) * S::kOutBytes);
        uint8_t *const cross = smem + kStages * S::kStageBytes + S::kWarps * S::kOutBytes;
        const int cross_pair = (warp - 2) / 4 * 2 + (part & 1), lower = part < 2;
        int acc = 0, turn = 0;
        uint32_t acc_phase = 0;
        const uint32_t arrive = PAIR ? peer_addr(&acc_empty[0], 0) : smem_addr(&acc_empty[0]);
        auto give_back = [&] {
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(arrive + acc * 8);
                else mbar_arrive(&acc_empty[acc]);
            }
            if (++acc == kAcc) { acc = 0; acc_phase ^= 1; }
        };
        for (int tile = first; tile < tiles; tile += step) {
            int m0, n0;
            place(tile, m0, n0);
            // what a lane has is a row; the epilogue's inputs of its first columns are on their way before the sums are there
            const int m = m0 + (S::kStacked ? part & 1 : part) * 32, row = min(m + lane, a.M - 1);
            float bias[2] = {0.0f, 0.0f};
            if (KIND <= kGated && a.bias) {
                bias[0] = a.bias[S::kStacked && !lower ? a.half + row : row];
                if (KIND == kGated && !S::kStacked) bias[1] = a.bias[a.half + row];
            }
            constexpr bool kExtra = sizeof(T) == 2 && (KIND == kForward || KIND == kInputGrad);
            uint4 extra[2][kPiece / 8];
            const bool has_extra = kExtra && a.extra && splits == 1 && c0 < TN;
            auto fetch_extra = [&](int i) {
                const int n = n0 + c0 + i;
                if (!has_extra || i >= S::kWarpColumns || n >= a.N) return;
                const __nv_bfloat16 *const p = static_cast<const __nv_bfloat16 *>(a.extra) + m * a.extra_stride + n;
                load_rows(extra[0], p, a.extra_stride, a.M - m, a.N - n, a.vec);
                if (KIND == kInputGrad && a.gated) load_rows(extra[1], p + a.half * a.extra_stride, a.extra_stride, a.M - m, a.N - n, a.vec);
            };
            fetch_extra(0);
            float sums[S::kPromote ? S::kWarpColumns : 1];
            bool ok = true;
            if constexpr (S::kPromote) {
#pragma unroll
                for (int i = 0; i < S::kWarpColumns; ++i) sums[i] = 0.0f;
                for (int c = k0; c < k1; c += a.chunk) {
                    ok = mbar_wait_warp(&acc_full[acc], acc_phase, &gave_up);
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint32_t at = tmem + ((uint32_t)(part * 32) << 16) + acc * S::kAccColumns + c0;
                    if (c0 < TN) {
#pragma unroll
                        for (int i = 0; i < S::kWarpColumns; i += kPiece) {
                            int v[kPiece];
                            tmem_load(at + i, v);
#pragma unroll
                            for (int j = 0; j < kPiece; ++j) sums[i + j] += __int_as_float(v[j]);
                        }
                    }
                    give_back();
                }
            } else {
                ok = mbar_wait_warp(&acc_full[acc], acc_phase, &gave_up);
                tcgen05_fence_after();
            }
            if (!ok) break;
            const uint32_t at = tmem + ((uint32_t)(part * 32) << 16) + acc * S::kAccColumns + c0;
            if (splits > 1) {
                // the stages are free: the tile's last product is done, and with it everything that read them
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
                    float *const to = reinterpret_cast<float *>(smem) + ((p * kTileM) + part * 32 + lane) * (TN + 4) + c0;
                    if (c0 < TN) {
#pragma unroll
                        for (int i = 0; i < S::kWarpColumns; i += kPiece) {
                            int v[kPiece];
                            if constexpr (S::kPromote) {
#pragma unroll
                                for (int j = 0; j < kPiece; ++j) v[j] = __float_as_int(sums[i + j]);
                            } else {
                                tmem_load(at + p * TN + i, v);
                            }
#pragma unroll
                            for (int j = 0; j < kPiece; j += 4) *reinterpret_cast<int4 *>(to + i + j) = make_int4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                        }
                    }
                }
                if constexpr (!S::kPromote) give_back();
                continue;
            }
            bool returned = S::kPromote;
            // (rolled where no registers are indexed: unrolled four times the epilogue's instructions do not stay in their cache)
#pragma unroll (S::kPromote ? S::kWarpColumns / kPiece : 1)
            for (int i = 0; i < S::kWarpColumns; i += kPiece) {
                const int n = n0 + c0 + i, left = a.N - n, rows = a.M - m;
                if (c0 >= TN || left <= 0) break;
                int v[kPiece], w[KIND == kGated ? kPiece : 1];
                if constexpr (S::kPromote) {
#pragma unroll
                    for (int j = 0; j < kPiece; ++j) v[j] = __float_as_int(sums[i + j]);
                } else {
                    tmem_load(at + i, v);
                    if constexpr (KIND == kGated && !S::kStacked) tmem_load(at + TN + i, w);
                    if (i + kPiece >= S::kWarpColumns || left <= kPiece) {        // the last of its columns: the next tile's products may have them
                        give_back();
                        returned = true;
                    }
                }
                uint4 out[kPiece / 8];
                // a number of each of the columns, made eight at a time: f(column) -> float
                auto made = [&](auto f) {
#pragma unroll
                    for (int q = 0; q < kPiece / 8; ++q) {
                        float r[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) r[j] = f(8 * q + j);
                        out[q] = pack<__nv_bfloat16>(r);
                    }
                };
                auto extra_of = [&](int which, int j) {
                    const uint32_t word = reinterpret_cast<const uint32_t *>(extra[which])[j / 2];
                    return __uint_as_float(j % 2 ? word & 0xffff0000u : word << 16);
                };
                __nv_bfloat16 *const z_base = KIND <= kGated && a.z_out ? static_cast<__nv_bfloat16 *>(a.z_out) + m * a.z_stride + n : nullptr;
                T *const base = static_cast<T *>(a.out) + m * a.out_stride + n;
                if constexpr (KIND == kForward) {
                    if (a.bias) {
#pragma unroll
                        for (int j = 0; j < kPiece; ++j) v[j] = __float_as_int(__int_as_float(v[j]) + bias[0]);
                    }
                    if (z_base) {
                        made([&](int j) { return __int_as_float(v[j]); });
                        store_rows(stage_out, out, z_base, a.z_stride, rows, left, a.vec);
                    }
                    with_activation(a.act, [&](auto act) {
#pragma unroll
                        for (int j = 0; j < kPiece; ++j) v[j] = __float_as_int(curve<decltype(act)::value, sizeof(T) == 2>(__int_as_float(v[j])).value);
                    });
                }
                if constexpr (sizeof(T) == 4) {
                    float r[kPiece];
#pragma unroll
                    for (int j = 0; j < kPiece; ++j) r[j] = __int_as_float(v[j]);
                    store_rows(stage_out, r, base, a.out_stride, a.extra ? static_cast<const float *>(a.extra) + m * a.extra_stride + n : nullptr, a.extra_stride,
                                  a.accumulate, rows, left, a.vec);
                } else if constexpr (KIND == kForward) {
                    if (a.extra) spread_rows(stage_out, extra[0], a.vec);
                    if (a.extra) made([&](int j) { return __int_as_float(v[j]) + extra_of(0, j); });
                    else made([&](int j) { return __int_as_float(v[j]); });
                    fetch_extra(i + kPiece);
                    store_rows(stage_out, out, base, a.out_stride, rows, left, a.vec);
                } else if constexpr (S::kStacked) {
                    if (a.bias) {
#pragma unroll
                        for (int j = 0; j < kPiece; ++j) v[j] = __float_as_int(__int_as_float(v[j]) + bias[0]);
                    }
                    const int b = turn & 1;
                    const uint32_t phase = turn >> 1 & 1;
                    uint4 *const at_cross = reinterpret_cast<uint4 *>(cross + (cross_pair * 2 + b) * 32 * kPiece * 4);
                    ++turn;
                    if (!lower) {
                        ok = mbar_wait_warp(&cross_empty[cross_pair][b], phase ^ 1, &gave_up);
                        if (!ok) break;
#pragma unroll
                        for (int q = 0; q < kPiece / 4; ++q)
                            at_cross[staged_piece<kPiece / 4>(lane, q)] = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&cross_full[cross_pair][b]);
                        if (z_base) {
                            made([&](int j) { return __int_as_float(v[j]); });
                            store_rows(stage_out, out, z_base + a.half * a.z_stride, a.z_stride, rows, left, a.vec);
                        }
                    } else {
                        ok = mbar_wait_warp(&cross_full[cross_pair][b], phase, &gave_up);
                        if (!ok) break;
#pragma unroll
                        for (int q = 0; q < kPiece / 4; ++q) {
                            const uint4 p = at_cross[staged_piece<kPiece / 4>(lane, q)];
                            w[4 * q] = (int)p.x; w[4 * q + 1] = (int)p.y; w[4 * q + 2] = (int)p.z; w[4 * q + 3] = (int)p.w;
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&cross_empty[cross_pair][b]);
                        with_activation(a.act, [&](auto act) { made([&](int j) { return curve<decltype(act)::value, sizeof(T) == 2>(__int_as_float(v[j])).value * __int_as_float(w[j]); }); });
                        store_rows(stage_out, out, base, a.out_stride, rows, left, a.vec);
                        if (z_base) {
                            made([&](int j) { return __int_as_float(v[j]); });
                            store_rows(stage_out, out, z_base, a.z_stride, rows, left, a.vec);
                        }
                    }
                } else if constexpr (KIND == kGated) {
                    if (a.bias) {
#pragma unroll
                        for (int j = 0; j < kPiece; ++j) {
                            v[j] = __float_as_int(__int_as_float(v[j]) + bias[0]);
                            w[j] = __float_as_int(__int_as_float(w[j]) + bias[1]);
                        }
                    }
                    with_activation(a.act, [&](auto act) { made([&](int j) { return curve<decltype(act)::value, sizeof(T) == 2>(__int_as_float(v[j])).value * __int_as_float(w[j]); }); });
                    store_rows(stage_out, out, base, a.out_stride, rows, left, a.vec);
                    if (z_base) {
                        made([&](int j) { return __int_as_float(v[j]); });
                        store_rows(stage_out, out, z_base, a.z_stride, rows, left, a.vec);
                        made([&](int j) { return __int_as_float(w[j]); });
                        store_rows(stage_out, out, z_base + a.half * a.z_stride, a.z_stride, rows, left, a.vec);
                    }
                } else if (a.gated) {
                    spread_rows(stage_out, extra[0], a.vec);
                    spread_rows(stage_out, extra[1], a.vec);
                    uint4 up[kPiece / 8];
                    with_activation(a.act, [&](auto act) {
#pragma unroll
                        for (int q = 0; q < kPiece / 8; ++q) {
                            float d[8], e[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const Curve k = curve<decltype(act)::value, sizeof(T) == 2>(extra_of(0, 8 * q + j));
                                const float s = __int_as_float(v[8 * q + j]);
                                d[j] = s * (extra_of(1, 8 * q + j) * k.slope);
                                e[j] = s * k.value;
                            }
                            out[q] = pack<__nv_bfloat16>(d);
                            up[q] = pack<__nv_bfloat16>(e);
                        }
                    });
                    fetch_extra(i + kPiece);
                    store_rows(stage_out, out, base, a.out_stride, rows, left, a.vec);
                    store_rows(stage_out, up, base + a.half * a.out_stride, a.out_stride, rows, left, a.vec);
                } else {
                    if (a.extra) spread_rows(stage_out, extra[0], a.vec);
                    if (a.extra) with_activation(a.act, [&](auto act) { made([&](int j) { return __int_as_float(v[j]) * curve<decltype(act)::value, sizeof(T) == 2>(extra_of(0, j)).slope; }); });
                    else made([&](int j) { return __int_as_float(v[j]); });
                    fetch_extra(i + kPiece);
                    store_rows(stage_out, out, base, a.out_stride, rows, left, a.vec);
                }
            }
            if (!ok) break;
            if (!returned) give_back();
        }
    }
    if (!PAIR && splits > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp >= 2 && !gave_up) {
            // a cluster has one tile; each of its CTAs finishes some of the rows
            int m0, n0;
            place(first, m0, n0);
            const int rows = kTileM / splits, r0 = (int)rank * rows;
            for (int e = threadIdx.x - 64; e < rows * (TN / 8); e += S::kThreads - 64) {
                const int r = r0 + e / (TN / 8), c = e % (TN / 8) * 8;
                if (m0 + r >= a.M || n0 + c >= a.N) continue;
                float s[2][8];
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
                    const uint32_t own = smem_addr(reinterpret_cast<float *>(smem) + (p * kTileM + r) * (TN + 4) + c);
                    int4 lo[kMostSplits], hi[kMostSplits];
#pragma unroll
                    for (int q = 0; q < kMostSplits; ++q)                   // all of them under way at a time
                        if (q < splits) { lo[q] = peer_load_v4(own, (uint32_t)q); hi[q] = peer_load_v4(own + 16, (uint32_t)q); }
#pragma unroll
                    for (int j = 0; j < 8; ++j) s[p][j] = 0.0f;
#pragma unroll
                    for (int q = 0; q < kMostSplits; ++q)
                        if (q < splits) {
                            s[p][0] += __int_as_float(lo[q].x); s[p][1] += __int_as_float(lo[q].y); s[p][2] += __int_as_float(lo[q].z); s[p][3] += __int_as_float(lo[q].w);
                            s[p][4] += __int_as_float(hi[q].x); s[p][5] += __int_as_float(hi[q].y); s[p][6] += __int_as_float(hi[q].z); s[p][7] += __int_as_float(hi[q].w);
                        }
                }
                finish_8<KIND, T>(a, m0 + r, n0 + c, s[0], s[kParts - 1]);
            }
        }
        __syncwarp();
        cluster_arrive();                                                 // nobody leaves while its sums may still be read
        cluster_wait();
    }
    __syncwarp();
    tcgen05_fence_before();
    if constexpr (PAIR) { cluster_arrive(); cluster_wait(); } else __syncthreads();
    tcgen05_fence_after();
    if (warp == 1) {
        if constexpr (PAIR) tmem_free_pair(tmem, S::kColumns);
        else tmem_free(tmem, S::kColumns);
    }
    if (threadIdx.x == 0 && gave_up) atomicCAS(a.fault, 0, kFaultBarrierTimeout);
}

// db = or += the sums of the rows of dy: a warp or a CTA of 8 a row, 16 bytes a lane, four of them under way
template <int W> __global__ void __launch_bounds__(256)
k_dense_bias_grad(const __nv_bfloat16 *__restrict__ dy, float *db, int O, int F, long long stride, int accumulate)
{
    grid_dependency();
    static_assert(W == 1 || W == 8, "a row is a warp's or a CTA's");
    const int lane = threadIdx.x & 31, warp = (int)threadIdx.x >> 5, part = warp % W, o = ((int)blockIdx.x * 8 + warp) / W;
    const __nv_bfloat16 *const row = dy + (long long)o * stride;
    float sum[8] = {};
    const unsigned whole = (unsigned)F & ~7u;
    constexpr unsigned step = W * 256;
    if (o < O)
        for (unsigned at = part * 256 + lane * 8; at < whole; at += 4 * step) {
            uint4 raw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[i] = at + i * step < whole ? *reinterpret_cast<const uint4 *>(row + at + i * step) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[8];
                unpack<__nv_bfloat16>(raw[i], v);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j] += v[j];
            }
        }
    if (o < O && part == 0 && lane < F - (int)whole) sum[0] += to_float(row[whole + lane]);
#pragma unroll
    for (int j = 1; j < 8; ++j) sum[0] += sum[j];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], d);
    if constexpr (W > 1) {
        __shared__ float s_sum[W];
        if (lane == 0) s_sum[warp] = sum[0];
        __syncthreads();
        for (int i = 1; i < W; ++i) sum[0] += s_sum[i];
    }
    if (o < O && part == 0 && lane == 0) db[o] = accumulate ? db[o] + sum[0] : sum[0];
}

// dW = db = 0 of a batch without frames
__global__ void __launch_bounds__(256) k_dense_no_frames(float *dW, float *db, int I, long long stride)
{
    grid_dependency();
    for (int i = threadIdx.x; i < I; i += 256)
        if (dW) dW[(long long)blockIdx.x * stride + i] = 0.0f;
    if (threadIdx.x == 0 && db) db[blockIdx.x] = 0.0f;
}

// ---- host side
struct Operand { const __nv_bfloat16 *p; long long size, rows, stride; };     // rows of `size` elements

template <int KIND, typename T, int TN, bool PAIR>
static int dense_tiles(const Operand &A, const Operand &B, const DenseArgs &a, cudaStream_t st)
{
    using S = DenseShape<KIND, T, TN, PAIR>;
    const TensorMapEncode encode = tensor_map_encode();
    BB200_REQUIRE(encode != nullptr, BBCU_ERR_NO_DEVICE);
    CUtensorMap map_a, map_b;
    auto map = [&](CUtensorMap *m, const Operand &o, int box_rows) {
        return tensor_map_rows(encode, m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, o.p, o.size, o.rows, o.stride * 2, box_rows) == CUDA_SUCCESS;
    };
    BB200_REQUIRE(map(&map_a, A, S::kAAcross ? kTileK : S::kOwnRows) && map(&map_b, B, S::kBAcross ? kTileK : S::kBRows), (int)cudaErrorInvalidValue);
    const long long tiles = ((long long)a.M + S::kRows - 1) / S::kRows * (((long long)a.N + TN - 1) / TN), sms = device_info().sm_count;
    BB200_REQUIRE(tiles < (1LL << 27), BBCU_ERR_TOO_LARGE);
    auto kernel = k_dense_tiles<KIND, T, TN, PAIR>;
    BB200_REQUIRE(allow_big_smem(kernel, S::kSmem), (int)cudaErrorInvalidValue);
    const unsigned cluster = PAIR ? 2u : (unsigned)a.splits;
    const long long slots = PAIR ? sms / 2 : sms;
    const unsigned grid = cluster * (unsigned)(!PAIR && a.splits > 1 ? tiles : tiles < slots ? tiles : slots);
    return launch_cluster(kernel, cluster, grid, S::kThreads, S::kSmem, st, map_a, map_b, a);
}

// The tensor cores cut the digits that do not fit their running sum, which drifts towards zero by 0.0154 half-units in the last place a term; fp32 outputs are taken
// out of them after every so many stages of k and added up in registers.  A 32-bit sum term after term is off by 0.3 sqrt(K) of those, a library's product, which has
// several sums, by 0.12 to 0.18 sqrt(K).  An output gets the second, 8 sqrt(K) terms at a time (0.12); a gradient, which is the time of a training step, the first,
// 16 sqrt(K) terms (0.25), since taking sums out stands in the products' way in TMEM: by 8 sqrt(K), 16 sqrt(K) and 768 terms dW of 4096 x 4096 x 2048 88, 76, 76 us,
// of 2000 x 5500 x 3001 84, 78, 78; y of 1024 x 4096 x 4096 64 us by 8 sqrt(K), 53 by 768 terms, its error 2.3e-7 and 6.4e-7, a library's in fp32 2.5e-7.
// At most 12 stages (dW of 4096 x 4096 x 8192 246, 239, 236 us at 8, 12, 16).
static int sums_chunk(int K, int terms_a_root) { return std::max(1, std::min(12, (int)std::lround(std::sqrt((double)K) * terms_a_root / kTileK))); }

// Columns a tile (0: by a pair of CTAs) and CTAs that share the k of one, by what they take in nanoseconds, measured with one tile an SM: a stage of k 325 whatever the
// columns (a CTA's 24 to 32 KB come at about 50 bytes a clock; both products of a gated block 505), by a pair 410; to start and to store 3700 and some for
// each column, by a pair 7000; to join sums in a cluster 1500 and more for columns and CTAs.  A cluster has one tile, so that there are no more of them than
// the device holds (clusters of eight: fewer than its SMs would make; 1024 x 1024 x 64 7.5 us by four CTAs, 12.9 where 16 clusters of eight took two rounds).
// Of 36 shapes from 420 x 70 x 512 to 4096 x 4096 x 1000 the choice is within 3 % of the best one, two within 9 %.
struct DenseTiles { int columns, splits; };
static DenseTiles choose_dense_tiles(int M, int N, int K, int parts, const int (&clusters)[4])
{
    const long long sms = device_info().sm_count, blocks = (K + kTileK - 1) / kTileK, tiles_m = ((long long)M + kTileM - 1) / kTileM;
    const long long pair_rows = parts == 2 ? kTileM : 2 * kTileM, pair_tiles = (M + pair_rows - 1) / pair_rows * (((long long)N + 255) / 256);
    DenseTiles best = {0, 1};
    long long least = (pair_tiles + sms / 2 - 1) / (sms / 2) * blocks * 410 + 7000;
    for (int columns = 32; columns <= 128; columns *= 2) {
        const long long tiles = tiles_m * (((long long)N + columns - 1) / columns);
        for (int splits = 1, i = 0; splits <= kMostSplits; splits *= 2, ++i) {
            if (splits > 1 && (tiles > clusters[i] || blocks < 2 * splits)) break;
            const long long rounds = splits > 1 ? 1 : (tiles + sms - 1) / sms;
            const long long cost = rounds * ((blocks + splits - 1) / splits) * (parts == 2 ? 505 : 325) + 3700 + columns * (parts == 2 ? 14 : 6) + (rounds - 1) * 8 * columns * parts +
                                   (splits > 1 ? 1500 + (splits > 2 ? 26 : 14) * columns * parts : 0);
            if (cost < least) { least = cost; best = {columns, splits}; }
        }
    }
    return best;
}

template <int KIND, typename T> static int dense_product(const Operand &A, const Operand &B, DenseArgs &a, cudaStream_t st)
{
    a.fault = fault_word();
    BB200_REQUIRE(a.fault != nullptr, BBCU_ERR_NO_DEVICE);
    int clusters[4];
    using S = DenseShape<KIND, T, 64, false>;
    auto kernel = k_dense_tiles<KIND, T, 64, false>;
    BB200_REQUIRE(allow_big_smem(kernel, S::kSmem), (int)cudaErrorInvalidValue);
    for (int i = 0; i < 4; ++i) clusters[i] = resident_clusters(reinterpret_cast<const void *>(kernel), 1 << i, S::kThreads, S::kSmem);
    const DenseTiles t = choose_dense_tiles(a.M, a.N, a.K, KIND == kGated ? 2 : 1, clusters);
    a.splits = t.splits;
    a.chunk = sums_chunk(a.K, KIND == kWeightGrad ? 16 : 8);
    switch (t.columns) {
    case 32: return dense_tiles<KIND, T, 32, false>(A, B, a, st);
    case 64: return dense_tiles<KIND, T, 64, false>(A, B, a, st);
    case 128: return dense_tiles<KIND, T, 128, false>(A, B, a, st);
    default: return dense_tiles<KIND, T, 256, true>(A, B, a, st);
    }
}

template <int KIND, typename T> static int dense_few(const __nv_bfloat16 *x, const __nv_bfloat16 *W, long long xs, long long ws, DenseArgs &a, cudaStream_t st)
{
    const int ctas = std::min(a.M, device_info().sm_count), rows = (a.M + ctas - 1) / ctas;
    int groups = 1;
    while (groups < kFewThreads / 32 && rows > 16 * groups) groups *= 2;
    const int chunk = std::min(few_chunk(a.N), (a.K + 31) / 32 * 32), smem = (a.N * (chunk + 8) + 8) * 2;
    a.chunk = sums_chunk(a.K, 8);
    auto kernel = k_dense_few<KIND, T>;
    BB200_REQUIRE(allow_big_smem(kernel, (kFewInputs + 9 * 8) * 2), (int)cudaErrorInvalidValue);
    launch(kernel, (unsigned)ctas, kFewThreads, (size_t)smem, st, x, W, xs, ws, a, groups, chunk);
    return launch_status();
}

// Sums for 16-bit outputs are not taken out on the way.  What the tensor cores cut of them stays below a tenth of a half step of bf16 up to 2^20 terms (1.4e-4
// of 2e-3; 4.6e-3 at 2^22).
constexpr int kMostExtent = 1 << 27, kMostCutTerms = 1 << 20;

// 2: rows on 32-byte boundaries, 1: on 16-byte ones
template <typename T> static int alignment(const T *p, long long stride)
{
    const unsigned long long both = reinterpret_cast<uintptr_t>(p) | (unsigned long long)(stride * (long long)sizeof(T));
    return both % 32 == 0 ? 2 : both % 16 == 0 ? 1 : 0;
}

static bool rows_on_16(const void *p, long long stride) { return frames_aligned<__nv_bfloat16>(p, stride); }

template <typename T>
static int dense_forward(bool gated, const bbcu_bf16_t *x_, const bbcu_bf16_t *W_, const float *bias, const T *residual, T *y, bbcu_bf16_t *z, int activation, int K, int O,
                         int F, int ws, int xs, int rs, int ys, int zs, bbcu_stream_t stream)
{
    const auto *x = reinterpret_cast<const __nv_bfloat16 *>(x_), *W = reinterpret_cast<const __nv_bfloat16 *>(W_);
    BB200_REQUIRE(K > 0 && O >= 0 && F >= 0 && activation >= BBCU_ACTIVATION_NONE && activation <= BBCU_ACTIVATION_SILU, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(K <= (sizeof(T) == 2 ? kMostCutTerms : kMostExtent) && O <= kMostExtent && F <= kMostExtent, BBCU_ERR_TOO_LARGE);
    BB200_REQUIRE(ws >= K && xs >= F && ys >= F && (!residual || rs >= F) && (!z || zs >= F) && rows_on_16(W, ws) && rows_on_16(x, xs), BBCU_ERR_BAD_STRIDE);
    if (F == 0 || O == 0) return BBCU_OK;
    BB200_REQUIRE_PTR(x); BB200_REQUIRE_PTR(W); BB200_REQUIRE_PTR(y);
    DenseArgs a{};
    a.bias = bias; a.extra = residual; a.out = y; a.z_out = z; a.act = activation;
    a.M = O; a.N = F; a.K = K; a.half = O; a.splits = 1;
    a.extra_stride = rs; a.out_stride = ys; a.z_stride = zs;
    a.vec = std::min({alignment(y, ys), residual ? alignment(residual, rs) : 2, z ? alignment(reinterpret_cast<const __nv_bfloat16 *>(z), zs) : 2});
    cudaStream_t st = as_stream(stream);
    const Operand A = {W, K, gated ? 2LL * O : O, ws}, B = {x, F, K, xs};
    if constexpr (sizeof(T) == 2) {
        if (gated) return F <= kFewFrames ? dense_few<kGated, T>(x, W, xs, ws, a, st) : dense_product<kGated, T>(A, B, a, st);
    }
    return F <= kFewFrames ? dense_few<kForward, T>(x, W, xs, ws, a, st) : dense_product<kForward, T>(A, B, a, st);
}

}   // namespace bb200

using namespace bb200;

extern "C" int bbcu_bf16_DenseAffine_Forward(const bbcu_bf16_t *x, const bbcu_bf16_t *W, const float *bias, const bbcu_bf16_t *residual, bbcu_bf16_t *y, bbcu_bf16_t *z,
                                             int activation, int input_node_size, int output_node_size, int frame_size, int w_node_stride, int x_frame_stride,
                                             int residual_frame_stride, int y_frame_stride, int z_frame_stride, bbcu_stream_t stream)
{
    return dense_forward<__nv_bfloat16>(false, x, W, bias, reinterpret_cast<const __nv_bfloat16 *>(residual), reinterpret_cast<__nv_bfloat16 *>(y), z, activation,
                                        input_node_size, output_node_size, frame_size, w_node_stride, x_frame_stride, residual_frame_stride, y_frame_stride,
                                        z_frame_stride, stream);
}

extern "C" int bbcu_bf16_fp32_DenseAffine_Forward(const bbcu_bf16_t *x, const bbcu_bf16_t *W, const float *bias, const float *residual, float *y, bbcu_bf16_t *z,
                                                  int activation, int input_node_size, int output_node_size, int frame_size, int w_node_stride, int x_frame_stride,
                                                  int residual_frame_stride, int y_frame_stride, int z_frame_stride, bbcu_stream_t stream)
{
    return dense_forward<float>(false, x, W, bias, residual, y, z, activation, input_node_size, output_node_size, frame_size, w_node_stride, x_frame_stride,
                                residual_frame_stride, y_frame_stride, z_frame_stride, stream);
}

extern "C" int bbcu_bf16_GatedDense_Forward(const bbcu_bf16_t *x, const bbcu_bf16_t *W, const float *bias, bbcu_bf16_t *y, bbcu_bf16_t *z, int activation, int input_node_size,
                                            int output_node_size, int frame_size, int w_node_stride, int x_frame_stride, int y_frame_stride, int z_frame_stride,
                                            bbcu_stream_t stream)
{
    return dense_forward<__nv_bfloat16>(true, x, W, bias, nullptr, reinterpret_cast<__nv_bfloat16 *>(y), z, activation, input_node_size, output_node_size, frame_size,
                                        w_node_stride, x_frame_stride, 0, y_frame_stride, z_frame_stride, stream);
}

extern "C" int bbcu_bf16_DenseAffine_BackwardInput(const bbcu_bf16_t *dy_, const bbcu_bf16_t *W_, const bbcu_bf16_t *z, bbcu_bf16_t *dx, int activation, int gated,
                                                   int input_node_size, int output_node_size, int frame_size, int w_node_stride, int dy_frame_stride,
                                                   int z_frame_stride, int dx_frame_stride, bbcu_stream_t stream)
{
    const auto *dy = reinterpret_cast<const __nv_bfloat16 *>(dy_), *W = reinterpret_cast<const __nv_bfloat16 *>(W_);
    const int I = input_node_size, O = output_node_size, F = frame_size;
    BB200_REQUIRE(I >= 0 && O > 0 && F >= 0 && activation >= BBCU_ACTIVATION_NONE && activation <= BBCU_ACTIVATION_SILU, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(I <= kMostExtent && O <= kMostCutTerms && F <= kMostExtent, BBCU_ERR_TOO_LARGE);
    BB200_REQUIRE(w_node_stride >= I && dy_frame_stride >= F && dx_frame_stride >= F && (!z || z_frame_stride >= F) && rows_on_16(W, w_node_stride) &&
                  rows_on_16(dy, dy_frame_stride), BBCU_ERR_BAD_STRIDE);
    if (F == 0 || I == 0) return BBCU_OK;
    BB200_REQUIRE_PTR(dy); BB200_REQUIRE_PTR(W); BB200_REQUIRE_PTR(dx);
    if (gated) BB200_REQUIRE_PTR(z);
    DenseArgs a{};
    a.extra = z; a.out = dx; a.act = activation; a.gated = gated != 0;
    a.M = I; a.N = F; a.K = O; a.half = I; a.splits = 1;
    a.extra_stride = z_frame_stride; a.out_stride = dx_frame_stride;
    a.vec = std::min(alignment(reinterpret_cast<const __nv_bfloat16 *>(dx), dx_frame_stride), z ? alignment(reinterpret_cast<const __nv_bfloat16 *>(z), z_frame_stride) : 2);
    return dense_product<kInputGrad, __nv_bfloat16>({W, I, O, w_node_stride}, {dy, F, O, dy_frame_stride}, a, as_stream(stream));
}

extern "C" int bbcu_bf16_DenseAffine_BackwardWeights(const bbcu_bf16_t *x_, const bbcu_bf16_t *dy_, float *dW, float *dbias, int accumulate, int input_node_size,
                                                     int output_node_size, int frame_size, int x_frame_stride, int dy_frame_stride, int dw_node_stride,
                                                     bbcu_stream_t stream)
{
    const auto *x = reinterpret_cast<const __nv_bfloat16 *>(x_), *dy = reinterpret_cast<const __nv_bfloat16 *>(dy_);
    const int I = input_node_size, O = output_node_size, F = frame_size;
    BB200_REQUIRE(I > 0 && O >= 0 && F >= 0, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(I <= kMostExtent && O <= kMostExtent && F <= kMostExtent, BBCU_ERR_TOO_LARGE);
    BB200_REQUIRE(x_frame_stride >= F && dy_frame_stride >= F && (!dW || dw_node_stride >= I) && rows_on_16(x, x_frame_stride) && rows_on_16(dy, dy_frame_stride),
                  BBCU_ERR_BAD_STRIDE);
    if (O == 0 || (!dW && !dbias)) return BBCU_OK;
    cudaStream_t st = as_stream(stream);
    if (F == 0) {
        if (!accumulate) launch(k_dense_no_frames, (unsigned)O, 256, 0, st, dW, dbias, I, (long long)dw_node_stride);
        return launch_status();
    }
    BB200_REQUIRE_PTR(dy);
    if (dbias) {
        // A warp a row where that gives every SM two CTAs, or where a row has no more than a warp's four loads; else a CTA a row.  By the warp and
        // by the CTA: 4096 rows x 1000 frames 2 and 7 us, 4096 x 8192 9 and 10, 1024 x 8192 4 and 3, 64 x 65536 24 and 4.
        if (O >= 16 * device_info().sm_count || F <= 1024)
            launch(k_dense_bias_grad<1>, (unsigned)((O + 7) / 8), 256, 0, st, dy, dbias, O, F, (long long)dy_frame_stride, accumulate);
        else launch(k_dense_bias_grad<8>, (unsigned)O, 256, 0, st, dy, dbias, O, F, (long long)dy_frame_stride, accumulate);
    }
    if (!dW) return launch_status();
    BB200_REQUIRE_PTR(x);
    DenseArgs a{};
    a.out = dW; a.accumulate = accumulate; a.act = BBCU_ACTIVATION_NONE;
    a.M = O; a.N = I; a.K = F; a.splits = 1;
    a.out_stride = dw_node_stride;
    a.vec = frames_aligned<float>(dW, dw_node_stride);
    return dense_product<kWeightGrad, float>({dy, F, O, dy_frame_stride}, {x, F, I, x_frame_stride}, a, st);
}
