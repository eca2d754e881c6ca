// Dense layer in 8-bit integers with a scale per frame and per output node, and the quantisers that make its operands.  (The reference's dense layers
// are fp32 through cuBLAS, include/bb/DenseAffine.h, and DepthwiseDenseAffineQuantize.h; it has no integer product.)
//
//   quantiser   per frame f of a frame buffer x[node][frame]: s = max_n |x| / 127,  q = rint(x / s) in [-127, 127], both in 32 bits, ties to even;
//               a frame of zeros has s = 0, one with a NaN or an infinity s = NaN, both q = 0.  The frames become rows, q[frame][node], 16-byte
//               pieces along the nodes, which is how the product reads both of its operands.  The channel form does the same to the rows of W[out][in].
//   product     y[o][f] = s_w[o] s_x[f] sum_k Wq[o][k] q[f][k] + bias[o],  the sum exact in 32-bit integers (at most 131071 inputs), y fp32 or bf16
#include <cuda.h>

#include "async_copy.cuh"
#include "frame_columns.cuh"
#include "tensor_core.cuh"

namespace bb200 {

constexpr int kQuantThreads = 256, kQuantRows = 256;      // rows of x that a CTA turns over
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

// Four numbers of a frame as a word of q.  x / scale comes through the reciprocal, off by less than 1e-4, and is rounded by adding 1.5 * 2^23, which
// leaves the integer in the lowest byte; where that could have decided the rounding, and for scales without a normal reciprocal, the quotient is divided
// out.  (The kernels are bound by their instructions, and the division costs more than all the rest.)
struct Quantizer {
    float scale, inv;
    bool plain;
    __device__ explicit Quantizer(float s) : scale(s), inv(1.0f / s), plain(s > 1e-36f && s < 1e36f) {}
    __device__ uint32_t operator()(float x0, float x1, float x2, float x3) const
    {
        constexpr float kRound = 12582912.0f;
        const float x[4] = {x0, x1, x2, x3};
        float worst = 0.0f;
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float t = x[i] * inv, n = t + kRound;
            worst = fmaxf(worst, fabsf(t - (n - kRound)));
            r[i] = __float_as_uint(n);
        }
        if (worst > 0.4999f || !plain) {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = (uint32_t)quantize(x[i], scale);
        }
        return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
    }
};

// the larger of the magnitudes of packed numbers, as integers: infinities and NaN are on top
template <typename T> __device__ __forceinline__ uint32_t packed_abs_max(uint32_t a, uint32_t b)
{
    return sizeof(T) == 4 ? max(a, b & 0x7fffffffu) : __vmaxu2(a, b & 0x7fff7fffu);
}

// A cluster has the columns of 128 (few frames: 32) bytes of a row; its CTAs take turns at the rows and join the largest magnitudes in the first CTA's shared memory.
template <typename T, int LPR, bool ALIGNED>
__global__ void __launch_bounds__(kQuantThreads, 4)
k_quantize_scale(const T *x, float *scale_out, int N, int F, long long xs)
{
    grid_dependency();
    constexpr int kBatch = 8;
    using Col = Column<T, LPR>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    __shared__ uint32_t red[8][kCols];
    __shared__ float part[kCols];
    const Col c;
    const uint32_t cl = cluster_size(), rank = cluster_rank();
    const int f0 = (int)(blockIdx.x / cl) * kCols, f = f0 + c.col, step = c.step * (int)cl;
    uint4 most = make_uint4(0, 0, 0, 0);
    for (int n = (int)rank * c.step + c.row; n < N; n += step * kBatch) {
        uint4 raw[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = n + i * step;
            raw[i] = m < N ? load_frames<T, ALIGNED>(x + (long long)m * xs, f, F) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            most.x = packed_abs_max<T>(most.x, raw[i].x); most.y = packed_abs_max<T>(most.y, raw[i].y);
            most.z = packed_abs_max<T>(most.z, raw[i].z); most.w = packed_abs_max<T>(most.w, raw[i].w);
        }
    }
    float v[kVec];
    unpack<T>(most, v);
    uint32_t top[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) top[j] = __float_as_uint(v[j]);
#pragma unroll
    for (int m = LPR; m < 32; m <<= 1)
#pragma unroll
        for (int j = 0; j < kVec; ++j) top[j] = max(top[j], __shfl_xor_sync(0xffffffffu, top[j], m));
    if (c.lane < LPR) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) red[c.warp][c.col + j] = top[j];
    }
    __syncthreads();
    uint32_t t = 0;
    if (threadIdx.x < kCols) {
        for (int w = 0; w < c.warps; ++w) t = max(t, red[w][threadIdx.x]);
        part[threadIdx.x] = __uint_as_float(t);
    }
    if (cl > 1) { cluster_arrive(); cluster_wait(); }
    if (rank == 0 && threadIdx.x < kCols && f0 + (int)threadIdx.x < F) {
        for (uint32_t r = 1; r < cl; ++r) t = max(t, __float_as_uint(peer_load(&part[threadIdx.x], r)));
        scale_out[f0 + threadIdx.x] = quant_scale(t);
    }
    if (cl > 1) { cluster_arrive(); cluster_wait(); }                     // nobody leaves while its part may still be read
}

// 256 rows x 128 bytes of x: a thread reads twice four neighbouring rows of its columns, so that four values of a frame are a word of q; the words cross
// through shared memory, in 16-byte pieces whose order differs from column to column so that no banks collide, and leave as lines of the frames' rows.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kQuantThreads)
k_quantize_apply(const T *x, int8_t *q, const float *__restrict__ scale_in, int N, int F, long long xs, long long qs)
{
    grid_dependency();
    constexpr int kLpr = 8, kPieces = kQuantRows / 16;
    using Col = Column<T, kLpr>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    __shared__ __align__(16) uint32_t tile[kCols][kQuantRows / 4];
    const Col c;
    const int f0 = (int)blockIdx.x * kCols, f = f0 + c.col, n0 = (int)blockIdx.y * kQuantRows, n = n0 + 4 * c.row;
    uint4 raw[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = n + 128 * h + i;
            raw[h][i] = m < N ? load_frames<T, ALIGNED>(x + (long long)m * xs, f, F) : make_uint4(0, 0, 0, 0);
        }
    float scale[kVec];
    load_columns(scale_in, f, F, scale);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float v[4][kVec];
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack<T>(raw[h][i], v[i]);
#pragma unroll
        for (int j = 0; j < kVec; ++j)
            tile[c.col + j][h * 32 + (c.row / 4 ^ c.lane % kLpr) * 4 + c.row % 4] = Quantizer(scale[j])(v[0][j], v[1][j], v[2][j], v[3][j]);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < kCols * kPieces; e += kQuantThreads) {
        const int col = e / kPieces, piece = e % kPieces, m = n0 + 16 * piece;
        if (f0 + col < F && m < N)
            *reinterpret_cast<uint4 *>(q + (long long)(f0 + col) * qs + m) = *reinterpret_cast<const uint4 *>(&tile[col][(piece ^ col / kVec) * 4]);
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

// Small calls in one launch: a cluster holds the columns of 64 bytes of a row in shared memory (see layer_norm.cu for the walk over the tiles), and a thread
// then takes 16 rows of a column, which are 16 bytes of q.
struct BitsMax { __device__ static float join(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); } };
constexpr int kQuantOnceRows = 16;
constexpr long long kQuantSmall = 1 << 18;                 // values (1020 x 200: 5.1 us, in two launches 8.4; 5000 x 70: 15.1 and 8.4)

template <typename T, int LPR>
__global__ void __launch_bounds__(kColumnThreads, 3)
k_quantize_once(const T *x, int8_t *q, float *scale_out, int N, int F, long long xs, long long qs, int rows, int tiles, int *fault)
{
    grid_dependency();
    using Col = Column<T, LPR>;
    constexpr int kVec = Col::kVec, kCols = Col::kCols;
    extern __shared__ __align__(16) uint8_t buffer[];
    __shared__ Exchange<1, kCols> tops[2];
    __shared__ int gave_up;
    const Col c;
    Cluster cl(&gave_up);
    const int clusters = (int)(gridDim.x / cl.size), cta_first = (int)cl.rank * c.step * rows, first = cta_first + c.row, piece = blockDim.x * 16;
    const int mine = min(rows, (N - first + c.step - 1) / c.step), cta_rows = min(c.step * rows, N - cta_first);
    const uint8_t *const at = buffer + threadIdx.x * 16;
    const long long x_step = c.step * xs;
    int tile = (int)(blockIdx.x / cl.size), f = tile * kCols + c.col;
    auto fetch = [&](int f) {
        if (f >= F) return;
        uint8_t *to = buffer + threadIdx.x * 16;
        const T *from = x + first * xs + f;
#pragma unroll 4
        for (int i = 0; i < mine; ++i, to += piece, from += x_step) cp_async16(to, from, true);
    };
    fetch(f);
    cl.meet(tops, buffer + rows * piece);
    uint32_t turn = 0;                                                    // the exchange is its lowest bit, the phase the next
    for (; tile < tiles; tile += clusters, f += clusters * kCols, ++turn) {
        cp_async_commit();
        cp_async_wait<0>();
        float top[1][kVec] = {};
        {
            const uint8_t *p = at;
#pragma unroll 4
            for (int i = 0; i < mine; ++i, p += piece) {
                float v[kVec];
                unpack<T>(*reinterpret_cast<const uint4 *>(p), v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) top[0][j] = BitsMax::join(top[0][j], fabsf(v[j]));
            }
        }
        Exchange<1, kCols> &e = tops[turn & 1];
        join_columns<BitsMax, 1, T, LPR>(top, c, e, cl, turn >> 1 & 1, [](int, float t) { return quant_scale(__float_as_uint(t)); });
        const int f0 = tile * kCols;
        if (cl.rank == 0 && threadIdx.x < kCols && f0 + (int)threadIdx.x < F) scale_out[f0 + threadIdx.x] = e.out[threadIdx.x];
        for (int i = threadIdx.x; i < (cta_rows + 15) / 16 * kCols; i += blockDim.x) {
            const int col = i % kCols, n = i / kCols * 16;
            if (f0 + col >= F) continue;
            const Quantizer quantize(e.out[col]);
            // (the distance between a thread's rows is a multiple of 16, so that the 16 are of one round)
            const uint8_t *const from = buffer + n / c.step * piece + (n % c.step * LPR + col / kVec) * 16 + col % kVec * sizeof(T);
            float v[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) v[r] = n + r < cta_rows ? to_float(*reinterpret_cast<const T *>(from + r * LPR * 16)) : 0.0f;
            uint32_t word[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) word[w] = quantize(v[4 * w], v[4 * w + 1], v[4 * w + 2], v[4 * w + 3]);
            *reinterpret_cast<uint4 *>(q + (long long)(f0 + col) * qs + cta_first + n) = make_uint4(word[0], word[1], word[2], word[3]);
        }
        __syncthreads();                                                  // nobody needs the tile any more
        fetch(f + clusters * kCols);
    }
    cl.leave(fault);
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

// An output from its sum.  The scales one after the other: their product may be outside of 32 bits where the output is not.
__device__ __forceinline__ float scaled(int sum, float w_scale, float q_scale, float bias) { return fmaf((float)sum * w_scale, q_scale, bias); }

// A single frame: what counts is to have W on its way.  A warp has a row of W, or one of `splits` parts of its inputs where there are few rows, and asks
// for 4096 bytes of it before it multiplies; q comes out of L1.  (Two rows a warp for two to eight frames: 9.9 to 22.7 us for 4096 x 4096, the tiles below 9.3.)
template <typename T>
__global__ void __launch_bounds__(256)
k_int8_dense_row(const int8_t *__restrict__ q, const float *__restrict__ q_scale, const int8_t *__restrict__ W, const float *__restrict__ w_scale,
                 const float *__restrict__ bias, T *y, int K, int O, long long ws, long long ys, int splits)
{
    grid_dependency();
    constexpr int kAhead = 8;
    __shared__ int red[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % splits, o = (int)blockIdx.x * (8 / splits) + warp / splits;
    const int steps = (K + 511) / 512, s0 = (int)((long long)steps * part / splits), s1 = (int)((long long)steps * (part + 1) / splits);
    const int8_t *const row = W + (long long)min(o, O - 1) * ws;
    int sum = 0;
    for (int s = s0; s < s1; s += kAhead) {
        int4 w[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int k = (s + a) * 512 + lane * 16;
            w[a] = s + a < s1 && k < K ? *reinterpret_cast<const int4 *>(row + k) : make_int4(0, 0, 0, 0);
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int k = (s + a) * 512 + lane * 16;
            if (s + a < s1 && k < K) {
                const int4 v = load_q(q, k, K);
                sum = __dp4a(w[a].w, v.w, __dp4a(w[a].z, v.z, __dp4a(w[a].y, v.y, __dp4a(w[a].x, v.x, sum))));
            }
        }
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (splits > 1) {
        if (lane == 0) red[warp] = sum;
        __syncthreads();
        if (part == 0)
            for (int i = 1; i < splits; ++i) sum += red[warp + i];
    }
    if (part == 0 && lane == 0 && o < O) y[(long long)o * ys] = from_float<T>(scaled(sum, w_scale[o], q_scale[0], bias ? bias[o] : 0.0f));
}

template <typename T>
static int int8_dense_row(const int8_t *q, const float *q_scale, const int8_t *W, const float *w_scale, const float *bias, T *y, int K, int O, int ws, int ys,
                          cudaStream_t st)
{
    int splits = 1;
    while (splits < 8 && (long long)O * splits < 16LL * device_info().sm_count && (K + 511) / 512 >= 2 * splits) splits *= 2;
    launch(k_int8_dense_row<T>, (unsigned)(((long long)O * splits + 7) / 8), 256, 0, st, q, q_scale, W, w_scale, bias, y, K, O, ws, ys, splits);
    return launch_status();
}

// ---- the product on the tensor cores: tiles of 128 output nodes x TN frames, D[o][f] = sum_k W[o][k] q[f][k] in TMEM (lane = output node, column =
// frame), 128 bytes of k a stage, brought by TMA into 128-byte swizzled rows.  Warp 0 copies, warp 1 issues the matrix instructions, warps 2-5 scale and
// store; the accumulator is double, so that the epilogue of a tile runs beside the products of the next.  Where there are fewer tiles than SMs, a
// cluster of CTAs shares the k of one tile: the integer partial sums cross through distributed shared memory (in any order: they are exact), and every
// CTA finishes its part of the columns.
constexpr int kGemmThreads = 192, kTileO = 128, kTileK = 128;
template <int TN> constexpr int kGemmStages = TN >= 128 ? 6 : 8;
template <int TN> constexpr int kStageBytes = (kTileO + TN) * kTileK;
template <int TN> constexpr int kGemmSmem = kGemmStages<TN> * kStageBytes<TN> + 1024;
constexpr int kMostSplits = 8;
constexpr int kTileGroup = 16;                           // tiles of output nodes that are walked together, so that their W and the q of some frames stay in L2

struct GemmArgs {
    const float *q_scale, *w_scale, *bias;
    int K, O, F, splits, vec;
    long long ys;
    int *fault;
};

// Columns of TMEM (`at`: a warp's 32 lanes, from column `c` on) to y, as many as make 128 bytes of a row: a lane has an output node, from o0 on, the columns
// are the frames f on, `scale` theirs.  The values cross through 4 KB of the warp's shared memory, in 16-byte pieces whose order differs from row to row
// so that no banks collide, and leave as whole lines of four rows a store.  (A store of 16 bytes by each lane for its own row touches 32 lines at a time:
// 8192 x 8192 x 1024 91 us, with the products done in 42.)
template <typename T, int TN> constexpr int kStoreColumns = TN < 128 / (int)sizeof(T) ? TN : 128 / (int)sizeof(T);      // (of a tile of TN frames)
template <typename T, int COLS>
__device__ __forceinline__ void store_columns(const GemmArgs &a, T *y, uint32_t at, int c, int o0, int f, float ws, float b, const float *scale, uint4 (*stage)[8])
{
    constexpr int kVec = kFramesPerVec<T>, kPieces = COLS / kVec;
    const int lane = threadIdx.x & 31;
    const bool whole = a.vec && f + COLS <= a.F;
#pragma unroll
    for (int h = 0; h < COLS; h += 32) {
        if (f + h >= a.F) break;
        int v[32];
        tmem_load_32(at + c + h, v);
#pragma unroll
        for (int i = 0; i < 32; i += kVec) {
            float r[kVec];
#pragma unroll
            for (int j = 0; j < kVec; ++j) r[j] = scaled(v[i + j], ws, scale[h + i + j], b);
            if (whole) {
                stage[lane][(h + i) / kVec ^ (lane & (kPieces - 1))] = pack<T>(r);
            } else if (o0 + lane < a.O) {
#pragma unroll
                for (int j = 0; j < kVec; ++j)
                    if (f + h + i + j < a.F) y[(long long)(o0 + lane) * a.ys + f + h + i + j] = from_float<T>(r[j]);
            }
        }
    }
    if (whole) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int row = (i * 32 + lane) / kPieces, piece = lane % kPieces;
            if (o0 + row < a.O) *reinterpret_cast<uint4 *>(y + (long long)(o0 + row) * a.ys + f + piece * kVec) = stage[row][piece ^ (row & (kPieces - 1))];
        }
        __syncwarp();
    }
}

template <typename T, int TN>
__global__ void __launch_bounds__(kGemmThreads, 1)
k_int8_dense_tiles(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q, T *y, const GemmArgs a)
{
    constexpr int kStages = kGemmStages<TN>, kAcc = 2, kColumns = kAcc * TN < 32 ? 32 : kAcc * TN;
    static_assert(kColumns <= 512 && (kColumns & (kColumns - 1)) == 0, "TMEM");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[kStages], empty[kStages], acc_full[kAcc], acc_empty[kAcc], drained;
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    __shared__ float s_scale[4][TN];                                      // of the frames of a tile, one copy an epilogue warp
    __shared__ uint4 stage_out[4][32][8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = a.splits > 1 ? cluster_rank() : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int s = 0; s < kAcc; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 4); }
        mbar_init(&drained, 1);
        gave_up = 0;
        mbar_init_fence();
        tma_prefetch(&map_w);
        tma_prefetch(&map_q);
    }
    if (warp == 1) tmem_alloc(&tmem_base, kColumns);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = tmem_base;
    grid_dependency();

    const int tiles_o = (a.O + kTileO - 1) / kTileO, tiles_f = (a.F + TN - 1) / TN, tiles = tiles_o * tiles_f;
    const int blocks_k = (a.K + kTileK - 1) / kTileK;
    const int k0 = (int)((long long)blocks_k * rank / a.splits), k1 = (int)((long long)blocks_k * (rank + 1) / a.splits);
    const int first = (int)blockIdx.x / a.splits, step = (int)gridDim.x / a.splits;
    auto place = [&](int tile, int &o0, int &f0) {
        const int group = tile / (kTileGroup * tiles_f), in = tile % (kTileGroup * tiles_f), rows = min(kTileGroup, tiles_o - group * kTileGroup);
        o0 = (group * kTileGroup + in % rows) * kTileO;
        f0 = in / rows * TN;
    };

    if (warp == 0 && lane == 0) {
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
            int o0, f0;
            place(tile, o0, f0);
            for (int kb = k0; kb < k1 && ok; ++kb) {
                ok = mbar_wait_one(&empty[stage], phase ^ 1, &gave_up);
                if (!ok) break;
                uint8_t *at = smem + stage * kStageBytes<TN>;
                mbar_arrive_expect_tx(&full[stage], kStageBytes<TN>);
                tma_load_2d(at, &map_w, kb * kTileK, o0, &full[stage]);
                tma_load_2d(at + kTileO * kTileK, &map_q, kb * kTileK, f0, &full[stage]);
                ++issued;
                if (++stage == kStages) { stage = 0; phase ^= 1; }
            }
        }
        // what is under way lands before the CTA leaves, also where a wait has run out
        for (int b = issued > kStages ? issued - kStages : 0; b < issued; ++b) mbar_wait_some(&full[b % kStages], (uint32_t)(b / kStages) & 1u, kDrainSpins);
    } else if (warp == 1 && lane == 0) {
        constexpr uint32_t kInstr = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TN >> 3) << 17) | ((uint32_t)(kTileO >> 4) << 24);     // s32 += s8 x s8
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
            ok = mbar_wait_one(&acc_empty[acc], acc_phase ^ 1, &gave_up);
            if (!ok) break;
            tcgen05_fence_after();
            for (int kb = k0; kb < k1; ++kb) {
                ok = mbar_wait_one(&full[stage], phase, &gave_up);
                if (!ok) break;
                tcgen05_fence_after();
                const uint32_t at = smem_addr(smem + stage * kStageBytes<TN>);
                const uint64_t da = smem_descriptor_128b(at), db = smem_descriptor_128b(at + kTileO * kTileK);
#pragma unroll
                for (int k = 0; k < kTileK / 32; ++k) mma_i8(tmem + acc * TN, da + 2 * k, db + 2 * k, kInstr, kb > k0 || k > 0);
                tcgen05_commit(&empty[stage]);
                if (++stage == kStages) { stage = 0; phase ^= 1; }
            }
            if (!ok) break;
            tcgen05_commit(&acc_full[acc]);
            if (++acc == kAcc) { acc = 0; acc_phase ^= 1; }
        }
        tcgen05_commit(&drained);                                         // no product is under way when the TMEM goes back
        mbar_wait_some(&drained, 0, kDrainSpins);
    } else if (warp >= 2) {
        const int part = warp & 3, row = part * 32 + lane;                // the lanes of TMEM that this warp may read
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int tile = first; tile < tiles; tile += step) {
            int o0, f0;
            place(tile, o0, f0);
            const int o = o0 + row;
            __syncwarp();
            for (int i = lane; i < TN; i += 32) s_scale[part][i] = f0 + i < a.F ? a.q_scale[f0 + i] : 0.0f;
            const float ws = o < a.O ? a.w_scale[o] : 0.0f, b = o < a.O && a.bias ? a.bias[o] : 0.0f;
            __syncwarp();
            if (!mbar_wait_warp(&acc_full[acc], acc_phase, &gave_up)) break;
            tcgen05_fence_after();
            const uint32_t at = tmem + ((uint32_t)(part * 32) << 16) + acc * TN;
            if (a.splits == 1) {
#pragma unroll 1
                for (int c = 0; c < TN; c += kStoreColumns<T, TN>) {
                    if (f0 + c >= a.F) break;
                    store_columns<T, kStoreColumns<T, TN>>(a, y, at, c, o0 + part * 32, f0 + c, ws, b, &s_scale[part][c], stage_out[part]);
                }
            } else {
                // the stages are free: the tile's last product is done, and with it everything that read them
                int *sums = reinterpret_cast<int *>(smem) + row * (TN + 4);
#pragma unroll 1
                for (int c = 0; c < TN; c += 32) {
                    int v[32];
                    tmem_load_32(at + c, v);
#pragma unroll
                    for (int i = 0; i < 32; i += 4) *reinterpret_cast<int4 *>(sums + c + i) = make_int4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                }
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[acc]);
            if (++acc == kAcc) { acc = 0; acc_phase ^= 1; }
        }
    }
    if (a.splits > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp >= 2 && !gave_up) {
            int o0, f0;
            place(first, o0, f0);
            const int row = (warp & 3) * 32 + lane, o = o0 + row, width = TN / a.splits, c0 = (int)rank * width;
            if (o < a.O) {
                const float ws = a.w_scale[o], b = a.bias ? a.bias[o] : 0.0f;
                const uint32_t own = smem_addr(reinterpret_cast<int *>(smem) + row * (TN + 4));
#pragma unroll 2
                for (int c = c0; c < c0 + width; c += 4) {
                    int4 v = make_int4(0, 0, 0, 0), p[kMostSplits];
#pragma unroll
                    for (int r = 0; r < kMostSplits; ++r)                   // all of them under way at a time
                        if (r < a.splits) p[r] = peer_load_v4(own + c * 4, (uint32_t)r);
#pragma unroll
                    for (int r = 0; r < kMostSplits; ++r)
                        if (r < a.splits) { v.x += p[r].x; v.y += p[r].y; v.z += p[r].z; v.w += p[r].w; }
                    const int sums[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (f0 + c + i < a.F) y[(long long)o * a.ys + f0 + c + i] = from_float<T>(scaled(sums[i], ws, s_scale[warp & 3][c + i], b));
                }
            }
        }
        __syncwarp();
        cluster_arrive();                                                 // nobody leaves while its sums may still be read
        cluster_wait();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    if (warp == 1) tmem_free(tmem, kColumns);
    if (threadIdx.x == 0 && gave_up) atomicCAS(a.fault, 0, kFaultBarrierTimeout);
}

// Large products: two CTAs on one tile of 256 output nodes x 256 frames.  Each brings 128 rows of either operand, the tensor cores of both work on all of
// them, and each CTA gets the sums of its 128 output nodes.  That halves what a CTA has to bring and read of q: alone, with 128 x 256, shared memory
// bounds the products (8192^3: 374 us, 79 % of the tensor cores' cycles).  The first CTA issues the products and has the barriers of what has arrived and
// of free accumulators; of consumed stages and finished sums each has its own.
constexpr int kPairN = 256, kPairStages = 6, kPairStageBytes = 2 * kTileO * kTileK, kPairSmem = kPairStages * kPairStageBytes + 1024, kPairGroup = 8;

template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 1)
k_int8_dense_pairs(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q, T *y, const GemmArgs a)
{
    constexpr int kAcc = 2, kColumns = kAcc * kPairN;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[kPairStages], empty[kPairStages], acc_full[kAcc], acc_empty[kAcc], drained;
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    __shared__ float s_scale[4][kPairN];
    __shared__ uint4 stage_out[4][32][8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int s = 0; s < kAcc; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 8); }
        mbar_init(&drained, 1);
        gave_up = 0;
        mbar_init_fence();
        tma_prefetch(&map_w);
        tma_prefetch(&map_q);
    }
    __syncwarp();
    if (warp == 1) tmem_alloc_pair(&tmem_base, kColumns);
    tcgen05_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    tcgen05_fence_after();
    const uint32_t tmem = tmem_base;
    grid_dependency();

    const int tiles_o = (a.O + 2 * kTileO - 1) / (2 * kTileO), tiles_f = (a.F + kPairN - 1) / kPairN, tiles = tiles_o * tiles_f;
    const int blocks_k = (a.K + kTileK - 1) / kTileK, first = (int)blockIdx.x / 2, step = (int)gridDim.x / 2;
    auto place = [&](int tile, int &o0, int &f0) {
        const int group = tile / (kPairGroup * tiles_f), in = tile % (kPairGroup * tiles_f), rows = min(kPairGroup, tiles_o - group * kPairGroup);
        o0 = (group * kPairGroup + in % rows) * 2 * kTileO + (int)rank * kTileO;
        f0 = in / rows * kPairN;
    };

    if (warp == 0 && lane == 0) {
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
            int o0, f0;
            place(tile, o0, f0);
            for (int kb = 0; kb < blocks_k; ++kb) {
                ok = mbar_wait_one(&empty[stage], phase ^ 1, &gave_up);
                if (!ok) break;
                uint8_t *at = smem + stage * kPairStageBytes;
                if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * kPairStageBytes);
                const uint32_t bar = peer_addr(&full[stage], 0);
                tma_load_2d_pair(at, &map_w, kb * kTileK, o0, bar);
                tma_load_2d_pair(at + kTileO * kTileK, &map_q, kb * kTileK, f0 + (int)rank * (kPairN / 2), bar);
                ++issued;
                if (++stage == kPairStages) { stage = 0; phase ^= 1; }
            }
        }
        // what is under way, for either CTA, lands before they leave, also where a wait has run out
        if (rank == 0)
            for (int b = issued > kPairStages ? issued - kPairStages : 0; b < issued; ++b)
                mbar_wait_some(&full[b % kPairStages], (uint32_t)(b / kPairStages) & 1u, kDrainSpins);
    } else if (warp == 1 && lane == 0 && rank == 0) {
        constexpr uint32_t kInstr = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kPairN >> 3) << 17) | ((uint32_t)(2 * kTileO >> 4) << 24);
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += step) {
            ok = mbar_wait_one(&acc_empty[acc], acc_phase ^ 1, &gave_up);
            if (!ok) break;
            tcgen05_fence_after();
            for (int kb = 0; kb < blocks_k; ++kb) {
                ok = mbar_wait_one(&full[stage], phase, &gave_up);
                if (!ok) break;
                tcgen05_fence_after();
                const uint32_t at = smem_addr(smem + stage * kPairStageBytes);
                const uint64_t da = smem_descriptor_128b(at), db = smem_descriptor_128b(at + kTileO * kTileK);
#pragma unroll
                for (int k = 0; k < kTileK / 32; ++k) mma_i8_pair(tmem + acc * kPairN, da + 2 * k, db + 2 * k, kInstr, kb > 0 || k > 0);
                tcgen05_commit_pair(&empty[stage]);
                if (++stage == kPairStages) { stage = 0; phase ^= 1; }
            }
            if (!ok) break;
            tcgen05_commit_pair(&acc_full[acc]);
            if (++acc == kAcc) { acc = 0; acc_phase ^= 1; }
        }
        tcgen05_commit_pair_own(&drained);                                // no product is under way when the TMEM goes back
        mbar_wait_some(&drained, 0, kDrainSpins);
    } else if (warp >= 2) {
        const int part = warp & 3, row = part * 32 + lane;
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int tile = first; tile < tiles; tile += step) {
            int o0, f0;
            place(tile, o0, f0);
            const int o = o0 + row;
            __syncwarp();
            for (int i = lane; i < kPairN; i += 32) s_scale[part][i] = f0 + i < a.F ? a.q_scale[f0 + i] : 0.0f;
            const float ws = o < a.O ? a.w_scale[o] : 0.0f, b = o < a.O && a.bias ? a.bias[o] : 0.0f;
            __syncwarp();
            if (!mbar_wait_warp(&acc_full[acc], acc_phase, &gave_up)) break;
            tcgen05_fence_after();
            const uint32_t at = tmem + ((uint32_t)(part * 32) << 16) + acc * kPairN;
#pragma unroll 1
            for (int c = 0; c < kPairN; c += kStoreColumns<T, kPairN>) {
                if (f0 + c >= a.F) break;
                store_columns<T, kStoreColumns<T, kPairN>>(a, y, at, c, o0 + part * 32, f0 + c, ws, b, &s_scale[part][c], stage_out[part]);
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(peer_addr(&acc_empty[acc], 0));
            if (++acc == kAcc) { acc = 0; acc_phase ^= 1; }
        }
    }
    __syncwarp();
    tcgen05_fence_before();
    cluster_arrive();
    cluster_wait();
    tcgen05_fence_after();
    if (warp == 1) tmem_free_pair(tmem, kColumns);
    if (threadIdx.x == 0 && gave_up) atomicCAS(a.fault, 0, kFaultBarrierTimeout);
}

// rows of 8-bit integers as TMA sees them: boxes of 128 bytes x `box_rows` rows; what lies beyond the inputs or the rows reads as zero
static int int8_rows_map(CUtensorMap *map, const int8_t *p, int K, int rows, long long stride, int box_rows)
{
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            fn = nullptr;
        }
        return reinterpret_cast<Encode>(fn);
    }();
    BB200_REQUIRE(encode != nullptr, BBCU_ERR_NO_DEVICE);
    const cuuint64_t size[2] = {(cuuint64_t)K, (cuuint64_t)rows}, pitch[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {(cuuint32_t)kTileK, (cuuint32_t)box_rows}, unit[2] = {1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(p), size, pitch, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? BBCU_OK : (int)cudaErrorInvalidValue;
}

template <typename T, int TN>
static int int8_dense_tiles(const int8_t *q, const int8_t *W, T *y, GemmArgs a, long long qs, long long ws, cudaStream_t st)
{
    CUtensorMap map_w, map_q;
    if (const int e = int8_rows_map(&map_w, W, a.K, a.O, ws, kTileO)) return e;
    if (const int e = int8_rows_map(&map_q, q, a.K, a.F, qs, TN)) return e;
    const long long tiles = ((long long)a.O + kTileO - 1) / kTileO * (((long long)a.F + TN - 1) / TN);
    BB200_REQUIRE(tiles < (1LL << 27), BBCU_ERR_TOO_LARGE);
    auto kernel = k_int8_dense_tiles<T, TN>;
    BB200_REQUIRE(allow_big_smem(kernel, kGemmSmem<TN>), (int)cudaErrorInvalidValue);
    const long long sms = device_info().sm_count;
    const unsigned grid = a.splits > 1 ? (unsigned)(tiles * a.splits) : (unsigned)(tiles < sms ? tiles : sms);
    return launch_cluster(kernel, (unsigned)a.splits, grid, kGemmThreads, kGemmSmem<TN>, st, map_w, map_q, y, a);
}

// Frames a tile (kPairN: by a pair of CTAs) and CTAs that share the inputs of one, by the clocks of an SM: rounds of tiles times blocks of 128 inputs times
// what a block costs, 2 (128 + frames) where shared memory takes in and gives out both operands at 128 bytes a clock, 512 for a pair, which the tensor
// cores bound; and about 12 for each column that is stored at the end, 2500 where sums cross a cluster.  (us, this choice and the best of others: 2048^3
// 14 by pairs and 15 by 128 columns; 4096 x 4096 x 16 9.5 by four CTAs, 25 by one.)
struct TileChoice { int columns, splits; };
static TileChoice choose_tiles(int K, int O, int F)
{
    const long long sms = device_info().sm_count, blocks = (K + kTileK - 1) / kTileK, tiles_o = ((long long)O + kTileO - 1) / kTileO;
    const long long pair_tiles = ((long long)O + 2 * kTileO - 1) / (2 * kTileO) * (((long long)F + kPairN - 1) / kPairN);
    TileChoice best = {kPairN, 1};
    long long least = (pair_tiles + sms / 2 - 1) / (sms / 2) * blocks * 512 + 12 * kPairN;
    for (int columns = 32; columns <= 128; columns *= 2) {
        const long long tiles = tiles_o * ((F + columns - 1) / columns);
        for (int splits = 1; splits <= kMostSplits; splits *= 2) {
            if (splits > 1 && (tiles * splits > sms || blocks < 2 * splits)) break;
            const long long cost = (tiles * splits + sms - 1) / sms * ((blocks + splits - 1) / splits) * 2 * (kTileO + columns) + 12 * columns + (splits > 1 ? 2500 : 0);
            if (cost < least) { least = cost; best = {columns, splits}; }
        }
    }
    return best;
}

template <typename T>
static int int8_dense_pairs(const int8_t *q, const int8_t *W, T *y, const GemmArgs &a, long long qs, long long ws, cudaStream_t st)
{
    CUtensorMap map_w, map_q;
    if (const int e = int8_rows_map(&map_w, W, a.K, a.O, ws, kTileO)) return e;
    if (const int e = int8_rows_map(&map_q, q, a.K, a.F, qs, kPairN / 2)) return e;
    const long long tiles = ((long long)a.O + 2 * kTileO - 1) / (2 * kTileO) * (((long long)a.F + kPairN - 1) / kPairN), pairs = device_info().sm_count / 2;
    BB200_REQUIRE(tiles < (1LL << 30), BBCU_ERR_TOO_LARGE);
    auto kernel = k_int8_dense_pairs<T>;
    BB200_REQUIRE(allow_big_smem(kernel, kPairSmem), (int)cudaErrorInvalidValue);
    return launch_cluster(kernel, 2u, (unsigned)(2 * (tiles < pairs ? tiles : pairs)), kGemmThreads, kPairSmem, st, map_w, map_q, y, a);
}

template <typename T>
static int quantize_frames(const T *x, int8_t *q, float *scale, int N, int F, int xs, int qs, bbcu_stream_t stream)
{
    BB200_REQUIRE(N > 0 && F >= 0, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(N <= (1 << 22), BBCU_ERR_TOO_LARGE);
    BB200_REQUIRE(xs >= F && qs >= (N + 15) / 16 * 16 && qs % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0, BBCU_ERR_BAD_STRIDE);
    if (F == 0) return BBCU_OK;
    BB200_REQUIRE_PTR(x); BB200_REQUIRE_PTR(q); BB200_REQUIRE_PTR(scale);
    cudaStream_t st = as_stream(stream);
    const bool aligned = frames_aligned<T>(x, xs);
    BB200_REQUIRE(F <= (1 << 30), BBCU_ERR_TOO_LARGE);
    if (ColumnPlan p = plan_columns<T>(N, F, 4, kQuantOnceRows, 8); aligned && p.cluster && (long long)N * F <= kQuantSmall) {
        const int per_warp = 32 / p.lanes;
        if (p.warps * per_warp % 16) ++p.warps;                           // a round of rows is whole 16-byte pieces of q
        p.rows = ((N + p.cluster - 1) / p.cluster + per_warp * p.warps - 1) / (per_warp * p.warps);
        int *fault = fault_word();
        BB200_REQUIRE(fault != nullptr, BBCU_ERR_NO_DEVICE);
        const int cols = p.lanes * kFramesPerVec<T>, once_tiles = (F + cols - 1) / cols, threads = 32 * p.warps;
        const int smem = p.rows * threads * 16 + (p.lanes == 2 ? exchange_bytes<1, Column<T, 2>::kCols>(p.cluster) : exchange_bytes<1, Column<T, 4>::kCols>(p.cluster));
        auto kernel = p.lanes == 2 ? k_quantize_once<T, 2> : k_quantize_once<T, 4>;
        BB200_REQUIRE(allow_big_smem(kernel, kQuantOnceRows * kColumnThreads * 16 + exchange_bytes<1, Column<T, 4>::kCols>(8)), (int)cudaErrorInvalidValue);
        const int clusters = std::min(once_tiles, resident_clusters(reinterpret_cast<const void *>(kernel), p.cluster, threads, smem));
        return launch_cluster(kernel, (unsigned)p.cluster, (unsigned)(clusters * p.cluster), threads, smem, st, x, q, scale, N, F, (long long)xs, (long long)qs, p.rows,
                              once_tiles, fault);
    }
    constexpr int kCols = Column<T, 8>::kCols;
    const long long tiles = ((long long)F + kCols - 1) / kCols, bands = ((long long)N + kQuantRows - 1) / kQuantRows;
    BB200_REQUIRE(bands <= 65535, BBCU_ERR_TOO_LARGE);
    const StreamingPlan s = plan_streaming<T>(N, F);
    auto scales = s.lanes == 2 ? (aligned ? k_quantize_scale<T, 2, true> : k_quantize_scale<T, 2, false>)
                               : (aligned ? k_quantize_scale<T, 8, true> : k_quantize_scale<T, 8, false>);
    if (const int e = launch_cluster(scales, s.cluster, s.ctas, kQuantThreads, 0, st, x, scale, N, F, (long long)xs)) return e;
    launch(aligned ? k_quantize_apply<T, true> : k_quantize_apply<T, false>, dim3((unsigned)tiles, (unsigned)bands), kQuantThreads, 0, st, x, q, scale, N, F, xs, qs);
    return launch_status();
}

template <typename T>
static int int8_dense(const int8_t *q, const float *q_scale, const int8_t *W, const float *w_scale, const float *bias, T *y, int K, int O, int F, int qs,
                      int ws, int ys, bbcu_stream_t stream)
{
    BB200_REQUIRE(K > 0 && O >= 0 && F >= 0, BBCU_ERR_BAD_SIZE);
    BB200_REQUIRE(K <= kMostInputs && O <= (1 << 30) && F <= (1 << 30), BBCU_ERR_TOO_LARGE);       // (counts are rounded up to whole tiles in 32 bits)
    const int least = (K + 15) / 16 * 16;
    BB200_REQUIRE(qs >= least && ws >= least && qs % 16 == 0 && ws % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(W) % 16 == 0 && ys >= F, BBCU_ERR_BAD_STRIDE);
    if (F == 0 || O == 0) return BBCU_OK;
    BB200_REQUIRE_PTR(q); BB200_REQUIRE_PTR(q_scale); BB200_REQUIRE_PTR(W); BB200_REQUIRE_PTR(w_scale); BB200_REQUIRE_PTR(y);
    cudaStream_t st = as_stream(stream);
    if (F == 1) return int8_dense_row<T>(q, q_scale, W, w_scale, bias, y, K, O, ws, ys, st);
    int *fault = fault_word();
    BB200_REQUIRE(fault != nullptr, BBCU_ERR_NO_DEVICE);
    GemmArgs a{q_scale, w_scale, bias, K, O, F, 1, frames_aligned<T>(y, ys), ys, fault};
    const TileChoice t = choose_tiles(K, O, F);
    if (t.columns == kPairN) return int8_dense_pairs<T>(q, W, y, a, qs, ws, st);
    a.splits = t.splits;
    const int tn = t.columns;
    return tn == 32 ? int8_dense_tiles<T, 32>(q, W, y, a, qs, ws, st) : tn == 64 ? int8_dense_tiles<T, 64>(q, W, y, a, qs, ws, st)
                    : int8_dense_tiles<T, 128>(q, W, y, a, qs, ws, st);
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
