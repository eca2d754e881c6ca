// Operators over the NODES of a frame (layer norm, the scales of the int8 quantiser, the softmax of the distillation loss) on node-major frame
// buffers of fp32 or bf16: a frame is a column, and a thread owns 16 bytes of a row, i.e. 4 or 8 neighbouring columns, for several rows.
//
// Common layout of a CTA: LPR lanes of a warp stand side by side along the frames (8 lanes: 128 bytes, 2 lanes: 32 bytes of a row), the 32 / LPR
// groups of a warp and the warps of the CTA one row below the other; a thread's further rows follow at a distance of all of them.  A cluster of
// 1 to 8 CTAs shares the rows of one column tile, so that a tile is read once and held in shared memory between the statistics and what is made of
// them; the column sums cross the warps through shared memory and the CTAs through distributed shared memory.
#pragma once

#include <algorithm>

#include <cuda_bf16.h>

#include "async_copy.cuh"
#include "common.cuh"

namespace bb200 {

template <typename T> constexpr int kFramesPerVec = 16 / (int)sizeof(T);

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of a row as 32-bit values
template <typename T> __device__ __forceinline__ void unpack(const uint4 &r, float (&v)[kFramesPerVec<T>]);
template <> __device__ __forceinline__ void unpack<float>(const uint4 &r, float (&v)[4])
{
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
}
template <> __device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4 &r, float (&v)[8])
{
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
}
template <typename T> __device__ __forceinline__ uint4 pack(const float (&v)[kFramesPerVec<T>]);
template <> __device__ __forceinline__ uint4 pack<float>(const float (&v)[4])
{
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
template <> __device__ __forceinline__ uint4 pack<__nv_bfloat16>(const float (&v)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t *>(&b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The frames f .. f + 15 bytes of a row; frames from F on come as whatever the row's padding holds (ALIGNED: the row reaches at least to the end of
// the vector, because its stride is a multiple of the vector) or as zeros.
template <typename T, bool ALIGNED> __device__ __forceinline__ uint4 load_frames(const T *row, int f, int F)
{
    if constexpr (ALIGNED) {
        return f < F ? *reinterpret_cast<const uint4 *>(row + f) : make_uint4(0, 0, 0, 0);
    } else {
        float v[kFramesPerVec<T>];
#pragma unroll
        for (int j = 0; j < kFramesPerVec<T>; ++j) v[j] = f + j < F ? to_float(row[f + j]) : 0.0f;
        return pack<T>(v);
    }
}

// stores the frames below F and nothing else
template <typename T, bool ALIGNED> __device__ __forceinline__ void store_frames(T *row, int f, int F, const float (&v)[kFramesPerVec<T>])
{
    if (ALIGNED && f + kFramesPerVec<T> <= F) {
        *reinterpret_cast<uint4 *>(row + f) = pack<T>(v);
    } else {
#pragma unroll
        for (int j = 0; j < kFramesPerVec<T>; ++j)
            if (f + j < F) row[f + j] = from_float<T>(v[j]);
    }
}

// a number of each of a thread's columns, 0 beyond the frames
template <int VEC> __device__ __forceinline__ void load_columns(const float *__restrict__ from, int f, int F, float (&v)[VEC])
{
    if (f + VEC <= F && (reinterpret_cast<uintptr_t>(from) & 15) == 0) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
            const float4 o = *reinterpret_cast<const float4 *>(from + f + j);
            v[j] = o.x; v[j + 1] = o.y; v[j + 2] = o.z; v[j + 3] = o.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = f + j < F ? from[f + j] : 0.0f;
    }
}

// ---- along the rows: the frames f0 .. f0 + 512 bytes of a row by a warp.  Rows on 16-byte boundaries: 16 bytes a lane; others: every 32nd frame a lane, so
// that the warp's narrow accesses lie side by side (distillation of 20000 x 777 bf16 at an odd stride: 89 us with 8 neighbours a lane).
template <typename T, bool ALIGNED> struct Line {
    static constexpr int kVec = kFramesPerVec<T>;
    int F, first;                                        // first frame of the lane
    __device__ Line(int f0, int lane, int frames) : F(frames), first(f0 + (ALIGNED ? lane * kVec : lane)) {}
    __device__ bool empty() const { return first >= F; }
    __device__ int frame(int j) const { return first + (ALIGNED ? j : 32 * j); }
    __device__ uint4 load(const T *row) const
    {
        if constexpr (ALIGNED) return load_frames<T, true>(row, first, F);
        float v[kVec];
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[j] = frame(j) < F ? to_float(row[frame(j)]) : 0.0f;
        return pack<T>(v);
    }
    __device__ void store(T *row, const float (&v)[kVec]) const
    {
        if constexpr (ALIGNED) {
            store_frames<T, true>(row, first, F, v);
        } else {
#pragma unroll
            for (int j = 0; j < kVec; ++j)
                if (frame(j) < F) row[frame(j)] = from_float<T>(v[j]);
        }
    }
    __device__ void load_columns(const float *__restrict__ from, float (&v)[kVec]) const
    {
        if constexpr (ALIGNED) {
            bb200::load_columns(from, first, F, v);
        } else {
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[j] = frame(j) < F ? from[frame(j)] : 0.0f;
        }
    }
};

template <typename T> inline bool frames_aligned(const void *p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * (long long)sizeof(T) % 16 == 0; }

// ---- clusters
__device__ __forceinline__ uint32_t cluster_rank()  { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size()  { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_arrive()    { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait()      { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer_addr(const void *own, uint32_t rank)
{
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(own)), "r"(rank));
    return at;
}
__device__ __forceinline__ float peer_load(const float *own, uint32_t rank)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_addr(own, rank)) : "memory");
    return v;
}
__device__ __forceinline__ double2 peer_load_double2(const double2 *own, uint32_t rank)
{
    double2 v;
    asm volatile("ld.shared::cluster.v2.f64 {%0, %1}, [%2];" : "=d"(v.x), "=d"(v.y) : "r"(peer_addr(own, rank)) : "memory");
    return v;
}
// a value for another CTA's shared memory, whose barrier counts the bytes when they have arrived
__device__ __forceinline__ void peer_send(uint32_t to, float v, uint32_t bar)
{
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(to), "f"(v), "r"(bar) : "memory");
}

// Launch with clusters of `cluster` CTAs (grid.x is a multiple of it).
template <typename... P, typename... A>
inline int launch_cluster(void (*kernel)(P...), unsigned cluster, dim3 grid, dim3 block, size_t smem, cudaStream_t st, A &&...args)
{
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    return launch_status();
}

// ---- a thread's place in the tile
template <typename T, int LPR> struct Column {
    static constexpr int kVec = kFramesPerVec<T>, kCols = LPR * kVec, kRowsPerWarp = 32 / LPR;
    int lane, warp, warps, row, step;            // first row of the thread in the CTA, distance between its rows
    int col;                                     // first of its columns in the tile
    __device__ Column()
    {
        lane = threadIdx.x & 31; warp = threadIdx.x >> 5; warps = blockDim.x >> 5;
        row = warp * kRowsPerWarp + lane / LPR;
        step = warps * kRowsPerWarp;
        col = lane % LPR * kVec;
    }
};

struct ColumnSum { __device__ static float join(float a, float b) { return a + b; }  static constexpr float none = 0.0f; };
struct ColumnMax { __device__ static float join(float a, float b) { return fmaxf(a, b); }  static constexpr float none = -INFINITY; };

constexpr int kColumnThreads = 256;

// Shared memory of one exchange of Q values a column; consecutive exchanges alternate between two of them, since a neighbour may still be reading.
// The parts of the cluster's CTAs, exchange_bytes(cluster) of them, lie in dynamic shared memory: their number is the launch's, and what they take decides
// how many CTAs an SM holds.
template <int Q, int COLS> struct Exchange {
    float red[kColumnThreads / 32][Q * COLS];
    __align__(16) float out[Q * COLS];
    float (*part)[Q * COLS];
    uint64_t bar;
};
template <int Q, int COLS> constexpr int exchange_bytes(int cluster) { return cluster > 1 ? 2 * cluster * Q * COLS * (int)sizeof(float) : 0; }

// A cluster of CTAs and what its exchanges have come to.  CTAs send their parts into the shared memory of all others, whose barriers count the bytes:
// unlike a barrier over the cluster, that does not wait for the stores of the tile before to be visible.
struct Cluster {
    uint32_t size, rank;
    int *gave_up;                                        // in shared memory: a wait ran out, all later ones are passed over
    __device__ Cluster(int *flag) : size(cluster_size()), rank(cluster_rank()), gave_up(flag) {}

    // before the first exchange: the barriers are there, and all CTAs run.  `parts`: exchange_bytes() of shared memory.
    template <int Q, int COLS> __device__ void meet(Exchange<Q, COLS> (&exchanges)[2], void *parts)
    {
        if (size == 1) return;
        if (threadIdx.x == 0) {
            *gave_up = 0;
            for (int i = 0; i < 2; ++i) {
                exchanges[i].part = reinterpret_cast<float (*)[Q * COLS]>(parts) + i * size;
                mbar_init(&exchanges[i].bar, 1);
            }
            mbar_init_fence();
        }
        cluster_arrive();
        cluster_wait();
    }
    // nobody leaves while something may still be sent to it
    __device__ void leave(int *fault)
    {
        if (size == 1) return;
        __syncthreads();
        if (threadIdx.x == 0 && *gave_up) atomicCAS(fault, 0, kFaultBarrierTimeout);
        cluster_arrive();
        cluster_wait();
    }
};

// Up to eight values `distance` apart, in their order; all of them on their way before the first is joined.
template <typename OP> __device__ __forceinline__ float join_parts(const float *from, int distance, int count)
{
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < count ? from[i * distance] : 0.0f;
    float s = v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i)
        if (i < count) s = OP::join(s, v[i]);
    return s;
}

// The way of v[Q][kVec] from the warps' lowest LPR lanes, which have their warp's columns, to what finish(q, joined) makes of a value over all rows of the tile,
// which comes back in v for the thread's own columns.  join_warps(from, distance, count) joins the parts of a CTA's warps, join_ctas those of a cluster's CTAs; one
// thread a value does so, since there are many threads and few columns.  `phase`: of the exchange's barrier, 0 and 1 in turn.
template <int Q, typename T, int LPR, typename WARPS, typename CTAS, typename FINISH>
__device__ __forceinline__ void exchange_columns(float (&v)[Q][kFramesPerVec<T>], const Column<T, LPR> &c, Exchange<Q, LPR * kFramesPerVec<T>> &e, const Cluster &cl,
                                                 uint32_t phase, WARPS join_warps, CTAS join_ctas, FINISH finish)
{
    constexpr int kVec = kFramesPerVec<T>, kCols = LPR * kVec;
    if (c.lane < LPR) {
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int j = 0; j < kVec; ++j) e.red[c.warp][q * kCols + c.col + j] = v[q][j];
    }
    if (cl.size > 1 && threadIdx.x == 0) mbar_arrive_expect_tx(&e.bar, cl.size * Q * kCols * (uint32_t)sizeof(float));
    __syncthreads();
    for (int i = threadIdx.x; i < Q * kCols; i += blockDim.x) {
        const float s = join_warps(&e.red[0][i], Q * kCols, c.warps);
        if (cl.size == 1) {
            e.out[i] = finish(i / kCols, s);
        } else {
            for (uint32_t r = 0; r < cl.size; ++r) peer_send(peer_addr(&e.part[cl.rank][i], r), s, peer_addr(&e.bar, r));
        }
    }
    if (cl.size > 1) {
        if (threadIdx.x / 32 * 32 < Q * kCols) {                          // warps that have something to join
            bool ok = *(volatile int *)cl.gave_up == 0;
            for (int i = 0; i < kWaitSpins && ok; ++i) {
                if (mbar_try_wait(&e.bar, phase)) break;
                if (i == kWaitSpins - 1) { *(volatile int *)cl.gave_up = 1; ok = false; }
            }
        }
        for (int i = threadIdx.x; i < Q * kCols; i += blockDim.x) e.out[i] = finish(i / kCols, join_ctas(&e.part[0][i], Q * kCols, (int)cl.size));
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int j = 0; j < kVec; j += 4) {
            const float4 o = *reinterpret_cast<const float4 *>(&e.out[q * kCols + c.col + j]);
            v[q][j] = o.x; v[q][j + 1] = o.y; v[q][j + 2] = o.z; v[q][j + 3] = o.w;
        }
}

// Joins v[Q][kVec] of all threads over all rows of the tile by a fixed order of operations.
template <typename OP, int Q, typename T, int LPR, typename FINISH>
__device__ __forceinline__ void join_columns(float (&v)[Q][kFramesPerVec<T>], const Column<T, LPR> &c, Exchange<Q, LPR * kFramesPerVec<T>> &e, const Cluster &cl,
                                             uint32_t phase, FINISH finish)
{
#pragma unroll
    for (int m = LPR; m < 32; m <<= 1)
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int j = 0; j < kFramesPerVec<T>; ++j) v[q][j] = OP::join(v[q][j], __shfl_xor_sync(0xffffffffu, v[q][j], m));
    exchange_columns<Q, T, LPR>(v, c, e, cl, phase, join_parts<OP>, join_parts<OP>, finish);
}

// How a kernel that streams over N rows is cut: `lanes` lanes along a row, 8 or, where those would leave most SMs without a cluster, 2; clusters that share
// a column tile, of as many CTAs as an SM holds four of and eight rounds of rows for each.  (Backward of 65536 x 64: 81 us by 8 lanes, 38 by 2; of 65536 x 1024,
// 256 CTAs by 8 lanes, 219 and 270.  One more doubling of the cluster, to a second round of CTAs, or clusters
// of 16, lost: layer norm of 16384 x 4096 bf16 72 us, 87 by clusters of 16 (its statistics have taken 2 us more since); 3000 x 5001 33 and 37.)
struct StreamingPlan { int lanes; unsigned cluster, ctas; };
template <typename T> inline StreamingPlan plan_streaming(int N, int F)
{
    const long long sms = device_info().sm_count;
    auto tiles = [&](int lanes) { return ((long long)F + lanes * kFramesPerVec<T> - 1) / (lanes * kFramesPerVec<T>); };
    const int lanes = tiles(8) * 8 < sms ? 2 : 8;
    unsigned cl = 1;
    while (cl < 8 && tiles(lanes) * cl <= 2 * sms && N > 256 / lanes * 8 * (int)cl) cl *= 2;
    return {lanes, cl, (unsigned)(tiles(lanes) * cl)};
}

// How a layer of N rows and F frames is cut: `lanes` lanes along a row, clusters of `cluster` CTAs, `most` at most (0: its columns are too long for one),
// of `warps` warps, `rows` rows a thread, at most `most_rows`.
struct ColumnPlan { int cluster, warps, rows, lanes; };
template <typename T>
inline ColumnPlan plan_columns(int N, int F, int lanes, int most_rows, int most)
{
    if (F <= 2 * kFramesPerVec<T>) lanes = 2;
    const int per_warp = 32 / lanes, most_warps = kColumnThreads / 32;
    const long long tiles = ((long long)F + lanes * kFramesPerVec<T> - 1) / (lanes * kFramesPerVec<T>), sms = device_info().sm_count;
    int cluster = 1;
    auto rows = [&] { return (N + cluster - 1) / cluster; };
    // as many CTAs as it takes to hold a column, and more where there would be few
    while (cluster < most && rows() > most_warps * per_warp * most_rows) cluster *= 2;
    if (rows() > most_warps * per_warp * most_rows) return {0, 0, 0, 0};
    while (cluster < most && tiles * cluster * 2 <= sms && rows() > most_warps * per_warp) cluster *= 2;
    const int warps = std::min(most_warps, (rows() + per_warp - 1) / per_warp);
    return {cluster, warps, (rows() + per_warp * warps - 1) / (per_warp * warps), lanes};
}

}   // namespace bb200
