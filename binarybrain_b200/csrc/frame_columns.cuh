// Operators over the NODES of a frame (layer norm, the scales of the int8 quantiser, the softmax of the distillation loss) on node-major frame
// buffers of fp32 or bf16: a frame is a column, and a thread owns 16 bytes of a row, i.e. 4 or 8 neighbouring columns, for several rows.
//
// Common layout of a CTA: LPR lanes of a warp stand side by side along the frames (8 lanes: 128 bytes, 2 lanes: 32 bytes of a row), the 32 / LPR
// groups of a warp and the warps of the CTA one row below the other; a thread's further rows follow at a distance of all of them.  A cluster of
// 1 to 16 CTAs shares the rows of one column tile, so that a tile is read once and held in registers between the statistics and what is made of
// them; the column sums cross the warps through shared memory and the CTAs through distributed shared memory.
#pragma once

#include <cuda_bf16.h>

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

template <typename T> inline bool frames_aligned(const void *p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * (long long)sizeof(T) % 16 == 0; }

// ---- clusters
__device__ __forceinline__ uint32_t cluster_rank()  { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size()  { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_arrive()    { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait()      { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float peer_load(const float *own, uint32_t rank)
{
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(own)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// Launch with clusters of `cluster` CTAs (grid.x is a multiple of it); 16 needs the kernel's opt-in.
bool allow_cluster_16_once(const void *kernel);
template <typename... P, typename... A>
inline int launch_cluster(void (*kernel)(P...), unsigned cluster, dim3 grid, dim3 block, size_t smem, cudaStream_t st, A &&...args)
{
    if (cluster > 8 && !allow_cluster_16_once(reinterpret_cast<const void *>(kernel))) return (int)cudaErrorInvalidClusterSize;
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

// Joins v[Q][kVec] over all rows of the tile (CTA, then cluster); every thread gets the result of its own columns, in the same order of operations
// everywhere.  `red`: warps * Q * kCols floats, `part`: Q * kCols floats, neither in use by an exchange that a neighbour may still be reading:
// consecutive exchanges alternate between two of each.
template <typename OP, int Q, typename T, int LPR>
__device__ __forceinline__ void join_columns(float (&v)[Q][kFramesPerVec<T>], const Column<T, LPR> &c, float *red, float *part, uint32_t cluster)
{
    constexpr int kVec = kFramesPerVec<T>, kCols = LPR * kVec;
#pragma unroll
    for (int m = LPR; m < 32; m <<= 1)
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[q][j] = OP::join(v[q][j], __shfl_xor_sync(0xffffffffu, v[q][j], m));
    if (c.lane < LPR) {
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int j = 0; j < kVec; ++j) red[(c.warp * Q + q) * kCols + c.col + j] = v[q][j];
    }
    __syncthreads();
    if (cluster == 1) {
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[q][j] = red[q * kCols + c.col + j];
        for (int w = 1; w < c.warps; ++w)
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int j = 0; j < kVec; ++j) v[q][j] = OP::join(v[q][j], red[(w * Q + q) * kCols + c.col + j]);
        return;
    }
    for (int i = threadIdx.x; i < Q * kCols; i += blockDim.x) {
        float s = red[i];
        for (int w = 1; w < c.warps; ++w) s = OP::join(s, red[w * Q * kCols + i]);
        part[i] = s;
    }
    cluster_arrive();
    cluster_wait();
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[q][j] = OP::none;
    for (uint32_t r = 0; r < cluster; ++r)
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[q][j] = OP::join(v[q][j], peer_load(part + q * kCols + c.col + j, r));
}

// No CTA of a cluster leaves while another may still read its shared memory.
__device__ __forceinline__ void cluster_leave(uint32_t cluster)
{
    if (cluster > 1) { cluster_arrive(); cluster_wait(); }
}

// How a layer of N rows and F frames is cut: clusters of `cluster` CTAs of `warps` warps, `rows` rows a thread.
struct ColumnPlan { int cluster, warps, rows; };

}   // namespace bb200
