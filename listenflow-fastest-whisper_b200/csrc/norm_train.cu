// sm_100a LayerNorm for training: forward with its statistics kept, and backward.
//
//   s = T(x + r)          mean, rstd of s over the row (fp32, population variance)
//   h = (s - mean) rstd   y = T(h gamma + beta)
//   w = dy gamma          dx = T(rstd (w - mean(w) - h mean(w h)) + dsum)
//   dgamma = sum over rows of dy h,  dbeta = sum over rows of dy
//
// T is the rows' type (fp16 or bf16); all arithmetic is fp32.  Both kernels are bound by
// DRAM: 2 bytes per element for each of x, r, s, y forward and dy, s, dsum, dx backward.
//
// A group of threads owns one row at a time, eight consecutive columns (16 bytes) per thread,
// so gamma, beta and the columns' dgamma and dbeta stay in registers for all of a group's
// rows.  Groups of a block run on their own (a named barrier each) and overlap one another's
// loads; R rows per step share the barriers of the row sums and put R times the loads in
// flight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "host_util.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace lffw {

namespace tnorm {

constexpr int kMaxThreads = 640;
constexpr int kMaxGroups = 15; // named barriers 1-15

struct Params {
    int64_t rows;
    int cols, groups, group_threads;
    const uint16_t *x, *residual; // forward
    uint16_t *sum, *y;
    const float *gamma, *beta;
    float eps;
    float *stats; // [2, rows]: mean, rstd
    const uint16_t *dy, *dsum; // backward; x holds s
    uint16_t *dx;
    float *partial;         // [blocks, 2, cols] column sums of each block, or, in a cluster,
    float *dgamma, *dbeta;  // the results themselves
};

constexpr int kClusterBlocks = 8;

template <bool kBf16>
__device__ __forceinline__ float2 unpack(uint32_t v)
{
    if (kBf16)
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
    __half2 h;
    memcpy(&h, &v, 4);
    return __half22float2(h);
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack(float lo, float hi)
{
    uint32_t r;
    if (kBf16)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint4 load16(const uint16_t *p)
{
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// Sums of N values over the group's threads; `slot` is the group's [warps][N] scratch.  The
// caller alternates slots: a slot is rewritten only after a later barrier.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float *slot, int warps, int barrier, int threads)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int o = 16; o; o >>= 1)
            v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (warps == 1)
        return;
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N; ++i)
            slot[warp * N + i] = v[i];
    asm volatile("barrier.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i)
        v[i] = 0.0f;
    for (int w = 0; w < warps; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] += slot[w * N + i];
}

__device__ __forceinline__ void load_floats(float (&f)[8], const float *p)
{
    const float4 lo = *reinterpret_cast<const float4 *>(p), hi = *reinterpret_cast<const float4 *>(p + 4);
    f[0] = lo.x, f[1] = lo.y, f[2] = lo.z, f[3] = lo.w;
    f[4] = hi.x, f[5] = hi.y, f[6] = hi.z, f[7] = hi.w;
}

// blockDim = (group_threads, groups).
template <int R, bool kBf16>
__global__ void __launch_bounds__(kMaxThreads, 1) forward_kernel(const Params p)
{
    __shared__ float scratch[2][kMaxGroups][16 * R];
    griddepcontrol_wait();
    griddepcontrol_launch_dependents();
    const int group = threadIdx.y, barrier = 1 + group;
    const int warps = p.group_threads / 32;
    const int col = threadIdx.x * 8;
    const bool active = col < p.cols;
    const float inv_cols = 1.0f / static_cast<float>(p.cols);
    float gamma[8] = {}, beta[8] = {};
    if (active) {
        load_floats(gamma, p.gamma + col);
        load_floats(beta, p.beta + col);
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * p.groups * R;
    for (int64_t row0 = (static_cast<int64_t>(blockIdx.x) * p.groups + group) * R; row0 < p.rows; row0 += step) {
        uint4 s[R], r[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            s[i] = r[i] = make_uint4(0u, 0u, 0u, 0u);
            if (active && row0 + i < p.rows) {
                s[i] = load16(p.x + (row0 + i) * p.cols + col);
                if (p.residual)
                    r[i] = load16(p.residual + (row0 + i) * p.cols + col);
            }
        }
        float total[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            uint32_t *sv = &s[i].x;
            const uint32_t *rv = &r[i].x;
            total[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 a = unpack<kBf16>(sv[j]);
                if (p.residual) {
                    // The residual stream is held in 16 bits: the norm reads the rounded sum.
                    const float2 b = unpack<kBf16>(rv[j]);
                    sv[j] = pack<kBf16>(a.x + b.x, a.y + b.y);
                    a = unpack<kBf16>(sv[j]);
                }
                total[i] += a.x + a.y;
            }
            if (p.sum && active && row0 + i < p.rows)
                *reinterpret_cast<uint4 *>(p.sum + (row0 + i) * p.cols + col) = s[i];
        }
        group_sum<R>(total, scratch[0][group], warps, barrier, p.group_threads);
        float var[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            total[i] *= inv_cols;
            var[i] = 0.0f;
            const uint32_t *sv = &s[i].x;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 a = unpack<kBf16>(sv[j]);
                const float u = a.x - total[i], v = a.y - total[i];
                var[i] += u * u + v * v;
            }
            if (!active)
                var[i] = 0.0f;
        }
        group_sum<R>(var, scratch[1][group], warps, barrier, p.group_threads);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (row0 + i >= p.rows)
                break;
            const float mean = total[i], rstd = rsqrtf(fmaf(var[i], inv_cols, p.eps));
            if (threadIdx.x == 0) {
                p.stats[row0 + i] = mean;
                p.stats[p.rows + row0 + i] = rstd;
            }
            if (!active)
                continue;
            const uint32_t *sv = &s[i].x;
            uint32_t out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 a = unpack<kBf16>(sv[j]);
                out[j] = pack<kBf16>(fmaf((a.x - mean) * rstd, gamma[2 * j], beta[2 * j]),
                                     fmaf((a.y - mean) * rstd, gamma[2 * j + 1], beta[2 * j + 1]));
            }
            *reinterpret_cast<uint4 *>(p.y + (row0 + i) * p.cols + col) = make_uint4(out[0], out[1], out[2], out[3]);
        }
    }
}

// kCluster: the grid is one cluster of eight blocks, which add up their column sums through
// distributed shared memory, so few rows need neither a workspace nor a second launch.
template <int R, bool kBf16, bool kCluster>
__global__ void __launch_bounds__(kMaxThreads, 1) backward_kernel(const Params p)
{
    __shared__ float scratch[2][kMaxGroups][16 * 2 * R];
    extern __shared__ float column_sums[]; // [groups - 1 (kCluster: groups)][2][cols]
    griddepcontrol_wait();
    griddepcontrol_launch_dependents();
    const int group = threadIdx.y, barrier = 1 + group;
    const int warps = p.group_threads / 32;
    const int col = threadIdx.x * 8;
    const bool active = col < p.cols;
    const float inv_cols = 1.0f / static_cast<float>(p.cols);
    float gamma[8] = {};
    if (active)
        load_floats(gamma, p.gamma + col);
    float dgamma[8] = {}, dbeta[8] = {};
    int turn = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * p.groups * R;
    for (int64_t row0 = (static_cast<int64_t>(blockIdx.x) * p.groups + group) * R; row0 < p.rows;
         row0 += step, turn ^= 1) {
        uint4 dy[R], s[R], ds[R];
        float mean[R], rstd[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            dy[i] = s[i] = ds[i] = make_uint4(0u, 0u, 0u, 0u);
            mean[i] = rstd[i] = 0.0f;
            if (row0 + i < p.rows) {
                const int64_t at = (row0 + i) * p.cols + col;
                if (active) {
                    dy[i] = load16(p.dy + at);
                    s[i] = load16(p.x + at);
                    if (p.dsum)
                        ds[i] = load16(p.dsum + at);
                }
                mean[i] = __ldg(p.stats + row0 + i);
                rstd[i] = __ldg(p.stats + p.rows + row0 + i);
            }
        }
        float sums[2 * R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            sums[2 * i] = sums[2 * i + 1] = 0.0f;
            const uint32_t *dv = &dy[i].x, *sv = &s[i].x;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 d = unpack<kBf16>(dv[j]), a = unpack<kBf16>(sv[j]);
                const float h0 = (a.x - mean[i]) * rstd[i], h1 = (a.y - mean[i]) * rstd[i];
                const float w0 = d.x * gamma[2 * j], w1 = d.y * gamma[2 * j + 1];
                sums[2 * i] += w0 + w1;
                sums[2 * i + 1] += w0 * h0 + w1 * h1;
                dgamma[2 * j] = fmaf(d.x, h0, dgamma[2 * j]);
                dgamma[2 * j + 1] = fmaf(d.y, h1, dgamma[2 * j + 1]);
                dbeta[2 * j] += d.x;
                dbeta[2 * j + 1] += d.y;
            }
        }
        if (!p.dx)
            continue;
        group_sum<2 * R>(sums, scratch[turn][group], warps, barrier, p.group_threads);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (row0 + i >= p.rows || !active)
                break;
            const float mw = sums[2 * i] * inv_cols, mwh = sums[2 * i + 1] * inv_cols;
            const uint32_t *dv = &dy[i].x, *sv = &s[i].x, *ev = &ds[i].x;
            uint32_t out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 d = unpack<kBf16>(dv[j]), a = unpack<kBf16>(sv[j]), e = unpack<kBf16>(ev[j]);
                const float h0 = (a.x - mean[i]) * rstd[i], h1 = (a.y - mean[i]) * rstd[i];
                const float g0 = fmaf(d.x, gamma[2 * j], -mw) - h0 * mwh;
                const float g1 = fmaf(d.y, gamma[2 * j + 1], -mw) - h1 * mwh;
                out[j] = pack<kBf16>(fmaf(g0, rstd[i], e.x), fmaf(g1, rstd[i], e.y));
            }
            *reinterpret_cast<uint4 *>(p.dx + (row0 + i) * p.cols + col) = make_uint4(out[0], out[1], out[2], out[3]);
        }
    }
    if (!p.dgamma)
        return;
    // The block's column sums, groups in order: the result does not depend on timing.
    if (group > 0 && active) {
        float *mine = column_sums + static_cast<size_t>(group - 1) * 2 * p.cols + col;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            mine[i] = dgamma[i];
            mine[p.cols + i] = dbeta[i];
        }
    }
    __syncthreads();
    float *block_sums = kCluster ? column_sums + static_cast<size_t>(p.groups - 1) * 2 * p.cols
                                 : p.partial + static_cast<size_t>(blockIdx.x) * 2 * p.cols;
    if (group == 0 && active) {
        for (int g = 0; g + 1 < p.groups; ++g) {
            const float *other = column_sums + static_cast<size_t>(g) * 2 * p.cols + col;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dgamma[i] += other[i];
                dbeta[i] += other[p.cols + i];
            }
        }
        float *out = block_sums + col;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            *reinterpret_cast<float4 *>(out + i) = make_float4(dgamma[i], dgamma[i + 1], dgamma[i + 2], dgamma[i + 3]);
            *reinterpret_cast<float4 *>(out + p.cols + i) =
                make_float4(dbeta[i], dbeta[i + 1], dbeta[i + 2], dbeta[i + 3]);
        }
    }
    if (kCluster) {
        cluster_sync();
        const uint32_t local = smem_u32(block_sums);
        const int thread = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
        for (int c = blockIdx.x * threads + thread; c < 2 * p.cols; c += kClusterBlocks * threads) {
            float v = 0.0f;
#pragma unroll
            for (uint32_t b = 0; b < kClusterBlocks; ++b)
                v += ld_shared_cluster_f32(map_to_rank(local + 4u * static_cast<uint32_t>(c), b));
            (c < p.cols ? p.dgamma : p.dbeta)[c < p.cols ? c : c - p.cols] = v;
        }
        cluster_sync(); // the peers' sums stay until every block has read them
    }
}

// Sums the blocks' partial dgamma | dbeta rows: 32 columns per block, 32 rows at a time.
__global__ void __launch_bounds__(1024) columns_kernel(const float *partial, int blocks, int cols, float *dgamma,
                                                       float *dbeta)
{
    __shared__ float sums[32][33];
    griddepcontrol_wait();
    griddepcontrol_launch_dependents();
    const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (c < 2 * cols)
        for (int b = part; b < blocks; b += 32)
            v += partial[static_cast<size_t>(b) * 2 * cols + c];
    sums[part][lane] = v;
    __syncthreads();
    // Warp `part` adds up column `part` of this block.
    v = sums[lane][part];
#pragma unroll
    for (int o = 16; o; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    const int out = blockIdx.x * 32 + part;
    if (lane == 0 && out < 2 * cols)
        (out < cols ? dgamma : dbeta)[out < cols ? out : out - cols] = v;
}

} // namespace tnorm

namespace {

using namespace tnorm;

int group_threads(int64_t cols) { return static_cast<int>((cols / 8 + 31) / 32 * 32); }
int group_count(int64_t cols) { return std::min(kMaxGroups, std::max(1, kMaxThreads / group_threads(cols))); }

// Rows per step: several once every group of the GPU has that many, else one, which spreads
// few rows over the most groups.
int grid_blocks(int64_t rows, int64_t cols, int rows_per_step)
{
    const int64_t per_block = static_cast<int64_t>(group_count(cols)) * rows_per_step;
    return static_cast<int>(std::min<int64_t>((rows + per_block - 1) / per_block, sm_count()));
}

constexpr int kForwardRows = 4, kBackwardRows = 2;

bool many_rows(int64_t rows, int64_t cols, int rows_per_step)
{
    return rows >= static_cast<int64_t>(sm_count()) * group_count(cols) * rows_per_step;
}

// Rows that one cluster of eight blocks handles in at most four steps of its groups, as fast
// as the whole GPU and a second launch would (20 x 1280: 4.2 + 2.1 us and the launch against
// one of 5 us).
bool one_cluster(int64_t rows, int64_t cols)
{
    return rows <= 4 * int64_t{kClusterBlocks} * group_count(cols) * kBackwardRows;
}

int backward_blocks(int64_t rows, int64_t cols)
{
    return grid_blocks(rows, cols, many_rows(rows, cols, kBackwardRows) ? kBackwardRows : 1);
}

template <class Kernel>
cudaError_t launch_groups(Kernel kernel, int blocks, int cluster, size_t smem, cudaStream_t stream, const Params &p)
{
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(blocks));
    config.blockDim = dim3(static_cast<unsigned>(p.group_threads), static_cast<unsigned>(p.groups));
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    config.attrs = attrs;
    config.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, kernel, p);
    count_launch();
    return err != cudaSuccess ? err : cudaGetLastError();
}

template <bool kBf16>
cudaError_t run_forward(const LayerNormTrainLaunch &L, const Params &p, cudaStream_t stream)
{
    if (many_rows(L.rows, L.cols, kForwardRows))
        return launch_groups(forward_kernel<kForwardRows, kBf16>, grid_blocks(L.rows, L.cols, kForwardRows), 1, 0,
                             stream, p);
    return launch_groups(forward_kernel<1, kBf16>, grid_blocks(L.rows, L.cols, 1), 1, 0, stream, p);
}

// Shared memory of the column sums: groups x 2 x cols floats, where groups x cols is at most
// 640 threads' 8 columns each (40 KB), under the 48 KB that every launch may use.
template <bool kBf16>
cudaError_t run_backward(const LayerNormTrainLaunch &L, const Params &p, cudaStream_t stream)
{
    const size_t sums = L.dgamma ? 2 * L.cols * sizeof(float) : 0;
    if (L.dgamma && one_cluster(L.rows, L.cols))
        return launch_groups(backward_kernel<kBackwardRows, kBf16, true>, kClusterBlocks, kClusterBlocks,
                             p.groups * sums, stream, p);
    const int blocks = backward_blocks(L.rows, L.cols);
    cudaError_t err = many_rows(L.rows, L.cols, kBackwardRows)
                          ? launch_groups(backward_kernel<kBackwardRows, kBf16, false>, blocks, 1,
                                          (p.groups - 1) * sums, stream, p)
                          : launch_groups(backward_kernel<1, kBf16, false>, blocks, 1, (p.groups - 1) * sums, stream, p);
    if (err == cudaSuccess && L.dgamma)
        err = launch_pdl(columns_kernel, dim3(static_cast<unsigned>((2 * L.cols + 31) / 32)), dim3(1024), stream,
                         static_cast<const float *>(p.partial), blocks, p.cols, L.dgamma, L.dbeta);
    return err;
}

} // namespace

int64_t layer_norm_grad_workspace(int64_t rows, int64_t cols)
{
    if (one_cluster(rows, cols))
        return 0;
    return static_cast<int64_t>(backward_blocks(rows, cols)) * 2 * cols * static_cast<int64_t>(sizeof(float));
}

cudaError_t launch_layer_norm_forward(const LayerNormTrainLaunch &L, cudaStream_t stream)
{
    Params p{};
    p.rows = L.rows;
    p.cols = static_cast<int>(L.cols);
    p.groups = group_count(L.cols);
    p.group_threads = group_threads(L.cols);
    p.x = L.x;
    p.residual = L.residual;
    p.sum = L.sum_out;
    p.y = L.y;
    p.gamma = L.gamma;
    p.beta = L.beta;
    p.eps = L.eps;
    p.stats = L.stats;
    return L.bf16 ? run_forward<true>(L, p, stream) : run_forward<false>(L, p, stream);
}

cudaError_t launch_layer_norm_backward(const LayerNormTrainLaunch &L, cudaStream_t stream)
{
    Params p{};
    p.rows = L.rows;
    p.cols = static_cast<int>(L.cols);
    p.groups = group_count(L.cols);
    p.group_threads = group_threads(L.cols);
    p.x = L.x;
    p.dy = L.dy;
    p.dsum = L.dsum;
    p.dx = L.dx;
    p.gamma = L.gamma;
    p.stats = L.stats;
    p.partial = static_cast<float *>(L.workspace);
    p.dgamma = L.dgamma;
    p.dbeta = L.dbeta;
    return L.bf16 ? run_backward<true>(L, p, stream) : run_backward<false>(L, p, stream);
}

} // namespace lffw
