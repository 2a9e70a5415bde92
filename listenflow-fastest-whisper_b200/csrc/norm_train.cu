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
// loads; R rows per step share the barriers of the row sums.
//
// With many rows each group has a ring of stages in shared memory, filled by bulk copies several
// steps ahead, so that the bytes in flight depend neither on registers nor on where in its step
// a group is.  With few rows (latency counts) the threads load their columns themselves.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstring>

#include "host_util.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace lffw {

namespace tnorm {

constexpr int kMaxThreads = 640;
constexpr int kMaxGroups = 15; // named barriers 1-15
constexpr int kMaxDepth = 8;

struct Params {
    int64_t rows;
    int cols, groups, group_threads;
    int depth; // stages of a group's ring
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

// fp32 pairs: one instruction rounds both lanes.
__device__ __forceinline__ uint64_t bits(float2 a)
{
    uint64_t x;
    memcpy(&x, &a, 8);
    return x;
}
__device__ __forceinline__ float2 pair(uint64_t x)
{
    float2 f;
    memcpy(&f, &x, 8);
    return f;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return pair(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return pair(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
    return pair(r);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

template <bool kBf16>
__device__ __forceinline__ uint32_t pack(float2 v)
{
    const float lo = v.x, hi = v.y;
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

// Waits, 2 s at most, for copies that a group's wait has given up on.
__device__ __forceinline__ bool landed_late(uint32_t bar, uint32_t parity)
{
    const uint64_t start = global_timer_ns();
    while (global_timer_ns() - start < 2000000000ull)
        if (mbar_try_wait(bar, parity))
            return true;
    return false;
}

// A group's ring.  A stage holds up to R rows of each of N arrays; the steps take the stages in
// turn.
template <int N, int R>
struct Ring {
    const uint16_t *arrays[N]; // null: not read
    uint32_t bars, data;       // shared-memory addresses
    int depth, cols;
    int64_t rows;
    int count; // arrays that are read
    int stage = 0;
    uint32_t phase = 0;

    __device__ __forceinline__ uint32_t row_bytes() const { return 2u * static_cast<uint32_t>(cols); }
    __device__ __forceinline__ uint32_t stage_at(int k) const
    {
        return data + static_cast<uint32_t>(k * N * R) * row_bytes();
    }
    // One thread: requests the rows from row0 on into stage k.
    __device__ __forceinline__ void fill(int k, int64_t row0) const
    {
        if (row0 >= rows)
            return;
        const int64_t left = rows - row0;
        const uint32_t bytes = static_cast<uint32_t>(left < R ? left : R) * row_bytes();
        mbar_arrive_expect_tx(bars + 8 * k, count * bytes);
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (arrays[n])
                bulk_load(stage_at(k) + static_cast<uint32_t>(n * R) * row_bytes(), arrays[n] + row0 * cols, bytes,
                          bars + 8 * k);
    }
    // All threads: the current stage's rows have landed (or the wait gave up and set the error
    // word; the group then goes on with what is there, so that its barriers are met).
    __device__ __forceinline__ void wait() const { mbar_wait(bars + 8 * stage, phase, kSiteProducerEmpty); }
    // One thread, once all of the group have read the current stage: requests the rows from row0 on
    // into it.  Where the wait gave up, the copies in flight are waited for first, in a group's last
    // steps too, so that none lands after the block has left its shared memory or reuses it.  (The
    // test costs nothing: 96000 x 1280, each direction alone, 176 and 156 us without it, 170 and 152
    // with it; the same after the steps instead of in them kept registers from these: 182 and 189.)
    __device__ __forceinline__ void refill(int64_t row0) const
    {
        if (mbar_test(bars + 8 * stage, phase) || landed_late(bars + 8 * stage, phase))
            fill(stage, row0);
    }
    // Eight columns of a row of the current stage.
    __device__ __forceinline__ uint4 load(uint32_t stage_col, int array, int row) const
    {
        uint4 v;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(stage_col + static_cast<uint32_t>(array * R + row) * row_bytes()));
        return v;
    }
    __device__ __forceinline__ void advance()
    {
        if (++stage == depth) {
            stage = 0;
            phase ^= 1u;
        }
    }
};

// The ring of this thread's group; its barriers are ready once the block has synchronised.
template <int N, int R>
__device__ __forceinline__ Ring<N, R> make_ring(uint64_t *bars, uint8_t *data, const Params &p)
{
    Ring<N, R> ring;
    const int group = threadIdx.y;
    ring.bars = smem_u32(bars + group * kMaxDepth);
    ring.depth = p.depth;
    ring.cols = p.cols;
    ring.rows = p.rows;
    ring.data = smem_u32(data) + static_cast<uint32_t>(group * p.depth * N * R) * ring.row_bytes();
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.depth; ++i)
            mbar_init(ring.bars + 8 * i, 1);
        fence_barrier_init();
    }
    __syncthreads();
    return ring;
}

// Sums of N (1, 2 or 4) values over the group's threads; `slot` is the group's [warps][N]
// scratch.  The caller alternates slots: a slot is rewritten only after a later barrier.
// Within a warp the values are halved along with the lanes (lanes 16-31 carry on with the
// second half of them, and so on), which takes N + 4 - log2(N) exchanges instead of 5 N.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float *slot, int warps, int barrier, int threads)
{
    static_assert(N == 1 || N == 2 || N == 4, "values");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float one;
    if (N == 4) {
        const bool high = lane & 16, odd = lane & 8;
        float a = high ? v[N / 2] : v[0], b = high ? v[N - 1] : v[1 % N];
        a += __shfl_xor_sync(0xffffffffu, high ? v[0] : v[N / 2], 16);
        b += __shfl_xor_sync(0xffffffffu, high ? v[1 % N] : v[N - 1], 16);
        one = odd ? b : a;
        one += __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
    } else if (N == 2) {
        const bool high = lane & 16;
        one = high ? v[N - 1] : v[0];
        one += __shfl_xor_sync(0xffffffffu, high ? v[0] : v[N - 1], 16);
        one += __shfl_xor_sync(0xffffffffu, one, 8);
    } else {
        one = v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
        one += __shfl_xor_sync(0xffffffffu, one, 8);
    }
#pragma unroll
    for (int o = 4; o; o >>= 1)
        one += __shfl_xor_sync(0xffffffffu, one, o);
    // Value i is now in the lanes from 32 i / N on.
    if (warps == 1) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] = __shfl_sync(0xffffffffu, one, 32 / N * i);
        __syncwarp(); // a barrier for memory too, as below: the caller may refill what was read
        return;
    }
    if (lane % (32 / N) == 0)
        slot[warp * N + lane / (32 / N)] = one;
    asm volatile("barrier.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
    if (N == 4) {
        float2 lo = both(0.0f), hi = both(0.0f);
        for (int w = 0; w < warps; ++w) {
            const float4 other = *reinterpret_cast<const float4 *>(slot + 4 * w);
            lo = add2(lo, make_float2(other.x, other.y));
            hi = add2(hi, make_float2(other.z, other.w));
        }
        v[0] = lo.x, v[1 % N] = lo.y, v[N / 2] = hi.x, v[N - 1] = hi.y;
    } else if (N == 2) {
        float2 sum = both(0.0f);
        for (int w = 0; w < warps; ++w)
            sum = add2(sum, *reinterpret_cast<const float2 *>(slot + 2 * w));
        v[0] = sum.x, v[N - 1] = sum.y;
    } else {
        v[0] = 0.0f;
        for (int w = 0; w < warps; ++w)
            v[0] += slot[w];
    }
}

__device__ __forceinline__ void load_floats(float2 (&f)[4], const float *p)
{
    const float4 lo = *reinterpret_cast<const float4 *>(p), hi = *reinterpret_cast<const float4 *>(p + 4);
    f[0] = make_float2(lo.x, lo.y), f[1] = make_float2(lo.z, lo.w);
    f[2] = make_float2(hi.x, hi.y), f[3] = make_float2(hi.z, hi.w);
}

// blockDim = (group_threads, groups).
template <int R, bool kBf16, bool kRing>
__global__ void __launch_bounds__(kMaxThreads, 1) forward_kernel(const Params p)
{
    __shared__ __align__(16) float scratch[2][kMaxGroups][16 * R];
    __shared__ uint64_t bars[kRing ? kMaxGroups * kMaxDepth : 1];
    extern __shared__ __align__(128) uint8_t ring_data[];
    Ring<2, R> ring;
    if (kRing)
        ring = make_ring<2, R>(bars, ring_data, p);
    griddepcontrol_wait();
    griddepcontrol_launch_dependents();
    const int group = threadIdx.y, barrier = 1 + group;
    const int warps = p.group_threads / 32;
    const int col = threadIdx.x * 8;
    const bool active = col < p.cols;
    const float inv_cols = 1.0f / static_cast<float>(p.cols);
    float2 gamma[4] = {}, beta[4] = {};
    if (active) {
        load_floats(gamma, p.gamma + col);
        load_floats(beta, p.beta + col);
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * p.groups * R;
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * p.groups + group) * R;
    if (kRing) {
        ring.arrays[0] = p.x;
        ring.arrays[1] = p.residual;
        ring.count = p.residual ? 2 : 1;
        if (threadIdx.x == 0)
            for (int i = 0; i < p.depth; ++i)
                ring.fill(i, first + i * step);
    }
    for (int64_t row0 = first; row0 < p.rows; row0 += step) {
        uint4 s[R], r[R];
        const uint32_t stage_col = ring.stage_at(ring.stage) + 2u * static_cast<uint32_t>(col);
        if (kRing)
            ring.wait();
#pragma unroll
        for (int i = 0; i < R; ++i) {
            s[i] = r[i] = make_uint4(0u, 0u, 0u, 0u);
            if (kRing) {
                if (active && row0 + i < p.rows) {
                    s[i] = ring.load(stage_col, 0, i);
                    if (p.residual)
                        r[i] = ring.load(stage_col, 1, i);
                }
            } else if (active && row0 + i < p.rows) {
                s[i] = load16(p.x + (row0 + i) * p.cols + col);
                if (p.residual)
                    r[i] = load16(p.residual + (row0 + i) * p.cols + col);
            }
        }
        float total[R];
        float2 f[R][4]; // the summed row, then its distance from the mean
#pragma unroll
        for (int i = 0; i < R; ++i) {
            uint32_t *sv = &s[i].x;
            const uint32_t *rv = &r[i].x;
            float2 sum = both(0.0f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[i][j] = unpack<kBf16>(sv[j]);
                if (p.residual) {
                    // The residual stream is held in 16 bits: the norm reads the rounded sum.
                    sv[j] = pack<kBf16>(add2(f[i][j], unpack<kBf16>(rv[j])));
                    f[i][j] = unpack<kBf16>(sv[j]);
                }
                sum = add2(sum, f[i][j]);
            }
            total[i] = sum.x + sum.y;
            if (p.sum && active && row0 + i < p.rows)
                *reinterpret_cast<uint4 *>(p.sum + (row0 + i) * p.cols + col) = s[i];
        }
        group_sum<R>(total, scratch[0][group], warps, barrier, p.group_threads);
        // Every thread of the group has read the step's stage.
        if (kRing && threadIdx.x == 0)
            ring.refill(row0 + p.depth * step);
        if (kRing)
            ring.advance();
        float var[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            total[i] *= inv_cols;
            float2 sum = both(0.0f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[i][j] = add2(f[i][j], both(-total[i]));
                sum = fma2(f[i][j], f[i][j], sum);
            }
            var[i] = active ? sum.x + sum.y : 0.0f;
        }
        group_sum<R>(var, scratch[1][group], warps, barrier, p.group_threads);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (row0 + i >= p.rows)
                break;
            const float rstd = rsqrtf(fmaf(var[i], inv_cols, p.eps));
            if (threadIdx.x == 0) {
                p.stats[row0 + i] = total[i];
                p.stats[p.rows + row0 + i] = rstd;
            }
            if (!active)
                continue;
            uint32_t out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                out[j] = pack<kBf16>(fma2(mul2(f[i][j], both(rstd)), gamma[j], beta[j]));
            *reinterpret_cast<uint4 *>(p.y + (row0 + i) * p.cols + col) = make_uint4(out[0], out[1], out[2], out[3]);
        }
    }
}

// kCluster: the grid is one cluster of eight blocks, which add up their column sums through
// distributed shared memory, so few rows need neither a workspace nor a second launch.
template <int R, bool kBf16, bool kCluster, bool kRing>
__global__ void __launch_bounds__(kMaxThreads, 1) backward_kernel(const Params p)
{
    __shared__ __align__(16) float scratch[2][kMaxGroups][16 * 2 * R];
    __shared__ uint64_t bars[kRing ? kMaxGroups * kMaxDepth : 1];
    // The rings, and after the last row (in their place) the column sums
    // [groups - 1 (kCluster: groups)][2][cols].
    extern __shared__ __align__(128) uint8_t ring_data[];
    float *column_sums = reinterpret_cast<float *>(ring_data);
    Ring<3, R> ring;
    if (kRing)
        ring = make_ring<3, R>(bars, ring_data, p);
    griddepcontrol_wait();
    griddepcontrol_launch_dependents();
    const int group = threadIdx.y, barrier = 1 + group;
    const int warps = p.group_threads / 32;
    const int col = threadIdx.x * 8;
    const bool active = col < p.cols;
    const float inv_cols = 1.0f / static_cast<float>(p.cols);
    float2 gamma[4] = {};
    if (active)
        load_floats(gamma, p.gamma + col);
    float2 dgamma[4] = {}, dbeta[4] = {};
    const int64_t step = static_cast<int64_t>(gridDim.x) * p.groups * R;
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * p.groups + group) * R;
    if (kRing) {
        ring.arrays[0] = p.dy;
        ring.arrays[1] = p.x;
        ring.arrays[2] = p.dsum;
        ring.count = p.dsum ? 3 : 2;
        if (threadIdx.x == 0)
            for (int i = 0; i < p.depth; ++i)
                ring.fill(i, first + i * step);
    }
    // The statistics of the next step's rows are requested a step ahead.
    float next_mean[R], next_rstd[R];
    auto load_stats = [&](int64_t row0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            next_mean[i] = row0 + i < p.rows ? p.stats[row0 + i] : 0.0f;
            next_rstd[i] = row0 + i < p.rows ? p.stats[p.rows + row0 + i] : 0.0f;
        }
    };
    load_stats(first);
    int turn = 0;
    for (int64_t row0 = first; row0 < p.rows; row0 += step, turn ^= 1) {
        uint4 dy[R], s[R], ds[R];
        float mean[R], rstd[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            dy[i] = s[i] = ds[i] = make_uint4(0u, 0u, 0u, 0u);
            mean[i] = next_mean[i];
            rstd[i] = next_rstd[i];
            if (row0 + i < p.rows) {
                const int64_t at = (row0 + i) * p.cols + col;
                if (active && !kRing) {
                    dy[i] = load16(p.dy + at);
                    s[i] = load16(p.x + at);
                    if (p.dsum)
                        ds[i] = load16(p.dsum + at);
                }
            }
        }
        load_stats(row0 + step);
        if (kRing) {
            const uint32_t stage_col = ring.stage_at(ring.stage) + 2u * static_cast<uint32_t>(col);
            ring.wait();
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (active && row0 + i < p.rows) {
                    dy[i] = ring.load(stage_col, 0, i);
                    s[i] = ring.load(stage_col, 1, i);
                    if (p.dsum)
                        ds[i] = ring.load(stage_col, 2, i);
                }
        }
        float sums[2 * R];
        float2 w[R][4], h[R][4];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const uint32_t *dv = &dy[i].x, *sv = &s[i].x;
            float2 sw = both(0.0f), swh = both(0.0f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 d = unpack<kBf16>(dv[j]);
                h[i][j] = mul2(add2(unpack<kBf16>(sv[j]), both(-mean[i])), both(rstd[i]));
                w[i][j] = mul2(d, gamma[j]);
                sw = add2(sw, w[i][j]);
                swh = fma2(w[i][j], h[i][j], swh);
                dgamma[j] = fma2(d, h[i][j], dgamma[j]);
                dbeta[j] = add2(dbeta[j], d);
            }
            sums[2 * i] = sw.x + sw.y;
            sums[2 * i + 1] = swh.x + swh.y;
        }
        if (!kRing && !p.dx)
            continue;
        group_sum<2 * R>(sums, scratch[turn][group], warps, barrier, p.group_threads);
        // Every thread of the group has read the step's stage.
        if (kRing && threadIdx.x == 0)
            ring.refill(row0 + p.depth * step);
        if (kRing)
            ring.advance();
        if (!p.dx)
            continue;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (row0 + i >= p.rows || !active)
                break;
            const float2 mw = both(-sums[2 * i] * inv_cols), mwh = both(-sums[2 * i + 1] * inv_cols);
            const uint32_t *ev = &ds[i].x;
            uint32_t out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                out[j] = pack<kBf16>(fma2(fma2(h[i][j], mwh, add2(w[i][j], mw)), both(rstd[i]), unpack<kBf16>(ev[j])));
            *reinterpret_cast<uint4 *>(p.dx + (row0 + i) * p.cols + col) = make_uint4(out[0], out[1], out[2], out[3]);
        }
    }
    if (!p.dgamma)
        return;
    // The block's column sums, groups in order: the result does not depend on timing.
    if (kRing)
        __syncthreads(); // every group is done with its ring
    if (group > 0 && active) {
        float2 *mine = reinterpret_cast<float2 *>(column_sums + static_cast<size_t>(group - 1) * 2 * p.cols + col);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mine[j] = dgamma[j];
            mine[p.cols / 2 + j] = dbeta[j];
        }
    }
    __syncthreads();
    float *block_sums = kCluster ? column_sums + static_cast<size_t>(p.groups - 1) * 2 * p.cols
                                 : p.partial + static_cast<size_t>(blockIdx.x) * 2 * p.cols;
    if (group == 0 && active) {
        for (int g = 0; g + 1 < p.groups; ++g) {
            const float2 *other =
                reinterpret_cast<const float2 *>(column_sums + static_cast<size_t>(g) * 2 * p.cols + col);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                dgamma[j] = add2(dgamma[j], other[j]);
                dbeta[j] = add2(dbeta[j], other[p.cols / 2 + j]);
            }
        }
        float2 *out = reinterpret_cast<float2 *>(block_sums + col);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            out[j] = dgamma[j];
            out[p.cols / 2 + j] = dbeta[j];
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

// Blocks that share the rows, at most one per SM.
int grid_blocks(int64_t rows, int64_t cols, int rows_per_step)
{
    const int64_t per_block = static_cast<int64_t>(group_count(cols)) * rows_per_step;
    return static_cast<int>(std::min<int64_t>((rows + per_block - 1) / per_block, sm_count()));
}

constexpr int kForwardRows = 2, kBackwardRows = 2;
constexpr int kRingBytes = 200 * 1024; // a block's rings

// Rings and several rows per step once every group of the GPU has that many rows, else one row
// per step, which spreads few rows over the most groups.  Forward of 512 x 1280: 2.7 us without
// rings, 3.3 with; 1184 x 1280: 4.1 and 3.5; 4000 x 1280: 11.0 and 8.3.
bool many_rows(int64_t rows, int64_t cols, int rows_per_step)
{
    return rows >= static_cast<int64_t>(sm_count()) * group_count(cols) * rows_per_step;
}

// Rows that one cluster of eight blocks handles in at most three steps of its groups.  It needs
// one launch and no workspace, some 4 us of a caller's time, and on the GPU takes as long as
// two launches over all SMs for one step (64 x 1280: 6.8 us against 6.2) and 2 to 4 us longer
// for three (128 x 1280: 8.2 against 5.8; at 256 rows it would be 11.5 against 6.2).
bool one_cluster(int64_t rows, int64_t cols)
{
    return rows <= 3 * int64_t{kClusterBlocks} * group_count(cols) * kBackwardRows;
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

// The kernel over rings: as many stages as fit.
template <auto kKernel>
cudaError_t launch_ring(int blocks, int stage_rows, size_t least, cudaStream_t stream, Params p)
{
    const int64_t stage = static_cast<int64_t>(p.groups) * stage_rows * p.cols * 2;
    p.depth = static_cast<int>(std::min<int64_t>(kMaxDepth, kRingBytes / stage));
    static std::atomic<bool> opted[kMaxDevices];
    const int device = current_device();
    if (!opted[device].load(std::memory_order_acquire)) {
        const cudaError_t err = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
        if (err != cudaSuccess)
            return err;
        opted[device].store(true, std::memory_order_release);
    }
    return launch_groups(kKernel, blocks, 1, std::max(static_cast<size_t>(p.depth * stage), least), stream, p);
}

template <bool kBf16>
cudaError_t run_forward(const LayerNormTrainLaunch &L, const Params &p, cudaStream_t stream)
{
    if (many_rows(L.rows, L.cols, kForwardRows))
        return launch_ring<forward_kernel<kForwardRows, kBf16, true>>(grid_blocks(L.rows, L.cols, kForwardRows),
                                                                      2 * kForwardRows, 0, stream, p);
    return launch_groups(forward_kernel<1, kBf16, false>, grid_blocks(L.rows, L.cols, 1), 1, 0, stream, p);
}

// Shared memory of the column sums: groups x 2 x cols floats, where groups x cols is at most
// 640 threads' 8 columns each (40 KB), under the 48 KB that every launch may use.
template <bool kBf16>
cudaError_t run_backward(const LayerNormTrainLaunch &L, const Params &p, cudaStream_t stream)
{
    const size_t sums = L.dgamma ? 2 * L.cols * sizeof(float) : 0;
    if (L.dgamma && one_cluster(L.rows, L.cols))
        return launch_groups(backward_kernel<kBackwardRows, kBf16, true, false>, kClusterBlocks, kClusterBlocks,
                             p.groups * sums, stream, p);
    const int blocks = backward_blocks(L.rows, L.cols);
    cudaError_t err = many_rows(L.rows, L.cols, kBackwardRows)
                          ? launch_ring<backward_kernel<kBackwardRows, kBf16, false, true>>(
                                blocks, 3 * kBackwardRows, (p.groups - 1) * sums, stream, p)
                          : launch_groups(backward_kernel<1, kBf16, false, false>, blocks, 1, (p.groups - 1) * sums,
                                          stream, p);
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

cudaError_t read_and_clear_norm_wait_error(int *site)
{
    int value = 0;
    cudaError_t err = cudaMemcpyFromSymbol(&value, g_device_error, sizeof(int));
    if (err == cudaSuccess && value != 0) {
        const int zero = 0;
        err = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
    }
    *site = value;
    return err;
}

} // namespace lffw
