// sm_100a kernels of the vocabulary losses: cross entropy against tokens and distillation
// from a teacher's top logits, over the logits z = x W^T of a token table W [V, d], forward
// and backward, without holding the logits.
//
//   loss     lse_i = log sum_v exp(z_iv / T)
//            loss_i = T^2 (sum_j t_ij log t_ij + S_i lse_i - sum_j t_ij z_{i,v_ij} / T)
//            (one target with t = 1 and T = 1: lse_i - z_i,label)
//   gradient G_iv = g_i T (exp(z_iv / T - lse_i) - t_iv),  dx = G W,  dW = G^T x
//
// Everything of size n x V runs through one tensor-core GEMM kernel in three forms:
//   kStats   z tiles, reduced in the epilogue to a running maximum, a sum of exponentials and
//            the targets' logits per row and column slice (merged by combine_kernel)
//   kGrad    z tiles again, turned in the epilogue into a piece of G (16 bits, a range of
//            vocabulary columns)
//   kBack    that piece times its rows of W (dx, summed over the pieces in fp32) and that piece
//            transposed times x (its rows of dW), one list of tiles shared out over the SMs
// A piece of G is the only n x (part of V) tensor that ever exists (all of V where 512 MB hold it).
//
// Rows without a target are left out of the gradients' products altogether.
//
// The work is bound by the tensor cores (2 n V d flops per product, four products in a training
// step: the logits are formed twice because they are not kept) once n exceeds a few hundred
// rows; below that it is bound by streaming W (and writing dW).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "host_util.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace lffw {

namespace vocab {

constexpr int kBM = 128;               // accumulator rows per CTA (TMEM lanes)
constexpr int kBK = 64;                // K elements per stage: one 128-byte swizzle row
constexpr int kUmmaK = 16;             // K of one kind::f16 MMA
constexpr int kSub = 32;               // columns per epilogue step
constexpr int kMaxBN = 256;            // widest tile
constexpr float kLog2e = 1.4426950408889634f;

enum Mode : int { kStats, kGrad, kBack };

// A label or a teacher token outside the vocabulary was met (see lffw_vocab_loss_error).
__device__ int g_token_error = 0;

// kPair: a cluster of two CTAs computes a 256 x bn tile with cta_group::2 MMAs, each CTA
// holding 128 rows of A, bn/2 rows of B and its half of the accumulator.  At 256 x 256 an SM's
// shared memory then takes 64 B/clk of TMA writes and 64 B/clk of MMA reads, its 128 B/clk; a
// 128 x 256 tile of one CTA would want 192.
// Operand layouts in shared memory (128-byte swizzle either way):
//   K-major   rows of 64 K elements, one TMA box
//   MN-major  64 K rows of 64 MN elements per TMA box, boxes stacked along MN
// x and W are K-major for z = x W^T; W is MN-major as B of G W; G and x are MN-major in G^T x.
// The tile width bn (a multiple of 16, of 32 in a pair, up to 256) is a launch parameter: the last dimension is
// cut into equal tiles instead of 256-wide ones and a remainder, and small problems into as
// many as the SMs share evenly.
template <bool kPair, int MODE>
struct Cfg {
    // Epilogue warps: per TMEM lane quarter two, each with half of a tile's columns, or four.
    // kGrad, whose epilogue is the longest, gains from sixteen where K is short (384: 24.8 ->
    // 22.3 us for 333 rows); the others are as fast or faster with eight (7168 x 1280 kStats
    // 634 -> 623 us).
    static constexpr int kEpiWarps = MODE == kGrad ? 16 : 8;
    static constexpr int kParts = kEpiWarps / 4;
    static constexpr int kThreads = 64 + 32 * kEpiWarps; // warp 0 TMA, warp 1 MMA, then the epilogue
    static constexpr int kTileM = kPair ? 2 * kBM : kBM;
    static constexpr int kABytes = kBM * 128;
    static constexpr int kBBytes = (kPair ? kMaxBN / 2 : kMaxBN) * 128; // this CTA's rows of B, at most
    static constexpr int kStageBytes = kABytes + kBBytes;
    // Per epilogue warp: kStats exchanges (maximum, sum, target product) of 32 rows, twice
    // (tile parity); the others stage 32-row x 64-byte stores.
    static constexpr int kBuffers = 16 / kEpiWarps;
    static constexpr int kStaging = MODE == kStats ? 2 * 3 * 32 * 4 : 2048 * kBuffers;
    static constexpr int kBarBytes = 256;
    static constexpr int kBudget = 232448 - 1024;
    static constexpr int kFit = (kBudget - kEpiWarps * kStaging - kBarBytes) / kStageBytes;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    static constexpr int kOffB = kStages * kABytes;
    static constexpr int kOffStaging = kOffB + kStages * kBBytes;
    static constexpr int kOffBar = kOffStaging + kEpiWarps * kStaging;
    static constexpr int kSmemBytes = kOffBar + kBarBytes + 1024;
    static constexpr int kTmemCols = 2 * kMaxBN; // two accumulators
    // Instruction descriptor without its operand types, major axes and N.
    static constexpr uint32_t kIdesc = (1u << 4) | (static_cast<uint32_t>(kTileM >> 4) << 24);
    static_assert(kStages >= 4 && kSmemBytes <= 232448, "shared memory budget");
    static_assert((2 * kStages + 5) * 8 + 8 <= kBarBytes, "barrier area");
};

// Up to this many rows G is held in two parts, its rounding to 16 bits and what that leaves off,
// as further rows from lo_row on (with x's rows once more): the products are then those of an
// unrounded G.  With more rows the roundings of G average out to as much as dx and dW's own
// (1.3 to 1.45 times the error of those alone, measured); with few, single large elements decide
// (1.9 times at 7 rows of 5 teacher's entries), and both parts fit one row tile of dx.  Backward
// over 51866 tokens with one part and with two: 7 x 512 40 and 42 us, 20 x 1280 83 and 87,
// 128 x 1280 93 and 108.
constexpr int kSplitRows = 128;

// The backward's shape, decided on the device once the rows that have a target are counted.
struct BackShape {
    int rows;       // that have a target
    int lo_row;     // where the second part's rows start (0: there is none)
    int all_rows;   // of G and x_used
    int kb_per;     // K blocks of one split of dx
    int splits;     // planes of dx
    int plane_rows; // rows from one plane to the next: all_rows, rounded up to a store's 32
};

// What the choice of dx's splits depends on.
struct BackCosts {
    int kbs, pieces;         // K blocks of dx in a piece, and pieces
    int n_tiles, dw_m_tiles; // tiles across x's width, and of dW down a piece (0: no dW)
    int units;               // CTA pairs
    int width;
    int plane_cap;           // rows of all planes together
    int part_rows;           // what lo_row is a multiple of
};

// A tile's start and epilogue, in K blocks' time (measured: a dW tile of 1 block takes 4.4
// blocks' time, one of 4 blocks 7.2).
constexpr int kTileBlocks = 3;

__host__ __device__ inline int ceil_int(int a, int b) { return (a + b - 1) / b; }

// lo_row for that many rows: whole stores of 32 rows, or (part_rows 8 or 16) a part of one, where a
// call has no more.
__host__ __device__ inline int second_part(int rows, int part_rows)
{
    return rows <= kSplitRows ? ceil_int(rows, part_rows) * part_rows : 0;
}

// Time of the backward's products with about `splits` K splits of dx, in K blocks of a CTA pair
// (infinity: not possible).  dx = G W has few tiles (rows x width) with a long K axis, a piece
// of the vocabulary; dx and dW tiles share one launch, so it takes the mean over the pairs or
// the rounds of dx tiles alone, whichever is longer, plus the fp32 planes' write and read at
// 1.6 MB per block's time (0.33 us at 5 TB/s).
__host__ __device__ inline float split_cost(const BackCosts &c, int rows, int splits, int &kb_per)
{
    kb_per = ceil_int(c.kbs, splits);
    const int used = ceil_int(c.kbs, kb_per), plane_rows = ceil_int(rows, 32) * 32;
    if ((splits > 1 && kb_per < 4) || static_cast<int64_t>(used) * plane_rows > c.plane_cap)
        return INFINITY;
    const float dx_tiles = static_cast<float>(ceil_int(rows, 2 * kBM)) * c.n_tiles * used;
    const float dx_time = static_cast<float>(kb_per + kTileBlocks);
    const float dw = static_cast<float>(c.dw_m_tiles) * c.n_tiles * (ceil_int(rows, kBK) + kTileBlocks);
    const float mean = (dx_tiles * dx_time + dw) / c.units;
    const float rounds = ceilf(dx_tiles / c.units) * dx_time;
    return fmaxf(mean, rounds) * c.pieces + static_cast<float>(used) * rows * c.width * (8.0f / 1.6e6f);
}

// One warp: the shape with the least cost.
__device__ __forceinline__ BackShape choose_shape(const BackCosts &c, int with_target, int lane)
{
    const int lo_row = second_part(with_target, c.part_rows), rows = lo_row + with_target;
    float best = INFINITY;
    int best_per = c.kbs;
    for (int splits = 1 + lane; splits <= c.units; splits += 32) {
        int per;
        const float cost = split_cost(c, rows, splits, per);
        if (cost < best) {
            best = cost;
            best_per = per;
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, best, o);
        const int other_per = __shfl_xor_sync(0xffffffffu, best_per, o);
        if (other < best || (other == best && other_per > best_per)) {
            best = other;
            best_per = other_per;
        }
    }
    return BackShape{with_target, lo_row, rows, best_per, ceil_int(c.kbs, best_per), ceil_int(rows, 32) * 32};
}

constexpr uint32_t kAMnMajor = 1u << 15, kBMnMajor = 1u << 16; // instruction descriptor bits

struct Params {
    int rows;                    // token rows (the most there can be; kBack: rows of G)
    int g_rows;                  // kGrad: rows that G has room for
    const BackShape *shape;      // kGrad and kBack: how many of them there are, and dx's splits
    int n, n_tiles;              // output columns: the vocabulary's (kStats, kGrad), x's width (kBack)
    int bn;                      // tile width
    int num_kb;                  // kStats, kGrad: K blocks (of x's width)
    int a_rows;                  // token rows of a K-major A tile that are loaded (kBM, or few rows rounded up)
    uint32_t idesc_bits;         // instruction descriptor's operand types and N
    // kStats and kGrad: column c is vocabulary entry col0 + c.
    int col0;
    float scale2;                // log2(e) / T
    const void *labels;          // kStats, one target: int32 or int64 per row
    int label_bytes;
    const int32_t *t_index;      // sorted target columns [rows, targets] (INT_MAX: none)
    const float *t_prob;
    int targets;
    float *part_max, *part_sum, *part_t; // [column tiles, rows]; part_t holds sum_j t_j z_j
    float *label_z;              // kStats, one target: z of the label
    const float *row_lse2, *row_gain; // kGrad: lse log2(e), and g T s
    // kBack
    int vocab;                   // the piece's vocabulary columns: K of dx, rows of dW
    int want_dx;
    int dw_tiles;                // tiles of dW (0: no dW)
    int accumulate;              // add to the fp32 planes
    const float *inv_gain;       // 1 / s
};

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Hands a drained accumulator back to the MMA issuer.  The reads of it have completed
// (tcgen05.wait::ld), so the arrival orders nothing else: a release at cluster scope would
// wait for this warp's global stores as well (it was a sixth of the epilogue's stalls).
__device__ __forceinline__ void release_accumulator(uint32_t cluster_bar)
{
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16)
{
    uint32_t r;
    if (bf16)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float2 unpack16(uint32_t v, bool bf16)
{
    if (bf16)
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
    __half2 h;
    memcpy(&h, &v, 4);
    return __half22float2(h);
}

// fp32 pair a * b + c, each lane rounded once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    uint64_t x, y, z, r;
    memcpy(&x, &a, 8);
    memcpy(&y, &b, 8);
    memcpy(&z, &c, 8);
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    float2 f;
    memcpy(&f, &r, 8);
    return f;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    uint64_t x, y, r;
    memcpy(&x, &a, 8);
    memcpy(&y, &b, 8);
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    float2 f;
    memcpy(&f, &r, 8);
    return f;
}

// v[c] for a c that differs from lane to lane: a five-level selection, since registers
// cannot be indexed.
__device__ __forceinline__ float select32(const uint32_t (&v)[32], int c)
{
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
        w[i] = (c & 1) ? v[2 * i + 1] : v[2 * i];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        w[i] = (c & 2) ? w[2 * i + 1] : w[2 * i];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = (c & 4) ? w[2 * i + 1] : w[2 * i];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        w[i] = (c & 8) ? w[2 * i + 1] : w[2 * i];
    return __uint_as_float((c & 16) ? w[1] : w[0]);
}

// First of the `count` sorted columns that is >= column.
__device__ __forceinline__ int lower_bound(const int32_t *cols, int count, int column)
{
    int lo = 0, hi = count;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cols[mid] < column)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int64_t load_label(const void *labels, int bytes, int64_t row)
{
    return bytes == 8 ? static_cast<const int64_t *>(labels)[row]
                      : static_cast<int64_t>(static_cast<const int32_t *>(labels)[row]);
}

__device__ __forceinline__ void tma_store_add_2d(const CUtensorMap *map, uint32_t src, int32_t x, int32_t y)
{
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(x), "r"(y)
                 : "memory");
}

// Matrix descriptor of an MN-major operand: 64-wide boxes of 64 K rows stacked along MN
// (8192 bytes apart, the leading offset), 8-row swizzle atoms stacked along K (1024 bytes,
// the stride offset).
__device__ __forceinline__ uint64_t desc_mn_boxes(uint32_t addr)
{
    uint64_t desc = static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
    desc |= static_cast<uint64_t>(8192u >> 4) << 16;
    desc |= static_cast<uint64_t>(1024u >> 4) << 32;
    desc |= static_cast<uint64_t>(1u) << 46;
    desc |= static_cast<uint64_t>(2u) << 61;
    return desc;
}

// tm_a, tm_b, tm_out: operands and output (G) of kStats and kGrad; G, W and the fp32 planes of
// dx in kBack.  tm_a2, tm_b2, tm_out2: G, x and dW of kBack.
template <bool kPair, int MODE, bool kBf16>
__global__ void __launch_bounds__(Cfg<kPair, MODE>::kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                const __grid_constant__ CUtensorMap tm_out, const __grid_constant__ CUtensorMap tm_a2,
                const __grid_constant__ CUtensorMap tm_b2, const __grid_constant__ CUtensorMap tm_out2, const Params p)
{
    using C = Cfg<kPair, MODE>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem);

    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    const uint32_t rank = kPair ? cluster_ctarank() : 0u;
    const bool leader = rank == 0;
    const int units = kPair ? static_cast<int>(gridDim.x / 2) : static_cast<int>(gridDim.x);
    const int unit = kPair ? static_cast<int>(blockIdx.x / 2) : static_cast<int>(blockIdx.x);
    const uint32_t bar_full = sbase + C::kOffBar;
    const uint32_t bar_empty = bar_full + 8 * C::kStages;
    const uint32_t bar_acc_full = bar_empty + 8 * C::kStages;
    const uint32_t bar_acc_empty = bar_acc_full + 16;
    const uint32_t bar_drain = bar_acc_empty + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::kOffBar + (2 * C::kStages + 5) * 8);

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(bar_acc_full + 8 * a, 1);
            mbar_init(bar_acc_empty + 8 * a, kPair ? 2 * C::kEpiWarps : C::kEpiWarps);
        }
        mbar_init(bar_drain, 1);
        fence_barrier_init();
        if (MODE != kBack || p.want_dx) {
            prefetch_tensor_map(&tm_a);
            prefetch_tensor_map(&tm_b);
            if (MODE != kStats)
                prefetch_tensor_map(&tm_out);
        }
        if (MODE == kBack && p.dw_tiles > 0) {
            prefetch_tensor_map(&tm_a2);
            prefetch_tensor_map(&tm_b2);
            prefetch_tensor_map(&tm_out2);
        }
    }
    if (warp == 1) {
        if (kPair) {
            tmem_alloc_pair(smem_u32(tmem_slot), C::kTmemCols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (kPair)
        cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    // Everything this grid reads (the weights too: an optimizer may just have written them)
    // and writes belongs to the previous kernel until it completes.  The next kernel may only
    // then start, so that its own early reads cannot pass that one either.
    // kStats after targets_kernel: x and W are complete since that one was let past its wait, and
    // only the epilogue reads its targets.
    const bool late = MODE == kStats && p.t_index != nullptr;
    if (!late || warp >= 2) {
        griddepcontrol_wait();
        griddepcontrol_launch_dependents();
    }

    BackShape shape{p.rows, 0, p.rows, 1, 0, 0};
    if (MODE != kStats)
        shape = *p.shape;
    const int rows = MODE == kBack ? shape.all_rows : shape.rows;
    struct Tile {
        int m0, n0, kb0, kbn, split;
        bool dw;
    };
    // The i-th tile of this CTA (pair): its first row, the tile's first column and its K blocks;
    // false past the last.  A function of i alone: the producer, the MMA issuer and the epilogue
    // agree.
    const int m_tiles = (rows + C::kTileM - 1) / C::kTileM;
    // kBack: the dx tiles (long: K is the piece of the vocabulary) are dealt out first, the dW
    // tiles (K: the rows) after them.  Where a last round of dx tiles leaves units without one,
    // those take as many dW tiles more as fit into its time; from then on every unit is level
    // again.
    const int dx_kbs = (p.vocab + kBK - 1) / kBK; // a last piece has fewer, and fewer splits
    const int dx_tiles = MODE == kBack && p.want_dx ? ceil_int(dx_kbs, shape.kb_per) * m_tiles * p.n_tiles : 0;
    const int dx_left = dx_tiles % units;
    const int dx_mine = dx_tiles / units + (unit < dx_left ? 1 : 0);
    const int dw_kbs = (rows + kBK - 1) / kBK;
    const int dw_extra = dx_left > 0 ? (shape.kb_per + kTileBlocks) / (dw_kbs + kTileBlocks) : 0;
    auto tile_at = [&](int i, Tile &tile) {
        tile.split = 0;
        tile.dw = false;
        if (MODE != kBack) {
            const int t = unit + i * units;
            if (t >= m_tiles * p.n_tiles)
                return false;
            tile.m0 = (t % m_tiles) * C::kTileM + static_cast<int>(rank) * kBM;
            tile.n0 = (t / m_tiles) * p.bn;
            tile.kb0 = 0;
            tile.kbn = p.num_kb;
            return true;
        }
        // Columns fastest: the units at work share panels of G.
        if (i < dx_mine) {
            const int t = unit + i * units;
            const int per_split = m_tiles * p.n_tiles;
            tile.split = t / per_split;
            const int r = t - tile.split * per_split;
            tile.m0 = (r / p.n_tiles) * C::kTileM + static_cast<int>(rank) * kBM;
            tile.n0 = (r % p.n_tiles) * p.bn;
            tile.kb0 = tile.split * shape.kb_per;
            tile.kbn = min(shape.kb_per, dx_kbs - tile.kb0);
            return true;
        }
        const int j = i - dx_mine;
        const bool early = unit >= dx_left;
        const int t = early && j < dw_extra
                          ? j * (units - dx_left) + unit - dx_left
                          : (units - dx_left) * dw_extra + (j - (early ? dw_extra : 0)) * units + unit;
        if (t >= p.dw_tiles)
            return false;
        tile.dw = true;
        tile.m0 = (t / p.n_tiles) * C::kTileM + static_cast<int>(rank) * kBM;
        tile.n0 = (t % p.n_tiles) * p.bn;
        tile.kb0 = 0;
        tile.kbn = dw_kbs;
        return true;
    };

    if (warp == 0) {
        // ---------------- TMA producer (one thread) ----------------
        if (lane == 0) {
            uint32_t used_mask = 0, parity_mask = 0;
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            auto load = [&](uint32_t dst, const CUtensorMap *map, uint32_t full, int x, int y) {
                if (kPair)
                    tma_load_2d_pair(dst, map, full, x, y);
                else
                    tma_load_2d(dst, map, full, x, y);
            };
            const int b_rows = kPair ? p.bn / 2 : p.bn; // this CTA's
            const int b_boxes = (b_rows + 63) / 64;     // MN-major
            Tile tile;
            for (int n = 0; ok && tile_at(n, tile); ++n) {
                const int b0 = tile.n0 + static_cast<int>(rank) * b_rows;
                const uint32_t tx = (kPair ? 2u : 1u) * (static_cast<uint32_t>(tile.dw ? kBM : p.a_rows) * 128u +
                                                         (MODE == kBack ? b_boxes * 8192u : b_rows * 128u));
                const CUtensorMap *map_b = tile.dw ? &tm_b2 : &tm_b;
                for (int i = 0; i < tile.kbn; ++i) {
                    if (!mbar_wait(bar_empty + 8 * s, ph ^ 1u, kSiteProducerEmpty)) {
                        ok = false;
                        break;
                    }
                    const int k0 = (tile.kb0 + i) * kBK;
                    if (leader)
                        mbar_arrive_expect_tx(bar_full + 8 * s, tx);
                    const uint32_t full = kPair ? map_to_rank(bar_full + 8 * s, 0) : bar_full + 8 * s;
                    const uint32_t a = sbase + s * C::kABytes;
                    const uint32_t b = sbase + C::kOffB + s * C::kBBytes;
                    if (MODE == kBack && tile.dw) {
#pragma unroll
                        for (int j = 0; j < kBM / 64; ++j)
                            load(a + j * 8192, &tm_a2, full, tile.m0 + 64 * j, k0);
                    } else {
                        load(a, &tm_a, full, k0, tile.m0);
                    }
                    if (MODE == kBack) {
                        for (int j = 0; j < b_boxes; ++j)
                            load(b + j * 8192, map_b, full, b0 + 64 * j, k0);
                    } else {
                        load(b, &tm_b, full, k0, b0);
                    }
                    used_mask |= 1u << s;
                    parity_mask = (parity_mask & ~(1u << s)) | (ph << s);
                    if (++s == C::kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
            // Every issued load must land before shared memory is released.  In a pair the
            // leader's full barriers count both CTAs' loads.
            if (leader)
                for (int i = 0; i < C::kStages; ++i)
                    if (used_mask & (1u << i)) {
                        const uint32_t par = (parity_mask >> i) & 1u;
                        for (int tries = 0; tries < (1 << 22) && !mbar_try_wait(bar_full + 8 * i, par); ++tries) {
                        }
                    }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (one thread of the leader) ----------------
        if (lane == 0 && leader) {
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            Tile tile;
            for (int n = 0; ok && tile_at(n, tile); ++n) {
                const bool a_mn = MODE == kBack && tile.dw;
                const uint32_t idesc =
                    C::kIdesc | p.idesc_bits | (a_mn ? kAMnMajor : 0u) | (MODE == kBack ? kBMnMajor : 0u);
                const uint32_t a = n & 1;
                const uint32_t acc_ph = (n >> 1) & 1;
                if (!mbar_wait(bar_acc_empty + 8 * a, acc_ph ^ 1u, kSiteMmaAccEmpty)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + a * kMaxBN;
                for (int i = 0; i < tile.kbn; ++i) {
                    if (!mbar_wait(bar_full + 8 * s, ph, kSiteMmaFull)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_addr = sbase + s * C::kABytes;
                    const uint32_t b_addr = sbase + C::kOffB + s * C::kBBytes;
#pragma unroll
                    for (int k = 0; k < kBK / kUmmaK; ++k) {
                        // 16 K elements: 32 bytes of a K-major row, or two 8-row atoms.
                        const uint64_t da = a_mn ? desc_mn_boxes(a_addr + k * 2048) : smem_desc_k_sw128(a_addr + k * 32);
                        const uint64_t db =
                            MODE == kBack ? desc_mn_boxes(b_addr + k * 2048) : smem_desc_k_sw128(b_addr + k * 32);
                        if (kPair)
                            mma_f16_pair(d_tmem, da, db, idesc, (i | k) != 0);
                        else
                            mma_f16(d_tmem, da, db, idesc, (i | k) != 0);
                    }
                    if (kPair)
                        mma_commit_pair_both(bar_empty + 8 * s);
                    else
                        mma_commit(bar_empty + 8 * s);
                    if (++s == C::kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
                if (ok) {
                    if (kPair)
                        mma_commit_pair_both(bar_acc_full + 8 * a);
                    else
                        mma_commit(bar_acc_full + 8 * a);
                }
            }
            // Drain: all MMAs issued by this thread complete before TMEM is freed.
            if (kPair)
                mma_commit_pair_local(bar_drain);
            else
                mma_commit(bar_drain);
            for (int tries = 0; tries < (1 << 22) && !mbar_try_wait(bar_drain, 0); ++tries) {
            }
        }
    } else {
        // ---------------- Epilogue: one row per lane ----------------
        const int ew = warp - 2;
        const int quarter = warp & 3;
        // This warp's columns: its share of the tile's 32-column steps.
        const int slice = ew >> 2;
        const int steps = (p.bn + kSub - 1) / kSub;
        const int col_begin = slice * steps / C::kParts * kSub;
        const int col_end = min((slice + 1) * steps / C::kParts * kSub, p.bn);
        const uint32_t acc_empty = kPair ? map_to_rank(bar_acc_empty, 0) : bar_acc_empty;
        uint8_t *staging = smem + C::kOffStaging + ew * C::kStaging;
        const uint32_t staging_s = smem_u32(staging);
        const float inv_gain = MODE == kBack ? *p.inv_gain : 1.0f;
        uint32_t stores = 0;
        // A staging buffer (32 rows x 64 B, 64-byte swizzle: chunk j of row r at j ^ ((r >> 1) & 3))
        // that its last store has read, its filling, and the fence before the next store.
        auto next_buffer = [&] {
            if (lane == 0)
                asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(C::kBuffers - 1) : "memory");
            __syncwarp();
            return C::kBuffers > 1 ? (stores++ & 1u) * 2048u : 0u;
        };
        auto put_row = [&](uint32_t buffer, int r, int j, uint4 w) {
            *reinterpret_cast<uint4 *>(staging + buffer + r * 64 + ((j ^ ((r >> 1) & 3)) * 16)) = w;
        };
        auto put = [&](uint32_t buffer, int j, uint4 w) { put_row(buffer, lane, j, w); };
        auto filled = [&] {
            fence_proxy_async_smem();
            __syncwarp();
        };
        Tile tile;
        for (int n = 0; tile_at(n, tile); ++n) {
            const uint32_t a = n & 1;
            const uint32_t acc_ph = (n >> 1) & 1;
            // G is also written (as zeros) for the rows that fill up a K block of dW.
            const int row_limit = MODE == kBack && tile.dw ? p.vocab
                                  : MODE != kGrad          ? rows
                                  : shape.lo_row > 0       ? shape.lo_row
                                                           : min((rows + kBK - 1) / kBK * kBK, p.g_rows);
            const int row0 = tile.m0 + quarter * 32;
            const int row = row0 + lane;
            const int col0 = tile.n0 + col_begin;
            const int col1 = min(tile.n0 + col_end, p.n);
            // Rows and columns of this warp that exist.
            const int width = row0 < row_limit ? col1 - col0 : 0;
            int subs = width > 0 ? (width + kSub - 1) / kSub : 0;

            // The row's next target column (relative to the piece), found while the MMAs run.
            int next = INT_MAX, entry = 0;
            const int32_t *row_cols = nullptr;
            float lse2 = 0.0f, gain = 0.0f;
            if (MODE != kBack && row < rows && subs > 0) {
                if (p.t_index) {
                    row_cols = p.t_index + static_cast<size_t>(row) * p.targets;
                    entry = lower_bound(row_cols, p.targets, p.col0 + col0);
                    if (entry < p.targets)
                        next = row_cols[entry] - p.col0; // INT_MAX - col0 never falls in a tile
                } else {
                    const int64_t label = load_label(p.labels, p.label_bytes, row);
                    if (label >= col0 && label < p.n)
                        next = static_cast<int>(label);
                }
                if (MODE == kGrad) {
                    lse2 = p.row_lse2[row];
                    gain = p.row_gain[row];
                }
            }
            // From the lowest finite value up, so that a logit of -infinity adds exp2(-infinity).
            float run_max = -FLT_MAX, run_sum = 0.0f, run_t = 0.0f;

            const bool ok = __all_sync(0xffffffffu, mbar_wait(bar_acc_full + 8 * a, acc_ph, kSiteEpilogueAccFull));
            if (!ok) {
                if (MODE != kStats)
                    break;
                subs = 0; // the error word is set; keep meeting the quarter's other warps
            }
            tc_fence_after();
            const uint32_t t_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + a * kMaxBN + col_begin;
#pragma unroll 1
            for (int sub = 0; sub < subs; ++sub) {
                const int c0 = col0 + sub * kSub;
                uint32_t v[32];
                tmem_ld_32x32b_x32(t_base + sub * kSub, v);
                tmem_wait_ld();
                if (sub == subs - 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (kPair)
                            release_accumulator(acc_empty + 8 * a);
                        else
                            mbar_arrive(acc_empty + 8 * a);
                    }
                }
                if (MODE == kStats) {
                    // Running maximum and sum of exp2(scale2 z - maximum).
                    if (col1 - c0 < kSub) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (c0 + i >= col1)
                                v[i] = 0xff800000u; // columns past the tile or the vocabulary: -infinity
                    }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            mx[j] = fmaxf(mx[j], fmaxf(__uint_as_float(v[i + 2 * j]), __uint_as_float(v[i + 2 * j + 1])));
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale2;
                    const float next_max = fmaxf(run_max, top);
                    const float2 ref = make_float2(-next_max, -next_max);
                    const float2 sc = make_float2(p.scale2, p.scale2);
                    float2 acc[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 e =
                            fma2(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), sc, ref);
                        acc[(i >> 1) & 1] = add2(acc[(i >> 1) & 1], make_float2(exp2_approx(e.x), exp2_approx(e.y)));
                    }
                    acc[0] = add2(acc[0], acc[1]);
                    run_sum = fmaf(run_sum, exp2_approx(run_max - next_max), acc[0].x + acc[0].y);
                    run_max = next_max;
                    // Targets of this step: rare, so one uniform test in the common case.
                    const int step_end = min(c0 + kSub, col1);
                    while (__any_sync(0xffffffffu, next < step_end)) {
                        if (next < step_end) {
                            const float z = select32(v, next - c0);
                            if (p.t_index) {
                                // A weight of 0 (a repeated token's later entries, an exponential that
                                // vanished) takes no part: z may be -infinity.
                                const float weight = p.t_prob[static_cast<size_t>(row) * p.targets + entry];
                                if (weight != 0.0f)
                                    run_t = fmaf(weight, z, run_t);
                                ++entry;
                                next = entry < p.targets ? row_cols[entry] - p.col0 : INT_MAX;
                            } else {
                                p.label_z[row] = z;
                                next = INT_MAX;
                            }
                        }
                    }
                    continue;
                }
                float f[32];
                if (MODE == kGrad) {
                    if (row0 + 32 > rows && row >= rows) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            v[i] = 0u; // whatever lay in the tile; times a gain of 0
                    }
                    const float2 ref = make_float2(-lse2, -lse2);
                    const float2 sc = make_float2(p.scale2, p.scale2);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 e =
                            fma2(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), sc, ref);
                        f[i] = exp2_approx(e.x) * gain;
                        f[i + 1] = exp2_approx(e.y) * gain;
                    }
                    while (__any_sync(0xffffffffu, next < c0 + kSub)) {
                        if (next < c0 + kSub) {
                            const int c = next - c0;
                            const float d = gain * p.t_prob[static_cast<size_t>(row) * p.targets + entry];
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                f[i] = i == c ? f[i] - d : f[i];
                            ++entry;
                            next = entry < p.targets ? row_cols[entry] - p.col0 : INT_MAX;
                        }
                    }
                }
                if (MODE == kBack && !tile.dw) {
                    // fp32, 16 columns at a time.
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const uint32_t buffer = next_buffer();
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            put(buffer, j,
                                make_uint4(v[16 * hf + 4 * j], v[16 * hf + 4 * j + 1], v[16 * hf + 4 * j + 2],
                                           v[16 * hf + 4 * j + 3]));
                        filled();
                        if (lane == 0) {
                            if (c0 + 16 * hf < p.n) {
                                const int plane_row = tile.split * shape.plane_rows + row0;
                                if (p.accumulate)
                                    tma_store_add_2d(&tm_out, staging_s + buffer, c0 + 16 * hf, plane_row);
                                else
                                    tma_store_2d(&tm_out, staging_s + buffer, c0 + 16 * hf, plane_row);
                            }
                            bulk_commit_group();
                        }
                    }
                    continue;
                }
                if (MODE == kBack) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        f[i] = __uint_as_float(v[i]) * inv_gain;
                }
                auto put16 = [&](uint32_t buffer, int r) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        put_row(buffer, r, j,
                                make_uint4(pack16(f[8 * j], f[8 * j + 1], kBf16), pack16(f[8 * j + 2], f[8 * j + 3], kBf16),
                                           pack16(f[8 * j + 4], f[8 * j + 5], kBf16),
                                           pack16(f[8 * j + 6], f[8 * j + 7], kBf16)));
                };
                auto store16 = [&](uint32_t buffer, int first_row) {
                    filled();
                    if (lane == 0) {
                        tma_store_2d(MODE == kBack ? &tm_out2 : &tm_out, staging_s + buffer, c0, first_row);
                        bulk_commit_group();
                    }
                };
                auto keep_rest = [&] { // what the rounding to 16 bits leaves off
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 kept = unpack16(pack16(f[i], f[i + 1], kBf16), kBf16);
                        f[i] -= kept.x;
                        f[i + 1] -= kept.y;
                    }
                };
                const uint32_t buffer = next_buffer();
                if (MODE == kGrad && shape.lo_row > 0 && shape.lo_row < 32) {
                    // Both parts in one store, which ends with them (G has no more rows).
                    if (lane < shape.lo_row) {
                        put16(buffer, lane);
                        keep_rest();
                        put16(buffer, shape.lo_row + lane);
                    }
                    store16(buffer, row0);
                    continue;
                }
                put16(buffer, lane);
                store16(buffer, row0);
                if (MODE == kGrad && shape.lo_row > 0) {
                    keep_rest();
                    const uint32_t again = next_buffer();
                    put16(again, lane);
                    store16(again, shape.lo_row + row0);
                }
            }
            if (subs == 0) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (kPair)
                        release_accumulator(acc_empty + 8 * a);
                    else
                        mbar_arrive(acc_empty + 8 * a);
                }
            }
            if (MODE == kStats) {
                // Merge the column slices of each row: the warps of a quarter meet on a
                // named barrier, and the first writes the tile's partial result.
                float *mine = reinterpret_cast<float *>(staging) + (n & 1) * 96;
                mine[lane] = run_max;
                mine[32 + lane] = run_sum;
                mine[64 + lane] = run_t;
                named_barrier_sync(1 + quarter, 32 * C::kParts);
                if (slice == 0 && row < rows) {
#pragma unroll
                    for (int j = 1; j < C::kParts; ++j) {
                        const float *other = mine + j * (4 * C::kStaging / 4);
                        const float m = other[lane];
                        const float next_max = fmaxf(run_max, m);
                        run_sum = fmaf(run_sum, exp2_approx(run_max - next_max),
                                       other[32 + lane] * exp2_approx(m - next_max));
                        run_max = next_max;
                        run_t += other[64 + lane];
                    }
                    const size_t at = static_cast<size_t>(tile.n0 / p.bn) * rows + row;
                    p.part_max[at] = run_max;
                    p.part_sum[at] = run_sum;
                    if (p.part_t)
                        p.part_t[at] = run_t;
                }
            }
        }
        if (MODE != kStats && lane == 0)
            bulk_wait_group0();
    }

    tc_fence_before();
    __syncthreads();
    if (kPair)
        cluster_sync(); // neither CTA leaves while its peer may still touch its barriers or TMEM
    if (warp == 1) {
        tc_fence_after();
        if (kPair)
            tmem_dealloc_pair(tmem_base, C::kTmemCols);
        else
            tmem_dealloc(tmem_base, C::kTmemCols);
    }
}

// ---- targets ------------------------------------------------------------------

__device__ __forceinline__ float load_float(const void *p, int dtype, size_t i)
{
    if (dtype == kTypeFloat)
        return static_cast<const float *>(p)[i];
    if (dtype == kTypeBf16)
        return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return __half2float(static_cast<const __half *>(p)[i]);
}

constexpr int kPrepWarps = 8;

struct Targets {
    int rows, vocab, count;
    const int32_t *tokens;
    const void *logits;
    int logit_type;
    float inv_temperature;
    int32_t *index; // sorted [rows, count]
    float *prob;
};

// Ascending bitonic sort of 32 R keys over a warp: key i of lane l is element 32 i + l, so
// distances from 32 up stay in a lane's registers and the others are lane exchanges.
template <int R>
__device__ __forceinline__ void sort_keys(uint32_t (&key)[R], int lane)
{
#pragma unroll
    for (int size = 2; size <= 32 * R; size *= 2) {
#pragma unroll
        for (int dist = size / 2; dist > 0; dist /= 2) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int e = 32 * i + lane;
                if (dist >= 32) {
                    const int j = i ^ (dist / 32);
                    if (j > i) {
                        const uint32_t lo = min(key[i], key[j]), hi = max(key[i], key[j]);
                        const bool up = (e & size) == 0;
                        key[i] = up ? lo : hi;
                        key[j] = up ? hi : lo;
                    }
                } else {
                    const uint32_t other = __shfl_xor_sync(0xffffffffu, key[i], dist);
                    const bool up = (e & size) == 0, low = (lane & dist) == 0;
                    key[i] = up == low ? min(key[i], other) : max(key[i], other);
                }
            }
        }
    }
}

// One warp lays out one row's teacher entries (up to 32 R): the softmax of the logits of the
// valid ones (token in the vocabulary, logit not -infinity) and their columns in ascending
// order, the rest INT_MAX.  A sort key is the column with the entry's number below it (22 + 8
// bits), so equal tokens keep their order.  Returns whether the row has any, with (negative
// entropy, sum) of its probabilities in 64 bits: the loss is a difference of terms near
// log(V), so it is formed from unrounded ones.  probs, keys: scratch of 32 R.
template <int R>
__device__ __forceinline__ bool sort_targets(const Targets &t, int row, int lane, float *probs, uint32_t *keys,
                                             double &entropy, double &total)
{
    constexpr uint32_t kNone = 0xFFFFFFFFu;
    const size_t base = static_cast<size_t>(row) * t.count;
    int32_t token[R];
    float z[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int j = lane + 32 * i;
        token[i] = j < t.count ? t.tokens[base + j] : -1;
        z[i] = j < t.count ? load_float(t.logits, t.logit_type, base + j) : 0.0f;
    }
    uint32_t key[R];
    float top = -INFINITY;
    bool has = false;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (token[i] >= t.vocab)
            g_token_error = 1;
        const bool valid = token[i] >= 0 && token[i] < t.vocab && z[i] != -INFINITY;
        // A finite logit stays finite: the lowest value of a type masks nothing.
        const float scaled = z[i] * t.inv_temperature;
        z[i] = isinf(scaled) && !isinf(z[i]) ? copysignf(FLT_MAX, z[i]) : scaled;
        key[i] = valid ? (static_cast<uint32_t>(token[i]) << 8) | static_cast<uint32_t>(lane + 32 * i) : kNone;
        z[i] = valid ? z[i] : -INFINITY;
        has |= valid;
        top = fmaxf(top, z[i]);
    }
    const bool any = __any_sync(0xffffffffu, has);
#pragma unroll
    for (int o = 16; o; o >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float e[R], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        e[i] = key[i] == kNone ? 0.0f : exp2f((z[i] - top) * kLog2e);
        sum += e[i];
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    entropy = 0.0;
    total = 0.0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const float prob = any ? e[i] / sum : 0.0f;
        probs[lane + 32 * i] = prob;
        if (key[i] != kNone) {
            entropy += static_cast<double>(prob) * (static_cast<double>(z[i]) - static_cast<double>(top));
            total += prob;
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        entropy += __shfl_xor_sync(0xffffffffu, entropy, o);
        total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    if (any)
        entropy -= total * log(static_cast<double>(sum));
    sort_keys<R>(key, lane);
#pragma unroll
    for (int i = 0; i < R; ++i)
        keys[lane + 32 * i] = key[i];
    __syncwarp();
    // A token that occurs several times has their sum at its first entry and 0 at the others, so
    // that dz subtracts it once: many small subtractions from a probability would each round.
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int j = lane + 32 * i;
        if (j < t.count) {
            const uint32_t col = key[i] >> 8;
            float prob = key[i] == kNone ? 0.0f : probs[key[i] & 255u];
            if (key[i] != kNone && j > 0 && keys[j - 1] >> 8 == col) {
                prob = 0.0f;
            } else if (key[i] != kNone && j + 1 < t.count && keys[j + 1] >> 8 == col) {
                double sum_of_equals = prob;
                for (int o = j + 1; o < t.count && keys[o] >> 8 == col; ++o)
                    sum_of_equals += probs[keys[o] & 255u];
                prob = static_cast<float>(sum_of_equals);
            }
            t.index[base + j] = key[i] == kNone ? INT_MAX : static_cast<int32_t>(col);
            t.prob[base + j] = prob;
        }
    }
    __syncwarp();
    return any;
}

// Sorted targets; in the forward (entropy, sum) per row, in the backward whether the row has any
// target (0, else -1).
template <int R>
__global__ void __launch_bounds__(32 * kPrepWarps) targets_kernel(const Targets t, double2 *row_terms, int32_t *marks)
{
    __shared__ float probs[kPrepWarps][32 * R];
    __shared__ uint32_t keys[kPrepWarps][32 * R];
    griddepcontrol_wait();
    griddepcontrol_launch_dependents();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int row = blockIdx.x * kPrepWarps + warp; row < t.rows; row += gridDim.x * kPrepWarps) {
        double entropy, total;
        const bool any = sort_targets<R>(t, row, lane, probs[warp], keys[warp], entropy, total);
        if (lane == 0 && row_terms)
            row_terms[row] = make_double2(entropy, total);
        if (lane == 0 && marks)
            marks[row] = any ? 0 : -1;
    }
}

struct Prepare {
    Targets t;            // the targets' place; a teacher's entries
    const int32_t *sorted_index; // a teacher's sorted targets, row by row, before the rows move
    const float *sorted_prob;
    const void *labels;   // one label per row, or a teacher's marks (0, -1 to be ignored)
    int label_bytes;
    int64_t ignore_index;
    float temperature;
    int width;            // elements per row of x, a multiple of 8
    int g_rows;           // rows of x_used, and of G
    const void *x;
    void *x_used;
    const float *lse, *grad;
    float *row_lse2, *row_gain, *inv_gain;
    int *row_at; // where each row went (-1: it has no target)
    BackCosts costs;
    BackShape *shape;
};

// A rounding is off by up to half a step of its value's binade, which is least, relative to the
// value, just under a power of two.  Most of G's weight is in the targets' elements, near -g T, so
// of four gains a quarter of an octave apart the one is taken that rounds the g T with the
// least squared error (loss gradients that are all alike then end up where steps are finest).
constexpr int kShares = 4;
__device__ __forceinline__ float gain_share(int i)
{
    return i == 0 ? 1.0f : i == 1 ? 1.18920712f : i == 2 ? 1.41421356f : 1.68179283f;
}

// Adds the squared step of g (a loss gradient times T) times each share.
__device__ __forceinline__ void add_steps(float (&steps)[kShares], float g)
{
#pragma unroll
    for (int k = 0; k < kShares; ++k) {
        const float step = __uint_as_float(__float_as_uint(g * gain_share(k)) & 0x7F800000u);
        steps[k] = fmaf(step, step, steps[k]);
    }
}

// The share with the least error; sums past fp32's range, up or down, leave the choice open.
__device__ __forceinline__ float best_share(const float (&steps)[kShares])
{
    float share = 1.0f, least = INFINITY;
#pragma unroll
    for (int k = 0; k < kShares; ++k) {
        const float error = steps[k] * (1.0f / (gain_share(k) * gain_share(k)));
        if (error < least) {
            least = error;
            share = gain_share(k);
        }
    }
    return share;
}

// The common gain s, a share times a power of two, puts max |g T s| in [2^13, 2^14) for any finite
// g from 2^-100 on: with |p - t| <= 1, G then fits fp16 (65504) and keeps 11 bits down to
// p = 2^-27 in the rows of the largest |g|, to 2^(k-27) in those of 2^-k of it.  Returns T s, since
// g T alone may pass fp32's range; thread 0 of block 0 keeps 1 / s, by which the products' fp32
// results are multiplied.  The exponent is taken of 2^-8 of the largest, which cannot overflow
// (top < 2^128, T <= 2^6, share < 2).
__device__ __forceinline__ float common_gain(float top, float temperature, float share, float *inv_gain)
{
    const int exponent = top > 0.0f ? min(max(ilogbf(top * 0x1p-8f * temperature * share) + 8, -100), 134) : 13;
    const float s = ldexpf(share, 13 - exponent);
    if (blockIdx.x == 0 && threadIdx.x == 0)
        *inv_gain = 1.0f / s;
    return temperature * s;
}

constexpr int kHeadVectors = 5; // 1280 elements of a row per lane group, requested ahead

// Backward's first step.  The rows that have a target move together, in order: their states,
// targets, lse and gain g T s.  The others (padding, in a batch of transcripts)
// take no part in the products, so whatever they hold, NaN included, reaches nothing and costs
// nothing.  Up to 255 zero rows follow, to the end of a tile, so that what a tile reads there
// adds nothing.  Each block counts the valid labels before its rows itself (a few KB of reads),
// which is why there is one large block per SM.
constexpr int kRowWarps = 32;
static_assert(kRowWarps == 32, "a lane per warp in the second step of a block's sums");
template <bool kTeacher>
__global__ void __launch_bounds__(32 * kRowWarps) prepare_rows_kernel(const Prepare p, int rows_per_block)
{
    __shared__ float warp_max[kRowWarps], warp_steps[kShares][kRowWarps];
    __shared__ int warp_before[kRowWarps], warp_total[kRowWarps];
    griddepcontrol_wait();
    griddepcontrol_launch_dependents();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int begin = min(static_cast<int>(blockIdx.x) * rows_per_block, p.t.rows);
    const int end = min(begin + rows_per_block, p.t.rows);
    auto valid = [&](int64_t label) { return label != p.ignore_index && label >= 0 && label < p.t.vocab; };
    float top = 0.0f;
    float steps[kShares] = {}; // sums of squared steps of g times each share
    int before = 0, total = 0;
    // The same sums in every block: over its warps, then in each warp over the warps' (a lane each).
    auto reduce = [&] {
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            before += __shfl_xor_sync(0xffffffffu, before, o);
            total += __shfl_xor_sync(0xffffffffu, total, o);
#pragma unroll
            for (int k = 0; k < kShares; ++k)
                steps[k] += __shfl_xor_sync(0xffffffffu, steps[k], o);
        }
    };
#pragma unroll 8
    for (int i = threadIdx.x; i < p.t.rows; i += 32 * kRowWarps) {
        const float grad = fabsf(p.grad[i]);
        const bool used = valid(load_label(p.labels, p.label_bytes, i));
        const float g = used && grad < INFINITY ? grad : 0.0f;
        top = fmaxf(top, g);
        before += used && i < begin;
        total += used;
        add_steps(steps, g * p.temperature);
    }
    reduce();
    if (lane == 0) {
        warp_max[warp] = top;
        warp_before[warp] = before;
        warp_total[warp] = total;
#pragma unroll
        for (int k = 0; k < kShares; ++k)
            warp_steps[k][warp] = steps[k];
    }
    __syncthreads();
    top = warp_max[lane];
    before = warp_before[lane];
    total = warp_total[lane];
#pragma unroll
    for (int k = 0; k < kShares; ++k)
        steps[k] = warp_steps[k][lane];
    reduce();
    const float gain = common_gain(top, p.temperature, best_share(steps), p.inv_gain);
    const int rows = max(total, 1), lo_row = second_part(rows, p.costs.part_rows); // a row of zeros where none has a target
    if (blockIdx.x == 0 && warp == 0) {
        const BackShape shape = choose_shape(p.costs, rows, lane);
        if (lane == 0)
            *p.shape = shape;
    }

    const int vectors = p.width / 8;
    const uint4 *x = static_cast<const uint4 *>(p.x);
    uint4 *x_used = static_cast<uint4 *>(p.x_used);
    for (int first = begin; first < end; first += 32) {
        const int64_t mine = first + lane < end ? load_label(p.labels, p.label_bytes, first + lane) : p.ignore_index;
        const uint32_t mask = __ballot_sync(0xffffffffu, valid(mine));
        if (warp == 0 && first + lane < end) {
            if (!valid(mine) && mine != p.ignore_index)
                g_token_error = 1;
            p.row_at[first + lane] = valid(mine) ? before + __popc(mask & ((1u << lane) - 1u)) : -1;
        }
        for (int j = warp; j < 32; j += kRowWarps) {
            if (!(mask >> j & 1u))
                continue;
            const int row = first + j, to = before + __popc(mask & ((1u << j) - 1u));
            const uint4 *src = x + static_cast<size_t>(row) * vectors;
            uint4 *dst = x_used + static_cast<size_t>(to) * vectors;
            uint4 head[kHeadVectors];
#pragma unroll
            for (int i = 0; i < kHeadVectors; ++i)
                if (lane + 32 * i < vectors)
                    head[i] = src[lane + 32 * i];
            for (int part = 0; part <= (lo_row > 0); ++part, dst += static_cast<size_t>(lo_row) * vectors) {
#pragma unroll
                for (int i = 0; i < kHeadVectors; ++i)
                    if (lane + 32 * i < vectors)
                        dst[lane + 32 * i] = head[i];
                for (int i = lane + 32 * kHeadVectors; i < vectors; i += 32)
                    dst[i] = src[i];
            }
            const int64_t label = __shfl_sync(0xffffffffu, mine, j);
            if (kTeacher) {
                const size_t entries_from = static_cast<size_t>(row) * p.t.count;
                const size_t entries_to = static_cast<size_t>(to) * p.t.count;
                for (int i = lane; i < p.t.count; i += 32) {
                    p.t.index[entries_to + i] = p.sorted_index[entries_from + i];
                    p.t.prob[entries_to + i] = p.sorted_prob[entries_from + i];
                }
            } else if (lane == 0) {
                p.t.index[to] = static_cast<int32_t>(label);
                p.t.prob[to] = 1.0f;
            }
            if (lane == 0) {
                p.row_lse2[to] = p.lse[row] * kLog2e;
                p.row_gain[to] = p.grad[row] * gain;
            }
        }
        before += __popc(mask);
    }
    const int tail = min((rows + 255) / 256 * 256, p.g_rows);
    for (int row = total + blockIdx.x * kRowWarps + warp; row < tail; row += gridDim.x * kRowWarps) {
        if (row < lo_row || row >= lo_row + total)
            for (int i = lane; i < vectors; i += 32)
                x_used[static_cast<size_t>(row) * vectors + i] = make_uint4(0u, 0u, 0u, 0u);
        if (row >= p.t.rows)
            continue;
        for (int i = lane; i < p.t.count; i += 32) {
            p.t.index[static_cast<size_t>(row) * p.t.count + i] = INT_MAX;
            p.t.prob[static_cast<size_t>(row) * p.t.count + i] = 0.0f;
        }
        if (lane == 0) {
            p.row_lse2[row] = 0.0f;
            p.row_gain[row] = 0.0f;
        }
    }
}

// The same with a teacher and few rows, none of which moves (a tile holds them all, so nothing
// would be saved): per row its sorted targets (up to 32 R), lse and gain,
// and a copy of x whose rows without a target are zero, so that whatever those hold, NaN
// included, reaches neither G nor dW.
template <int R>
__global__ void __launch_bounds__(32 * kPrepWarps) prepare_teacher_kernel(const Prepare p)
{
    __shared__ float probs[kPrepWarps][32 * R];
    __shared__ uint32_t keys[kPrepWarps][32 * R];
    __shared__ float warp_max[kPrepWarps], warp_steps[kPrepWarps][kShares];
    griddepcontrol_wait();
    griddepcontrol_launch_dependents();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    // The largest finite |g| of the rows that have an entry: every block looks at all of them, a
    // row per thread (there are kTeacherMoveRows at most).  A row's first entry says mostly
    // that it has one; a row whose first is left out matters only if its |g| is larger than
    // those, and its warp then reads the others.
    auto is_entry = [&](size_t at) {
        const int32_t token = p.t.tokens[at];
        return token >= 0 && token < p.t.vocab && load_float(p.t.logits, p.t.logit_type, at) != -INFINITY;
    };
    auto block_max = [&](float v) {
#pragma unroll
        for (int o = 16; o; o >>= 1)
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
        if (lane == 0)
            warp_max[warp] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < kPrepWarps; ++i)
            v = fmaxf(v, warp_max[i]);
        return v;
    };
    const int mine = threadIdx.x;
    float g = 0.0f;
    bool known = true;
    if (mine < p.t.rows) {
        g = fabsf(p.grad[mine]);
        g = g < INFINITY ? g : 0.0f;
        known = is_entry(static_cast<size_t>(mine) * p.t.count);
    }
    float top = block_max(known ? g : 0.0f);
    const bool open = !known && g > top;
    if (__syncthreads_or(open)) {
        float more = top;
        for (uint32_t rows = __ballot_sync(0xffffffffu, open); rows; rows &= rows - 1u) {
            const int from = __ffs(rows) - 1;
            const size_t base = static_cast<size_t>(warp * 32 + from) * p.t.count;
            bool has = false;
            for (int i = lane; i < p.t.count; i += 32)
                has |= is_entry(base + i);
            const float g_there = __shfl_sync(0xffffffffu, g, from);
            if (__any_sync(0xffffffffu, has))
                more = fmaxf(more, g_there);
        }
        top = block_max(more);
    }
    const int lo_row = second_part(p.t.rows, p.costs.part_rows);
    float share = 1.0f;
    if (lo_row == 0) { // the rows known to have an entry decide
        float steps[kShares] = {};
        add_steps(steps, known ? g * p.temperature : 0.0f);
#pragma unroll
        for (int k = 0; k < kShares; ++k) {
#pragma unroll
            for (int o = 16; o; o >>= 1)
                steps[k] += __shfl_xor_sync(0xffffffffu, steps[k], o);
            if (lane == 0)
                warp_steps[warp][k] = steps[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kShares; ++k) {
            steps[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < kPrepWarps; ++i)
                steps[k] += warp_steps[i][k];
        }
        share = best_share(steps);
    }
    const float gain = common_gain(top, p.temperature, share, p.inv_gain);
    if (blockIdx.x == 0 && warp == 0) {
        const BackShape shape = choose_shape(p.costs, p.t.rows, lane);
        if (lane == 0)
            *p.shape = shape;
    }

    const int vectors = p.width / 8;
    for (int row = blockIdx.x * kPrepWarps + warp; row < p.g_rows; row += gridDim.x * kPrepWarps) {
        if (row < lo_row + p.t.rows && row >= p.t.rows && row >= lo_row)
            continue; // the second part: with the first
        if (row >= p.t.rows) {
            for (int i = lane; i < vectors; i += 32)
                static_cast<uint4 *>(p.x_used)[static_cast<size_t>(row) * vectors + i] = make_uint4(0u, 0u, 0u, 0u);
            continue;
        }
        const size_t base = static_cast<size_t>(row) * vectors;
        const uint4 *src = static_cast<const uint4 *>(p.x) + base;
        uint4 *dst = static_cast<uint4 *>(p.x_used) + base;
        // The start of the row is requested before its targets are known.
        uint4 head[kHeadVectors];
#pragma unroll
        for (int i = 0; i < kHeadVectors; ++i)
            if (lane + 32 * i < vectors)
                head[i] = src[lane + 32 * i];
        double entropy, total;
        const bool any = sort_targets<R>(p.t, row, lane, probs[warp], keys[warp], entropy, total);
        if (lane == 0) {
            p.row_lse2[row] = any ? p.lse[row] * kLog2e : 0.0f;
            p.row_gain[row] = any ? p.grad[row] * gain : 0.0f;
        }
        for (int part = 0; part <= (lo_row > 0); ++part, dst += static_cast<size_t>(lo_row) * vectors) {
#pragma unroll
            for (int i = 0; i < kHeadVectors; ++i)
                if (lane + 32 * i < vectors)
                    dst[lane + 32 * i] = any ? head[i] : make_uint4(0u, 0u, 0u, 0u);
            for (int i = lane + 32 * kHeadVectors; i < vectors; i += 32)
                dst[i] = any ? src[i] : make_uint4(0u, 0u, 0u, 0u);
        }
    }
}

// ---- forward's last step ---------------------------------------------------------

struct Combine {
    int rows, slices, vocab, width;
    const float *part_max, *part_sum, *part_t;
    const float *label_z;
    const void *x, *weight;
    const void *labels; // one per row, or null with the teacher's row_terms
    int label_bytes;
    int64_t ignore_index;
    const double2 *row_terms;
    float temperature;
    float *losses, *lse;
};

template <bool kBf16>
__device__ __forceinline__ float dot16(uint4 a, uint4 b, float acc)
{
    const uint32_t *u = &a.x, *v = &b.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = unpack16(u[i], kBf16), q = unpack16(v[i], kBf16);
        acc = fmaf(p.x, q.x, acc);
        acc = fmaf(p.y, q.y, acc);
    }
    return acc;
}

// The label's logit as an fp32 dot product by one warp (0 for a label outside the vocabulary).
// The tensor cores truncate each of the width / 16 steps of a logit's sum, which shifts large
// logits, the label's above all, by some 1e-6 of their value.  One dot product per row
// replaces the label's logit where it enters: the loss and, by its probability, the lse.
// Its operands are the call's inputs, complete since the kernel before this one was let past its
// own wait, so it runs before this kernel's.
template <bool kBf16>
__device__ __forceinline__ float label_product(const Combine &p, int row, int lane)
{
    float z = 0.0f;
    const int64_t label = load_label(p.labels, p.label_bytes, row);
    if (label >= 0 && label < p.vocab) {
        const uint4 *a = static_cast<const uint4 *>(p.x) + static_cast<size_t>(row) * (p.width / 8);
        const uint4 *b = static_cast<const uint4 *>(p.weight) + static_cast<size_t>(label) * (p.width / 8);
#pragma unroll 5
        for (int i = lane; i < p.width / 8; i += 32)
            z = dot16<kBf16>(a[i], b[i], z);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
        z += __shfl_xor_sync(0xffffffffu, z, o);
    return z;
}

// One row's loss and lse from its merged maximum, sum and target product.  In 64 bits: the
// loss is a difference of terms near log(V).
__device__ __forceinline__ void write_row(const Combine &p, int row, float mx, float sum, double target, float label_z)
{
    double lse = static_cast<double>(mx) * 0.69314718055994530942 + log(static_cast<double>(sum));
    double loss = 0.0;
    if (p.row_terms) {
        const double2 terms = p.row_terms[row];
        if (terms.y != 0.0) {
            const double temperature = p.temperature;
            loss = temperature * temperature * (terms.x + terms.y * lse - target / temperature);
        }
    } else {
        const int64_t label = load_label(p.labels, p.label_bytes, row);
        if (label >= 0 && label < p.vocab) {
            const double formed = p.label_z[row];
            // One of the two sums may pass fp32's range on its way where the other does not: the
            // finite one counts.
            double z = label_z;
            if (isfinite(formed) && isfinite(z))
                lse -= exp(formed - lse) * (formed - z);
            else if (isfinite(formed))
                z = formed;
            else if (isfinite(z)) // left out of the sum as -infinity
                lse = fmax(lse, z) + log1p(exp(-fabs(lse - z)));
            if (label != p.ignore_index)
                loss = lse - z;
        } else if (label != p.ignore_index) {
            g_token_error = 1;
        }
    }
    p.lse[row] = static_cast<float>(lse);
    p.losses[row] = static_cast<float>(loss);
}

constexpr int kBatch = 8; // partial results of a thread in flight together

// Merges tiles first, first + step, ... of a row.
__device__ __forceinline__ void merge_tiles(const Combine &p, int row, int first, int step, float &mx, float &sum,
                                            double &target)
{
    for (; first < p.slices; first += kBatch * step) {
        float m[kBatch], v[kBatch], t[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int i = first + j * step;
            m[j] = -INFINITY;
            v[j] = t[j] = 0.0f;
            if (i < p.slices) {
                const size_t at = static_cast<size_t>(i) * p.rows + row;
                m[j] = p.part_max[at];
                v[j] = p.part_sum[at];
                if (p.part_t)
                    t[j] = p.part_t[at];
            }
        }
        float next = mx;
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            next = fmaxf(next, m[j]);
        sum *= mx == -INFINITY ? 0.0f : exp2f(mx - next);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (first + j * step < p.slices)
                sum = fmaf(v[j], exp2f(m[j] - next), sum);
            target += t[j];
        }
        mx = next;
    }
}

// Merges (mx, sum, target) with another; an empty side (maximum -infinity, sum 0) adds nothing.
__device__ __forceinline__ void merge_pair(float &mx, float &sum, double &target, float m, float s, double t)
{
    const float next = fmaxf(mx, m);
    sum = (mx == -INFINITY && sum == 0.0f ? 0.0f : sum * exp2f(mx - next)) +
          (m == -INFINITY && s == 0.0f ? 0.0f : s * exp2f(m - next));
    mx = next;
    target += t;
}

// Forward's last step, in a fixed order.  Many rows: 32 rows per block, lane = row (coalesced),
// warps over the column tiles.
constexpr int kCombineGroups = 16;
template <bool kBf16>
__global__ void __launch_bounds__(32 * kCombineGroups) combine_kernel(const Combine p)
{
    __shared__ float s_max[kCombineGroups][32], s_sum[kCombineGroups][32];
    __shared__ double s_t[kCombineGroups][32];
    __shared__ float s_label[32];
    const int group = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int row = blockIdx.x * 32 + lane;
    for (int i = group; p.labels && i < 32 && blockIdx.x * 32 + i < p.rows; i += kCombineGroups) {
        const float z = label_product<kBf16>(p, blockIdx.x * 32 + i, lane);
        if (lane == 0)
            s_label[i] = z;
    }
    griddepcontrol_wait();
    griddepcontrol_launch_dependents();
    float mx = -INFINITY, sum = 0.0f;
    double target = 0.0;
    if (row < p.rows)
        merge_tiles(p, row, group, kCombineGroups, mx, sum, target);
    s_max[group][lane] = mx;
    s_sum[group][lane] = sum;
    s_t[group][lane] = target;
    __syncthreads();
    if (group != 0 || row >= p.rows)
        return;
    for (int i = 1; i < kCombineGroups && i < p.slices; ++i)
        merge_pair(mx, sum, target, s_max[i][lane], s_sum[i][lane], s_t[i][lane]);
    write_row(p, row, mx, sum, target, s_label[lane]);
}

// Few rows: a warp per row, lanes over the column tiles, so that every row's chain is short.
constexpr int kCombineRowWarps = 4;
template <bool kBf16>
__global__ void __launch_bounds__(32 * kCombineRowWarps) combine_rows_kernel(const Combine p)
{
    const int row = blockIdx.x * kCombineRowWarps + threadIdx.x / 32, lane = threadIdx.x % 32;
    const float label_z = p.labels && row < p.rows ? label_product<kBf16>(p, row, lane) : 0.0f;
    griddepcontrol_wait();
    griddepcontrol_launch_dependents();
    if (row >= p.rows)
        return;
    float mx = -INFINITY, sum = 0.0f;
    double target = 0.0;
    merge_tiles(p, row, lane, 32, mx, sum, target);
#pragma unroll
    for (int o = 16; o; o >>= 1)
        merge_pair(mx, sum, target, __shfl_down_sync(0xffffffffu, mx, o), __shfl_down_sync(0xffffffffu, sum, o),
                   __shfl_down_sync(0xffffffffu, target, o));
    if (lane == 0)
        write_row(p, row, mx, sum, target, label_z);
}

// dx = sum of the fp32 planes (one per K split; both parts' rows), in a fixed order, times 1 / s;
// rows that moved come from where they went, rows without a target are zero.
// Few planes, many rows: eight elements per thread, runs of four rows per block, in flight together.
template <bool kBf16>
__global__ void __launch_bounds__(256) planes_kernel(const float *planes, const BackShape *shape, int rows, int width,
                                                     const int *row_at, const float *inv_gain, uint4 *dx)
{
    constexpr int kRows = 4;
    // From the backward's first kernel, which the one before this waited for.
    const float inv = *inv_gain;
    const int vectors = width / 8;
    const int count = shape->splits, parts = shape->lo_row > 0 ? 2 : 1;
    const size_t plane = static_cast<size_t>(shape->plane_rows) * vectors; // in pairs of float4
    const size_t part = static_cast<size_t>(shape->lo_row) * vectors;
    griddepcontrol_wait();
    griddepcontrol_launch_dependents();
    const float4 *all = reinterpret_cast<const float4 *>(planes);
    for (int row0 = blockIdx.x * kRows; row0 < rows; row0 += gridDim.x * kRows) {
        int from[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            from[r] = row0 + r >= rows ? -1 : row_at ? row_at[row0 + r] : row0 + r;
        for (int i = threadIdx.x; i < vectors; i += blockDim.x) {
            float f[kRows][8] = {};
            for (int s = 0; s < count * parts; ++s) {
                float4 v[kRows][2];
#pragma unroll
                for (int r = 0; r < kRows; ++r)
                    if (from[r] >= 0) {
                        const float4 *src = all + 2 * (plane * (s / parts) + part * (s % parts) +
                                                       static_cast<size_t>(from[r]) * vectors + i);
                        v[r][0] = src[0];
                        v[r][1] = src[1];
                    } else {
                        v[r][0] = v[r][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    const float4 lo = v[r][0], hi = v[r][1];
                    f[r][0] += lo.x, f[r][1] += lo.y, f[r][2] += lo.z, f[r][3] += lo.w;
                    f[r][4] += hi.x, f[r][5] += hi.y, f[r][6] += hi.z, f[r][7] += hi.w;
                }
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r)
                if (row0 + r < rows)
                    dx[static_cast<size_t>(row0 + r) * vectors + i] =
                        make_uint4(pack16(f[r][0] * inv, f[r][1] * inv, kBf16), pack16(f[r][2] * inv, f[r][3] * inv, kBf16),
                                   pack16(f[r][4] * inv, f[r][5] * inv, kBf16), pack16(f[r][6] * inv, f[r][7] * inv, kBf16));
        }
    }
}

// Many planes, few rows: a block sums one row's 256 columns, four per thread; its kPlaneGroups
// groups of threads take every kPlaneGroups-th plane and meet in shared memory, so that a
// thread waits for few loads in turn.
constexpr int kPlaneColumns = 256, kPlaneGroups = 8;
template <bool kBf16>
__global__ void __launch_bounds__(kPlaneColumns / 4 * kPlaneGroups)
    planes_row_kernel(const float *planes, const BackShape *shape, int width, const int *row_at, const float *inv_gain,
                      uint2 *dx)
{
    __shared__ float4 sums[kPlaneGroups][kPlaneColumns / 4];
    const float inv = *inv_gain;
    const int row = blockIdx.y, group = threadIdx.y;
    const int column = blockIdx.x * kPlaneColumns / 4 + threadIdx.x, columns = width / 4; // in float4
    const int from = row_at ? row_at[row] : row;
    const int lo_row = shape->lo_row, count = shape->splits;
    const size_t plane = static_cast<size_t>(shape->plane_rows) * columns;
    griddepcontrol_wait();
    griddepcontrol_launch_dependents();
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](const float4 &v) { sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w; };
    if (from >= 0 && column < columns) {
        const float4 *src = reinterpret_cast<const float4 *>(planes) + static_cast<size_t>(from) * columns + column;
        const size_t part = static_cast<size_t>(lo_row) * columns;
#pragma unroll 5
        for (int s = group; s < count; s += kPlaneGroups) {
            add(src[plane * s]);
            if (lo_row > 0)
                add(src[plane * s + part]);
        }
    }
    sums[group][threadIdx.x] = sum;
    __syncthreads();
    if (group != 0 || column >= columns)
        return;
#pragma unroll
    for (int g = 1; g < kPlaneGroups; ++g)
        add(sums[g][threadIdx.x]);
    dx[static_cast<size_t>(row) * columns + column] =
        make_uint2(pack16(sum.x * inv, sum.y * inv, kBf16), pack16(sum.z * inv, sum.w * inv, kBf16));
}

} // namespace vocab

// ---- host ---------------------------------------------------------------------------

namespace {

using namespace vocab;

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Up to this many rows one CTA computes a tile instead of a pair: the rows fit one
// accumulator and W is streamed once.  128 x 1280 x 51866: forward 28.7 us and backward 108 us,
// with pairs 29.8 and 111.
constexpr int64_t kSingleRows = 128;

// Up to this many rows the forward's last step takes a warp per row; above, its strided reads
// cost more than they save.  Whole forward over 384: 333 rows 22.2 us with a warp per row, 25.8
// with 32 rows per block; 1024 rows 35.8 and 37.1; 2048 rows 71.5 and 66.0.
constexpr int64_t kCombineRows = 1024;

// Up to this many planes (or above kPlaneRows rows, a grid's y) dx is summed by runs of rows, else
// a row at a time.  Backward by runs and by row: 2240 x 1024, one plane, 510 and 580 us; 1024 x
// 384, five planes, 127 and 128; 700 x 384, six, 98 and 95; 333 x 384, nine, 74 and 65.
constexpr int64_t kFewPlanes = 5, kPlaneRows = 65535;

// Bytes of one piece of G: the memory a step may take for it, whatever its rows.  Larger pieces
// are faster (14336 x 1280 x 51866: 6.07 ms with 256 MB, 5.94 with 512, 5.82 with all of G).
constexpr int64_t kPieceBytes = int64_t{512} << 20;

// Calls f with the entries per lane (1, 2, 4 or 8) that hold `targets` entries in a warp.
template <class F>
cudaError_t per_lane(int targets, F f)
{
    static_assert(kVocabMaxTargets == 256, "eight entries per lane, and entry numbers of 8 bits in the sort keys");
    if (targets <= 32)
        return f(std::integral_constant<int, 1>{});
    if (targets <= 64)
        return f(std::integral_constant<int, 2>{});
    if (targets <= 128)
        return f(std::integral_constant<int, 4>{});
    return f(std::integral_constant<int, 8>{});
}

struct Arena {
    uint8_t *base;
    int64_t used = 0;
    template <class T>
    T *take(int64_t count)
    {
        T *at = reinterpret_cast<T *>(base + used);
        used += round_up(count * static_cast<int64_t>(sizeof(T)), 256);
        return at;
    }
};

// Width of the equal tiles (multiples of 32) that cover `columns`.
int even_width(int64_t columns)
{
    return static_cast<int>(round_up(ceil_div(columns, ceil_div(columns, kMaxBN)), 32));
}

// Width of z's tiles over `columns`: the one that finishes first, by rounds of the persistent
// CTAs times a tile's time, which grows with its width, a fixed part for A's reads (about 32
// columns' worth) and its start and epilogue (about three K blocks of 256).  20 x 51866: 295
// tiles of 176 for 148 SMs, where 203 of 256 would leave the second round half empty.
int logits_width(int64_t rows, int64_t columns, int64_t width, bool single, int align)
{
    const int64_t units = single ? sm_count() : sm_count() / 2;
    const int64_t m_tiles = ceil_div(rows, single ? kBM : 2 * kBM);
    const int64_t kbs = ceil_div(width, kBK);
    int best = kMaxBN;
    int64_t best_cost = INT64_MAX;
    for (int bn = kMaxBN; bn >= 128; bn -= align) {
        const int64_t rounds = ceil_div(m_tiles * ceil_div(columns, bn), units);
        const int64_t cost = rounds * (kbs * (bn + 32) + 3 * 288);
        if (cost < best_cost) {
            best_cost = cost;
            best = bn;
        }
    }
    return best;
}

struct ForwardPlan {
    bool single;
    int bn;
    int64_t slices; // column tiles
    float *part_max, *part_sum, *part_t, *label_z, *t_prob;
    int32_t *t_index;
    double2 *row_terms;
    int64_t bytes;
};

ForwardPlan plan_forward(const VocabLossLaunch &L, void *workspace)
{
    ForwardPlan f{};
    Arena arena{static_cast<uint8_t *>(workspace)};
    f.single = L.rows <= kSingleRows;
    f.bn = logits_width(L.rows, L.vocab, L.width, f.single, f.single ? 16 : 32);
    f.slices = ceil_div(L.vocab, f.bn);
    f.part_max = arena.take<float>(f.slices * L.rows);
    f.part_sum = arena.take<float>(f.slices * L.rows);
    if (L.targets > 0) {
        f.part_t = arena.take<float>(f.slices * L.rows);
        f.t_index = arena.take<int32_t>(L.rows * L.targets);
        f.t_prob = arena.take<float>(L.rows * L.targets);
        f.row_terms = arena.take<double2>(L.rows);
    } else {
        f.label_z = arena.take<float>(L.rows);
    }
    f.bytes = arena.used;
    return f;
}

// Up to this many rows (a row per thread of prepare_teacher_kernel) a teacher's rows without an
// entry stay where they are: the others would
// fill as many tiles without them, and moving them takes one more launch.  Above it padding costs
// nothing.  Backward, 32 entries, 51866 tokens, moved / in place, us: 256 rows of 512 63 / 57, a
// third of them padding 60 / 57; 300 rows 76 / 73, a third 62 / 72; 1024 rows 150 / 148, a
// third 117 / 140; 2240 rows of 1280, a third 524-586 / 623.
constexpr int64_t kTeacherMoveRows = 256;
static_assert(kTeacherMoveRows == 32 * kPrepWarps, "prepare_teacher_kernel: a row per thread");

// Rows that G and x_used have room for: all of a call's, or both parts of a few.  A part of 8 or 16
// rows, where a call has no more, puts both into one store of 32.  Backward over 51865 tokens with
// those and with 32 always, us: 1 x 384 39.9 and 41.0; 7 x 512 of 5 teacher's entries 46.2 and 47.7;
// 16 x 1280 96.1 and 96.8.
int part_rows(int64_t rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : 32; }
int64_t rows_of_g(int64_t rows)
{
    return std::max<int64_t>(rows, 2 * second_part(static_cast<int>(std::min<int64_t>(rows, kSplitRows)), part_rows(rows)));
}

struct BackwardPlan {
    bool single;             // kGrad by one CTA per tile
    bool moves;              // rows without a target are left out
    int targets;
    int64_t g_rows;
    int64_t piece, pieces;   // vocabulary columns per piece of G
    int64_t ldg;             // elements per row of a piece
    int grad_bn, width_bn;   // tile widths over a piece's columns, and over x's width
    BackCosts costs;
    int64_t splits;          // K splits of dx if every row has a target
    float *row_lse2, *row_gain, *inv_gain, *t_prob, *sorted_prob, *dx_planes;
    int32_t *t_index, *sorted_index, *marks;
    BackShape *shape;
    int *row_at;
    void *x_used, *g;
    int64_t bytes;
};

BackwardPlan plan_backward(const VocabLossLaunch &L, void *workspace)
{
    BackwardPlan b{};
    Arena arena{static_cast<uint8_t *>(workspace)};
    b.single = L.rows <= kSingleRows;
    b.moves = L.targets == 0 || L.rows > kTeacherMoveRows;
    b.targets = L.targets > 0 ? L.targets : 1;
    b.g_rows = rows_of_g(L.rows);
    const int64_t most = std::max<int64_t>(256, kPieceBytes / 2 / b.g_rows / 256 * 256);
    b.pieces = ceil_div(L.vocab, most);
    b.piece = std::min(L.vocab, round_up(ceil_div(L.vocab, b.pieces), 256));
    b.pieces = ceil_div(L.vocab, b.piece);
    b.ldg = round_up(b.piece, 64);
    b.grad_bn = logits_width(L.rows, b.piece, L.width, b.single, 32);
    b.width_bn = even_width(L.width);
    b.costs.kbs = static_cast<int>(ceil_div(b.piece, kBK));
    b.costs.pieces = static_cast<int>(b.pieces);
    b.costs.n_tiles = static_cast<int>(ceil_div(L.width, b.width_bn));
    b.costs.dw_m_tiles = L.dweight ? static_cast<int>(ceil_div(b.piece, 2 * kBM)) : 0;
    b.costs.units = sm_count() / 2;
    b.costs.width = static_cast<int>(L.width);
    b.costs.plane_cap = INT_MAX;
    b.costs.part_rows = part_rows(L.rows);
    float least = INFINITY;
    int kb_per = 1;
    for (int s = 1; s <= b.costs.units; ++s) {
        const float cost =
            split_cost(b.costs, static_cast<int>(L.rows <= kSplitRows ? b.g_rows : L.rows), s, kb_per);
        if (cost < least) {
            least = cost;
            b.splits = ceil_div(b.costs.kbs, kb_per);
        }
    }
    // Planes for those splits, or twice as many where that is at most 16 MB: fewer rows than
    // there can be may want more of them.
    const int64_t plane_rows = b.splits * round_up(b.g_rows, 32);
    b.costs.plane_cap = static_cast<int>(
        std::min<int64_t>(std::max(plane_rows, std::min(2 * plane_rows, (int64_t{16} << 20) / (4 * L.width))), INT_MAX));
    b.row_lse2 = arena.take<float>(L.rows);
    b.row_gain = arena.take<float>(L.rows);
    b.inv_gain = arena.take<float>(1);
    b.t_index = arena.take<int32_t>(L.rows * b.targets);
    b.t_prob = arena.take<float>(L.rows * b.targets);
    if (b.moves)
        b.row_at = arena.take<int>(L.rows);
    if (b.moves && L.targets > 0) {
        b.marks = arena.take<int32_t>(L.rows);
        b.sorted_index = arena.take<int32_t>(L.rows * b.targets);
        b.sorted_prob = arena.take<float>(L.rows * b.targets);
    }
    b.shape = arena.take<BackShape>(1);
    b.x_used = arena.take<uint16_t>(b.g_rows * L.width);
    b.g = arena.take<uint16_t>(b.g_rows * b.ldg);
    if (L.dx)
        b.dx_planes = arena.take<float>(b.costs.plane_cap * L.width);
    b.bytes = arena.used;
    return b;
}

// fp16/bf16 operand [rows, cols], rows `ld` elements apart.
bool map16(CUtensorMap *map, bool bf16, const void *base, int64_t rows, int64_t cols, int64_t ld, int box_cols,
           int box_rows, CUtensorMapSwizzle swizzle)
{
    return make_map_ld(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, base, rows,
                       cols, ld, static_cast<uint32_t>(box_cols), static_cast<uint32_t>(box_rows), swizzle);
}

// Rows of an A tile that are loaded.  Few rows (one CTA's tile) are loaded as such: the rest of
// the tile keeps what shared memory held, and only rows of the accumulator that nothing reads
// are computed from it.
int tile_rows(int64_t rows) { return static_cast<int>(rows < kBM ? round_up(rows, 8) : kBM); }

// An operand of a GEMM: K-major ([mn, k] in memory) or MN-major ([k, mn]).
bool operand_map(CUtensorMap *map, bool bf16, bool mn_major, const void *base, int64_t rows, int64_t cols, int64_t ld,
                 int mn_rows)
{
    return mn_major ? map16(map, bf16, base, rows, cols, ld, 64, kBK, CU_TENSOR_MAP_SWIZZLE_128B)
                    : map16(map, bf16, base, rows, cols, ld, kBK, mn_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// maps: A, B, output, and kBack's second A, B, output.  `tiles`: the most there can be.
template <bool kPair, int MODE, bool kBf16>
cudaError_t launch_one(const CUtensorMap (&maps)[6], int64_t tiles, Params p, cudaStream_t stream)
{
    using C = Cfg<kPair, MODE>;
    auto kernel = gemm_kernel<kPair, MODE, kBf16>;
    static std::atomic<bool> opted[kMaxDevices];
    const int device = current_device();
    if (!opted[device].load(std::memory_order_acquire)) {
        const cudaError_t err =
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
        if (err != cudaSuccess)
            return err;
        opted[device].store(true, std::memory_order_release);
    }
    p.a_rows = tile_rows(p.rows);
    p.idesc_bits = (kBf16 ? (1u << 7) | (1u << 10) : 0u) | (static_cast<uint32_t>(p.bn >> 3) << 17);
    const int64_t units = kPair ? sm_count() / 2 : sm_count();
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(std::min(tiles, units) * (kPair ? 2 : 1)));
    config.blockDim = dim3(C::kThreads);
    config.dynamicSmemBytes = C::kSmemBytes;
    config.stream = stream;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    config.numAttrs = 1;
    if (kPair) {
        attrs[1].id = cudaLaunchAttributeClusterDimension;
        attrs[1].val.clusterDim.x = 2;
        attrs[1].val.clusterDim.y = 1;
        attrs[1].val.clusterDim.z = 1;
        config.numAttrs = 2;
    }
    config.attrs = attrs;
    const cudaError_t err = cudaLaunchKernelEx(&config, kernel, maps[0], maps[1], maps[2], maps[3], maps[4], maps[5], p);
    count_launch();
    return err != cudaSuccess ? err : cudaGetLastError();
}

// z tiles: x [rows, width] times columns [col0, col0 + cols) of W^T.
template <int MODE, bool kBf16>
cudaError_t launch_logits(const VocabLossLaunch &L, const void *x, int64_t col0, int64_t cols, int bn, bool single,
                          const CUtensorMap *out, Params p, cudaStream_t stream)
{
    CUtensorMap maps[6] = {};
    const uint16_t *w = static_cast<const uint16_t *>(L.weight) + col0 * L.width;
    if (!operand_map(&maps[0], kBf16, false, x, L.rows, L.width, L.width, tile_rows(L.rows)) ||
        !operand_map(&maps[1], kBf16, false, w, cols, L.width, L.width, single ? bn : bn / 2))
        return cudaErrorInvalidValue;
    if (out)
        maps[2] = *out;
    p.rows = static_cast<int>(L.rows);
    p.n = static_cast<int>(cols);
    p.bn = bn;
    p.n_tiles = static_cast<int>(ceil_div(cols, bn));
    p.num_kb = static_cast<int>(ceil_div(L.width, kBK));
    p.col0 = static_cast<int>(col0);
    p.scale2 = static_cast<float>(1.4426950408889634 / static_cast<double>(L.temperature));
    const int64_t tiles = ceil_div(L.rows, single ? kBM : 2 * kBM) * p.n_tiles;
    return single ? launch_one<false, MODE, kBf16>(maps, tiles, p, stream)
                  : launch_one<true, MODE, kBf16>(maps, tiles, p, stream);
}

template <bool kBf16>
cudaError_t run_forward(const VocabLossLaunch &L, cudaStream_t stream)
{
    const ForwardPlan f = plan_forward(L, L.workspace);
    cudaError_t err;
    Params p{};
    if (L.targets > 0) {
        Targets t{};
        t.rows = static_cast<int>(L.rows);
        t.vocab = static_cast<int>(L.vocab);
        t.count = L.targets;
        t.tokens = L.teacher_tokens;
        t.logits = L.teacher_logits;
        t.logit_type = L.teacher_type;
        t.inv_temperature = 1.0f / L.temperature;
        t.index = f.t_index;
        t.prob = f.t_prob;
        const int64_t blocks = std::min<int64_t>(ceil_div(L.rows, kPrepWarps), 8 * sm_count());
        err = per_lane(L.targets, [&](auto r) {
            return launch_pdl(targets_kernel<decltype(r)::value>, dim3(static_cast<unsigned>(blocks)),
                              dim3(32 * kPrepWarps), stream, t, f.row_terms, static_cast<int32_t *>(nullptr));
        });
        if (err != cudaSuccess)
            return err;
        p.t_index = f.t_index;
        p.t_prob = f.t_prob;
        p.targets = L.targets;
    }
    p.labels = L.labels;
    p.label_bytes = L.label_bytes;
    p.part_max = f.part_max;
    p.part_sum = f.part_sum;
    p.part_t = f.part_t;
    p.label_z = f.label_z;
    err = launch_logits<kStats, kBf16>(L, L.x, 0, L.vocab, f.bn, f.single, nullptr, p, stream);
    if (err != cudaSuccess)
        return err;
    Combine c{};
    c.rows = static_cast<int>(L.rows);
    c.slices = static_cast<int>(f.slices);
    c.vocab = static_cast<int>(L.vocab);
    c.width = static_cast<int>(L.width);
    c.x = L.x;
    c.weight = L.weight;
    c.part_max = f.part_max;
    c.part_sum = f.part_sum;
    c.part_t = f.part_t;
    c.label_z = f.label_z;
    c.labels = L.targets > 0 ? nullptr : L.labels;
    c.label_bytes = L.label_bytes;
    c.ignore_index = L.ignore_index;
    c.row_terms = f.row_terms;
    c.temperature = L.temperature;
    c.losses = L.losses;
    c.lse = L.lse_out;
    if (L.rows <= kCombineRows)
        return launch_pdl(combine_rows_kernel<kBf16>, dim3(static_cast<unsigned>(ceil_div(L.rows, kCombineRowWarps))),
                          dim3(32 * kCombineRowWarps), stream, c);
    return launch_pdl(combine_kernel<kBf16>, dim3(static_cast<unsigned>(ceil_div(L.rows, 32))), dim3(32 * kCombineGroups),
                      stream, c);
}

// dx (added up in the planes) and dW's rows from the piece of G over columns [col0, col0 + cols).
template <bool kBf16>
cudaError_t launch_back(const VocabLossLaunch &L, const BackwardPlan &b, int64_t col0, int64_t cols,
                        cudaStream_t stream)
{
    CUtensorMap maps[6] = {};
    Params p{};
    p.rows = static_cast<int>(b.g_rows);
    p.shape = b.shape;
    p.n = static_cast<int>(L.width);
    p.bn = b.width_bn;
    p.n_tiles = static_cast<int>(ceil_div(L.width, b.width_bn));
    p.vocab = static_cast<int>(cols);
    p.inv_gain = b.inv_gain;
    p.accumulate = col0 > 0 ? 1 : 0;
    int64_t tiles = 0;
    if (L.dx) {
        const uint16_t *w = static_cast<const uint16_t *>(L.weight) + col0 * L.width;
        const int64_t dims[2] = {L.width, b.costs.plane_cap};
        const int64_t strides[1] = {L.width * 4};
        const uint32_t box[2] = {16u, 32u};
        if (!operand_map(&maps[0], kBf16, false, b.g, b.g_rows, cols, b.ldg, tile_rows(b.g_rows)) ||
            !operand_map(&maps[1], kBf16, true, w, cols, L.width, L.width, 0) ||
            !make_map_nd(&maps[2], CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, b.dx_planes, dims, strides, box,
                         CU_TENSOR_MAP_SWIZZLE_64B))
            return cudaErrorInvalidValue;
        p.want_dx = 1;
        tiles += 2 * b.splits * ceil_div(b.g_rows, 2 * kBM) * p.n_tiles;
    }
    if (L.dweight) {
        uint16_t *dw = static_cast<uint16_t *>(L.dweight) + col0 * L.width;
        if (!operand_map(&maps[3], kBf16, true, b.g, b.g_rows, cols, b.ldg, 0) ||
            !operand_map(&maps[4], kBf16, true, b.x_used, b.g_rows, L.width, L.width, 0) ||
            !map16(&maps[5], kBf16, dw, cols, L.width, L.width, kSub, 32, CU_TENSOR_MAP_SWIZZLE_64B))
            return cudaErrorInvalidValue;
        p.dw_tiles = static_cast<int>(ceil_div(cols, 2 * kBM) * p.n_tiles);
        tiles += p.dw_tiles;
    }
    return launch_one<true, kBack, kBf16>(maps, tiles, p, stream);
}

template <bool kBf16>
cudaError_t run_backward(const VocabLossLaunch &L, cudaStream_t stream)
{
    const BackwardPlan b = plan_backward(L, L.workspace);
    Prepare q{};
    q.t.rows = static_cast<int>(L.rows);
    q.t.vocab = static_cast<int>(L.vocab);
    q.t.count = b.targets;
    q.t.tokens = L.targets > 0 ? L.teacher_tokens : nullptr;
    q.t.logits = L.teacher_logits;
    q.t.logit_type = L.teacher_type;
    q.t.inv_temperature = 1.0f / L.temperature;
    q.t.index = b.t_index;
    q.t.prob = b.t_prob;
    q.labels = L.labels;
    q.label_bytes = L.label_bytes;
    q.ignore_index = L.ignore_index;
    q.temperature = L.temperature;
    q.width = static_cast<int>(L.width);
    q.g_rows = static_cast<int>(b.g_rows);
    q.x = L.x;
    q.x_used = b.x_used;
    q.lse = L.lse_in;
    q.grad = L.dloss;
    q.row_lse2 = b.row_lse2;
    q.row_gain = b.row_gain;
    q.inv_gain = b.inv_gain;
    q.row_at = b.row_at;
    q.costs = b.costs;
    q.shape = b.shape;
    const dim3 teacher_grid(static_cast<unsigned>(std::min<int64_t>(ceil_div(L.rows, kPrepWarps), 8 * sm_count())));
    const int64_t per_block = round_up(ceil_div(L.rows, sm_count()), kRowWarps);
    const dim3 row_grid(static_cast<unsigned>(ceil_div(L.rows, per_block)));
    cudaError_t err;
    if (L.targets == 0) {
        err = launch_pdl(prepare_rows_kernel<false>, row_grid, dim3(32 * kRowWarps), stream, q,
                         static_cast<int>(per_block));
    } else if (!b.moves) {
        err = per_lane(L.targets, [&](auto r) {
            return launch_pdl(prepare_teacher_kernel<decltype(r)::value>, teacher_grid, dim3(32 * kPrepWarps), stream, q);
        });
    } else {
        Targets t = q.t;
        t.index = b.sorted_index;
        t.prob = b.sorted_prob;
        err = per_lane(L.targets, [&](auto r) {
            return launch_pdl(targets_kernel<decltype(r)::value>, teacher_grid, dim3(32 * kPrepWarps), stream, t,
                              static_cast<double2 *>(nullptr), b.marks);
        });
        q.sorted_index = b.sorted_index;
        q.sorted_prob = b.sorted_prob;
        q.labels = b.marks;
        q.label_bytes = 4;
        q.ignore_index = -1;
        if (err == cudaSuccess)
            err = launch_pdl(prepare_rows_kernel<true>, row_grid, dim3(32 * kRowWarps), stream, q,
                             static_cast<int>(per_block));
    }
    if (err != cudaSuccess)
        return err;
    for (int64_t col0 = 0; col0 < L.vocab; col0 += b.piece) {
        const int64_t cols = std::min(b.piece, L.vocab - col0);
        CUtensorMap out;
        if (!map16(&out, kBf16, b.g, b.g_rows, cols, b.ldg, kSub, 32, CU_TENSOR_MAP_SWIZZLE_64B))
            return cudaErrorInvalidValue;
        Params p{};
        p.shape = b.shape;
        p.g_rows = static_cast<int>(b.g_rows);
        p.t_index = b.t_index;
        p.t_prob = b.t_prob;
        p.targets = b.targets;
        p.row_lse2 = b.row_lse2;
        p.row_gain = b.row_gain;
        err = launch_logits<kGrad, kBf16>(L, b.x_used, col0, cols, b.grad_bn, b.single, &out, p, stream);
        if (err == cudaSuccess)
            err = launch_back<kBf16>(L, b, col0, cols, stream);
        if (err != cudaSuccess)
            return err;
    }
    if (L.dx) {
        const float *planes = b.dx_planes;
        const BackShape *shape = b.shape;
        const int *row_at = b.row_at;
        const float *inv_gain = b.inv_gain;
        const int width = static_cast<int>(L.width);
        if (b.splits <= kFewPlanes || L.rows > kPlaneRows) {
            const int64_t threads = std::min<int64_t>(round_up(L.width / 8, 32), 256);
            const int64_t blocks = std::min<int64_t>(ceil_div(L.rows, 4), 4096 / threads * sm_count());
            err = launch_pdl(planes_kernel<kBf16>, dim3(static_cast<unsigned>(blocks)),
                             dim3(static_cast<unsigned>(threads)), stream, planes, shape, static_cast<int>(L.rows), width,
                             row_at, inv_gain, static_cast<uint4 *>(L.dx));
        } else {
            err = launch_pdl(planes_row_kernel<kBf16>,
                             dim3(static_cast<unsigned>(ceil_div(L.width, kPlaneColumns)), static_cast<unsigned>(L.rows)),
                             dim3(kPlaneColumns / 4, kPlaneGroups), stream, planes, shape, width, row_at, inv_gain,
                             static_cast<uint2 *>(L.dx));
        }
    }
    return err;
}

} // namespace

int64_t vocab_loss_workspace(const VocabLossLaunch &L, bool backward)
{
    return backward ? plan_backward(L, nullptr).bytes : plan_forward(L, nullptr).bytes;
}

cudaError_t launch_vocab_loss(const VocabLossLaunch &L, cudaStream_t stream)
{
    return L.bf16 ? run_forward<true>(L, stream) : run_forward<false>(L, stream);
}

cudaError_t launch_vocab_loss_grad(const VocabLossLaunch &L, cudaStream_t stream)
{
    return L.bf16 ? run_backward<true>(L, stream) : run_backward<false>(L, stream);
}

int read_and_clear_token_error()
{
    // The copies follow the default stream's work only: what other streams hold is waited for first.
    // A word that is set between the copies is part of the 1 that is then returned.
    if (cudaDeviceSynchronize() != cudaSuccess)
        return -1;
    int value = 0;
    if (cudaMemcpyFromSymbol(&value, vocab::g_token_error, sizeof(int)) != cudaSuccess)
        return -1;
    const int zero = 0;
    if (value != 0 && cudaMemcpyToSymbol(vocab::g_token_error, &zero, sizeof(int)) != cudaSuccess)
        return -1;
    return value;
}

cudaError_t read_and_clear_vocab_wait_error(int *site)
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
