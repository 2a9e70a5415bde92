// Host-side helpers of the kernel launchers: tensor maps, device properties, the
// shared-memory opt-in and launches with programmatic stream serialisation.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <mutex>
#include <set>
#include <utility>

#include "launch.h"

namespace lffw {

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                   const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                   const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled()
{
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult status{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &status) ==
                cudaSuccess &&
            status == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(ptr);
    });
    return fn;
}

// 2-D row-major tensor [rows, cols] with `elem` bytes per element.
// 2-D tensor map over [rows, cols] elements whose rows are `ld` elements apart
// (ld >= cols: a column window of a wider matrix).
inline bool make_map_ld(CUtensorMap *map, CUtensorMapDataType type, int elem, const void *base, int64_t rows,
                 int64_t cols, int64_t ld, uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle)
{
    EncodeTiledFn fn = encode_tiled();
    if (!fn)
        return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld * elem)};
    const cuuint32_t box[2] = {box_cols, box_rows};
    const cuuint32_t estrides[2] = {1, 1};
    return fn(map, type, 2, const_cast<void *>(base), dims, strides, box, estrides,
              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

inline bool make_map(CUtensorMap *map, CUtensorMapDataType type, int elem, const void *base, int64_t rows,
              int64_t cols, uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle)
{
    EncodeTiledFn fn = encode_tiled();
    if (!fn)
        return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols * elem)};
    const cuuint32_t box[2] = {box_cols, box_rows};
    const cuuint32_t estrides[2] = {1, 1};
    return fn(map, type, 2, const_cast<void *>(base), dims, strides, box, estrides,
              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// N-d tensor map (rank <= 5): dims[0] is the contiguous axis, strides_bytes[i]
// the byte step of axis i + 1.
inline bool make_map_nd(CUtensorMap *map, CUtensorMapDataType type, int rank, const void *base, const int64_t *dims,
                 const int64_t *strides_bytes, const uint32_t *box, CUtensorMapSwizzle swizzle)
{
    EncodeTiledFn fn = encode_tiled();
    if (!fn || rank < 1 || rank > 5)
        return false;
    cuuint64_t d[5], st[4];
    cuuint32_t b[5], es[5];
    for (int i = 0; i < rank; ++i) {
        d[i] = static_cast<cuuint64_t>(dims[i]);
        b[i] = box[i];
        es[i] = 1;
        if (i + 1 < rank)
            st[i] = static_cast<cuuint64_t>(strides_bytes[i]);
    }
    return fn(map, type, static_cast<cuuint32_t>(rank), const_cast<void *>(base), d, st, b, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kMaxDevices = 64;

inline int current_device()
{
    int device = 0;
    cudaGetDevice(&device);
    return device >= 0 && device < kMaxDevices ? device : 0;
}

inline int sm_count()
{
    static std::atomic<int> cache[kMaxDevices];
    const int device = current_device();
    int count = cache[device].load(std::memory_order_relaxed);
    if (count <= 0) {
        cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device);
        count = count > 0 ? count : 148;
        cache[device].store(count, std::memory_order_relaxed);
    }
    return count;
}

// cudaFuncSetAttribute(MaxDynamicSharedMemorySize) once per (kernel, device).
// Keyed by the kernel's address: template instances share a pointer type.
template <class Kernel>
cudaError_t ensure_smem(Kernel kernel, int bytes)
{
    static std::mutex lock;
    static std::set<std::pair<const void *, int>> done;
    const std::pair<const void *, int> key{reinterpret_cast<const void *>(kernel), current_device()};
    std::lock_guard<std::mutex> guard(lock);
    if (done.count(key))
        return cudaSuccess;
    cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err == cudaSuccess)
        done.insert(key);
    return err;
}

// Launches with programmatic stream serialisation: the kernel waits for the
// previous grid (griddepcontrol.wait) before reading anything it wrote.
template <class Kernel, class... Args>
cudaError_t launch_pdl(Kernel kernel, dim3 grid, dim3 block, cudaStream_t stream, Args... args)
{
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = block;
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, kernel, args...);
    count_launch();
    return err != cudaSuccess ? err : cudaGetLastError();
}

} // namespace lffw
