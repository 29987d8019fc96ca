// tmap.cuh -- 2-D TMA tensor maps, encoded through the driver entry point and
// cached per host thread.
//
// A tensor map only describes an address range (base, extents, strides, box,
// swizzle), never the contents, so a map made for the same description is
// always valid again; caching it takes cuTensorMapEncodeTiled (several
// microseconds of host time) off every launch.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

namespace b200q8 {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

typedef CUresult (*CtxGetCurrentFn)(CUcontext*);

inline void* driver_entry(const char* name)
{
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q{};
    const bool found = cudaGetDriverEntryPoint(name, &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess;
    cudaGetLastError();
    return found ? ptr : nullptr;
}

inline EncodeTiledFn encode_fn()
{
    static const EncodeTiledFn fn = reinterpret_cast<EncodeTiledFn>(driver_entry("cuTensorMapEncodeTiled"));
    return fn;
}

// The encoder needs a context, and a host thread whose first CUDA call this is has none yet (asking for the
// device's number binds none): the current device's primary context, as a launch would bind it.
inline bool bind_context()
{
    static const CtxGetCurrentFn current = reinterpret_cast<CtxGetCurrentFn>(driver_entry("cuCtxGetCurrent"));
    CUcontext ctx = nullptr;
    if (current && current(&ctx) == CUDA_SUCCESS && ctx) return true;
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}

struct TmapDesc {
    const void* base;
    uint64_t inner, outer;    // extents in elements (inner = contiguous dimension)
    uint64_t row_bytes;       // stride of the outer dimension
    uint32_t box_inner, box_outer;
    int dtype;                // CUtensorMapDataType
    int swizzle;              // CUtensorMapSwizzle
    bool operator==(const TmapDesc& o) const { return memcmp(this, &o, sizeof(TmapDesc)) == 0; }
};

// Row-major 2-D map with zero fill out of range; false if the driver refuses it.
inline bool tmap_2d(CUtensorMap* out, const TmapDesc& d)
{
    constexpr int kEntries = 64;
    struct Cache {
        TmapDesc key[kEntries];
        CUtensorMap map[kEntries];
        int used = 0, next = 0;
    };
    static thread_local Cache c;
    for (int i = 0; i < c.used; i++)
        if (c.key[i] == d) {
            *out = c.map[i];
            return true;
        }
    EncodeTiledFn enc = encode_fn();
    if (!enc || !bind_context()) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)d.inner, (cuuint64_t)d.outer};
    const cuuint64_t strides[1] = {(cuuint64_t)d.row_bytes};
    const cuuint32_t box[2] = {d.box_inner, d.box_outer};
    const cuuint32_t es[2] = {1, 1};
    CUtensorMap m;
    if (enc(&m, (CUtensorMapDataType)d.dtype, 2, const_cast<void*>(d.base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, (CUtensorMapSwizzle)d.swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return false;
    const int slot = c.used < kEntries ? c.used++ : (c.next++ % kEntries);
    c.key[slot] = d;
    c.map[slot] = m;
    *out = m;
    return true;
}

}  // namespace b200q8
