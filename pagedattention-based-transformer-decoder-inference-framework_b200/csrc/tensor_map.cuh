// tensor_map.cuh -- the driver's encoder of TMA tensor maps, without linking the driver library.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

namespace pa {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static inline EncodeTiledFn driver_encode_tiled() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres) == cudaSuccess && qres == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}

// A driver call fails on a host thread that has no context yet: the runtime binds the device's primary one at a thread's first launch or allocation,
// and the encoder may come before both.  So it is bound here and the call repeated.
static inline CUresult encode_tiled(CUtensorMap* map, CUtensorMapDataType type, cuuint32_t rank, void* ptr, const cuuint64_t* dims, const cuuint64_t* strides,
                                    const cuuint32_t* box, const cuuint32_t* elem_strides, CUtensorMapInterleave interleave, CUtensorMapSwizzle swizzle,
                                    CUtensorMapL2promotion promotion, CUtensorMapFloatOOBfill fill) {
    const EncodeTiledFn fn = driver_encode_tiled();
    const CUresult r = fn(map, type, rank, ptr, dims, strides, box, elem_strides, interleave, swizzle, promotion, fill);
    int dev = 0;
    if (r == CUDA_SUCCESS || cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return r;
    return fn(map, type, rank, ptr, dims, strides, box, elem_strides, interleave, swizzle, promotion, fill);
}
// null: the driver has no encoder
static inline EncodeTiledFn encode_fn() { return driver_encode_tiled() ? encode_tiled : nullptr; }

}  // namespace pa
