// The driver's encoder of tensor maps, found once.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

typedef CUresult (*encode_tiled_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                    const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                    CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static inline encode_tiled_fn tensor_map_encoder() {
    static encode_tiled_fn encode = nullptr;
    if (!encode) {
        cudaDriverEntryPointQueryResult qr;
        void* fn = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qr) == cudaSuccess && fn &&
            qr == cudaDriverEntryPointSuccess)
            encode = (encode_tiled_fn)fn;
    }
    return encode;
}
