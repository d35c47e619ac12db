// Host side of the tensor-core kernels: tensor maps.
#include "tensor.cuh"

namespace p2b {

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (EncodeTiled)p;
    }();
    return fn;
}

// A thread that has made no runtime call yet has no context, and the driver's call does not bring it about as the runtime's calls do.
template <class Call> static CUresult with_context(Call call) {
    CUresult rc = call();
    int device = 0;
    if (rc == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) rc = call();
    return rc;
}

int encode_rows(CUtensorMap* map, const void* base, int element, int64_t columns, int64_t rows, int64_t stride_bytes, int box_rows) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return set_error(P2B_ERR_STATE, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / element), (cuuint32_t)box_rows}, steps[2] = {1, 1};
    const CUresult rc = with_context([&] {
        return encode(map, element == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2,
                      const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    });
    if (rc != CUDA_SUCCESS)
        return set_error(P2B_ERR_ARG, "tensor map of %lld x %lld elements refused (%d)", (long long)rows, (long long)columns, (int)rc);
    return P2B_OK;
}

int encode_pieces(CUtensorMap* map, const void* base, int64_t pieces) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return set_error(P2B_ERR_STATE, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t dims[2] = {128, (cuuint64_t)pieces * 8}, strides[1] = {128};
    const cuuint32_t box[2] = {128, 8}, steps[2] = {1, 1};
    const CUresult rc = with_context([&] {
        return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    });
    if (rc != CUDA_SUCCESS) return set_error(P2B_ERR_ARG, "tensor map of %lld pieces refused (%d)", (long long)pieces, (int)rc);
    return P2B_OK;
}

}  // namespace p2b
