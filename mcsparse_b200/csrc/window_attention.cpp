// Which kernels a windowed-attention call runs on, and the tensor maps of the tensor-core ones.
#include "api_common.h"
#include "window_maps.h"

namespace mcsp_b200 {

namespace {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, looked up once (the library links no libcuda).
EncodeTiled encoder() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

}  // namespace

bool head_map(CUtensorMap* map, const AttentionTensor& t, int64_t tokens, int heads, int dim, macaDataType type, int rows) {
    const EncodeTiled encode = encoder();
    if (encode == nullptr) return false;
    const bool shared = t.head == 0 || heads == 1;
    const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)(shared ? 1 : heads), (cuuint64_t)(tokens > 0 ? tokens : 1)};
    // (a stride of a dimension of one is never used; it only has to be a legal one)
    const cuuint64_t strides[2] = {(cuuint64_t)(shared ? 256 : t.head * 2), (cuuint64_t)(tokens <= 1 ? 256 : t.token * 2)};
    const cuuint32_t box[3] = {64, 1, (cuuint32_t)rows}, step[3] = {1, 1, 1};
    return encode(map, type == MACA_R_16BF ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, t.p, dims, strides,
                  box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The tensor cores take 16-bit types whose rows and strides are multiples of 16 bytes; a scale of 0 (every score equal, also
// the masked ones' -inf times 0) and everything else go to the kernels that walk row by row.
static bool tensor_cores(const AttentionArgs& a) {
    return a.type != MACA_R_32F && a.scale != 0.0f && a.total_q > 0 && a.total_k > 0 &&
           window_tensor_ready(a.q, a.total_q, a.q_heads, a.dim) && window_tensor_ready(a.k, a.total_k, a.kv_heads, a.dim) &&
           window_tensor_ready(a.v, a.total_k, a.kv_heads, a.dim) && window_tensor_ready(a.o, a.total_q, a.q_heads, a.dim);
}

cudaError_t window_attention(cudaStream_t s, const AttentionArgs& a) {
    if (a.total_q == 0 || a.batch == 0) return cudaSuccess;
    if (tensor_cores(a)) {
        const cudaError_t e = window_forward_mma(s, a);
        if (e != cudaErrorNotSupported) return e;
    }
    return window_rows_forward(s, a);
}

size_t window_attention_backward_bytes(const AttentionArgs& a) {
    return a.type != MACA_R_32F ? window_backward_mma_bytes(a) : 256;
}

cudaError_t window_attention_backward(cudaStream_t s, const AttentionArgs& a, void* buffer) {
    if (a.batch == 0) return cudaSuccess;
    if (tensor_cores(a) && window_tensor_ready(a.d_o, a.total_q, a.q_heads, a.dim) && window_tensor_ready(a.dq, a.total_q, a.q_heads, a.dim) &&
        window_tensor_ready(a.dk, a.total_k, a.kv_heads, a.dim) && window_tensor_ready(a.dv, a.total_k, a.kv_heads, a.dim)) {
        const cudaError_t e = window_backward_mma(s, a, buffer);
        if (e != cudaErrorNotSupported) return e;
    }
    return window_rows_backward(s, a);
}

size_t window_attention_decode_bytes(const DecodeArgs& a) { return a.type != MACA_R_32F ? window_decode_mma_bytes(a) : 256; }

cudaError_t window_attention_decode(cudaStream_t s, const DecodeArgs& a, void* buffer) {
    if (a.batch == 0) return cudaSuccess;
    return window_decode_ready(a) ? window_decode_mma(s, a, buffer) : window_rows_decode(s, a);
}

}  // namespace mcsp_b200
