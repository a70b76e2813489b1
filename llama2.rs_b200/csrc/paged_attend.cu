// l2_kv_attend: which kernel takes which sequences, and the TMA maps of a cache.
#include <cuda_runtime.h>

#include <algorithm>

#include "paged_attend.h"

namespace l2 {

cudaError_t kv_map(CUtensorMap* map, const KvPool& p, const void* base, int type, int head_size, int tile) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<Encode> known{nullptr};
    Encode encode = known.load(std::memory_order_acquire);
    if (!encode) {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult r;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r);
        if (e != cudaSuccess) return e;
        if (r != cudaDriverEntryPointSuccess || !f) return cudaErrorSymbolNotFound;
        encode = reinterpret_cast<Encode>(f);
        known.store(encode, std::memory_order_release);
    }
    const int size = type == L2_I8 ? 1 : 2, page = 1 << p.page_shift;
    const cuuint64_t dims[4] = {(cuuint64_t)head_size, (cuuint64_t)page, (cuuint64_t)p.n_kv_heads, (cuuint64_t)p.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)p.pos_stride * size, (cuuint64_t)p.head_stride * size, (cuuint64_t)p.page_stride * size};
    const cuuint32_t box[4] = {(cuuint32_t)std::min(head_size, 128 / size), (cuuint32_t)std::min(page, tile), 1, 1}, step[4] = {1, 1, 1, 1};
    // (A row of 256 bytes comes in two copies: the first brings both halves to the L2, 115 -> 112 us for 672 MB of them; rows of 128 take 112 us as they are, 125 in pairs.)
    const CUresult r = encode(map, type == L2_I8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type == L2_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                              const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              head_size * size == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, head_size * size == 256 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

size_t kv_attend_work(const KvStep& s, const KvPool& p, int n_heads, int type, int head_size, int sms) {  // the kernels run one after the other
    const int group = n_heads / p.n_kv_heads;
    return std::max<size_t>(16, std::max(kv_rows_work(s, p, group, type, head_size, sms), kv_tc_work(s, p, group, head_size, sms)));
}

cudaError_t launch_kv_attend(const KvAttendParams& p, int type, int head_size, int sms, cudaStream_t st) {
    if (cudaError_t e = launch_kv_rows(p, type, head_size, sms, st)) return e;
    return launch_kv_tc(p, type, head_size, sms, st);
}

}  // namespace l2
