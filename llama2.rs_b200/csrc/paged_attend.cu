// l2_kv_attend: which sequences which kernel takes, and the simplest form, for the sequences that no other takes.  A warp has one row and query
// head and walks the positions that the row sees, with the running maximum and sum of the softmax; lanes split the head's elements.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kernels.cuh"
#include "paged_attend.h"

namespace l2 {

namespace {

template <int T, int HD>
__global__ void __launch_bounds__(128) kv_attend_kernel(const __grid_constant__ KvAttendParams P, const int lim) {
    constexpr int N = HD / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int head = blockIdx.x, kvh = head / P.group;
    for (int r = blockIdx.y * 4 + warp; r < P.step.n_rows; r += gridDim.y * 4) {
        const int b = kv_find_seq(P.step, r);
        const KvSeq s = kv_seq(P.step, P.pool.page_shift, b);
        if (r < s.row0 || r >= s.row0 + s.n || (int64_t)s.n * P.group <= lim) continue;
        const int pos = s.kv - s.n + (r - s.row0), d = lane * N;
        float q[N], acc[N] = {}, m = -INFINITY, l = 0.0f;
        for (int i = 0; i < N; i++) {
            const int64_t e = r * P.q.row_stride + head * P.q.head_stride + d + i;
            q[i] = P.q.type == L2_F16 ? __half2float(reinterpret_cast<const __half*>(P.q.data)[e]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(P.q.data)[e]);
        }
        const int from = P.window ? max(0, pos - P.window + 1) : 0;
        for (int j = 0; j <= pos; j++) {
            if (j < from && j >= P.sinks) j = from;
            const int page = kv_page(P.step, P.pool, b, j), at = j & ((1 << P.pool.page_shift) - 1);
            const int64_t e = (int64_t)page * P.pool.page_stride + at * P.pool.pos_stride + kvh * P.pool.head_stride + d;
            float k[N] = {}, v[N] = {};
            if (page >= 0) {
                float ks = 1.0f, vs = 1.0f;
                if constexpr (T == L2_I8) {
                    const int64_t at_s = ((int64_t)page * P.pool.n_kv_heads + kvh << P.pool.page_shift) + at;
                    ks = P.pool.ks[at_s]; vs = P.pool.vs[at_s];
                }
                for (int i = 0; i < N; i++) {
                    if constexpr (T == L2_I8) { k[i] = P.pool.k[e + i] * ks; v[i] = P.pool.v[e + i] * vs; }
                    else {
                        using E = typename KvElem<T>::type;
                        k[i] = (float)reinterpret_cast<const E*>(P.pool.k)[e + i];
                        v[i] = (float)reinterpret_cast<const E*>(P.pool.v)[e + i];
                    }
                }
            }
            float x = 0.0f;
            for (int i = 0; i < N; i++) x += q[i] * k[i];
            for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
            x *= P.scale_log2;
            const float m1 = fmaxf(m, x), ref = m1 == -INFINITY ? 0.0f : m1, f = exp2f(m - ref), p = exp2f(x - ref);  // (a NaN reaches acc through p)
            for (int i = 0; i < N; i++) acc[i] = acc[i] * f + p * v[i];
            l = l * f + p;
            m = m1;
        }
        for (int i = 0; i < N; i++) {
            const int64_t e = r * P.out.row_stride + head * P.out.head_stride + d + i;
            const float y = pos < 0 ? 0.0f : acc[i] / l;
            if (P.out.type == L2_F32) reinterpret_cast<float*>(P.out.data)[e] = y;
            else if (P.out.type == L2_F16) reinterpret_cast<__half*>(P.out.data)[e] = __float2half(y);
            else reinterpret_cast<__nv_bfloat16*>(P.out.data)[e] = __float2bfloat16(y);
        }
    }
}

}  // namespace

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
    const CUresult r = encode(map, type == L2_I8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type == L2_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                              const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              head_size * size == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

size_t kv_attend_work(const KvStep& s, const KvPool& p, int n_heads, int, int head_size, int sms) {
    return std::max<size_t>(16, kv_rows_work(s, p, n_heads / p.n_kv_heads, head_size, sms));
}

cudaError_t launch_kv_attend(const KvAttendParams& p, int type, int head_size, int sms, cudaStream_t st) {
    if (cudaError_t e = launch_kv_rows(p, type, head_size, sms, st)) return e;
    const int lim = kv_rows_limit(p.step, p.group);
    if ((int64_t)p.step.max_rows * p.group <= lim) return cudaSuccess;
    const dim3 grid(p.q.heads, std::min((p.step.n_rows + 3) / 4, 65535));
    auto go = [&](auto t, auto hd) { kv_attend_kernel<decltype(t)::value, decltype(hd)::value><<<grid, 128, 0, st>>>(p, lim); };
    auto by_size = [&](auto t) { head_size == 128 ? go(t, std::integral_constant<int, 128>()) : go(t, std::integral_constant<int, 64>()); };
    if (type == L2_F16) by_size(std::integral_constant<int, L2_F16>());
    else if (type == L2_BF16) by_size(std::integral_constant<int, L2_BF16>());
    else by_size(std::integral_constant<int, L2_I8>());
    g_launches++;
    return cudaGetLastError();
}

}  // namespace l2
