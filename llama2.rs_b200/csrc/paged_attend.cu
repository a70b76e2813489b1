// Attention of a batch's rows over the paged cache: the simplest form that is right for every case.  A warp has one row and query head
// and walks the positions that the row sees, with the running maximum and sum of the softmax; lanes split the head's elements.
#include <cuda_runtime.h>

#include <type_traits>

#include "kernels.cuh"
#include "paged.cuh"

namespace l2 {

namespace {

template <int T, int HD>
__global__ void __launch_bounds__(128) kv_attend_kernel(const __grid_constant__ KvAttendParams P) {
    constexpr int N = HD / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int head = blockIdx.x, kvh = head / P.group;
    for (int r = blockIdx.y * 4 + warp; r < P.step.n_rows; r += gridDim.y * 4) {
        const int b = kv_find_seq(P.step, r);
        const KvSeq s = kv_seq(P.step, P.pool.page_shift, b);
        if (r < s.row0 || r >= s.row0 + s.n) continue;
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

size_t kv_attend_work(const KvStep&, const KvPool&, int, int, int, int) { return 16; }

cudaError_t launch_kv_attend(const KvAttendParams& p, int type, int head_size, int, cudaStream_t st) {
    const dim3 grid(p.q.heads, std::min((p.step.n_rows + 3) / 4, 65535));
    auto go = [&](auto t, auto hd) { kv_attend_kernel<decltype(t)::value, decltype(hd)::value><<<grid, 128, 0, st>>>(p); };
    auto by_size = [&](auto t) { head_size == 128 ? go(t, std::integral_constant<int, 128>()) : go(t, std::integral_constant<int, 64>()); };
    if (type == L2_F16) by_size(std::integral_constant<int, L2_F16>());
    else if (type == L2_BF16) by_size(std::integral_constant<int, L2_BF16>());
    else by_size(std::integral_constant<int, L2_I8>());
    g_launches++;
    return cudaGetLastError();
}

}  // namespace l2
