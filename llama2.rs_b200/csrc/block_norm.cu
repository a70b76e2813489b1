// Norms before and after a block, with its gate, its scale and the residual stream in one pass (l2_block_norm):
//   t = y / sqrt(mean(y^2) + eps) w,   r = x + s g t,   out = r / sqrt(mean(r^2) + eps) v
// A row is read once and stays in registers between the two sums; x is on its way while y's sum is formed.  Bound by memory where rows are many, else by the trip to
// memory and the two meetings of a row's threads.  Rows longer than 16384 (32 elements a thread, x and r beside one another in 64 registers) go through local memory in part, 600 to 800 bytes a
// thread: 400 rows of 28672 take 39 us where their bytes need 21, 400 of 16384 22 where they need 12.
// 8191 rows of 8192, bf16 beside an f32 residual (805 MB): 126 us, 6.4 TB/s (a plain copy 6.5; with the next row on its way into shared memory meanwhile, two CTAs an SM, 130, and rows of 2048 55 us instead of 36).  A row of 4096 with 200 of them or one: 4 us, which is latency.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "host_common.h"
#include "kernels.cuh"
#include "model.h"
#include "paged_attend.h"
#include "paged_device.cuh"

namespace l2 {

namespace {

struct BnRows { char* data; int64_t stride; int type; };
struct BnParams {
    BnRows block, residual, gate, residual_out, out;
    const float* post; const float* pre;
    float scale, eps;
    int rows, dim;
};

// V elements as they lie in memory (of 32 bits, or two a word), and as f32
template <int V> struct BnRaw { uint32_t w[V]; };
template <int V>
__device__ __forceinline__ BnRaw<V> bn_load(const BnRows& a, int64_t row, int e) {
    BnRaw<V> r;
    const int64_t at = row * a.stride + e;
    if constexpr (V == 4) {
        if (a.type == L2_F32) {
            const uint4 x = __ldcs(reinterpret_cast<const uint4*>(a.data + 4 * at));
            r.w[0] = x.x; r.w[1] = x.y; r.w[2] = x.z; r.w[3] = x.w;
        } else {
            const uint2 x = __ldcs(reinterpret_cast<const uint2*>(a.data + 2 * at));
            r.w[0] = x.x; r.w[1] = x.y; r.w[2] = r.w[3] = 0u;
        }
    } else {
        if (a.type == L2_F32) r.w[0] = __ldcs(reinterpret_cast<const uint32_t*>(a.data + 4 * at));
        else r.w[0] = __ldcs(reinterpret_cast<const unsigned short*>(a.data + 2 * at));
    }
    return r;
}
template <int V>
__device__ __forceinline__ void bn_values(const BnRaw<V>& r, int type, float* x) {  // (branches, all threads the same way: a choice at every element is three conversions each)
    if (type == L2_F32) {
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = __uint_as_float(r.w[i]);
    } else if (type == L2_BF16) {
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = __uint_as_float(V == 4 && i % 2 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = __half2float(__ushort_as_half((unsigned short)(V == 4 ? r.w[i / 2] >> (16 * (i % 2)) : r.w[0])));
    }
}
template <int V>
__device__ __forceinline__ void bn_store(const BnRows& a, int64_t row, int e, const float* x) {
    const int64_t at = row * a.stride + e;
    if (a.type == L2_F32) {
        if constexpr (V == 4) __stcs(reinterpret_cast<float4*>(a.data + 4 * at), make_float4(x[0], x[1], x[2], x[3]));
        else *reinterpret_cast<float*>(a.data + 4 * at) = x[0];
    } else if constexpr (V == 4) {
        uint32_t w[2];
        if (a.type == L2_F16) {
            const __half2 p = __floats2half2_rn(x[0], x[1]), q = __floats2half2_rn(x[2], x[3]);
            w[0] = *reinterpret_cast<const uint32_t*>(&p); w[1] = *reinterpret_cast<const uint32_t*>(&q);
        } else {
            const __nv_bfloat162 p = __floats2bfloat162_rn(x[0], x[1]), q = __floats2bfloat162_rn(x[2], x[3]);
            w[0] = *reinterpret_cast<const uint32_t*>(&p); w[1] = *reinterpret_cast<const uint32_t*>(&q);
        }
        __stcs(reinterpret_cast<uint2*>(a.data + 2 * at), make_uint2(w[0], w[1]));
    } else if (a.type == L2_F16) {
        reinterpret_cast<__half*>(a.data)[at] = __float2half_rn(x[0]);
    } else {
        reinterpret_cast<__nv_bfloat16*>(a.data)[at] = __float2bfloat16_rn(x[0]);
    }
}

// The sum over a row's threads: a warp, or the CTA (scratch: a word a warp, used in turn with another).
template <bool WARP>
__device__ __forceinline__ float bn_sum(float x, float* scratch) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if constexpr (!WARP) {
        const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
        if (lane == 0) scratch[threadIdx.x >> 5] = x;
        __syncthreads();
        x = lane < warps ? scratch[lane] : 0.0f;
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    }
    return x;
}

// f with the type as a constant: loops over a thread's elements go inside, so that there is one choice an array.
template <class F>
__device__ __forceinline__ void bn_by_type(int type, F f) {
    if (type == L2_F32) f(std::integral_constant<int, L2_F32>());
    else if (type == L2_BF16) f(std::integral_constant<int, L2_BF16>());
    else f(std::integral_constant<int, L2_F16>());
}
__device__ __forceinline__ BnRows bn_of(BnRows a, int type) { a.type = type; return a; }

// E elements a thread, V of them side by side.  WARP: a warp has a row, else a CTA.
template <int E, int V, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) block_norm_kernel(const __grid_constant__ BnParams P) {
    constexpr int N = E / V;
    __shared__ float scratch[2][32];
    const int threads = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int64_t step = WARP ? (int64_t)gridDim.x * (blockDim.x >> 5) : gridDim.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x; row < P.rows; row += step) {
        BnRaw<V> y[N], x[N];
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int i = 0; i < V; i++) y[n].w[i] = x[n].w[i] = 0u;
        auto load = [&](const BnRows& from, BnRaw<V>* to) {
            bn_by_type(from.type, [&](auto type) {
#pragma unroll
                for (int n = 0; n < N; n++) {
                    const int e = (n * threads + t) * V;
                    if (e < P.dim) to[n] = bn_load<V>(bn_of(from, decltype(type)::value), row, e);
                }
            });
        };
        if (P.block.data) load(P.block, y);
        if (P.residual.data) load(P.residual, x);
        float r[E];
        bn_by_type(P.block.type, [&](auto type) {
#pragma unroll
            for (int n = 0; n < N; n++) bn_values<V>(y[n], decltype(type)::value, r + n * V);
        });
        if (P.post) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < E; i++) sum = fmaf(r[i], r[i], sum);
            sum = bn_sum<WARP>(sum, scratch[0]);
            const float f = 1.0f / sqrtf(sum / (float)P.dim + P.eps);
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int e = (n * threads + t) * V;
                if (e < P.dim) {
                    float w[V];
                    if constexpr (V == 4) { const float4 q = *reinterpret_cast<const float4*>(P.post + e); w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w; }
                    else w[0] = P.post[e];
#pragma unroll
                    for (int i = 0; i < V; i++) r[n * V + i] = r[n * V + i] * f * w[i];
                }
            }
        }
        if (P.gate.data) {
            bn_by_type(P.gate.type, [&](auto type) {
#pragma unroll
                for (int n = 0; n < N; n++) {
                    const int e = (n * threads + t) * V;
                    if (e >= P.dim) continue;
                    float g[V];
                    bn_values<V>(bn_load<V>(bn_of(P.gate, decltype(type)::value), row, e), decltype(type)::value, g);
#pragma unroll
                    for (int i = 0; i < V; i++) r[n * V + i] *= g[i];
                }
            });
        }
        bn_by_type(P.residual.type, [&](auto type) {
#pragma unroll
            for (int n = 0; n < N; n++) {
                float v[V];
                bn_values<V>(x[n], decltype(type)::value, v);
#pragma unroll
                for (int i = 0; i < V; i++) r[n * V + i] = fmaf(P.scale, r[n * V + i], v[i]);
            }
        });
        if (P.residual_out.data)
            bn_by_type(P.residual_out.type, [&](auto type) {
#pragma unroll
                for (int n = 0; n < N; n++) {
                    const int e = (n * threads + t) * V;
                    if (e < P.dim) bn_store<V>(bn_of(P.residual_out, decltype(type)::value), row, e, r + n * V);
                }
            });
        if (!P.out.data) {
            if (!WARP && P.post) __syncthreads();  // (the scratch of this row's sum, before the next row's)
            continue;
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < E; i++) sum = fmaf(r[i], r[i], sum);
        sum = bn_sum<WARP>(sum, scratch[1]);
        const float f = 1.0f / sqrtf(sum / (float)P.dim + P.eps);
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int e = (n * threads + t) * V;
            if (e >= P.dim) continue;
            float w[V];
#pragma unroll
            for (int i = 0; i < V; i++) w[i] = 1.0f;
            if (P.pre) {
                if constexpr (V == 4) { const float4 q = *reinterpret_cast<const float4*>(P.pre + e); w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w; }
                else w[0] = P.pre[e];
            }
#pragma unroll
            for (int i = 0; i < V; i++) r[n * V + i] = r[n * V + i] * f * w[i];
        }
        bn_by_type(P.out.type, [&](auto type) {
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int e = (n * threads + t) * V;
                if (e < P.dim) bn_store<V>(bn_of(P.out, decltype(type)::value), row, e, r + n * V);
            }
        });
        if constexpr (!WARP) {
            if (!P.post) __syncthreads();  // (the scratch of one row's second sum, before the next row's)
        }
    }
}

int bn_bytes(int type) { return type == L2_F32 ? 4 : 2; }

// `quads`: whether all arrays can be taken four elements at a time
int check_rows(const char* who, const char* what, const l2_rows& a, const l2_block_norm_args* args, bool written, BnRows* out, bool* quads) {
    out->data = static_cast<char*>(a.data); out->stride = a.row_stride; out->type = a.type;
    if (!a.data) { out->type = L2_F32; return L2_OK; }
    if (a.type != L2_F32 && a.type != L2_F16 && a.type != L2_BF16) return fail(L2_EINVAL, "%s: %s is f32, f16 or bf16 (type %d)", who, what, a.type);
    const int size = bn_bytes(a.type);
    if (reinterpret_cast<uintptr_t>(a.data) % size) return fail(L2_EINVAL, "%s: %s does not start on a boundary of its elements", who, what);
    if (a.row_stride < 0 || a.row_stride > ((int64_t)1 << 40) || (written && args->rows > 1 && a.row_stride < args->dim))
        return fail(L2_EINVAL, "%s: %s has rows %lld elements apart", who, what, (long long)a.row_stride);
    if (reinterpret_cast<uintptr_t>(a.data) % (4 * size) || (args->rows > 1 && a.row_stride % 4)) *quads = false;
    return L2_OK;
}
RowSpan span(const BnRows& a, int rows, int dim) { return {reinterpret_cast<uintptr_t>(a.data), a.stride * bn_bytes(a.type), a.data ? rows : 0, (int64_t)dim * bn_bytes(a.type)}; }
bool same(const BnRows& a, const BnRows& b, int rows) { return a.data && a.data == b.data && a.type == b.type && (rows < 2 || a.stride == b.stride); }

}  // namespace

}  // namespace l2

using namespace l2;

extern "C" int l2_block_norm(const l2_block_norm_args* a, void* cuda_stream) {
    clear_error();
    const char* who = "l2_block_norm";
    if (!a) return fail(L2_EINVAL, "%s: no arguments", who);
    BnParams P{};
    bool quads = a->dim % 4 == 0;
    if (a->rows < 0 || a->dim < 1 || a->dim > 32768) return fail(L2_EINVAL, "%s: %d rows of %d elements (1 to 32768)", who, a->rows, a->dim);
    if (int rc = check_rows(who, "block", a->block, a, false, &P.block, &quads)) return rc;
    if (int rc = check_rows(who, "residual", a->residual, a, false, &P.residual, &quads)) return rc;
    if (int rc = check_rows(who, "gate", a->gate, a, false, &P.gate, &quads)) return rc;
    if (int rc = check_rows(who, "residual_out", a->residual_out, a, true, &P.residual_out, &quads)) return rc;
    if (int rc = check_rows(who, "out", a->out, a, true, &P.out, &quads)) return rc;
    if (a->rows) {  // (arrays of no rows may have no address)
        if (!P.block.data && !P.residual.data) return fail(L2_EINVAL, "%s: neither block nor residual", who);
        if (!P.residual_out.data && !P.out.data) return fail(L2_EINVAL, "%s: neither residual_out nor out", who);
        if (!P.block.data && (P.gate.data || a->post_weight)) return fail(L2_EINVAL, "%s: a gate or post_weight without a block", who);
    }
    if (!(a->eps >= 0.0f) || !(a->eps < 1e30f) || !(a->scale - a->scale == 0.0f)) return fail(L2_EINVAL, "%s: scale %g, eps %g", who, a->scale, a->eps);
    const float* weights[2] = {a->post_weight, a->pre_weight};
    for (const float* w : weights) {
        if (reinterpret_cast<uintptr_t>(w) & 3) return fail(L2_EINVAL, "%s: weights that do not start on a 4-byte boundary", who);
        if (reinterpret_cast<uintptr_t>(w) & 15) quads = false;
    }
    if (a->rows) {
        // (in place: every element is written by the thread that has read it, or, of out, after its row has been read)
        const RowSpan w[2] = {span(P.residual_out, a->rows, a->dim), span(P.out, a->rows, a->dim)};
        const BnRows* read[3] = {&P.block, &P.residual, &P.gate};
        bool fine = rows_apart(w[0], w[1]);
        for (int i = 0; i < 2; i++) {
            for (int k = 0; k < 3; k++)
                fine &= rows_apart(w[i], span(*read[k], a->rows, a->dim)) || (i == 0 && k == 1 && same(P.residual_out, P.residual, a->rows)) || (i == 1 && k == 0 && same(P.out, P.block, a->rows));
            for (const float* v : weights) fine &= !v || rows_apart(w[i], {reinterpret_cast<uintptr_t>(v), 0, 1, 4 * (int64_t)a->dim});
        }
        if (!fine) return fail(L2_EINVAL, "%s: results overlap one another or what is read", who);
    }
    P.post = a->post_weight; P.pre = a->pre_weight; P.scale = a->scale; P.eps = a->eps; P.rows = a->rows; P.dim = a->dim;
    int sms;
    if (int rc = kv_device(&sms)) return rc;
    if (!a->rows) return L2_OK;
    // A row in a warp where there are many rows that 32 threads hold (5000 rows of 512: 6.7 us, with a CTA a row 9.6; 148 rows: 3.1 and 2.5).  Else a CTA a row.  With four elements a
    // thread, or eight of rows longer than 4096, as long as an SM gets no more than 1024 threads that way (592 rows of 1024: 3.3 us, with 16 elements 4.5; 148 of 4096: 3.8 and 4.6;
    // 200 of 5120: 4.7 and 5.1); else with 16, or 32 of rows longer than 16384 (740 of 1024: 4.6 us, with four 5.2; 222 of 4096: 4.9 and 6.6).
    const bool warp = a->dim <= 512 && a->rows >= 4 * sms;
    int elements = 4, threads = 32;
    auto widen = [&]() {
        while (elements < 32 && 1024 * elements < a->dim) elements *= 2;
        threads = std::min(1024, (a->dim + 32 * elements - 1) / (32 * elements) * 32);
    };
    if (warp) {
        while (elements < 16 && 32 * elements < a->dim) elements *= 2;
    } else {
        widen();
        if (elements < 16 && (int64_t)a->rows * threads > 1024 * sms) { elements = 16; widen(); }
    }
    auto go = [&](auto e, auto v, auto w) {
        constexpr bool W = decltype(w)::value;
        const int64_t ctas = W ? ((int64_t)a->rows + 7) / 8 : a->rows, most = (int64_t)sms * (W ? 8 : std::max(1, 2048 / threads));
        return kv_launch(block_norm_kernel<decltype(e)::value, decltype(v)::value, W>, dim3((unsigned)std::min(ctas, most)), W ? 256 : threads, 0, static_cast<cudaStream_t>(cuda_stream), P);
    };
    auto by_e = [&](auto v, auto w) {
        if (elements == 4) return go(std::integral_constant<int, 4>(), v, w);
        if (elements == 8) return go(std::integral_constant<int, 8>(), v, w);
        if (elements == 16) return go(std::integral_constant<int, 16>(), v, w);
        if constexpr (decltype(w)::value) return cudaErrorInvalidValue;  // (a warp has rows of up to 512)
        else return go(std::integral_constant<int, 32>(), v, w);
    };
    auto by_v = [&](auto w) { return quads ? by_e(std::integral_constant<int, 4>(), w) : by_e(std::integral_constant<int, 1>(), w); };
    L2_CUDA(warp ? by_v(std::true_type()) : by_v(std::false_type()));
    return L2_OK;
}
