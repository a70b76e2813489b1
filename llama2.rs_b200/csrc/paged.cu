// Paged KV cache: the C entries (checks of arguments), writing rows into pages and reading them back.
//
//   16 bits:  cache = round(x)
//   8 bits:   a = max |x| over a row and head, scale = a / 127, cache = rint(x * (127 / a)), and back: value = cache * scale
//   4 bits:   zero = bf16 at or below min x, scale = least bf16 with 15 scale >= max x - zero, cache = rint((x - zero) / scale), value = zero + scale * cache.  Both are
//             rounded outwards, so that cache stays in 0 .. 15 and no element lies more than half a step off, but for the roundings of x - zero and 1 / scale (15 x 2^-23 of a step); bf16 because it has f32's range in half the bytes (a pair beside
//             the 64 bytes of a head of 128)
//   RoPE:     (a, b) = (x[d], x[d + hd/2]) turned by the angle of the row's position, first: a' = a c - b s, b' = b c + a s, or, as the
//             token loop of this library does it in place, b' = b c + a' s
//
// Both are copies: what they cannot do without is each row read once and written once, and nothing is used twice.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "host_common.h"
#include "kernels.cuh"
#include "model.h"
#include "paged_attend.h"

namespace l2 {

int kv_device(int* sms) {
    static std::atomic<int> known[64];  // SM counts of devices looked at before (zero: none yet)
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return fail(L2_ECUDA, "no usable CUDA device (%s); this library has no CPU fallback", cudaGetErrorString(e));
    if (dev < 0 || dev >= 64) return fail(L2_EINVAL, "device ordinal %d unsupported", dev);
    int n = known[dev].load(std::memory_order_acquire);
    if (!n) {
        int major = 0;
        const cudaError_t a = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
        if (a != cudaSuccess) return fail(L2_ECUDA, "no usable CUDA device (%s); this library has no CPU fallback", cudaGetErrorString(a));
        if (major < 10) return fail(L2_ECUDA, "device %d: this library is built for sm_100a only", dev);
        L2_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        known[dev].store(n, std::memory_order_release);
    }
    *sms = n;
    return L2_OK;
}

namespace {

constexpr int KV_THREADS = 256, KV_WARPS = KV_THREADS / 32, KV_MAX_ROWS = 16;
constexpr int KV_AT_ONCE = 2, KV_READ_AT_ONCE = 4;  // heads that a group of threads has under way

struct KvCopyParams {
    KvPool pool;
    KvStep step;
    KvRows k, v, q, q_out;
    const float* cos; const float* sin;
    int rope_len, rope_in_place;
    int rows;  // of a CTA
    uint32_t by_heads, by_q_heads;  // reciprocals of the kv heads (kv_read_kernel: twice as many) and of q's
};

// Where a row's position is; by one warp a row, the rows of a CTA side by side: three or four loads that depend on one another, once a row.
struct KvPlace { int64_t at, scale; int pos; };  // elements of the pool (-1: no page), of the scales; position, -1: a row that is left out
__device__ __forceinline__ KvPlace kv_place(const KvCopyParams& P, int r) {
    KvPlace w{-1, 0, -1};
    if (r >= P.step.n_rows) return w;
    const int b = kv_find_seq(P.step, r);
    const KvSeq s = kv_seq(P.step, P.pool.page_shift, b);
    if (P.step.kv_len[b] != s.kv) return w;  // (a length beyond the table: what lies at its end belongs to other rows)
    const int pos = s.kv - s.n + (r - s.row0);
    if (r < s.row0 || r >= s.row0 + s.n || pos < 0) return w;
    if (P.cos && pos >= P.rope_len) { kv_report(P.step.status, L2_KV_BAD_ROPE); return w; }
    w.pos = pos;
    const int page = kv_page(P.step, P.pool, b, pos), in = pos & ((1 << P.pool.page_shift) - 1);
    if (page < 0) return w;
    w.at = (int64_t)page * P.pool.page_stride + in * P.pool.pos_stride;
    w.scale = ((int64_t)page * P.pool.n_kv_heads << P.pool.page_shift) + in;
    return w;
}
// u / n by n's reciprocal, 2^32 / n rounded up: exact for u n < 2^32, and u and n stay below 2^13 (n = 1: the reciprocal is taken as 0)
__device__ __forceinline__ int kv_div(int u, uint32_t by) { return by ? (int)__umulhi((uint32_t)u, by) : u; }
__device__ __forceinline__ void kv_places(const KvCopyParams& P, int r0, KvPlace* place) {
    for (int i = threadIdx.x >> 5; i < P.rows; i += KV_WARPS) {
        const KvPlace w = kv_place(P, r0 + i);
        if ((threadIdx.x & 31) == 0) place[i] = w;
    }
    __syncthreads();
}

// two f32 rounded to T, the first in the low half
template <int T>
__device__ __forceinline__ uint32_t kv_pack(float a, float b) {
    uint32_t r;
    if constexpr (T == L2_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// Eight elements as they lie in memory, as f32, and back.
template <int T> struct KvRaw { uint4 w[T == L2_F32 ? 2 : 1]; };
template <int T>
__device__ __forceinline__ KvRaw<T> load_raw(const char* p) {
    KvRaw<T> r;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r.w) / 16); i++) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
template <int T>
__device__ __forceinline__ void to_f32(const KvRaw<T>& r, float* x) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (T == L2_F32) x[i] = __uint_as_float(w[i]);
        else if constexpr (T == L2_F16) x[i] = __half2float(__ushort_as_half((unsigned short)(w[i / 2] >> (16 * (i % 2)))));
        else x[i] = __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
}
template <int T>
__device__ __forceinline__ void store8(char* base, int64_t e, const float* x) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = x[j];
    if constexpr (T == L2_F32) kv_store8(reinterpret_cast<float*>(base) + e, y);
    else if constexpr (T == L2_F16) kv_store8(reinterpret_cast<__half*>(base) + e, y);
    else kv_store8(reinterpret_cast<__nv_bfloat16*>(base) + e, y);
}
// ... that nobody here reads again
template <int T>
__device__ __forceinline__ void stream8(char* base, int64_t e, const float* x) {
    if constexpr (T == L2_F32) {
        float4* p = reinterpret_cast<float4*>(base + 4 * e);
        __stcs(p, make_float4(x[0], x[1], x[2], x[3]));
        __stcs(p + 1, make_float4(x[4], x[5], x[6], x[7]));
    } else {
        __stcs(reinterpret_cast<uint4*>(base + 2 * e), make_uint4(kv_pack<T>(x[0], x[1]), kv_pack<T>(x[2], x[3]), kv_pack<T>(x[4], x[5]), kv_pack<T>(x[6], x[7])));
    }
}
__device__ __forceinline__ float min_nan(float a, float x) {  // NaN if one of them is
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float x) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(x));
    return y;
}
__device__ __forceinline__ float max_abs(float a, float x) {  // NaN if one of them is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(fabsf(x)));
    return y;
}

// A CTA has a few rows (blockIdx.y) of k, v or q (blockIdx.x modulo their number), or a part of one row's heads.  HD / 16 threads have a head, eight
// elements each of its first half and the same of its second: whole lines, and the pairs that RoPE turns in one thread.
// Latency of loads and instructions, then bandwidth, bound it: 7900 rows of 2 x 40 heads of 128, bf16 to int8 (242 MB), take 51 us (4.8 TB/s).  A row a CTA,
// whose look-ups nothing hid, took 76; so did 16 elements of one run a thread with conversion instructions and 110 registers (18 instructions an element).
// To 4 bits (213 MB) 53 us: instructions bound it, 17 an element for two extremes, a rounding and the packing.
template <int T, int HD>
__global__ void __launch_bounds__(KV_THREADS, 4) kv_append_kernel(const __grid_constant__ KvCopyParams P) {
    constexpr bool I8 = T == L2_I8, U4 = T == L2_U4;
    constexpr int LANES = HD / 16, GROUPS = KV_THREADS / LANES, HALF = HD / 2;
    __shared__ KvPlace place[KV_MAX_ROWS];
    const int sub = threadIdx.x % LANES, grp = threadIdx.x / LANES, d = 8 * sub;
    const int arrays = P.q.data ? 3 : 2, what = blockIdx.x % arrays, part = blockIdx.x / arrays, parts = gridDim.x / arrays;  // what: 0 k, 1 v, 2 q
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const KvRows& from = what == 0 ? P.k : what == 1 ? P.v : P.q;
    const int heads = from.heads, units = P.rows * heads;
    const uint32_t by_heads = what == 2 ? P.by_q_heads : P.by_heads;
    const bool turn = P.cos && what != 1;
    char* const to = what == 1 ? P.pool.v : P.pool.k;
    float* const scales = what == 1 ? P.pool.vs : P.pool.ks;
    for (int r0 = blockIdx.y * P.rows; r0 < P.step.n_rows; r0 += gridDim.y * P.rows) {
        kv_places(P, r0, place);
        auto run = [&](auto type) {
            constexpr int IN = decltype(type)::value, SIZE = IN == L2_F32 ? 4 : 2;
#pragma unroll 1
            for (int u0 = part * GROUPS; u0 < units; u0 += parts * GROUPS * KV_AT_ONCE) {  // (whole warps stay together for the shuffles)
                KvRaw<IN> raw[KV_AT_ONCE][2];
                int row[KV_AT_ONCE], head[KV_AT_ONCE];
                bool mine[KV_AT_ONCE];
#pragma unroll
                for (int a = 0; a < KV_AT_ONCE; a++) {
                    const int u = u0 + a * parts * GROUPS + grp;
                    row[a] = kv_div(u, by_heads);
                    head[a] = u - row[a] * heads;
                    mine[a] = u < units && place[row[a]].pos >= 0;
                    raw[a][0] = raw[a][1] = {};
                    if (mine[a]) {
                        const char* p = from.data + ((int64_t)(r0 + row[a]) * from.row_stride + head[a] * from.head_stride + d) * SIZE;
                        raw[a][0] = load_raw<IN>(p);
                        raw[a][1] = load_raw<IN>(p + HALF * SIZE);
                    }
                }
#pragma unroll
                for (int a = 0; a < KV_AT_ONCE; a++) {
                    if (u0 + a * parts * GROUPS >= units) break;  // (whole CTAs)
                    float x[16];
                    to_f32(raw[a][0], x);
                    to_f32(raw[a][1], x + 8);
                    const int at_row = mine[a] ? row[a] : 0;
                    if (turn) {  // products and their sum are rounded one by one, as written
                        const int64_t e = (int64_t)max(place[at_row].pos, 0) * HALF + d;
                        float c[8], s[8];
                        to_f32(load_raw<L2_F32>(reinterpret_cast<const char*>(P.cos + e)), c);
                        to_f32(load_raw<L2_F32>(reinterpret_cast<const char*>(P.sin + e)), s);
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float y = x[i], z = x[i + 8];
                            x[i] = __fsub_rn(__fmul_rn(y, c[i]), __fmul_rn(z, s[i]));
                            x[i + 8] = __fadd_rn(__fmul_rn(P.rope_in_place ? x[i] : y, s[i]), __fmul_rn(z, c[i]));
                        }
                    }
                    if (what == 2) {
                        if (!mine[a]) continue;
                        const int64_t e = (int64_t)(r0 + row[a]) * P.q_out.row_stride + head[a] * P.q_out.head_stride + d;
                        auto out = [&](auto t) { store8<decltype(t)::value>(P.q_out.data, e, x); store8<decltype(t)::value>(P.q_out.data, e + HALF, x + 8); };
                        if (P.q_out.type == L2_F32) out(std::integral_constant<int, L2_F32>());
                        else if (P.q_out.type == L2_F16) out(std::integral_constant<int, L2_F16>());
                        else out(std::integral_constant<int, L2_BF16>());
                        continue;
                    }
                    const int64_t e = place[at_row].at + head[a] * P.pool.head_stride + d;
                    const bool store = mine[a] && place[at_row].at >= 0;
                    if constexpr (I8) {
                        float m = 0.0f;
#pragma unroll
                        for (int i = 0; i < 16; i++) m = max_abs(m, x[i]);
#pragma unroll
                        for (int o = LANES / 2; o; o >>= 1) m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, o));
                        const bool finite = m < INFINITY, zero = m < 0x1p-100f;
                        const float inv = zero ? 0.0f : __fmul_rn(__frcp_rn(m), 127.0f);
                        // (|x| inv is at most 127 and a few units in the last place.  Added to 1.5 x 2^23 it is rounded to a whole number, to nearest even, whose
                        // two's complement is the low byte: a conversion instruction takes four times as long.  What is not finite gives any byte: the scale is NaN.)
                        uint32_t b[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inv), 12582912.0f));
#pragma unroll
                        for (int i = 0; i < 16; i += 4) b[i / 4] = __byte_perm(__byte_perm(b[i], b[i + 1], 0x0040), __byte_perm(b[i + 2], b[i + 3], 0x0040), 0x5410);
                        if (!store) continue;
                        *reinterpret_cast<uint2*>(to + e) = make_uint2(b[0], b[1]);
                        *reinterpret_cast<uint2*>(to + e + HALF) = make_uint2(b[2], b[3]);
                        if (sub == 0) scales[place[at_row].scale + ((int64_t)head[a] << P.pool.page_shift)] =
                            !finite ? __int_as_float(0x7fc00000) : zero ? 0.0f : __fmul_rn(m, 1.0f / 127.0f);
                    } else if constexpr (U4) {
                        float lo = x[0], hi = x[0];
#pragma unroll
                        for (int i = 1; i < 16; i++) { lo = min_nan(lo, x[i]); hi = max_nan(hi, x[i]); }
#pragma unroll
                        for (int o = LANES / 2; o; o >>= 1) { lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o)); hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o)); }
                        const uint32_t low = __float_as_uint(lo);
                        const float zero = __uint_as_float((low + (lo < 0.0f ? 0xffffu : 0u)) & 0xffff0000u), span = __fsub_rn(hi, zero);
                        uint32_t step = __float_as_uint(__fmul_rn(span, 1.0f / 15.0f)) & 0xffff0000u;  // (15 times a bf16 number is exact)
                        if (__fmul_rn(__uint_as_float(step), 15.0f) < span) step += 0x10000u;
                        const bool finite = span < INFINITY, flat = span < 0x1p-100f;
                        const float inv = flat ? 0.0f : __frcp_rn(__uint_as_float(step));
                        // ((x - zero) inv is at most 15 and a few units in the last place.  One rounding to a whole number, as above, of the exact product: rows of 16 bits often
                        // lie next to the middle of a step.  What the number 1.5 x 2^23 adds to all eight is taken off the word.)
                        uint32_t w[2] = {0u, 0u};
#pragma unroll
                        for (int i = 7; i >= 0; i--) {
                            w[0] = (w[0] << 4) + __float_as_uint(__fmaf_rn(__fsub_rn(x[i], zero), inv, 12582912.0f));
                            w[1] = (w[1] << 4) + __float_as_uint(__fmaf_rn(__fsub_rn(x[8 + i], zero), inv, 12582912.0f));
                        }
                        if (!store) continue;
                        constexpr uint32_t ADDED = 0x4b400000u * 0x11111111u;
                        *reinterpret_cast<uint32_t*>(to + e / 2) = w[0] - ADDED;
                        *reinterpret_cast<uint32_t*>(to + (e + HALF) / 2) = w[1] - ADDED;
                        if (sub == 0) reinterpret_cast<uint32_t*>(scales)[place[at_row].scale + ((int64_t)head[a] << P.pool.page_shift)] =
                            !finite ? 0x7fc07fc0u : __float_as_uint(zero) | (flat ? 0u : step >> 16);
                    } else if (store) {
                        store8<T>(to, e, x);
                        store8<T>(to, e + HALF, x + 8);
                    }
                }
            }
        };
        if (from.type == L2_F32) run(std::integral_constant<int, L2_F32>());
        else if (from.type == L2_F16) run(std::integral_constant<int, L2_F16>());
        else run(std::integral_constant<int, L2_BF16>());
        __syncthreads();
    }
}

// Bound by memory.  190,000 rows of 2 x 8 heads of 128, int8 to bf16 (1.2 GB): 210 us, 5.6 TB/s (a plain copy of as much: 6.0).  Five CTAs an SM at 48
// registers, although the int8 forms then spill 13 words: with four and ordinary stores it took 218 us, with six 233.
// 7900 rows of 2 x 40 heads of 128, 4 bits to bf16 (207 MB): 42 us, 4.9 TB/s; issue slots are 63 % busy.
template <int T, int HD>
__global__ void __launch_bounds__(KV_THREADS, 5) kv_read_kernel(const __grid_constant__ KvCopyParams P) {
    constexpr bool I8 = T == L2_I8, U4 = T == L2_U4;
    constexpr int N = I8 || U4 ? 16 : 8, LANES = HD / N, GROUPS = KV_THREADS / LANES;
    __shared__ KvPlace place[KV_MAX_ROWS];
    const int d = N * (threadIdx.x % LANES), grp = threadIdx.x / LANES, heads = P.pool.n_kv_heads, units = 2 * P.rows * heads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int r0 = blockIdx.y * P.rows; r0 < P.step.n_rows; r0 += gridDim.y * P.rows) {
        kv_places(P, r0, place);
#pragma unroll 1
        for (int u0 = blockIdx.x * GROUPS + grp; u0 < units; u0 += gridDim.x * GROUPS * KV_READ_AT_ONCE) {
            uint4 x[KV_READ_AT_ONCE];
            float f[KV_READ_AT_ONCE];
#pragma unroll
            for (int a = 0; a < KV_READ_AT_ONCE; a++) {
                const int u = u0 + a * gridDim.x * GROUPS, r = kv_div(u, P.by_heads), h = u - r * 2 * heads, head = h < heads ? h : h - heads;
                x[a] = make_uint4(0, 0, 0, 0);
                f[a] = 0.0f;
                if (u < units && place[r].at >= 0) {
                    const char* from = h < heads ? P.pool.k : P.pool.v;
                    if constexpr (U4) {
                        const uint2 w = __ldcs(reinterpret_cast<const uint2*>(from + (place[r].at + head * P.pool.head_stride + d) / 2));
                        x[a].x = w.x; x[a].y = w.y;
                    } else {
                        x[a] = __ldcs(reinterpret_cast<const uint4*>(from + (place[r].at + head * P.pool.head_stride + d) * (I8 ? 1 : 2)));
                    }
                    if constexpr (I8 || U4) f[a] = (h < heads ? P.pool.ks : P.pool.vs)[place[r].scale + ((int64_t)head << P.pool.page_shift)];
                }
            }
#pragma unroll
            for (int a = 0; a < KV_READ_AT_ONCE; a++) {
                const int u = u0 + a * gridDim.x * GROUPS, r = kv_div(u, P.by_heads), h = u - r * 2 * heads, head = h < heads ? h : h - heads;
                if (u >= units || place[r].pos < 0) continue;
                const KvRows& to = h < heads ? P.k : P.v;
                float y[N];
                const uint32_t w[4] = {x[a].x, x[a].y, x[a].z, x[a].w}, pair = __float_as_uint(f[a]);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    // 2^23 + 128 + byte, less 2^23 + 128: exact, and no conversion instruction
                    if constexpr (I8) y[i] = (__uint_as_float(__byte_perm(w[i / 4] ^ 0x80808080u, 0x4b000000u, 0x7540 | (i % 4))) - 8388736.0f) * f[a];
                    else if constexpr (U4) y[i] = __fmaf_rn(__uint_as_float((w[i / 8] >> (4 * (i % 8)) & 15u) | 0x4b000000u) - 8388608.0f, kv_pair_scale(pair), kv_pair_zero(pair));
                    else if constexpr (T == L2_F16) y[i] = __half2float(__ushort_as_half((unsigned short)(w[i / 2] >> (16 * (i % 2)))));
                    else y[i] = __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
                }
                const int64_t e = (int64_t)(r0 + r) * to.row_stride + head * to.head_stride + d;
                auto put = [&](auto t) {
#pragma unroll
                    for (int i = 0; i < N; i += 8) stream8<decltype(t)::value>(to.data, e + i, y + i);
                };
                if (to.type == T) __stcs(reinterpret_cast<uint4*>(to.data + 2 * e), x[a]);
                else if (to.type == L2_F32) put(std::integral_constant<int, L2_F32>());
                else if (to.type == L2_F16) put(std::integral_constant<int, L2_F16>());
                else put(std::integral_constant<int, L2_BF16>());
            }
        }
        __syncthreads();
    }
}

int elem_bits(int type) { return type == L2_F32 ? 32 : type == L2_I8 ? 8 : type == L2_U4 ? 4 : 16; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether runs of head_size elements lie apart, each dimension's steps beyond all that is inside it (as every array that is a part of a larger one has it).
struct KvDim { int64_t stride, extent; };
template <size_t N>
bool apart(KvDim (&d)[N], int head_size) {
    std::sort(d, d + N, [](const KvDim& a, const KvDim& b) { return a.stride < b.stride; });
    __int128 span = head_size;
    for (const KvDim& x : d) {
        if (x.extent <= 1) continue;
        if (x.stride < span) return false;
        span += (__int128)x.stride * (x.extent - 1);
    }
    return true;
}

int check_pages(const char* who, const l2_kv_pages* p, KvPool* out) {
    if (!p) return fail(L2_EINVAL, "%s: no pages", who);
    if (p->type != L2_F16 && p->type != L2_BF16 && p->type != L2_I8 && p->type != L2_U4) return fail(L2_EINVAL, "%s: a cache is f16, bf16, int8 or u4 (type %d)", who, p->type);
    if (p->head_size != 64 && p->head_size != 128) return fail(L2_EINVAL, "%s: head size %d (64 or 128)", who, p->head_size);
    int shift = 3;
    while (shift < 8 && (1 << shift) < p->page_size) shift++;
    if ((1 << shift) != p->page_size) return fail(L2_EINVAL, "%s: page size %d (8, 16, 32, 64, 128 or 256)", who, p->page_size);
    if (p->n_pages < 1 || p->n_kv_heads < 1 || p->n_kv_heads > 1024) return fail(L2_EINVAL, "%s: %d pages, %d kv heads", who, p->n_pages, p->n_kv_heads);
    if (!p->k || !p->v || !aligned16(p->k) || !aligned16(p->v)) return fail(L2_EINVAL, "%s: k and v must start on a 16-byte boundary", who);
    const int64_t s[3] = {p->page_stride, p->position_stride, p->head_stride};
    const int least = 128 / elem_bits(p->type);
    for (int64_t x : s)
        if (x < least || x % least || x > ((int64_t)1 << 36)) return fail(L2_EINVAL, "%s: a stride of %lld elements (multiples of 16 bytes)", who, (long long)x);
    KvDim dims[3] = {{p->page_stride, p->n_pages}, {p->position_stride, p->page_size}, {p->head_stride, p->n_kv_heads}};
    if (!apart(dims, p->head_size)) return fail(L2_EINVAL, "%s: pages, positions or heads overlap", who);
    if ((p->type == L2_I8 || p->type == L2_U4) && (!p->k_scale || !p->v_scale || !aligned16(p->k_scale) || !aligned16(p->v_scale)))
        return fail(L2_EINVAL, "%s: an int8 or u4 cache needs scales that start on a 16-byte boundary", who);
    out->k = static_cast<char*>(p->k); out->v = static_cast<char*>(p->v);
    out->ks = p->k_scale; out->vs = p->v_scale;
    out->page_stride = p->page_stride; out->pos_stride = p->position_stride; out->head_stride = p->head_stride;
    out->n_pages = p->n_pages; out->page_shift = shift; out->n_kv_heads = p->n_kv_heads;
    return L2_OK;
}

int check_batch(const char* who, const l2_kv_batch* b, int page_size, KvStep* out) {
    if (!b) return fail(L2_EINVAL, "%s: no batch", who);
    if (b->n_seqs < 0 || b->n_rows < 0 || b->max_rows < 0 || b->table_width < 0) return fail(L2_EINVAL, "%s: a negative size", who);
    if ((int64_t)b->table_width * page_size > (1 << 30) || b->n_rows > (1 << 30)) return fail(L2_ERANGE, "%s: more than 2^30 positions or rows", who);
    if (b->n_seqs > 65536) return fail(L2_EINVAL, "%s: %d sequences (at most 65536)", who, b->n_seqs);
    if (b->n_seqs && (!b->kv_len || !b->row_start || (b->table_width && !b->page_table))) return fail(L2_EINVAL, "%s: null device pointer", who);
    out->table = b->page_table; out->kv_len = b->kv_len; out->row_start = b->row_start; out->status = b->status;
    out->n_seqs = b->n_seqs; out->width = b->table_width; out->n_rows = b->n_rows; out->max_rows = b->max_rows;
    return L2_OK;
}

// (rows that are read may lie on one another: one row for all, by a stride of 0)
int check_rows(const char* who, const char* what, const l2_kv_rows* r, const l2_kv_batch* b, int head_size, int heads, bool written, KvRows* out) {
    if (!r) return fail(L2_EINVAL, "%s: no %s", who, what);
    if (r->type != L2_F32 && r->type != L2_F16 && r->type != L2_BF16) return fail(L2_EINVAL, "%s: %s is f32, f16 or bf16 (type %d)", who, what, r->type);
    if (r->heads != heads) return fail(L2_EINVAL, "%s: %s has %d heads, not %d", who, what, r->heads, heads);
    if (b->n_rows && (!r->data || !aligned16(r->data))) return fail(L2_EINVAL, "%s: %s must start on a 16-byte boundary", who, what);
    const int least = 128 / elem_bits(r->type);
    if ((b->n_rows > 1 && (r->row_stride % least || r->row_stride < 0)) || (heads > 1 && (r->head_stride % least || r->head_stride < 0)))
        return fail(L2_EINVAL, "%s: %s has strides of %lld and %lld elements (multiples of 16 bytes)", who, what, (long long)r->row_stride, (long long)r->head_stride);
    out->data = static_cast<char*>(r->data); out->row_stride = r->row_stride; out->head_stride = r->head_stride;
    out->type = r->type; out->heads = heads;
    KvDim dims[2] = {{r->row_stride, b->n_rows}, {r->head_stride, heads}};
    if (written && !apart(dims, head_size)) return fail(L2_EINVAL, "%s: rows or heads of %s overlap", who, what);
    return L2_OK;
}

// Rows and heads as rows for rows_apart: the wider of the two strides is that of rows, the other belongs to their width.
RowSpan span(const KvRows& r, int n_rows, int head_size) {
    const int64_t size = elem_bits(r.type) / 8;
    int64_t rows = n_rows, row = rows > 1 ? r.row_stride : 0, heads = r.heads, head = heads > 1 ? r.head_stride : 0;
    if (row && row < head) { std::swap(row, head); std::swap(rows, heads); }
    return {reinterpret_cast<uintptr_t>(r.data), row * size, rows, ((heads - 1) * head + head_size) * size};
}

// What attention asks of the heads and sizes, before anything divides by them: query heads per kv head, and tiles that are counted in 31 bits.
int check_heads(const char* who, const l2_kv_pages* p, const l2_kv_batch* b, int n_heads) {
    if (n_heads < 1 || n_heads % p->n_kv_heads || n_heads / p->n_kv_heads > 64)
        return fail(L2_EINVAL, "%s: %d query heads, %d kv heads (1 to 64 times as many)", who, n_heads, p->n_kv_heads);
    const int64_t positions = (int64_t)b->table_width * p->page_size;
    if (((int64_t)b->max_rows * (n_heads / p->n_kv_heads) / 64 + 1) * ((positions + 127) / 128 + 1) >> 31)
        return fail(L2_ERANGE, "%s: %d rows of a sequence over %lld positions (more than 2^31 tiles)", who, b->max_rows, (long long)positions);
    return L2_OK;
}

template <class F>
cudaError_t by_type(int type, int head_size, F f) {
    if (head_size == 128) {
        if (type == L2_F16) return f(std::integral_constant<int, L2_F16>(), std::integral_constant<int, 128>());
        if (type == L2_BF16) return f(std::integral_constant<int, L2_BF16>(), std::integral_constant<int, 128>());
        if (type == L2_U4) return f(std::integral_constant<int, L2_U4>(), std::integral_constant<int, 128>());
        return f(std::integral_constant<int, L2_I8>(), std::integral_constant<int, 128>());
    }
    if (type == L2_F16) return f(std::integral_constant<int, L2_F16>(), std::integral_constant<int, 64>());
    if (type == L2_BF16) return f(std::integral_constant<int, L2_BF16>(), std::integral_constant<int, 64>());
    if (type == L2_U4) return f(std::integral_constant<int, L2_U4>(), std::integral_constant<int, 64>());
    return f(std::integral_constant<int, L2_I8>(), std::integral_constant<int, 64>());
}

// Rows of a CTA and CTAs of a copy: `rounds` rounds of a CTA's groups of threads, where that leaves four CTAs an SM (a CTA's look-ups are a chain of loads, which
// few rows would not pay for); a row's heads in several CTAs where the rows alone do not fill the device.
dim3 copy_grid(KvCopyParams& P, int heads, int arrays, int groups, int rounds, int sms) {
    const int n = P.step.n_rows;
    P.rows = std::max(1, std::min({KV_MAX_ROWS, rounds * groups / heads, (int)((int64_t)n * arrays / (4 * sms))}));
    const int y = (n + P.rows - 1) / P.rows, x = std::min((P.rows * heads + groups - 1) / groups, std::max(1, 4 * sms / (y * arrays)));
    return dim3(x * arrays, std::min(y, 65535));
}
uint32_t reciprocal(int n) { return n > 1 ? (uint32_t)((((uint64_t)1 << 32) + n - 1) / n) : 0; }

}  // namespace

}  // namespace l2

using namespace l2;

extern "C" int l2_kv_append(const l2_kv_pages* pages, const l2_kv_batch* batch, const l2_kv_rows* k, const l2_kv_rows* v, const l2_kv_rows* q,
                            const l2_kv_rows* q_out, const float* rope_cos, const float* rope_sin, int rope_len, void* cuda_stream) {
    return l2_kv_append_rope(pages, batch, k, v, q, q_out, rope_cos, rope_sin, rope_len, L2_ROPE_PAIRS, cuda_stream);
}

extern "C" int l2_kv_append_rope(const l2_kv_pages* pages, const l2_kv_batch* batch, const l2_kv_rows* k, const l2_kv_rows* v, const l2_kv_rows* q,
                                 const l2_kv_rows* q_out, const float* rope_cos, const float* rope_sin, int rope_len, int rotation, void* cuda_stream) {
    clear_error();
    const char* who = "l2_kv_append";
    KvCopyParams P{};
    if (int rc = check_pages(who, pages, &P.pool)) return rc;
    if (int rc = check_batch(who, batch, pages->page_size, &P.step)) return rc;
    if (int rc = check_rows(who, "k", k, batch, pages->head_size, pages->n_kv_heads, false, &P.k)) return rc;
    if (int rc = check_rows(who, "v", v, batch, pages->head_size, pages->n_kv_heads, false, &P.v)) return rc;
    if (!q != !q_out) return fail(L2_EINVAL, "%s: q and q_out go together", who);
    if (q) {
        if (q->heads < 1 || q->heads > 4096) return fail(L2_EINVAL, "%s: q has %d heads", who, q->heads);
        if (int rc = check_rows(who, "q", q, batch, pages->head_size, q->heads, false, &P.q)) return rc;
        if (int rc = check_rows(who, "q_out", q_out, batch, pages->head_size, q->heads, true, &P.q_out)) return rc;
    }
    if (!rope_cos != !rope_sin || (rope_cos && (rope_len < 1 || !aligned16(rope_cos) || !aligned16(rope_sin))))
        return fail(L2_EINVAL, "%s: both rope tables, on a 16-byte boundary, of at least one position", who);
    if (rotation != L2_ROPE_PAIRS && rotation != L2_ROPE_MODEL) return fail(L2_EINVAL, "%s: rotation %d (L2_ROPE_PAIRS or L2_ROPE_MODEL)", who, rotation);
    P.cos = rope_cos; P.sin = rope_sin; P.rope_len = rope_len; P.rope_in_place = rotation == L2_ROPE_MODEL;
    int sms;
    if (int rc = kv_device(&sms)) return rc;
    if (!batch->n_rows || !batch->n_seqs) return L2_OK;
    const dim3 grid = copy_grid(P, std::max(pages->n_kv_heads, q ? q->heads : 0), q ? 3 : 2, KV_THREADS / (pages->head_size / 16), 8, sms);
    P.by_heads = reciprocal(pages->n_kv_heads);
    P.by_q_heads = reciprocal(q ? q->heads : 1);
    L2_CUDA(by_type(pages->type, pages->head_size, [&](auto t, auto hd) {
        return kv_launch(kv_append_kernel<decltype(t)::value, decltype(hd)::value>, grid, KV_THREADS, 0, static_cast<cudaStream_t>(cuda_stream), P);
    }));
    return L2_OK;
}

extern "C" int l2_kv_read(const l2_kv_pages* pages, const l2_kv_batch* batch, const l2_kv_rows* k, const l2_kv_rows* v, void* cuda_stream) {
    clear_error();
    const char* who = "l2_kv_read";
    KvCopyParams P{};
    if (int rc = check_pages(who, pages, &P.pool)) return rc;
    if (int rc = check_batch(who, batch, pages->page_size, &P.step)) return rc;
    if (int rc = check_rows(who, "k", k, batch, pages->head_size, pages->n_kv_heads, true, &P.k)) return rc;
    if (int rc = check_rows(who, "v", v, batch, pages->head_size, pages->n_kv_heads, true, &P.v)) return rc;
    int sms;
    if (int rc = kv_device(&sms)) return rc;
    if (!batch->n_rows || !batch->n_seqs) return L2_OK;
    const dim3 grid = copy_grid(P, 2 * pages->n_kv_heads, 1, KV_THREADS / (pages->head_size / (pages->type == L2_I8 || pages->type == L2_U4 ? 16 : 8)), 8, sms);
    P.by_heads = reciprocal(2 * pages->n_kv_heads);
    L2_CUDA(by_type(pages->type, pages->head_size, [&](auto t, auto hd) {
        return kv_launch(kv_read_kernel<decltype(t)::value, decltype(hd)::value>, grid, KV_THREADS, 0, static_cast<cudaStream_t>(cuda_stream), P);
    }));
    return L2_OK;
}

extern "C" size_t l2_kv_attend_workspace_bytes(const l2_kv_pages* pages, const l2_kv_batch* batch, int n_heads) {
    clear_error();
    const char* who = "l2_kv_attend_workspace_bytes";
    KvPool pool;
    KvStep step;
    int sms;
    if (check_pages(who, pages, &pool) || check_batch(who, batch, pages->page_size, &step) || check_heads(who, pages, batch, n_heads) || kv_device(&sms)) return 0;
    return kv_attend_work(step, pool, n_heads, pages->type, pages->head_size, sms);
}

extern "C" int l2_kv_attend(const l2_kv_pages* pages, const l2_kv_batch* batch, const l2_kv_rows* q, const l2_kv_rows* out, float scale, int window, int sinks,
                            void* workspace, size_t workspace_bytes, void* cuda_stream) {
    clear_error();
    const char* who = "l2_kv_attend";
    KvAttendParams P{};
    if (int rc = check_pages(who, pages, &P.pool)) return rc;
    if (int rc = check_batch(who, batch, pages->page_size, &P.step)) return rc;
    if (!q) return fail(L2_EINVAL, "%s: no q", who);
    if (int rc = check_heads(who, pages, batch, q->heads)) return rc;
    if (int rc = check_rows(who, "q", q, batch, pages->head_size, q->heads, false, &P.q)) return rc;
    if (int rc = check_rows(who, "out", out, batch, pages->head_size, q->heads, true, &P.out)) return rc;
    if (q->type == L2_F32 || (pages->type != L2_I8 && pages->type != L2_U4 && q->type != pages->type))
        return fail(L2_EINVAL, "%s: q must be of the cache's type (f16 or bf16 with an int8 or u4 cache)", who);
    if (out->type != L2_F32 && out->type != q->type) return fail(L2_EINVAL, "%s: out must be of q's type or f32", who);
    // (of 4 bits some rows may be taken again behind the first results: see paged_tc.cu)
    if (pages->type == L2_U4 && batch->n_rows && !rows_apart(span(P.out, batch->n_rows, pages->head_size), span(P.q, batch->n_rows, pages->head_size)))
        return fail(L2_EINVAL, "%s: out overlaps q, which a u4 cache does not allow", who);
    if (window < 0 || sinks < 0 || !(scale > 0.0f) || !(scale < 1e30f)) return fail(L2_EINVAL, "%s: window %d, sinks %d, scale %g", who, window, sinks, scale);
    int sms;
    if (int rc = kv_device(&sms)) return rc;
    const size_t need = kv_attend_work(P.step, P.pool, q->heads, pages->type, pages->head_size, sms);
    if (workspace_bytes < need || (need && (!workspace || !aligned16(workspace)))) return fail(L2_EINVAL, "%s: a workspace of %zu bytes on a 16-byte boundary needed", who, need);
    if (!batch->n_rows || !batch->n_seqs) return L2_OK;
    P.scale_log2 = scale * 1.4426950408889634f;
    // (a window as wide as the table leaves nothing out; below that, positions and windows of up to 2^30 can be added and subtracted in 32 bits)
    P.window = window < (int64_t)batch->table_width << P.pool.page_shift ? window : 0;
    P.sinks = P.window ? sinks : 0;
    P.group = q->heads / pages->n_kv_heads;
    P.group_inv = (65536 + P.group - 1) / P.group;
    P.work = workspace;
    L2_CUDA(launch_kv_attend(P, pages->type, pages->head_size, sms, static_cast<cudaStream_t>(cuda_stream)));
    return L2_OK;
}
