// Paged KV cache: the C entries (checks of arguments), writing rows into pages and reading them back.
//
//   16 bits:  cache = round(x)
//   8 bits:   a = max |x| over a row and head, scale = a / 127, cache = rint(x * (127 / a)), and back: value = cache * scale
//   RoPE:     (x[d], x[d + hd/2]) turned by the angle of the row's position, first
//
// Both are copies: what they cannot do without is each row read once and written once, and nothing is used twice.
#include <cuda_runtime.h>

#include <atomic>

#include "host_common.h"
#include "kernels.cuh"
#include "model.h"
#include "paged.cuh"

namespace l2 {

namespace {

constexpr int KV_THREADS = 256;

struct KvCopyParams {
    KvPool pool;
    KvStep step;
    KvRows k, v, q, q_out;
    const float* cos; const float* sin;
    int rope_len;
};

// One row a CTA (blockIdx.y strides over the rows), LANES = hd / 8 threads for a head, 8 elements each.
template <int T, int HD>
__global__ void __launch_bounds__(KV_THREADS) kv_append_kernel(const __grid_constant__ KvCopyParams P) {
    constexpr int LANES = HD / 8, GROUPS = KV_THREADS / LANES;
    const int sub = threadIdx.x % LANES, grp = threadIdx.x / LANES, d = 8 * sub, half = HD / 2;
    const int kvh = P.pool.n_kv_heads, units = 2 * kvh + (P.q.data ? P.q.heads : 0);
    for (int r = blockIdx.y; r < P.step.n_rows; r += gridDim.y) {
        const int b = kv_find_seq(P.step, r);
        const KvSeq s = kv_seq(P.step, P.pool.page_shift, b);
        const int pos = s.kv - s.n + (r - s.row0);
        if (r < s.row0 || r >= s.row0 + s.n || pos < 0) continue;
        if (P.cos && pos >= P.rope_len) { kv_report(P.step.status, L2_KV_BAD_ROPE); continue; }
        const int page = kv_page(P.step, P.pool, b, pos), at = pos & ((1 << P.pool.page_shift) - 1);
        for (int u0 = blockIdx.x * GROUPS; u0 < units; u0 += gridDim.x * GROUPS) {  // (whole warps stay together for the shuffles)
            const int u = min(u0 + grp, units - 1);
            const bool mine = u0 + grp < units;
            const int what = u < kvh ? 0 : u < 2 * kvh ? 1 : 2, head = u - what * kvh;
            float x[8];
            kv_load8(what == 0 ? P.k : what == 1 ? P.v : P.q, r, head, d, x);
            if (P.cos) {  // products and their sum are rounded one by one, as written
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = __shfl_xor_sync(0xffffffffu, x[i], LANES / 2);
                if (what != 1) {
                    const int e = d & (half - 1);
                    float c[8], w[8];
                    kv_load8(P.cos + (size_t)pos * half + e, c);
                    kv_load8(P.sin + (size_t)pos * half + e, w);
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        x[i] = d < half ? __fsub_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], w[i])) : __fadd_rn(__fmul_rn(y[i], w[i]), __fmul_rn(x[i], c[i]));
                }
            }
            if (what == 2) {
                if (mine) kv_store8(P.q_out, r, head, d, x);
                if constexpr (T != L2_I8) continue;
            }
            const int64_t e = (int64_t)page * P.pool.page_stride + at * P.pool.pos_stride + head * P.pool.head_stride + d;
            char* to = what == 1 ? P.pool.v : P.pool.k;
            if constexpr (T == L2_I8) {
                // the row's largest magnitude, as bits: of non-negative floats the order of the bits is that of the values, NaN above all
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
                for (int o = LANES / 2; o; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                const float a = __uint_as_float(most);
                const bool finite = most < 0x7f800000u, zero = a < 0x1p-100f;
                const float inv = finite && !zero ? __fmul_rn(__frcp_rn(a), 127.0f) : 0.0f;
                uint32_t w[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int v = finite ? max(-127, min(127, __float2int_rn(__fmul_rn(x[i], inv)))) : 0;
                    w[i / 4] |= (uint32_t)(v & 255) << (8 * (i % 4));
                }
                if (!mine || page < 0 || what == 2) continue;
                *reinterpret_cast<uint2*>(to + e) = make_uint2(w[0], w[1]);
                if (sub == 0) (what == 1 ? P.pool.vs : P.pool.ks)[((int64_t)page * kvh + head << P.pool.page_shift) + at] =
                    !finite ? __int_as_float(0x7fc00000) : zero ? 0.0f : __fmul_rn(a, 1.0f / 127.0f);
            } else {
                using E = typename KvElem<T>::type;
                if (mine && page >= 0) kv_store8(reinterpret_cast<E*>(to) + e, x);
            }
        }
    }
}

template <int T, int HD>
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(const __grid_constant__ KvCopyParams P) {
    constexpr int LANES = HD / 8, GROUPS = KV_THREADS / LANES;
    const int d = 8 * (threadIdx.x % LANES), grp = threadIdx.x / LANES, kvh = P.pool.n_kv_heads;
    for (int r = blockIdx.y; r < P.step.n_rows; r += gridDim.y) {
        const int b = kv_find_seq(P.step, r);
        const KvSeq s = kv_seq(P.step, P.pool.page_shift, b);
        const int pos = s.kv - s.n + (r - s.row0);
        if (r < s.row0 || r >= s.row0 + s.n || pos < 0) continue;
        const int page = kv_page(P.step, P.pool, b, pos), at = pos & ((1 << P.pool.page_shift) - 1);
        for (int u = blockIdx.x * GROUPS + grp; u < 2 * kvh; u += gridDim.x * GROUPS) {
            const int what = u >= kvh, head = u - what * kvh;
            float x[8] = {};
            if (page >= 0) {
                const int64_t e = (int64_t)page * P.pool.page_stride + at * P.pool.pos_stride + head * P.pool.head_stride + d;
                const char* from = what ? P.pool.v : P.pool.k;
                if constexpr (T == L2_I8) {
                    const float f = (what ? P.pool.vs : P.pool.ks)[((int64_t)page * kvh + head << P.pool.page_shift) + at];
                    kv_load8(reinterpret_cast<const int8_t*>(from) + e, x);
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] *= f;
                } else {
                    kv_load8(reinterpret_cast<const typename KvElem<T>::type*>(from) + e, x);
                }
            }
            kv_store8(what ? P.v : P.k, r, head, d, x);
        }
    }
}

// SM count of the current device; L2_ECUDA where there is none that this library runs on.
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

int elem_bytes(int type) { return type == L2_F32 ? 4 : type == L2_I8 ? 1 : 2; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_pages(const char* who, const l2_kv_pages* p, KvPool* out) {
    if (!p) return fail(L2_EINVAL, "%s: no pages", who);
    if (p->type != L2_F16 && p->type != L2_BF16 && p->type != L2_I8) return fail(L2_EINVAL, "%s: a cache is f16, bf16 or int8 (type %d)", who, p->type);
    if (p->head_size != 64 && p->head_size != 128) return fail(L2_EINVAL, "%s: head size %d (64 or 128)", who, p->head_size);
    int shift = 3;
    while (shift < 8 && (1 << shift) < p->page_size) shift++;
    if ((1 << shift) != p->page_size) return fail(L2_EINVAL, "%s: page size %d (8, 16, 32, 64, 128 or 256)", who, p->page_size);
    if (p->n_pages < 1 || p->n_kv_heads < 1 || p->n_kv_heads > 1024) return fail(L2_EINVAL, "%s: %d pages, %d kv heads", who, p->n_pages, p->n_kv_heads);
    if (!p->k || !p->v || !aligned16(p->k) || !aligned16(p->v)) return fail(L2_EINVAL, "%s: k and v must start on a 16-byte boundary", who);
    const int64_t s[3] = {p->page_stride, p->position_stride, p->head_stride};
    const int least = 16 / elem_bytes(p->type);
    for (int64_t x : s)
        if (x < least || x % least || x > ((int64_t)1 << 36)) return fail(L2_EINVAL, "%s: a stride of %lld elements (multiples of 16 bytes)", who, (long long)x);
    if ((p->position_stride < p->head_size && p->page_size > 1) || (p->head_stride < p->head_size && p->n_kv_heads > 1))
        return fail(L2_EINVAL, "%s: positions or heads overlap", who);
    if (p->type == L2_I8 && (!p->k_scale || !p->v_scale || !aligned16(p->k_scale) || !aligned16(p->v_scale)))
        return fail(L2_EINVAL, "%s: an int8 cache needs scales that start on a 16-byte boundary", who);
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

int check_rows(const char* who, const char* what, const l2_kv_rows* r, const l2_kv_batch* b, int head_size, int heads, KvRows* out) {
    if (!r) return fail(L2_EINVAL, "%s: no %s", who, what);
    if (r->type != L2_F32 && r->type != L2_F16 && r->type != L2_BF16) return fail(L2_EINVAL, "%s: %s is f32, f16 or bf16 (type %d)", who, what, r->type);
    if (r->heads != heads) return fail(L2_EINVAL, "%s: %s has %d heads, not %d", who, what, r->heads, heads);
    if (b->n_rows && (!r->data || !aligned16(r->data))) return fail(L2_EINVAL, "%s: %s must start on a 16-byte boundary", who, what);
    const int least = 16 / elem_bytes(r->type);
    if ((b->n_rows > 1 && (r->row_stride % least || r->row_stride < 0)) || (heads > 1 && (r->head_stride % least || r->head_stride < 0)))
        return fail(L2_EINVAL, "%s: %s has strides of %lld and %lld elements (multiples of 16 bytes)", who, what, (long long)r->row_stride, (long long)r->head_stride);
    out->data = static_cast<char*>(r->data); out->row_stride = r->row_stride; out->head_stride = r->head_stride;
    out->type = r->type; out->heads = heads;
    (void)head_size;
    return L2_OK;
}

template <class F>
int by_type(int type, int head_size, F f) {
    if (head_size == 128) {
        if (type == L2_F16) return f(std::integral_constant<int, L2_F16>(), std::integral_constant<int, 128>());
        if (type == L2_BF16) return f(std::integral_constant<int, L2_BF16>(), std::integral_constant<int, 128>());
        return f(std::integral_constant<int, L2_I8>(), std::integral_constant<int, 128>());
    }
    if (type == L2_F16) return f(std::integral_constant<int, L2_F16>(), std::integral_constant<int, 64>());
    if (type == L2_BF16) return f(std::integral_constant<int, L2_BF16>(), std::integral_constant<int, 64>());
    return f(std::integral_constant<int, L2_I8>(), std::integral_constant<int, 64>());
}

// CTAs of a copy: a row's heads in one CTA where the rows fill the device, spread over several where they do not.
dim3 copy_grid(int rows, int units, int head_size, int sms) {
    const int groups = KV_THREADS / (head_size / 8), blocks = (units + groups - 1) / groups;
    const int x = std::min(blocks, std::max(1, 4 * sms / std::max(1, rows)));
    return dim3(x, std::min(rows, 65535));
}

}  // namespace

}  // namespace l2

using namespace l2;

extern "C" int l2_kv_append(const l2_kv_pages* pages, const l2_kv_batch* batch, const l2_kv_rows* k, const l2_kv_rows* v, const l2_kv_rows* q,
                            const l2_kv_rows* q_out, const float* rope_cos, const float* rope_sin, int rope_len, void* cuda_stream) {
    clear_error();
    const char* who = "l2_kv_append";
    KvCopyParams P{};
    if (int rc = check_pages(who, pages, &P.pool)) return rc;
    if (int rc = check_batch(who, batch, pages->page_size, &P.step)) return rc;
    if (int rc = check_rows(who, "k", k, batch, pages->head_size, pages->n_kv_heads, &P.k)) return rc;
    if (int rc = check_rows(who, "v", v, batch, pages->head_size, pages->n_kv_heads, &P.v)) return rc;
    if (!q != !q_out) return fail(L2_EINVAL, "%s: q and q_out go together", who);
    if (q) {
        if (q->heads < 1) return fail(L2_EINVAL, "%s: q has %d heads", who, q->heads);
        if (int rc = check_rows(who, "q", q, batch, pages->head_size, q->heads, &P.q)) return rc;
        if (int rc = check_rows(who, "q_out", q_out, batch, pages->head_size, q->heads, &P.q_out)) return rc;
    }
    if (!rope_cos != !rope_sin || (rope_cos && (rope_len < 1 || !aligned16(rope_cos) || !aligned16(rope_sin))))
        return fail(L2_EINVAL, "%s: both rope tables, on a 16-byte boundary, of at least one position", who);
    P.cos = rope_cos; P.sin = rope_sin; P.rope_len = rope_len;
    int sms;
    if (int rc = kv_device(&sms)) return rc;
    if (!batch->n_rows || !batch->n_seqs) return L2_OK;
    const dim3 grid = copy_grid(batch->n_rows, 2 * pages->n_kv_heads + (q ? q->heads : 0), pages->head_size, sms);
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    by_type(pages->type, pages->head_size, [&](auto t, auto hd) {
        kv_append_kernel<decltype(t)::value, decltype(hd)::value><<<grid, KV_THREADS, 0, st>>>(P);
        return 0;
    });
    g_launches++;
    L2_CUDA(cudaGetLastError());
    return L2_OK;
}

extern "C" int l2_kv_read(const l2_kv_pages* pages, const l2_kv_batch* batch, const l2_kv_rows* k, const l2_kv_rows* v, void* cuda_stream) {
    clear_error();
    const char* who = "l2_kv_read";
    KvCopyParams P{};
    if (int rc = check_pages(who, pages, &P.pool)) return rc;
    if (int rc = check_batch(who, batch, pages->page_size, &P.step)) return rc;
    if (int rc = check_rows(who, "k", k, batch, pages->head_size, pages->n_kv_heads, &P.k)) return rc;
    if (int rc = check_rows(who, "v", v, batch, pages->head_size, pages->n_kv_heads, &P.v)) return rc;
    int sms;
    if (int rc = kv_device(&sms)) return rc;
    if (!batch->n_rows || !batch->n_seqs) return L2_OK;
    const dim3 grid = copy_grid(batch->n_rows, 2 * pages->n_kv_heads, pages->head_size, sms);
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    by_type(pages->type, pages->head_size, [&](auto t, auto hd) {
        kv_read_kernel<decltype(t)::value, decltype(hd)::value><<<grid, KV_THREADS, 0, st>>>(P);
        return 0;
    });
    g_launches++;
    L2_CUDA(cudaGetLastError());
    return L2_OK;
}

extern "C" size_t l2_kv_attend_workspace_bytes(const l2_kv_pages* pages, const l2_kv_batch* batch, int n_heads) {
    clear_error();
    const char* who = "l2_kv_attend_workspace_bytes";
    KvPool pool;
    KvStep step;
    int sms;
    if (check_pages(who, pages, &pool) || check_batch(who, batch, pages->page_size, &step) || kv_device(&sms)) return 0;
    if (n_heads < 1 || n_heads % pool.n_kv_heads) { fail(L2_EINVAL, "%s: %d heads, %d kv heads", who, n_heads, pool.n_kv_heads); return 0; }
    return kv_attend_work(step, pool, n_heads, pages->head_size, sms);
}

extern "C" int l2_kv_attend(const l2_kv_pages* pages, const l2_kv_batch* batch, const l2_kv_rows* q, const l2_kv_rows* out, float scale, int window, int sinks,
                            void* workspace, size_t workspace_bytes, void* cuda_stream) {
    clear_error();
    const char* who = "l2_kv_attend";
    KvAttendParams P{};
    if (int rc = check_pages(who, pages, &P.pool)) return rc;
    if (int rc = check_batch(who, batch, pages->page_size, &P.step)) return rc;
    if (!q || q->heads < 1 || q->heads % pages->n_kv_heads || q->heads / pages->n_kv_heads > 64)
        return fail(L2_EINVAL, "%s: the heads of q must be 1 to 64 times the kv heads", who);
    if (int rc = check_rows(who, "q", q, batch, pages->head_size, q->heads, &P.q)) return rc;
    if (int rc = check_rows(who, "out", out, batch, pages->head_size, q->heads, &P.out)) return rc;
    if (q->type == L2_F32 || (pages->type != L2_I8 && q->type != pages->type)) return fail(L2_EINVAL, "%s: q must be of the cache's type (f16 or bf16 with an int8 cache)", who);
    if (out->type != L2_F32 && out->type != q->type) return fail(L2_EINVAL, "%s: out must be of q's type or f32", who);
    if (window < 0 || sinks < 0 || !(scale > 0.0f) || !(scale < 1e30f)) return fail(L2_EINVAL, "%s: window %d, sinks %d, scale %g", who, window, sinks, scale);
    int sms;
    if (int rc = kv_device(&sms)) return rc;
    const size_t need = kv_attend_work(P.step, P.pool, q->heads, pages->head_size, sms);
    if (workspace_bytes < need || (need && (!workspace || !aligned16(workspace)))) return fail(L2_EINVAL, "%s: a workspace of %zu bytes on a 16-byte boundary needed", who, need);
    if (!batch->n_rows || !batch->n_seqs) return L2_OK;
    P.scale_log2 = scale * 1.4426950408889634f;
    P.window = window; P.sinks = window ? sinks : 0;
    P.group = q->heads / pages->n_kv_heads;
    P.group_inv = (65536 + P.group - 1) / P.group;
    P.work = workspace;
    L2_CUDA(launch_kv_attend(P, pages->type, pages->head_size, sms, static_cast<cudaStream_t>(cuda_stream)));
    return L2_OK;
}
