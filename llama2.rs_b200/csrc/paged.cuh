// Paged KV cache: parameter records and device helpers shared by paged.cu and the attention kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/llama2_b200.h"

namespace l2 {

struct KvPool {  // l2_kv_pages as the kernels take it
    char* k; char* v;
    float* ks; float* vs;
    int64_t page_stride, pos_stride, head_stride;  // elements
    int n_pages, page_shift, n_kv_heads;
};
struct KvStep {  // l2_kv_batch
    const int* table; const int* kv_len; const int* row_start;
    int* status;
    int n_seqs, width, n_rows, max_rows;
};
struct KvRows {
    char* data;
    int64_t row_stride, head_stride;
    int type, heads;
};

struct KvAttendParams {
    KvPool pool;
    KvStep step;
    KvRows q, out;
    float scale_log2;   // scale * log2(e): scores in powers of two
    int window, sinks;  // window 0: all
    int group;          // query heads per kv head
    int group_inv;      // 2^16 / group, rounded up
    void* work;
};

// One sequence of a step, with what is out of range put right (and reported once, by the caller's choice).
struct KvSeq { int row0, n, kv; };

#ifdef __CUDACC__
// (The kernels are launched programmatically: lengths and tables may be written by the kernel in front, for whose end they wait, so nothing here is read through
// the read-only path.)
__device__ __forceinline__ void kv_report(int* status, int bit) { if (status) atomicOr(status, bit); }

__device__ __forceinline__ KvSeq kv_seq(const KvStep& s, int page_shift, int b) {
    KvSeq q;
    q.row0 = s.row_start[b];
    const int64_t n = (int64_t)s.row_start[b + 1] - q.row0;
    q.n = (int)n;
    if (q.row0 < 0 || n < 0 || n > s.max_rows || q.row0 + n > s.n_rows) { kv_report(s.status, L2_KV_BAD_ROWS); q.row0 = 0; q.n = 0; }
    q.kv = s.kv_len[b];
    const int64_t most = (int64_t)s.width << page_shift;
    if (q.kv < 0 || q.kv > most) { kv_report(s.status, L2_KV_BAD_LENGTH); q.kv = q.kv < 0 ? 0 : (int)most; }
    return q;
}

// The page of position j of sequence b, or -1 where the table's entry is none.
__device__ __forceinline__ int kv_page(const KvStep& s, const KvPool& p, int b, int j) {
    const int page = s.table[(size_t)b * s.width + (j >> p.page_shift)];
    if ((unsigned)page >= (unsigned)p.n_pages) { kv_report(s.status, L2_KV_BAD_PAGE); return -1; }
    return page;
}

// The sequence that row r belongs to, by the whole warp: the last b with row_start[b] <= r (the caller checks r against kv_seq(b)).
__device__ __forceinline__ int kv_find_seq(const KvStep& s, int r) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = s.n_seqs;  // the answer is in lo .. lo + n - 1
    while (n > 1) {
        const int step = (n + 31) / 32, at = lo + lane * step;
        const unsigned below = __ballot_sync(0xffffffffu, lane * step < n && s.row_start[at] <= r);
        const int k = below ? 31 - __clz(below) : 0;
        n = min(step, n - k * step);
        lo += k * step;
    }
    return lo;
}

// 8 f32 stored as a type
__device__ __forceinline__ void kv_store8(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void kv_store8(__half* p, const float (&x)[8]) {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
}
__device__ __forceinline__ void kv_store8(__nv_bfloat16* p, const float (&x)[8]) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
}
#endif

cudaError_t launch_kv_attend(const KvAttendParams& p, int type, int head_size, int sms, cudaStream_t st);
size_t kv_attend_work(const KvStep& s, const KvPool& p, int n_heads, int type, int head_size, int sms);

}  // namespace l2
