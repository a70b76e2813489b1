// Tables of a step on the device: l2_kv_plan (rows, pages from the free list, lengths, slots) and l2_kv_release, which takes back what it gave.
//
//   plan:    n_b rows more for sequence b:  row_start = exclusive sum of n,  pages_b = ceil((len_b + n_b) / page) - ceil(len_b / page),
//            page i of all of them (sequence by sequence, in the order of their positions) = free[count - 1 - i],  slot = page * page_size + offset
//   release: positions from keep_b on, and those that a window has left behind, go: page i of all of them to free[count + total - 1 - i],
//            so that a release of what a plan has added leaves lists and tables as they were
//
// A few kilobytes and a chain of dependent loads: nothing but latency.  So one launch of one cluster, and work shared out by rows and by entries, not by sequences (long prompts
// often stand side by side: with a warp for a sequence's pages, 24 of them among 500, 42,000 rows, took 79 us for a plan and a release; now 15, and 8.5 for 256 sequences with a row each).  Every CTA sums up all sequences by itself, in shared memory, which costs less than
// asking the others; they meet once, before the first writes what another may still read.  Nothing goes through atomics, and the order of pages does not depend on who was first.
// A release with a window looks at every entry between the sinks and the window, those given back before too: 8 sequences of 5,000 positions in pages of 16 take 4.8 us, of 60,000 123.
#include <cuda_runtime.h>

#include <algorithm>

#include "host_common.h"
#include "kernels.cuh"
#include "model.h"
#include "paged_attend.h"

namespace l2 {

namespace {

constexpr int TB_CLUSTER = 8, TB_MOST = 1024, TB_WARPS = TB_MOST / 32;  // CTAs and threads at most
constexpr int TB_SEQS = 16384;  // whose sums a CTA's shared memory holds

struct TbParams {
    int* table; int* kv_len; int* free_pages; int* free_count; int* status;
    int n_seqs, width, n_pages, page_shift;
    const int* counts;  // plan: new rows; release: lengths to keep, or NULL
    int* row_start; long long* slots; int* positions;
    int n_rows, max_rows;
    int window, sinks;
};

__device__ __forceinline__ void tb_sync(int ctas) {  // of the cluster
    if (ctas == 1) { __syncthreads(); return; }
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ long long tb_remote(const long long* p, int cta) {
    uint32_t at;
    long long v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(cta));
    asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ long long tb_scan(long long v) {  // inclusive, over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += u;
    }
    return v;
}

// Exclusive sums of N numbers a thread over the CTA, and their totals.
template <int N>
__device__ __forceinline__ void tb_sums(const long long (&v)[N], long long (&before)[N], long long (&total)[N], long long (*scratch)[N]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();  // (scratch is free)
#pragma unroll
    for (int i = 0; i < N; i++) {
        const long long s = tb_scan(v[i]);
        before[i] = s - v[i];
        if (lane == 31) scratch[warp][i] = s;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        const long long s = tb_scan(lane < (int)(blockDim.x >> 5) ? scratch[lane][i] : 0);
        total[i] = __shfl_sync(0xffffffffu, s, 31);
        const long long w = __shfl_sync(0xffffffffu, s, warp ? warp - 1 : 0);
        if (warp) before[i] += w;
    }
}

// The number of free pages, put right (and reported) where it cannot be one.
__device__ __forceinline__ int tb_free(const TbParams& P, bool report) {
    const int n = *P.free_count;
    if (n >= 0 && n <= P.n_pages) return n;
    if (report) kv_report(P.status, L2_KV_BAD_PAGE);
    return n < 0 ? 0 : P.n_pages;
}
__device__ __forceinline__ int tb_pages(const TbParams& P, long long positions) { return (int)((positions + (1 << P.page_shift) - 1) >> P.page_shift); }
__device__ __forceinline__ bool tb_is_page(const TbParams& P, int e) { return (unsigned)e < (unsigned)P.n_pages; }
// The last of n ascending numbers that is not above x (the first is not).
__device__ __forceinline__ int tb_find(const int* a, int n, int x) {
    int lo = 0;
    for (int hi = n; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(TB_MOST) kv_plan_kernel(const __grid_constant__ TbParams P) {
    extern __shared__ int tb_smem[];
    int* const starts = tb_smem;                      // [n_seqs + 1] first rows
    int* const taken = tb_smem + P.n_seqs + 1;        // [n_seqs + 1] pages taken in front of a sequence
    int* const lengths = tb_smem + 2 * P.n_seqs + 2;  // [n_seqs] before the step
    __shared__ long long scratch[TB_WARPS][2];
    const int tid = threadIdx.x, threads = blockDim.x, cta = blockIdx.x, ctas = gridDim.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int count = tb_free(P, cta == 0 && tid == 0);
    // ---- rows and pages of all sequences.  (Sums that pass 31 bits are of steps without room, whose sums nobody uses.)
    long long all[2] = {0, 0};
    for (int b0 = 0; b0 < P.n_seqs; b0 += threads) {
        const int b = b0 + tid;
        long long v[2] = {0, 0}, before[2], total[2];
        if (b < P.n_seqs) {
            const int len = P.kv_len[b];
            int n = P.counts[b], wrong = 0;
            if (n < 0 || n > P.max_rows) { wrong = L2_KV_BAD_ROWS; n = 0; }
            if (len < 0 || (long long)len + n > (long long)P.width << P.page_shift) { wrong |= L2_KV_BAD_LENGTH; n = 0; }
            if (wrong && cta == 0) kv_report(P.status, wrong);
            v[0] = n;
            if (n) v[1] = tb_pages(P, (long long)len + n) - tb_pages(P, len);
            lengths[b] = len;
        }
        tb_sums<2>(v, before, total, scratch);
        if (b < P.n_seqs) { starts[b] = (int)(all[0] + before[0]); taken[b] = (int)(all[1] + before[1]); }
        all[0] += total[0];
        all[1] += total[1];
    }
    const bool room = all[0] <= P.n_rows && all[1] <= count;
    const int rows = room ? (int)all[0] : 0, pages = room ? (int)all[1] : 0;
    if (tid == 0) { starts[P.n_seqs] = rows; taken[P.n_seqs] = pages; }
    tb_sync(ctas);  // all have read the lengths and the number of free pages
    if (cta == 0 && tid == 0) {
        if (!room) kv_report(P.status, L2_KV_NO_ROOM);  // nothing changes, and no sequence brings rows
        else *P.free_count = count - pages;
        P.row_start[P.n_seqs] = rows;
    }
    for (int b = cta * threads + tid; b < P.n_seqs; b += ctas * threads) {
        P.row_start[b] = room ? starts[b] : 0;
        const int n = room ? starts[b + 1] - starts[b] : 0;
        if (n) P.kv_len[b] = lengths[b] + n;
    }
    // page i of the step: of the free list, from its end
    auto page = [&](int i) {
        const int e = P.free_pages[count - 1 - i];
        if (tb_is_page(P, e)) return e;
        kv_report(P.status, L2_KV_BAD_PAGE);
        return -1;
    };
    if (!P.slots && !P.positions) {
        for (int i = cta * threads + tid; i < pages; i += ctas * threads) {
            const int b = tb_find(taken, P.n_seqs, i);  // (the last sequence with so many in front: the one that takes it)
            P.table[(size_t)b * P.width + tb_pages(P, lengths[b]) + i - taken[b]] = page(i);
        }
        return;
    }
    // ---- a slot and a position for every row, a few rows a thread; the first row of a new page brings it into the table
    const int mask = (1 << P.page_shift) - 1;
    constexpr int N = 4;
    const bool wide = ((reinterpret_cast<uintptr_t>(P.slots) | reinterpret_cast<uintptr_t>(P.positions)) & 15) == 0;
    for (int r0 = N * (cta * threads + tid); r0 < P.n_rows; r0 += N * ctas * threads) {
        long long slot[N];
        int pos[N];
        int b = r0 < rows ? tb_find(starts, P.n_seqs, r0) : 0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int r = r0 + i;
            slot[i] = pos[i] = -1;
            if (r >= rows) continue;
            while (r >= starts[b + 1]) b++;
            const int len = lengths[b], have = tb_pages(P, len);
            pos[i] = len + r - starts[b];
            const int at = pos[i] >> P.page_shift;
            int* const entry = P.table + (size_t)b * P.width + at;
            int e;
            if (at >= have) {
                e = page(taken[b] + at - have);
                if ((pos[i] & mask) == 0) *entry = e;
            } else {
                e = *entry;
                if (!tb_is_page(P, e)) { kv_report(P.status, L2_KV_BAD_PAGE); e = -1; }
            }
            if (e >= 0) slot[i] = ((long long)e << P.page_shift) + (pos[i] & mask);
        }
        if (wide && r0 + N <= P.n_rows) {  // (every array that there is starts on a boundary of 16 bytes)
            if (P.slots) {
                reinterpret_cast<longlong2*>(P.slots + r0)[0] = make_longlong2(slot[0], slot[1]);
                reinterpret_cast<longlong2*>(P.slots + r0)[1] = make_longlong2(slot[2], slot[3]);
            }
            if (P.positions) *reinterpret_cast<int4*>(P.positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
            continue;
        }
#pragma unroll
        for (int i = 0; i < N; i++)
            if (r0 + i < P.n_rows) {
                if (P.slots) P.slots[r0 + i] = slot[i];
                if (P.positions) P.positions[r0 + i] = pos[i];
            }
    }
}

// Entries of a sequence that go, behind the window and from the length to keep on: first[0] .. first[0] + n[0] - 1, then first[1] .. first[1] + n[1] - 1.
struct TbGone { int first[2], n[2]; };
__device__ __forceinline__ TbGone tb_gone(const TbParams& P, int len, int keep) {
    TbGone g;
    g.first[1] = tb_pages(P, keep);
    g.n[1] = tb_pages(P, len) - g.first[1];
    g.first[0] = g.n[0] = 0;
    if (P.window) {  // the next row, at position keep, sees none from keep - window on back, but for the sinks
        g.first[0] = (int)min((long long)g.first[1], ((long long)P.sinks + (1 << P.page_shift) - 1) >> P.page_shift);
        g.n[0] = max(0, (max(0, keep - P.window + 1) >> P.page_shift) - g.first[0]);
    }
    return g;
}

__global__ void __launch_bounds__(TB_MOST) kv_release_kernel(const __grid_constant__ TbParams P) {
    extern __shared__ int tb_smem[];
    int* const from = tb_smem;                     // [n_seqs] entries in front of a sequence's
    int* const lengths = tb_smem + P.n_seqs;       // [n_seqs]
    int* const kept = tb_smem + 2 * P.n_seqs;      // [n_seqs]
    __shared__ long long scratch[TB_WARPS][1], mine;
    const int tid = threadIdx.x, threads = blockDim.x, cta = blockIdx.x, ctas = gridDim.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int count = tb_free(P, cta == 0 && tid == 0);
    long long entries = 0;
    for (int b0 = 0; b0 < P.n_seqs; b0 += threads) {
        const int b = b0 + tid;
        long long v[1] = {0}, before[1], total[1];
        if (b < P.n_seqs) {
            int len = P.kv_len[b], keep = P.counts ? P.counts[b] : len;
            if (len < 0 || len > (long long)P.width << P.page_shift || keep < 0) {  // left as it is
                if (cta == 0) kv_report(P.status, L2_KV_BAD_LENGTH);
                lengths[b] = kept[b] = -1;
            } else {
                lengths[b] = len;
                kept[b] = min(len, keep);
                const TbGone g = tb_gone(P, len, kept[b]);
                v[0] = g.n[0] + g.n[1];
            }
        }
        tb_sums<1>(v, before, total, scratch);
        if (b < P.n_seqs) from[b] = (int)(entries + before[0]);
        entries += total[0];
    }
    __syncthreads();
    // ---- a run of the entries for each CTA.  The pages among them are counted, then put on the list below those of the entries in front
    const int per = (int)((entries + ctas - 1) / ctas), e0 = (int)min(entries, (long long)cta * per), e1 = (int)min(entries, (long long)e0 + per);
    auto find = [&](int i) {  // entry i of all, in the tables
        const int b = tb_find(from, P.n_seqs, i);
        const TbGone g = tb_gone(P, lengths[b], kept[b]);
        const int k = i - from[b];
        return P.table + (size_t)b * P.width + (k < g.n[0] ? g.first[0] + k : g.first[1] + k - g.n[0]);
    };
    int* at = nullptr;
    int e = -1;
    long long v[1] = {0}, before[1], total[1];
    for (int i0 = e0; i0 < e1; i0 += threads) {
        at = nullptr;
        e = -1;
        if (i0 + tid < e1) {
            at = find(i0 + tid);
            e = *at;
            if (tb_is_page(P, e)) v[0]++;
            else if (e != -1) kv_report(P.status, L2_KV_BAD_PAGE);
        }
    }
    const bool once = e1 - e0 <= threads;  // (at and e are then what they will be below)
    tb_sums<1>(v, before, total, scratch);
    if (tid == 0) mine = total[0];
    tb_sync(ctas);  // (also: all have read the lengths and the number of free pages)
    long long others = 0;
    if ((tid & 31) < ctas) others = ctas == 1 ? mine : tb_remote(&mine, tid & 31);
    const long long inc = tb_scan(others), all = __shfl_sync(0xffffffffu, inc, ctas - 1);
    long long front = __shfl_sync(0xffffffffu, inc - others, cta);
    if (cta == 0 && tid == 0) {
        if (all > P.n_pages - count) kv_report(P.status, L2_KV_BAD_PAGE);  // (more pages than there are: some were in two tables)
        *P.free_count = (int)min((long long)P.n_pages, count + all);
    }
    for (int i0 = e0; i0 < e1; i0 += threads) {
        if (!once) {
            at = nullptr;
            e = -1;
            if (i0 + tid < e1) { at = find(i0 + tid); e = *at; }
            v[0] = tb_is_page(P, e);
            tb_sums<1>(v, before, total, scratch);
        }
        if (at && tb_is_page(P, e)) {
            const long long to = count + all - 1 - (front + before[0]);
            if (to >= 0 && to < P.n_pages) P.free_pages[to] = e;
            *at = -1;
        }
        front += total[0];
    }
    for (int b = cta * threads + tid; b < P.n_seqs; b += ctas * threads)
        if (kept[b] < lengths[b]) P.kv_len[b] = kept[b];
    tb_sync(ctas);  // (nobody reads this CTA's shared memory any more)
}

int check_tables(const char* who, const l2_kv_tables* t, TbParams* out) {
    if (!t) return fail(L2_EINVAL, "%s: no tables", who);
    int shift = 3;
    while (shift < 8 && (1 << shift) < t->page_size) shift++;
    if ((1 << shift) != t->page_size) return fail(L2_EINVAL, "%s: page size %d (8, 16, 32, 64, 128 or 256)", who, t->page_size);
    if (t->n_seqs < 0 || t->n_seqs > TB_SEQS || t->table_width < 0 || t->n_pages < 1) return fail(L2_EINVAL, "%s: %d sequences (at most %d), tables of %d, %d pages", who, t->n_seqs, TB_SEQS, t->table_width, t->n_pages);
    if ((int64_t)t->table_width * t->page_size > (1 << 30) || (int64_t)t->n_seqs * t->table_width > (1 << 30)) return fail(L2_ERANGE, "%s: more than 2^30 positions, or entries of tables", who);
    if (!t->free_pages || !t->free_count || (t->n_seqs && (!t->kv_len || (t->table_width && !t->page_table)))) return fail(L2_EINVAL, "%s: null device pointer", who);
    const void* words[] = {t->page_table, t->kv_len, t->free_pages, t->free_count, t->status};
    for (const void* p : words)
        if (reinterpret_cast<uintptr_t>(p) & 3) return fail(L2_EINVAL, "%s: an array that does not start on a 4-byte boundary", who);
    out->table = t->page_table; out->kv_len = t->kv_len; out->free_pages = t->free_pages; out->free_count = t->free_count; out->status = t->status;
    out->n_seqs = t->n_seqs; out->width = t->table_width; out->n_pages = t->n_pages; out->page_shift = shift;
    return L2_OK;
}

// One cluster for so many rows or entries, launched programmatically.
cudaError_t tb_launch(void (*kernel)(const TbParams), const TbParams& P, int64_t items, KvOnce& once, cudaStream_t st) {
    // (few rows: fewer warps to meet; else as many as there are, two rows or so a thread)
    const int threads = items <= 1024 && P.n_seqs <= 512 ? 256 : TB_MOST;
    const int64_t ctas = (items + 2 * threads - 1) / (2 * threads);
    const int smem = (3 * P.n_seqs + 2) * (int)sizeof(int);
    if (smem > 40 * 1024)
        if (cudaError_t e = once.shared_memory(reinterpret_cast<const void*>(kernel), (3 * TB_SEQS + 2) * (int)sizeof(int))) return e;
    int n = 1;
    while (n < TB_CLUSTER && n < ctas) n *= 2;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3(n);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = n; attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = n > 1 ? 2 : 1;
    g_launches++;
    return cudaLaunchKernelEx(&cfg, kernel, P);
}

}  // namespace

}  // namespace l2

using namespace l2;

extern "C" int l2_kv_plan(const l2_kv_tables* tables, const int32_t* new_rows, int32_t* row_start, int64_t* slots, int32_t* positions, int n_rows, int max_rows, void* cuda_stream) {
    clear_error();
    const char* who = "l2_kv_plan";
    TbParams P{};
    if (int rc = check_tables(who, tables, &P)) return rc;
    if (n_rows < 0 || max_rows < 0 || n_rows > (1 << 30)) return fail(L2_EINVAL, "%s: %d rows, at most %d of a sequence", who, n_rows, max_rows);
    if ((P.n_seqs && !new_rows) || !row_start) return fail(L2_EINVAL, "%s: null device pointer", who);
    if ((reinterpret_cast<uintptr_t>(new_rows) & 3) || (reinterpret_cast<uintptr_t>(row_start) & 3) || (reinterpret_cast<uintptr_t>(positions) & 3) || (reinterpret_cast<uintptr_t>(slots) & 7))
        return fail(L2_EINVAL, "%s: an array that does not start on a boundary of its elements", who);
    P.counts = new_rows; P.row_start = row_start; P.slots = reinterpret_cast<long long*>(slots); P.positions = positions; P.n_rows = n_rows; P.max_rows = max_rows;
    int sms;
    if (int rc = kv_device(&sms)) return rc;
    static KvOnce once;
    L2_CUDA(tb_launch(kv_plan_kernel, P, n_rows, once, static_cast<cudaStream_t>(cuda_stream)));
    return L2_OK;
}

extern "C" int l2_kv_release(const l2_kv_tables* tables, const int32_t* keep, int window, int sinks, void* cuda_stream) {
    clear_error();
    const char* who = "l2_kv_release";
    TbParams P{};
    if (int rc = check_tables(who, tables, &P)) return rc;
    if (window < 0 || sinks < 0) return fail(L2_EINVAL, "%s: window %d, sinks %d", who, window, sinks);
    if (reinterpret_cast<uintptr_t>(keep) & 3) return fail(L2_EINVAL, "%s: an array that does not start on a 4-byte boundary", who);
    P.counts = keep; P.window = window; P.sinks = sinks;
    int sms;
    if (int rc = kv_device(&sms)) return rc;
    if (!P.n_seqs) return L2_OK;
    static KvOnce once;
    L2_CUDA(tb_launch(kv_release_kernel, P, std::min<int64_t>((int64_t)P.n_seqs * P.width, 16 * (int64_t)P.n_seqs), once, static_cast<cudaStream_t>(cuda_stream)));
    return L2_OK;
}
