// Tables of a step on the device: l2_kv_plan (rows, pages from the free list, lengths, slots) and l2_kv_release, which takes back what it gave.
//
//   plan:    n_b rows more for sequence b:  row_start = exclusive sum of n,  pages_b = ceil((len_b + n_b) / page) - ceil(len_b / page),
//            page i of all of them (sequence by sequence, in the order of their positions) = free[count - 1 - i],  slot = page * page_size + offset
//   release: positions from keep_b on, and those that a window has left behind, go: page i of all of them to free[count + total - 1 - i],
//            so that a release of what a plan has added leaves lists and tables as they were
//
// A few kilobytes and a chain of dependent loads: nothing but latency.  So one launch of one cluster: a CTA has a run of sequences, a thread a sequence (pages of one that has many: the
// lanes of its warp), and the sums in front of a CTA's run come from the others' shared memory.  Nothing goes through atomics, and the order of pages does not depend on who was first.
#include <cuda_runtime.h>

#include <algorithm>

#include "host_common.h"
#include "kernels.cuh"
#include "model.h"
#include "paged_attend.h"

namespace l2 {

namespace {

constexpr int TB_THREADS = 512, TB_WARPS = TB_THREADS / 32, TB_CLUSTER = 8;
constexpr int TB_STARTS = 8192;  // first rows that a CTA keeps in shared memory
constexpr int TB_ALONE = 4;      // pages that a lane takes by itself

struct TbParams {
    int* table; int* kv_len; int* free_pages; int* free_count; int* status;
    int n_seqs, width, n_pages, page_shift;
    const int* counts;  // plan: new rows; release: lengths to keep, or NULL
    int* row_start; long long* slots; int* positions;
    int n_rows, max_rows;
    int window, sinks;
    int per;            // sequences of a CTA
};

__device__ __forceinline__ void tb_sync(int ctas) {  // of the cluster, what was written to memory included
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
        const long long s = tb_scan(lane < TB_WARPS ? scratch[lane][i] : 0);
        total[i] = __shfl_sync(0xffffffffu, s, TB_WARPS - 1);
        const long long w = __shfl_sync(0xffffffffu, s, warp ? warp - 1 : 0);
        if (warp) before[i] += w;
    }
}

// What the CTAs in front of this one have, and all of them: mine is this CTA's totals, in shared memory.
template <int N>
__device__ __forceinline__ void tb_cluster(const long long (*mine)[N], int cta, int ctas, long long (&before)[N], long long (&total)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int lane = threadIdx.x & 31;
        long long s = 0;
        if (lane < ctas) s = ctas == 1 ? (*mine)[i] : tb_remote(&(*mine)[i], lane);
        const long long inc = tb_scan(s);
        total[i] = __shfl_sync(0xffffffffu, inc, ctas - 1);
        before[i] = __shfl_sync(0xffffffffu, inc - s, cta);
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

struct TbPlan { int len, n, have, need; };  // positions, new rows; pages before and after
__device__ __forceinline__ TbPlan tb_plan(const TbParams& P, int b, bool report) {
    TbPlan s{P.kv_len[b], P.counts[b], 0, 0};
    const long long most = (long long)P.width << P.page_shift;
    int wrong = 0;
    if (s.n < 0 || s.n > P.max_rows) { wrong = L2_KV_BAD_ROWS; s.n = 0; }
    if (s.len < 0 || (long long)s.len + s.n > most) { wrong |= L2_KV_BAD_LENGTH; s.n = 0; }
    if (wrong && report) kv_report(P.status, wrong);
    if (s.n) { s.have = tb_pages(P, s.len); s.need = tb_pages(P, (long long)s.len + s.n); }
    return s;
}

__global__ void __launch_bounds__(TB_THREADS) kv_plan_kernel(const __grid_constant__ TbParams P) {
    __shared__ long long scratch[TB_WARPS][2], mine[1][2];
    __shared__ int starts[TB_STARTS + 1];
    const int tid = threadIdx.x, lane = tid & 31, cta = blockIdx.x, ctas = gridDim.x;
    const int b0 = min((long long)P.n_seqs, (long long)cta * P.per), b1 = min((long long)P.n_seqs, (long long)b0 + P.per);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int count = tb_free(P, cta == 0 && tid == 0);
    // ---- rows and pages of this CTA's sequences; the first of a thread stays in registers
    TbPlan first{0, 0, 0, 0};
    long long sum[2] = {0, 0}, before[2], total[2];
    for (int b = b0 + tid; b < b1; b += TB_THREADS) {
        const TbPlan s = tb_plan(P, b, true);
        if (b == b0 + tid) first = s;
        sum[0] += s.n;
        sum[1] += s.need - s.have;
    }
    tb_sums<2>(sum, before, total, scratch);
    if (tid == 0) { mine[0][0] = total[0]; mine[0][1] = total[1]; }
    tb_sync(ctas);
    long long front[2], all[2];
    tb_cluster<2>(mine, cta, ctas, front, all);
    const bool room = all[0] <= P.n_rows && all[1] <= count;
    if (!room) {  // nothing changes, and no sequence brings rows
        if (cta == 0 && tid == 0) kv_report(P.status, L2_KV_NO_ROOM);
        for (int b = b0 + tid; b < b1; b += TB_THREADS) P.row_start[b] = 0;
        if (cta == 0 && tid == 0) P.row_start[P.n_seqs] = 0;
        all[0] = 0;
    } else {
        if (cta == 0 && tid == 0) { *P.free_count = count - (int)all[1]; P.row_start[P.n_seqs] = (int)all[0]; }
        const bool once = b1 - b0 <= TB_THREADS;
        for (int c0 = b0; c0 < b1; c0 += TB_THREADS) {
            const int b = c0 + tid;
            TbPlan s = first;
            if (c0 != b0) s = b < b1 ? tb_plan(P, b, false) : TbPlan{0, 0, 0, 0};
            long long at[2] = {before[0], before[1]};
            if (!once) {
                const long long v[2] = {s.n, s.need - s.have};
                long long t[2];
                tb_sums<2>(v, at, t, scratch);
                at[0] += front[0]; at[1] += front[1];
                front[0] += t[0]; front[1] += t[1];
            } else {
                at[0] += front[0]; at[1] += front[1];
            }
            if (b < b1) {
                P.row_start[b] = (int)at[0];
                if (s.n) P.kv_len[b] = s.len + s.n;
            }
            // pages: of the free list from its end
            auto take = [&](int seq, int have, int from, int i) {
                int page = P.free_pages[count - 1 - (from + i)];
                if ((unsigned)page >= (unsigned)P.n_pages) { kv_report(P.status, L2_KV_BAD_PAGE); page = -1; }
                P.table[(size_t)seq * P.width + have + i] = page;
            };
            const int n = s.need - s.have, from = (int)at[1];
            if (n <= TB_ALONE)
                for (int i = 0; i < n; i++) take(b, s.have, from, i);
            for (unsigned many = __ballot_sync(0xffffffffu, n > TB_ALONE); many; many &= many - 1) {
                const int src = __ffs(many) - 1;
                const int m = __shfl_sync(0xffffffffu, n, src), f = __shfl_sync(0xffffffffu, from, src), h = __shfl_sync(0xffffffffu, s.have, src);
                for (int i = lane; i < m; i += 32) take(b - lane + src, h, f, i);
            }
        }
    }
    tb_sync(ctas);  // (also: nobody reads this CTA's shared memory any more)
    if (!P.slots && !P.positions) return;
    // ---- a slot and a position for every row, four rows a thread
    // (What other CTAs have written is read past the L1.)
    const bool near = P.n_seqs <= TB_STARTS;
    if (near) {
        for (int b = tid; b <= P.n_seqs; b += TB_THREADS) starts[b] = __ldcg(P.row_start + b);
        __syncthreads();
    }
    auto start = [&](int b) { return near ? starts[b] : __ldcg(P.row_start + b); };
    const int rows = (int)all[0], mask = (1 << P.page_shift) - 1;
    for (int r0 = 4 * (cta * TB_THREADS + tid); r0 < P.n_rows; r0 += 4 * ctas * TB_THREADS) {
        int b = 0, end = 0, len = 0;
        if (r0 < rows) {  // the last sequence that begins at r0 or before
            int hi = P.n_seqs;
            while (hi - b > 1) {
                const int mid = (b + hi) >> 1;
                if (start(mid) <= r0) b = mid;
                else hi = mid;
            }
            end = start(b + 1);
            len = __ldcg(P.kv_len + b);
        }
        long long slot[4];
        int pos[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = r0 + i;
            slot[i] = pos[i] = -1;
            if (r >= rows) continue;
            while (r >= end) { b++; end = start(b + 1); if (r < end) len = __ldcg(P.kv_len + b); }
            pos[i] = len - (end - r);
            const int page = __ldcg(P.table + (size_t)b * P.width + (pos[i] >> P.page_shift));
            if ((unsigned)page < (unsigned)P.n_pages) slot[i] = ((long long)page << P.page_shift) + (pos[i] & mask);
            else kv_report(P.status, L2_KV_BAD_PAGE);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (r0 + i < P.n_rows) {
                if (P.slots) P.slots[r0 + i] = slot[i];
                if (P.positions) P.positions[r0 + i] = pos[i];
            }
    }
}

// Pages of a sequence that go: entries lo[0] .. hi[0] - 1 (behind the window) and lo[1] .. hi[1] - 1 (from the length to keep on).
struct TbRelease { int len, keep, lo[2], hi[2]; };
__device__ __forceinline__ TbRelease tb_release(const TbParams& P, int b, bool report) {
    TbRelease s{P.kv_len[b], 0, {0, 0}, {0, 0}};
    const long long most = (long long)P.width << P.page_shift;
    const int keep = P.counts ? P.counts[b] : s.len;
    s.keep = min(s.len, keep);
    if (s.len < 0 || s.len > most || keep < 0) {  // left as it is
        if (report) kv_report(P.status, L2_KV_BAD_LENGTH);
        s.keep = s.len;
        return s;
    }
    s.lo[1] = tb_pages(P, s.keep);
    s.hi[1] = tb_pages(P, s.len);
    if (P.window) {  // the next row, at position keep, sees none from keep - window on back, but for the sinks
        s.lo[0] = (int)min((long long)s.lo[1], ((long long)P.sinks + (1 << P.page_shift) - 1) >> P.page_shift);
        s.hi[0] = max(s.lo[0], max(0, s.keep - P.window + 1) >> P.page_shift);
    }
    return s;
}

__global__ void __launch_bounds__(TB_THREADS) kv_release_kernel(const __grid_constant__ TbParams P) {
    __shared__ long long scratch[TB_WARPS][1], mine[1][1];
    const int tid = threadIdx.x, lane = tid & 31, cta = blockIdx.x, ctas = gridDim.x;
    const int b0 = min((long long)P.n_seqs, (long long)cta * P.per), b1 = min((long long)P.n_seqs, (long long)b0 + P.per);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int count = tb_free(P, cta == 0 && tid == 0);
    // f(entry, its place in the free list) for the pages of the lanes' sequences that go, from `place` down; how many they are
    auto walk = [&](const TbRelease& s, int b, bool report, long long place, auto f) {
        int pages = 0;
        auto look = [&](int seq, int i) {
            const int e = P.table[(size_t)seq * P.width + i];
            const bool is = (unsigned)e < (unsigned)P.n_pages;
            if (!is && e != -1 && report) kv_report(P.status, L2_KV_BAD_PAGE);
            return is;
        };
        const int n = s.hi[0] - s.lo[0] + s.hi[1] - s.lo[1];
        if (n <= 2 * TB_ALONE) {
            for (int k = 0; k < n; k++) {
                const int i = k < s.hi[0] - s.lo[0] ? s.lo[0] + k : s.lo[1] + k - (s.hi[0] - s.lo[0]);
                if (look(b, i)) f((size_t)b * P.width + i, place - pages++);
            }
        }
        for (unsigned many = __ballot_sync(0xffffffffu, n > 2 * TB_ALONE); many; many &= many - 1) {
            const int src = __ffs(many) - 1;
            int at = 0;
            const long long top = __shfl_sync(0xffffffffu, place, src);
#pragma unroll
            for (int part = 0; part < 2; part++) {
                const int lo = __shfl_sync(0xffffffffu, s.lo[part], src), hi = __shfl_sync(0xffffffffu, s.hi[part], src);
                for (int i0 = lo; i0 < hi; i0 += 32) {
                    const bool is = i0 + lane < hi && look(b - lane + src, i0 + lane);
                    const unsigned votes = __ballot_sync(0xffffffffu, is);
                    if (is) f((size_t)(b - lane + src) * P.width + i0 + lane, top - at - __popc(votes & ((1u << lane) - 1)));
                    at += __popc(votes);
                }
            }
            if (lane == src) pages = at;
        }
        return pages;
    };
    auto nothing = [](size_t, long long) {};
    TbRelease first{0, 0, {0, 0}, {0, 0}};
    int first_pages = 0;
    long long sum[1] = {0}, before[1], total[1];
    for (int c0 = b0; c0 < b1; c0 += TB_THREADS) {
        const int b = c0 + tid;
        TbRelease s{0, 0, {0, 0}, {0, 0}};
        if (b < b1) s = tb_release(P, b, true);
        const int pages = walk(s, b, true, 0, nothing);
        if (c0 == b0) { first = s; first_pages = pages; }
        sum[0] += pages;
    }
    tb_sums<1>(sum, before, total, scratch);
    if (tid == 0) mine[0][0] = total[0];
    tb_sync(ctas);
    long long front[1], all[1];
    tb_cluster<1>(mine, cta, ctas, front, all);
    if (cta == 0 && tid == 0) {
        if (all[0] > P.n_pages - count) kv_report(P.status, L2_KV_BAD_PAGE);  // (more pages than there are: some were in two tables)
        *P.free_count = (int)min((long long)P.n_pages, count + all[0]);
    }
    const bool once = b1 - b0 <= TB_THREADS;
    for (int c0 = b0; c0 < b1; c0 += TB_THREADS) {
        const int b = c0 + tid;
        TbRelease s = first;
        long long at = before[0];
        if (!once) {
            int pages = first_pages;
            if (c0 != b0) {
                s = b < b1 ? tb_release(P, b, false) : TbRelease{0, 0, {0, 0}, {0, 0}};
                pages = walk(s, b, false, 0, nothing);
            }
            const long long v[1] = {pages};
            long long a[1], t[1];
            tb_sums<1>(v, a, t, scratch);
            at = a[0] + front[0];
            front[0] += t[0];
        } else {
            at += front[0];
        }
        walk(s, b, false, count + all[0] - 1 - at, [&](size_t entry, long long to) {
            if (to >= 0 && to < P.n_pages) P.free_pages[to] = P.table[entry];
            P.table[entry] = -1;
        });
        if (b < b1 && s.keep != s.len) P.kv_len[b] = s.keep;
    }
    tb_sync(ctas);  // (nobody reads this CTA's shared memory any more)
}

int check_tables(const char* who, const l2_kv_tables* t, TbParams* out) {
    if (!t) return fail(L2_EINVAL, "%s: no tables", who);
    int shift = 3;
    while (shift < 8 && (1 << shift) < t->page_size) shift++;
    if ((1 << shift) != t->page_size) return fail(L2_EINVAL, "%s: page size %d (8, 16, 32, 64, 128 or 256)", who, t->page_size);
    if (t->n_seqs < 0 || t->n_seqs > 65536 || t->table_width < 0 || t->n_pages < 1) return fail(L2_EINVAL, "%s: %d sequences (at most 65536), tables of %d, %d pages", who, t->n_seqs, t->table_width, t->n_pages);
    if ((int64_t)t->table_width * t->page_size > (1 << 30)) return fail(L2_ERANGE, "%s: more than 2^30 positions", who);
    if (!t->free_pages || !t->free_count || (t->n_seqs && (!t->kv_len || (t->table_width && !t->page_table)))) return fail(L2_EINVAL, "%s: null device pointer", who);
    const void* words[] = {t->page_table, t->kv_len, t->free_pages, t->free_count, t->status};
    for (const void* p : words)
        if (reinterpret_cast<uintptr_t>(p) & 3) return fail(L2_EINVAL, "%s: an array that does not start on a 4-byte boundary", who);
    out->table = t->page_table; out->kv_len = t->kv_len; out->free_pages = t->free_pages; out->free_count = t->free_count; out->status = t->status;
    out->n_seqs = t->n_seqs; out->width = t->table_width; out->n_pages = t->n_pages; out->page_shift = shift;
    return L2_OK;
}

// One cluster of `ctas`, launched programmatically.
cudaError_t tb_launch(void (*kernel)(const TbParams), TbParams& P, int64_t ctas, cudaStream_t st) {
    int n = 1;
    while (n < TB_CLUSTER && n < ctas) n *= 2;
    P.per = (P.n_seqs + n - 1) / n;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3(n);
    cfg.blockDim = dim3(TB_THREADS);
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
    const int64_t by_rows = slots || positions ? (n_rows + 4 * TB_THREADS - 1) / (4 * TB_THREADS) : 1;
    L2_CUDA(tb_launch(kv_plan_kernel, P, std::max<int64_t>(by_rows, (P.n_seqs + TB_THREADS - 1) / TB_THREADS), static_cast<cudaStream_t>(cuda_stream)));
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
    L2_CUDA(tb_launch(kv_release_kernel, P, (P.n_seqs + TB_THREADS - 1) / TB_THREADS, static_cast<cudaStream_t>(cuda_stream)));
    return L2_OK;
}
