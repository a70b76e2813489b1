// Host side of l2_kv_attend's kernels.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "kernels.cuh"
#include "paged.cuh"

namespace l2 {

// Sets a kernel's opt-in shared memory once per device (a static of the launch).
struct KvOnce {
    std::atomic<uint64_t> done{0};
    cudaError_t shared_memory(const void* kernel, int bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess || (done.load(std::memory_order_acquire) >> dev & 1)) return e;
        if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) == cudaSuccess) done.fetch_or(1ull << dev, std::memory_order_release);
        return e;
    }
};

// Launched programmatically: a kernel's launch overlaps the one in front of it, for whose end it waits before it reads anything.
template <class... A>
cudaError_t kv_launch(void (*kernel)(A...), dim3 grid, int threads, size_t smem, cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    g_launches++;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The pool as a TMA tensor (element, position in the page, kv head, page); a copy brings up to `tile` positions of one page and head, 128 bytes wide (or a
// row, where that is less), swizzled accordingly.
cudaError_t kv_map(CUtensorMap* map, const KvPool& p, const void* base, int type, int head_size, int tile);

// Sequences with at most this many rows (tokens x query heads per kv head) are taken by the kernel for few rows, the others by the tcgen05 kernel: all of a
// batch whose largest sequence is that small, the single tokens of another; 0: none (there is room for as many rows as the largest sequence has for
// every one: a batch of one kind, which one kernel takes whole).
int kv_rows_limit(const KvStep& s, int group);
size_t kv_rows_work(const KvStep& s, const KvPool& p, int group, int type, int head_size, int sms);
cudaError_t launch_kv_rows(const KvAttendParams& p, int type, int head_size, int sms, cudaStream_t st);

// The others: tcgen05.
size_t kv_tc_work(const KvStep& s, const KvPool& p, int group, int head_size, int sms);
cudaError_t launch_kv_tc(const KvAttendParams& p, int type, int head_size, int sms, cudaStream_t st);

}  // namespace l2
