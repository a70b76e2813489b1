// Device pieces shared by the kernels of l2_kv_attend: bounded mbarrier waits, TMA copies of page runs, the tiles a block of rows sees,
// and the line of tiles that a launch divides over its CTAs.
#pragma once

#include <cuda.h>

#include "paged.cuh"

namespace l2 {

// ---- mbarriers and copies ---------------------------------------------------------------------------------------------

constexpr uint32_t KV_WAIT_LIMIT = 1u << 22;

__device__ __forceinline__ uint32_t kv_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void kv_bar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(kv_smem(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void kv_bar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(kv_smem(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void kv_bar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(kv_smem(bar)) : "memory");
}
__device__ __forceinline__ bool kv_bar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(kv_smem(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// A wait that ends: after KV_WAIT_LIMIT polls, or soon after another thread has given up, it fails, and later ones return at once.
struct KvWait {
    volatile int* failed;
    bool dead = false;
    __device__ __forceinline__ void operator()(uint64_t* bar, uint32_t parity) {
        if (dead) return;
#pragma unroll 1
        for (uint32_t i = 0; i < KV_WAIT_LIMIT; i++) {
            if (kv_bar_try(bar, parity)) return;
            if ((i & 63) == 63 && *failed) break;
        }
        dead = true;
        *failed = 1;
    }
};
__device__ __forceinline__ void kv_tma4(uint32_t dst, const CUtensorMap* map, int x, int pos, int head, int page, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(pos), "r"(head), "r"(page), "r"(kv_smem(bar)) : "memory");
}
__device__ __forceinline__ void kv_bulk(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(kv_smem(bar)) : "memory");
}
__device__ __forceinline__ float kv_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---- what a block of rows sees -----------------------------------------------------------------------------------------
// Rows at positions lo_pos .. hi_pos of a sequence see positions in tiles of TS: the tiles of the sinks (first `sink_tiles`), then those from
// `first` on; `tiles` in all, at least one (rows that see nothing still have a result to write).
template <int TS>
struct KvView {
    int lo_pos, hi_pos, sink_tiles, first, tiles;
    __device__ __forceinline__ KvView() {}
    __device__ __forceinline__ KvView(int lo, int hi, int window, int sinks) : lo_pos(lo), hi_pos(hi) {
        const int end = (hi + TS) / TS;  // (hi >= -1) tiles up to the last position seen
        first = window ? max(0, lo - window + 1) / TS : 0;
        sink_tiles = (min(sinks, max(0, lo + 1)) + TS - 1) / TS;
        if (sink_tiles >= first) sink_tiles = first = 0;
        tiles = max(1, sink_tiles + end - first);
    }
    __device__ __forceinline__ int base(int t) const { return (t < sink_tiles ? t : first + t - sink_tiles) * TS; }
    // every row sees every position of the tile
    __device__ __forceinline__ bool whole(int base, int window, int sinks) const {
        return base + TS <= lo_pos + 1 && (!window || base > hi_pos - window || base + TS <= sinks);
    }
    // some row sees some position of base .. base + n - 1
    __device__ __forceinline__ bool any(int base, int n, int window, int sinks) const {
        return base <= hi_pos && (!window || base + n > lo_pos - window + 1 || base < sinks);
    }
};
__device__ __forceinline__ bool kv_sees(int pos, int j, int window, int sinks) {
    return j <= pos && (!window || pos - j < window || j < sinks);
}

}  // namespace l2
