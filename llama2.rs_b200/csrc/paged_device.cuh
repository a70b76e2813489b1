// Device pieces shared by the kernels of l2_kv_attend: bounded mbarrier waits, TMA copies of page runs, the tiles a block of rows sees,
// and the line of tiles that a launch divides over its CTAs.
#pragma once

#include <cuda.h>

#include "paged.cuh"

namespace l2 {

// ---- mbarriers and copies ---------------------------------------------------------------------------------------------

constexpr uint32_t KV_WAIT_LIMIT = 1u << 22;  // polls, each parked for up to 4 us

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
// A wait that ends: after KV_WAIT_LIMIT polls, or soon after another thread has given up; *failed is set then.
struct KvWait {
    volatile int* failed;
    __device__ __forceinline__ void operator()(uint64_t* bar, uint32_t parity) const {
        if (kv_bar_try(bar, parity)) return;
#pragma unroll 1
        for (uint32_t i = 0; !kv_bar_try(bar, parity); i++)
            if (i == KV_WAIT_LIMIT || ((i & 15) == 0 && *failed)) { *failed = 1; return; }
    }
    __device__ __forceinline__ bool over() const { return __any_sync(0xffffffffu, *failed); }  // (by whole warps)
};
__device__ __forceinline__ void kv_prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void kv_tma4(uint32_t dst, const CUtensorMap* map, int x, int pos, int head, int page, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(pos), "r"(head), "r"(page), "r"(kv_smem(bar)) : "memory");
}
// 16 bytes by a thread, zeros where there is nothing to bring; its arrival at `bar` follows when it has landed (one of those the barrier counts).
__device__ __forceinline__ void kv_copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void kv_copy16_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(kv_smem(bar)) : "memory");
}
__device__ __forceinline__ float kv_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// x 2^d for d <= 0 (d = -inf: 0), in two steps: 2^d alone may be too small for a normal number where the product is none too small
struct KvScale {
    float h;
    __device__ __forceinline__ explicit KvScale(float d) : h(kv_exp2(0.5f * d)) {}
    __device__ __forceinline__ float operator()(float x) const { return x * h * h; }
};

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

// ---- the line of tiles -----------------------------------------------------------------------------------------------------
// The tiles of all sequences one after the other; CTA c of `ctas` takes positions c * per .. of it, per = total / ctas rounded up.
struct KvSpot { int64_t per, total, start; int b; };  // its length; the sequence that a CTA's first position is in and where that begins (-1: there is none)

__device__ __forceinline__ int64_t kv_quotient(int64_t a, int64_t b) {  // of numbers that are hardly ever beyond 32 bits
    return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
__device__ __forceinline__ int64_t kv_scan(int64_t v) {  // inclusive sum over the warp
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// By a warp, for up to 32 sequences: v the tiles of the lane's sequence; src the sequence found (0 where there is none).
__device__ __forceinline__ KvSpot kv_locate_few(int64_t v, int cta, int ctas, int* src) {
    KvSpot spot{0, 0, -1, 32};
    const int64_t inc = kv_scan(v);
    spot.total = __shfl_sync(0xffffffffu, inc, 31);
    spot.per = kv_quotient(spot.total + ctas - 1, ctas);
    const int64_t at = spot.per * cta;
    *src = 0;
    if (at >= spot.total) return spot;
    spot.b = *src = __ffs(__ballot_sync(0xffffffffu, inc > at)) - 1;
    spot.start = __shfl_sync(0xffffffffu, inc - v, *src);
    return spot;
}

// By all threads of a CTA of THREADS.  len(b): tiles of sequence b, called by whole warps, 0 for b >= n.  Scratch: THREADS / 32 + 2 words of shared memory.
// Up to 32 sequences: every warp by itself (with barriers between, the search took 3100 clocks of a kernel that takes 13000 for one token of one sequence).
template <int THREADS, class Len>
__device__ __forceinline__ KvSpot kv_locate(int n, int cta, int ctas, int64_t* scratch, Len len) {
    constexpr int WARPS = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (n <= 32) {
        int src;
        return kv_locate_few(len(lane), cta, ctas, &src);
    }
    KvSpot spot{0, 0, -1, n};
    const int64_t mine = len(tid);
    int64_t sum = mine;
    for (int b0 = THREADS; b0 < n; b0 += THREADS) sum += len(b0 + tid);
    sum = kv_scan(sum);
    if (lane == 31) scratch[warp] = sum;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; w++) spot.total += scratch[w];
    spot.per = kv_quotient(spot.total + ctas - 1, ctas);
    const int64_t at = spot.per * cta;
    if (at >= spot.total) return spot;
    int64_t before = 0;
    for (int b0 = 0; b0 < n; b0 += THREADS) {
        const int64_t v = b0 == 0 ? mine : len(b0 + tid);
        const int64_t inc = kv_scan(v);
        __syncthreads();
        if (lane == 31) scratch[warp] = inc;
        if (tid == 0) scratch[WARPS] = -1;
        __syncthreads();
        int64_t base = before, chunk = 0;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            if (w < warp) base += scratch[w];
            chunk += scratch[w];
        }
        const int64_t from = base + inc - v;
        if (from <= at && at < from + v) { scratch[WARPS] = b0 + tid; scratch[WARPS + 1] = from; }
        __syncthreads();
        if (scratch[WARPS] >= 0) { spot.b = (int)scratch[WARPS]; spot.start = scratch[WARPS + 1]; break; }
        before += chunk;
    }
    return spot;
}

// What a CTA leaves for the kernel that adds the pieces of a block of rows: the block that begins in it and goes on in the next CTAs.
struct alignas(16) KvCut {
    int pieces;     // CTAs that have a piece; 0: no block begins here and goes on
    int slot;       // of this CTA's piece: 0 its first, 1 its last
    int rows, head; // of the block
    int64_t row0;   // of the row arrays
    int lo_pos, pad;
};
__device__ __forceinline__ KvCut* kv_cuts(void* work) { return static_cast<KvCut*>(work); }
__host__ __device__ constexpr size_t kv_cut_bytes(int ctas) { return (size_t)ctas * sizeof(KvCut); }

// Behind the cuts: partial results of a CTA's first (slot 0) and last piece: `rows` times hd floats, then `rows` times (m, l).
__device__ __forceinline__ float* kv_part(void* work, int ctas, int rows, int hd, int64_t cta, int slot) {
    return reinterpret_cast<float*>(static_cast<char*>(work) + kv_cut_bytes(ctas)) + (cta * 2 + slot) * rows * (hd + 2);
}

__device__ __forceinline__ void kv_store1(const KvRows& o, int64_t e, float x) {
    if (o.type == L2_F32) reinterpret_cast<float*>(o.data)[e] = x;
    else if (o.type == L2_F16) reinterpret_cast<__half*>(o.data)[e] = __float2half_rn(x);
    else reinterpret_cast<__nv_bfloat16*>(o.data)[e] = __float2bfloat16_rn(x);
}

// ---- bytes as 16-bit numbers -------------------------------------------------------------------------------------------------
// The 16-bit numbers of bytes SEL & 3 and SEL >> 4 & 3 of w (two's complement), exact.
template <bool BF, uint32_t SEL>
__device__ __forceinline__ uint32_t widen(uint32_t w) {
    uint32_t r;
    constexpr uint32_t sel = 0x4040u | (SEL & 15u) | ((SEL >> 4) & 15u) << 8;
    if constexpr (BF) {  // 0x4300 | x is 128 + x for x < 128: 128 + (low seven bits) minus 128 or, for a negative byte, 256
        const uint32_t t = __byte_perm(w, 0, sel);
        uint32_t a, b;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(a) : "r"(t), "r"(0x007f007fu), "r"(0x43004300u));
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(b) : "r"(t), "r"(0x00800080u), "r"(0x43004300u));
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    } else {             // 0x6400 | x is 1024 + x: with the sign bit turned over, 1024 + 128 + byte
        const uint32_t t = __byte_perm(w ^ 0x80808080u, 0x64646464u, sel);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(t), "r"(0x64806480u));
    }
    return r;
}
template <bool BF> __device__ __forceinline__ uint32_t not_finite(uint32_t v) {  // non-zero where one of the two is NaN or infinite
    constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
    return ((v & E) == E) | ((v & (E << 16)) == (E << 16));
}
template <bool BF> __device__ __forceinline__ uint32_t only_finite(uint32_t v) {
    constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
    if ((v & E) == E) v &= 0xffff0000u;
    if ((v & (E << 16)) == (E << 16)) v &= 0x0000ffffu;
    return v;
}
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    uint32_t r;
    if constexpr (BF) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

}  // namespace l2
