// l2_kv_attend for sequences with many rows (chunks of a prompt, whole prompts): tcgen05 matrix products, softmax in registers.
//
// A block of up to 256 rows (tokens x query heads of one kv head) of one sequence, as two tiles Q0, Q1 of 128, walks tiles of 128 positions:
//   S = Q K^T (tensor memory),  P = 2^(scale S - m) (over S, 16 bits),  O += P V (tensor memory),  l += sum P,   out = O / l
// m is a row's maximum of some earlier tile: it is raised, and O and l scaled, only when a score exceeds it by more than 2^8 (the sums
// are f32: a common factor costs nothing).
//
// What bounds it.  A tile of positions is four products of 128 x 128 x 128, 2048 clocks of the tensor cores at their peak; 32768 exponentials, 2048 clocks of the
// special function units; and, because S is taken 64 positions at a time, 320 KB through shared memory at 128 bytes a clock, 2500.  A whole prompt (8191 tokens, 32
// heads of 128, bf16) takes about 3500 clocks a tile: 540 us on one input (1021 TFLOP/s of 1621 measured), 640 to 660 between others, as the chip's power allows.
// Counters of that prompt: tensor pipe 52 %, special functions 52 %, shared memory 53 % (48 for the products, 5 for the rest): none is full, the chain
// scores, softmax, product of the two row tiles is what is left.
// Measured on the way (the same prompt): one warp issuing for both tiles of rows 1017 us (an issue takes 75 to 85 clocks, whatever its size, and a wait some hundred); two
// 918; S in halves 803; Q requested eight lines at once 656; pieces planned by one warp, so that next to nothing spills (12 bytes; int8 196, 64 wide 132), 598; room on the line for a block's other costs 539.
// Not kept: exponentials on the FMA units (1, 2 or 4 of 16: 559 to 565 against 556), the two groups of softmax taking turns (608 against 598), a predicate in place of
// the branch around the issue (569 against 556).  An int8 cache costs about 1500 clocks a tile more (scales of 64 positions
// a thread and their products, and bytes to widen: 512 tokens of 64 heads behind 14,488 positions take 360 us on one input, 252 without either and 350 without one of them; four rows
// a quad of threads, so that each thread reads a quarter of the scales, took 349, but 40 rows a kv head 58 instead of 52).
//
// Work.  The tiles of positions of all (sequence, kv head, block) triples form one line, cut evenly over the SMs, with room in front of every
// block for what it costs besides its tiles (without it the SM with most blocks of that prompt took 1.13 times the mean); a block that a cut
// goes through leaves a partial (m, l, O) in each piece, which kv_tc_combine_kernel adds in order.  Causal blocks of different lengths,
// windows and ragged sequences need no other balance.
//
// Roles (they meet only through mbarriers):
//   warps 0, 2      one thread each issues the products of Q0 and of Q1, for 64 positions at a time, S in two halves of its room in turn: O += P V of one half,
//                   S = Q K of the same half of the next tile, and so on; the softmax finds the next scores ready
//   warp 1          K and V tiles by TMA into one ring, a copy a page run
//   warp 3          plans the pieces of the CTA, a few ahead, and leaves the kernel behind this one a record of the block that the CTA's end cuts
//   warps 4-7, 8-11 softmax of Q0 and Q1, a row a thread; they bring Q, and the result out
//   warps 12-15     16-bit caches: tiles that some row sees in part are searched for values that are not finite: 0 x NaN is NaN, and a row must not be
//                   reached by what it does not see.  They are taken out before the product and added to the rows that see them at the end.
//                   int8 caches: they turn the bytes into 16-bit numbers (K q's type, V bf16, exact); scales are applied to the scores and to the
//                   probabilities.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kernels.cuh"
#include "paged_attend.h"
#include "paged_device.cuh"

namespace l2 {

namespace {

constexpr int KT_TILE = 128, KT_SUB = 64, KT_ROWS = 256, KT_THREADS = 512;
constexpr int KT_MMA_WARP = 0, KT_COPY_WARP = 1, KT_PLAN_WARP = 3, KT_ROW_WARP = 4, KT_HELP_WARP = 12;
constexpr int KT_SCALE_SLOTS = 4;
// What a block costs besides its tiles, in tiles.  2 or 8 instead: 12 sequences with 5 tokens 9 % slower (int8 3 and 9 %); a prompt of 4095 tokens with heads of 64 4 %
// faster and 6 % slower; chunks of 512 over long caches within 1 % (int8 with heads of 64: 1 % faster, 4 % slower).
constexpr int KT_SETUP = 4;
constexpr int KT_RAISE = 8;  // powers of two that a score may exceed m by

template <int CT, int HD>
struct KtShape {
    static constexpr bool I8 = CT == L2_I8;
    static constexpr int SLOT = KT_TILE * HD * 2;                     // K or V of a tile in 16 bits
    static constexpr int RAW = I8 ? KT_TILE * HD : 0;                 // ... in 8
    static constexpr int SLOTS = HD == 64 ? 6 : I8 ? 3 : 5, RAWS = I8 ? (HD == 64 ? 4 : 3) : 0;
    static constexpr int SCALES = I8 ? KT_SCALE_SLOTS * 2 * KT_TILE * 4 : 0;
    static constexpr int Q_BYTES = 2 * SLOT;
    // (always more than half of an SM's shared memory: one CTA, one owner of the tensor memory, per SM)
    static constexpr int SMEM = 1024 + Q_BYTES + SLOTS * SLOT + RAWS * RAW + SCALES > 120 * 1024 ? 1024 + Q_BYTES + SLOTS * SLOT + RAWS * RAW + SCALES : 120 * 1024;
    static_assert(SMEM <= 226 * 1024, "shared memory");
};

__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo_units) { return ((saddr >> 4) & 0x3FFFu) | (lbo_units << 16); }
constexpr uint32_t KT_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);  // 8 rows of 128 bytes 1024 bytes apart, 128-byte swizzle
// D (+)= A B: A and B in shared memory, or A in tensor memory
template <bool ACC>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 da, db;\nsetp.ne.b32 p, %5, 0;\nmov.b64 da, {%1, %3};\nmov.b64 db, {%2, %3};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n}"
                 ::"r"(d), "r"(a_lo), "r"(b_lo), "n"(KT_DESC_HI), "r"(idesc), "n"(ACC ? 1 : 0) : "memory");
}
template <bool ACC>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 db;\nsetp.ne.b32 p, %5, 0;\nmov.b64 db, {%2, %3};\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}"
                 ::"r"(d), "r"(a), "r"(b_lo), "n"(KT_DESC_HI), "r"(idesc), "n"(ACC ? 1 : 0) : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(kv_smem(bar)) : "memory");
}
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
#define KT_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define KT_W8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t* v, uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : KT_R8(v, 0), KT_R8(v, 8), KT_R8(v, 16), KT_R8(v, 24) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t* v, uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : KT_R8(v, 0), KT_R8(v, 8) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
                 ::KT_W8(v, 0), KT_W8(v, 8), KT_W8(v, 16), KT_W8(v, 24), "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::KT_W8(v, 0), KT_W8(v, 8), "r"(addr) : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ unsigned long long pair(float a, float b) {
    unsigned long long d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 unpair(unsigned long long d) {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(d));
    return v;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// byte offset of 16-byte chunk c of row r in a tile of 128 rows: halves of 128 bytes one after the other, 128-byte swizzle (rows of 64 bytes: 64-byte swizzle)
__device__ __forceinline__ uint32_t kt_offset(int r, int c) { return (c >> 3) * (KT_TILE * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4); }
__device__ __forceinline__ uint32_t kt_offset64(int r, int c) { return r * 64 + ((c ^ ((r >> 1) & 3)) << 4); }

// ---- the line: sequence by sequence, kv head by kv head, block by block, tile by tile ---------------------------------------
struct KtBlocks { KvSeq s; int tokens, n; };  // blocks of a sequence, of `tokens` tokens; n = 0: not this kernel's
__device__ __forceinline__ KtBlocks kt_blocks(const KvAttendParams& P, int lim, int b) {
    KtBlocks k;
    k.tokens = KT_ROWS / P.group;
    k.n = 0;
    if (b >= P.step.n_seqs) { k.s = KvSeq{0, 0, 0}; return k; }
    k.s = kv_seq(P.step, P.pool.page_shift, b);
    if ((int64_t)k.s.n * P.group > lim) k.n = (k.s.n + k.tokens - 1) / k.tokens;
    return k;
}
__device__ __forceinline__ KvView<KT_TILE> kt_view(const KvAttendParams& P, const KtBlocks& k, int block) {
    const int t0 = block * k.tokens, t1 = min(k.s.n, t0 + k.tokens), p = k.s.kv - k.s.n;
    return KvView<KT_TILE>(p + t0, p + t1 - 1, P.window, P.sinks);
}
// Tiles of one kv head of the lane's sequence, by the whole warp (each lane its own sequence).  (The host refuses steps where they could pass 31 bits.)
__device__ __forceinline__ int kt_tiles(const KvAttendParams& P, KtBlocks k) {
    const int lane = threadIdx.x & 31;
    int sum = 0;
    if (k.n <= 4) {
#pragma unroll 1
        for (int i = 0; i < k.n; i++) sum += KT_SETUP + kt_view(P, k, i).tiles;
    }
    unsigned many = __ballot_sync(0xffffffffu, k.n > 4);
#pragma unroll 1
    while (many) {  // the warp's lanes share the blocks of a long one
        const int src = __ffs(many) - 1;
        many &= many - 1;
        KtBlocks q = k;
        q.s.n = __shfl_sync(0xffffffffu, k.s.n, src);
        q.s.kv = __shfl_sync(0xffffffffu, k.s.kv, src);
        q.n = __shfl_sync(0xffffffffu, k.n, src);
        int x = 0;
#pragma unroll 1
        for (int i = lane; i < q.n; i += 32) x += KT_SETUP + kt_view(P, q, i).tiles;
        x = __reduce_add_sync(0xffffffffu, x);
        if (lane == src) sum = x;
    }
    return sum;
}
// The block that tile `at` of a head of the sequence is in, and the tiles in front of it; by the whole warp, all lanes with the same arguments.
__device__ __forceinline__ int kt_find_block(const KvAttendParams& P, const KtBlocks& k, int at, int* before) {
    const int lane = threadIdx.x & 31;
    int base = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < k.n; i0 += 32) {
        const int mine = i0 + lane < k.n ? KT_SETUP + kt_view(P, k, i0 + lane).tiles : 0;
        int v = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        const unsigned past = __ballot_sync(0xffffffffu, base + v > at);
        if (past) {
            const int l = __ffs(past) - 1;
            *before = base + __shfl_sync(0xffffffffu, v - mine, l);
            return i0 + l;
        }
        base += __shfl_sync(0xffffffffu, v, 31);
    }
    *before = base;
    return k.n - 1;
}

// row / group for the rows of a block: exact for rows below 256, groups up to 64 (the error of the rounded-up reciprocal stays below 1 / group)
__device__ __forceinline__ int kt_token(const KvAttendParams& P, int row) { return row * P.group_inv >> 16; }

struct KtWalk {
    int64_t w, w1, per;
    int b, head, block, skip;  // skip: tiles of the first block that belong to the CTA in front
    KtBlocks k;
    KvView<KT_TILE> view;
    int t0, t1, rows, index;   // rows of the block; pieces before this one
    // k and tiles: the blocks of the spot's sequence, and the tiles of one of its kv heads
    __device__ __forceinline__ KtWalk(const KvAttendParams& P, const KvSpot& spot, const KtBlocks& blocks, int tiles) : k(blocks) {
        per = spot.per;
        w = per * blockIdx.x;
        w1 = min(spot.total, w + per);
        b = spot.b; index = -1; head = block = skip = 0;
        if (w >= w1) return;
        const int64_t in = w - spot.start;
        head = (int)kv_quotient(in, tiles);
        const int at = (int)(in - (int64_t)head * tiles);
        int before = 0;
        if (k.n > 1) block = kt_find_block(P, k, at, &before);
        skip = at - before;
        block--;  // (next() goes on to it)
    }
    __device__ __forceinline__ bool next(const KvAttendParams& P, int lim) {
#pragma unroll 1
        while (w < w1) {
            if (++block >= k.n) {
                block = 0;
                if (++head == P.pool.n_kv_heads) {
                    head = 0;
                    do k = kt_blocks(P, lim, ++b); while (!k.n && b < P.step.n_seqs);
                }
            }
            view = kt_view(P, k, block);
            const int at = skip, end = (int)min((int64_t)view.tiles + KT_SETUP, at + (w1 - w));  // of the block's place on the line, whose first KT_SETUP are no tiles
            skip = 0;
            w += end - at;
            t0 = max(0, at - KT_SETUP);
            t1 = end - KT_SETUP;
            if (t1 <= t0) continue;  // (the block's tiles begin in the next CTA)
            rows = min(k.tokens, k.s.n - block * k.tokens) * P.group;
            index++;
            return true;
        }
        return false;
    }
};

// One piece as the roles read it (shared memory): tiles t0 .. t1 - 1 of positions of a block of rows.
struct KtPiece {
    int on;                             // 0: no more pieces
    int t0, t1, tiles, sink_tiles, first;
    int lo_pos, hi_pos, lo[2], hi[2];   // positions of the block's rows, and of those of each tile of rows (hi -1: it has none, and sees nothing)
    int rows, head, b, index;           // index: pieces before this one
    int64_t row0;                       // of the row arrays
    __device__ __forceinline__ KvView<KT_TILE> view(int lo, int hi) const {
        KvView<KT_TILE> v;
        v.lo_pos = lo; v.hi_pos = hi; v.sink_tiles = sink_tiles; v.first = first; v.tiles = tiles;
        return v;
    }
    __device__ __forceinline__ KvView<KT_TILE> part(int i) const { return view(lo[i], hi[i]); }
    __device__ __forceinline__ int base(int t) const { return (t < sink_tiles ? t : first + t - sink_tiles) * KT_TILE; }
    // A bit for each of the tiles t .. t + 31 of positions (of this piece) of which f(first position) holds; by the whole warp.  What is decided once for 32
    // tiles, and by a vote, is in uniform registers, and so is all that follows from it.
    template <class F> __device__ __forceinline__ uint32_t bits(int t, F f) const {
        const int mine = t + (threadIdx.x & 31);
        return __ballot_sync(0xffffffffu, mine >= t0 && mine < t1 && f(base(mine)));
    }
};
constexpr int KT_PIECES = 4;

template <int CT, bool QB, int HD>
__global__ void __launch_bounds__(KT_THREADS, 1) kv_tc_kernel(const __grid_constant__ KvAttendParams P, const int lim, const __grid_constant__ CUtensorMap map_k,
                                                              const __grid_constant__ CUtensorMap map_v) {
    using S = KtShape<CT, HD>;
    constexpr bool I8 = S::I8, PB = I8 || QB;
    constexpr int LANES = HD / 8;
    constexpr uint32_t S_COL = 0, O_COL = 256;                   // tensor memory: S0 S1 O0 O1, 128 columns each; P over S
    // Probabilities carry a factor of 2^BIAS, so that small ones are normal numbers: f16 at most 2^(7 + KT_RAISE); f32 and bf16 have room (2^95 for a V).
    constexpr float BIAS = PB ? 24.0f : 7.0f;
    extern __shared__ __align__(1024) uint8_t kt_smem[];
    __shared__ __align__(8) uint64_t full[S::SLOTS], empty[S::SLOTS], ready[S::SLOTS], raw_full[I8 ? S::RAWS : 1], raw_empty[I8 ? S::RAWS : 1],
        sc_full[KT_SCALE_SLOTS], sc_empty[KT_SCALE_SLOTS], q_full[2], s_full[2][2], p_full[2][2], pv_done[2][2], drained[2];
    __shared__ int64_t scratch[KT_THREADS / 32 + 2];
    __shared__ __align__(8) uint64_t piece_full[KT_PIECES], piece_empty[KT_PIECES], row_meet[2];
    __shared__ KtPiece pieces[KT_PIECES];
    __shared__ uint32_t tmem_s;
    __shared__ volatile int failed;
    __shared__ volatile int odd[8];  // by piece: values that are not finite have been taken out of a V tile
    uint8_t* sq = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(kt_smem) + 1023) & ~(uintptr_t)1023);  // Q0, Q1
    uint8_t* ring = sq + S::Q_BYTES;
    uint8_t* raw = ring + S::SLOTS * S::SLOT;
    float* scales = reinterpret_cast<float*>(raw + S::RAWS * S::RAW);  // [slot][k, v][position]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // (Code that runs once comes from far away, 100 clocks and more for eight instructions: every warp prepares a little.)
    if (warp == 4 && lane < S::SLOTS) { kv_bar_init(&full[lane], I8 ? 4 : 1); kv_bar_init(&empty[lane], I8 ? 2 : 6); kv_bar_init(&ready[lane], 4); }
    if (I8 && warp == 5 && lane < S::RAWS) { kv_bar_init(&raw_full[lane], 1); kv_bar_init(&raw_empty[lane], 4); }
    if (I8 && warp == 6 && lane < KT_SCALE_SLOTS) { kv_bar_init(&sc_full[lane], 32); kv_bar_init(&sc_empty[lane], 8); }
    if (warp == 7 && lane < KT_PIECES) { kv_bar_init(&piece_full[lane], 1); kv_bar_init(&piece_empty[lane], 15); }
    if (warp == 8 && lane < 2) { kv_bar_init(&q_full[lane], 128); kv_bar_init(&drained[lane], 1); kv_bar_init(&row_meet[lane], 4); }
    if (warp == 9 && lane < 4) { kv_bar_init(&s_full[0][0] + lane, 1); kv_bar_init(&p_full[0][0] + lane, 4); kv_bar_init(&pv_done[0][0] + lane, 1); }
    if (warp == 10 && lane < 8) odd[lane] = 0;
    if (tid == 0) failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (warp == KT_MMA_WARP) {  // all 512 columns of tensor memory
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(kv_smem(&tmem_s)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == KT_COPY_WARP && lane < 2) kv_prefetch_map(lane ? &map_v : &map_k);
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (rows, lengths and the cache may come from the kernel in front)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    KvSpot spot{0, 0, -1, 0};
    if (P.step.n_seqs > 32) spot = kv_locate<KT_THREADS>(P.step.n_seqs, blockIdx.x, gridDim.x, scratch, [&](int b) { return (int64_t)kt_tiles(P, kt_blocks(P, lim, b)) * P.pool.n_kv_heads; });
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_s;
    const KvWait wait{&failed};
    // Pieces are planned by one warp and read by the others from a ring: the walk's state would cost each role thirty registers.
    auto piece_at = [&](uint32_t n) -> const KtPiece& { wait(&piece_full[n % KT_PIECES], (n / KT_PIECES) & 1u); return pieces[n % KT_PIECES]; };
    auto is_one = [&](const KtPiece& piece) { return __any_sync(0xffffffffu, piece.on) && !wait.over(); };
    auto give_back = [&](uint32_t n) { __syncwarp(); if (lane == 0) kv_bar_arrive(&piece_empty[n % KT_PIECES]); };

    if (warp >= KT_ROW_WARP && warp < KT_HELP_WARP) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        // ================= softmax: a row a thread ============================================================================
        const int i = (warp - KT_ROW_WARP) >> 2, row = 128 * i + (tid & 127);
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, s_row = tmem + lanes + S_COL + 128 * i, o_at = tmem + lanes + O_COL + 128 * i;
        uint32_t s_ph = 0, sc = 0, sc_ph = 0;
        // Q of a piece is requested while the result of the piece in front is still on its way out.  HD / 8 threads have a row.
        constexpr int Q_ROWS = 128 / LANES, Q_N = 128 / Q_ROWS;  // rows at once, and of a thread
        uint4 qx[Q_N];
        auto request_q = [&](const KtPiece& piece) {
            const char* const from = P.q.data + 2 * (piece.row0 * P.q.row_stride + (int64_t)piece.head * P.group * P.q.head_stride + 8 * (tid % LANES));
            const int rows = piece.rows;
#pragma unroll
            for (int n = 0; n < Q_N; n++) {  // (rows that there are not: zeros)
                const int f = 128 * i + (tid & 127) / LANES + n * Q_ROWS, k = kt_token(P, f);
                qx[n] = make_uint4(0, 0, 0, 0);
                if (f < rows) qx[n] = *reinterpret_cast<const uint4*>(from + 2 * (k * P.q.row_stride + (int64_t)(f - k * P.group) * P.q.head_stride));
            }
        };
        uint32_t meet_ph = 0;
        auto meet = [&]() {  // of the four warps
            __syncwarp();
            if (lane == 0) kv_bar_arrive(&row_meet[i]);
            wait(&row_meet[i], meet_ph);
            meet_ph ^= 1u;
            __syncwarp();
        };
        bool more = is_one(piece_at(0));
        if (more) request_q(pieces[0]);
        for (uint32_t n = 0; more; n++) {
            const KtPiece& walk = pieces[n % KT_PIECES];
            const KvView<KT_TILE> mine = walk.part(i);
            const int t0 = walk.t0, t1 = walk.t1;
            const int tok = kt_token(P, min(row, walk.rows - 1));
            const int pos = walk.lo_pos + tok;
            auto any = [&](int base) { return mine.any(base, KT_TILE, P.window, P.sinks); };
            uint32_t some = 0;  // this tile of rows sees something in the piece
            for (int t = t0; t < t1 && !some; t += 32) some = walk.bits(t, any);
            if (some) {  // Q, swizzled as the products want it
#pragma unroll
                for (int n = 0; n < Q_N; n++) *reinterpret_cast<uint4*>(sq + i * S::SLOT + kt_offset((tid & 127) / LANES + n * Q_ROWS, tid % LANES)) = qx[n];
                fence_async();
                kv_bar_arrive(&q_full[i]);
            }
            float m = -INFINITY, l = 0.0f;
            int seen = 0;      // halves of tiles seen
            uint32_t on = 0, all = 0;  // by tile of positions: seen by some row; by every row
#pragma unroll 1
            for (int t = t0; t < t1; t++, on >>= 1, all >>= 1) {
                if ((t - t0) % 32 == 0) {
                    on = walk.bits(t, any);
                    all = walk.bits(t, [&](int base) { return mine.whole(base, P.window, P.sinks); });
                }
                if (!(on & 1u)) {
                    if constexpr (I8) {
                        wait(&sc_full[sc], sc_ph);
                        __syncwarp();
                        if (lane == 0) kv_bar_arrive(&sc_empty[sc]);
                        if (++sc == KT_SCALE_SLOTS) { sc = 0; sc_ph ^= 1u; }
                    }
                    continue;
                }
                const bool whole = all & 1u;
                if constexpr (I8) wait(&sc_full[sc], sc_ph);
#pragma unroll 1
                for (int h = 0; h < 2; h++, seen++) {
                    const float* ks = scales + sc * 2 * KT_TILE + KT_SUB * h;
                    const uint32_t s_at = s_row + KT_SUB * h;
                    uint32_t x[KT_SUB];
                    wait(&s_full[i][h], s_ph);
                    __syncwarp();
                    fence_after();
                    tmem_ld32(x, s_at);
                    tmem_ld32(x + 32, s_at + 32);
                    wait_ld();
                    if constexpr (I8) {
#pragma unroll
                        for (int j = 0; j < KT_SUB; j += 4) {
                            const float4 k = *reinterpret_cast<const float4*>(ks + j);
                            const float2 a = unpair(mul2(pair(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), pair(k.x, k.y)));
                            const float2 b = unpair(mul2(pair(__uint_as_float(x[j + 2]), __uint_as_float(x[j + 3])), pair(k.z, k.w)));
                            x[j] = __float_as_uint(a.x); x[j + 1] = __float_as_uint(a.y); x[j + 2] = __float_as_uint(b.x); x[j + 3] = __float_as_uint(b.y);
                        }
                    }
                    auto visible = [&]() {  // a bit for each of the 64 positions: j <= hi and (j > lo or j < sinks)
                        const int base = walk.base(t) + KT_SUB * h;
                        auto below = [](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };
                        return below(pos - base + 1) & (P.window ? ~below(pos - P.window - base + 1) | below(P.sinks - base) : ~0ull);
                    };
                    if (!whole) {
                        const unsigned long long bits = visible();
#pragma unroll
                        for (int j = 0; j < KT_SUB; j++)
                            if (!(bits >> j & 1ull)) x[j] = 0xff800000u;
                    }
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int j = 0; j < KT_SUB; j += 8)
#pragma unroll
                        for (int c = 0; c < 4; c++) top[c] = fmaxf(top[c], fmaxf(__uint_as_float(x[j + c]), __uint_as_float(x[j + 4 + c])));
                    const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * P.scale_log2 - BIAS;
                    const bool raise = most > m + KT_RAISE;
                    if (__any_sync(0xffffffffu, raise)) {
                        const float m1 = raise ? most : m;  // (a row's result does not depend on the others of its warp)
                        const KvScale f(m1 == -INFINITY ? 0.0f : m - m1);
                        m = m1;
                        l = f(l);
                        if (seen) {  // O is this thread's when the product in front has written it
                            wait(&pv_done[i][h ^ 1], h ? s_ph : s_ph ^ 1u);
                            __syncwarp();
                            fence_after();
#pragma unroll 1
                            for (int c = 0; c < HD; c += 16) {
                                uint32_t o[16];
                                tmem_ld16(o, o_at + c);
                                wait_ld();
#pragma unroll
                                for (int j = 0; j < 16; j++) o[j] = __float_as_uint(f(__uint_as_float(o[j])));
                                tmem_st16(o_at + c, o);
                            }
                        }
                    }
                    const float ref = m == -INFINITY ? 0.0f : m;
                    const unsigned long long f2 = pair(P.scale_log2, P.scale_log2), r2 = pair(-ref, -ref);
                    unsigned long long sum[2] = {0ull, 0ull};
                    auto probabilities = [&](auto is_whole) {  // (an int8 cache with the choice at every element: 378 us instead of 362)
                        uint32_t p16[KT_SUB / 2];
                        float4 v4 = make_float4(0.f, 0.f, 0.f, 0.f);
                        const unsigned long long bits = decltype(is_whole)::value ? 0ull : visible();
#pragma unroll
                        for (int j = 0; j < KT_SUB; j += 2) {
                            const float2 e = unpair(fma2(pair(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), f2, r2));
                            float2 p = make_float2(kv_exp2(e.x), kv_exp2(e.y));
                            sum[(j >> 1) & 1] = add2(sum[(j >> 1) & 1], pair(p.x, p.y));
                            if constexpr (I8) {
                                if (j % 4 == 0) v4 = *reinterpret_cast<const float4*>(ks + KT_TILE + j);
                                const float2 v = j % 4 ? make_float2(v4.z, v4.w) : make_float2(v4.x, v4.y);
                                if constexpr (decltype(is_whole)::value) p = unpair(mul2(pair(p.x, p.y), pair(v.x, v.y)));
                                else p = make_float2(bits >> j & 1ull ? p.x * v.x : 0.0f, bits >> j & 2ull ? p.y * v.y : 0.0f);  // (what is not seen may have any scale)
                            }
                            p16[j / 2] = pack16<PB>(p.x, p.y);
                        }
                        tmem_st32(s_at, p16);
                    };
                    if (!I8 || whole) probabilities(std::true_type());
                    else probabilities(std::false_type());
                    const float2 s0 = unpair(sum[0]), s1 = unpair(sum[1]);
                    l += (s0.x + s0.y) + (s1.x + s1.y);
                    wait_st();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) kv_bar_arrive(&p_full[i][h]);
                }
                s_ph ^= 1u;
                if constexpr (I8) {
                    if (lane == 0) kv_bar_arrive(&sc_empty[sc]);
                    if (++sc == KT_SCALE_SLOTS) { sc = 0; sc_ph ^= 1u; }
                }
            }
            // ---- the result of the piece
            more = is_one(piece_at(n + 1));
            if (more) request_q(pieces[(n + 1) % KT_PIECES]);
            const bool done = t0 == 0 && t1 == walk.tiles, started = seen > 0;
            if (started) {
                wait(&pv_done[i][1], s_ph ^ 1u);
                __syncwarp();
                fence_after();
            }
            if (128 * i >= walk.rows) { give_back(n); continue; }  // (this tile has no rows)
            const bool fix = !I8 && started && odd[walk.index & 7];
            float* part = kv_part(P.work, gridDim.x, KT_ROWS, HD, blockIdx.x, walk.index ? 1 : 0);
            const float inv = done && pos >= 0 ? 1.0f / l : 1.0f;
            // A whole block's result goes through this tile's room of Q (its products are done), so that rows leave in whole lines.
            uint8_t* stage = sq + i * S::SLOT;
            const int wide = P.out.type == L2_F32 ? 4 : 2, cols = HD * 2 / wide;  // bytes of an element, columns at a time
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                if (started) { tmem_ld32(o, o_at + c); wait_ld(); }
                else {
#pragma unroll
                    for (int j = 0; j < 32; j++) o[j] = 0u;
                }
                if constexpr (!I8) {
                    if (fix) {  // rare: the values that were taken out, one by one, to the rows that see them
#pragma unroll 1
                        for (int t = walk.t0; t < walk.t1; t++) {
                            const int base = walk.base(t);
                            if (!mine.any(base, KT_TILE, P.window, P.sinks) || mine.whole(base, P.window, P.sinks)) {
                                const KvView<KT_TILE> other = walk.part(i ^ 1);  // (taken out for the other tile's rows)
                                if (!mine.any(base, KT_TILE, P.window, P.sinks) || !other.any(base, KT_TILE, P.window, P.sinks) || other.whole(base, P.window, P.sinks)) continue;
                            }
#pragma unroll 1
                            for (int j = base; j < base + KT_TILE; j++) {
                                if (!kv_sees(pos, j, P.window, P.sinks)) continue;
                                const int page = kv_page(P.step, P.pool, walk.b, j);
                                if (page < 0) continue;
                                const uint16_t* v = reinterpret_cast<const uint16_t*>(P.pool.v) + (int64_t)page * P.pool.page_stride +
                                                    (j & ((1 << P.pool.page_shift) - 1)) * P.pool.pos_stride + walk.head * P.pool.head_stride + c;
#pragma unroll
                                for (int e = 0; e < 32; e++) {
                                    const uint16_t bits = v[e];
                                    if (not_finite<QB>(bits)) o[e] = __float_as_uint(__uint_as_float(o[e]) + (QB ? __uint_as_float((uint32_t)bits << 16) : __half2float(__ushort_as_half(bits))));
                                }
                            }
                        }
                    }
                }
                if (!done) {  // partial results: [4 columns][row][4], so that a warp's rows are side by side
#pragma unroll
                    for (int j = 0; j < 32; j += 4) *reinterpret_cast<uint4*>(part + ((c + j) / 4 * KT_ROWS + row) * 4) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                    continue;
                }
                const float f = pos < 0 ? 0.0f : inv;
                if (pos < 0) {
#pragma unroll
                    for (int j = 0; j < 32; j++) o[j] = 0u;
                }
                const int in = c % cols, r = tid & 127;
                auto y = [&](int j) { return __uint_as_float(o[j]) * f; };
                if (wide == 4) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(stage + kt_offset(r, (in + j) / 4)) = make_float4(y(j), y(j + 1), y(j + 2), y(j + 3));
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                        *reinterpret_cast<uint4*>(stage + kt_offset(r, (in + j) / 8)) = make_uint4(pack16<QB>(y(j), y(j + 1)), pack16<QB>(y(j + 2), y(j + 3)), pack16<QB>(y(j + 4), y(j + 5)), pack16<QB>(y(j + 6), y(j + 7)));
                }
                if (in + 32 < cols) continue;
                meet();
                const int ch = tid % LANES;
                char* const out = P.out.data + ((walk.row0) * P.out.row_stride + (int64_t)walk.head * P.group * P.out.head_stride + (c + 32 - cols)) * wide + 16 * ch;
#pragma unroll
                for (int n0 = 0; n0 < Q_N; n0 += 4) {
                    uint4 w[4];
#pragma unroll
                    for (int n = 0; n < 4; n++) w[n] = *reinterpret_cast<const uint4*>(stage + kt_offset((tid & 127) / LANES + (n0 + n) * Q_ROWS, ch));
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        const int fl = 128 * i + (tid & 127) / LANES + (n0 + n) * Q_ROWS, k = kt_token(P, fl);
                        if (fl < walk.rows) *reinterpret_cast<uint4*>(out + (k * P.out.row_stride + (int64_t)(fl - k * P.group) * P.out.head_stride) * wide) = w[n];
                    }
                }
                meet();
            }
            if (!done) *reinterpret_cast<float2*>(part + KT_ROWS * HD + 2 * row) = make_float2(m, l);
            fence_before();
            give_back(n);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == KT_MMA_WARP || warp == KT_MMA_WARP + 2) {
            // ================= products of one tile of rows =====================================================================
            // (All of the tensor memory is this CTA's: it starts at 0.  The operands are uniform registers: the whole warp walks, one elected lane issues.)
            const int i = warp == KT_MMA_WARP ? 0 : 1;
            const bool leader = elect();
            constexpr uint32_t fmt = QB ? 1u : 0u, fmt_p = PB ? 1u : 0u;
            constexpr uint32_t idesc_s = (1u << 4) | (fmt << 7) | (fmt << 10) | (((uint32_t)KT_SUB >> 3) << 17) | ((128u >> 4) << 24);
            constexpr uint32_t idesc_o = (1u << 4) | (fmt_p << 7) | (fmt_p << 10) | (1u << 16) | (((uint32_t)HD >> 3) << 17) | ((128u >> 4) << 24);  // V: elements contiguous
            const uint32_t s_col = S_COL + 128 * i, o_col = O_COL + 128 * i, q_lo = desc_lo(kv_smem(sq + i * S::SLOT), 1), k_lo = desc_lo(kv_smem(ring), 1),
                           v_lo = desc_lo(kv_smem(ring), KT_TILE * 128 / 16);
            uint32_t slot = 0, ph = 0, ready_ph = 0, q_ph = 0, p_ph = 0;  // ready_ph: a bit for each slot
            auto step = [&]() { if (++slot == S::SLOTS) { slot = 0; ph ^= 1u; } };
            for (uint32_t n = 0;; n++) {
                const KtPiece& walk = piece_at(n);
                if (!is_one(walk)) break;
                const KvView<KT_TILE> mine = walk.part(i), other = walk.part(i ^ 1);
                auto any = [&](int base) { return mine.any(base, KT_TILE, P.window, P.sinks); };
                const int t0 = __reduce_max_sync(0xffffffffu, walk.t0), t1 = __reduce_max_sync(0xffffffffu, walk.t1);
                uint32_t begun = 0;  // S has been computed (1), O has been written (2)
                auto scores = [&](int h) {  // S of half a tile, from the K tile in the current slot
                    if (!(begun & 1u)) { wait(&q_full[i], q_ph); q_ph ^= 1u; begun |= 1u; }
                    __syncwarp();
                    fence_after();
                    const uint32_t k_at = k_lo + slot * (S::SLOT / 16) + h * (KT_SUB * 128 / 16), d = s_col + KT_SUB * h;
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < HD / 16; k++) {
                            const uint32_t off = (k / 4) * (KT_TILE * 128 / 16) + (k % 4) * 2;
                            if (k == 0) mma_ss<false>(d, q_lo + off, k_at + off, idesc_s);
                            else mma_ss<true>(d, q_lo + off, k_at + off, idesc_s);
                        }
                        commit(&s_full[i][h]);
                    }
                    __syncwarp();
                };
                uint32_t on = walk.bits(t0, any);
                wait(&full[slot], ph);
                if (on & 1u) { scores(0); scores(1); }
                if (leader) commit(&empty[slot]);
                __syncwarp();
                step();
#pragma unroll 1
                for (int tc = t0; tc < t1; tc += 32) {
                    const uint32_t part = I8 ? 0u : walk.bits(tc, [&](int base) {
                        return (any(base) && !mine.whole(base, P.window, P.sinks)) || (other.any(base, KT_TILE, P.window, P.sinks) && !other.whole(base, P.window, P.sinks)); });
                    on = walk.bits(tc, any);
                    const uint32_t next = walk.bits(tc + 1, any);
                    const int tiles = min(32, t1 - tc);
#pragma unroll 1
                    for (int b = 0; b < tiles; b++) {
                        const uint32_t v_slot = slot, v_ph = ph;
                        step();
                        const bool more = tc + b + 1 < t1;
                        wait(&full[v_slot], v_ph);
                        if (part >> b & 1u) { wait(&ready[v_slot], ready_ph >> v_slot & 1u); ready_ph ^= 1u << v_slot; }
                        if (more) wait(&full[slot], ph);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            if (on >> b & 1u) {
                                wait(&p_full[i][h], p_ph);
                                __syncwarp();
                                fence_after();
                                const uint32_t v_at = v_lo + v_slot * (S::SLOT / 16) + h * (KT_SUB * 128 / 16), a = s_col + KT_SUB * h;
                                if (leader) {
                                    if (begun & 2u) mma_ts<true>(o_col, a, v_at, idesc_o);
                                    else mma_ts<false>(o_col, a, v_at, idesc_o);
#pragma unroll
                                    for (int k = 1; k < KT_SUB / 16; k++) mma_ts<true>(o_col, a + 8 * k, v_at + k * (16 * 128 / 16), idesc_o);
                                    commit(&pv_done[i][h]);
                                }
                                begun |= 2u;
                                __syncwarp();
                            }
                            if (next >> b & 1u) scores(h);
                        }
                        p_ph ^= on >> b & 1u;
                        if (leader) {
                            commit(&empty[v_slot]);
                            if (more) commit(&empty[slot]);
                        }
                        __syncwarp();
                        if (more) step();
                    }
                }
                give_back(n);
            }
            if (failed) {  // products still under way read shared memory: a bounded time to end
                if (leader) commit(&drained[i]);
                __syncwarp();
                for (int n = 0; n < 1024 && !kv_bar_try(&drained[i], 0); n++) {}
            }
        } else if (warp == KT_COPY_WARP) {
            // ================= copies: lane l brings run l of a tile ==============================================================
            const int R = min(KT_TILE, 1 << P.pool.page_shift), runs = KT_TILE / R;
            constexpr int RB = HD * (I8 ? 1 : 2), W = RB < 128 ? RB : 128;  // bytes of a row, of a copy's row
            uint32_t slot = 0, ph = 1, sc = 0, sc_ph = 1;
            bool over = false;
            for (uint32_t n = 0; !over; n++) {
                const KtPiece& walk = piece_at(n);
                if (!is_one(walk)) break;
                const KvView<KT_TILE> view = walk.view(walk.lo_pos, walk.hi_pos);
                const int t0 = walk.t0, t1 = walk.t1, head = walk.head, b = walk.b;
                auto page_of = [&](int t) {  // the page of this lane's run of tile t, n_pages (zeros) where no row sees it or there is none
                    const int j = view.base(t) + lane * R;
                    if (lane >= runs || !view.any(j, R, P.window, P.sinks)) return P.pool.n_pages;
                    const int x = kv_page(P.step, P.pool, b, j);
                    return x >= 0 ? x : P.pool.n_pages;
                };
                int page = page_of(t0);
                for (int t = t0; t < t1; t++) {
                    const int j = view.base(t) + lane * R, at = j & ((1 << P.pool.page_shift) - 1);
                    const int ahead = t + 1 < t1 ? page_of(t + 1) : P.pool.n_pages;
                    if constexpr (I8) {
                        wait(&sc_empty[sc], sc_ph);
                        if ((over = wait.over())) break;
                        // four positions a lane, of K and of V
                        const int x = 4 * lane, of = __shfl_sync(0xffffffffu, page, x / R);
                        const bool there = of < P.pool.n_pages;
                        const int64_t e = ((int64_t)(there ? of : 0) * P.pool.n_kv_heads + head << P.pool.page_shift) + ((view.base(t) + x) & ((1 << P.pool.page_shift) - 1));
                        const uint32_t to = kv_smem(scales + sc * 2 * KT_TILE + x);
                        kv_copy16(to, P.pool.ks + e, there);
                        kv_copy16(to + 4 * KT_TILE, P.pool.vs + e, there);
                        kv_copy16_arrive(&sc_full[sc]);
                        if (++sc == KT_SCALE_SLOTS) { sc = 0; sc_ph ^= 1u; }
                    }
#pragma unroll
                    for (int kv = 0; kv < 2; kv++) {
                        uint64_t *f = I8 ? &raw_full[slot] : &full[slot], *e = I8 ? &raw_empty[slot] : &empty[slot];
                        wait(e, ph);
                        if ((over = wait.over())) break;
                        if (lane == 0) kv_bar_expect(f, KT_TILE * RB);
                        __syncwarp();
                        if (lane < runs) {
                            const uint32_t to = kv_smem(I8 ? raw + slot * S::RAW : ring + slot * S::SLOT) + lane * R * W;
#pragma unroll
                            for (int h = 0; h < RB / W; h++) kv_tma4(to + h * (KT_TILE * 128), kv ? &map_v : &map_k, h * 64, at, head, page, f);
                        }
                        if (++slot == (I8 ? S::RAWS : S::SLOTS)) { slot = 0; ph ^= 1u; }
                    }
                    if (over) break;
                    page = ahead;
                }
                give_back(n);
            }
        } else if (warp == KT_PLAN_WARP) {
            // ================= pieces, and what the next kernel has to know of them ===================================================
            // (up to 32 sequences: a lane has one)
            const bool few = P.step.n_seqs <= 32;
            KtBlocks k = kt_blocks(P, lim, few ? lane : spot.b);
            int tiles = kt_tiles(P, k);
            if (few) {
                int src;
                spot = kv_locate_few((int64_t)tiles * P.pool.n_kv_heads, blockIdx.x, gridDim.x, &src);
                k.s.row0 = __shfl_sync(0xffffffffu, k.s.row0, src);
                k.s.n = __shfl_sync(0xffffffffu, k.s.n, src);
                k.s.kv = __shfl_sync(0xffffffffu, k.s.kv, src);
                k.n = __shfl_sync(0xffffffffu, k.n, src);
                tiles = __shfl_sync(0xffffffffu, tiles, src);
            }
            KtWalk walk(P, spot, k, tiles);
            KvCut cut{0, 0, 0, 0, 0, 0, 0};
            bool more = true;
            for (uint32_t n = 0; more; n++) {
                more = walk.next(P, lim);
                const int64_t row0 = (int64_t)walk.k.s.row0 + walk.block * walk.k.tokens;
                if (more && walk.t0 == 0 && walk.t1 < walk.view.tiles)
                    cut = KvCut{(int)kv_quotient(walk.w - walk.t1 + walk.view.tiles - 1, walk.per) - (int)blockIdx.x + 1, walk.index ? 1 : 0, walk.rows, walk.head, row0, walk.view.lo_pos, 0};
                wait(&piece_empty[n % KT_PIECES], (n / KT_PIECES & 1u) ^ 1u);
                if (wait.over()) break;
                if (lane == 0) {
                    KtPiece& p = pieces[n % KT_PIECES];
                    p.on = more;
                    if (more) {
                        p.t0 = walk.t0; p.t1 = walk.t1; p.tiles = walk.view.tiles; p.sink_tiles = walk.view.sink_tiles; p.first = walk.view.first;
                        p.lo_pos = walk.view.lo_pos; p.hi_pos = walk.view.hi_pos;
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const int lo = 128 * i, hi = min(walk.rows, lo + 128) - 1;
                            p.lo[i] = walk.view.lo_pos + kt_token(P, lo);
                            p.hi[i] = hi < lo ? -1 : walk.view.lo_pos + kt_token(P, hi);
                        }
                        p.rows = walk.rows; p.head = walk.head; p.b = walk.b; p.index = walk.index; p.row0 = row0;
                    }
                    kv_bar_arrive(&piece_full[n % KT_PIECES]);
                }
                __syncwarp();
            }
            if (lane == 0) kv_cuts(P.work)[blockIdx.x] = cut;
        } else if (warp >= KT_HELP_WARP) {
            const int r = tid & 127;
            if constexpr (I8) {
                // ================= bytes to 16-bit numbers: a position a thread ==================================================
                uint32_t rs = 0, rph = 0, slot = 0, ph = 1;
                for (uint32_t n = 0;; n++) {
                    const KtPiece& walk = piece_at(n);
                    if (!is_one(walk)) break;
#pragma unroll 1
                    for (int left = 2 * (walk.t1 - walk.t0), kv = 0; left > 0; left--, kv ^= 1) {
                        wait(&raw_full[rs], rph);
                        wait(&empty[slot], ph);
                        __syncwarp();
                        const uint8_t* from = raw + rs * S::RAW;
                        uint8_t* to = ring + slot * S::SLOT;
                        auto turn = [&](auto bf) {
                            constexpr bool BF = decltype(bf)::value;
#pragma unroll
                            for (int c = 0; c < HD / 16; c++) {
                                const uint4 w = *reinterpret_cast<const uint4*>(from + (HD == 64 ? kt_offset64(r, c) : kt_offset(r, c)));
                                *reinterpret_cast<uint4*>(to + kt_offset(r, 2 * c)) = make_uint4(widen<BF, 0x10>(w.x), widen<BF, 0x32>(w.x), widen<BF, 0x10>(w.y), widen<BF, 0x32>(w.y));
                                *reinterpret_cast<uint4*>(to + kt_offset(r, 2 * c + 1)) = make_uint4(widen<BF, 0x10>(w.z), widen<BF, 0x32>(w.z), widen<BF, 0x10>(w.w), widen<BF, 0x32>(w.w));
                            }
                        };
                        if (kv || QB) turn(std::true_type());
                        else turn(std::false_type());
                        fence_async();
                        __syncwarp();
                        if (lane == 0) { kv_bar_arrive(&raw_empty[rs]); kv_bar_arrive(&full[slot]); }
                        if (++rs == (uint32_t)S::RAWS) { rs = 0; rph ^= 1u; }
                        if (++slot == (uint32_t)S::SLOTS) { slot = 0; ph ^= 1u; }
                    }
                    give_back(n);
                }
            } else {
                // ================= V tiles that some row sees in part: only finite values stay ===================================
                // (they see every slot of the ring and give it back with the products: neither can be a round ahead of the other)
                uint32_t slot = 0, ph = 0;
                auto step = [&]() {
                    __syncwarp();
                    if (lane == 0) kv_bar_arrive(&empty[slot]);
                    if (++slot == S::SLOTS) { slot = 0; ph ^= 1u; }
                };
                for (uint32_t n = 0;; n++) {
                    const KtPiece& walk = piece_at(n);
                    if (!is_one(walk)) break;
                    const KvView<KT_TILE> see[2] = {walk.part(0), walk.part(1)};
                    const int t0 = walk.t0, t1 = walk.t1;
                    if (tid == KT_HELP_WARP * 32) odd[(walk.index + 4) & 7] = 0;  // (a piece to come)
#pragma unroll 1
                    for (int t = t0; t < t1; t++) {
                        const int base = walk.base(t);
                        wait(&full[slot], ph);
                        step();
                        bool part = false;
#pragma unroll
                        for (int i = 0; i < 2; i++) part |= see[i].any(base, KT_TILE, P.window, P.sinks) && !see[i].whole(base, P.window, P.sinks);
                        wait(&full[slot], ph);
                        if (part) {
                            uint8_t* v = ring + slot * S::SLOT;
                            uint32_t found = 0;
#pragma unroll
                            for (int c = 0; c < HD / 8; c++) {
                                uint4* at = reinterpret_cast<uint4*>(v + kt_offset(r, c));
                                uint4 w = *at;
                                if (not_finite<QB>(w.x) | not_finite<QB>(w.y) | not_finite<QB>(w.z) | not_finite<QB>(w.w)) {
                                    found = 1;
                                    *at = make_uint4(only_finite<QB>(w.x), only_finite<QB>(w.y), only_finite<QB>(w.z), only_finite<QB>(w.w));
                                }
                            }
                            if (found) { odd[walk.index & 7] = 1; __threadfence_block(); }
                            fence_async();
                            __syncwarp();
                            if (lane == 0) kv_bar_arrive(&ready[slot]);
                        }
                        step();
                    }
                    give_back(n);
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    if (failed) {  // copies may still be on their way into this CTA's shared memory: a bounded time to land
        uint64_t* bar = tid < S::SLOTS ? &full[tid] : tid < S::SLOTS + S::RAWS ? &raw_full[tid - S::SLOTS] : tid < S::SLOTS + S::RAWS + KT_SCALE_SLOTS && I8 ? &sc_full[tid - S::SLOTS - S::RAWS] : nullptr;
        if (bar)
            for (int i = 0; i < 64; i++) { kv_bar_try(bar, 0); kv_bar_try(bar, 1); }
        if (tid == 0) kv_report(P.step.status, L2_KV_TIMEOUT);
    }
    if (warp == KT_MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Adds the pieces of the block of rows that begins in CTA x of the launch in front and goes on in the next.  A thread has a row and eight columns; the lanes of a
// warp have rows side by side, as the pieces lie; blockIdx.z has 64 columns (one sequence of 5 x 8 rows, 18 pieces a kv head: 24.2 -> 22.5 us).
template <int HD>
__global__ void __launch_bounds__(256) kv_tc_combine_kernel(const __grid_constant__ KvAttendParams P, const int ctas) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const KvCut cut = kv_cuts(P.work)[blockIdx.x];
    const int r = blockIdx.y * 32 + (threadIdx.x & 31);
    if (!cut.pieces || r >= cut.rows) return;
    auto piece = [&](int i) { return kv_part(P.work, ctas, KT_ROWS, HD, blockIdx.x + i, i == 0 ? cut.slot : 0); };
    float top = -INFINITY, sum = 0.0f;
#pragma unroll 8
    for (int i = 0; i < cut.pieces; i++) top = fmaxf(top, piece(i)[KT_ROWS * HD + 2 * r]);
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll 8
    for (int i = 0; i < cut.pieces; i++) {
        const float2 ml = *reinterpret_cast<const float2*>(piece(i) + KT_ROWS * HD + 2 * r);
        sum += KvScale(ml.x - ref)(ml.y);
    }
    const int tok = kt_token(P, r), pos = cut.lo_pos + tok;
    const int64_t e = (cut.row0 + tok) * P.out.row_stride + (int64_t)(cut.head * P.group + r - tok * P.group) * P.out.head_stride;
    const float inv = 1.0f / sum;
    const int d = 8 * (threadIdx.x >> 5) + 64 * blockIdx.z;
    float y[8] = {};
#pragma unroll 4
    for (int i = 0; i < cut.pieces; i++) {
        const float* p = piece(i);
        const KvScale f(p[KT_ROWS * HD + 2 * r] - ref);
        const float4 a = *reinterpret_cast<const float4*>(p + (d / 4 * KT_ROWS + r) * 4), b = *reinterpret_cast<const float4*>(p + ((d / 4 + 1) * KT_ROWS + r) * 4);
        y[0] += f(a.x); y[1] += f(a.y); y[2] += f(a.z); y[3] += f(a.w);
        y[4] += f(b.x); y[5] += f(b.y); y[6] += f(b.z); y[7] += f(b.w);
    }
#pragma unroll
    for (int x = 0; x < 8; x++) y[x] = pos < 0 ? 0.0f : y[x] * inv;
    if (P.out.type == L2_F32) kv_store8(reinterpret_cast<float*>(P.out.data) + e + d, y);
    else if (P.out.type == L2_F16) kv_store8(reinterpret_cast<__half*>(P.out.data) + e + d, y);
    else kv_store8(reinterpret_cast<__nv_bfloat16*>(P.out.data) + e + d, y);
}

// CTAs of a launch: one an SM, no more than the line can be long (which is KT_SETUP + 1 or more)
int kt_grid(const KvStep& s, const KvPool& p, int group, int sms) {
    const int64_t blocks = s.n_rows / (KT_ROWS / group) + s.n_seqs;
    return (int)std::min<int64_t>(sms, blocks * p.n_kv_heads * ((((int64_t)s.width << p.page_shift) + KT_TILE - 1) / KT_TILE + 1 + KT_SETUP));
}

bool kt_needed(const KvStep& s, int group) { return (int64_t)s.max_rows * group > kv_rows_limit(s, group); }

}  // namespace

size_t kv_tc_work(const KvStep& s, const KvPool& p, int group, int head_size, int sms) {
    if (!kt_needed(s, group)) return 0;
    const int grid = kt_grid(s, p, group, sms);
    return kv_cut_bytes(grid) + (size_t)grid * 2 * KT_ROWS * (head_size + 2) * sizeof(float);
}

cudaError_t launch_kv_tc(const KvAttendParams& p, int type, int head_size, int sms, cudaStream_t st) {
    if (!kt_needed(p.step, p.group)) return cudaSuccess;
    const int lim = kv_rows_limit(p.step, p.group), grid = kt_grid(p.step, p.pool, p.group, sms);
    CUtensorMap mk, mv;
    if (cudaError_t e = kv_map(&mk, p.pool, p.pool.k, type, head_size, KT_TILE)) return e;
    if (cudaError_t e = kv_map(&mv, p.pool, p.pool.v, type, head_size, KT_TILE)) return e;
    auto go = [&](auto t, auto b, auto h) {
        constexpr int T = decltype(t)::value, HD = decltype(h)::value;
        auto kernel = kv_tc_kernel<T, decltype(b)::value, HD>;
        static KvOnce once;
        if (cudaError_t x = once.shared_memory(reinterpret_cast<const void*>(kernel), KtShape<T, HD>::SMEM)) return x;
        return kv_launch(kernel, dim3(grid), KT_THREADS, KtShape<T, HD>::SMEM, st, p, lim, mk, mv);
    };
    auto by_hd = [&](auto t, auto b) { return head_size == 128 ? go(t, b, std::integral_constant<int, 128>()) : go(t, b, std::integral_constant<int, 64>()); };
    const bool qb = p.q.type == L2_BF16;
    const cudaError_t e = type == L2_F16 ? by_hd(std::integral_constant<int, L2_F16>(), std::false_type())
                        : type == L2_BF16 ? by_hd(std::integral_constant<int, L2_BF16>(), std::true_type())
                        : qb ? by_hd(std::integral_constant<int, L2_I8>(), std::true_type()) : by_hd(std::integral_constant<int, L2_I8>(), std::false_type());
    if (e != cudaSuccess) return e;
    auto combine = head_size == 128 ? kv_tc_combine_kernel<128> : kv_tc_combine_kernel<64>;
    return kv_launch(combine, dim3(grid - 1, KT_ROWS / 32, head_size / 64), 256, 0, st, p, grid);
}

}  // namespace l2
