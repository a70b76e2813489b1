// l2_kv_attend for sequences with few rows (tokens x query heads of a kv head: single tokens, drafted tokens).
//
// For one kv head of one sequence, with the rows' queries Q (8 NT rows at most), keys K and values V:
//   S^T = K Q^T,  P^T = 2^(scale S^T - m),  O^T += V^T P^T,  l += sum P,   out = O / l
// m is a row's maximum of some earlier tile, raised (O and l scaled) only when a score exceeds it by more than 2^8.  The products are taken transposed: positions (S^T)
// and head elements (O^T) are the 16 rows of an mma.sync, the few query rows its 8 columns, so that one row wastes 7 of 8, not 15 of 16.
//
// What bounds it: reading the cache, once, by TMA, while the matrix work of a tile hides behind the copies of the next.  bf16, 8 sequences of 40 heads, 4096 positions each
// (672 MB): 114 us, 5.9 TB/s.  int8, 64 sequences of 8 kv heads with 8 query heads (565 MB): 115 to 123 us, 4.6 to 4.9 TB/s, for most of the time bound by the instructions that
// widen V (173 us while a compiler made two instructions of each of their logic operations, 194 with tiles of 64 positions).
//
// Work.  The tiles of all (sequence, kv head) pairs form one line, cut evenly over the CTAs whatever the lengths are, with room in front of every pair for what it costs
// besides its tiles (134 -> 119 us for that int8 step); a pair that a cut goes through leaves a partial (m, l, O) in each piece, which kv_rows_combine_kernel adds in
// order.  The cuts are found on the device: the host does not know the lengths.
//
// Roles: warps 0-3 take 16 or 32 positions of a tile each, with a softmax of their own, and meet at the end of a piece; warp 4 fills a ring of
// tiles with TMA copies, one a page run (and the scales of an int8 cache, 16 bytes a lane).
//
// An int8 cache is multiplied as it is stored: K as q's type and V as bf16, both exact; the scale of a position is applied to its score and to
// its probability.  (The probabilities times scales are rounded to bf16 even where q is f16: they can leave f16's range.)
// Up to eight rows: K goes into integer products (s8) as it is, and a row of Q as four signed digits of 8 bits, 2^30 for the power of two above its largest
// element.  Only where they hold every element of all rows exactly (f16: always below 64): beside a large element that K has no part in, what a small one
// loses would decide.  Else K is widened for these rows as for more of them.  (64 sequences, 8 kv heads: 115 us; 122 with K always widened; 116 with three
// digits, which fail to hold one piece in six of normally distributed bf16, 112 with three and the loss.)
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kernels.cuh"
#include "paged_device.cuh"
#include "paged_attend.h"

namespace l2 {

namespace {

constexpr int KR_WARPS = 4, KR_THREADS = (KR_WARPS + 1) * 32, KR_MAX_STAGES = 12;
// What a pair costs besides its tiles, in tiles.  1 or 4 instead, steps of 40 to 64 sequences: int8, 8 rows a kv head 1.5 % slower and up to 1.5 % slower (heads of 64: 3 %, none);
// 16 rows a kv head, int8 5 % slower and 7 % faster, bf16 5 % slower and 1 % faster; bf16 with heads of 64 no difference.
constexpr int KR_SETUP = 2;
constexpr int KR_JOIN = 2;  // CTAs that add the pieces of a pair (with 4 or 8, a step of 64 sequences takes 2 or 5 us longer: CTAs without work)
constexpr int KR_RAISE = 8;  // powers of two that a score may exceed the running maximum by before that is raised
constexpr int KR_DIGITS = 4;  // of Q against int8 K
constexpr int KR_SMEM = 111 * 1024;  // of a CTA: two on an SM, with what is static and reserved

// A variant: 16 KB of K and as much of V in a tile, 64 or 128 positions, of which a warp has 16 or 32 (an int8 cache in tiles of 64 was bound by the
// chain of a warp's step, 2000 clocks whatever the bytes).
// Shared memory: Q and the ring; the warps' results meet in the slot of a piece's last tile.
template <int CT, int HD, int NT>
struct KrShape {
    static constexpr bool I8 = CT == L2_I8;
    static constexpr int ROWS = 8 * NT, ROW_BYTES = HD * (I8 ? 1 : 2);
    static constexpr int TILE = ROW_BYTES == 256 ? 64 : 128, PER_WARP = TILE / KR_WARPS, MB = PER_WARP / 16;
    static constexpr int DIGITS = I8 && NT == 1 ? KR_DIGITS : 0;                // of Q, where it can be in digits
    static constexpr int Q_PITCH = 2 * HD + 16, D_PITCH = HD + 16, D_PLANE = ROWS * D_PITCH;  // bytes between rows of Q, of a digit (no bank conflicts); of a digit's plane
    static constexpr int KV_BYTES = TILE * ROW_BYTES;                           // K or V of a tile
    static constexpr int SCALE_BYTES = I8 ? TILE * 4 : 0;
    static constexpr int STAGE = (2 * (KV_BYTES + SCALE_BYTES) + 1023) / 1024 * 1024;
    static constexpr int FIXED = 1024 + ROWS * Q_PITCH + DIGITS * D_PLANE;
    static constexpr int STAGES = (KR_SMEM - FIXED) / STAGE < KR_MAX_STAGES ? (KR_SMEM - FIXED) / STAGE : KR_MAX_STAGES;
    static constexpr int SMEM = FIXED + STAGES * STAGE;
    static_assert(STAGES >= 2 && KR_WARPS * ROWS * HD * 4 <= STAGE, "ring");
};

// Where 16-byte chunk c16 of row r of a tile is: rows of 128 bytes (two halves of a tile one after the other) or 64, as the TMA swizzles them.
template <int ROW_BYTES, int TILE>
__device__ __forceinline__ uint32_t kr_offset(int r, int c16) {
    if constexpr (ROW_BYTES == 64) return r * 64 + ((c16 ^ ((r >> 1) & 3)) << 4);
    else return (c16 >> 3) * (TILE * 128) + r * 128 + (((c16 & 7) ^ (r & 7)) << 4);
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float from_int(int x) { return __int_as_float(x + 0x4b400000) - 12582912.0f; }  // |x| < 2^22, exact
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The line of tiles: sequence by sequence, kv head by kv head, tile by tile.
template <int TILE>
struct KrSeq {
    KvSeq s;
    KvView<TILE> view;
    int rows;  // tokens x group, 0: not this kernel's
    __device__ __forceinline__ KrSeq() {}
    __device__ __forceinline__ KrSeq(const KvAttendParams& P, int lim, int b) {
        s = kv_seq(P.step, P.pool.page_shift, b);
        const int64_t n = (int64_t)s.n * P.group;
        rows = n <= lim ? (int)n : 0;
        view = KvView<TILE>(s.kv - s.n, s.kv - 1, P.window, P.sinks);
    }
};
template <int TILE>
__device__ __forceinline__ int64_t kr_length(const KvAttendParams& P, int lim, int b) {
    if (b >= P.step.n_seqs) return 0;
    const KrSeq<TILE> q(P, lim, b);
    return q.rows ? (int64_t)(q.view.tiles + KR_SETUP) * P.pool.n_kv_heads : 0;
}

// A CTA's piece of the line, one (sequence, kv head) at a time.
template <int TILE>
struct KrWalk {
    int64_t w, w1, start, per;
    int b;
    KrSeq<TILE> q;
    int head, t0, t1;
    bool first;  // the piece is the CTA's first
    __device__ __forceinline__ KrWalk(const KvAttendParams& P, int lim, const KvSpot& spot) {
        per = spot.per;
        w = per * blockIdx.x;
        w1 = min(spot.total, w + per);
        start = spot.start; b = spot.b;
        first = true;
        t0 = -1;
        if (w < w1) q = KrSeq<TILE>(P, lim, b);
    }
    __device__ __forceinline__ bool next(const KvAttendParams& P, int lim) {
        if (t0 >= 0) first = false;
#pragma unroll 1
        while (w < w1) {
            int64_t length = q.rows ? (int64_t)(q.view.tiles + KR_SETUP) * P.pool.n_kv_heads : 0;
            while (w >= start + length) {
                start += length;
                q = KrSeq<TILE>(P, lim, ++b);
                length = q.rows ? (int64_t)(q.view.tiles + KR_SETUP) * P.pool.n_kv_heads : 0;
            }
            const int64_t in = w - start;
            const int place = q.view.tiles + KR_SETUP;  // of a pair on the line, whose first KR_SETUP are no tiles
            head = (int)kv_quotient(in, place);
            const int at = (int)(in - (int64_t)head * place), end = (int)min((int64_t)place, at + (w1 - w));
            w += end - at;
            if (end <= KR_SETUP) continue;  // (the pair's tiles begin in the next CTA)
            t0 = max(0, at - KR_SETUP);
            t1 = end - KR_SETUP;
            return true;
        }
        return false;
    }
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == q.view.tiles; }
};

// CT: cache type; QB: q is bf16, else f16
// (Eight rows: no spills.  Sixteen: int8 with heads of 128 spills 236 bytes, 16 bits 24.)
template <int CT, bool QB, int HD, int NT>
__global__ void __launch_bounds__(KR_THREADS, 2) kv_rows_kernel(const __grid_constant__ KvAttendParams P, const int lim, const __grid_constant__ CUtensorMap map_k,
                                                               const __grid_constant__ CUtensorMap map_v) {
    using S = KrShape<CT, HD, NT>;
    constexpr bool I8 = S::I8, PB = I8 || QB;       // probabilities and V in bf16
    constexpr int KS = HD / 16, MT = HD / 16, RB = S::ROW_BYTES, TILE = S::TILE, MB = S::MB;
    constexpr float BIAS = PB ? 24.0f : 7.0f;       // probabilities carry a factor of 2^BIAS, so that small ones are normal numbers; f16 at most 2^(7 + KR_RAISE)
    extern __shared__ __align__(1024) uint8_t kr_smem[];
    __shared__ __align__(8) uint64_t full[S::STAGES], empty[S::STAGES];
    __shared__ int64_t scratch[KR_THREADS / 32 + 2];
    __shared__ float meet_ml[KR_WARPS][S::ROWS][2];
    __shared__ float q_factor[S::ROWS];  // of a row's digits
    __shared__ volatile int failed;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(kr_smem) + 1023) & ~(uintptr_t)1023);
    uint8_t* sq = ring + S::STAGES * S::STAGE;
    uint8_t* sd = sq + S::ROWS * S::Q_PITCH;  // the digits
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < S::STAGES; i++) { kv_bar_init(&full[i], I8 ? 33 : 1); kv_bar_init(&empty[i], KR_WARPS); }
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == KR_WARPS && lane < 2) kv_prefetch_map(lane ? &map_v : &map_k);
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (rows, lengths and the cache may come from the kernel in front)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const KvSpot spot = kv_locate<KR_THREADS>(P.step.n_seqs, blockIdx.x, gridDim.x, scratch, [&](int b) { return kr_length<TILE>(P, lim, b); });
    __syncthreads();
    KrWalk<TILE> walk(P, lim, spot);
    const KvWait wait{&failed};

    if (warp == KR_WARPS) {
        // ================= copies: lane l brings run l of a tile ==============================================================
        // Pages are looked up for 32 runs at once, and for the next 32 while these are copied: a look-up takes as long as a tile's arithmetic.
        const int R = min(TILE, 1 << P.pool.page_shift), runs = TILE / R, ahead = 32 / runs;
        uint32_t st = 0, ph = 1;
        bool over = false;
        while (!over && walk.next(P, lim)) {
            const KvView<TILE>& view = walk.q.view;
            auto look_up = [&](int t) {  // lane l: run l % runs of tile t + l / runs; n_pages (a copy from there gives zeros) where no row sees it or there is none
                const int mine = t + lane / runs, j = view.base(mine) + lane % runs * R;
                if (mine >= walk.t1 || !view.any(j, R, P.window, P.sinks)) return P.pool.n_pages;
                const int x = kv_page(P.step, P.pool, walk.b, j);
                return x >= 0 ? x : P.pool.n_pages;
            };
            int pages = 0, next = look_up(walk.t0);
            for (int t = walk.t0, k = 0; t < walk.t1; t++, k = k + 1 == ahead ? 0 : k + 1) {
                if (k == 0) { pages = next; next = look_up(t + ahead); }
                const int j = view.base(t), page = __shfl_sync(0xffffffffu, pages, k * runs + lane % runs);
                wait(&empty[st], ph);
                if ((over = wait.over())) break;
                uint8_t* stage = ring + st * S::STAGE;
                if (lane == 0) kv_bar_expect(&full[st], 2 * S::KV_BYTES);
                __syncwarp();
                if (lane < runs) {
                    const int at = (j + lane * R) & ((1 << P.pool.page_shift) - 1);
                    const uint32_t k_to = kv_smem(stage), v_to = k_to + S::KV_BYTES;
#pragma unroll
                    for (int h = 0; h < (RB + 127) / 128; h++) {
                        const uint32_t to = h * (TILE * 128) + lane * R * min(RB, 128);
                        kv_tma4(k_to + to, &map_k, h * 64, at, walk.head, page, &full[st]);
                        kv_tma4(v_to + to, &map_v, h * 64, at, walk.head, page, &full[st]);
                    }
                }
                if constexpr (I8) {  // the scales: four positions a lane, of K and of V
                    const int pos = 4 * lane, of = __shfl_sync(0xffffffffu, pages, k * runs + pos / R);
                    const bool there = of < P.pool.n_pages;
                    const int64_t e = ((int64_t)(there ? of : 0) * P.pool.n_kv_heads + walk.head << P.pool.page_shift) + ((j + pos) & ((1 << P.pool.page_shift) - 1));
                    const uint32_t to = kv_smem(stage + 2 * S::KV_BYTES) + 16 * lane;
                    kv_copy16(to, P.pool.ks + e, there);
                    kv_copy16(to + S::SCALE_BYTES, P.pool.vs + e, there);
                    kv_copy16_arrive(&full[st]);
                }
                if (++st == S::STAGES) { st = 0; ph ^= 1u; }
            }
        }
    } else {
        // ================= matrix work ========================================================================================
        const int c = lane & 3, g8 = lane >> 2;
        uint32_t st = 0, ph = 0;
        // Q of a piece is requested while the results of the piece in front meet.
        constexpr int Q_N = S::ROWS * (HD / 8) / (KR_WARPS * 32) + (S::ROWS * (HD / 8) % (KR_WARPS * 32) != 0);
        uint4 qx[Q_N];
        auto request_q = [&]() {  // (rows beyond the last are zeros)
#pragma unroll
            for (int n = 0; n < Q_N; n++) {
                const int u = tid + n * KR_WARPS * 32, r = u / (HD / 8), ch = u % (HD / 8), tok = r / P.group;
                qx[n] = make_uint4(0, 0, 0, 0);
                if (r < walk.q.rows)
                    qx[n] = *reinterpret_cast<const uint4*>(P.q.data + 2 * ((walk.q.s.row0 + tok) * P.q.row_stride + (int64_t)(walk.head * P.group + r - tok * P.group) * P.q.head_stride + ch * 8));
            }
        };
        bool more = walk.next(P, lim);
        if (more) request_q();
        while (more) {
            const KvView<TILE> view = walk.q.view;
            const int rows = walk.q.rows, G = P.group, t0 = walk.t0, t1 = walk.t1;
            asm volatile("bar.sync 1, 128;" ::: "memory");  // (everybody has read the piece before's)
#pragma unroll
            for (int n = 0; n < Q_N; n++) {
                const int u = tid + n * KR_WARPS * 32, r = u / (HD / 8), ch = u % (HD / 8);
                if (r < S::ROWS) *reinterpret_cast<uint4*>(sq + r * S::Q_PITCH + ch * 16) = qx[n];
            }
            bool digits = false;  // Q is in digits: they hold every element of all rows
            if constexpr (S::DIGITS > 0) {
                const int r = tid / (HD / 8), ch = tid % (HD / 8);
                float x[8], most = 0.0f;
                const uint32_t w[4] = {qx[0].x, qx[0].y, qx[0].z, qx[0].w};
                bool held = true;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    x[k] = QB ? __uint_as_float(k % 2 ? w[k / 2] & 0xffff0000u : w[k / 2] << 16) : __half2float(__ushort_as_half((unsigned short)(w[k / 2] >> (16 * (k % 2)))));
                    held &= fabsf(x[k]) < INFINITY;
                    most = fmaxf(most, fabsf(x[k]));
                }
#pragma unroll
                for (int o = 1; o < HD / 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                constexpr int BITS = 8 * S::DIGITS - 2;
                const int e = max((int)(__float_as_uint(most) >> 23) - 126, BITS - 122);  // most < 2^e; 2^(BITS - e) and its inverse are normal numbers
                const float up = __uint_as_float((uint32_t)(BITS - e + 127) << 23);
                uint32_t plane[S::DIGITS][2] = {};
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float y = x[k] * up;
                    const int whole = __float2int_rn(y);
                    held &= (float)whole == y;
                    constexpr uint32_t HALF = 0x80808080u >> (32 - 8 * S::DIGITS);
                    const uint32_t v = ((uint32_t)whole + HALF) ^ HALF;  // balanced digits
#pragma unroll
                    for (int p = 0; p < S::DIGITS; p++) plane[p][k / 4] |= (v >> (8 * p) & 255u) << (8 * (k % 4));
                }
                if (r < S::ROWS) {
#pragma unroll
                    for (int p = 0; p < S::DIGITS; p++) *reinterpret_cast<uint2*>(sd + p * S::D_PLANE + r * S::D_PITCH + 8 * ch) = make_uint2(plane[p][0], plane[p][1]);
                    if (ch == 0) q_factor[r] = __uint_as_float((uint32_t)(e - BITS + 127) << 23);
                }
                uint32_t all;
                asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.and.pred q, 1, 128, p;\nselp.u32 %0, 1, 0, q;\n}" : "=r"(all) : "r"((uint32_t)held) : "memory");
                digits = __all_sync(0xffffffffu, all);  // (a vote's result is uniform)
            } else {
                asm volatile("bar.sync 1, 128;" ::: "memory");
            }
            // Q^T as the second factor: columns 8 nt .., two words for each 16 elements (digits: for each 32, of each digit)
            constexpr int Q_WORDS = S::DIGITS * HD / 32 > NT * KS ? S::DIGITS * HD / 32 : NT * KS;
            uint32_t qr[Q_WORDS][2];
            float by_row[2] = {1.0f, 1.0f};
            if (digits) {
#pragma unroll
                for (int a = 0; a < S::DIGITS; a++)
#pragma unroll
                    for (int c2 = 0; c2 < HD / 32; c2++) {
                        const uint8_t* p = sd + a * S::D_PLANE + g8 * S::D_PITCH + c2 * 32 + 4 * c;
                        qr[a * (HD / 32) + c2][0] = *reinterpret_cast<const uint32_t*>(p);
                        qr[a * (HD / 32) + c2][1] = *reinterpret_cast<const uint32_t*>(p + 16);
                    }
                by_row[0] = q_factor[2 * c]; by_row[1] = q_factor[2 * c + 1];
            } else {
#pragma unroll
                for (int a = 0; a < NT; a++)
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) {
                        const uint8_t* p = sq + (8 * a + g8) * S::Q_PITCH + ks * 32;
                        if constexpr (I8) { const uint2 x = *reinterpret_cast<const uint2*>(p + 8 * c); qr[a * KS + ks][0] = x.x; qr[a * KS + ks][1] = x.y; }
                        else { qr[a * KS + ks][0] = *reinterpret_cast<const uint32_t*>(p + 4 * c); qr[a * KS + ks][1] = *reinterpret_cast<const uint32_t*>(p + 16 + 4 * c); }
                    }
            }
            int pos[NT][2];  // positions of this thread's two rows of each eight
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) pos[nt][e] = view.lo_pos + (8 * nt + 2 * c + e) / G;

            float o[MT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                m[nt][0] = m[nt][1] = -INFINITY;
                l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
                for (int mt = 0; mt < MT; mt++) o[mt][nt][0] = o[mt][nt][1] = o[mt][nt][2] = o[mt][nt][3] = 0.0f;
            }
#pragma unroll 1
            for (int t = t0; t < t1; t++) {
                const int base = view.base(t);
                const bool whole = view.whole(base, P.window, P.sinks);
                wait(&full[st], ph);
                __syncwarp();
                const uint8_t* stage = ring + st * S::STAGE;
                const uint32_t k_at = kv_smem(stage), v_at = k_at + S::KV_BYTES;
                // ---- scores of this warp's positions, 16 at a time: rows g8 and g8 + 8, columns 2 c and 2 c + 1
                float s[MB][NT][4];
#pragma unroll
                for (int mb = 0; mb < MB; mb++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) s[mb][nt][0] = s[mb][nt][1] = s[mb][nt][2] = s[mb][nt][3] = 0.0f;
                const int kr = S::PER_WARP * warp + (lane & 15);
                auto by_k = [&](int mb, int ks, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) mma<QB>(s[mb][nt], a0, a1, a2, a3, qr[nt * KS + ks][0], qr[nt * KS + ks][1]);
                };
                if (digits) {
                    constexpr int N = S::DIGITS ? S::DIGITS : 1;
                    int d[MB][N][4] = {};
#pragma unroll
                    for (int c2 = 0; c2 < HD / 32; c2++)
#pragma unroll
                        for (int mb = 0; mb < MB; mb++) {
                            uint32_t a[4];
                            ldsm4(a, k_at + kr_offset<RB, TILE>(kr + 16 * mb, 2 * c2 + (lane >> 4)));
#pragma unroll
                            for (int p = 0; p < N; p++) mma_s8(d[mb][p], a, qr[p * (HD / 32) + c2][0], qr[p * (HD / 32) + c2][1]);
                        }
#pragma unroll
                    for (int mb = 0; mb < MB; mb++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            float x = from_int(d[mb][0][i]);
#pragma unroll
                            for (int p = 1; p < N; p++) x = fmaf(from_int(d[mb][p][i]), (float)(1 << (8 * p)), x);
                            s[mb][0][i] = by_row[i & 1] * x;
                        }
                } else if constexpr (I8) {
#pragma unroll
                    for (int c2 = 0; c2 < KS / 2; c2++)  // 32 elements; of each 16, element 4 c + i is k index 2 c + i (i < 2) or 8 + 2 c + i - 2
#pragma unroll
                        for (int mb = 0; mb < MB; mb++) {
                            uint32_t a[4];
                            ldsm4(a, k_at + kr_offset<RB, TILE>(kr + 16 * mb, 2 * c2 + (lane >> 4)));
                            by_k(mb, 2 * c2, widen<QB, 0x10>(a[0]), widen<QB, 0x10>(a[1]), widen<QB, 0x32>(a[0]), widen<QB, 0x32>(a[1]));
                            by_k(mb, 2 * c2 + 1, widen<QB, 0x10>(a[2]), widen<QB, 0x10>(a[3]), widen<QB, 0x32>(a[2]), widen<QB, 0x32>(a[3]));
                        }
                } else {
#pragma unroll
                    for (int ks = 0; ks < KS; ks++)
#pragma unroll
                        for (int mb = 0; mb < MB; mb++) {
                            uint32_t a[4];
                            ldsm4(a, k_at + kr_offset<RB, TILE>(kr + 16 * mb, 2 * ks + (lane >> 4)));
                            by_k(mb, ks, a[0], a[1], a[2], a[3]);
                        }
                }
                // ---- softmax
                const int j0 = base + S::PER_WARP * warp + g8;  // this thread's positions: j0 + 16 mb, and 8 more
                auto sees = [&](int nt, int mb, int i) { return kv_sees(pos[nt][i & 1], j0 + 16 * mb + 8 * (i >> 1), P.window, P.sinks); };
                float v_scale[MB][2], most[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) most[nt][0] = most[nt][1] = -INFINITY;
#pragma unroll
                for (int mb = 0; mb < MB; mb++) {
                    float f0 = P.scale_log2, f1 = P.scale_log2;
                    if constexpr (I8) {
                        const float* sc = reinterpret_cast<const float*>(stage + 2 * S::KV_BYTES) + S::PER_WARP * warp + 16 * mb + g8;
                        f0 *= sc[0]; f1 *= sc[8];
                        v_scale[mb][0] = sc[TILE]; v_scale[mb][1] = sc[TILE + 8];
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        s[mb][nt][0] *= f0; s[mb][nt][1] *= f0; s[mb][nt][2] *= f1; s[mb][nt][3] *= f1;
                        if (!whole) {
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                if (!sees(nt, mb, i)) s[mb][nt][i] = -INFINITY;
                        }
                        most[nt][0] = fmaxf(most[nt][0], fmaxf(s[mb][nt][0], s[mb][nt][2]));
                        most[nt][1] = fmaxf(most[nt][1], fmaxf(s[mb][nt][1], s[mb][nt][3]));
                    }
                }
                bool raise = false;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) raise |= most[nt][0] - BIAS > m[nt][0] + KR_RAISE || most[nt][1] - BIAS > m[nt][1] + KR_RAISE;
                if (__any_sync(0xffffffffu, raise)) {  // seldom: only then do the lanes of a row need their common maximum
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float x = most[nt][e] - BIAS;
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                            const float m1 = x > m[nt][e] + KR_RAISE ? x : m[nt][e];  // (a row's result does not depend on the others)
                            const KvScale f(m1 == -INFINITY ? 0.0f : m[nt][e] - m1);
                            m[nt][e] = m1;
                            l[nt][e] = f(l[nt][e]);
#pragma unroll
                            for (int mt = 0; mt < MT; mt++) { o[mt][nt][e] = f(o[mt][nt][e]); o[mt][nt][e + 2] = f(o[mt][nt][e + 2]); }
                        }
                }
                uint32_t pb[MB][NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const float ref[2] = {m[nt][0] == -INFINITY ? 0.0f : m[nt][0], m[nt][1] == -INFINITY ? 0.0f : m[nt][1]};
#pragma unroll
                    for (int mb = 0; mb < MB; mb++) {
                        float p[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            p[i] = kv_exp2(s[mb][nt][i] - ref[i & 1]);
                            l[nt][i & 1] += p[i];
                            if constexpr (I8) p[i] = !whole && !sees(nt, mb, i) ? 0.0f : p[i] * v_scale[mb][i >> 1];
                        }
                        pb[mb][nt][0] = transpose8(pack16<PB>(p[0], p[1]));
                        pb[mb][nt][1] = transpose8(pack16<PB>(p[2], p[3]));
                    }
                }
                // ---- O^T += V^T P^T
                const int vr = S::PER_WARP * warp + (lane & 7) + 8 * (lane >> 4);
#pragma unroll
                for (int mb = 0; mb < MB; mb++) {
                    if constexpr (I8) {
#pragma unroll
                        for (int m2 = 0; m2 < (MT + 1) / 2; m2++) {  // 32 elements; row i of a product is element 2 i, row 8 + i element 2 i + 1
                            uint32_t a[4];
                            ldsm4_t(a, v_at + kr_offset<RB, TILE>(vr + 16 * mb, 2 * m2 + ((lane >> 3) & 1)));
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const uint32_t x0 = widen<true, 0x20>(a[h]), x1 = widen<true, 0x31>(a[h]), x2 = widen<true, 0x20>(a[h + 2]), x3 = widen<true, 0x31>(a[h + 2]);
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) mma<true>(o[2 * m2 + h][nt], x0, x1, x2, x3, pb[mb][nt][0], pb[mb][nt][1]);
                            }
                        }
                    } else {
                        bool odd = false;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            uint32_t a[4];
                            ldsm4_t(a, v_at + kr_offset<RB, TILE>(vr + 16 * mb, 2 * mt + ((lane >> 3) & 1)));
                            if (!whole) {  // 0 x NaN is NaN: a value that some row does not see may only be multiplied where it is finite
                                if (__any_sync(0xffffffffu, not_finite<PB>(a[0]) | not_finite<PB>(a[1]) | not_finite<PB>(a[2]) | not_finite<PB>(a[3]))) {
                                    odd = true;
#pragma unroll
                                    for (int i = 0; i < 4; i++) a[i] = only_finite<PB>(a[i]);
                                }
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) mma<PB>(o[mt][nt], a[0], a[1], a[2], a[3], pb[mb][nt][0], pb[mb][nt][1]);
                        }
                        if (odd) {  // rare: the values that are not finite, one by one, to the rows that see them
#pragma unroll 1
                            for (int i = 0; i < 16; i++) {
                                const int r = S::PER_WARP * warp + 16 * mb + i;
#pragma unroll
                                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                                    for (int h = 0; h < 2; h++) {
                                        const uint16_t bits = *reinterpret_cast<const uint16_t*>(stage + S::KV_BYTES + kr_offset<RB, TILE>(r, 2 * mt + h) + 2 * g8);
                                        if (not_finite<PB>(bits)) {
                                            const float x = PB ? __uint_as_float((uint32_t)bits << 16) : __half2float(__ushort_as_half(bits));
#pragma unroll
                                            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                                                for (int e = 0; e < 2; e++)
                                                    if (kv_sees(pos[nt][e], base + r, P.window, P.sinks)) o[mt][nt][2 * h + e] += x;
                                        }
                                    }
                            }
                        }
                    }
                }
                if (t + 1 < t1) {  // (the last tile's slot is kept for the meeting)
                    __syncwarp();
                    if (lane == 0) kv_bar_arrive(&empty[st]);
                    if (++st == S::STAGES) { st = 0; ph ^= 1u; }
                }
            }
            const int head = walk.head;
            const int64_t row0 = walk.q.s.row0;
            const bool done = walk.whole();
            float* part = kv_part(P.work, gridDim.x, S::ROWS, HD, blockIdx.x, walk.first ? 0 : 1);
            if (tid == 0) {  // what the kernel behind this one has to know of the CTA's last piece
                KvCut cut{0, 0, 0, 0, 0, 0, 0};
                if (t0 == 0 && !done) cut = KvCut{(int)kv_quotient(walk.w - t1 + view.tiles - 1, walk.per) - (int)blockIdx.x + 1, walk.first ? 0 : 1, rows, head, row0, view.lo_pos, 0};
                kv_cuts(P.work)[blockIdx.x] = cut;
            }
            more = walk.next(P, lim);
            if (more) request_q();
            // ---- the four warps' results meet: a common maximum, then each warp adds a quarter of the elements, in the order of the warps
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float x = l[nt][e];
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    if (g8 == 0) { meet_ml[warp][8 * nt + 2 * c + e][0] = m[nt][e]; meet_ml[warp][8 * nt + 2 * c + e][1] = x; }
                }
            asm volatile("bar.sync 1, 128;" ::: "memory");  // (and everybody is done with the last tile)
            float4* meet = reinterpret_cast<float4*>(ring + st * S::STAGE);  // [warp][product][lane]
            float lsum[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int r = 8 * nt + 2 * c + e;
                    float top = -INFINITY;
#pragma unroll
                    for (int w = 0; w < KR_WARPS; w++) top = fmaxf(top, meet_ml[w][r][0]);
                    const float ref = top == -INFINITY ? 0.0f : top;
                    lsum[nt][e] = 0.0f;
#pragma unroll
                    for (int w = 0; w < KR_WARPS; w++) lsum[nt][e] += KvScale(meet_ml[w][r][0] - ref)(meet_ml[w][r][1]);
                    const KvScale f(m[nt][e] - ref);
                    m[nt][e] = top;
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) { o[mt][nt][e] = f(o[mt][nt][e]); o[mt][nt][e + 2] = f(o[mt][nt][e + 2]); }
                }
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) meet[(warp * MT * NT + mt * NT + nt) * 32 + lane] = make_float4(o[mt][nt][0], o[mt][nt][1], o[mt][nt][2], o[mt][nt][3]);
            asm volatile("bar.sync 1, 128;" ::: "memory");
            constexpr int SHARE = MT / KR_WARPS;  // products of a warp
#pragma unroll
            for (int x = 0; x < SHARE; x++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const int mt = SHARE * warp + x;
                    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int w = 0; w < KR_WARPS; w++) {
                        const float4 z = meet[(w * MT * NT + mt * NT + nt) * 32 + lane];
                        y[0] += z.x; y[1] += z.y; y[2] += z.z; y[3] += z.w;
                    }
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int r = 8 * nt + 2 * c + e;
                        if (r >= rows) continue;
                        const int tok = r / G;
                        const int64_t at = (row0 + tok) * P.out.row_stride + (int64_t)(head * G + r - tok * G) * P.out.head_stride;
                        const float inv = 1.0f / lsum[nt][e];
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int d = I8 ? 16 * mt + 2 * g8 + h : 16 * mt + 8 * h + g8;
                            if (done) kv_store1(P.out, at + d, pos[nt][e] < 0 ? 0.0f : y[2 * h + e] * inv);
                            else part[r * HD + d] = y[2 * h + e];
                        }
                        if (!done && warp == 0 && x == 0 && g8 == 0) *reinterpret_cast<float2*>(part + S::ROWS * HD + 2 * r) = make_float2(m[nt][e], lsum[nt][e]);
                    }
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (the slot goes back to the copies)
            __syncwarp();
            if (lane == 0) kv_bar_arrive(&empty[st]);
            if (++st == S::STAGES) { st = 0; ph ^= 1u; }
        }
        if (tid == 0 && walk.t0 < 0) kv_cuts(P.work)[blockIdx.x].pieces = 0;  // (a CTA without work)
    }
    __syncthreads();
    if (failed) {  // copies may still be on their way into this CTA's shared memory: a bounded time to land
        if (tid < S::STAGES)
            for (int i = 0; i < 64; i++) { kv_bar_try(&full[tid], 0); kv_bar_try(&full[tid], 1); }
        if (tid == 0) kv_report(P.step.status, L2_KV_TIMEOUT);
    }
}

// Adds the pieces of the pair that begins in CTA x of the launch in front and goes on in the next.
// HD / 4 threads for a row; with few rows the others take pieces of the same row, and meet in order.  The rows go over KR_JOIN CTAs.
// One sequence of 60,000 positions and 8 kv heads (int8, 37 pieces a pair): attention 37 us; 46 with one CTA a pair and each thread walking all maxima and sums.
template <int HD>
__global__ void __launch_bounds__(256) kv_rows_combine_kernel(const __grid_constant__ KvAttendParams P, const int ctas, const int part_rows) {
    constexpr int LANES = HD / 4, SLOTS = 256 / LANES;
    __shared__ float4 sums[256];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const KvCut cut = kv_cuts(P.work)[blockIdx.x];
    if (!cut.pieces) return;
    auto piece = [&](int i) { return kv_part(P.work, ctas, part_rows, HD, blockIdx.x + i, i == 0 ? cut.slot : 0); };
    int width = 1;  // rows side by side
    while (width * (int)gridDim.y < cut.rows && width < SLOTS) width <<= 1;
    const int share = SLOTS / width, slot = threadIdx.x / LANES, d = 4 * (threadIdx.x % LANES), mine = slot / width;
    for (int r0 = blockIdx.y * width; r0 < cut.rows; r0 += gridDim.y * width) {
        const int r = r0 + slot % width;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.0f;
        const bool on = r < cut.rows;
        // the common maximum and the sum: piece i by thread i % LANES of the row
        const int ml = part_rows * HD + 2 * r;
        float top = -INFINITY;
        for (int i = threadIdx.x % LANES; i < cut.pieces; i += LANES) if (on) top = fmaxf(top, piece(i)[ml]);
#pragma unroll
        for (int x = 1; x < LANES; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float ref = top == -INFINITY ? 0.0f : top;
        for (int i = threadIdx.x % LANES; i < cut.pieces; i += LANES) if (on) sum += KvScale(piece(i)[ml] - ref)(piece(i)[ml + 1]);
#pragma unroll
        for (int x = 1; x < LANES; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        if (on) {
#pragma unroll 8
            for (int i = mine; i < cut.pieces; i += share) {
                const float* p = piece(i);
                const KvScale f(p[ml] - ref);
                const float4 x = *reinterpret_cast<const float4*>(p + r * HD + d);
                acc.x += f(x.x); acc.y += f(x.y); acc.z += f(x.z); acc.w += f(x.w);
            }
        }
        if (share > 1) {
            sums[threadIdx.x] = acc;
            __syncthreads();
            for (int i = 1; i < share && mine == 0; i++) {
                const float4 x = sums[threadIdx.x + i * width * LANES];
                acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
            }
            __syncthreads();
        }
        if (on && mine == 0) {
            const int tok = r / P.group, pos = cut.lo_pos + tok;
            const int64_t e = (cut.row0 + tok) * P.out.row_stride + (int64_t)(cut.head * P.group + r - tok * P.group) * P.out.head_stride + d;
            const float inv = 1.0f / sum;
            const float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
            for (int i = 0; i < 4; i++) kv_store1(P.out, e + i, pos < 0 ? 0.0f : y[i]);
        }
    }
}

template <class F>
cudaError_t kr_by_variant(int type, bool qb, int hd, int nt, F f) {
    auto by_nt = [&](auto t, auto b, auto h) {
        return nt == 1 ? f(t, b, h, std::integral_constant<int, 1>()) : f(t, b, h, std::integral_constant<int, 2>());
    };
    auto by_hd = [&](auto t, auto b) { return hd == 128 ? by_nt(t, b, std::integral_constant<int, 128>()) : by_nt(t, b, std::integral_constant<int, 64>()); };
    if (type == L2_F16) return by_hd(std::integral_constant<int, L2_F16>(), std::false_type());
    if (type == L2_BF16) return by_hd(std::integral_constant<int, L2_BF16>(), std::true_type());
    return qb ? by_hd(std::integral_constant<int, L2_I8>(), std::true_type()) : by_hd(std::integral_constant<int, L2_I8>(), std::false_type());
}

int kr_nt(int lim) { return lim <= 8 ? 1 : 2; }
int kr_tile(int type, int head_size) { return head_size * (type == L2_I8 ? 1 : 2) == 256 ? 64 : 128; }
// CTAs of a launch: two an SM, no more than the line can be long (which is KR_SETUP + 1 or more)
int kr_grid(const KvStep& s, const KvPool& p, int tile, int sms) {
    const int64_t tiles = (int64_t)s.n_seqs * p.n_kv_heads * ((((int64_t)s.width << p.page_shift) + tile - 1) / tile + 1 + KR_SETUP);
    return (int)std::min<int64_t>(2 * sms, tiles);
}

}  // namespace

int kv_rows_limit(const KvStep& s, int group) {
    const int64_t most = (int64_t)s.max_rows * group;
    if (most <= 16) return std::max(1, (int)most);  // (0, a step said to bring no rows: somebody has to look whether that is so)
    return group <= 16 && (int64_t)s.n_seqs * s.max_rows > s.n_rows ? group : 0;
}

size_t kv_rows_work(const KvStep& s, const KvPool& p, int group, int type, int head_size, int sms) {
    const int lim = kv_rows_limit(s, group);
    if (!lim) return 0;
    const int grid = kr_grid(s, p, kr_tile(type, head_size), sms);
    return kv_cut_bytes(grid) + (size_t)grid * 2 * 8 * kr_nt(lim) * (head_size + 2) * sizeof(float);
}

cudaError_t launch_kv_rows(const KvAttendParams& p, int type, int head_size, int sms, cudaStream_t st) {
    const int lim = kv_rows_limit(p.step, p.group);
    if (!lim) return cudaSuccess;
    const int tile = kr_tile(type, head_size);
    CUtensorMap mk, mv;
    if (cudaError_t e = kv_map(&mk, p.pool, p.pool.k, type, head_size, tile)) return e;
    if (cudaError_t e = kv_map(&mv, p.pool, p.pool.v, type, head_size, tile)) return e;
    const int nt = kr_nt(lim), grid = kr_grid(p.step, p.pool, tile, sms);
    cudaError_t e = kr_by_variant(type, p.q.type == L2_BF16, head_size, nt, [&](auto t, auto b, auto h, auto n) {
        constexpr int T = decltype(t)::value, HD = decltype(h)::value, NT = decltype(n)::value;
        auto kernel = kv_rows_kernel<T, decltype(b)::value, HD, NT>;
        static KvOnce once;
        if (cudaError_t x = once.shared_memory(reinterpret_cast<const void*>(kernel), KrShape<T, HD, NT>::SMEM)) return x;
        return kv_launch(kernel, dim3(grid), KR_THREADS, KrShape<T, HD, NT>::SMEM, st, p, lim, mk, mv);
    });
    if (e != cudaSuccess) return e;
    auto combine = head_size == 128 ? kv_rows_combine_kernel<128> : kv_rows_combine_kernel<64>;
    return kv_launch(combine, dim3(grid - 1, KR_JOIN), 256, 0, st, p, grid, 8 * nt);
}

}  // namespace l2
