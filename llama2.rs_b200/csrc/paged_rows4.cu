// l2_kv_attend over a cache in 4 bits for sequences with few rows (tokens x query heads of a kv head: single tokens, drafted tokens).
//
// With u the numbers of 0 .. 15, a pair (scale, zero) for every position of K (s, z) and of V (t, y), and for a row of Q its sum g:
//   score_j = s_j (u_j . q) + z_j g,    out = sum_j (p_j t_j) u_j + (sum_j p_j y_j) for every element alike
// so only the numbers themselves go through the matrix products, exactly, and what belongs to a position is two operations a score.
//
// A number is used as it lies in the word.  f16 holds u 2^-24 as the bits of u, and 16 u 2^-24 as the bits of 16 u: a mask of a word with eight numbers
// gives two elements of a factor, and a shift by 8 and the same masks the others: five instructions for eight elements (eleven, where numbers are made by adding to a
// larger one and taking that off again, or one of 128 that stays in the sums).  Products and sums are f32 and hold 2^-48.  The two kinds of numbers (u and 16 u) have sums of their own in
// the scores and rows of their own in O^T.
// Q is in f16, a row times a power of two that brings its largest element to 2^15 or more, the elements of odd index as a sixteenth (their numbers are 16 u): half of f16's
// smallest step, 2^-25, is 2^-40 of the row's largest for an even element, 2^-36 for an odd one.
// p t h is rounded to f16, with h a power of two a row: it follows the largest p t seen, so that the scales may have any size (2^-60 to 2^90) beside one another.
//
// Work.  A warp has one kv head of a piece of a sequence, in steps of 32 positions.  Four, two or one heads side by side (as many as divide their number) are a CTA's, so that the 64
// bytes that a head has of a position come from memory together with its neighbours'; with fewer heads than warps the warps of a head share the steps, and meet at the end of a
// piece.  The tiles of all (sequence, heads) form one line, cut evenly over the CTAs, with room in front for what a piece costs besides its tiles; what a cut goes through leaves partial
// (m, l, O), which kv_rows4_combine_kernel adds in order.
//
// Copies.  Every warp of products has a warp of copies that brings its positions, 16 bytes a lane, up to three or four steps ahead, across the ends of pieces; the two meet through
// mbarriers only.  64 sequences of 8 kv heads and 64 query heads, up to 8192 positions (292 MB): 80 us.  By the warps of products themselves 84 (a copy waits where memory is busy, and all
// behind it); by TMA, one warp for four, 93, of which the copies alone took 84: it brings a row of 64 bytes every 4.5 clocks, where it could bring one of 128.  What bounds it now: a start of
// some 13 us (place on the line, table, first positions, first step), then copies (alone 66 us with the start) and steps (alone 68 us) that hide each other in part.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kernels.cuh"
#include "paged_attend.h"
#include "paged_device.cuh"

namespace l2 {

namespace {

constexpr int R4_WARPS = 4, R4_THREADS = 2 * 32 * R4_WARPS;  // warps of products, and as many of copies
constexpr int R4_CTAS = 2;   // of an SM
constexpr int R4_SETUP = 3;  // what a piece costs besides its tiles, in tiles (at the size above 2: 1.5 us longer, 5: 1.1)
constexpr int R4_RAISE = 8;  // powers of two that a score may exceed the running maximum by before that is raised
constexpr float R4_BIAS = 24.0f;  // probabilities carry a factor of 2^24

template <int HD, int NT>
struct R4Shape {
    static constexpr int ROWS = 8 * NT, STEP = NT == 1 ? 64 : 32;          // positions of a warp's step
    static constexpr int ROW = HD / 2, KV = STEP * ROW, SLOT = 2 * KV + 2 * STEP * 4;
    static constexpr int O_BYTES = ROWS * HD * 4, MEET = 2 * (O_BYTES + ROWS * 8);  // a warp's results; of two warps
    static constexpr int SLOTS = NT == 1 && HD == 128 ? 3 : 4;
    __host__ __device__ static constexpr int smem(int wph) { return R4_WARPS * SLOTS * SLOT + (wph > 1 ? MEET : 0); }
    static_assert(R4_CTAS * (smem(4) + 2048) <= 228 * 1024, "shared memory");
};

// Heads of a CTA, and the warps of a head.
struct R4Split { int heads, wph; };
__host__ __device__ constexpr R4Split r4_split(int n_kv_heads) { return n_kv_heads % 4 == 0 ? R4Split{4, 1} : n_kv_heads % 2 == 0 ? R4Split{2, 2} : R4Split{1, 4}; }
// The line's tiles: a step of each warp of a head (64 positions where that would be less).
constexpr int r4_least_shift(int wph, int nt) { return nt == 1 ? wph == 1 ? 6 : wph == 2 ? 7 : 8 : wph == 4 ? 7 : 6; }

// Where 16-byte chunk c of row r is: no bank conflicts for eight rows side by side
template <int ROW>
__device__ __forceinline__ uint32_t r4_offset(int r, int c) {
    if constexpr (ROW == 32) return r * 32 + ((c ^ ((r >> 2) & 1)) << 4);
    else return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}
__device__ __forceinline__ void r4_copy(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ int64_t r4_times(int n, int64_t bytes) {  // (n is not negative; two instructions where a product of 64 bits takes more)
    return (int64_t)((uint64_t)(uint32_t)n * (uint32_t)bytes + ((uint64_t)((uint32_t)n * (uint32_t)(bytes >> 32)) << 32));
}
__device__ __forceinline__ void r4_copy_if(uint32_t dst, const void* src, bool there) {  // (zeros where there is nothing to bring)
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// What rows at positions lo .. hi see, in tiles of 2^shift: KvView with a size that is not known before the call.
struct R4View {
    int lo, hi, sink_tiles, first, tiles;
    __device__ __forceinline__ R4View() {}
    __device__ __forceinline__ R4View(int lo_pos, int hi_pos, int window, int sinks, int shift) : lo(lo_pos), hi(hi_pos) {
        const int end = (hi + (1 << shift)) >> shift;
        first = window ? max(0, lo - window + 1) >> shift : 0;
        sink_tiles = (min(sinks, max(0, lo + 1)) + (1 << shift) - 1) >> shift;
        if (sink_tiles >= first) sink_tiles = first = 0;
        tiles = max(1, sink_tiles + end - first);
    }
    __device__ __forceinline__ int base(int t, int shift) const { return (t < sink_tiles ? t : first + t - sink_tiles) << shift; }
    __device__ __forceinline__ bool whole(int base, int n, int window, int sinks) const { return base + n <= lo + 1 && (!window || base > hi - window || base + n <= sinks); }
    __device__ __forceinline__ bool any(int base, int n, int window, int sinks) const { return base <= hi && (!window || base + n > lo - window + 1 || base < sinks); }
};

struct R4Seq {
    KvSeq s;
    R4View view;
    int rows;  // tokens x group, 0: not this kernel's
    __device__ __forceinline__ R4Seq() {}
    __device__ __forceinline__ R4Seq(const KvAttendParams& P, int lim, int shift, int b) {
        s = kv_seq(P.step, P.pool.page_shift, b);
        const int64_t n = (int64_t)s.n * P.group;
        rows = n <= lim ? (int)n : 0;
        view = R4View(s.kv - s.n, s.kv - 1, P.window, P.sinks, shift);
    }
    __device__ __forceinline__ int length(int units) const { return rows ? (view.tiles + R4_SETUP) * units : 0; }  // on the line
};

// A CTA's part of the line, one (sequence, heads) at a time.  (The line is shorter than 2^31: the host takes tiles that are large enough.)
struct R4Walk {
    int w, w1, start, per, b;
    R4Seq q;
    int unit, t0, t1;
    bool first;  // the piece is the CTA's first
    __device__ __forceinline__ R4Walk() {}
    // Where the CTA's part begins, by every warp for itself; a lane has four sequences of 128.
    __device__ __forceinline__ R4Walk(const KvAttendParams& P, int lim, int shift, int units) {
        const int lane = threadIdx.x & 31;
        auto lengths = [&](int b0, int (&v)[4]) {  // their sum over the lanes up to this one
            int sum = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = b0 + 4 * lane + i;
                v[i] = at < P.step.n_seqs ? R4Seq(P, lim, shift, at).length(units) : 0;
                sum += v[i];
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += u;
            }
            return sum;
        };
        int v[4], inc = lengths(0, v), total = __shfl_sync(0xffffffffu, inc, 31);
#pragma unroll 1
        for (int b0 = 128; b0 < P.step.n_seqs; b0 += 128) {
            int x[4];
            total += __shfl_sync(0xffffffffu, lengths(b0, x), 31);
        }
        per = (int)(((uint32_t)total + gridDim.x - 1) / gridDim.x);
        w = (int)min((int64_t)total, (int64_t)per * blockIdx.x);
        w1 = (int)min((int64_t)total, (int64_t)w + per);
        first = true;
        t0 = -1; t1 = 0;
        start = 0; b = 0;
        if (w >= w1) return;
        int front = 0;
#pragma unroll 1
        for (int b0 = 0;; b0 += 128) {
            if (b0) inc = lengths(b0, v);
            const unsigned past = __ballot_sync(0xffffffffu, front + inc > w);
            if (past) {
                const int src = __ffs(past) - 1;
                int at = front + inc - (v[0] + v[1] + v[2] + v[3]), i = 0;  // (of the lane found, the sequence that w is in)
#pragma unroll
                for (int k = 0; k < 3; k++)
                    if (i == k && at + v[k] <= w) { at += v[k]; i = k + 1; }
                start = __shfl_sync(0xffffffffu, at, src);
                b = b0 + 4 * src + __shfl_sync(0xffffffffu, i, src);
                break;
            }
            front += __shfl_sync(0xffffffffu, inc, 31);
        }
        q = R4Seq(P, lim, shift, b);
    }
    __device__ __forceinline__ bool next(const KvAttendParams& P, int lim, int shift, int units) {
        if (t0 >= 0) first = false;
#pragma unroll 1
        while (w < w1) {
            int length = q.length(units);
            while (w - start >= length) {
                start += length;
                q = R4Seq(P, lim, shift, ++b);
                length = q.length(units);
            }
            const int in = w - start, place = q.view.tiles + R4_SETUP;  // of a unit on the line, whose first R4_SETUP are no tiles
            unit = (uint32_t)in / (uint32_t)place;
            const int at = in - unit * place, end = min(place, at + (w1 - w));
            w += end - at;
            if (end <= R4_SETUP) continue;  // (its tiles begin in the next CTA)
            t0 = max(0, at - R4_SETUP);
            t1 = end - R4_SETUP;
            return true;
        }
        return false;
    }
};

// What the products of a piece have to know of it: left by the copies, which are ahead.
struct R4Piece {
    int64_t row0;  // of the row arrays
    int rows, head, lo_pos, whole_slot;  // whole_slot: -1 where the piece is all of its unit, else which of the CTA's two partial results it is
};

// Partial results of a CTA's first (slot 0) and last piece, a head each: `rows` times hd floats, then `rows` times (m, l).
__device__ __forceinline__ float* r4_part(void* work, int ctas, int heads, int rows, int hd, int64_t cta, int slot, int h) {
    return reinterpret_cast<float*>(static_cast<char*>(work) + kv_cut_bytes(ctas)) + ((cta * 2 + slot) * heads + h) * rows * (hd + 2);
}
__device__ __forceinline__ void r4_store4(const KvRows& o, int64_t e, float a, float b, float c, float d) {
    if (o.type == L2_F32) *reinterpret_cast<float4*>(o.data + 4 * e) = make_float4(a, b, c, d);
    else if (o.type == L2_F16) *reinterpret_cast<uint2*>(o.data + 2 * e) = make_uint2(pack16<false>(a, b), pack16<false>(c, d));
    else *reinterpret_cast<uint2*>(o.data + 2 * e) = make_uint2(pack16<true>(a, b), pack16<true>(c, d));
}

// ---- a step: 32 positions of a warp ------------------------------------------------------------------------------------------
constexpr int R4_TOP = 6;              // h is chosen so that the largest p t h is between 2^this and twice as much ...
constexpr uint32_t R4_LIMIT = 0x7800;  // ... and again where one reaches 2^15 (in f16)

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {  // onto zeros
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t max_abs_f16(uint32_t a, uint32_t b) {  // of magnitudes; the sign is either
    uint32_t r;
    asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// 2^k with 2^R4_TOP <= w 2^k < 2^(R4_TOP + 1), within 2^-100 .. 2^64 (w = 0: what it was)
__device__ __forceinline__ float r4_factor(float w, float before) {
    const int e = (int)(__float_as_uint(w) >> 23);  // (w is not negative; NaN and infinity: 255)
    return w > 0.0f ? __uint_as_float((uint32_t)min(max(127 + R4_TOP + 127 - e, 27), 191) << 23) : before;
}

// What a warp keeps of its rows, as the threads have them: rows 8 nt + 2 c and 8 nt + 2 c + 1
template <int HD, int NT>
struct R4Rows {
    uint32_t q[HD / 32][NT][4];  // of 32 elements: the words of elements 8 c + {0, 4}, {2, 6} and, a sixteenth, of {1, 5}, {3, 7}
    float by[NT][2], sum[NT][2]; // a score is `by` times (s (u . q) + z sum), in powers of two
    int pos[NT][2];
    float m[NT][2], l[NT][2], y[NT][2], h[NT][2];
    float o[HD / 16][NT][4];
    int state;                   // (of the warp) 0: no row has an m yet, 1: some have none, 2: all have one
};
struct R4Lane { uint32_t k, v; };  // a lane's places in a slot for the fragments of K and of V

// slot: the step's in shared memory (K, V, pairs of K, of V); first: its first position.  Position 4 i + 2 mb + half is row 16 mb + 8 half + i of the products, so that a thread's four
// positions, i = g8, lie side by side; 32 more for every two mb more.
// Nothing looks for a score above m in front of the exponentials: f32 has room for 2^100 in the sums and f16 for 2^15 in p t h, and a step with rows that pass either, or have no m yet,
// is done again with a larger m and a smaller h for these rows.
template <int HD, int NT>
__device__ __forceinline__ void r4_step(const KvAttendParams& P, R4Rows<HD, NT>& r, const R4Lane& at, const uint8_t* slot, int first, bool whole) {
    using S = R4Shape<HD, NT>;
    constexpr int MB = S::STEP / 16, CH = HD / 32;  // (blocks of 32 positions, of two MB each)
    constexpr uint32_t LO = 0x000f000fu, HI = 0x00f000f0u;
    const uint32_t base = kv_smem(slot);
    const int j0 = first + 4 * ((threadIdx.x & 31) >> 2);
    // ---- u . q of the positions, rows 2 c and 2 c + 1
    float s[MB][NT][4];
#pragma unroll
    for (int c2 = 0; c2 < CH / 2; c2++)
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            uint32_t a[4];
            ldsm4(a, base + (at.k ^ (32 * c2)) + 16 * mb * S::ROW);
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t a0 = a[2 * x], a1 = a[2 * x + 1], b0 = a0 >> 8, b1 = a1 >> 8;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const uint32_t (&q)[4] = r.q[2 * c2 + x][nt];
                    if (c2 == 0 && x == 0) mma_f16_new(s[mb][nt], a0 & LO, a1 & LO, b0 & LO, b1 & LO, q[0], q[1]);
                    else mma_f16(s[mb][nt], a0 & LO, a1 & LO, b0 & LO, b1 & LO, q[0], q[1]);
                    mma_f16(s[mb][nt], a0 & HI, a1 & HI, b0 & HI, b1 & HI, q[2], q[3]);
                }
            }
        }
    // ---- scores, in units of `by`
    uint32_t kw[2 * MB], vw[2 * MB];
#pragma unroll
    for (int b = 0; b < MB / 2; b++) {
        const uint4 k = *reinterpret_cast<const uint4*>(slot + 2 * S::KV + 128 * b + 16 * ((threadIdx.x & 31) >> 2)), v = *reinterpret_cast<const uint4*>(slot + 2 * S::KV + 4 * S::STEP + 128 * b + 16 * ((threadIdx.x & 31) >> 2));
        kw[4 * b] = k.x; kw[4 * b + 1] = k.y; kw[4 * b + 2] = k.z; kw[4 * b + 3] = k.w;
        vw[4 * b] = v.x; vw[4 * b + 1] = v.y; vw[4 * b + 2] = v.z; vw[4 * b + 3] = v.w;
    }
    auto sees = [&](int nt, int mb, int i) { return kv_sees(r.pos[nt][i & 1], j0 + 32 * (mb / 2) + 2 * (mb % 2) + (i >> 1), P.window, P.sinks); };
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t w = kw[2 * mb + (i >> 1)];
                s[mb][nt][i] = fmaf(kv_pair_scale(w), s[mb][nt][i], kv_pair_zero(w) * r.sum[nt][i & 1]);
            }
    if (!whole) {
#pragma unroll
        for (int mb = 0; mb < MB; mb++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (!sees(nt, mb, i)) s[mb][nt][i] = -INFINITY;
    }
    // ---- probabilities, and with the scales of V and h (what a row does not see may have any)
    float l[NT][2], y[NT][2];
    uint32_t pb[MB][NT][2];
    auto probabilities = [&](auto is_whole) {
        uint32_t top = 0;
        float most = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const float ref[2] = {r.m[nt][0] == -INFINITY ? 0.0f : r.m[nt][0], r.m[nt][1] == -INFINITY ? 0.0f : r.m[nt][1]};
            l[nt][0] = r.l[nt][0]; l[nt][1] = r.l[nt][1];
            y[nt][0] = r.y[nt][0]; y[nt][1] = r.y[nt][1];
#pragma unroll
            for (int mb = 0; mb < MB; mb++)
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const float t = kv_pair_scale(vw[2 * mb + half]), zero = kv_pair_zero(vw[2 * mb + half]);
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float p = kv_exp2(fmaf(s[mb][nt][2 * half + e], r.by[nt][e], -ref[e]));
                        l[nt][e] += p;
                        w[e] = p;
                        if (decltype(is_whole)::value || sees(nt, mb, 2 * half + e)) {
                            y[nt][e] = fmaf(p, zero, y[nt][e]);
                            w[e] = p * (t * r.h[nt][e]);
                        }
                    }
                    pb[mb][nt][half] = pack16<false>(w[0], w[1]);
                    top = max_abs_f16(top, pb[mb][nt][half]);
                }
            most = fmaxf(most, fmaxf(l[nt][0], l[nt][1]));
        }
        top &= 0x7fff7fffu;
        return most >= 0x1p100f || (top & 0xffffu) >= R4_LIMIT || (top >> 16) >= R4_LIMIT;
    };
    // (A loop, so that the probabilities are in the code once: one token of one sequence 13.5 -> 13.0 us, a window of 13B heads 55.7 -> 54.8)
    bool ready = false;  // m and h hold for this step
#pragma unroll 1
    for (bool first = r.state == 0;; first = false) {
        if (!first) {
            const bool over = whole ? probabilities(std::true_type()) : probabilities(std::false_type());
            if (ready || !(__any_sync(0xffffffffu, over) || r.state != 2)) break;
        }
        // seldom: a row's m is raised, or its h lowered, and what was summed is scaled.  Only of rows that need it: a row's result does not depend on the others.
        bool none = false;
        uint32_t needs = ~0u;  // a bit a row
        if (r.state) {
            needs = 0u;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    bool mine = r.m[nt][e] == -INFINITY || l[nt][e] >= 0x1p100f;
#pragma unroll
                    for (int mb = 0; mb < MB; mb++) mine |= (pb[mb][nt][0] >> (16 * e) & 0x7fffu) >= R4_LIMIT || (pb[mb][nt][1] >> (16 * e) & 0x7fffu) >= R4_LIMIT;
                    if (__ballot_sync(0xffffffffu, mine) & 0x11111111u << (threadIdx.x & 3)) needs |= 1u << (2 * nt + e);
                }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                auto over_lanes = [](float x) {  // the largest of the lanes that have the row
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                };
                const bool row_needs = needs >> (2 * nt + e) & 1u;
                float x = -INFINITY, w = 0.0f;
#pragma unroll
                for (int mb = 0; mb < MB; mb++)
#pragma unroll
                    for (int half = 0; half < 2; half++) x = fmaxf(x, s[mb][nt][2 * half + e]);
                x = over_lanes(x) * r.by[nt][e] - R4_BIAS;
                const bool up = row_needs && x > r.m[nt][e] + R4_RAISE;
                const float m1 = up ? x : r.m[nt][e];
                const KvScale f(m1 == -INFINITY ? 0.0f : r.m[nt][e] - m1);
                r.m[nt][e] = m1;
                none |= m1 == -INFINITY;
                r.l[nt][e] = f(r.l[nt][e]);
                r.y[nt][e] = f(r.y[nt][e]);
#pragma unroll
                for (int mb = 0; mb < MB; mb++)
#pragma unroll
                    for (int half = 0; half < 2; half++)
                        if (whole || sees(nt, mb, 2 * half + e))
                            w = fmaxf(w, fabsf(kv_exp2(fmaf(s[mb][nt][2 * half + e], r.by[nt][e], m1 == -INFINITY ? 0.0f : -m1)) * kv_pair_scale(vw[2 * mb + half])));
                w = over_lanes(w);
                const float h1 = row_needs && (up || w * r.h[nt][e] >= 32768.0f * 0.99f) ? r4_factor(w, r.h[nt][e]) : r.h[nt][e];
                // (in two steps: the power of two between the two h may be beyond f32)
                const int k = (int)(__float_as_uint(h1) >> 23) - (int)(__float_as_uint(r.h[nt][e]) >> 23);
                const float a = __uint_as_float((uint32_t)(127 + k / 2) << 23), b = __uint_as_float((uint32_t)(127 + k - k / 2) << 23);
                r.h[nt][e] = h1;
#pragma unroll
                for (int mt = 0; mt < HD / 16; mt++) {
                    r.o[mt][nt][e] = f(r.o[mt][nt][e]) * a * b;
                    r.o[mt][nt][e + 2] = f(r.o[mt][nt][e + 2]) * a * b;
                }
            }
        r.state = __any_sync(0xffffffffu, none) ? 1 : 2;
        ready = true;
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) { r.l[nt][e] = l[nt][e]; r.y[nt][e] = y[nt][e]; }
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) { pb[mb][nt][0] = transpose8(pb[mb][nt][0]); pb[mb][nt][1] = transpose8(pb[mb][nt][1]); }
    // ---- O^T += U^T P^T.  Of 32 elements (a chunk) the product 2 chunk + i has elements 4 g8 + 2 i in its rows g8, 4 g8 + 2 i + 1 in its rows g8 + 8
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int c2 = 0; c2 < CH / 2; c2++) {
            uint32_t a[4];
            ldsm4_t(a, base + S::KV + (at.v ^ (32 * c2)) + 16 * mb * S::ROW);
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t a0 = a[x], a1 = a[x + 2], b0 = a0 >> 8, b1 = a1 >> 8;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    mma_f16(r.o[2 * (2 * c2 + x)][nt], a0 & LO, a0 & HI, a1 & LO, a1 & HI, pb[mb][nt][0], pb[mb][nt][1]);
                    mma_f16(r.o[2 * (2 * c2 + x) + 1][nt], b0 & LO, b0 & HI, b1 & LO, b1 & HI, pb[mb][nt][0], pb[mb][nt][1]);
                }
            }
        }
}

// ---- the kernel ----------------------------------------------------------------------------------------------------------------
// QB: q is bf16, else f16
template <bool QB, int HD, int NT>
__global__ void __launch_bounds__(R4_THREADS, R4_CTAS) kv_rows4_kernel(const __grid_constant__ KvAttendParams P, const int lim, const int shift) {
    using S = R4Shape<HD, NT>;
    constexpr int CHUNKS = S::ROW / 16, PER_COPY = 32 / CHUNKS, PAIR_LANES = S::STEP / 4, COPIES = S::STEP / PER_COPY;  // 16-byte chunks of a row; positions of a copy by the warp, copies of a step
    extern __shared__ __align__(128) uint8_t r4_smem[];
    __shared__ R4Piece pieces[R4_WARPS][4];
    __shared__ __align__(8) uint64_t full[R4_WARPS][4], empty[R4_WARPS][4], met[2];
    __shared__ volatile int failed;
    __shared__ int2 marks[R4_WARPS][4];  // of a slot: the step's first position; bit 0: every row sees all of it, 1: some row sees something, 2: the piece's last step, 3: there is none
    const int tid = threadIdx.x, warp = (tid >> 5) % R4_WARPS, lane = tid & 31, g8 = lane >> 2, c = lane & 3;
    const R4Split split = r4_split(P.pool.n_kv_heads);
    const int units = P.pool.n_kv_heads / split.heads, of_head = warp / split.wph, share = warp % split.wph;  // this warp's head of the unit, its place among that one's warps
    const int steps = (1 << shift) / (S::STEP * split.wph), slots = S::SLOTS;
    uint8_t* const ring = r4_smem + warp * slots * S::SLOT;
    if (tid < R4_WARPS * 4) { kv_bar_init(&full[0][0] + tid, 33); kv_bar_init(&empty[0][0] + tid, 1); }
    if (tid < 2) kv_bar_init(&met[tid], split.wph);
    if (tid == 0) failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    const KvWait wait{&failed};

    // (registers: 128 x (72 + 184) of the 256 x 128 that the launch has; 56 + 200 leaves more of the copies' addresses in memory: 1.2 us longer)
    if (tid >= 32 * R4_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        // ================= copies ==========================================================================================================
        asm volatile("griddepcontrol.wait;" ::: "memory");  // (rows, lengths and the cache may come from the kernel in front)
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        R4Walk walk(P, lim, shift, units);
        const bool first_warp = tid == 32 * R4_WARPS;
        if (first_warp) kv_cuts(P.work)[blockIdx.x].pieces = 0;  // (no unit that begins here goes on, until one does)
        int pages = 0, next_pages = 0, page0 = 0, next0 = -1;  // a lane has entry page0 + lane of the table
        uint32_t there = 0;                                    // which of them are pages
        // Of K, where the lane's 16 bytes of the head's first position are, and its row of a copy from there on; and of the pairs.  V lies as far behind K everywhere.
        const char *k_lane = nullptr, *pair_lane = nullptr;
        const int64_t to_v = P.pool.v - P.pool.k, page_bytes = P.pool.page_stride / 2, pos_bytes = P.pool.pos_stride / 2;
        const int mask = (1 << P.pool.page_shift) - 1, pair_page = P.pool.n_kv_heads << P.pool.page_shift + 2;
        // position r of 32 is row 8 (r % 4) + r / 4 of theirs
        constexpr int SIDE = PER_COPY / 4, IN_BLOCK = 32 / PER_COPY;
        const uint32_t lane_row = ((lane / CHUNKS & 3) * 8 + (lane / CHUNKS >> 2)) * S::ROW, lane_chunk = 16 * (lane % CHUNKS);
        static_assert(SIDE * S::ROW == 128, "the rows of a copy behind those of the one in front");
        auto look_up = [&](int first) {  // the entries that some row sees, as they are (nothing waits for them before they are needed); -2: none of these
            const int i = first + lane;
            if (i > walk.q.view.hi >> P.pool.page_shift || (P.window && !walk.q.view.any(i << P.pool.page_shift, 1 << P.pool.page_shift, P.window, P.sinks))) return -2;
            return P.step.table[(size_t)walk.b * P.step.width + i];
        };
        uint32_t put = 0, ph = 1;
        auto give = [&](int first, int flags) {  // the slot's copies and what it is, to the warp of products
            kv_copy16_arrive(&full[warp][put]);
            if (lane == 0) {
                marks[warp][put] = make_int2(first, flags);
                kv_bar_arrive(&full[warp][put]);
            }
            if (++put == slots) { put = 0; ph ^= 1u; }
        };
        bool over = false;
#pragma unroll 1
        for (int begun = 0; !over && walk.next(P, lim, shift, units); begun++) {
            const int head = walk.unit * split.heads + of_head;
            const bool done = walk.t0 == 0 && walk.t1 == walk.q.view.tiles;
            if (first_warp && walk.t0 == 0 && !done)  // what the kernel behind this one has to know of the CTA's last piece
                kv_cuts(P.work)[blockIdx.x] = KvCut{(int)((uint32_t)(walk.w - walk.t1 + walk.q.view.tiles - 1) / (uint32_t)walk.per) - (int)blockIdx.x + 1, walk.first ? 0 : 1, walk.q.rows,
                                                    walk.unit * split.heads, walk.q.s.row0, walk.q.view.lo, 0};
            k_lane = P.pool.k + (int64_t)head * (P.pool.head_stride / 2) + lane_chunk + (PER_COPY <= 8 || mask >= PER_COPY - 1 ? lane / CHUNKS : lane / CHUNKS & mask) * pos_bytes;
            pair_lane = reinterpret_cast<const char*>(lane < PAIR_LANES ? P.pool.ks : P.pool.vs) + (((int64_t)head << P.pool.page_shift) + (4 * (lane % PAIR_LANES) & mask)) * 4;
            page0 = next0 = -1 << 20;
            const R4View& view = walk.q.view;
#pragma unroll 1
            for (int t = walk.t0, k = 0; t < walk.t1;) {
                const int j0 = view.base(t, shift) + (k * split.wph + share) * S::STEP;
                bool some = j0 <= view.hi, whole = j0 + S::STEP <= view.lo + 1;
                if (P.window) { some = view.any(j0, S::STEP, P.window, P.sinks); whole = view.whole(j0, S::STEP, P.window, P.sinks); }
                wait(&empty[warp][put], ph);
                if ((over = wait.over())) break;
                if (t == walk.t0 && k == 0 && lane == 0) pieces[warp][begun & 3] = R4Piece{walk.q.s.row0, walk.q.rows, head, walk.q.view.lo, done ? -1 : walk.first ? 0 : 1};
                const uint32_t to = kv_smem(ring + put * S::SLOT);
                if (some) {
                    const int want = j0 >> P.pool.page_shift, last = (j0 + S::STEP - 1) >> P.pool.page_shift;
                    if (want < page0 || last > page0 + 31) {
                        if (want == next0) { pages = next_pages; page0 = next0; }
                        else { page0 = want; pages = look_up(page0); }
                        next0 = page0 + 32;  // (steps go on by whole pages, or within one, and by a divisor of 32 of them)
                        next_pages = look_up(next0);
                        if (pages != -2 && (unsigned)pages >= (unsigned)P.pool.n_pages) kv_report(P.step.status, L2_KV_BAD_PAGE);
                        if ((unsigned)pages >= (unsigned)P.pool.n_pages) pages = -1;
                        there = __ballot_sync(0xffffffffu, pages >= 0);
                    }
                    // (a step begins a page or lies inside one)
                    const int in = j0 & mask, p0 = (j0 >> P.pool.page_shift) - page0;
                    const uint32_t need = (2u << (S::STEP - 1 >> P.pool.page_shift)) - 1;
                    if ((there >> p0 & need) == need) {
                        const uint32_t at = to + lane_row + lane_chunk;
                        auto copies = [&](auto n) {  // of a step with so many pages
                            constexpr int PER_PAGE = S::STEP / decltype(n)::value;
                            const char* from = k_lane;
#pragma unroll
                            for (int i = 0; i < COPIES; i++) {
                                if (PER_COPY > PER_PAGE || i * PER_COPY % PER_PAGE == 0) {
                                    from = k_lane + r4_times(__shfl_sync(0xffffffffu, pages, p0 + i * PER_COPY / PER_PAGE + (PER_COPY > PER_PAGE ? lane / CHUNKS / PER_PAGE : 0)), page_bytes);
                                    if (PER_PAGE == S::STEP) from += r4_times(in, pos_bytes);
                                } else {
                                    from += PER_COPY * pos_bytes;
                                }
                                const uint32_t off = (at ^ 16 * (i % IN_BLOCK)) + 128 * (i % IN_BLOCK) + 32 * S::ROW * (i / IN_BLOCK);
                                r4_copy(off, from);
                                r4_copy(off + S::KV, from + to_v);
                            }
                        };
                        if (P.pool.page_shift == 4) copies(std::integral_constant<int, S::STEP / 16>());
                        else if (P.pool.page_shift == 5) copies(std::integral_constant<int, S::STEP / 32>());
                        else if (P.pool.page_shift == 3) copies(std::integral_constant<int, S::STEP / 8>());
                        else copies(std::integral_constant<int, 1>());
                        // the pairs: four positions a lane, of K by the first lanes, of V by the next
                        const int page = __shfl_sync(0xffffffffu, pages, p0 + (4 * (lane % PAIR_LANES) >> P.pool.page_shift));
                        if (2 * PAIR_LANES == 32 || lane < 2 * PAIR_LANES) r4_copy(to + 2 * S::KV + 16 * lane, pair_lane + (uint64_t)(uint32_t)page * (uint32_t)pair_page + 4 * in);
                    } else {  // zeros where there is no page
#pragma unroll 1
                        for (int i = 0; i < COPIES; i++) {
                            const int page = __shfl_sync(0xffffffffu, pages, p0 + (i * PER_COPY >> P.pool.page_shift) + (PER_COPY <= 8 ? 0 : lane / CHUNKS >> P.pool.page_shift));
                            const char* const from = k_lane + r4_times(max(page, 0), page_bytes) + (in + (i * PER_COPY & mask)) * pos_bytes;
                            const uint32_t off = to + lane_row + 128 * (i % IN_BLOCK) + 32 * S::ROW * (i / IN_BLOCK) + (lane_chunk ^ (16 * (i % IN_BLOCK)));
                            r4_copy_if(off, from, page >= 0);
                            r4_copy_if(off + S::KV, from + to_v, page >= 0);
                        }
                        const int page = __shfl_sync(0xffffffffu, pages, p0 + (4 * (lane % PAIR_LANES) >> P.pool.page_shift));
                        if (2 * PAIR_LANES == 32 || lane < 2 * PAIR_LANES) r4_copy_if(to + 2 * S::KV + 16 * lane, pair_lane + (uint64_t)(uint32_t)max(page, 0) * (uint32_t)pair_page + 4 * in, page >= 0);
                    }
                }
                if (++k == steps) { k = 0; t++; }
                give(j0, (int)whole | (int)some << 1 | (int)(t >= walk.t1) << 2);
            }
        }
        if (!over) {
            wait(&empty[warp][put], ph);
            give(0, 8);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (lane == 0 && failed) kv_report(P.step.status, L2_KV_TIMEOUT);
        return;
    }

    // ================= products ========================================================================================================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    R4Rows<HD, NT> r;
    const R4Lane at{r4_offset<S::ROW>(lane & 15, lane >> 4), r4_offset<S::ROW>((lane & 7) + 8 * (lane >> 4), (lane >> 3) & 1)};
    R4Piece piece{};
    bool fresh = true;
    int ended = 0;
    uint32_t get = 0, ph = 0, met_ph = 0;
#pragma unroll 1
    while (true) {
        wait(&full[warp][get], ph);
        if (wait.over()) break;
        const int2 mark = marks[warp][get];
        if (mark.y & 8) break;
        if (fresh) {  // a new piece: Q, in f16, of eight elements the words (0, 4), (2, 6), (1, 5), (3, 7), as the numbers of a word of K come out
            piece = pieces[warp][ended & 3];
            fresh = false;
            r.state = 0;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const int row = 8 * nt + g8, tok = row / P.group;
                uint4 x[HD / 32];
#pragma unroll
                for (int ch = 0; ch < HD / 32; ch++) {
                    x[ch] = make_uint4(0, 0, 0, 0);
                    if (row < piece.rows)
                        x[ch] = *reinterpret_cast<const uint4*>(P.q.data + 2 * ((piece.row0 + tok) * P.q.row_stride + (int64_t)(piece.head * P.group + row - tok * P.group) * P.q.head_stride + 32 * ch + 8 * c));
                }
                float up = 1.0f, by = 1.0f, sum = 0.0f;
                auto element = [&](const uint4& v, int i) {
                    const uint32_t w = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
                    return QB ? __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16) : __half2float(__ushort_as_half((unsigned short)(w >> (16 * (i % 2)))));
                };
                {
                    float top = 0.0f;
#pragma unroll
                    for (int ch = 0; ch < HD / 32; ch++)
#pragma unroll
                        for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(element(x[ch], i)));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    kv_q_factors(top, &up, &by);
                }
#pragma unroll
                for (int ch = 0; ch < HD / 32; ch++) {
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) { y[i] = element(x[ch], i) * up; sum += y[i]; }
                    r.q[ch][nt][0] = pack16<false>(y[0], y[4]); r.q[ch][nt][1] = pack16<false>(y[2], y[6]);
                    r.q[ch][nt][2] = pack16<false>(y[1] * 0.0625f, y[5] * 0.0625f); r.q[ch][nt][3] = pack16<false>(y[3] * 0.0625f, y[7] * 0.0625f);
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                // (rows are g8 here, and 2 c and 2 c + 1 below; the products are of numbers times 2^-24)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    r.by[nt][e] = __shfl_sync(0xffffffffu, by, 4 * (2 * c + e)) * (P.scale_log2 * 0x1p24f);
                    r.sum[nt][e] = __shfl_sync(0xffffffffu, sum, 4 * (2 * c + e)) * 0x1p-24f;
                    r.pos[nt][e] = piece.lo_pos + min(8 * nt + 2 * c + e, piece.rows - 1) / P.group;  // (rows that there are not see no more than the last)
                    r.m[nt][e] = -INFINITY;
                    r.l[nt][e] = r.y[nt][e] = 0.0f;
                    r.h[nt][e] = 1.0f;
                }
#pragma unroll
                for (int mt = 0; mt < HD / 16; mt++) r.o[mt][nt][0] = r.o[mt][nt][1] = r.o[mt][nt][2] = r.o[mt][nt][3] = 0.0f;
            }
        }
        if (mark.y & 2) r4_step<HD, NT>(P, r, at, ring + get * S::SLOT, mark.x, mark.y & 1);
        __syncwarp();
        if (lane == 0) kv_bar_arrive(&empty[warp][get]);  // (the slot is free)
        if (++get == slots) { get = 0; ph ^= 1u; }
        if (!(mark.y & 4)) continue;

        // ---- the piece's end: sums over the lanes that have the row, in units of 2^-m, with what the zeros give every element
        fresh = true;
        ended++;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float y = r.y[nt][e], l = r.l[nt][e];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) { y += __shfl_xor_sync(0xffffffffu, y, o); l += __shfl_xor_sync(0xffffffffu, l, o); }
                r.l[nt][e] = l;
                const float by = 0x1p20f / r.h[nt][e];  // (a power of two between 2^-44 and 2^120)
#pragma unroll
                for (int mt = 0; mt < HD / 16; mt++) {
                    r.o[mt][nt][e] = fmaf(r.o[mt][nt][e], 16.0f * by, y);
                    r.o[mt][nt][e + 2] = fmaf(r.o[mt][nt][e + 2], by, y);
                }
            }
        if (split.wph > 1) {  // the warps of a head meet: the upper half leaves its results for the lower, and again
            uint8_t* const room = r4_smem + R4_WARPS * slots * S::SLOT;
            auto meet = [&]() {
                __syncwarp();
                if (lane == 0) kv_bar_arrive(&met[of_head]);
                wait(&met[of_head], met_ph);
                met_ph ^= 1u;
                __syncwarp();
            };
#pragma unroll 1
            for (int half = split.wph / 2; half; half >>= 1) {
                float4* const o = reinterpret_cast<float4*>(room + (split.wph == 2 ? of_head : share % half) * (S::O_BYTES + S::ROWS * 8));
                float2* const ml = reinterpret_cast<float2*>(o + S::O_BYTES / 16);
                if (share >= half && share < 2 * half) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                        for (int mt = 0; mt < HD / 16; mt++) o[(mt * NT + nt) * 32 + lane] = make_float4(r.o[mt][nt][0], r.o[mt][nt][1], r.o[mt][nt][2], r.o[mt][nt][3]);
                        if (g8 == 0) {
                            ml[8 * nt + 2 * c] = make_float2(r.m[nt][0], r.l[nt][0]);
                            ml[8 * nt + 2 * c + 1] = make_float2(r.m[nt][1], r.l[nt][1]);
                        }
                    }
                }
                meet();
                if (share < half) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float fa[2], fb[2];  // (2^d for d <= 0 as two factors: see KvScale)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float2 x = ml[8 * nt + 2 * c + e];
                            const float top = fmaxf(r.m[nt][e], x.x), ref = top == -INFINITY ? 0.0f : top;
                            const KvScale f(r.m[nt][e] - ref), g(x.x - ref);
                            r.m[nt][e] = top;
                            r.l[nt][e] = f(r.l[nt][e]) + g(x.y);
                            fa[e] = f.h; fb[e] = g.h;
                        }
#pragma unroll
                        for (int mt = 0; mt < HD / 16; mt++) {
                            const float4 x = o[(mt * NT + nt) * 32 + lane];
                            const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int i = 0; i < 4; i++) r.o[mt][nt][i] = r.o[mt][nt][i] * fa[i & 1] * fa[i & 1] + v[i] * fb[i & 1] * fb[i & 1];
                        }
                    }
                }
                meet();  // (the room is free)
            }
        }
        if (share == 0) {
            float* const part = r4_part(P.work, gridDim.x, split.heads, S::ROWS, HD, blockIdx.x, max(0, piece.whole_slot), of_head);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int row = 8 * nt + 2 * c + e;
                    if (row >= piece.rows) continue;
                    const int tok = row / P.group;
                    const int64_t at = (piece.row0 + tok) * P.out.row_stride + (int64_t)(piece.head * P.group + row - tok * P.group) * P.out.head_stride;
                    const bool sees = r.pos[nt][e] >= 0;
                    const float inv = 1.0f / r.l[nt][e];
#pragma unroll
                    for (int ch = 0; ch < HD / 32; ch++) {
                        const float v[4] = {r.o[2 * ch][nt][e], r.o[2 * ch][nt][e + 2], r.o[2 * ch + 1][nt][e], r.o[2 * ch + 1][nt][e + 2]};
                        const int d = 32 * ch + 4 * g8;
                        if (piece.whole_slot >= 0) *reinterpret_cast<float4*>(part + row * HD + d) = make_float4(v[0], v[1], v[2], v[3]);
                        else if (sees) r4_store4(P.out, at + d, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                        else r4_store4(P.out, at + d, 0.0f, 0.0f, 0.0f, 0.0f);
                    }
                    if (piece.whole_slot >= 0 && g8 == 0) *reinterpret_cast<float2*>(part + S::ROWS * HD + 2 * row) = make_float2(r.m[nt][e], r.l[nt][e]);
                }
        }
    }
    if (lane == 0 && failed) kv_report(P.step.status, L2_KV_TIMEOUT);
}

// Adds the pieces of the unit that begins in CTA x of the launch in front and goes on in the next; blockIdx.y has one of its heads.
// HD / 4 threads for a row; with few rows the others take pieces of the same row, and meet in order.
template <int HD>
__global__ void __launch_bounds__(256) kv_rows4_combine_kernel(const __grid_constant__ KvAttendParams P, const int ctas, const int part_rows) {
    constexpr int LANES = HD / 4, SLOTS = 256 / LANES;
    __shared__ float4 sums[256];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const KvCut cut = kv_cuts(P.work)[blockIdx.x];
    if (!cut.pieces) return;
    auto piece = [&](int i) { return r4_part(P.work, ctas, gridDim.y, part_rows, HD, blockIdx.x + i, i == 0 ? cut.slot : 0, blockIdx.y); };
    const int head = cut.head + blockIdx.y;
    int width = 1;  // rows side by side
    while (width < cut.rows && width < SLOTS) width <<= 1;
    const int share = SLOTS / width, slot = threadIdx.x / LANES, d = 4 * (threadIdx.x % LANES), mine = slot / width;
    for (int r0 = 0; r0 < cut.rows; r0 += width) {
        const int r = r0 + slot % width;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.0f;
        const bool on = r < cut.rows;
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
            const int64_t e = (cut.row0 + tok) * P.out.row_stride + (int64_t)(head * P.group + r - tok * P.group) * P.out.head_stride + d;
            const float inv = 1.0f / sum;
            if (pos < 0) r4_store4(P.out, e, 0.0f, 0.0f, 0.0f, 0.0f);
            else r4_store4(P.out, e, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        }
    }
}

int r4_nt(int lim) { return lim <= 8 ? 1 : 2; }
// Tiles that are so large that the line stays below 2^31, and the CTAs of a launch: no more than the line can be long (which is R4_SETUP + 1 or more).
struct R4Grid { int shift, ctas; };
R4Grid r4_grid(const KvStep& s, const KvPool& p, int nt, int sms) {
    const R4Split split = r4_split(p.n_kv_heads);
    for (int shift = r4_least_shift(split.wph, nt);; shift++) {
        const int64_t most = (int64_t)s.n_seqs * (p.n_kv_heads / split.heads) * (((((int64_t)s.width << p.page_shift) + (1 << shift) - 1) >> shift) + 1 + R4_SETUP);
        if (most < ((int64_t)1 << 31) - 65536 || shift == 30)
            return {shift, (int)std::min<int64_t>(R4_CTAS * sms, most)};
    }
}

}  // namespace

size_t kv_rows4_work(const KvStep& s, const KvPool& p, int lim, int head_size, int sms) {
    const int nt = r4_nt(lim), grid = r4_grid(s, p, nt, sms).ctas;
    return kv_cut_bytes(grid) + (size_t)grid * 2 * r4_split(p.n_kv_heads).heads * 8 * nt * (head_size + 2) * sizeof(float);
}

cudaError_t launch_kv_rows4(const KvAttendParams& p, int lim, int head_size, int sms, cudaStream_t st) {
    const int nt = r4_nt(lim);
    const R4Grid of = r4_grid(p.step, p.pool, nt, sms);
    const int grid = of.ctas;
    const R4Split split = r4_split(p.pool.n_kv_heads);
    auto go = [&](auto b, auto h, auto n) {
        using S = R4Shape<decltype(h)::value, decltype(n)::value>;
        auto kernel = kv_rows4_kernel<decltype(b)::value, decltype(h)::value, decltype(n)::value>;
        static KvOnce once;
        if (cudaError_t x = once.shared_memory(reinterpret_cast<const void*>(kernel), std::max(S::smem(1), S::smem(4)))) return x;
        return kv_launch(kernel, dim3(grid), R4_THREADS, S::smem(split.wph), st, p, lim, of.shift);
    };
    auto by_nt = [&](auto b, auto h) { return nt == 1 ? go(b, h, std::integral_constant<int, 1>()) : go(b, h, std::integral_constant<int, 2>()); };
    auto by_hd = [&](auto b) { return head_size == 128 ? by_nt(b, std::integral_constant<int, 128>()) : by_nt(b, std::integral_constant<int, 64>()); };
    const cudaError_t e = p.q.type == L2_BF16 ? by_hd(std::true_type()) : by_hd(std::false_type());
    if (e != cudaSuccess || grid < 2) return e;
    auto combine = head_size == 128 ? kv_rows4_combine_kernel<128> : kv_rows4_combine_kernel<64>;
    return kv_launch(combine, dim3(grid - 1, split.heads), 256, 0, st, p, grid, 8 * nt);
}

}  // namespace l2