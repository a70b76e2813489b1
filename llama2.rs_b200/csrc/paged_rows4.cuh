// A step of kv_rows_kernel over a cache in 4 bits: 32 positions of a warp.
//
// With u the numbers of 0 .. 15, a pair (scale, zero) for every position of K (s, z) and of V (t, y), and for a row of Q its sum g:
//   score_j = s_j (u_j . q) + z_j g,    out = sum_j (p_j t_j) u_j + (sum_j p_j y_j) for every element alike
// so only the numbers themselves go through the matrix products, exactly, and what belongs to a position is two operations a score.
//
// A number is used as it lies in the word.  f16 holds u 2^-24 as the bits of u, and 16 u 2^-24 as the bits of 16 u: a mask of a word with eight numbers
// gives two elements of a factor, and a shift by 8 and the same masks the others: five instructions for eight elements (eleven, where numbers are made by adding to a
// larger one and taking that off again, or one of 128 that stays in the sums).  Products and sums are f32 and hold 2^-48.  The two kinds of numbers (u and 16 u) have sums of their own in
// the scores and rows of their own in O^T.
// Q is in f16 as it is, or a row of bf16 times a power of two that brings its largest element to 2^15 or more: an element is resolved to 2^-39 of the
// row's largest, which is below what the sum g keeps of it.
// p t h is rounded to f16, with h a power of two a row: it follows the largest p t seen, so that the scales may have any size (2^-60 to 2^90) beside one another.
#pragma once

#include <type_traits>

#include "paged_device.cuh"

namespace l2 {

constexpr float KR4_TOP = 64.0f;       // h is chosen so that the largest p t h is between this and twice as much ...
constexpr uint32_t KR4_LIMIT = 0x7800;  // ... and again where one reaches 2^15 (in f16)

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t max_f16(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// 2^k with KR4_TOP <= w 2^k < 2 KR4_TOP, within 2^-100 .. 2^64 (w = 0: what it was)
__device__ __forceinline__ float kr4_factor(float w, float before) {
    const int e = (int)(__float_as_uint(w) >> 23);  // (w is not negative; NaN and infinity: 255)
    return w > 0.0f ? __uint_as_float((uint32_t)min(max(127 + 6 + 127 - e, 27), 191) << 23) : before;
}

// For a row of bf16 whose largest element is `most`: a power of two that brings it to 2^15 .. 2^16 (f16 holds 65504, bf16 goes up to 65280 there), and its inverse, both normal
// numbers.  (Elements of 2^118 and more are beyond f16 then, and the row gives NaN.)
__device__ __forceinline__ void kr4_q_factors(float most, float* up, float* by) {
    const int e = most > 0.0f ? min(max((int)(__float_as_uint(most) >> 23), 16), 244) : 142;
    *up = __uint_as_float((uint32_t)(127 + 127 + 15 - e) << 23);
    *by = __uint_as_float((uint32_t)(e - 15) << 23);
}

// What a warp keeps of its rows, as the threads have them: rows 8 nt + 2 c and 8 nt + 2 c + 1
template <int HD, int NT>
struct Kr4Rows {
    uint32_t q[HD / 32][NT][4];  // of 32 elements: the words of elements 8 c + {0, 4}, {2, 6}, {1, 5}, {3, 7}
    float by[NT][2], sum[NT][2]; // a score is `by` times (s (u . q) + z sum), in powers of two
    int pos[NT][2];
    float m[NT][2], l[NT][2], y[NT][2], h[NT][2];
    float o[HD / 16][NT][4];
};

// k_at, v_at: the tile's K and V in shared memory, `row` the first of the 32 positions in it, k_pair and v_pair those of this thread's first position (row + g8);
// j0 the position of the row `row + g8`.
template <int HD, int NT, class Offset, class Ldsm, class LdsmT, class Transpose>
__device__ __forceinline__ void kr4_step(const KvAttendParams& P, Kr4Rows<HD, NT>& r, uint32_t k_at, uint32_t v_at, int row, const uint32_t* k_pair, const uint32_t* v_pair, int j0,
                                         bool whole, float bias, float raise_by, Offset offset, Ldsm ldsm, LdsmT ldsm_t, Transpose transpose) {
    constexpr int CH = HD / 32, MB = 2;
    constexpr uint32_t LO = 0x000f000fu, HI = 0x00f000f0u;
    const int lane = threadIdx.x & 31;
    // ---- u . q of the positions g8 and g8 + 8 of 16, rows 2 c and 2 c + 1
    float s[MB][NT][4], s16[MB][NT][4];
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[mb][nt][i] = s16[mb][nt][i] = 0.0f;
#pragma unroll
    for (int c2 = 0; c2 < CH / 2; c2++)
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            uint32_t a[4];
            ldsm(a, k_at + offset(row + 16 * mb + (lane & 15), 2 * c2 + (lane >> 4)));
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t a0 = a[2 * x], a1 = a[2 * x + 1], b0 = a0 >> 8, b1 = a1 >> 8;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const uint32_t (&q)[4] = r.q[2 * c2 + x][nt];
                    mma_f16(s[mb][nt], a0 & LO, a1 & LO, b0 & LO, b1 & LO, q[0], q[1]);
                    mma_f16(s16[mb][nt], a0 & HI, a1 & HI, b0 & HI, b1 & HI, q[2], q[3]);
                }
            }
        }
    // ---- scores, in units of `by`
    auto sees = [&](int nt, int mb, int i) { return kv_sees(r.pos[nt][i & 1], j0 + 16 * mb + 8 * (i >> 1), P.window, P.sinks); };
    float most[NT][2], t[MB][2], y[MB][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) most[nt][0] = most[nt][1] = -INFINITY;
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t kw = k_pair[16 * mb + 8 * half], vw = v_pair[16 * mb + 8 * half];
            const float scale = kv_pair_scale(kw), zero = kv_pair_zero(kw);
            t[mb][half] = kv_pair_scale(vw);
            y[mb][half] = kv_pair_zero(vw);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float& x = s[mb][nt][2 * half + e];
                    x = fmaf(scale, fmaf(s16[mb][nt][2 * half + e], 0.0625f, x), zero * r.sum[nt][e]);
                }
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
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 4; i++) most[nt][i & 1] = fmaxf(most[nt][i & 1], s[mb][nt][i]);
    // ---- a row's maximum is raised, and what was summed is scaled (seldom)
    bool raise = false;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) raise |= most[nt][e] * r.by[nt][e] - bias > r.m[nt][e] + raise_by;
    auto over_lanes = [](float x) {  // the largest of the lanes that have the row
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
    };
    auto scale_o = [&](int nt, int e, float by) {
#pragma unroll
        for (int mt = 0; mt < HD / 16; mt++) { r.o[mt][nt][e] *= by; r.o[mt][nt][e + 2] *= by; }
    };
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float x = over_lanes(most[nt][e]) * r.by[nt][e] - bias;
                const bool up = x > r.m[nt][e] + raise_by;
                const float m1 = up ? x : r.m[nt][e];  // (a row's result does not depend on the others)
                const KvScale f(m1 == -INFINITY ? 0.0f : r.m[nt][e] - m1);
                r.m[nt][e] = m1;
                r.l[nt][e] = f(r.l[nt][e]);
                r.y[nt][e] = f(r.y[nt][e]);
                float w = 0.0f;
#pragma unroll
                for (int mb = 0; mb < MB; mb++)
#pragma unroll
                    for (int half = 0; half < 2; half++) if (whole || sees(nt, mb, 2 * half + e)) w = fmaxf(w, fabsf(kv_exp2(fmaf(s[mb][nt][2 * half + e], r.by[nt][e], -m1)) * t[mb][half]));
                w = over_lanes(w);
                const float h1 = up ? kr4_factor(w, r.h[nt][e]) : r.h[nt][e];
#pragma unroll
                for (int mt = 0; mt < HD / 16; mt++) { r.o[mt][nt][e] = f(r.o[mt][nt][e]); r.o[mt][nt][e + 2] = f(r.o[mt][nt][e + 2]); }
                scale_o(nt, e, h1 / r.h[nt][e]);
                r.h[nt][e] = h1;
            }
    }
    // ---- probabilities, and with the scales of V (what a row does not see may have any)
    uint32_t top = 0;
    auto probabilities = [&](auto is_whole) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float ref = r.m[nt][e] == -INFINITY ? 0.0f : r.m[nt][e];
#pragma unroll
                for (int mb = 0; mb < MB; mb++)
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        float& x = s[mb][nt][2 * half + e];
                        x = kv_exp2(fmaf(x, r.by[nt][e], -ref));
                        r.l[nt][e] += x;
                        if (decltype(is_whole)::value || sees(nt, mb, 2 * half + e)) {
                            r.y[nt][e] = fmaf(x, y[mb][half], r.y[nt][e]);
                            x *= t[mb][half];
                        }
                    }
            }
    };
    if (whole) probabilities(std::true_type());
    else probabilities(std::false_type());
    uint32_t pb[MB][NT][2];
    auto pack = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int mb = 0; mb < MB; mb++)
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    pb[mb][nt][half] = pack16<false>(s[mb][nt][2 * half] * r.h[nt][0], s[mb][nt][2 * half + 1] * r.h[nt][1]);
                    top = max_f16(top, pb[mb][nt][half] & 0x7fff7fffu);
                }
    };
    pack();
    if (__any_sync(0xffffffffu, (top & 0xffffu) >= KR4_LIMIT || (top >> 16) >= KR4_LIMIT)) {  // (seldom: a scale of V larger than those before)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float w = 0.0f;
#pragma unroll
                for (int mb = 0; mb < MB; mb++)
#pragma unroll
                    for (int half = 0; half < 2; half++) w = fmaxf(w, fabsf(s[mb][nt][2 * half + e]));
                w = over_lanes(w);
                const float h1 = w * r.h[nt][e] >= 32768.0f * 0.99f ? kr4_factor(w, r.h[nt][e]) : r.h[nt][e];
                scale_o(nt, e, h1 / r.h[nt][e]);
                r.h[nt][e] = h1;
            }
        pack();
    }
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) { pb[mb][nt][0] = transpose(pb[mb][nt][0]); pb[mb][nt][1] = transpose(pb[mb][nt][1]); }
    // ---- O^T += U^T P^T.  Of 32 elements (a chunk) the product 2 chunk + i has elements 4 g8 + 2 i in its rows g8, 4 g8 + 2 i + 1 in its rows g8 + 8
#pragma unroll
    for (int mb = 0; mb < MB; mb++)
#pragma unroll
        for (int c2 = 0; c2 < CH / 2; c2++) {
            uint32_t a[4];
            ldsm_t(a, v_at + offset(row + 16 * mb + (lane & 7) + 8 * (lane >> 4), 2 * c2 + ((lane >> 3) & 1)));
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

}  // namespace l2
