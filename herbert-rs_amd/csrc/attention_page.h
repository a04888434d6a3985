// Pieces of the bfloat16 attention kernels that work on pages of 64 keys with the 32x32x16 MFMA: the order of a page's keys, the
// masked online softmax of a page, and the products of a step whose pages lie in LDS.
#pragma once
#include "common.h"
#include "lds_read.h"
#include <math.h>

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

#define PAGE 64

// MFMA row rho (0..31) of a key block -> key within the block.
// rho = 16h + 8b + 4g + r  ->  16h + 8g + 4b + r  (h, b, g in {0,1}, r in 0..3)
__device__ __forceinline__ int perm(int rho) {
    return (rho & 16) | ((rho & 4) << 1) | ((rho & 8) >> 1) | (rho & 3);
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Capped scores: s <- cap tanh(s / cap), in the units of the raw dot products (cap = softcap / scale, so that
// the scaled score is softcap tanh(scale s / softcap)). tanh t = 1 - 2 / (1 + e^(2t)): e^(2t) infinite gives 1,
// zero gives -1.
__device__ __forceinline__ void cap_scores(f32x16 st[2], float cap) {
    const float k = 2.0f * 1.4426950408889634f / cap;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float e = fast_exp2(st[kb][i] * k);
            st[kb][i] = cap - 2.0f * cap * __builtin_amdgcn_rcpf(1.0f + e);
        }
}

// accumulator element i of lane group g2 of key block kb -> key within the page
__device__ __forceinline__ int acc_key(int kb, int g2, int i) { return kb * 32 + 16 * (i >> 3) + 8 * g2 + (i & 7); }

// One page of scores: mask, online-softmax update, P^T as MFMA operands.
// st[kb]: S^T accumulators (raw dot products). c = scale * log2(e).
// Keys k with lo <= page0 + k <= hi (and the sequence's first `keep`) are visible; MASKED = false: the caller
// knows that all are.
// m is the reference of the exponents, not always the maximum: it is moved up (and the sums so
// far scaled by corr < 1) only when a score exceeds it by more than 8 / c, that is when a
// probability would exceed 2^8 times the largest so far; till then corr is 1 and the caller
// need not touch its sums. Any reference gives the same quotient in the end.
__device__ __forceinline__ float max_with_other_half(float v) {
    // lanes i and i ^ 32 exchange their values without a trip through LDS
    const unsigned u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

#define RESCALE_LOG2 8.0f

// A sink: a score without key or value that the softmax's denominator of a head also holds, exp(sink),
// unscaled, once. It joins the sum at the end, in the units of the reference m that the sum was taken
// against (raw scores; c = scale * log2 e): 2^(sink * log2 e - m c). m lags behind the largest score by
// at most RESCALE_LOG2, so the share neither overflows nor loses digits that count; an infinite share
// (a sink far above every score) gives the output 0, its limit.
__device__ __forceinline__ float sink_share(float sink, float m, float c) {
    return fast_exp2(sink * 1.4426950408889634f - (m == -INFINITY ? 0.f : m * c));
}
template <bool MASKED>
__device__ __forceinline__ void softmax_page(f32x16 st[2], int g2, int page0, int lo, int hi, float c,
                                             float& m, float& l, float& corr, bf16x8 pb[2][2], int keep = 0) {
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (MASKED) {
                const int key = page0 + acc_key(kb, g2, i);
                st[kb][i] = ((key >= lo || key < keep) && key <= hi) ? st[kb][i] : -INFINITY;
            }
            mx = fmaxf(mx, st[kb][i]);
        }
    mx = max_with_other_half(mx);
    corr = 1.0f;
    if ((mx - m) * c > RESCALE_LOG2 || m == -INFINITY) {       // (-inf) - (-inf) is NaN: compares false
        const float m_new = (mx == -INFINITY) ? m : mx;
        corr = (m == -INFINITY) ? 0.f : fast_exp2((m - m_new) * c);
        m = m_new;
    }
    const float mc = (m == -INFINITY) ? 0.f : m * c;
    float sum = 0.f;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float p = fast_exp2(fmaf(st[kb][i], c, -mc));
            sum += p;
            pb[kb][i >> 3][i & 7] = (__bf16)p;
        }
    l = l * corr + sum;      // this lane's keys only; the two halves are added at the end
}

// oacc *= corr, unless corr is 1 in every lane
template <int NACC>
__device__ __forceinline__ void rescale(f32x16 (&oacc)[NACC], float corr) {
    if (__builtin_amdgcn_ballot_w64(corr != 1.0f) == 0) return;
#pragma unroll
    for (int d = 0; d < NACC; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[d][i] *= corr;
}

// The first half of softmax_page alone: mask, the page's largest score, the reference moved up if
// need be. Returns m * c (what is taken off the scaled scores), corr as softmax_page does.
template <bool MASKED>
__device__ __forceinline__ float softmax_reference(f32x16 st[2], int g2, int page0, int lo, int hi, float c,
                                                   float& m, float& corr, int keep = 0) {
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (MASKED) {
                const int key = page0 + acc_key(kb, g2, i);
                st[kb][i] = ((key >= lo || key < keep) && key <= hi) ? st[kb][i] : -INFINITY;
            }
            mx = fmaxf(mx, st[kb][i]);
        }
    mx = max_with_other_half(mx);
    corr = 1.0f;
    if ((mx - m) * c > RESCALE_LOG2 || m == -INFINITY) {
        const float m_new = (mx == -INFINITY) ? m : mx;
        corr = (m == -INFINITY) ? 0.f : fast_exp2((m - m_new) * c);
        m = m_new;
    }
    return (m == -INFINITY) ? 0.f : m * c;
}

// What a lane needs to find its operands in the LDS stages of a page's keys and values.
struct PrefillLane {
    int c32, g2, krow, k_read[2], v_swz;
};

// The matrix products of one step of the prompt kernels, in the order in which they are issued:
// the scores of the next page S (HD / 8 of them: k-step j / 2 of key block j % 2) and this page's
// P V (four groups of 8 probabilities x HD / 32 blocks of the output). Between them go the
// exponentials, one group of 8 ahead of the P V products that use it, so that the vector units
// work in the shadow of the matrix cores within the wave itself: a wave issues in order, and a
// run of MFMAs followed by a run of exponentials would leave each unit idle in turn.
//   phase 0:        S[0, Q)                                 exp of group 0
//   phase g = 1..3: S[g Q, (g + 1) Q), P V of group g - 1   exp of group g
//   phase 4:        P V of group 3
// with Q = HD / 32. The LDS operand of a product is read AHEAD products before it is used.
// kst: the stage of the next page's keys; vst: the stage of this page's values. After the last
// page the scores "of the next" are worked out all the same, from whatever that stage holds,
// and never looked at: a second copy of the code without them costs more registers than a wave has.
// STARTED: nxt already holds what the scores start from (else zero).
template <int HD, bool STARTED = false>
__device__ __forceinline__ void prefill_step_products(const bf16* kst, const bf16* vst, f32x16 (&st)[2],
                                                      f32x16 (&nxt)[2], f32x16 (&oacc)[HD / 32],
                                                      const bf16x8 (&qreg)[HD / 16], const PrefillLane& ln, float c,
                                                      float mc, float corr, float& l) {
    constexpr int Q = HD / 32, NM = 8 * Q, AHEAD = 3;
    const int c32 = ln.c32, g2 = ln.g2, krow = ln.krow, v_swz = ln.v_swz;
    // product n of the step: is it a score product, and which
    auto is_s = [](int n) { return n < Q || (n < 7 * Q && (n - Q) % (2 * Q) < Q); };
    auto s_index = [](int n) { return n < Q ? n : ((n - Q) / (2 * Q) + 1) * Q + (n - Q) % (2 * Q); };
    auto pv_group = [](int n) { return n < 7 * Q ? (n - Q) / (2 * Q) : 3; };
    auto pv_block = [](int n) { return n < 7 * Q ? (n - Q) % (2 * Q) - Q : n - 7 * Q; };
    constexpr int KRPB = 128 / HD > 0 ? 128 / HD : 1;
    // (an address is a lane's own part, shared by the two key blocks of a k-step and by the output
    // blocks of a group of probabilities, plus a constant that goes into the instruction)
    auto operand = [&](auto n_tag) -> bf16x8 {
        constexpr int n = decltype(n_tag)::value;
        if constexpr (is_s(n)) {
            constexpr int j = s_index(n), ks = j / 2, kb = j % 2;
            return lds_read_ahead<kb * 32 * HD * 2>(kst + krow * HD + (((2 * ks + g2) ^ ln.k_read[0]) * 8));
        } else {
            constexpr int g = pv_group(n), d = pv_block(n), kb = g >> 1, h2 = g & 1;
            return lds_read_ahead<d * 32 * PAGE * 2>(vst + c32 * PAGE + (((kb * 4 + h2 * 2 + g2) ^ v_swz) * 8));
        }
    };
    (void)KRPB;
    if (!STARTED) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) nxt[kb][e] = 0.f;
    }
    bf16x8 ops[NM];
    bf16x8 pb[4];
    float sum = 0.f;
    // exponential e (0..7) of group g: element 8 * (g & 1) + e of key block g >> 1
    auto exponential = [&](int g, int e) {
        const float p = fast_exp2(fmaf(st[g >> 1][8 * (g & 1) + e], c, -mc));
        sum += p;
        pb[g][e] = (__bf16)p;
    };
    static_for<0, AHEAD>([&](auto t) { ops[decltype(t)::value] = operand(t); });
    static_for<0, NM>([&](auto t) {
        constexpr int n = decltype(t)::value;
        if constexpr (n + AHEAD < NM) ops[n + AHEAD] = operand(std::integral_constant<int, n + AHEAD>{});
        // the reads behind product n's own may still be on their way: AHEAD of them, fewer at the end
        lds_wait<(n + AHEAD < NM ? AHEAD : NM - 1 - n)>(ops[n]);
        if constexpr (is_s(n)) {
            constexpr int j = s_index(n);
            nxt[j % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ops[n], qreg[j / 2], nxt[j % 2], 0, 0, 0);
        } else {
            constexpr int d = pv_block(n);
            oacc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ops[n], pb[pv_group(n)], oacc[d], 0, 0, 0);
        }
        // the exponentials that go with this product: those of phase g are dealt out over the
        // phase's products (phase 0 has Q of them, the others 2 Q)
        if constexpr (n < 7 * Q) {
            constexpr int g = n < Q ? 0 : (n - Q) / (2 * Q) + 1;
            constexpr int in_phase = n < Q ? n : (n - Q) % (2 * Q), of = n < Q ? Q : 2 * Q;
#pragma unroll
            for (int e = in_phase * 8 / of; e < (in_phase + 1) * 8 / of; ++e) exponential(g, e);
        }
        __builtin_amdgcn_sched_barrier(0);
    });
    l = l * corr + sum;      // this lane's keys only; the two halves are added at the end
}
