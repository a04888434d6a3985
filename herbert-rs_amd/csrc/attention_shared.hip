// Attention of a step whose sequences share pages of the cache: a page that several sequences hold is read once for all
// of them.
//
// The host cuts the step into items: some tokens (rows) x some neighbouring pages that all of them see through the same page table. A
// sequence's pages lie in several items (those of the whole batch, of its branch, its own), so an item leaves for
// every (row, query head) of its own a partial result, the reference m of the exponents, the sum l of 2^((s - m) c) and the
// output O = sum 2^((s - m) c) v, and a second kernel adds a token's up:
//   out = sum_i 2^((m_i - M) c) O_i / (sum_i 2^((m_i - M) c) l_i + the sink's share),  M = max m_i, c = scale * log2 e.
// The columns of an item are (row, head of the group): with a group of G query heads to a kv head, 32 / G sequences fill the
// 32 columns of a matrix product that one sequence alone leaves mostly empty.
//
// Cache layout as in the other attention kernels: keys [page, kv head, 64 tokens, hd], values [page, kv head, hd, 64 tokens].
// In xigh/herbert-rs every sequence has a cache of its own (crates/backends/backend_common/src/kv_cache.rs:270-273) and
// attends over it alone; the sums are those of crates/backends/backend_common/src/attention_common.rs:20-124.
#include "attention_page.h"
#include "mfma_f32.h"

HB_MODULE_ERROR_SLOT()

// What an item says, 8 numbers each: its first row in the order of the rows, how many (0: nothing here), the sequence whose
// page table names its pages, its first page and the one behind its last, its first partial result.
#define ITEM_INTS 8
struct Item {
    int row0, rows, seq, page0, page1, part0;
    __device__ __forceinline__ explicit Item(const int* p)
        : row0(p[0]), rows(p[1]), seq(p[2]), page0(p[3]), page1(p[4]), part0(p[5]) {}
};

// ---------------------------------------------------------------- bfloat16
// The values of a page that some column does not see whole, before their product: those of keys that no column sees are whatever lay
// in the page and become zeros, since a weight of zero does not hide what is not finite. (va: rows d * 32 + c32, keys kb * 32 +
// h2 * 16 + g2 * 8 + e.)
template <int HD>
__device__ __forceinline__ void hide_values(bf16x8 (&va)[HD / 32][2][2], int page0, int g2, int seen_last) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
            const int seen = seen_last + 1 - (page0 + kb * 32 + h2 * 16 + g2 * 8);      // of the eight
            u32x4 keep;
#pragma unroll
            for (int i = 0; i < 4; ++i) keep[i] = seen >= 2 * i + 2 ? 0xffffffffu : seen == 2 * i + 1 ? 0xffffu : 0u;
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
                va[d][kb][h2] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, va[d][kb][h2]) & keep);
        }
}

// What is left of them that is not finite is taken out of the product as well and added here, one key after another, to the
// columns that see it. (pb: this lane's weights of its column; a row of the output is entry d * 32 + 8 (i / 4) + 4 g2 + i % 4.)
template <int HD>
__device__ __forceinline__ void add_not_finite(bf16x8 (&va)[HD / 32][2][2], const bf16x8 (&pb)[2][2], f32x16 (&oacc)[HD / 32],
                                               const bf16* values, int page0, int pos, int c32, int g2) {
    bool any = false;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool finite = fabsf((float)va[d][kb][h2][e]) < INFINITY;
                    any |= !finite;
                    va[d][kb][h2][e] = finite ? va[d][kb][h2][e] : (__bf16)0.f;
                }
    if (__builtin_amdgcn_ballot_w64(any) == 0) return;
#pragma unroll 1
    for (int j = 0; j < PAGE; ++j) {
        const int kb = j >> 5, h2 = (j >> 4) & 1, from = c32 + 32 * ((j >> 3) & 1), e = j & 7;
        float w = 0.f;
#pragma unroll
        for (int x = 0; x < 32; ++x)
            if (x == kb * 16 + h2 * 8 + e) w = (float)pb[x >> 4][(x >> 3) & 1][x & 7];
        w = __shfl(w, from, 64);
        if (page0 + j > pos) continue;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float v = hb_to_float(values[(d * 32 + 8 * (i >> 2) + 4 * g2 + (i & 3)) * PAGE + j]);
                if (!(fabsf(v) < INFINITY)) oacc[d][i] = fmaf(w, v, oacc[d][i]);
            }
    }
}

// A workgroup: an item x a kv head. Its four waves are as many tiles of 32 columns as the item fills (1, 2 or 4); where those are
// fewer than four the waves of a tile take the pages in turn and add up their results through LDS.
// S^T = K Q^T and O^T = V^T P^T as in the decode kernel: operands stream from memory into registers, P stays there.
template <int HD>
__global__ void __launch_bounds__(256)
attn_shared_kernel(const bf16* __restrict__ q, const bf16* __restrict__ k_cache, const bf16* __restrict__ v_cache,
                   float* __restrict__ partial_o, float* __restrict__ partial_ml, const int* __restrict__ items,
                   const int* __restrict__ order, const int* __restrict__ positions, const int* __restrict__ slots,
                   const int* __restrict__ page_table, int max_pages, int nq, int nkv, float c, float cap) {
    constexpr int HANDED = (HD / 2 + 2) * 64;                     // floats that a wave hands over
    extern __shared__ __attribute__((aligned(16))) float handed[];   // [3][HANDED]
    const int kvh = blockIdx.x % nkv;
    const Item it(items + (size_t)(blockIdx.x / nkv) * ITEM_INTS);
    if (it.rows == 0) return;
    const int G = nq / nkv, cols = it.rows * G;
    const int tiles = cols <= 32 ? 1 : cols <= 64 ? 2 : 4, phases = 4 / tiles;
    const int lane = threadIdx.x & 63, c32 = lane & 31, g2 = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = wave % tiles, phase = wave / tiles;
    const int col = tile * 32 + c32;
    const bool mine = col < cols;
    const int r = (mine ? col : cols - 1) / G, head = kvh * G + (mine ? col : cols - 1) % G;
    const int token = order[it.row0 + r];
    const int pos = positions[token];
    int seen_last = pos, seen_first = pos;                        // the last key that some, and that every column sees
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        seen_last = max(seen_last, __shfl_xor(seen_last, off, 64));
        seen_first = min(seen_first, __shfl_xor(seen_first, off, 64));
    }
    const int* pt = page_table + (size_t)slots[it.seq] * max_pages;
    const int page_end = tile * 32 < cols ? min(it.page1, seen_last / PAGE + 1) : 0;

    bf16x8 qreg[HD / 16];
    {
        const bf16* qrow = q + ((size_t)token * nq + head) * HD + g2 * (HD / 2);
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) qreg[s] = *(const bf16x8*)(qrow + s * 8);
    }
    f32x16 oacc[HD / 32];
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[d][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    const int krow = perm(c32);
    bf16x8 ka[2][HD / 16];
    bf16x8 va[HD / 32][2][2];
    auto load_keys = [&](int p) {
        const bf16* kp = k_cache + ((size_t)pt[p] * nkv + kvh) * PAGE * HD + g2 * (HD / 2);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int s = 0; s < HD / 16; ++s) ka[kb][s] = *(const bf16x8*)(kp + (kb * 32 + krow) * HD + s * 8);
    };
    auto load_values = [&](int p) {
        const bf16* vp = v_cache + ((size_t)pt[p] * nkv + kvh) * HD * PAGE + g2 * 8;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int h2 = 0; h2 < 2; ++h2) va[d][kb][h2] = *(const bf16x8*)(vp + (d * 32 + c32) * PAGE + kb * 32 + h2 * 16);
    };
    int p = it.page0 + phase;
    if (p < page_end) {
        load_keys(p);
        load_values(p);
    }
    for (; p < page_end; p += phases) {
        f32x16 st[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) st[kb][i] = 0.f;
#pragma unroll
            for (int s = 0; s < HD / 16; ++s)
                st[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[kb][s], qreg[s], st[kb], 0, 0, 0);
        }
        if (p + phases < page_end) load_keys(p + phases);
        float corr;
        bf16x8 pb[2][2];
        if (cap != 0.f) cap_scores(st, cap);
        const int page0 = p * PAGE;
        if (page0 + PAGE - 1 <= seen_first) {
            softmax_page<false>(st, g2, page0, 0, pos, c, m, l, corr, pb);
        } else {
            softmax_page<true>(st, g2, page0, 0, pos, c, m, l, corr, pb);
            hide_values<HD>(va, page0, g2, seen_last);
        }
        rescale(oacc, corr);
        if (page0 + PAGE - 1 > seen_first && seen_first != seen_last)
            add_not_finite<HD>(va, pb, oacc, v_cache + ((size_t)pt[p] * nkv + kvh) * HD * PAGE, page0, pos, c32, g2);
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int h2 = 0; h2 < 2; ++h2)
                    oacc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[d][kb][h2], pb[kb][h2], oacc[d], 0, 0, 0);
        if (p + phases < page_end) load_values(p + phases);
    }
    l += __shfl_xor(l, 32, 64);
    if (phases > 1) {
        if (phase > 0) {
            float* const hand = handed + (wave - tiles) * HANDED + lane;
            hand[0] = m;
            hand[64] = l;
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) hand[(2 + d * 16 + i) * 64] = oacc[d][i];
        }
        __syncthreads();
        if (phase > 0) return;
        float top = m;
        for (int f = 1; f < phases; ++f) top = fmaxf(top, handed[((f - 1) * tiles + tile) * HANDED + lane]);
        const float own = m == -INFINITY ? 0.f : fast_exp2((m - top) * c);
        l *= own;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) oacc[d][i] *= own;
        for (int f = 1; f < phases; ++f) {
            const float* const hand = handed + ((f - 1) * tiles + tile) * HANDED + lane;
            const float share = hand[0] == -INFINITY ? 0.f : fast_exp2((hand[0] - top) * c);
            l = fmaf(share, hand[64], l);
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) oacc[d][i] = fmaf(share, hand[(2 + d * 16 + i) * 64], oacc[d][i]);
        }
        m = top;
    }
    if (!mine) return;
    const size_t part = (size_t)(it.part0 + r) * nq + head;
    if (g2 == 0) {
        partial_ml[part * 2] = m;
        partial_ml[part * 2 + 1] = l;
    }
    float* const po = partial_o + part * HD;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int qd = 0; qd < 4; ++qd)
            *(f32x4*)(po + d * 32 + 8 * qd + 4 * g2) =
                f32x4{oacc[d][4 * qd], oacc[d][4 * qd + 1], oacc[d][4 * qd + 2], oacc[d][4 * qd + 3]};
}

// ---------------------------------------------------------------- float32
// A workgroup of four waves: an item x a kv head x 16 of its columns. The products are chains of fmaf on the matrix cores
// (mfma_f32.h), as in the float32 attention over pages of a sequence's own: a wave scores 16 of a page's 64 keys, the scores meet in LDS,
// and each wave owns a quarter of the head's entries of the output.
template <int NB>
__global__ void __launch_bounds__(256)
attn_shared_f32_kernel(const float* __restrict__ q, const float* __restrict__ k_cache, const float* __restrict__ v_cache,
                       float* __restrict__ partial_o, float* __restrict__ partial_ml, const int* __restrict__ items,
                       const int* __restrict__ order, const int* __restrict__ positions, const int* __restrict__ slots,
                       const int* __restrict__ page_table, int max_pages, int nq, int nkv, int hd, float scale, float softcap,
                       int col_tiles) {
    constexpr int DB = 4 * NB, QLD = 16 * DB + 4, SLD = PAGE + 4;
    __shared__ __attribute__((aligned(16))) float qs[16 * QLD], ss[16 * SLD];
    __shared__ float tops[4][16];
    const int kvh = blockIdx.x % nkv, col_tile = blockIdx.x / nkv % col_tiles;
    const Item it(items + (size_t)(blockIdx.x / nkv / col_tiles) * ITEM_INTS);
    if (it.rows == 0) return;
    const int G = nq / nkv, cols = it.rows * G, col0 = col_tile * 16;
    if (col0 >= cols) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, g4 = lane >> 4;
    // the queries, zeros beyond the head's entries and in columns that are nobody's, every 16 entries transposed
    for (int i = tid; i < 16 * 16 * DB; i += 256) {
        const int cl = col0 + i / (16 * DB), d = i % (16 * DB);
        float v = 0.f;
        if (cl < cols && d < hd) v = q[((size_t)order[it.row0 + cl / G] * nq + kvh * G + cl % G) * hd + d];
        qs[(i / (16 * DB)) * QLD + (d & ~15) + 4 * (d & 3) + ((d >> 2) & 3)] = v;
    }
    const int col = col0 + r;
    const bool mine = col < cols;
    const int row = (mine ? col : cols - 1) / G, head = kvh * G + (mine ? col : cols - 1) % G;
    const int pos = positions[order[it.row0 + row]];
    int seen_last = pos, seen_first = pos;
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
        seen_last = max(seen_last, __shfl_xor(seen_last, off, 64));
        seen_first = min(seen_first, __shfl_xor(seen_first, off, 64));
    }
    const int* pt = page_table + (size_t)slots[it.seq] * max_pages;
    const int page_end = min(it.page1, seen_last / PAGE + 1);
    f32x4 acc[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    f32x4 key[DB], val[NB][4];
    auto load_keys = [&](int p) {
        const float* at = k_cache + (((size_t)pt[p] * nkv + kvh) * PAGE + 16 * wave + r) * hd;
#pragma unroll
        for (int b = 0; b < DB; ++b) key[b] = load_quad<true>(at + (16 * b + 4 * g4 < hd ? 16 * b + 4 * g4 : 0), 4);
    };
    auto load_values = [&](int p) {
        const float* at = v_cache + ((size_t)pt[p] * nkv + kvh) * hd * PAGE + 4 * g4;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int d = 16 * (wave + 4 * i) + r;
#pragma unroll
            for (int b = 0; b < 4; ++b) val[i][b] = load_quad<true>(at + (d < hd ? d : 0) * PAGE + 16 * b, 4);
        }
    };
    if (it.page0 < page_end) {
        load_keys(it.page0);
        load_values(it.page0);
    }
    __syncthreads();
    for (int p = it.page0; p < page_end; ++p) {
        const int page0 = p * PAGE, next = p + 1 < page_end ? p + 1 : p;
        if (hd < 16 * DB)
#pragma unroll
            for (int b = 0; b < DB; ++b) key[b] = 16 * b + 4 * g4 < hd ? key[b] : f32x4{0.f, 0.f, 0.f, 0.f};
        f32x4 dots = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < DB; ++b) {
            transpose_quads(key[b]);
            const f32x4 qq = *(const f32x4*)&qs[r * QLD + 16 * b + 4 * g4];
#pragma unroll
            for (int s = 0; s < 4; ++s) dots = mfma_k4(key[b][s], qq[s], dots);
        }
        load_keys(next);
        dots *= scale;
        if (softcap > 0.f)
#pragma unroll
            for (int e = 0; e < 4; ++e) dots[e] = softcap * tanhf(dots[e] / softcap);
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            dots[e] = page0 + 16 * wave + 4 * g4 + e <= pos ? dots[e] : -INFINITY;
            top = fmaxf(top, dots[e]);
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (g4 == 0) tops[wave][r] = top;
        hb_workgroup_barrier();                       // (and the weights of the page before have been read)
        const float m_new = fmaxf(m, fmaxf(fmaxf(tops[0][r], tops[1][r]), fmaxf(tops[2][r], tops[3][r])));
        const float corr = m == -INFINITY ? 0.f : expf(m - m_new);
        m = m_new;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool there = dots[e] != -INFINITY;
            const float weight = expf(there ? dots[e] - m_new : 0.f);
            ss[r * SLD + 16 * wave + 4 * e + g4] = there ? weight : 0.f;
        }
        hb_workgroup_barrier();
        f32x4 w[4];                                   // this lane's share of its column: keys 16 b + 4 s + g4
#pragma unroll
        for (int b = 0; b < 4; ++b) w[b] = *(const f32x4*)&ss[r * SLD + 16 * b + 4 * g4];
        const f32x4 t = (w[0] + w[2]) + (w[1] + w[3]);
        float sum = (t[0] + t[2]) + (t[1] + t[3]);
        sum += __shfl_xor(sum, 32, 64);
        sum += __shfl_xor(sum, 16, 64);
        l = l * corr + sum;
        const bool masked = page0 + PAGE - 1 > seen_first;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            acc[i] *= corr;
            const int d0 = 16 * (wave + 4 * i);
            f32x4 (&v)[4] = val[i];
            // a key that no column sees, or an entry beyond the head: its value is whatever lay there, and a weight of zero
            // does not hide what is not finite
            if (masked || hd < 16 * DB)
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[b][e] = d0 + r < hd && page0 + 16 * b + 4 * g4 + e <= seen_last ? v[b][e] : 0.f;
            float nothing = 0.f;                      // (or NaN)
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) nothing = fmaf(v[b][e], 0.f, nothing);
            if (masked && __any(!(nothing == 0.f))) {
                // a value without a finite size that some columns see and others do not: one key after another
                const float* const at = v_cache + ((size_t)pt[p] * nkv + kvh) * hd * PAGE;
                for (int j = 0; j < PAGE; ++j) {
                    const int in = j & 15, s = in >> 2, k = in & 3;
                    const f32x4 wb = j < 16 ? w[0] : j < 32 ? w[1] : j < 48 ? w[2] : w[3];
                    const float mine_w = __shfl(s == 0 ? wb[0] : s == 1 ? wb[1] : s == 2 ? wb[2] : wb[3], 16 * k + r, 64);
                    if (page0 + j > pos) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (d0 + 4 * g4 + e < hd) acc[i][e] = fmaf(mine_w, at[(d0 + 4 * g4 + e) * PAGE + j], acc[i][e]);
                }
            } else {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    transpose_quads(v[b]);
#pragma unroll
                    for (int s = 0; s < 4; ++s) acc[i] = mfma_k4(v[b][s], w[b][s], acc[i]);
                }
            }
        }
        load_values(next);
    }
    if (!mine) return;
    const size_t part = (size_t)(it.part0 + row) * nq + head;
    if (wave == 0 && g4 == 0) {
        partial_ml[part * 2] = m;
        partial_ml[part * 2 + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = 16 * (wave + 4 * i) + 4 * g4 + e;
            if (d < hd) partial_o[part * hd + d] = acc[i][e];
        }
}

// ---------------------------------------------------------------- joining
// A wave a (token, query head): the partial results parts[part_start[t] ..] of the t-th row, in their order. T: the type that
// leaves; c: what a difference of references is multiplied by for a power of two (float32: natural units, expf).
template <class T, int E>
__global__ void __launch_bounds__(256)
attn_shared_join_kernel(const float* __restrict__ partial_o, const float* __restrict__ partial_ml, T* __restrict__ out,
                        const int* __restrict__ order, const int* __restrict__ part_start, const int* __restrict__ parts,
                        int n_rows, int nq, int hd, float c, const float* __restrict__ sinks) {
    constexpr bool EXACT = sizeof(T) == 4;
    const int lane = threadIdx.x & 63;
    const int at = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = at / nq, h = at % nq;
    if (t >= n_rows) return;
    const int first = part_start[t], n = part_start[t + 1] - first;
    auto weight = [&](float m, float top) { return m == -INFINITY ? 0.f : EXACT ? expf(m - top) : fast_exp2((m - top) * c); };
    float top = -INFINITY;
    for (int s = lane; s < n; s += 64) top = fmaxf(top, partial_ml[((size_t)parts[first + s] * nq + h) * 2]);
    top = hb_wave_max(top);
    float acc[E], total = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int s0 = 0; s0 < n; s0 += 64) {
        int part = 0;
        float w = 0.f, term = 0.f;
        if (s0 + lane < n) {
            part = parts[first + s0 + lane];
            const float2 ml = ((const float2*)partial_ml)[(size_t)part * nq + h];
            w = weight(ml.x, top);
            term = w * ml.y;
        }
        total += hb_wave_sum(term);
        const int here = n - s0 < 64 ? n - s0 : 64;
        for (int s = 0; s < here; ++s) {
            const float ws = __shfl(w, s, 64);
            const float* po = partial_o + ((size_t)__shfl(part, s, 64) * nq + h) * hd;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int d = E * lane + e;
                if (d < hd) acc[e] = fmaf(ws, po[d], acc[e]);
            }
        }
    }
    if (sinks) total += EXACT ? expf(sinks[h] - (top == -INFINITY ? 0.f : top)) : sink_share(sinks[h], top, c);
    const float inv = total > 0.f || total != total ? 1.0f / total : 0.f;
    T* const dst = out + ((size_t)order[t] * nq + h) * hd;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = E * lane + e;
        if (d < hd) dst[d] = hb_from_float<T>(acc[e] * inv);
    }
}

// q, out [T, nq hd]; keys [pages, nkv, 64, hd], values [pages, nkv, hd, 64]; one storage type. items [n_items, 8]; order [n_rows],
// part_start [n_rows + 1], parts [...]; partial_o [partial results, nq, hd], partial_ml [partial results, nq, 2]. max_rows: the most
// rows of an item. softcap 0: none; sinks [nq] or null.
extern "C" int hb_attn_shared(const void* q, const void* k_cache, const void* v_cache, void* out, int dtype, float* partial_o,
                              float* partial_ml, const int* items, int n_items, int max_rows, const int* order,
                              const int* part_start, const int* parts, int n_rows, const int* positions, const int* slots,
                              const int* page_table, int max_pages, int nq, int nkv, int hd, float scale, float softcap,
                              const float* sinks, hipStream_t stream) {
    HB_REQUIRE(n_rows > 0 && n_items > 0 && nq > 0 && nkv > 0 && nq % nkv == 0, "shared attention: empty input, or heads that do not group");
    HB_REQUIRE(scale > 0.f && softcap >= 0.f, "shared attention: the scale must be positive, a cap of the scores too");
    const int G = nq / nkv;
    const long long rows_of_heads = (long long)n_rows * nq;
    HB_REQUIRE(rows_of_heads <= 0x7fffffffLL - 4, "shared attention: too many rows for the grid");
    const dim3 join((unsigned)((rows_of_heads + 3) / 4));
    if (dtype == HB_BF16) {
        HB_REQUIRE(hd == 32 || hd == 64 || hd == 128, "shared attention: bfloat16 heads of 32, 64 or 128, not %d", hd);
        HB_REQUIRE((long long)max_rows * G <= 128, "shared attention: items of %d rows x %d heads exceed 128 columns", max_rows, G);
        HB_REQUIRE((long long)n_items * nkv <= 0x7fffffffLL, "shared attention: too many items for the grid");
        const float c = scale * 1.4426950408889634f, cap = softcap > 0.f ? softcap / scale : 0.f;
        const dim3 grid((unsigned)(n_items * nkv));
#define HB_SHARED(HD, E)                                                                                                     \
        {                                                                                                                    \
            constexpr int lds = 3 * (HD / 2 + 2) * 64 * 4;                                                                   \
            attn_shared_kernel<HD><<<grid, 256, lds, stream>>>((const bf16*)q, (const bf16*)k_cache, (const bf16*)v_cache,   \
                                                               partial_o, partial_ml, items, order, positions, slots,        \
                                                               page_table, max_pages, nq, nkv, c, cap);                      \
            HB_CHECK_LAUNCH("shared attention");                                                                             \
            attn_shared_join_kernel<bf16, E><<<join, 256, 0, stream>>>(partial_o, partial_ml, (bf16*)out, order, part_start, \
                                                                       parts, n_rows, nq, hd, c, sinks);                     \
        }
        if (hd == 32) HB_SHARED(32, 1)
        else if (hd == 64) HB_SHARED(64, 1)
        else HB_SHARED(128, 2)
#undef HB_SHARED
    } else if (dtype == HB_F32) {
        HB_REQUIRE(hd > 0 && hd <= 256 && hd % 4 == 0, "shared attention: float32 heads of up to 256 entries in whole quads, not %d", hd);
        HB_REQUIRE(((uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0, "shared attention: pages on 16-byte borders");
        const long long col_tiles = ((long long)max_rows * G + 15) / 16;
        HB_REQUIRE((long long)n_items * nkv * col_tiles <= 0x7fffffffLL, "shared attention: too many items for the grid");
        const dim3 grid((unsigned)(n_items * nkv * col_tiles));
#define HB_SHARED(NB, E)                                                                                                       \
        {                                                                                                                      \
            attn_shared_f32_kernel<NB><<<grid, 256, 0, stream>>>((const float*)q, (const float*)k_cache, (const float*)v_cache, \
                                                                 partial_o, partial_ml, items, order, positions, slots,        \
                                                                 page_table, max_pages, nq, nkv, hd, scale, softcap,           \
                                                                 (int)col_tiles);                                              \
            HB_CHECK_LAUNCH("shared attention");                                                                               \
            attn_shared_join_kernel<float, E><<<join, 256, 0, stream>>>(partial_o, partial_ml, (float*)out, order, part_start, \
                                                                        parts, n_rows, nq, hd, 0.f, sinks);                    \
        }
        if (hd <= 64) HB_SHARED(1, 1)
        else if (hd <= 128) HB_SHARED(2, 2)
        else HB_SHARED(4, 4)
#undef HB_SHARED
    } else {
        HB_REQUIRE(false, "shared attention: unknown dtype %d", dtype);
    }
    HB_CHECK_LAUNCH("shared attention: joining");
    return 0;
}
