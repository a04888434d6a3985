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

// What an item says, 8 numbers each: its first row in the order of the rows, how many (0: nothing here), the slot whose
// page table names its pages, its first page and the one behind its last, where its rows' places among the partial results are
// listed, whether there is a place in its pages that one of its rows does not see, and a number that is not used.
#define ITEM_INTS 8
struct Item {
    int row0, rows, slot, page0, page1, list0, masked;
    __device__ __forceinline__ explicit Item(const int* p)
        : row0(p[0]), rows(p[1]), slot(p[2]), page0(p[3]), page1(p[4]), list0(p[5]), masked(p[6]) {}
};

// ---------------------------------------------------------------- bfloat16
// A workgroup is an item x a kv head, four waves. S^T = K Q^T and O^T = V^T P^T as in the other attention kernels.
//
// Wide items (more than 64 columns, every page seen whole): a wave is a tile of 32 columns, the pages go through a ring of LDS stages
// once for all four, the next page's scores on the matrix cores while this one's exponentials are worked out.
// Narrow ones: operands stream from memory into registers, half a page at a time, in 16 x 16 x 32 products, whose operands are 64
// neighbouring bytes of a row; a wave has 16 or 32 columns, the waves of a tile (four, or two each of two tiles) take the pages
// in turn and add up their results through LDS. A sequence's own rows over the pages that they see in part (CAUSAL) are
// narrow, too, in tiles of 16 columns. In steps of short contexts a sequence is an item and its result the row's (out), nothing is joined.
// 256 registers and 68 KB of LDS: two workgroups a CU, so that items that wait for memory and items that compute overlap.
// Scores, exponentials, their sums and the outputs are float32. An exponential is rounded to bfloat16 (2^-8 of itself at most) before it meets its value, since the products
// take bfloat16 alone, and a head and a rest of it would double the second half of the matrix work; its sum is that of the unrounded ones. Against 64 bits results
// are off by 0.0017 to 0.0023 of their root mean square, where the exact ones rounded to bfloat16 are by 0.0017. No sum's order changes: the same call gives the same bits.
// 8/32 heads of 128, microseconds (join apart, caches warm; cold, join and all: 97, 38, 23.4 and 14.5): 128 answers to 32,768 tokens 86 to 92 (0.75 PFLOP/s; the products are 39 % of the time and the softmax's vector
// work 37 %, partly side by side; with 64 columns a wave 120, since registers were moved between files), 64 to 8,192 29 (108 MB at 3.7 TB/s), 48 questions
// behind 6 texts 20.6 (82 MB at 4.0 TB/s), 8 answers to 4,096 10.4, where a page a wave is a chain of loads. The first form, every item
// streamed from memory in 32 x 32 x 16 products: 280 and 77 with the join, where these take 97 and 34.
template <int HD>
struct SharedSizes {
    static constexpr int STAGE = PAGE * HD;
    static constexpr int RING = 4 * STAGE * 2;                                     // two stages of keys, two of values
    static constexpr int SUMS = 4 * 2 * (HD / 16) * 64 * 16;                       // four waves' sums
    static constexpr int HANDED = SUMS + 4 * 2 * 64 * 8;                           // and their references and denominators
    static constexpr int LDS = RING > HANDED ? RING : HANDED;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float max_of_rows(float v) {        // over the four lanes 16 apart
    const unsigned u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return max_with_other_half(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

// What the kernel's two forms share.
struct SharedArgs {
    const bf16 *q, *k_cache, *v_cache;
    float *partial_o, *partial_ml;
    const int *order, *positions, *parts;
    int nq, nkv, kvh, G;
    float c, cap;
    bf16* out;                          // where every row is one item's: its result; else null
    const float* sinks;
};

// A narrow item's wave: NT tiles of 16 columns from column col0 on, every phases-th page of the item from the phase-th on. With more than one
// phase all waves of the workgroup come here (there is a barrier).
// An operand of half a page: keys (row 4 g + i of block b: key 8 g + 4 b + i, so that a lane's scores are 8 neighbouring keys), g = lane / 16.
template <int HD, int NT, bool CAUSAL>
__device__ __forceinline__ void narrow_item(const SharedArgs& A, const Item& it, const int* pt, int cols, int col0, int phase, int phases,
                                            int wave, int lane, char* lds) {
    constexpr int STEPS = HD / 32, BLOCKS = HD / 16, STAGE = PAGE * HD;
    constexpr int DEPTH = NT == 1 && !CAUSAL ? 2 : 1;    // halves of a page in flight
    const int c16 = lane & 15, g = lane >> 4;
    int token[NT], head[NT], place[NT], pos[NT];
    bool mine[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int col = col0 + 16 * t + c16;
        mine[t] = col < cols;
        const int r = (mine[t] ? col : cols - 1) / A.G;
        head[t] = A.kvh * A.G + (mine[t] ? col : cols - 1) % A.G;
        token[t] = A.order[it.row0 + r];
        place[t] = A.parts[it.list0 + r];
        pos[t] = 0x7ffffffe;
    }
    bf16x8 ka[DEPTH][2][STEPS], va[DEPTH][BLOCKS], qreg[NT][STEPS];
    const int k_lane = (8 * (c16 >> 2) + (c16 & 3)) * HD + g * 8, v_lane = c16 * PAGE + g * 8;
    // (h: half of a page, 2 x its place among the item's pages + which)
    auto load_keys = [&](int page, int h, bf16x8 (&k)[2][STEPS]) {
        const bf16* kp = A.k_cache + ((size_t)page * A.nkv + A.kvh) * STAGE + (h & 1) * 32 * HD + k_lane;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int s = 0; s < STEPS; ++s) k[b][s] = *(const bf16x8*)(kp + b * 4 * HD + s * 32);
    };
    auto load_values = [&](int page, int h, bf16x8 (&v)[BLOCKS]) {
        const bf16* vp = A.v_cache + ((size_t)page * A.nkv + A.kvh) * STAGE + (h & 1) * 32 + v_lane;
#pragma unroll
        for (int d = 0; d < BLOCKS; ++d) v[d] = *(const bf16x8*)(vp + d * 16 * PAGE);
    };
    const int halves = col0 < cols ? 2 * (it.page1 - it.page0) : 0;
    auto next = [&](int h) { return (h & 1) ? h + 2 * phases - 1 : h + 1; };      // this wave's next half
    int h = 2 * phase;
    if (h < halves) {                                     // (a page is two halves: the second is there too)
        const int page = pt[it.page0 + phase];
        load_keys(page, h, ka[0]);
        load_values(page, h, va[0]);
        if constexpr (DEPTH == 2) {
            load_keys(page, h + 1, ka[1]);
            load_values(page, h + 1, va[1]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const bf16* qrow = A.q + ((size_t)token[t] * A.nq + head[t]) * HD + g * 8;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) qreg[t][s] = *(const bf16x8*)(qrow + s * 32);
    }
    int seen_last = 0x7ffffffe;                           // what the last of the columns sees
    if (it.masked) {
        seen_last = -1;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            pos[t] = A.positions[token[t]];
            seen_last = max(seen_last, pos[t]);
        }
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) seen_last = max(seen_last, __shfl_xor(seen_last, off, 64));
    }
    uint32_t odd = 0;
    f32x4 oacc[NT][BLOCKS];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int d = 0; d < BLOCKS; ++d) oacc[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    auto half = [&](auto more_tag, bf16x8 (&k)[2][STEPS], bf16x8 (&v)[BLOCKS]) {
        constexpr bool MORE = decltype(more_tag)::value;  // there is a half whose operands take these registers next
        const int key0 = it.page0 * PAGE + h * 32;
        const int following = DEPTH == 2 ? h + 2 * phases : next(h), page = MORE ? pt[it.page0 + (following >> 1)] : 0;
        f32x4 st[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                st[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < STEPS; ++s) st[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[b][s], qreg[t][s], st[t][b], 0, 0, 0);
            }
        __builtin_amdgcn_sched_barrier(0);
        if (MORE) load_keys(page, following, k);
        __builtin_amdgcn_sched_barrier(0);
        bf16x8 pb[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float x = st[t][i >> 2][i & 3];
                if (A.cap != 0.f) x = A.cap - 2.0f * A.cap * __builtin_amdgcn_rcpf(1.0f + fast_exp2(x * (2.0f * 1.4426950408889634f / A.cap)));
                x = key0 + 8 * g + i <= pos[t] ? x : -INFINITY;
                st[t][i >> 2][i & 3] = x;
                mx = fmaxf(mx, x);
            }
            mx = max_of_rows(mx);
            float corr = 1.0f;                            // (the reference moves up lazily: see softmax_page)
            if ((mx - m[t]) * A.c > RESCALE_LOG2 || m[t] == -INFINITY) {
                const float m_new = (mx == -INFINITY) ? m[t] : mx;
                corr = (m[t] == -INFINITY) ? 0.f : fast_exp2((m[t] - m_new) * A.c);
                m[t] = m_new;
            }
            const float mc = (m[t] == -INFINITY) ? 0.f : m[t] * A.c;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float p = fast_exp2(fmaf(st[t][i >> 2][i & 3], A.c, -mc));
                sum += p;
                pb[t][i] = (__bf16)p;
            }
            l[t] = l[t] * corr + sum;
            if (__builtin_amdgcn_ballot_w64(corr != 1.0f) != 0)
#pragma unroll
                for (int d = 0; d < BLOCKS; ++d) oacc[t][d] *= corr;
        }
        // Values of keys that no column sees are whatever lay in the page and become zeros: a weight of zero does not hide what
        // is not finite. (The registers of the values themselves stay as they are: changed under a condition within this loop, the
        // compiler took some of them for temporaries.)
        const int seen = seen_last + 1 - (key0 + 8 * g);                 // of this lane's eight
        u32x4 keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) keep[i] = seen >= 2 * i + 2 ? 0xffffffffu : seen == 2 * i + 1 ? 0xffffu : 0u;
#pragma unroll
        for (int d = 0; d < BLOCKS; ++d) {
            u32x4 x = __builtin_bit_cast(u32x4, v[d]) & keep;
            if constexpr (CAUSAL) {
                // A value without a size that only some of the columns see is taken out of the product; the rows are marked, and
                // the kernel that joins looks for it. (An exponent of ones: its lowest bit added carries into the sign's
                // place; two numbers a word.)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t ones = (((x[i] & 0x7f807f80u) + 0x00800080u) >> 15) & 0x00010001u;
                    x[i] &= ~((ones << 16) - ones);
                    odd |= ones;
                }
            }
            const bf16x8 clean = __builtin_bit_cast(bf16x8, x);
#pragma unroll
            for (int t = 0; t < NT; ++t) oacc[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(clean, pb[t], oacc[t][d], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (MORE) load_values(page, following, v);
        __builtin_amdgcn_sched_barrier(0);
        h = next(h);
    };
    // Within the loop every load is issued, whatever the item: the compiler counts what is in flight, and waits for all of it where it cannot.
    __builtin_amdgcn_s_waitcnt(0x0f70);                   // (no load is left: of the queries, that is, which the loop then need not wait for)
    if (h < halves) {
        const std::true_type more;
        const std::false_type last;
        while ((DEPTH == 2 ? h + 2 * phases : next(h)) < halves) {
            half(more, ka[0], va[0]);
            if constexpr (DEPTH == 2) half(more, ka[1], va[1]);
        }
        half(last, ka[0], va[0]);
        if constexpr (DEPTH == 2) half(last, ka[1], va[1]);
    }
    const bool marked = CAUSAL && __builtin_amdgcn_ballot_w64(odd != 0) != 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        l[t] += __shfl_xor(l[t], 16, 64);
        l[t] += __shfl_xor(l[t], 32, 64);
        if (marked) l[t] = -l[t];                         // (a mark: sums are not below zero)
    }
    // (factor: of a whole result, see whole)
    auto leave = [&](int t, int d, float factor) {
        if (!mine[t]) return;
        if (!CAUSAL && A.out) {
            bf16x4 b;
#pragma unroll
            for (int e = 0; e < 4; ++e) b[e] = (__bf16)(oacc[t][d][e] * factor);
            *(bf16x4*)(A.out + ((size_t)token[t] * A.nq + head[t]) * HD + d * 16 + 4 * g) = b;
        } else {
            *(f32x4*)(A.partial_o + ((size_t)place[t] * A.nq + head[t]) * HD + d * 16 + 4 * g) = oacc[t][d];
        }
    };
    auto whole = [&](int t, float top, float total) {
        if (CAUSAL || !A.out) return 0.f;
        if (A.sinks) total += sink_share(A.sinks[head[t]], top, A.c);
        return total > 0.f || total != total ? 1.0f / total : 0.f;
    };
    auto leave_ml = [&](int t, float top, float total) {
        if (mine[t] && g == 0 && (CAUSAL || !A.out)) ((float2*)A.partial_ml)[(size_t)place[t] * A.nq + head[t]] = make_float2(top, total);
    };
    // the waves of a tile add up what they have: each the blocks that are its own (the x-th: phase x % PHASES)
    auto join = [&](auto phases_tag) {
        constexpr int PHASES = decltype(phases_tag)::value, TILES = 4 / PHASES;
        f32x4* const sums = (f32x4*)lds;                                 // [wave][tile and block][lane]
        float2* const ml = (float2*)(lds + SharedSizes<HD>::SUMS);       // [wave][tile][lane]
        const int tile = wave % TILES;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            ml[(wave * NT + t) * 64 + lane] = make_float2(m[t], l[t]);
#pragma unroll
            for (int d = 0; d < BLOCKS; ++d)
                if ((t * BLOCKS + d) % PHASES != phase) sums[((wave * NT + t) * BLOCKS + d) * 64 + lane] = oacc[t][d];
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float2 other[PHASES];
            float top = -INFINITY, total = 0.f;
#pragma unroll
            for (int f = 0; f < PHASES; ++f) {
                other[f] = ml[((f * TILES + tile) * NT + t) * 64 + lane];
                top = fmaxf(top, other[f].x);
            }
#pragma unroll
            for (int f = 0; f < PHASES; ++f) {
                other[f].x = other[f].x == -INFINITY ? 0.f : fast_exp2((other[f].x - top) * A.c);
                total = fmaf(other[f].x, CAUSAL ? fabsf(other[f].y) : other[f].y, total);
            }
            if constexpr (CAUSAL) {
                bool some = false;
#pragma unroll
                for (int f = 0; f < PHASES; ++f) some |= __float_as_uint(other[f].y) >> 31;
                total = some ? -total : total;
            }
            const float factor = whole(t, top, total);
#pragma unroll
            for (int d = 0; d < BLOCKS; ++d) {
                if ((t * BLOCKS + d) % PHASES != phase) continue;
                f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < PHASES; ++f) {
                    f32x4 x = oacc[t][d];
                    if (f != phase) x = sums[(((f * TILES + tile) * NT + t) * BLOCKS + d) * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = fmaf(other[f].x, x[e], o[e]);
                }
                oacc[t][d] = o;
                leave(t, d, factor);
            }
            if (phase == 0) leave_ml(t, top, total);
        }
    };
    if (phases == 4) {
        join(std::integral_constant<int, 4>{});
    } else if (phases == 2) {
        join(std::integral_constant<int, 2>{});
    } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            leave_ml(t, m[t], l[t]);
            const float factor = whole(t, m[t], l[t]);
#pragma unroll
            for (int d = 0; d < BLOCKS; ++d) leave(t, d, factor);
        }
    }
}

// A wide item's wave: 32 columns from column col0 on (active: some of them exist). All four waves come here.
template <int HD>
__device__ __forceinline__ void wide_item(const SharedArgs& A, const Item& it, const int* pt, int cols, int wave, int lane, bf16* lds) {
    constexpr int BLOCKS = HD / 32, STAGE = PAGE * HD;
    constexpr int KCH = HD / 8, KRPB = 128 / HD > 0 ? 128 / HD : 1, KROWS = 512 / HD, LOADS = HD / 32;
    const int c32 = lane & 31, g2 = lane >> 5, krow = perm(c32);
    bf16* const Ks = lds;
    bf16* const Vs = Ks + 2 * STAGE;
    const int n = it.page1 - it.page0;
    const bool active = wave * 32 < cols;
    int k_off[LOADS], v_off[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int instr = wave * LOADS + i;
        const int kr = instr * KROWS + lane / KCH;
        k_off[i] = kr * HD + (((lane % KCH) ^ ((kr / KRPB) % KCH)) * 8);
        const int vr = instr * 8 + lane / 8;
        v_off[i] = vr * PAGE + (((lane & 7) ^ ((vr >> 1) & 7)) * 8);
    }
    auto issue_keys = [&](int i, int stage) {
        const bf16* kp = A.k_cache + ((size_t)pt[it.page0 + i] * A.nkv + A.kvh) * STAGE;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) hb_load_to_lds(kp + k_off[j], Ks + stage * STAGE + (wave * LOADS + j) * 512);
    };
    auto issue_values = [&](int i, int stage) {
        const bf16* vp = A.v_cache + ((size_t)pt[it.page0 + i] * A.nkv + A.kvh) * STAGE;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) hb_load_to_lds(vp + v_off[j], Vs + stage * STAGE + (wave * LOADS + j) * 512);
    };
    issue_keys(0, 0);
    issue_values(0, 0);
    if (n > 1) issue_keys(1, 1);
    const int col = wave * 32 + c32;
    const bool mine = col < cols;
    const int r = (mine ? col : cols - 1) / A.G, head = A.kvh * A.G + (mine ? col : cols - 1) % A.G;
    const int token = A.order[it.row0 + r], place = A.parts[it.list0 + r];
    bf16x8 qreg[HD / 16];
    {
        const bf16* qrow = A.q + ((size_t)token * A.nq + head) * HD + g2 * 8;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) qreg[s] = *(const bf16x8*)(qrow + s * 16);
    }
    f32x16 oacc[BLOCKS];
#pragma unroll
    for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[d][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    PrefillLane ln;
    ln.c32 = c32;
    ln.g2 = g2;
    ln.krow = krow;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) ln.k_read[kb] = ((kb * 32 + krow) / KRPB) % KCH;
    ln.v_swz = (c32 >> 1) & 7;
    auto step = [&](auto parity_tag, int i, f32x16 (&st)[2], f32x16 (&nxt)[2]) {
        // landed, for every wave after the barrier: the values of this page and the keys of the next; and
        // nobody reads any more the stages that the next loads fill
        hb_wait_vmcnt<0>();
        hb_workgroup_barrier();
        if (i + 2 < n) issue_keys(i + 2, i & 1);
        if (i + 1 < n) issue_values(i + 1, (i + 1) & 1);
        if (!active) return;
        float corr;
        if (A.cap != 0.f) cap_scores(st, A.cap);
        const float mc = softmax_reference<false>(st, g2, 0, 0, 0, A.c, m, corr);
        rescale(oacc, corr);
        constexpr int PAR = decltype(parity_tag)::value;
        prefill_step_products<HD>(Ks + ((PAR + 1) & 1) * STAGE, Vs + PAR * STAGE, st, nxt, oacc, qreg, ln, A.c, mc, corr, l);
    };
    hb_wait_vmcnt<0>();
    hb_workgroup_barrier();
    f32x16 sa[2], sb[2];
    if (active) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) sa[kb][i] = 0.f;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const bf16x8 ka = *(const bf16x8*)(Ks + (kb * 32 + krow) * HD + (((2 * s + g2) ^ ln.k_read[kb]) * 8));
                sa[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka, qreg[s], sa[kb], 0, 0, 0);
            }
    }
    for (int i = 0; i < n; i += 2) {
        step(std::integral_constant<int, 0>{}, i, sa, sb);
        if (i + 1 < n) step(std::integral_constant<int, 1>{}, i + 1, sb, sa);
    }
    l += __shfl_xor(l, 32, 64);
    if (!mine) return;
    const size_t part = (size_t)place * A.nq + head;
    if (g2 == 0) ((float2*)A.partial_ml)[part] = make_float2(m, l);
    float* const po = A.partial_o + part * HD;
#pragma unroll
    for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
        for (int qd = 0; qd < 4; ++qd)
            *(f32x4*)(po + d * 32 + 8 * qd + 4 * g2) = f32x4{oacc[d][4 * qd], oacc[d][4 * qd + 1], oacc[d][4 * qd + 2], oacc[d][4 * qd + 3]};
}

// CAUSAL: there are items of several columns that see different places.
template <int HD, bool CAUSAL>
__global__ void __launch_bounds__(256, 2)
attn_shared_kernel(const bf16* __restrict__ q, const bf16* __restrict__ k_cache, const bf16* __restrict__ v_cache,
                   float* __restrict__ partial_o, float* __restrict__ partial_ml, const int* __restrict__ items,
                   const int* __restrict__ order, const int* __restrict__ parts, const int* __restrict__ positions,
                   const int* __restrict__ page_table, int max_pages, int nq, int nkv, float c, float cap, bf16* __restrict__ out,
                   const float* __restrict__ sinks) {
    // (of the launch, not of the kernel: see the prompt kernels)
    extern __shared__ __attribute__((aligned(1024))) char shared_lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Item it(items + (size_t)(blockIdx.x / nkv) * ITEM_INTS);
    if (it.rows == 0) return;
    const SharedArgs A = {q, k_cache, v_cache, partial_o, partial_ml, order, positions, parts, nq, nkv, (int)(blockIdx.x % nkv), nq / nkv, c, cap, out, sinks};
    const int cols = it.rows * A.G;
    const int* pt = page_table + (size_t)it.slot * max_pages;
    if (cols > 64) {
        wide_item<HD>(A, it, pt, cols, wave, lane, (bf16*)shared_lds);
        return;
    }
    // (what is looked for in items of a sequence's own rows takes registers that a wave of 32 columns does not have)
    const bool small = CAUSAL ? it.masked || cols <= 16 : cols <= 16;
    const int tiles = small ? (cols <= 16 ? 1 : cols <= 32 ? 2 : 4) : cols <= 32 ? 1 : 2, phases = 4 / tiles;
    const int tile = wave % tiles, phase = wave / tiles;
    if (small) narrow_item<HD, 1, CAUSAL>(A, it, pt, cols, tile * 16, phase, phases, wave, lane, shared_lds);
    else narrow_item<HD, 2, false>(A, it, pt, cols, tile * 32, phase, phases, wave, lane, shared_lds);
}

// ---------------------------------------------------------------- float32
// A workgroup of four waves: an item x a kv head x 16 of its columns. The products are chains of fmaf on the matrix cores
// (mfma_f32.h), as in the float32 attention over pages of a sequence's own: a wave scores 16 of a page's 64 keys, the scores meet in LDS,
// and each wave owns a quarter of the head's entries of the output. Two barriers a page. Bound by that chain: 5 answers to 1,500 tokens, 16/8 heads of 128, 15.8 MB
// in 9.9 us; 16 to 2,048 24 us with the join (one sequence after another: 103).
template <int NB>
__global__ void __launch_bounds__(256)
attn_shared_f32_kernel(const float* __restrict__ q, const float* __restrict__ k_cache, const float* __restrict__ v_cache,
                       float* __restrict__ partial_o, float* __restrict__ partial_ml, const int* __restrict__ items,
                       const int* __restrict__ order, const int* __restrict__ parts, const int* __restrict__ positions,
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
    const int* pt = page_table + (size_t)it.slot * max_pages;
    const int col = col0 + r;
    const bool mine = col < cols;
    const int row = (mine ? col : cols - 1) / G, head = kvh * G + (mine ? col : cols - 1) % G;
    const int pos = positions[order[it.row0 + row]], place = parts[it.list0 + row];
    // the queries, zeros beyond the head's entries and in columns that are nobody's, every 16 entries transposed: 16 threads a column
    {
        const int mc = tid >> 4, cl = col0 + mc;
        const float* src = q + ((size_t)order[it.row0 + (cl < cols ? cl : cols - 1) / G] * nq + kvh * G + (cl < cols ? cl : cols - 1) % G) * hd;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int d = 4 * ((tid & 15) + 16 * i);
            const f32x4 v = d < hd && cl < cols ? *(const f32x4*)(src + d) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; ++e) qs[mc * QLD + (d & ~15) + 4 * e + ((d >> 2) & 3)] = v[e];
        }
    }
    int seen_last = pos, seen_first = pos;
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
        seen_last = max(seen_last, __shfl_xor(seen_last, off, 64));
        seen_first = min(seen_first, __shfl_xor(seen_first, off, 64));
    }
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
        const int page0 = p * PAGE;
        const bool more = p + 1 < page_end;
        if (hd < 16 * DB)
#pragma unroll
            for (int b = 0; b < DB; ++b) key[b] = 16 * b + 4 * g4 < hd ? key[b] : f32x4{0.f, 0.f, 0.f, 0.f};
        // (four chains side by side: a quarter of the roundings one after the other, and none waits for another)
        f32x4 chain[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) chain[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < DB; ++b) {
            transpose_quads(key[b]);
            const f32x4 qq = *(const f32x4*)&qs[r * QLD + 16 * b + 4 * g4];
#pragma unroll
            for (int s = 0; s < 4; ++s) chain[b & 3] = mfma_k4(key[b][s], qq[s], chain[b & 3]);
        }
        f32x4 dots = (chain[0] + chain[1]) + (chain[2] + chain[3]);
        if (more) load_keys(p + 1);
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
                f32x4 half[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};     // (of the page)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    transpose_quads(v[b]);
#pragma unroll
                    for (int s = 0; s < 4; ++s) half[b & 1] = mfma_k4(v[b][s], w[b][s], half[b & 1]);
                }
                acc[i] += half[0] + half[1];
            }
        }
        if (more) load_values(p + 1);
    }
    if (!mine) return;
    const size_t part = (size_t)place * nq + head;
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
// Where the values that rows of one sequence see lie: for rows whose partial results are marked (a sum with a sign), because a value without a
// size was taken out of a product (CAUSAL: there may be such).
struct Spoiled {
    const bf16* v_cache;
    const int *positions, *seq_of, *slots, *page_table;
    int max_pages, nkv;
};

// What the sum over all values that a row sees becomes if some of them have no size: entry d of a head.
__device__ __forceinline__ float spoiled_sum(const Spoiled& s, float sum, int token, int kvh, int d, int hd) {
    const int pos = s.positions[token];
    const int* pt = s.page_table + (size_t)s.slots[s.seq_of[token]] * s.max_pages;
    bool plus = false, minus = false, nan = false;
#pragma unroll 1
    for (int j = 0; j <= pos; ++j) {
        const float v = hb_to_float(s.v_cache[(((size_t)pt[j / PAGE] * s.nkv + kvh) * hd + d) * PAGE + j % PAGE]);
        plus |= v == INFINITY;
        minus |= v == -INFINITY;
        nan |= v != v;
    }
    if (nan || (plus && minus)) return __uint_as_float(0x7fc00000u);
    return plus ? INFINITY : minus ? -INFINITY : sum;
}

// Bound by latency (3 us for a few results a row, 5.4 for 64 rows of 32 heads in 16 parts each, 17 MB) and for many rows by reading what the items left (516 rows, five parts each, 43 MB: 10.5 us).
// LANES lanes a (token, query head), four entries each: the partial results part_start[t] .. part_start[t + 1] - 1 of the t-th row, in their
// order. T: the type that leaves; c: what a difference of references is multiplied by for a power of two (float32: natural units,
// expf). A chain of three waits: where they lie, the results with their references, and the store.
template <class T, int LANES, bool CAUSAL>
__global__ void __launch_bounds__(256)
attn_shared_join_kernel(const float* __restrict__ partial_o, const float* __restrict__ partial_ml, T* __restrict__ out,
                        const int* __restrict__ order, const int* __restrict__ part_start, int n_rows, int nq, int hd, float c,
                        const float* __restrict__ sinks, Spoiled spoiled) {
    constexpr bool EXACT = sizeof(T) == 4;
    constexpr int AHEAD = 8;
    const int lane = threadIdx.x % LANES;
    const int at = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const bool exists = at < n_rows * nq;                 // (lanes of others go along: a wave's exchanges are among LANES)
    const int t = exists ? at / nq : 0, h = exists ? at % nq : 0;
    const int first = part_start[t], n = part_start[t + 1] - first, row = order[t];
    const bool there = 4 * lane < hd;
    const float* const po = partial_o + ((size_t)first * nq + h) * hd + (there ? 4 * lane : 0);
    const float2* const ml = (const float2*)partial_ml + (size_t)first * nq + h;
    const size_t stride = (size_t)nq * hd;
    f32x4 v[AHEAD];
    auto ask = [&](int s) {                               // (places beyond the last: the last, with a weight of 0)
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) v[u] = *(const f32x4*)(po + (size_t)(s + u < n ? s + u : n - 1) * stride);
    };
    ask(0);
    auto weight = [&](float m, float top) { return m == -INFINITY ? 0.f : EXACT ? expf(m - top) : fast_exp2((m - top) * c); };
    float top = -INFINITY;
    float2 kept = make_float2(-INFINITY, 0.f);            // this lane's, of the first LANES
    for (int s = lane; s < n; s += LANES) {
        const float2 x = ml[(size_t)s * nq];
        if (s == lane) kept = x;
        top = fmaxf(top, x.x);
    }
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, LANES));
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
    bool marked = false;
    for (int s0 = 0; s0 < n; s0 += LANES) {
        if (s0 > 0) kept = s0 + lane < n ? ml[(size_t)(s0 + lane) * nq] : make_float2(-INFINITY, 0.f);
        if constexpr (CAUSAL) {
            marked |= kept.y < 0.f;
            kept.y = fabsf(kept.y);
        }
        const float w = weight(kept.x, top);
        total = fmaf(w, kept.y, total);
        const int here = n - s0 < LANES ? n - s0 : LANES;
        for (int s = 0; s < here; s += AHEAD) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const float ws = __shfl(w, (s + u) % LANES, LANES);
                const bool counts = s + u < here;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = counts ? fmaf(ws, v[u][e], acc[e]) : acc[e];
            }
            if (s0 + s + AHEAD < n) ask(s0 + s + AHEAD);
        }
    }
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) {
        total += __shfl_xor(total, off, LANES);
        if (CAUSAL) marked |= __shfl_xor((int)marked, off, LANES) != 0;
    }
    if (sinks) total += EXACT ? expf(sinks[h] - (top == -INFINITY ? 0.f : top)) : sink_share(sinks[h], top, c);
    const float inv = total > 0.f || total != total ? 1.0f / total : 0.f;
    if (!there || !exists) return;
    if constexpr (CAUSAL) {
        if (marked)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = spoiled_sum(spoiled, acc[e], row, h / (nq / spoiled.nkv), 4 * lane + e, hd);
    }
    T* const dst = out + ((size_t)row * nq + h) * hd + 4 * lane;
    if constexpr (EXACT) {
        *(f32x4*)dst = acc * inv;
    } else {
        bf16x4 b;
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = (__bf16)(acc[e] * inv);
        *(bf16x4*)dst = b;
    }
}

// q, out [T, nq hd]; keys [pages, nkv, 64, hd], values [pages, nkv, hd, 64]; one storage type. items [n_items, 8]; order [n_rows]; part_start [n_rows + 1]: where a row's partial results begin; parts: the places of the items' rows among
// them; partial_o [partial results, nq, hd], partial_ml [partial results, nq, 2]. max_rows: the most rows of an item;
// causal: some rows are of one sequence (seq_of [n_rows], slots [sequences]: only then looked at). direct (bfloat16, not causal, items of at most 64
// columns): every row is in one item, whose result is the row's. softcap 0: none; sinks [nq] or null.
extern "C" int hb_attn_shared(const void* q, const void* k_cache, const void* v_cache, void* out, int dtype, float* partial_o,
                              float* partial_ml, const int* items, int n_items, int max_rows, int causal, int direct, const int* order,
                              const int* part_start, const int* parts, int n_rows, const int* positions,
                              const int* seq_of, const int* slots, const int* page_table, int max_pages, int nq, int nkv, int hd, float scale, float softcap,
                              const float* sinks, hipStream_t stream) {
    HB_REQUIRE(n_rows > 0 && n_items > 0 && nq > 0 && nkv > 0 && nq % nkv == 0, "shared attention: empty input, or heads that do not group");
    HB_REQUIRE(scale > 0.f && softcap >= 0.f, "shared attention: the scale must be positive, a cap of the scores too");
    HB_REQUIRE(((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)partial_o | (uintptr_t)out) % 16 == 0,
               "shared attention: queries and pages lie on 16-byte borders");
    const int G = nq / nkv;
    const long long rows_of_heads = (long long)n_rows * nq;
    HB_REQUIRE(rows_of_heads <= 0x7fffffffLL / 64, "shared attention: too many rows for the grid");
    auto join = [&](int lanes) { return dim3((unsigned)((rows_of_heads * lanes + 255) / 256)); };
    if (dtype == HB_BF16) {
        HB_REQUIRE(hd == 32 || hd == 64 || hd == 128, "shared attention: bfloat16 heads of 32, 64 or 128, not %d", hd);
        HB_REQUIRE((long long)max_rows * G <= 128, "shared attention: items of %d rows x %d heads exceed 128 columns", max_rows, G);
        HB_REQUIRE((long long)n_items * nkv <= 0x7fffffffLL, "shared attention: too many items for the grid");
        HB_REQUIRE(!direct || (!causal && (long long)max_rows * G <= 64), "shared attention: items that are whole rows' have at most 64 columns, a token a sequence");
        const float c = scale * 1.4426950408889634f, cap = softcap > 0.f ? softcap / scale : 0.f;
        const Spoiled spoiled = {(const bf16*)v_cache, positions, seq_of, slots, page_table, max_pages, nkv};
        const dim3 grid((unsigned)(n_items * nkv));
#define HB_SHARED_KERNEL(HD, CAUSAL)                                                                                       \
        {                                                                                                                    \
            constexpr int lds = SharedSizes<HD>::LDS;                                                                        \
            static const hipError_t allowed = hipFuncSetAttribute((const void*)attn_shared_kernel<HD, CAUSAL>,               \
                                                                  hipFuncAttributeMaxDynamicSharedMemorySize, lds);          \
            HB_REQUIRE(allowed == hipSuccess, "shared attention: %d bytes of LDS refused: %s", lds, hipGetErrorString(allowed)); \
            attn_shared_kernel<HD, CAUSAL><<<grid, 256, lds, stream>>>(                                                      \
                (const bf16*)q, (const bf16*)k_cache, (const bf16*)v_cache, partial_o, partial_ml, items, order, parts, positions, \
                page_table, max_pages, nq, nkv, c, cap, direct ? (bf16*)out : nullptr, sinks);                               \
            HB_CHECK_LAUNCH("shared attention");                                                                             \
            if (!direct) attn_shared_join_kernel<bf16, HD / 4, CAUSAL><<<join(HD / 4), 256, 0, stream>>>(partial_o, partial_ml, (bf16*)out, order,     \
                                                                               part_start, n_rows, nq, hd, c, sinks, spoiled); \
        }
#define HB_SHARED(HD)                                                                                                        \
        {                                                                                                                    \
            if (causal) HB_SHARED_KERNEL(HD, true)                                                                        \
            else HB_SHARED_KERNEL(HD, false)                                                                              \
        }
        if (hd == 32) HB_SHARED(32)
        else if (hd == 64) HB_SHARED(64)
        else HB_SHARED(128)
#undef HB_SHARED
#undef HB_SHARED_KERNEL
    } else if (dtype == HB_F32) {
        HB_REQUIRE(!direct, "shared attention: float32 items leave parts of rows");
        HB_REQUIRE(hd > 0 && hd <= 256 && hd % 4 == 0, "shared attention: float32 heads of up to 256 entries in whole quads, not %d", hd);
        const long long col_tiles = ((long long)max_rows * G + 15) / 16;
        HB_REQUIRE((long long)n_items * nkv * col_tiles <= 0x7fffffffLL, "shared attention: too many items for the grid");
        const dim3 grid((unsigned)(n_items * nkv * col_tiles));
#define HB_SHARED(NB, LANES)                                                                                                      \
        {                                                                                                                      \
            attn_shared_f32_kernel<NB><<<grid, 256, 0, stream>>>((const float*)q, (const float*)k_cache, (const float*)v_cache, \
                                                                 partial_o, partial_ml, items, order, parts, positions,        \
                                                                 page_table, max_pages, nq, nkv, hd, scale, softcap,           \
                                                                 (int)col_tiles);                                              \
            HB_CHECK_LAUNCH("shared attention");                                                                               \
            attn_shared_join_kernel<float, LANES, false><<<join(LANES), 256, 0, stream>>>(partial_o, partial_ml, (float*)out, order, part_start, \
                                                                        n_rows, nq, hd, 0.f, sinks, Spoiled{});                    \
        }
        if (hd <= 64) HB_SHARED(1, 16)
        else if (hd <= 128) HB_SHARED(2, 32)
        else HB_SHARED(4, 64)
#undef HB_SHARED
    } else {
        HB_REQUIRE(false, "shared attention: unknown dtype %d", dtype);
    }
    HB_CHECK_LAUNCH("shared attention: joining");
    return 0;
}
