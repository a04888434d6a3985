// What a step's logits say of given tokens: for every row x of V logits and its token t
//   log p(t) = x_t - m - log S,   S = sum e^(x - m),   m = max x,
//   entropy  = log S - T / S,     T = sum (x - m) e^(x - m)   (-inf: e^-inf = 0, and 0 (-inf) counts as 0),
// and the `top` largest logits with their log p, larger first and the lower id first among equals.
//
// Bound by reading the logits once. A row is cut into chunks of 4,096, a workgroup of 256 threads each, which holds its chunk in
// registers (16 a thread), finds its (m, S, T) and its own `top` largest; a second kernel adds a row's chunks up:
//   S = sum S_c e^(m_c - m),   T = sum (T_c + (m_c - m) S_c) e^(m_c - m).
// A row of one chunk needs no second kernel.
// 2,048 rows of 151,936 in 201 to 213 us, 6.1 TB/s: HBM. With alternatives by instructions: 64 rows and 20 of them 14.4 us for the chunks (39 MB; about 520 instructions a wave, a
// quarter of them alternatives; chunks of 8,192 took as long for 64 rows and 0.9 us more for one), 5 us for the rows; one row 5.2 and 4.0, near the least that two kernels take.
// The reference computes a softmax on the host to draw a token (crates/core/src/sampler.rs:72-145) and reports no
// probabilities.
#include "common.h"
#include <math.h>
#include <type_traits>

HB_MODULE_ERROR_SLOT()

#define CHUNK 4096
#define THREADS 256
#define PER (CHUNK / THREADS)
#define MAX_TOP 64
#define LISTED 1024        // candidates that are listed
#define RANKED 128         // and ranked

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// A logit and its id as one number, larger for what comes first: the value's order in the upper half, the id's complement
// in the lower one. 0 is none (a NaN's key is as good as any: such a row is refused as a whole).
__device__ __forceinline__ uint64_t key_of(float v, int id) {
    const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);       // (-0 equals 0)
    return ((uint64_t)((u & 0x80000000u) ? ~u : (u | 0x80000000u)) << 32) | (uint32_t)~id;
}
__device__ __forceinline__ int id_of(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

// e^u for u from -150 (e^-150 is 0 in 32 bits) to 0 by the hardware's power of two; the rounding of u log2 e, which grows with |u|, is
// put back.
__device__ __forceinline__ float exp_of(float u) {
    const float t = u * 1.44269502f;
    const float left = fmaf(u, 1.92596303e-8f, fmaf(u, 1.44269502f, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e * left, 0.693147182f, e);
}
__device__ __forceinline__ float at_least_nothing(float u) { return u < -150.f ? -150.f : u; }      // (a NaN stays one)

__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int off) {
    const uint32_t lo = __shfl_xor((int)(uint32_t)v, off, 64), hi = __shfl_xor((int)(uint32_t)(v >> 32), off, 64);
    return ((uint64_t)hi << 32) | lo;
}

// How many of the wave's lanes say so.
__device__ __forceinline__ int in_wave(bool is) { return __popcll(__builtin_amdgcn_ballot_w64(is)); }

struct Selecting {
    uint64_t list[LISTED], last[RANKED];
    uint64_t groups[64];
    int above[THREADS / 64][64], count;
};

// A bound from which there are `most` keys or fewer, but `top` at least: between lo, from which there are `count`, and hi, from which there
// are fewer than `top`, by halving. of(bound): how many of the wave's keys lie at or above a bound.
template <class Of>
__device__ uint64_t narrowed(Selecting& sh, int top, int most, uint64_t lo, uint64_t hi, int count, Of of) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int turn = 0; count > most && hi - lo > 1; turn ^= 1) {      // (two places in turn: one barrier)
        const uint64_t mid = lo + (hi - lo) / 2;
        int n = of(mid);
        if (lane == 0) sh.above[wave][turn] = n;
        __syncthreads();
        n = (sh.above[0][turn] + sh.above[1][turn]) + (sh.above[2][turn] + sh.above[3][turn]);
        if (n >= top) {
            lo = mid;
            count = n;
        } else {
            hi = mid;
        }
    }
    return lo;
}

// The `top` largest of the keys that a workgroup holds, written by put(rank, key): ranks 0 .. top - 1, those that there is no key
// for with the key 0. largest: the thread's own largest key; each(bound, f) hands f the thread's keys from bound on, and may hand it others;
// counted(bound): how many the wave's are.
// The n-th largest of the 64 largest keys of four threads each bounds the n largest of all from below. The keys at or above it are listed,
// mostly few; where they are many, the bound is moved up by halving first (an order of the keys in memory that puts the largest side by side
// leaves up to 16 for each of them). The last ones are ranked by counting.
template <class Each, class Counted, class Put>
__device__ void select_top(Selecting& sh, int top, uint64_t largest, Each each, Counted counted, Put put) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t g = largest;
#pragma unroll
    for (int off = 1; off <= 2; off <<= 1) {
        const uint64_t o = shfl_xor_u64(g, off);
        g = o > g ? o : g;
    }
    if ((tid & 3) == 0) sh.groups[tid >> 2] = g;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    const uint64_t of_lane = sh.groups[lane];             // (a wave counts a quarter of the groups that lie above)
    int above = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) above += sh.groups[16 * wave + i] > of_lane ? 1 : 0;
    sh.above[wave][lane] = above;
    __syncthreads();
    above = (sh.above[0][lane] + sh.above[1][lane]) + (sh.above[2][lane] + sh.above[3][lane]);
    // (keys are of different ids, only 0 may be there twice: no group has the n-th place, and every key counts)
    const uint64_t found = __builtin_amdgcn_ballot_w64(above == top - 1 && of_lane != 0);
    uint64_t bound = found ? sh.groups[__ffsll((unsigned long long)found) - 1] : 1;
    auto list = [&](uint64_t* to, int room, auto keys) {
        keys([&](uint64_t key) {
            if (key >= bound) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < room) to[at] = key;
            }
        });
        __syncthreads();
        return sh.count;
    };
    auto of_thread = [&](auto f) { each(bound, f); };
    int count = list(sh.list, LISTED, of_thread);
    const uint64_t* ranked = sh.list;
    if (count > RANKED) {
        uint64_t hi = of_lane;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const uint64_t o = shfl_xor_u64(hi, off);
            hi = o > hi ? o : hi;
        }
        ++hi;
        const bool listed = count <= LISTED;
        const int n = count;
        auto of_list = [&](auto f) {
            for (int i = tid; i < n; i += THREADS) f(sh.list[i]);
        };
        if (listed)
            bound = narrowed(sh, top, RANKED, bound, hi, n, [&](uint64_t from) {
                int c = 0;
                for (int i = tid; i - tid < n; i += THREADS) c += in_wave(i < n && sh.list[i] >= from);
                return c;
            });
        else
            bound = narrowed(sh, top, RANKED, bound, hi, n, counted);
        __syncthreads();                                  // (the count has been read)
        if (tid == 0) sh.count = 0;
        __syncthreads();
        count = listed ? list(sh.last, RANKED, of_list) : list(sh.last, RANKED, of_thread);
        if (count > RANKED) count = RANKED;
        ranked = sh.last;
    }
    int each_by = 1;                                      // threads that count for one of them
    while (each_by < 64 && 2 * each_by * count <= THREADS) each_by *= 2;
    const int i = tid / each_by, part = tid % each_by;    // (THREADS / each_by >= count)
    const uint64_t mine = ranked[i < count ? i : 0];
    above = 0;
#pragma unroll 8
    for (int j = part; j < count; j += each_by) above += ranked[j] > mine ? 1 : 0;
    for (int off = each_by / 2; off > 0; off >>= 1) above += __shfl_xor(above, off, 64);
    if (i < count && part == 0 && above < top) put(above, mine);
    for (int n = count + tid; n < top; n += THREADS) put(n, (uint64_t)0);
}

// A row's results from its m, S and T: what the row's threads share.
struct Row {
    float m, log_s;
    bool bad;            // NaN or +inf among the logits, or nothing above -inf: no distribution
};
__device__ __forceinline__ Row row_of(float m, float S) {
    Row r;
    r.m = m;
    r.bad = !(S > 0.f && S < INFINITY);
    r.log_s = logf(S);
    return r;
}
__device__ __forceinline__ void leave_token(const Row& r, float S, float T, const float* row, int V, int token, float* chosen,
                                            float* entropy) {
    const float nan = __uint_as_float(0x7fc00000u);
    *chosen = r.bad || token < 0 || token >= V ? nan : (row[token] - r.m) - r.log_s;
    *entropy = r.bad ? nan : fmaxf(r.log_s - T / S, 0.f);
}
__device__ __forceinline__ void leave_top(const Row& r, uint64_t key, int* id, float* best) {
    *id = r.bad ? -1 : id_of(key);
    *best = r.bad ? __uint_as_float(0x7fc00000u) : (value_of(key) - r.m) - r.log_s;
}

// stats [row][chunk]: (m, S, T); keys [row][rank][chunk], so that neighbours are alike in rank. One chunk a row: the row's results themselves.
// (seven waves a SIMD hold the registers; eight, with one of them in memory, take as long)
template <bool TOP>
__global__ void __launch_bounds__(THREADS, 7)
logprob_chunk_kernel(const float* __restrict__ logits, int V, const int* __restrict__ tokens, float* __restrict__ chosen,
                     float* __restrict__ entropy, int* __restrict__ ids, float* __restrict__ best, int top, int chunks,
                     float4* __restrict__ stats, uint64_t* __restrict__ keys) {
    __shared__ float red[3][THREADS / 64];
    __shared__ std::conditional_t<TOP, Selecting, int> sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t r = blockIdx.x / chunks;
    const int chunk = blockIdx.x % chunks, first = chunk * CHUNK, len = V - first < CHUNK ? V - first : CHUNK;
    const float* row = logits + r * V;
    float x[PER];
#pragma unroll
    for (int j = 0; j < PER / 4; ++j) {
        const int at = (j * THREADS + tid) * 4;
        if (at + 4 <= len) {
            const f32x4u v = *(const f32x4u*)(row + first + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * j + e] = v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * j + e] = at + e < len ? row[first + at + e] : -INFINITY;
        }
    }
    float mine = x[0];
    int which = 0;
#pragma unroll
    for (int i = 1; i < PER; ++i) {
        const bool more = x[i] > mine;
        mine = more ? x[i] : mine;
        which = more ? i : which;
    }
    float m = hb_wave_max(fmaxf(mine, -INFINITY));        // (of what is a number)
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    float S = 0.f, T = 0.f;                               // (a NaN ends up in S)
    if (m != -INFINITY) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float u = at_least_nothing(x[i] - m), e = exp_of(u);
            S += e;
            T = fmaf(e, u, T);
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) S = x[i] != x[i] ? x[i] : S;
    }
    S = hb_wave_sum(S);
    T = hb_wave_sum(T);
    if (lane == 0) red[1][wave] = S, red[2][wave] = T;
    __syncthreads();
    S = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    T = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
    const Row whole = row_of(m, S);
    if (tid == 0) {
        if (chunks > 1) stats[r * chunks + chunk] = make_float4(m, S, T, 0.f);
        else leave_token(whole, S, T, row, V, tokens[r], chosen + r, entropy + r);
    }
    if constexpr (TOP) {
        auto id_at = [&](int i) { return ((i >> 2) * THREADS + tid) * 4 + (i & 3); };
        const uint64_t largest = id_at(which) < len ? key_of(mine, first + id_at(which)) : (uint64_t)0;
        select_top(sh, top, largest, [&](uint64_t bound, auto f) {
            const float least = bound > 1 ? value_of(bound) : -INFINITY;
            if (mine >= least) f(largest);
            int n = 0;                                    // (few threads have a second one)
#pragma unroll
            for (int i = 0; i < PER; ++i) n += x[i] >= least ? 1 : 0;
            if (n > 1)
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (x[i] >= least && i != which) f(id_at(i) < len ? key_of(x[i], first + id_at(i)) : (uint64_t)0);
        }, [&](uint64_t bound) {
            // (a bound need not be a logit's key: below all of them, and between those of -0, of which there are none, and 0)
            const uint64_t lowest = (uint64_t)0x007fffffu << 32, zero = (uint64_t)0x80000000u << 32;
            bound = bound < lowest ? lowest : (uint32_t)(bound >> 32) == 0x7fffffffu ? zero : bound;
            const float least = value_of(bound);
            const int last = (int)min(~(uint32_t)bound, (uint32_t)(first + len - 1)) - first;
            int n = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) n += in_wave(x[i] > least || (x[i] == least && id_at(i) <= last));
            return n;
        }, [&](int rank, uint64_t key) {
            if (chunks > 1) keys[(r * top + rank) * chunks + chunk] = key;
            else leave_top(whole, key, ids + r * top + rank, best + r * top + rank);
        });
    }
}

// A workgroup a row: its chunks added up, in a fixed order.
template <bool TOP>
__global__ void __launch_bounds__(THREADS)
logprob_row_kernel(const float* __restrict__ logits, int V, const int* __restrict__ tokens, float* __restrict__ chosen,
                   float* __restrict__ entropy, int* __restrict__ ids, float* __restrict__ best, int top, int chunks,
                   const float4* __restrict__ stats, const uint64_t* __restrict__ keys) {
    __shared__ float red[3][THREADS / 64];
    __shared__ std::conditional_t<TOP, Selecting, int> sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t r = blockIdx.x;
    stats += r * chunks;
    float m = -INFINITY;
    for (int c = tid; c < chunks; c += THREADS) m = fmaxf(m, stats[c].x);
    m = hb_wave_max(m);
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    float S = 0.f, T = 0.f;
    for (int c = tid; c < chunks; c += THREADS) {
        const float4 s = stats[c];
        if (s.x == -INFINITY) {
            S += s.y;                      // nothing, or NaN
            continue;
        }
        const float down = at_least_nothing(s.x - m), e = exp_of(down);
        S = fmaf(e, s.y, S);
        T = fmaf(e, fmaf(down, s.y, s.z), T);
    }
    S = hb_wave_sum(S);
    T = hb_wave_sum(T);
    if (lane == 0) red[1][wave] = S, red[2][wave] = T;
    __syncthreads();
    S = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    T = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
    const Row whole = row_of(m, S);
    if (tid == 0) leave_token(whole, S, T, logits + r * V, V, tokens[r], chosen + r, entropy + r);
    if constexpr (TOP) {
        keys += r * chunks * top;
        const int n = chunks * top;
        uint64_t largest = 0;
        for (int i = tid; i < n; i += THREADS) largest = keys[i] > largest ? keys[i] : largest;
        select_top(sh, top, largest, [&](uint64_t, auto f) {
            for (int i = tid; i < n; i += THREADS) f(keys[i]);
        }, [&](uint64_t bound) {
            int c = 0;
            for (int i = tid; i - tid < n; i += THREADS) c += in_wave(i < n && keys[i] >= bound);
            return c;
        }, [&](int rank, uint64_t key) { leave_top(whole, key, ids + r * top + rank, best + r * top + rank); });
    }
}

// logits [R, V], tokens [R] -> chosen [R], entropy [R]; top > 0: ids, best [R, top]. stats: 4 floats for every row and chunk of 4,096, keys: 2
// floats' room for every one of their `top` (both only for V > 4,096).
extern "C" int hb_token_logprobs(const float* logits, int R, int V, const int* tokens, float* chosen, float* entropy, int* ids,
                                 float* best, int top, void* stats, void* keys, hipStream_t stream) {
    HB_REQUIRE(R > 0 && V > 0 && top >= 0 && top <= MAX_TOP && top <= V, "log probabilities: bad sizes (R=%d, V=%d, top=%d)", R, V, top);
    HB_REQUIRE(top == 0 || (ids && best), "log probabilities: no room for %d alternatives", top);
    const int chunks = (V - 1) / CHUNK + 1;
    HB_REQUIRE((long long)R * chunks <= 0x7fffffffLL, "log probabilities: too many rows for the grid");
    HB_REQUIRE(chunks == 1 || (stats && (top == 0 || keys)), "log probabilities: rows of more than %d logits need room for their chunks", CHUNK);
    const unsigned grid = (unsigned)(R * chunks);
    if (top > 0) logprob_chunk_kernel<true><<<grid, THREADS, 0, stream>>>(logits, V, tokens, chosen, entropy, ids, best, top, chunks, (float4*)stats, (uint64_t*)keys);
    else logprob_chunk_kernel<false><<<grid, THREADS, 0, stream>>>(logits, V, tokens, chosen, entropy, ids, best, top, chunks, (float4*)stats, (uint64_t*)keys);
    HB_CHECK_LAUNCH("log probabilities");
    if (chunks > 1) {
        if (top > 0) logprob_row_kernel<true><<<R, THREADS, 0, stream>>>(logits, V, tokens, chosen, entropy, ids, best, top, chunks, (const float4*)stats, (const uint64_t*)keys);
        else logprob_row_kernel<false><<<R, THREADS, 0, stream>>>(logits, V, tokens, chosen, entropy, ids, best, top, chunks, (const float4*)stats, (const uint64_t*)keys);
        HB_CHECK_LAUNCH("log probabilities: rows");
    }
    return 0;
}
