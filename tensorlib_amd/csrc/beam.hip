// Beam search: selection over beams and vocabulary, and the reordering of the beams' token histories.
//
// Every beam of a request continues with every token at  score + logit - log sum exp(logits);  the best n of a request
// go on, equal scores in the order of (beam, token).  A finished beam has one continuation, its end token at its own
// score.  Scores are compared in fp64: as fp32 they would be rounded by 2^-20 at a score of -20.  A row's sum takes fp32
// exponentials and is fp32 within a thread and fp64 from there on.  Its relative error, which is its logarithm's absolute one, is
// at most 2^-23 for an exponential, 0.8 2^-23 for its argument and eight additions of 2^-24 in turn: below 2^-20.  Continuations
// of different beams that lie closer may come in either order; within a beam the logits alone decide.  (Relative to the largest
// term, as the pick takes it where that has most of the sum, its own 1.8 2^-23 are added, and what the two share drops out.)
//
// Bound by the one pass over the logits (2 bytes each), small requests by latency.  First launch: one workgroup per (row,
// slice of the vocabulary) holds its slice in registers and leaves the slice's maximum, its sum and its best n
// candidates in order: within a row the order of the logits is the order of the scores, so no sum is needed for that.
// Second launch: one workgroup per request joins the rows' sums and picks.
//
// The best n of many: the n-th largest of the threads' maxima, or the least of what each wavefront's share of n threads reaches,
// is a bound that at least n elements reach; it is found bit by bit, a ballot each.  What reaches it (some fifteen candidates
// for n = 8 out of 8192 random logits) goes to a list in LDS, where every candidate counts those before it: its rank is its
// place in the answer.  A list that overflows (values in an order that defeats the bound) is given up for n rounds of a maximum
// over the workgroup.
//
// 24 requests of 8 beams over 100003 tokens: 13 + 5.5 us (38 MB: 6 us at the rate of a plain read; the vector pipes are busy
// for 7 us of the first launch, and its workgroups do not all run at a time).  1 request of 4 beams over 32000: 4 + 4 us,
// two launches and their memory latencies.  64 beams over 100003, 64 selected: 120 us, most of it the second launch.
#include <algorithm>
#include <cmath>

#include "paged.h"

namespace tl {

typedef unsigned long long u64;

constexpr int kBeamThreads = 256;
constexpr int kBeamWaves = kBeamThreads / 64;
constexpr int kIndexBits = 13;                            // of a logit in its slice
constexpr int kMaxSelect = 64;
constexpr int kList = 1024;

struct SliceStats {
    double sum;                                           // of 2^(logit log2 e - top), NaN if the slice holds NaN or +inf
    float top;                                            // a whole number, kLowest for nothing but -inf
    float most;                                           // the largest logit; anything if the sum is NaN or 0
};

struct BeamArgs {
    const half_t* logits;
    size_t logits_stride;
    const float* scores;
    const uint8_t* finished;
    float* scores_out;
    int *tokens_out, *parents_out;
    SliceStats* stats;                                    // [row][slice]
    unsigned* best;                                       // [row][slice][n_select]
    FastDiv by_row;                                       // candidates per row in the second launch
    int n_beams, vocab, n_select, end_token, n_slices, slice;
};

// Larger is better: the logit's order (the two zeros are equal), then the lower index in the slice.  Never 0.
__device__ __forceinline__ unsigned key_of(half_t x) {
    unsigned b = __builtin_bit_cast(unsigned short, x);
    if (b == 0x8000u) b = 0;
    return b & 0x8000u ? (~b & 0xffffu) : (b | 0x8000u);
}
__device__ __forceinline__ unsigned candidate(half_t x, int index) { return (key_of(x) << kIndexBits) | (unsigned)((1 << kIndexBits) - 1 - index); }
__device__ __forceinline__ float candidate_logit(unsigned c) {
    unsigned b = c >> kIndexBits;
    b = b & 0x8000u ? (b & 0x7fffu) : (~b & 0xffffu);
    return (float)__builtin_bit_cast(half_t, (unsigned short)b);
}
__device__ __forceinline__ int candidate_index(unsigned c) { return (1 << kIndexBits) - 1 - (int)(c & ((1u << kIndexBits) - 1)); }

// One step of a reduction over lanes whose f does not care for the order of its operands: v joined with the value of the lane
// whose number differs in one bit, for values that are equal within groups of 2^BIT adjacent lanes (what the steps before
// leave behind).  All in the vector pipe: quads, mirrored halves of 8 and 16, then swapped rows of 16 and 32.
template <int BIT, class F>
__device__ __forceinline__ unsigned join_word(unsigned v, F f) {
    if constexpr (BIT < 4) {
        constexpr int ctrl = BIT == 0 ? 0xB1 : BIT == 1 ? 0x4E : BIT == 2 ? 0x141 : 0x140;
        return f(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true));
    } else {
        const auto r = BIT == 4 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return f(r[0], r[1]);
    }
}
template <int BIT, class T, class F>
__device__ __forceinline__ T join(T v, F f) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, join_word<BIT>(__builtin_bit_cast(unsigned, v), [&](unsigned a, unsigned b) {
            return __builtin_bit_cast(unsigned, f(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b)));
        }));
    } else {
        const uint2 w = __builtin_bit_cast(uint2, v);
        unsigned other;
        const unsigned x = join_word<BIT>(w.x, [&](unsigned a, unsigned b) { other = b; return a; });
        unsigned other_y;
        const unsigned y = join_word<BIT>(w.y, [&](unsigned a, unsigned b) { other_y = b; return a; });
        return f(__builtin_bit_cast(T, uint2{x, y}), __builtin_bit_cast(T, uint2{other, other_y}));
    }
}
template <class T, class F>
__device__ __forceinline__ T over_wave(T v, F f) {
    v = join<0>(v, [&](T a, T b) { return f(a, b, 0); });
    v = join<1>(v, [&](T a, T b) { return f(a, b, 1); });
    v = join<2>(v, [&](T a, T b) { return f(a, b, 2); });
    v = join<3>(v, [&](T a, T b) { return f(a, b, 3); });
    v = join<4>(v, [&](T a, T b) { return f(a, b, 4); });
    return join<5>(v, [&](T a, T b) { return f(a, b, 5); });
}
template <class T>
__device__ __forceinline__ T wave_max(T v) {
    return over_wave(v, [](T a, T b, int) { return b > a ? b : a; });
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
    return over_wave(v, [](T a, T b, int) { return a + b; });
}
// The n-th largest of the wavefront's keys without its lowest 12 bits, bit by bit from the top: of a float's place eleven bits
// of the fraction are left, close enough for a bound, and 0.25 us less than with all 32 in turn.
__device__ __forceinline__ unsigned nth_largest(unsigned key, int n) {
    unsigned found = 0;
#pragma unroll
    for (int bit = 31; bit >= 12; --bit) {
        const unsigned trial = found | (1u << bit);
        if ((int)__popcll(__ballot(key >= trial)) >= n) found = trial;
    }
    return found;
}
// The n-th largest of the wavefront's candidates, or one a little smaller: by the logit, and by the index too where many have
// that logit (a row that is masked but for a few tokens).
__device__ __forceinline__ unsigned nth_candidate(unsigned c, int n) {
    unsigned found = 0;
    int reached = 64;
    auto bits = [&](int from, int to) {
#pragma unroll
        for (int bit = from; bit >= to; --bit) {
            const unsigned trial = found | (1u << bit);
            const int k = (int)__popcll(__ballot(c >= trial));
            if (k >= n) {
                found = trial;
                reached = k;
            }
        }
    };
    bits(kIndexBits + 15, kIndexBits);
    if (reached > 2 * n + 4) bits(kIndexBits - 1, 0);
    return found;
}
// A float's place in the order of floats, and back.
__device__ __forceinline__ unsigned order_of(float f) {
    const unsigned b = __builtin_bit_cast(unsigned, f);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_order(unsigned o) { return __builtin_bit_cast(float, o ^ (o >> 31 ? 0x80000000u : 0xffffffffu)); }

// log2 e is kLog2e (1 + d), and 2^(x log2 e) is 2^(x kLog2e) e^(x kLog2e d ln 2).  The second factor is taken once for eight
// elements, at the whole number c above the largest x kLog2e.  An element a factor of 2^-t below 2^c is then off by t d ln 2 =
// t 0.93e-8, which its share of the sum makes 2.5e-8 at most, less than half an fp32 rounding (192 rows of 100003: 23.7 -> 23.3 us).
constexpr float kLog2e = 1.4426950216293335f, kLog2eRest = 9.253347e-9f;       // the latter d ln 2
constexpr float kLowest = -131072.f;                      // below every finite half times log2 e
__device__ __forceinline__ float whole_above(float most) { return fmaxf(ceilf(most * kLog2e), kLowest); }
__device__ __forceinline__ float power_of(float x, float c) { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2e, -c)); }
__device__ __forceinline__ float with_rest(float sum, float c) {
    const float rest = c * kLog2eRest;
    return __builtin_fmaf(sum, __builtin_fmaf(0.5f * rest, rest, rest), sum);     // e^rest to its square, at most 8.8e-4
}
__device__ __forceinline__ int exponent_of(float c, float reference) { return (int)fmaxf(c - reference, -1024.f); }

// NV: 16-byte pieces of logits per thread; a slice is NV * 2048 of them.
template <int NV>
__global__ void __launch_bounds__(kBeamThreads) beam_rows_kernel(BeamArgs A) {
    constexpr int SLICE = NV * kBeamThreads * 8;
    static_assert(SLICE <= 1 << kIndexBits, "index bits");
    __shared__ __align__(16) unsigned s_list[kList];
    __shared__ unsigned s_bound[kBeamWaves], s_best[kBeamWaves];
    __shared__ float s_c[kBeamWaves];
    __shared__ double s_sum[kBeamWaves];
    __shared__ int s_count;
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x, wave = tid / 64;
    if (A.finished && A.finished[row]) return;
    const int v0 = slice * SLICE;
    const int n = A.vocab - v0 < SLICE ? A.vocab - v0 : SLICE;
    const half_t* x = A.logits + (size_t)row * A.logits_stride + v0;
    half8_t v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = (j * kBeamThreads + tid) * 8;
        if (i + 8 <= n) {
            __builtin_memcpy(&v[j], x + i, 16);           // rows of an odd vocabulary start at any even address
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = i + e < n ? x[i + e] : (half_t)-INFINITY;
        }
    }
    if (tid == 0) s_count = 0;
    // Piece by piece as they arrive: its largest logit, and the sum of 2^(x log2 e - c) with a whole number c of its own, so that
    // sums with other c join without rounding.  A piece of -inf has a c below all others and a sum of 0; NaN and +inf show
    // as NaN.
    half_t most[NV], top = (half_t)-INFINITY;
    float part[NV], c[NV], c_thread = kLowest;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        half2_t m[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = half2_t{v[j][2 * e], v[j][2 * e + 1]};
        m[0] = __builtin_elementwise_max(__builtin_elementwise_max(m[0], m[1]), __builtin_elementwise_max(m[2], m[3]));
        most[j] = __builtin_elementwise_max(m[0][0], m[0][1]);
        top = __builtin_elementwise_max(top, most[j]);
        c[j] = whole_above((float)most[j]);
        c_thread = fmaxf(c_thread, c[j]);
        float p[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e % 2] += power_of((float)v[j][e], c[j]);
        }
        part[j] = with_rest(p[0] + p[1], c[j]);
    }
    float mine_sum = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) mine_sum += ldexpf(part[j], exponent_of(c[j], c_thread));
    int first = NV - 1;                                   // the first piece that holds it
#pragma unroll
    for (int j = NV - 2; j >= 0; --j)
        if (most[j] == top) first = j;
    // the candidate of the piece's last element is at most the thread's best: still a bound that enough elements reach
    const unsigned mine_least = candidate(top, (first * kBeamThreads + tid) * 8 + 7);
    // Either every wavefront's share of n_select, the least of which n_select threads reach together, or, where the last one has
    // little to choose from, the best of what n_select threads of one reach.
    const bool shared = n >= kBeamThreads * 7;
    const unsigned bound = nth_candidate(mine_least, shared ? (A.n_select + kBeamWaves - 1) / kBeamWaves : A.n_select);
    const float c_wave = wave_max(c_thread);
    const double sum_wave = wave_sum((double)ldexpf(mine_sum, exponent_of(c_thread, c_wave)));
    if (tid % 64 == 0) {
        s_bound[wave] = bound;
        s_c[wave] = c_wave;
        s_sum[wave] = sum_wave;
    }
    __syncthreads();
    unsigned reach = s_bound[0];
#pragma unroll
    for (int w = 1; w < kBeamWaves; ++w) reach = shared ? min(reach, s_bound[w]) : max(reach, s_bound[w]);
    SliceStats* stats = A.stats + (size_t)row * A.n_slices + slice;
    if (tid == 0) {
        float c_slice = kLowest;
        double sum = 0.0;
        for (int w = 0; w < kBeamWaves; ++w) c_slice = fmaxf(c_slice, s_c[w]);
        for (int w = 0; w < kBeamWaves; ++w) sum += ldexp(s_sum[w], exponent_of(s_c[w], c_slice));
        stats->sum = sum;
        stats->top = c_slice;
    }
    // what reaches the bound
    const half_t reach_value = (half_t)candidate_logit(reach);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (!(most[j] >= reach_value)) continue;
        unsigned hits = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) hits |= v[j][e] >= reach_value ? 1u << e : 0u;
        const uint4 w = __builtin_bit_cast(uint4, v[j]);
        while (hits) {                                    // one or two lanes, once, as a rule
            const int e = __builtin_ctz(hits);
            hits &= hits - 1;
            const unsigned pair = e < 4 ? (e < 2 ? w.x : w.y) : (e < 6 ? w.z : w.w);
            const int i = (j * kBeamThreads + tid) * 8 + e;
            const unsigned cand = candidate(__builtin_bit_cast(half_t, (unsigned short)(pair >> (e % 2 * 16))), i);
            if (cand >= reach && i < n) {
                const int at = atomicAdd(&s_count, 1);
                if (at < kList) s_list[at] = cand;
            }
        }
    }
    __syncthreads();
    unsigned* best = A.best + ((size_t)row * A.n_slices + slice) * A.n_select;
    const int count = s_count;
    if (count <= kList) {
        // several threads count for each candidate where there are enough
        const int parts = count <= kBeamThreads / 8 ? 8 : count <= kBeamThreads / 4 ? 4 : count <= kBeamThreads / 2 ? 2 : 1;
        for (int i = tid / parts; i < count; i += kBeamThreads) {      // once if parts > 1: all of a candidate's lanes come along
            const unsigned mine = s_list[i];
            int rank = 0;
            for (int k = tid % parts * 4; k < count; k += parts * 4) {     // what stands behind the list's end is masked
                const uint4 a = *reinterpret_cast<const uint4*>(s_list + k);
                rank += (a.x > mine) + (k + 1 < count && a.y > mine) + (k + 2 < count && a.z > mine) + (k + 3 < count && a.w > mine);
            }
            if (parts >= 2) rank = join<0>(rank, [](int a, int b) { return a + b; });
            if (parts >= 4) rank = join<1>(rank, [](int a, int b) { return a + b; });
            if (parts == 8) rank = join<2>(rank, [](int a, int b) { return a + b; });
            if (tid % parts == 0 && rank < A.n_select) best[rank] = mine;
            if (tid % parts == 0 && rank == 0) stats->most = candidate_logit(mine);
        }
        for (int i = count + tid; i < A.n_select; i += kBeamThreads) best[i] = 0;       // the slice has no more
        return;
    }
    unsigned below = ~0u;
    for (int k = 0; k < A.n_select; ++k) {
        unsigned mine = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = (j * kBeamThreads + tid) * 8 + e;
                const unsigned cand = candidate(v[j][e], i);
                if (i < n && cand < below && cand > mine) mine = cand;
            }
        mine = wave_max(mine);
        __syncthreads();
        if (tid % 64 == 0) s_best[wave] = mine;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kBeamWaves; ++w) mine = max(mine, s_best[w]);
        if (tid == 0) best[k] = mine;
        if (tid == 0 && k == 0) stats->most = candidate_logit(mine);
        below = mine;
    }
}

// A continuation of a request: better by score, then by the lower place.
struct Choice {
    double score;
    u64 place;                                            // beam, then token
};
__device__ __forceinline__ bool better(const Choice& a, const Choice& b) { return a.score > b.score || (a.score == b.score && a.place < b.place); }

constexpr int kHeld = 4;                                  // continuations a thread keeps in registers

template <int THREADS>
__global__ void __launch_bounds__(THREADS) beam_pick_kernel(BeamArgs A) {
    constexpr int kPickThreads = THREADS, kPickWaves = THREADS / 64;
    __shared__ Choice s_list[kList];
    __shared__ Choice s_best[kPickWaves];
    __shared__ Choice s_last;
    __shared__ unsigned s_bound[kPickWaves], s_share[kPickWaves];
    __shared__ int s_count;
    extern __shared__ double s_base[];                    // per beam: score - log sum, then how it continues
    int* s_kind = reinterpret_cast<int*>(s_base + A.n_beams);
    enum { kDead, kAlive, kFinished };
    const int request = blockIdx.x, tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    const int row0 = request * A.n_beams;
    const int per_row = A.n_slices * A.n_select;
    const unsigned total = (unsigned)A.n_beams * A.by_row.d;
    const u64 none = ~0ull;
    // the first candidates are under way while the sums are joined
    unsigned held[kHeld];
#pragma unroll
    for (int x = 0; x < kHeld; ++x) {
        unsigned at = 0, b = 0;
        const unsigned i = x * kPickThreads + tid;
        if (i < total) b = A.by_row.divmod(i, at);
        held[x] = i < total && (int)at < per_row ? A.best[(size_t)(row0 + b) * per_row + at] : 0;
    }
    for (int b = wave; b < A.n_beams; b += kPickWaves) {
        const double score = (double)A.scores[row0 + b];
        const bool done = A.finished && A.finished[row0 + b];
        const SliceStats* st = A.stats + (size_t)(row0 + b) * A.n_slices;
        // a finished row has left nothing there, and nothing of what is read for it is used
        SliceStats mine = lane < A.n_slices ? st[lane] : SliceStats{0.0, -INFINITY, -INFINITY};
        float top = mine.top, most = mine.most;
        for (int s = lane + 64; s < A.n_slices; s += 64) {
            top = fmaxf(top, st[s].top);
            most = fmaxf(most, st[s].most);
        }
        top = wave_max(top);
        most = wave_max(most);
        double sum = 0.0;
        for (int s = lane;;) {
            if (mine.sum != 0.0) sum += mine.sum * exp2((double)mine.top - (double)top);
            s += 64;
            if (s >= A.n_slices) break;
            mine = st[s];
        }
        sum = wave_sum(sum);
        // Where one token has most of the sum, the logarithm is taken relative to that token's own term, computed as it was in
        // the sum: the error of its exponential drops out, and a row with one token left continues with probability 1 to the bit.
        const double own = (double)with_rest(power_of(most, top), top);
        const double log_sum = sum < 2.0 * own ? (double)most + log(sum / own) : (double)top * 0.69314718055994530942 + log(sum);
        const double base = done ? score : score - log_sum;
        if (lane == 0) {
            const bool finite = base > -INFINITY && base < INFINITY;
            s_base[b] = finite ? base : -INFINITY;
            s_kind[b] = done ? kFinished : finite ? kAlive : kDead;
        }
    }
    if (tid == 0) s_count = 0;
    __syncthreads();
    // the i-th possible continuation, given its entry of `best`; place none: there is none behind this number
    auto choice_of = [&](unsigned i, unsigned e) -> Choice {
        unsigned at;
        const int b = (int)A.by_row.divmod(i, at);
        const double base = s_base[b];
        const int kind = s_kind[b];
        if (kind != kAlive) {                             // the end token at the beam's score; all else at -inf, lowest first
            const bool end = kind == kFinished && (int)at == A.n_select;
            if ((int)at > A.n_select || (!end && ((int)at >= A.vocab || (kind == kFinished && (int)at == A.end_token)))) return {-INFINITY, none};
            return {end ? base : (double)-INFINITY, (u64)b << 32 | (end ? (unsigned)A.end_token : at)};
        }
        if (e == 0) return {-INFINITY, none};
        return {base + (double)candidate_logit(e), (u64)b << 32 | ((at / A.n_select) * A.slice + candidate_index(e))};
    };
    auto entry = [&](unsigned i) -> unsigned {
        unsigned at;
        const int b = (int)A.by_row.divmod(i, at);
        return s_kind[b] == kAlive && (int)at < per_row ? A.best[(size_t)(row0 + b) * per_row + at] : 0;
    };
    auto choice = [&](unsigned i) -> Choice { return choice_of(i, entry(i)); };
    // f of the continuations that are not held, several of whose entries are under way together
    auto others = [&](auto f) {
        for (unsigned i0 = kHeld * kPickThreads + tid; i0 < total; i0 += 4 * kPickThreads) {
            unsigned e[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) e[x] = i0 + x * kPickThreads < total ? entry(i0 + x * kPickThreads) : 0;
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (i0 + x * kPickThreads < total) f(choice_of(i0 + x * kPickThreads, e[x]));
        }
    };
    auto put = [&](int k, const Choice& c) {
        const size_t o = (size_t)request * A.n_select + k;
        A.scores_out[o] = (float)c.score;
        A.tokens_out[o] = (int)(c.place & 0xffffffffu);
        A.parents_out[o] = row0 + (int)(c.place >> 32);
    };
    Choice kept[kHeld];
    double mine = -INFINITY;
#pragma unroll
    for (int x = 0; x < kHeld; ++x) {
        const unsigned i = x * kPickThreads + tid;
        kept[x] = {-INFINITY, none};
        if (i < total) kept[x] = choice_of(i, held[x]);
        mine = fmax(mine, kept[x].score);
    }
    others([&](const Choice& c) { mine = fmax(mine, c.score); });
    // the n-th largest of a wavefront's threads, as a float that is not above it: scores of one beam in neighbouring threads
    // are in order already, and groups of them would make a loose bound
    float low = (float)mine;
    if ((double)low > mine) low = from_order(order_of(low) - 1);
    const unsigned bound = nth_largest(order_of(low), A.n_select);
    // each wavefront's share of n_select, the smallest of which n_select threads reach too: of many, the closer bound
    unsigned share = 0;
    if (A.n_select > kPickWaves / 2) share = nth_largest(order_of(low), (A.n_select + kPickWaves - 1) / kPickWaves);
    if (lane == 0) {
        s_bound[wave] = bound;
        s_share[wave] = ~share;
    }
    __syncthreads();
    const unsigned closer = max(wave_max(s_bound[lane % kPickWaves]), ~wave_max(s_share[lane % kPickWaves]));
    const double reach = (double)from_order(max(closer, order_of(-INFINITY)));
    auto list = [&](const Choice& c) {
        if (c.place == none || !(c.score >= reach)) return;
        const int at = atomicAdd(&s_count, 1);
        if (at < kList) s_list[at] = c;
    };
#pragma unroll
    for (int x = 0; x < kHeld; ++x) list(kept[x]);
    others(list);
    __syncthreads();
    const int count = s_count;
    if (count <= kList) {                                 // at least n_select: the bound says so, or everything is in it
        // Several threads count for each choice of a short list.  A list may be longer than the workgroup (512 threads, up to kList
        // choices): then a thread takes two.  With parts > 1 there is one turn, and all of a choice's lanes are in it together.
        const int parts = count <= kPickThreads / 8 ? 8 : count <= kPickThreads / 4 ? 4 : 1;
        for (int i = tid / parts; i < count; i += kPickThreads) {
            const Choice c = s_list[i];
            int rank = 0;
            for (int k = tid % parts; k < count; k += parts) rank += better(s_list[k], c);
            if (parts >= 4) {
                rank = join<0>(rank, [](int a, int b) { return a + b; });
                rank = join<1>(rank, [](int a, int b) { return a + b; });
            }
            if (parts == 8) rank = join<2>(rank, [](int a, int b) { return a + b; });
            if (tid % parts == 0 && rank < A.n_select) put(rank, c);
        }
        return;
    }
    Choice last = {INFINITY, 0};
    for (int k = 0; k < A.n_select; ++k) {
        Choice top = {-INFINITY, none};
        for (unsigned i = tid; i < total; i += kPickThreads) {
            const Choice c = choice(i);
            if (c.place != none && (k == 0 || better(last, c)) && better(c, top)) top = c;
        }
#pragma unroll
        for (int d = 32; d >= 1; d /= 2) {
            const Choice o = {__shfl_xor(top.score, d, 64), __shfl_xor(top.place, d, 64)};
            if (better(o, top)) top = o;
        }
        if (lane == 0) s_best[wave] = top;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kPickWaves; ++w)
                if (better(s_best[w], top)) top = s_best[w];
            s_last = top;
            put(k, top);
        }
        __syncthreads();
        last = s_last;
    }
}

// Vocabulary per workgroup of the first launch: 8192, or 2048 where that leaves compute units without work (both
// launches and the histories, 4 rows of 32000: 10.5 us, 11.4 with 8192; 192 rows of 100003: 23 us with 8192, 28 with 2048).
constexpr size_t kManySlices = 256;
static size_t slices_of(int pieces, int vocab) {
    const size_t slice = (size_t)pieces * kBeamThreads * 8;
    return ((size_t)vocab + slice - 1) / slice;
}
static int pieces_of(size_t rows, int vocab) { return rows * slices_of(4, vocab) >= kManySlices ? 4 : 1; }
static size_t slice_bytes(int n_select) { return sizeof(SliceStats) + (size_t)n_select * sizeof(unsigned); }

struct AdvanceArgs {
    const int *history, *lens;
    const uint8_t* finished;
    const int *parents, *tokens;
    int *history_out, *lens_out;
    uint8_t* finished_out;
    int n_in, stride, end_token;
};

__global__ void __launch_bounds__(256) beam_advance_kernel(AdvanceArgs A) {
    const int row = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x;
    const int parent = A.parents[row];
    const bool has = parent >= 0 && parent < A.n_in;
    const int len = has ? min(max(A.lens[parent], 0), A.stride) : 0;
    const bool done = !has || (A.finished && A.finished[parent]);
    const int token = A.tokens[row];
    const bool room = len < A.stride;
    if (c < A.stride) A.history_out[(size_t)row * A.stride + c] = c < len ? A.history[(size_t)parent * A.stride + c] : c == len && !done ? token : 0;
    if (c == 0) {
        A.lens_out[row] = len + (!done && room);
        A.finished_out[row] = done || !room || token == A.end_token;
    }
}

}  // namespace tl

extern "C" {

size_t tl_beam_select_workspace(int n_batch, int n_beams, int vocab, int n_select) {
    if (n_batch <= 0 || n_beams <= 0 || vocab <= 0 || n_select <= 0) return 0;
    const size_t rows = (size_t)n_batch * n_beams;
    // Calls in short slices have fewer than kManySlices long ones, so at most four times as many.
    const size_t few = std::min(rows * tl::slices_of(1, vocab), 4 * (tl::kManySlices - 1));
    return std::max(rows * tl::slices_of(4, vocab), few) * tl::slice_bytes(n_select);
}

int tl_beam_select_f16(float* scores_out, int* tokens_out, int* parents_out, const void* logits, size_t logits_stride, const float* scores,
                       const uint8_t* finished, int n_batch, int n_beams, int vocab, int n_select, int end_token, void* workspace,
                       size_t workspace_bytes) {
    using namespace tl;
    const char* what = "tl_beam_select_f16";
    TL_REQUIRE(n_batch >= 0 && n_beams >= 1 && vocab >= 1 && n_select >= 1, "%s: sizes out of range", what);
    if (n_select > kMaxSelect || n_beams > 1024) return set_error(TL_ELIMIT, "%s: selects at most %d of at most 1024 beams", what, kMaxSelect);
    TL_REQUIRE((size_t)n_select <= (size_t)n_beams * vocab, "%s: %d continuations of %d beams over %d tokens do not exist", what, n_select, n_beams, vocab);
    TL_REQUIRE(!finished || (end_token >= 0 && end_token < vocab), "%s: end token %d is outside the vocabulary", what, end_token);
    if (n_batch == 0) return TL_OK;
    TL_REQUIRE(scores_out && tokens_out && parents_out && logits && scores, "%s: null pointer", what);
    TL_REQUIRE((reinterpret_cast<uintptr_t>(logits) & 1u) == 0, "%s: misaligned logits", what);
    TL_REQUIRE(logits_stride >= (size_t)vocab || (n_batch == 1 && n_beams == 1), "%s: the row stride must cover the vocabulary", what);
    const size_t rows = (size_t)n_batch * n_beams;
    if (rows > 65535) return set_error(TL_ELIMIT, "%s: %zu rows, at most 65535", what, rows);
    const int pieces = pieces_of(rows, vocab);
    const size_t slices = slices_of(pieces, vocab);
    const size_t per_row = slices * n_select > (size_t)n_select + 1 ? slices * n_select : (size_t)n_select + 1;
    if (per_row * n_beams >= (1u << 31)) return set_error(TL_ELIMIT, "%s: a vocabulary of %d is too large for %d beams", what, vocab, n_beams);
    const size_t need = rows * slices * slice_bytes(n_select);
    TL_REQUIRE(workspace && workspace_bytes >= need && aligned16(workspace), "%s: needs an aligned workspace of %zu bytes, got %zu", what, need,
               workspace ? workspace_bytes : (size_t)0);
    TL_ENSURE_INIT();
    BeamArgs A{};
    A.logits = static_cast<const half_t*>(logits);
    A.logits_stride = logits_stride;
    A.scores = scores;
    A.finished = finished;
    A.scores_out = scores_out;
    A.tokens_out = tokens_out;
    A.parents_out = parents_out;
    A.stats = static_cast<SliceStats*>(workspace);
    A.best = reinterpret_cast<unsigned*>(A.stats + rows * slices);
    A.by_row = FastDiv((unsigned)per_row);
    A.n_beams = n_beams;
    A.vocab = vocab;
    A.n_select = n_select;
    A.end_token = end_token;
    A.n_slices = (int)slices;
    A.slice = pieces * kBeamThreads * 8;
    const dim3 grid((unsigned)slices, (unsigned)rows);
    if (pieces == 4) beam_rows_kernel<4><<<grid, kBeamThreads, 0, stream()>>>(A);
    else beam_rows_kernel<1><<<grid, kBeamThreads, 0, stream()>>>(A);
    TL_CHECK_LAUNCH("beam_rows_kernel");
    // 512 threads where they hold all continuations and have a wavefront for each beam (4 beams x 32000: 9.8 us, 10.1 with 1024)
    const size_t lds = n_beams * (sizeof(double) + sizeof(int));
    if (n_beams <= 8 && per_row * n_beams <= kHeld * 512) beam_pick_kernel<512><<<n_batch, 512, lds, stream()>>>(A);
    else beam_pick_kernel<1024><<<n_batch, 1024, lds, stream()>>>(A);
    TL_CHECK_LAUNCH("beam_pick_kernel");
    return TL_OK;
}

int tl_beam_advance(int* history_out, int* lens_out, uint8_t* finished_out, const int* history, const int* lens, const uint8_t* finished,
                    const int* parents, const int* tokens, int n_in, int n_out, int stride, int end_token) {
    using namespace tl;
    const char* what = "tl_beam_advance";
    TL_REQUIRE(n_in >= 0 && n_out >= 0 && stride >= 1, "%s: sizes out of range", what);
    if (n_out > 65535) return set_error(TL_ELIMIT, "%s: %d rows, at most 65535", what, n_out);
    if (n_out == 0) return TL_OK;
    TL_REQUIRE(history_out && lens_out && finished_out && parents && tokens && (n_in == 0 || (history && lens)), "%s: null pointer", what);
    TL_REQUIRE(history_out != history && lens_out != lens && finished_out != finished, "%s: the new histories must not lie over the old ones", what);
    TL_ENSURE_INIT();
    AdvanceArgs A{history, lens, finished, parents, tokens, history_out, lens_out, finished_out, n_in, stride, end_token};
    beam_advance_kernel<<<dim3((stride + 255) / 256, n_out), 256, 0, stream()>>>(A);
    TL_CHECK_LAUNCH("beam_advance_kernel");
    return TL_OK;
}

}  // extern "C"
