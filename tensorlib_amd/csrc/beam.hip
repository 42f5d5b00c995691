// Beam search: selection over beams and vocabulary, and the reordering of the beams' token histories.
//
// Every beam of a request continues with every token at  score + logit - log sum exp(logits);  the best n of a request
// go on, equal scores in the order of (beam, token).  A finished beam has one continuation, its end token at its own
// score.  The sum of a row is held in fp64 and scores are compared in fp64: candidates of different beams may lie
// closer than an fp32 rounding.
//
// Bound by the one pass over the logits (2 bytes each; small requests by latency).  First launch: one workgroup per
// (row, slice of the vocabulary) holds its slice in registers, leaves the slice's maximum and sum and its best n
// candidates: within a row, the order of the logits is the order of the scores, so no sum is needed for that.  Second
// launch: one workgroup per request joins the rows' sums and picks.
#include <cmath>

#include "tl_internal.h"

namespace tl {

typedef unsigned long long u64;

constexpr int kBeamThreads = 256;
constexpr int kPerThread = 32;                            // logits a thread holds
constexpr int kSlice = kBeamThreads * kPerThread;
constexpr int kMaxSelect = 64;

struct SliceStats {
    double sum;                                           // of exp(logit - top)
    float top;
    float pad;
};

struct BeamArgs {
    const half_t* logits;
    size_t logits_stride;
    const float* scores;
    const uint8_t* finished;
    float* scores_out;
    int *tokens_out, *parents_out;
    SliceStats* stats;                                    // [row][slice]
    u64* best;                                            // [row][slice][n_select]
    int n_beams, vocab, n_select, end_token, n_slices;
};

// Larger is better: the logit's order (the two zeros are equal), then the lower index.  Never 0.
__device__ __forceinline__ u64 candidate(half_t x, int index) {
    unsigned b = __builtin_bit_cast(unsigned short, x);
    if (b == 0x8000u) b = 0;
    b = b & 0x8000u ? (~b & 0xffffu) : (b | 0x8000u);
    return ((u64)b << 32) | (unsigned)~index;
}
__device__ __forceinline__ float candidate_logit(u64 c) {
    unsigned b = (unsigned)(c >> 32);
    b = b & 0x8000u ? (b & 0x7fffu) : (~b & 0xffffu);
    return (float)__builtin_bit_cast(half_t, (unsigned short)b);
}
__device__ __forceinline__ int candidate_index(u64 c) { return (int)~(unsigned)c; }

__device__ __forceinline__ u64 wave_max(u64 v) {
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) {
        const u64 o = __shfl_xor(v, d, 64);
        v = o > v ? o : v;
    }
    return v;
}

// exp(d) for d <= 0 to about an ulp: the product with log2 e is carried in two floats.
__device__ __forceinline__ float exp_of(float d) {
    const float hi = d * 1.4426950408889634f;
    const float lo = __builtin_fmaf(d, 1.4426950408889634f, -hi) + d * 1.9259629911266175e-8f;
    const float e = __builtin_amdgcn_exp2f(hi);
    return d == -INFINITY ? 0.f : __builtin_fmaf(e, lo * 0.6931471805599453f, e);
}

__global__ void __launch_bounds__(kBeamThreads) beam_rows_kernel(BeamArgs A) {
    __shared__ u64 s_best[kBeamThreads / 64];
    __shared__ float s_top[kBeamThreads / 64];
    __shared__ double s_sum[kBeamThreads / 64];
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    if (A.finished && A.finished[row]) return;
    const int v0 = slice * kSlice;
    const int n = A.vocab - v0 < kSlice ? A.vocab - v0 : kSlice;
    const half_t* x = A.logits + (size_t)row * A.logits_stride + v0;
    half_t v[kPerThread];
    float top = -INFINITY;
    bool odd = false;                                     // NaN or +inf: the row has no probabilities
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int i = j * kBeamThreads + tid;
        v[j] = i < n ? x[i] : (half_t)-INFINITY;
        odd |= !((float)v[j] < INFINITY);
        top = fmaxf(top, (float)v[j]);
    }
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
    if (tid % 64 == 0) s_top[tid / 64] = top;
    odd = __syncthreads_or(odd);
    for (int w = 0; w < kBeamThreads / 64; ++w) top = fmaxf(top, s_top[w]);
    double sum = 0.0;
    if (top > -INFINITY && !odd) {
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) sum += (double)exp_of((float)v[j] - top);
    }
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) sum += __shfl_xor(sum, d, 64);
    if (tid % 64 == 0) s_sum[tid / 64] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.0;
        for (int w = 0; w < kBeamThreads / 64; ++w) sum += s_sum[w];
        A.stats[(size_t)row * A.n_slices + slice] = {odd ? (double)NAN : sum, top, 0.f};
    }
    u64 bound = ~0ull;                                    // candidates below it have not been taken
    u64* best = A.best + ((size_t)row * A.n_slices + slice) * A.n_select;
    for (int k = 0; k < A.n_select; ++k) {
        u64 mine = 0;
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) {
            const int i = j * kBeamThreads + tid;
            const u64 c = candidate(v[j], v0 + i);
            if (i < n && c < bound && c > mine) mine = c;
        }
        mine = wave_max(mine);
        __syncthreads();
        if (tid % 64 == 0) s_best[tid / 64] = mine;
        __syncthreads();
        mine = s_best[0];
        for (int w = 1; w < kBeamThreads / 64; ++w) mine = s_best[w] > mine ? s_best[w] : mine;
        if (tid == 0) best[k] = mine;                     // 0: the slice has no more
        bound = mine;
    }
}

// A continuation of a request: better by score, then by the lower place beam * vocab + token.
struct Choice {
    double score;
    u64 place;
};
__device__ __forceinline__ bool better(const Choice& a, const Choice& b) { return a.score > b.score || (a.score == b.score && a.place < b.place); }

__global__ void __launch_bounds__(kBeamThreads) beam_pick_kernel(BeamArgs A) {
    __shared__ Choice s_best[kBeamThreads / 64];
    __shared__ Choice s_last;
    extern __shared__ double s_base[];                    // per beam: score - log sum, or -inf for a beam without continuations
    const int request = blockIdx.x, tid = threadIdx.x;
    for (int b = tid; b < A.n_beams; b += kBeamThreads) {
        const int row = request * A.n_beams + b;
        const double score = (double)A.scores[row];
        double base = -INFINITY;
        if (A.finished && A.finished[row]) {
            base = score;
        } else {
            const SliceStats* st = A.stats + (size_t)row * A.n_slices;
            float top = -INFINITY;
            for (int s = 0; s < A.n_slices; ++s) top = fmaxf(top, st[s].top);
            double sum = 0.0;
            for (int s = 0; s < A.n_slices; ++s)
                sum += st[s].sum == 0.0 ? 0.0 : st[s].sum * exp((double)st[s].top - (double)top);
            base = score - ((double)top + log(sum));
        }
        s_base[b] = base > -INFINITY && base < INFINITY ? base : -INFINITY;
    }
    __syncthreads();
    const int per_row = A.n_slices * A.n_select;
    const u64 none = ~0ull;
    Choice last = {INFINITY, 0};
    bool first = true;
    for (int k = 0; k < A.n_select; ++k) {
        Choice mine = {-INFINITY, none};
        for (int b = 0; b < A.n_beams; ++b) {
            const int row = request * A.n_beams + b;
            const double base = s_base[b];
            const bool done = A.finished && A.finished[row];
            const bool dead = !(base > -INFINITY);
            const int count = done || dead ? A.n_select + 1 : per_row;
            for (int i = tid; i < count; i += kBeamThreads) {
                Choice c;
                if (done || dead) {                       // the end token at the beam's score; all else at -inf, lowest first
                    if (i >= A.vocab && !(done && i == A.n_select)) continue;
                    const bool end = done && i == A.n_select;
                    if (done && !end && i == A.end_token) continue;
                    c = {end ? base : (double)-INFINITY, (u64)b * A.vocab + (end ? A.end_token : i)};
                } else {
                    const u64 e = A.best[(size_t)row * per_row + i];
                    if (e == 0) continue;
                    c = {base + (double)candidate_logit(e), (u64)b * A.vocab + candidate_index(e)};
                }
                if ((first || better(last, c)) && better(c, mine)) mine = c;
            }
        }
#pragma unroll
        for (int d = 32; d >= 1; d /= 2) {
            const Choice o = {__shfl_xor(mine.score, d, 64), __shfl_xor(mine.place, d, 64)};
            if (better(o, mine)) mine = o;
        }
        if (tid % 64 == 0) s_best[tid / 64] = mine;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kBeamThreads / 64; ++w)
                if (better(s_best[w], mine)) mine = s_best[w];
            s_last = mine;
            const size_t o = (size_t)request * A.n_select + k;
            A.scores_out[o] = (float)mine.score;
            A.tokens_out[o] = (int)(mine.place % A.vocab);
            A.parents_out[o] = request * A.n_beams + (int)(mine.place / A.vocab);
        }
        __syncthreads();
        last = s_last;
        first = false;
    }
}

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
    const size_t slices = ((size_t)vocab + tl::kSlice - 1) / tl::kSlice;
    return (size_t)n_batch * n_beams * slices * (sizeof(tl::SliceStats) + (size_t)n_select * sizeof(tl::u64));
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
    const size_t slices = ((size_t)vocab + kSlice - 1) / kSlice;
    if (rows > 65535) return set_error(TL_ELIMIT, "%s: %zu rows, at most 65535", what, rows);
    const size_t need = tl_beam_select_workspace(n_batch, n_beams, vocab, n_select);
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
    A.best = reinterpret_cast<u64*>(A.stats + rows * slices);
    A.n_beams = n_beams;
    A.vocab = vocab;
    A.n_select = n_select;
    A.end_token = end_token;
    A.n_slices = (int)slices;
    beam_rows_kernel<<<dim3((unsigned)slices, (unsigned)rows), kBeamThreads, 0, stream()>>>(A);
    TL_CHECK_LAUNCH("beam_rows_kernel");
    beam_pick_kernel<<<n_batch, kBeamThreads, n_beams * sizeof(double), stream()>>>(A);
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
