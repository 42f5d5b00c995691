// Attention of one new token per sequence over the pages of a key-value cache, kv heads shared by groups of query heads.
//
//   out[b, h, :] = sum_t p_t V[t, g(h), :] / sum_t p_t,   p_t = exp(scale q.K_t - max),   t < lens[b]
//
// Bound by memory: K and V are read once (4 len kv_heads head_dim bytes).  The length is cut into chunks, one workgroup
// per (sequence, kv head, chunk), four wavefronts that take 16 or 32 positions each in turn; more than one chunk leaves
// fp32 partials (max, sum, weighted values) for a second launch to join.  Chunks with no positions leave at once.
//
// Both products run on the matrix cores with the query heads of a group as the 16 columns of a tile; a group of one wastes
// 15 columns, and the matrix cores are still busy for less than a tenth of the time.  The scores are K (16 positions x
// dims) times Q^T: lane (n = lane % 16, g = lane / 16) ends up with head n and positions 4 g + r of each tile.  That is
// what the second product, V^T (dims x positions) times the weights, wants as its right operand, positions being free to
// stand in any order along k.  For the left one each lane loads 16-byte pieces of exactly those positions of V, and the
// eight positions of one dimension come together within the lane: no LDS, no exchange between lanes.  A weight goes in
// as the sum of two halves, 22 bits of it.  (The fp32 product, which takes the weights as they are, has operand
// layouts that need no exchange at all; its rate made 0.9 us of a 32-position turn: 13.7 against 12.4 us for 1 x 2048
// positions of 32 heads, 108 against 92 us for 16 x 8000 positions of 256 dims.)
//
// Measured (one pass, both launches): 64 sequences of 65 to 4097 positions, 32 heads on 8 of 128: 106 us = 5.2 TB/s; in
// the middle of the launch the memory runs at 6.0, the rest is the first requests' and the last workgroups' time.
// 4 sequences of 100001 to 131072, 64 heads on 8: 320 us = 5.95 TB/s.  1 x 2048, 32 heads: 12.0 us, of which the two
// launches of an empty problem take 8.
#include <algorithm>
#include <cmath>

#include "paged.h"

namespace tl {

constexpr int kWaves = 4;
constexpr int kMinChunk = 128, kMaxChunk = 1024;   // positions of a workgroup, a power of two
constexpr int kGroupTile = 16;            // query heads that share a pass over K and V
constexpr float kLog2e = 1.4426950408889634f;
// Weights are kept 2^12 times as large as exp(score - max), in the sum too.  As two halves, the first truncated and the second
// rounded, a weight is off by at most 2^-21 of itself; where the parts are subnormal or raised to kTiny, by less than 2 kTiny,
// which is 2^-35 of the largest weight.
constexpr float kWeightLog2 = 12.f;
constexpr float kTiny = 5.9604644775390625e-8f;   // 2^-24, the smallest positive half

struct PagedAttnArgs {
    half_t* out;
    const half_t* q;
    size_t q_stride;
    tl_kv_pages cache;
    const int* tables;
    size_t table_stride;
    const int* lens;
    float* part_o;                        // [seq][split][head][head_dim]
    float2* part_ml;                      // [seq][split][head] (max in log2 units, sum)
    FastDiv by_page, by_heads, by_splits; // grid: (kv head tile) fastest, then split, then sequence
    int n_heads, group, group_tiles, max_len, chunk, n_splits, turn_heads;
    float scale_log2;
};

// f over the four lanes of a column (16 and 32 apart), by swapping rows of lanes in the vector pipe.  (The elements are copied
// out of the returned vector first: a bit cast of an element itself reads element 0.)
template <class F>
__device__ __forceinline__ float over_column(float v, F f) {
    const unsigned a = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    const unsigned r0 = r[0], r1 = r[1];
    const unsigned b = __builtin_bit_cast(unsigned, f(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1)));
    const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    const unsigned q0 = q[0], q1 = q[1];
    return f(__builtin_bit_cast(float, q0), __builtin_bit_cast(float, q1));
}

// LDS: the offsets of the chunk's positions, then every wavefront's weighted values of every head of the tile.
template <int DP>
static size_t attention_lds(int chunk, int group) {
    return chunk * sizeof(long) + (size_t)kWaves * (group < kGroupTile ? group : kGroupTile) * DP * sizeof(float);
}

// DP: head_dim rounded up to 64, 128 or 256 (EXACT: equal to it).  U: 16-position tiles per turn of a wavefront; one for
// DP 256, whose rows fill twice the registers.  STREAM: V, whose rows come a whole line per request, is read past the caches (K
// comes half a line per request, and the second half has to find the first one's line).
template <int DP, bool EXACT, bool STREAM>
__global__ void __launch_bounds__(256, 2) paged_attention_kernel(PagedAttnArgs A) {
    constexpr int U = DP == 256 ? 1 : 2;
    constexpr int kTile = 16 * U;         // positions of a turn
    constexpr int VD = DP / 16;           // dims of V per lane
    typedef _Float16 vpiece __attribute__((ext_vector_type(VD < 8 ? VD : 8)));
    constexpr int VP = VD / (VD < 8 ? VD : 8);
    constexpr int KJ = DP / 32;
    typedef _Float16 weights __attribute__((ext_vector_type(4 * U)));
    extern __shared__ __align__(16) unsigned char s_dynamic[];
    __shared__ float s_ml[kWaves][2][kGroupTile];

    unsigned head_tile, split;
    const unsigned pair = A.by_heads.divmod(blockIdx.x, head_tile), seq = A.by_splits.divmod(pair, split);
    // Workgroups go to the eight dies in turn, so eight kv heads in order would leave each die with one of them, whose rows lie in
    // one eighth of its L2's channels: the heads of each next pair start elsewhere.
    if (A.turn_heads) A.by_heads.divmod(head_tile + (pair + pair / 2 + pair / 4) % 65536, head_tile);
    const int t0 = (int)split * A.chunk;
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int col = lane % 16, grp = lane / 16;
    const int kv_head = (int)head_tile / A.group_tiles;
    const int g0 = ((int)head_tile % A.group_tiles) * kGroupTile;
    const int heads = A.group - g0 < kGroupTile ? A.group - g0 : kGroupTile;
    const int head0 = kv_head * A.group + g0;
    const int D = EXACT ? DP : A.cache.head_dim;
    long* s_slot = reinterpret_cast<long*>(s_dynamic) + wave * (A.chunk / kWaves);         // the wavefront's own positions
    float* s_o = reinterpret_cast<float*>(s_dynamic + A.chunk * sizeof(long));             // [wave][head][DP]

    // The length, the chunk's table entries and the queries are requested together, before any of them is needed.  A
    // wavefront looks up its own positions only (a turn's of every four), so no barrier stands before its first rows.
    const int* table = A.tables + (size_t)seq * A.table_stride;
    constexpr int LOOKUPS = kMaxChunk / (kWaves * 64);
    int page[LOOKUPS];
    unsigned row[LOOKUPS];
#pragma unroll
    for (int x = 0; x < LOOKUPS; ++x) {
        const int i = (x * (64 / kTile) + lane / kTile) * (kWaves * kTile) + wave * kTile + lane % kTile;      // position in the chunk
        page[x] = 0;
        row[x] = 0;
        if (i < A.chunk) {
            const unsigned at = A.by_page.divmod((unsigned)t0 + (unsigned)i, row[x]);
            if (at < A.table_stride) page[x] = table[at];
        }
    }
    // queries: column = head, 8 dims per lane group; columns past the group and dims past the head hold zeros
    half8_t qf[KJ];
    const half8_t zero8 = {0, 0, 0, 0, 0, 0, 0, 0};
    {
        const half_t* q = A.q + (size_t)seq * A.q_stride + (size_t)(head0 + (col < heads ? col : 0)) * D;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
            const int d = 32 * j + 8 * grp;
            qf[j] = *reinterpret_cast<const half8_t*>(q + (EXACT || d < D ? d : 0));
        }
    }
    const int len = A.lens[seq];
    // a length beyond what the tables or the caller's bound cover: the first chunk answers NaN for the sequence
    const bool too_long = len > 0 && (len > A.max_len || (size_t)A.by_page.div((unsigned)len - 1u) >= A.table_stride);
    if (split != 0 && (too_long || t0 >= len)) return;
    if (len <= 0 || too_long) {           // nothing to attend to: zeros
        const half_t fill = too_long ? (half_t)NAN : (half_t)0.f;
        half_t* o = A.out + ((size_t)seq * A.n_heads + head0) * D;
        for (int i = tid; i < heads * D; i += 256) o[i] = fill;
        return;
    }
    const int n = len - t0 < A.chunk ? len - t0 : A.chunk;
    // element offsets of the positions; a page id out of range poisons the result and reads page 0
    bool bad = false;
#pragma unroll
    for (int x = 0; x < LOOKUPS; ++x) {
        const int i = (x * (64 / kTile) + lane / kTile) * (kWaves * kTile) + wave * kTile + lane % kTile;
        if (page[x] < 0 || page[x] >= A.cache.n_pages) {
            bad |= i < n;
            page[x] = 0;
        }
        if (i < A.chunk)
            s_slot[x * 64 + lane] = (long)((size_t)page[x] * A.cache.page_stride + (size_t)row[x] * A.cache.row_stride);
    }
    bad = __any(bad);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // other lanes read these offsets
#pragma unroll
    for (int j = 0; j < KJ; ++j)
        if (col >= heads || (!EXACT && 32 * j + 8 * grp >= D)) qf[j] = zero8;

    const half_t* kbase = static_cast<const half_t*>(A.cache.k) + (size_t)kv_head * A.cache.head_stride;
    const half_t* vbase = static_cast<const half_t*>(A.cache.v) + (size_t)kv_head * A.cache.head_stride;
    half8_t kf[U][KJ];
    vpiece vf[U][4][VP];
    // Rows of the wavefront's turn `s` (16 U positions).  Positions behind the end read what their table entry names, page
    // 0 if it names none: inside the cache in any case.  The fences keep the requests where they stand: the compiler
    // would move those of the next turn's V behind the wait for its K.
    auto load_k = [&](int s) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const half_t* p = kbase + s_slot[s * kTile + 16 * u + col];
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                const int d = 32 * j + 8 * grp;
                kf[u][j] = *reinterpret_cast<const half8_t*>(p + (EXACT || d < D ? d : 0));
            }
        }
        asm volatile("" ::: "memory");
    };
    auto load_v = [&](int s) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const half_t* p = vbase + s_slot[s * kTile + 16 * u + 4 * grp + r];
#pragma unroll
                for (int x = 0; x < VP; ++x) {
                    const int d = VP == 1 ? col * VD : 8 * col + 128 * x;      // a row's line is in one request
                    const vpiece* v = reinterpret_cast<const vpiece*>(p + (EXACT || d < D ? d : 0));
                    vf[u][r][x] = STREAM ? __builtin_nontemporal_load(v) : *v;
                }
            }
        asm volatile("" ::: "memory");
    };

    float4_t acc[VD];
#pragma unroll
    for (int i = 0; i < VD; ++i) acc[i] = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;         // running maximum (whole column) and this lane's share of the sum
    int t = wave * kTile, turn = 0;
    if (t < n) {
        load_k(0);
        load_v(0);
    }
    for (; t < n; t += kWaves * kTile, ++turn) {
        float4_t sc[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            sc[u] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                half8_t a = kf[u][j];
                if (!EXACT && 32 * j + 8 * grp >= D) a = zero8;
                sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[j], sc[u], 0, 0, 0);
            }
        }
        const int next = t + kWaves * kTile;
        if (next < n) load_k(turn + 1);
        float p[U][4];
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[u][r] = t + 16 * u + 4 * grp + r < n ? sc[u][r] * A.scale_log2 : -INFINITY;
                mx = fmaxf(mx, p[u][r]);
            }
        mx = over_column(mx, [](float a, float b) { return fmaxf(a, b); });
        const float m_new = fmaxf(m, mx);
        const float base = m_new == -INFINITY ? 0.f : m_new;   // a column of -inf so far has weights of zero
        const float alpha = __builtin_amdgcn_exp2f(m - base);
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < VD; ++i) acc[i] *= alpha;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[u][r] = __builtin_amdgcn_exp2f(p[u][r] - base + kWeightLog2);
                l += p[u][r];
            }
        if (t + kTile > n) {              // what lies behind the end may hold anything, and 0 times it must be 0
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (t + 16 * u + 4 * grp + r >= n) {
#pragma unroll
                        for (int x = 0; x < VP; ++x) vf[u][r][x] = (vpiece)(half_t)0.f;
                    }
        }
        // p as the sum of two halves.  hi is rounded towards zero and neither part of a
        // positive weight becomes zero, so that an infinite value keeps its sign.  The eight (four) positions of a lane
        // come together as A[row = dims, k = position] by exchanges within the lane.
        weights hi, lo;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float x = p[u][r], tiny = x > 0.f ? kTiny : 0.f;
                const half_t h = (half_t)__builtin_amdgcn_cvt_pkrtz(fmaxf(x, tiny), 0.f)[0];
                hi[4 * u + r] = h;
                lo[4 * u + r] = (half_t)fmaxf(x - (float)h, tiny);
            }
#pragma unroll
        for (int i = 0; i < VD; ++i) {
            weights a;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) a[4 * u + r] = vf[u][r][i / 8][i % 8];
            if constexpr (U == 2) {
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, hi, acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, lo, acc[i], 0, 0, 0);
            } else {
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x16f16(a, hi, acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x16f16(a, lo, acc[i], 0, 0, 0);
            }
        }
        if (next < n) load_v(turn + 1);
    }

    // join the wavefronts: lane (col, grp) holds head col, dims (4 grp + r) * VD + i
    l = over_column(l, [](float a, float b) { return a + b; });
    if (grp == 0) {
        s_ml[wave][0][col] = m;
        s_ml[wave][1][col] = bad ? NAN : l;
    }
    if (col < heads) {
#pragma unroll
        for (int i = 0; i < VD; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) s_o[(wave * heads + col) * DP + (VP == 1 ? (4 * grp + r) * VD + i : 8 * (4 * grp + r) + 128 * (i / 8) + i % 8)] = acc[i][r];
    }
    __syncthreads();
    const bool whole = len <= A.chunk;    // the only chunk: the result itself
    const size_t part = ((size_t)seq * A.n_splits + split) * A.n_heads + head0;
    for (int i = tid; i < heads * D; i += 256) {
        const int h = i / D, d = i % D;
        float mw[kWaves], top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            mw[w] = s_ml[w][0][h];
            top = fmaxf(top, mw[w]);
        }
        float sum = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = mw[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw[w] - top);   // 0 * NaN stays NaN
            sum += f * s_ml[w][1][h];
            o += f * s_o[(w * heads + h) * DP + d];
        }
        if (whole) {
            A.out[((size_t)seq * A.n_heads + head0) * D + i] = (half_t)(o / sum);
        } else {
            A.part_o[part * D + i] = o;
            if (d == 0) A.part_ml[part + h] = make_float2(top, sum);
        }
    }
}

// Joins the chunks of one (head, sequence): D / 4 threads take four dims each of every n-th chunk, several chunks' loads in
// flight together (a dependent load per chunk would cost a memory latency each), then the groups of threads join in LDS.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) paged_attention_join_kernel(PagedAttnArgs A) {
    constexpr int U = 8;
    __shared__ float4_t s_o[THREADS];
    __shared__ float s_m[THREADS], s_l[THREADS];
    const int h = blockIdx.x, seq = blockIdx.y, D = A.cache.head_dim;
    const int per = D / 4, groups = THREADS / per;
    const int grp = threadIdx.x / per, d = (threadIdx.x % per) * 4;
    const size_t part = (size_t)seq * A.n_splits * A.n_heads + h;
    // A turn of chunks.  The first one's are requested before the length is known, one memory latency less (1 x 2048: 12.6 ->
    // 12.0 us); what lies behind the length is not looked at.
    float2 ml[U];
    float4_t x[U];
    auto load = [&](int i0, int n) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * groups;
            if (i >= n) break;
            const size_t at = part + (size_t)i * A.n_heads;
            ml[u] = A.part_ml[at];
            x[u] = *reinterpret_cast<const float4_t*>(A.part_o + at * D + d);
        }
    };
    if (grp < groups) load(grp, A.n_splits);
    const int len = A.lens[seq];
    if (len <= A.chunk || len > A.max_len || (size_t)((len - 1) / A.cache.page_size) >= A.table_stride) return;
    const int n = (len + A.chunk - 1) / A.chunk;
    float m = -INFINITY, l = 0.f;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
    if (grp < groups) {
        for (int i0 = grp; i0 < n; i0 += U * groups) {
            if (i0 != grp) load(i0, n);
            float m_new = m;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i0 + u * groups < n) m_new = fmaxf(m_new, ml[u].x);
            const float base = m_new == -INFINITY ? 0.f : m_new;
            const float f0 = __builtin_amdgcn_exp2f(m - base);
            l *= f0;
            o *= f0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i0 + u * groups >= n) break;
                const float f = __builtin_amdgcn_exp2f(ml[u].x - base);
                l += ml[u].y * f;
                o += x[u] * f;
            }
            m = m_new;
        }
    }
    s_m[threadIdx.x] = m;
    s_l[threadIdx.x] = l;
    s_o[threadIdx.x] = o;
    __syncthreads();
    if (grp != 0) return;
    for (int g = 1; g < groups; ++g) m = fmaxf(m, s_m[threadIdx.x + g * per]);
    const float base = m == -INFINITY ? 0.f : m;
    l = 0.f;
    o = {0.f, 0.f, 0.f, 0.f};
    for (int g = 0; g < groups; ++g) {
        const float f = __builtin_amdgcn_exp2f(s_m[threadIdx.x + g * per] - base);
        l += s_l[threadIdx.x + g * per] * f;
        o += s_o[threadIdx.x + g * per] * f;
    }
    half4_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (half_t)(o[i] / l);
    *reinterpret_cast<half4_t*>(A.out + ((size_t)seq * A.n_heads + h) * D + d) = r;
}

constexpr double kUnits = 256.0, kMany = 6 * kUnits;
constexpr int kLongContext = 32768;
static double dims_of(int head_dim) { return head_dim <= 64 ? 0.5 : head_dim <= 128 ? 1.0 : 2.0; }

// Positions per workgroup.  With fewer workgroups than six times the 256 compute units, the least of: positions that the fullest
// unit goes through one after the other, 42 more for each workgroup it is given, 240 for the join (in units of 128 dims, fitted
// to thirty sizes).  It cuts 1 x 4096 on 8 kv heads into chunks of 128 (10.2 us, 13.7 with 512), 1 x 131072 on one into 512
// (20.5, 28.2 with 128), 2 x 60000 on 2 into 1024 (29.5, 37 with 128), and leaves 64 x 700 on 8 whole (29.5, 42 with 512).  With
// more: 512, since the last workgroups of a ragged batch then end close together (64 of 65 to 4097 positions on 8, heads in order: 114 us,
// 117 with 1024, 135 with 128), 1024 for long contexts, where the partials are what can be saved (4 x 131072: 320, 332 with 512),
// and where it leaves sequences whole (200 x 600: 60, 87 with 512).
static int chunk_of(int n_seqs, int head_tiles, int head_dim, int max_len) {
    const double tiles = (double)n_seqs * head_tiles, dims = dims_of(head_dim);
    int best = kMaxChunk;
    if (tiles * ceil(max_len / 512.0) * dims >= kMany) {
        if (max_len > kMaxChunk && max_len <= kLongContext) best = kMaxChunk / 2;
    } else {
        double least = 1e300;
        for (int chunk = kMaxChunk; chunk >= kMinChunk; chunk /= 2) {
            const double groups = tiles * ceil((double)max_len / chunk);
            const double time = ceil(groups / kUnits) * (chunk < max_len ? chunk : max_len) * dims + 42.0 * groups / kUnits + (chunk < max_len ? 240.0 : 0.0);
            if (time < least) {
                best = chunk;
                least = time;
            }
        }
    }
    while (best > kMinChunk && best / 2 >= max_len) best /= 2;
    return best;
}
// At least the chunks, of all sequences together, of any call with at most n_seqs sequences and a bound of at most max_len.  Calls with
// many workgroups have chunks of 512 up to kLongContext and of 1024 beyond.  The others have n_seqs * head_tiles * ceil(max_len / 512) below
// kMany / dims, and in chunks of 128, the smallest, at most four times as many.  Up to 128 positions are one chunk.
static size_t most_chunks(int n_seqs, int head_tiles, int head_dim, int max_len) {
    if (max_len <= kMinChunk) return 0;
    const double n = n_seqs, most = kMany / (dims_of(head_dim) * head_tiles);
    double chunks = n * ceil(max_len / (double)kMinChunk);
    if (n * ceil(max_len / 512.0) >= most) {
        const double many = n * std::max(ceil(std::min(max_len, kLongContext) / 512.0), ceil(max_len / (double)kMaxChunk));
        chunks = std::min(chunks, std::max(many, ceil(4.0 * most)));
    }
    return (size_t)(ceil(chunks / n) * n);
}
static int group_tiles_of(int n_heads, int n_kv_heads) { return (n_heads / n_kv_heads + kGroupTile - 1) / kGroupTile; }

template <int DP>
static void launch_paged_attention(const PagedAttnArgs& A, unsigned blocks, bool past) {
    const size_t lds = attention_lds<DP>(A.chunk, A.group);
    auto kernel = A.cache.head_dim == DP ? (past ? paged_attention_kernel<DP, true, true> : paged_attention_kernel<DP, true, false>)
                                         : (past ? paged_attention_kernel<DP, false, true> : paged_attention_kernel<DP, false, false>);
    kernel<<<blocks, 256, lds, stream()>>>(A);
}

}  // namespace tl

extern "C" {

size_t tl_paged_attention_workspace(int n_seqs, int n_heads, int n_kv_heads, int head_dim, int max_len) {
    if (n_seqs <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || head_dim <= 0 || max_len <= 0) return 0;
    return tl::most_chunks(n_seqs, n_kv_heads * tl::group_tiles_of(n_heads, n_kv_heads), head_dim, max_len) * n_heads * ((size_t)head_dim + 2) * sizeof(float);
}

size_t tl_paged_attention_workspace_of_call(int n_seqs, int n_heads, int n_kv_heads, int head_dim, int max_len) {
    if (n_seqs <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || head_dim <= 0 || max_len <= 0) return 0;
    const int chunk = tl::chunk_of(n_seqs, n_kv_heads * tl::group_tiles_of(n_heads, n_kv_heads), head_dim, max_len);
    const size_t splits = ((size_t)max_len + chunk - 1) / chunk;
    return splits <= 1 ? 0 : splits * n_seqs * n_heads * ((size_t)head_dim + 2) * sizeof(float);
}

int tl_paged_attention_f16(void* out, const void* q, size_t q_stride, const tl_kv_pages* cache, const int* tables, size_t table_stride,
                           const int* lens, int n_seqs, int n_heads, int max_len, float scale, void* workspace, size_t workspace_bytes) {
    using namespace tl;
    const char* what = "tl_paged_attention_f16";
    int rc = check_kv_pages(cache, what);
    if (rc != TL_OK) return rc;
    TL_REQUIRE(n_seqs >= 0 && n_heads >= 1 && max_len >= 0, "%s: sizes out of range", what);
    TL_REQUIRE(n_heads % cache->n_kv_heads == 0, "%s: %d query heads do not share %d kv heads evenly", what, n_heads, cache->n_kv_heads);
    TL_REQUIRE(std::isfinite(scale), "%s: scale must be finite", what);
    if (n_seqs == 0) return TL_OK;
    TL_REQUIRE(out && q && lens && (tables || table_stride == 0), "%s: null pointer", what);
    TL_REQUIRE((reinterpret_cast<uintptr_t>(out) & 7u) == 0, "%s: the output must be 8-byte aligned", what);
    TL_REQUIRE(aligned16(q) && (n_seqs == 1 || q_stride % 8 == 0), "%s: query rows must be 16-byte aligned", what);
    TL_REQUIRE(n_seqs == 1 || q_stride >= (size_t)n_heads * cache->head_dim, "%s: the query stride must cover the heads", what);
    PagedAttnArgs A{};
    A.group = n_heads / cache->n_kv_heads;
    A.group_tiles = group_tiles_of(n_heads, cache->n_kv_heads);
    const int head_tiles = cache->n_kv_heads * A.group_tiles;
    A.chunk = chunk_of(n_seqs, head_tiles, cache->head_dim, max_len);
    A.n_splits = max_len <= A.chunk ? 1 : (int)(((size_t)max_len + A.chunk - 1) / A.chunk);
    const size_t parts = (size_t)n_seqs * A.n_splits * n_heads;
    if (A.n_splits > 1) {
        const size_t need = parts * ((size_t)cache->head_dim + 2) * sizeof(float);
        TL_REQUIRE(workspace && workspace_bytes >= need, "%s: needs a workspace of %zu bytes, got %zu", what, need, workspace ? workspace_bytes : (size_t)0);
        TL_REQUIRE(aligned16(workspace), "%s: the workspace must be 16-byte aligned", what);
    }
    const double blocks = (double)n_seqs * A.n_splits * head_tiles;
    // threads of one dimension of a grid are counted in 32 bits
    if (blocks >= 16777216.0 || (A.n_splits > 1 && n_heads >= 4194304) || n_seqs > 65535) return set_error(TL_ELIMIT, "%s: %d sequences of up to %d positions are too many for one call", what, n_seqs, max_len);
    TL_ENSURE_INIT();
    A.out = static_cast<half_t*>(out);
    A.q = static_cast<const half_t*>(q);
    A.q_stride = q_stride;
    A.cache = *cache;
    A.tables = tables;
    A.table_stride = table_stride;
    A.lens = lens;
    A.part_o = static_cast<float*>(workspace);
    A.part_ml = reinterpret_cast<float2*>(A.part_o + parts * cache->head_dim);
    A.by_page = FastDiv((unsigned)cache->page_size);
    A.by_heads = FastDiv((unsigned)head_tiles);
    A.by_splits = FastDiv((unsigned)A.n_splits);
    A.n_heads = n_heads;
    A.max_len = max_len;
    A.scale_log2 = scale * kLog2e;
    // 64 ragged sequences of 8 kv heads of 128: 106 us, 114 in order; with few workgroups 2 % the other way (3 x 9000: 27.3, 27.0)
    A.turn_heads = blocks > 1024.0;
    // V past the caches if what the sequences may read is more than the 256 MB of the last-level one and one pass reads it
    // (4 x 131072: 320 against 352 us, 64 ragged sequences 115 against 121; a cache of 66 MB that had stayed there 24 against 21)
    const bool past = A.group_tiles == 1 && (double)n_seqs * max_len * cache->n_kv_heads * cache->head_dim * 4.0 >= 268435456.0;
    if (cache->head_dim <= 64) launch_paged_attention<64>(A, (unsigned)blocks, past);
    else if (cache->head_dim <= 128) launch_paged_attention<128>(A, (unsigned)blocks, past);
    else launch_paged_attention<256>(A, (unsigned)blocks, past);
    TL_CHECK_LAUNCH("paged_attention_kernel");
    if (A.n_splits > 1) {
        // 256 threads where they cover the chunks in one round trip (16 x 8000 positions of 64 dims: 22 us, 24 with 1024),
        // else 1024 (1 x 32768 in 256 chunks: 40 us, 45 with 256)
        if (A.n_splits <= 8 * (256 / (cache->head_dim / 4))) paged_attention_join_kernel<256><<<dim3(n_heads, n_seqs), 256, 0, stream()>>>(A);
        else paged_attention_join_kernel<1024><<<dim3(n_heads, n_seqs), 1024, 0, stream()>>>(A);
        TL_CHECK_LAUNCH("paged_attention_join_kernel");
    }
    return TL_OK;
}

}  // extern "C"
