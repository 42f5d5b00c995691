// Attention of one new token per sequence over the pages of a key-value cache, kv heads shared by groups of query heads.
//
//   out[b, h, :] = sum_t p_t V[t, g(h), :] / sum_t p_t,   p_t = exp(scale q.K_t - max),   t < lens[b]
//
// Bound by memory: K and V are read once (4 len kv_heads head_dim bytes).  The length is cut into chunks, one workgroup
// per (sequence, kv head, chunk), four wavefronts that take 32 positions each in turn; more than one chunk leaves fp32
// partials (max, sum, weighted values) for a second launch to join.  Chunks with no positions leave at once.
//
// Both products run on the matrix cores with the query heads of a group as the 16 columns of a tile (a group of one
// wastes 15 columns, and the matrix cores still have three times the rate that the memory can feed).  The scores are
// K (16 positions x dims) times Q^T, f16 in, fp32 out: lane (n = lane % 16, g = lane / 16) ends up with head n and
// positions 4 g + r.  The values then go through the fp32 product, 16 x 4 by 4 x 16, whose operand layouts are exactly
// that: step r takes position 4 g + r from lane group g, p from the registers that the scores were in, and V converted
// to fp32 on the way, one dimension of its 16-byte piece per instruction.  No transposition, no LDS round trip, and no
// rounding of p.
#include <cmath>

#include "paged.h"

namespace tl {

constexpr int kWaves = 4;
constexpr int kTile = 32;                 // positions of a wavefront's turn
constexpr int kMaxChunk = 2048;           // positions of a workgroup
constexpr int kGroupTile = 16;            // query heads that share a pass over K and V
constexpr float kLog2e = 1.4426950408889634f;

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
    int n_heads, group, group_tiles, max_len, chunk, n_splits;
    float scale_log2;
};

template <int DP, bool EXACT>
__global__ void __launch_bounds__(256, DP == 256 ? 1 : 2) paged_attention_kernel(PagedAttnArgs A) {
    constexpr int VD = DP / 16;           // dims of V per lane
    typedef _Float16 vpiece __attribute__((ext_vector_type(VD < 8 ? VD : 8)));
    constexpr int VP = VD / (VD < 8 ? VD : 8);
    constexpr int KJ = DP / 32;
    __shared__ long s_slot[kMaxChunk];
    __shared__ float s_ml[kWaves][2][kGroupTile];
    __shared__ float s_o[kWaves][kGroupTile][DP];
    __shared__ int s_bad;

    unsigned head_tile, split;
    const unsigned seq = A.by_splits.divmod(A.by_heads.divmod(blockIdx.x, head_tile), split);
    const int len = A.lens[seq];
    const int t0 = (int)split * A.chunk;
    // a length beyond what the tables or the caller's bound cover: the first chunk answers NaN for the sequence
    const bool too_long = len > A.max_len || (size_t)(len > 0 ? (len - 1) / A.cache.page_size : 0) >= A.table_stride;
    if (split != 0 && (too_long || t0 >= len)) return;
    const int kv_head = (int)head_tile / A.group_tiles;
    const int g0 = ((int)head_tile % A.group_tiles) * kGroupTile;
    const int heads = A.group - g0 < kGroupTile ? A.group - g0 : kGroupTile;
    const int head0 = kv_head * A.group + g0;
    const int D = EXACT ? DP : A.cache.head_dim;
    const int tid = threadIdx.x;
    if (len <= 0 || too_long) {           // nothing to attend to: zeros
        const half_t fill = too_long ? (half_t)NAN : (half_t)0.f;
        half_t* o = A.out + ((size_t)seq * A.n_heads + head0) * D;
        for (int i = tid; i < heads * D; i += 256) o[i] = fill;
        return;
    }
    const int n = len - t0 < A.chunk ? len - t0 : A.chunk;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    // element offset of every position of the chunk; a page id out of range poisons the result and reads page 0
    const int* table = A.tables + (size_t)seq * A.table_stride;
    for (int i = tid; i < n; i += 256) {
        unsigned row;
        const unsigned at = A.by_page.divmod((unsigned)(t0 + i), row);
        int page = table[at];
        if (page < 0 || page >= A.cache.n_pages) { page = 0; s_bad = 1; }
        s_slot[i] = (long)((size_t)page * A.cache.page_stride + (size_t)row * A.cache.row_stride);
    }
    const int lane = tid % 64, wave = tid / 64;
    const int col = lane % 16, grp = lane / 16;
    // queries: column = head, 8 dims per lane group; columns past the group and dims past the head hold zeros
    half8_t qf[KJ];
    const half8_t zero8 = {0, 0, 0, 0, 0, 0, 0, 0};
    {
        const half_t* q = A.q + (size_t)seq * A.q_stride + (size_t)(head0 + (col < heads ? col : 0)) * D;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
            const int d = 32 * j + 8 * grp;
            qf[j] = col < heads && (EXACT || d < D) ? *reinterpret_cast<const half8_t*>(q + (EXACT || d < D ? d : 0)) : zero8;
        }
    }
    __syncthreads();

    const half_t* kbase = static_cast<const half_t*>(A.cache.k) + (size_t)kv_head * A.cache.head_stride;
    const half_t* vbase = static_cast<const half_t*>(A.cache.v) + (size_t)kv_head * A.cache.head_stride;
    half8_t kf[2][KJ];
    vpiece vf[2][4][VP];
    auto load_k = [&](int t) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = t + 16 * u + col;
            const half_t* p = kbase + s_slot[i < n ? i : n - 1];
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                const int d = 32 * j + 8 * grp;
                kf[u][j] = *reinterpret_cast<const half8_t*>(p + (EXACT || d < D ? d : 0));
            }
        }
    };
    auto load_v = [&](int t) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = t + 16 * u + 4 * grp + r;
                const half_t* p = vbase + s_slot[i < n ? i : n - 1];
#pragma unroll
                for (int x = 0; x < VP; ++x) {
                    const int d = col * VD + 8 * x;
                    vf[u][r][x] = *reinterpret_cast<const vpiece*>(p + (EXACT || d < D ? d : 0));
                }
            }
    };

    float4_t acc[VD];
#pragma unroll
    for (int i = 0; i < VD; ++i) acc[i] = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;         // running maximum (whole column) and this lane's share of the sum
    int t = wave * kTile;
    if (t < n) {
        load_k(t);
        load_v(t);
    }
    for (; t < n; t += kWaves * kTile) {
        float4_t sc[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            sc[u] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                half8_t a = kf[u][j];
                if (!EXACT && 32 * j + 8 * grp >= D) a = zero8;
                sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[j], sc[u], 0, 0, 0);
            }
        }
        const int next = t + kWaves * kTile;
        if (next < n) load_k(next);
        float p[2][4];
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[u][r] = t + 16 * u + 4 * grp + r < n ? sc[u][r] * A.scale_log2 : -INFINITY;
                mx = fmaxf(mx, p[u][r]);
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m_new = fmaxf(m, mx);
        const float base = m_new == -INFINITY ? 0.f : m_new;   // a column of -inf so far has weights of zero
        const float alpha = __builtin_amdgcn_exp2f(m - base);
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < VD; ++i) acc[i] *= alpha;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[u][r] = __builtin_amdgcn_exp2f(p[u][r] - base);
                l += p[u][r];
            }
        if (t + kTile > n) {              // what lies behind the end may hold anything, and 0 times it must be 0
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (t + 16 * u + 4 * grp + r >= n) {
#pragma unroll
                        for (int x = 0; x < VP; ++x) vf[u][r][x] = (vpiece)(half_t)0.f;
                    }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < VD; ++i)
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)vf[u][r][i / 8][i % 8], p[u][r], acc[i], 0, 0, 0);
        if (next < n) load_v(next);
    }

    // join the wavefronts: lane (col, grp) holds head col, dims (4 grp + r) * VD + i
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (grp == 0) {
        s_ml[wave][0][col] = m;
        s_ml[wave][1][col] = l;
    }
    if (col < heads) {
#pragma unroll
        for (int i = 0; i < VD; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) s_o[wave][col][(4 * grp + r) * VD + i] = acc[i][r];
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
            const float f = mw[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw[w] - top);
            sum += f * s_ml[w][1][h];
            o += f * s_o[w][h][d];
        }
        if (s_bad) sum = NAN;
        if (whole) {
            A.out[((size_t)seq * A.n_heads + head0) * D + i] = (half_t)(o / sum);
        } else {
            A.part_o[part * D + i] = o;
            if (d == 0) A.part_ml[part + h] = make_float2(top, sum);
        }
    }
}

// Joins the chunks of one (head, sequence): D threads, the chunks in order.
__global__ void __launch_bounds__(256) paged_attention_join_kernel(PagedAttnArgs A) {
    const int h = blockIdx.x, seq = blockIdx.y, D = A.cache.head_dim, d = threadIdx.x;
    const int len = A.lens[seq];
    if (len <= A.chunk || len > A.max_len || (size_t)((len - 1) / A.cache.page_size) >= A.table_stride) return;
    const int n = (len + A.chunk - 1) / A.chunk;
    if (d >= D) return;
    const size_t part = (size_t)seq * A.n_splits * A.n_heads + h;
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int i = 0; i < n; ++i) {
        const float2 ml = A.part_ml[part + (size_t)i * A.n_heads];
        const float x = A.part_o[(part + (size_t)i * A.n_heads) * D + d];
        const float m_new = fmaxf(m, ml.x);
        const float base = m_new == -INFINITY ? 0.f : m_new;
        const float f0 = __builtin_amdgcn_exp2f(m - base), f1 = __builtin_amdgcn_exp2f(ml.x - base);
        l = l * f0 + ml.y * f1;
        o = o * f0 + x * f1;
        m = m_new;
    }
    A.out[((size_t)seq * A.n_heads + h) * D + d] = (half_t)(o / l);
}

// Positions per workgroup: as many as leave about four workgroups per compute unit (256 of them).
static int chunk_of(int n_seqs, int head_tiles, int max_len) {
    int chunk = kMaxChunk;
    while (chunk > kWaves * kTile && (double)n_seqs * head_tiles * ((max_len + (double)chunk - 1) / chunk) < 1024.0) chunk /= 2;
    return chunk;
}
static int group_tiles_of(int n_heads, int n_kv_heads) { return (n_heads / n_kv_heads + kGroupTile - 1) / kGroupTile; }

template <int DP>
static void launch_paged_attention(const PagedAttnArgs& A, unsigned blocks) {
    if (A.cache.head_dim == DP) paged_attention_kernel<DP, true><<<blocks, 256, 0, stream()>>>(A);
    else paged_attention_kernel<DP, false><<<blocks, 256, 0, stream()>>>(A);
}

}  // namespace tl

extern "C" {

size_t tl_paged_attention_workspace(int n_seqs, int n_heads, int n_kv_heads, int head_dim, int max_len) {
    if (n_seqs <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || head_dim <= 0 || max_len <= 0) return 0;
    const int chunk = tl::chunk_of(n_seqs, n_kv_heads * tl::group_tiles_of(n_heads, n_kv_heads), max_len);
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
    TL_REQUIRE(aligned16(q) && (n_seqs == 1 || q_stride % 8 == 0), "%s: query rows must be 16-byte aligned", what);
    TL_REQUIRE(n_seqs == 1 || q_stride >= (size_t)n_heads * cache->head_dim, "%s: the query stride must cover the heads", what);
    PagedAttnArgs A{};
    A.group = n_heads / cache->n_kv_heads;
    A.group_tiles = group_tiles_of(n_heads, cache->n_kv_heads);
    const int head_tiles = cache->n_kv_heads * A.group_tiles;
    A.chunk = chunk_of(n_seqs, head_tiles, max_len);
    A.n_splits = max_len <= A.chunk ? 1 : (int)(((size_t)max_len + A.chunk - 1) / A.chunk);
    const size_t parts = (size_t)n_seqs * A.n_splits * n_heads;
    if (A.n_splits > 1) {
        const size_t need = parts * ((size_t)cache->head_dim + 2) * sizeof(float);
        TL_REQUIRE(workspace && workspace_bytes >= need, "%s: needs a workspace of %zu bytes, got %zu", what, need, workspace ? workspace_bytes : (size_t)0);
        TL_REQUIRE(aligned16(workspace), "%s: the workspace must be 16-byte aligned", what);
    }
    const double blocks = (double)n_seqs * A.n_splits * head_tiles;
    if (blocks >= 2147483648.0 || n_seqs > 65535) return set_error(TL_ELIMIT, "%s: %d sequences of up to %d positions are too many for one call", what, n_seqs, max_len);
    TL_ENSURE_INIT();
    A.out = static_cast<half_t*>(out);
    A.q = static_cast<const half_t*>(q);
    A.q_stride = q_stride;
    A.cache = *cache;
    A.tables = tables;
    A.table_stride = table_stride;
    A.lens = lens;
    A.part_ml = static_cast<float2*>(workspace);
    A.part_o = static_cast<float*>(workspace) + 2 * parts;
    A.by_page = FastDiv((unsigned)cache->page_size);
    A.by_heads = FastDiv((unsigned)head_tiles);
    A.by_splits = FastDiv((unsigned)A.n_splits);
    A.n_heads = n_heads;
    A.max_len = max_len;
    A.scale_log2 = scale * kLog2e;
    if (cache->head_dim <= 64) launch_paged_attention<64>(A, (unsigned)blocks);
    else if (cache->head_dim <= 128) launch_paged_attention<128>(A, (unsigned)blocks);
    else launch_paged_attention<256>(A, (unsigned)blocks);
    TL_CHECK_LAUNCH("paged_attention_kernel");
    if (A.n_splits > 1) {
        paged_attention_join_kernel<<<dim3(n_heads, n_seqs), cache->head_dim <= 64 ? 64 : cache->head_dim <= 128 ? 128 : 256, 0, stream()>>>(A);
        TL_CHECK_LAUNCH("paged_attention_join_kernel");
    }
    return TL_OK;
}

}  // extern "C"
