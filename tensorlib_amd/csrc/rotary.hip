// Rotary positions for batches of tokens: any part of the head, pairs interleaved or half a rotated part apart,
// frequencies given per pair, positions from a device array; alone, or fused with the write of keys and values to the
// pages of a cache.
//
// A pair (a, b) at position p becomes m (a cos t - b sin t), m (a sin t + b cos t) with t = p f_i.  The angle is formed
// and reduced to half a turn in fp64: at p = 10^5 an fp32 product would be off by 2^-24 p = 0.006 rad.  Sine, cosine
// and the rotation itself are fp32, rounded to half once.
//
// Bound by memory: every value is read and written once (4 bytes), the positions, frequencies and tables come from L2.
// 16001 prompt tokens of 32 query and 8 kv heads of 128 take 70 us, 5.6 TB/s; a single token 3.4 us, a launch.
#include <cmath>

#include "paged.h"

namespace tl {

struct RotaryArgs {
    half_t* q_out;
    const half_t* q;
    const half_t* k;
    const half_t* v;
    size_t q_out_stride, q_stride, k_stride, v_stride;
    const int* positions;
    const int* seq_ids;
    const double* freq;
    const int* tables;
    size_t table_stride;
    tl_kv_pages cache;
    FastDiv by_units, by_groups, by_page;
    int n_seqs, n_heads, n_kv, head_dim, rotary_dim;
    float magnitude;
    unsigned total;
};

// cos and sin of position * radians_per_position, times the magnitude.
__device__ __forceinline__ void turn(int position, double radians_per_position, float magnitude, float& c, float& s) {
    double t = (double)position * (radians_per_position * 0.15915494309189533577);   // turns
    t -= rint(t);
    sincospif(2.0f * (float)t, &s, &c);
    c *= magnitude;
    s *= magnitude;
}

// Where the head rows of one token come from and go to: rows [0, n_heads) are query heads, the next n_kv keys, the last
// n_kv values.  dst is null where nothing is stored (a token without a page).
struct Row {
    const half_t* src;
    half_t* dst;
    bool rotated;
};
__device__ __forceinline__ Row row_of(const RotaryArgs& A, size_t token, int row, long slot) {
    if (row < A.n_heads) return {A.q + token * A.q_stride + (size_t)row * A.head_dim, A.q_out + token * A.q_out_stride + (size_t)row * A.head_dim, true};
    row -= A.n_heads;
    const bool key = row < A.n_kv;
    if (!key) row -= A.n_kv;
    const half_t* src = (key ? A.k + token * A.k_stride : A.v + token * A.v_stride) + (size_t)row * A.head_dim;
    half_t* base = static_cast<half_t*>(key ? A.cache.k : A.cache.v);
    return {src, slot < 0 ? nullptr : base + slot + (size_t)row * A.cache.head_stride, key};
}
// Element offset of a token's cache row (head 0), -1 if it has none: a sequence, position or page out of range.
__device__ __forceinline__ long slot_of(const RotaryArgs& A, size_t token, int position) {
    if (A.n_kv == 0) return -1;
    const size_t seq = A.seq_ids ? (size_t)(long)A.seq_ids[token] : token;
    if (seq >= (size_t)A.n_seqs || position < 0) return -1;      // a negative id is a huge unsigned one
    unsigned row;
    const unsigned at = A.by_page.divmod((unsigned)position, row);
    if (at >= A.table_stride) return -1;
    const int page = A.tables[seq * A.table_stride + at];
    if (page < 0 || page >= A.cache.n_pages) return -1;
    return (long)((size_t)page * A.cache.page_stride + (size_t)row * A.cache.row_stride);
}

// One thread: one unit of `ROWS` head rows of a token.  A unit is two pieces of VEC elements that pair up (HALF, rotary_dim a
// multiple of 2 VEC), or one of VEC / 2 adjacent pairs (rotary_dim a multiple of VEC); behind the rotated part, one piece
// that is copied.  The rows of a thread share their angles, and their loads are in flight together.
template <bool HALF, int VEC, int ROWS, bool STREAM_IN, bool STREAM_OUT>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs A) {
    typedef _Float16 piece __attribute__((ext_vector_type(VEC)));
    const unsigned id = blockIdx.x * 256u + threadIdx.x;
    if (id >= A.total) return;
    unsigned unit, group;
    const unsigned token = A.by_groups.divmod(A.by_units.divmod(id, unit), group);
    const int position = A.positions[token];
    const int pairing = HALF ? A.rotary_dim / (2 * VEC) : A.rotary_dim / VEC;     // units of the rotated part
    const bool turned = (int)unit < pairing;
    const int at = turned || !HALF ? (int)unit * VEC : (int)unit * VEC + A.rotary_dim / 2;
    const int other = at + A.rotary_dim / 2;
    const int n_rows = A.n_heads + 2 * A.n_kv;
    const long slot = (int)(group * ROWS + ROWS) > A.n_heads ? slot_of(A, token, position) : -1;

    auto load = [](const half_t* p) {
        const piece* v = reinterpret_cast<const piece*>(p);
        return STREAM_IN ? __builtin_nontemporal_load(v) : *v;
    };
    auto store = [](half_t* p, piece x) {
        piece* v = reinterpret_cast<piece*>(p);
        if (STREAM_OUT) __builtin_nontemporal_store(x, v);
        else *v = x;
    };
    Row r[ROWS];
    piece a[ROWS], b[ROWS];
    bool any = false;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        const int row = (int)group * ROWS + j;
        r[j] = row < n_rows ? row_of(A, token, row, slot) : Row{nullptr, nullptr, false};
        any |= r[j].rotated;
        if (r[j].dst) {
            a[j] = load(r[j].src + at);
            if (HALF && turned) b[j] = load(r[j].src + other);
        }
    }
    constexpr int ANGLES = HALF ? VEC : VEC / 2;
    float c[ANGLES], s[ANGLES];
    if (turned && any) {
#pragma unroll
        for (int i = 0; i < ANGLES; ++i) turn(position, A.freq[HALF ? at + i : at / 2 + i], A.magnitude, c[i], s[i]);
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        if (!r[j].dst) continue;
        if (turned && r[j].rotated) {
            if constexpr (HALF) {
#pragma unroll
                for (int i = 0; i < ANGLES; ++i) {
                    const float x = (float)a[j][i], y = (float)b[j][i];
                    a[j][i] = (half_t)(x * c[i] - y * s[i]);
                    b[j][i] = (half_t)(x * s[i] + y * c[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < ANGLES; ++i) {
                    const float x = (float)a[j][2 * i], y = (float)a[j][2 * i + 1];
                    a[j][2 * i] = (half_t)(x * c[i] - y * s[i]);
                    a[j][2 * i + 1] = (half_t)(x * s[i] + y * c[i]);
                }
            }
        }
        store(r[j].dst + at, a[j]);
        if (HALF && turned) store(r[j].dst + other, b[j]);
    }
}

// Any even rotary_dim, any alignment: one thread per pair, behind the rotated part per two neighbours.
__global__ void __launch_bounds__(256) rotary_pairs_kernel(RotaryArgs A, int interleaved) {
    const unsigned id = blockIdx.x * 256u + threadIdx.x;
    if (id >= A.total) return;
    unsigned unit, row;
    const unsigned token = A.by_groups.divmod(A.by_units.divmod(id, unit), row);
    const int position = A.positions[token];
    const Row r = row_of(A, token, (int)row, (int)row >= A.n_heads ? slot_of(A, token, position) : -1);
    if (!r.dst) return;
    const int half_rd = A.rotary_dim / 2;
    const bool turned = (int)unit < half_rd;
    int i0 = 2 * (int)unit, i1 = i0 + 1;
    if (turned && !interleaved) { i0 = (int)unit; i1 = i0 + half_rd; }
    if (i1 >= A.head_dim) {                      // an odd head_dim's last element
        if (r.dst + i0 != r.src + i0) r.dst[i0] = r.src[i0];
        return;
    }
    float x = (float)r.src[i0], y = (float)r.src[i1];
    if (turned && r.rotated) {
        float c, s;
        turn(position, A.freq[unit], A.magnitude, c, s);
        const float x1 = x * c - y * s;
        y = x * s + y * c;
        x = x1;
    }
    r.dst[i0] = (half_t)x;
    r.dst[i1] = (half_t)y;
}

static uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// From this many values on two rows per thread, and stores past the caches (1024 tokens of 32 + 8 + 8 heads of 128: 7.1 us, 9.2 the
// other way; 16000 of 8 + 8 + 8 of 96: 31 against 41); below, one row and plain accesses (64 tokens 3.6 against 4.2 us).
constexpr double kManyValues = 4194304.0;
// From this many on what is read and written exceeds the last-level cache.  Loads go past it too if a request's pieces make
// whole lines (16001 tokens of 32 + 8 + 8 heads of 128: 69 us, 72 with plain loads).  Where a head is two halves that pair up and
// not whole half lines, plain stores are better (40000 of 8 + 8 + 8 of 96: 84 against 98 us), at an odd number of pieces always (16000 of
// 8 + 8 + 8 of 80: 36 against 45).
constexpr double kPastCache = 67108864.0;

template <bool HALF, int VEC>
static void launch_rotary_pieces(const RotaryArgs& A, unsigned blocks, bool many, bool in, bool out) {
    if (!many) rotary_kernel<HALF, VEC, 1, false, false><<<blocks, 256, 0, stream()>>>(A);
    else if (VEC == 8 && in) rotary_kernel<HALF, VEC, 2, VEC == 8, true><<<blocks, 256, 0, stream()>>>(A);
    else if (HALF && VEC == 8 && !out) rotary_kernel<HALF, VEC, 2, false, !(HALF && VEC == 8)><<<blocks, 256, 0, stream()>>>(A);
    else rotary_kernel<HALF, VEC, 2, false, true><<<blocks, 256, 0, stream()>>>(A);
}

// alignment: all addresses and row strides in bytes, or-ed: a power of two that divides it divides them all.
static int launch_rotary(RotaryArgs& A, int n_tokens, int layout, uintptr_t alignment, const char* what) {
    const bool half = layout == TL_ROTARY_HALF;
    const long n_rows = A.n_heads + 2L * A.n_kv;
    int vec = 8;                          // the widest pieces that fit
    while (vec > 1 && (alignment % (2u * vec) || A.head_dim % vec || A.rotary_dim % (half ? 2 * vec : vec))) vec /= 2;
    const int units = vec == 1 ? (int)((A.head_dim + 1L) / 2) : half ? (A.head_dim - A.rotary_dim / 2) / vec : A.head_dim / vec;
    const double values = (double)n_tokens * n_rows * A.head_dim;
    const bool many = vec > 1 && values >= kManyValues, past = values >= kPastCache;
    const int run = half ? A.rotary_dim / 2 : A.head_dim;      // elements next to each other in one request
    const bool in = past && run % 64 == 0 && A.head_dim % 64 == 0, out = !half || A.rotary_dim < A.head_dim || run % (past ? 32 : 16) == 0;
    const long groups = many ? (n_rows + 1) / 2 : n_rows;
    const double total = (double)n_tokens * groups * units;
    if (total >= 2147483648.0 || n_rows > 0x7fffffff)
        return set_error(TL_ELIMIT, "%s: %d tokens of %ld heads of %d are too many for one call", what, n_tokens, n_rows, A.head_dim);
    TL_ENSURE_INIT();
    A.total = (unsigned)total;
    A.by_units = FastDiv((unsigned)units);
    A.by_groups = FastDiv((unsigned)groups);
    const unsigned blocks = (A.total + 255u) / 256u;
    if (vec == 1) rotary_pairs_kernel<<<blocks, 256, 0, stream()>>>(A, half ? 0 : 1);
    else if (half) (vec == 8 ? launch_rotary_pieces<true, 8> : vec == 4 ? launch_rotary_pieces<true, 4> : launch_rotary_pieces<true, 2>)(A, blocks, many, in, out);
    else (vec == 8 ? launch_rotary_pieces<false, 8> : vec == 4 ? launch_rotary_pieces<false, 4> : launch_rotary_pieces<false, 2>)(A, blocks, many, in, out);
    TL_CHECK_LAUNCH("rotary_kernel");
    return TL_OK;
}

static int check_rotary(const char* what, const int* positions, const double* freq, int rotary_dim, int layout, float magnitude, int n_tokens,
                        int n_heads, int head_dim) {
    TL_REQUIRE(n_tokens >= 0 && n_heads >= 0, "%s: negative size", what);
    TL_REQUIRE(head_dim >= 1 && rotary_dim >= 0 && rotary_dim <= head_dim && rotary_dim % 2 == 0,
               "%s: rotary_dim %d must be even and at most head_dim %d", what, rotary_dim, head_dim);
    TL_REQUIRE(layout == TL_ROTARY_INTERLEAVED || layout == TL_ROTARY_HALF, "%s: unknown layout %d", what, layout);
    TL_REQUIRE(std::isfinite(magnitude), "%s: magnitude must be finite", what);
    TL_REQUIRE(n_tokens == 0 || (positions && (freq || rotary_dim == 0)), "%s: null pointer", what);
    return TL_OK;
}

}  // namespace tl

extern "C" {

int tl_rotary_frequencies(double* host_out, int rotary_dim, double base, int scaling, double factor, double original_context,
                          double slow_turns, double fast_turns) {
    TL_REQUIRE(host_out != nullptr, "tl_rotary_frequencies: null pointer");
    TL_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0, "tl_rotary_frequencies: rotary_dim %d must be even and positive", rotary_dim);
    TL_REQUIRE(std::isfinite(base) && base > 0.0, "tl_rotary_frequencies: base must be positive");
    TL_REQUIRE(scaling >= TL_ROTARY_SCALE_NONE && scaling <= TL_ROTARY_SCALE_PARTS, "tl_rotary_frequencies: unknown scaling %d", scaling);
    TL_REQUIRE(scaling == TL_ROTARY_SCALE_NONE || (std::isfinite(factor) && factor > 0.0), "tl_rotary_frequencies: factor must be positive");
    if (scaling == TL_ROTARY_SCALE_PARTS)
        TL_REQUIRE(std::isfinite(original_context) && original_context > 0.0 && std::isfinite(slow_turns) && std::isfinite(fast_turns) && fast_turns > slow_turns,
                   "tl_rotary_frequencies: needs original_context > 0 and fast_turns > slow_turns");
    if (scaling == TL_ROTARY_SCALE_BASE) {
        TL_REQUIRE(rotary_dim > 2, "tl_rotary_frequencies: a change of base needs rotary_dim > 2");
        base *= std::pow(factor, (double)rotary_dim / (rotary_dim - 2));
    }
    for (int i = 0; i < rotary_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rotary_dim);
        if (scaling == TL_ROTARY_SCALE_LINEAR) f /= factor;
        if (scaling == TL_ROTARY_SCALE_PARTS) {
            const double turns = original_context * f / 6.283185307179586476925;
            double keep = (turns - slow_turns) / (fast_turns - slow_turns);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
            f = f * keep + f / factor * (1.0 - keep);
        }
        host_out[i] = f;
    }
    return TL_OK;
}

int tl_rotary_f16(void* out, size_t out_stride, const void* in, size_t in_stride, const int* positions, const double* freq, int rotary_dim,
                  int layout, float magnitude, int n_tokens, int n_heads, int head_dim) {
    using namespace tl;
    int rc = check_rotary("tl_rotary_f16", positions, freq, rotary_dim, layout, magnitude, n_tokens, n_heads, head_dim);
    if (rc != TL_OK) return rc;
    if (n_tokens == 0 || n_heads == 0) return TL_OK;
    TL_REQUIRE(out && in, "tl_rotary_f16: null pointer");
    const size_t width = (size_t)n_heads * head_dim;
    TL_REQUIRE(n_tokens == 1 || (in_stride >= width && out_stride >= width), "tl_rotary_f16: row strides must cover the heads");
    TL_REQUIRE(out != in || out_stride == in_stride || n_tokens == 1, "tl_rotary_f16: in place needs equal strides");
    RotaryArgs A{};
    A.q_out = static_cast<half_t*>(out);
    A.q = static_cast<const half_t*>(in);
    A.q_out_stride = out_stride;
    A.q_stride = in_stride;
    A.positions = positions;
    A.freq = freq;
    A.by_page = FastDiv(1);
    A.n_heads = n_heads;
    A.head_dim = head_dim;
    A.rotary_dim = rotary_dim;
    A.magnitude = magnitude;
    const uintptr_t strides = n_tokens == 1 ? 0 : 2 * (in_stride | out_stride);
    return launch_rotary(A, n_tokens, layout, address(out) | address(in) | strides, "tl_rotary_f16");
}

int tl_rotary_kv_pages_f16(void* q_out, const void* q, size_t q_stride, const void* k, size_t k_stride, const void* v, size_t v_stride,
                           const int* positions, const int* seq_ids, const double* freq, int rotary_dim, int layout, float magnitude,
                           int n_tokens, int n_heads, const tl_kv_pages* cache, const int* tables, size_t table_stride, int n_seqs) {
    using namespace tl;
    const char* what = "tl_rotary_kv_pages_f16";
    int rc = check_kv_pages(cache, what);
    if (rc != TL_OK) return rc;
    rc = check_rotary(what, positions, freq, rotary_dim, layout, magnitude, n_tokens, n_heads, cache->head_dim);
    if (rc != TL_OK) return rc;
    if (n_tokens == 0) return TL_OK;
    TL_REQUIRE(n_seqs >= 0, "%s: negative size", what);
    TL_REQUIRE(k && v && (tables || n_seqs == 0 || table_stride == 0), "%s: null pointer", what);
    TL_REQUIRE(n_heads == 0 || (q && q_out), "%s: null pointer", what);
    const size_t D = (size_t)cache->head_dim;
    if (n_tokens > 1)
        TL_REQUIRE(q_stride >= n_heads * D && k_stride >= cache->n_kv_heads * D && v_stride >= cache->n_kv_heads * D,
                   "%s: row strides must cover the heads", what);
    RotaryArgs A{};
    A.q_out = static_cast<half_t*>(q_out);
    A.q = static_cast<const half_t*>(q);
    A.k = static_cast<const half_t*>(k);
    A.v = static_cast<const half_t*>(v);
    A.q_out_stride = n_heads * D;
    A.q_stride = q_stride;
    A.k_stride = k_stride;
    A.v_stride = v_stride;
    A.positions = positions;
    A.seq_ids = seq_ids;
    A.freq = freq;
    A.tables = tables;
    A.table_stride = table_stride;
    A.cache = *cache;
    A.by_page = FastDiv((unsigned)cache->page_size);
    A.n_seqs = n_seqs;
    A.n_heads = n_heads;
    A.n_kv = cache->n_kv_heads;
    A.head_dim = cache->head_dim;
    A.rotary_dim = rotary_dim;
    A.magnitude = magnitude;
    const uintptr_t strides = n_tokens == 1 ? 0 : 2 * (q_stride | k_stride | v_stride);
    return launch_rotary(A, n_tokens, layout, address(q_out) | address(q) | address(k) | address(v) | strides, what);
}

}  // extern "C"
