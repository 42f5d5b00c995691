// Bookkeeping and copies of the pages of a key-value cache.
//
// State, all int32 on the device: tables [n_seqs, table_stride] (a sequence's pages in order, -1 behind them),
// lens [n_seqs] (cached positions), refs [n_pages] (how many table entries name a page; 0 = free).  A page is shared
// only while it is full: a fork gives every further child its own copy of a partly filled last page, so a sequence may
// always write behind its last position.  New pages are the lowest free ids, handed out in row order, so results do not
// depend on scheduling.  Reference counts change by integer atomics, whose order cannot matter.
//
// What these cost is launches and latency; only the page copies move data worth a bound (2 x bytes at copy rate).
#include "paged.h"

namespace tl {

constexpr int kThreads = 1024;
constexpr int kMaxSeqs = 8192;             // the rows' prefix sums sit in LDS

__device__ __forceinline__ int pages_of(int len, int page_size, int table_stride) {
    if (len <= 0) return 0;
    const int p = (len - 1) / page_size + 1;
    return p < table_stride ? p : table_stride;
}

// Exclusive prefix sums of one value per thread over a workgroup of 1024; *total receives the sum.
__device__ __forceinline__ int block_scan(int v, int* total) {
    __shared__ int s_wave[kThreads / 64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    int x = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    __syncthreads();                       // the previous call's sums have been read
    if (lane == 63) s_wave[wave] = x;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        const int s = s_wave[w];
        if (w < wave) before += s;
        all += s;
    }
    *total = all;
    return before + x - v;
}

// The number of free pages, counted up to `enough` at least if there are as many (one workgroup).
__device__ int count_free(const int* refs, int n_pages, int enough) {
    int found = 0;
    for (int p0 = 0; p0 < n_pages && found < enough; p0 += 4 * kThreads) {
        int mine = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int p = p0 + (int)threadIdx.x * 4 + j;
            if (p < n_pages && refs[p] == 0) ++mine;
        }
        int total;
        block_scan(mine, &total);
        found += total;
    }
    return found;
}

// Calls take(k, page) for the `wanted` lowest free pages, k counting from 0 in page order (one workgroup).
template <class F>
__device__ void take_free(int* refs, int n_pages, int wanted, F take) {
    int found = 0;
    for (int p0 = 0; p0 < n_pages && found < wanted; p0 += 4 * kThreads) {
        const int p = p0 + (int)threadIdx.x * 4;
        bool free_[4];
        int mine = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            free_[j] = p + j < n_pages && refs[p + j] == 0;
            mine += free_[j];
        }
        int total;
        int k = found + block_scan(mine, &total);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!free_[j]) continue;
            if (k < wanted) {
                refs[p + j] = 1;
                take(k, p + j);
            }
            ++k;
        }
        found += total;
    }
}

// ---- states that fit one workgroup: the whole operation in one launch, the reference counts in registers or LDS ----

constexpr int kPer = 16;                   // pages per thread
constexpr int kSmallPages = kPer * kThreads;
constexpr int kSmallSeqs = kThreads;       // a thread per row
constexpr size_t kSmallEntries = 65536;    // table entries

// The thread's pages [per tid, per tid + per), per = n_pages / 1024 rounded up; pages past the end count as taken.
struct MyPages {
    int ref[kPer], per;
    __device__ __forceinline__ int page(int j) const { return (int)threadIdx.x * per + j; }
    __device__ __forceinline__ void load(const int* refs, int n_pages) {
        per = (n_pages + kThreads - 1) / kThreads;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            ref[j] = 1;
            if (j < per && page(j) < n_pages) ref[j] = refs[page(j)];
        }
    }
    // How many of the thread's pages fulfil a condition on (page, count).
    template <class F>
    __device__ __forceinline__ int count(F f) const {
        int n = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (j < per) n += f(page(j), ref[j]);
        return n;
    }
    __device__ __forceinline__ int free_count() const {
        return count([](int, int r) { return r == 0; });
    }
    // Gives away those of the thread's free pages whose rank in page order, from `rank` on, is below `wanted`.
    template <class F>
    __device__ __forceinline__ void take(int rank, int wanted, F give) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (j < per && ref[j] == 0) {
                if (rank < wanted) give(rank, page(j));
                ++rank;
            }
        }
    }
};

struct ForkArgs {
    const int *tables, *lens, *refs, *parents;
    int *tables_out, *lens_out, *refs_out, *copy_src, *copy_dst, *missing;
    int n_seqs, table_stride, n_pages, page_size;
    FastDiv by_vectors;                    // table entries of a row, in steps of VEC
};

// VEC: table entries a thread moves at a time, 4 where rows are 16-byte aligned.
template <int VEC>
__global__ void __launch_bounds__(kThreads) pages_fork_small_kernel(ForkArgs A) {
    __shared__ int s_len[kSmallSeqs], s_pages[kSmallSeqs], s_parent[kSmallSeqs], s_first[kSmallSeqs], s_page[kSmallSeqs];
    extern __shared__ int s_refs[];
    const int r = threadIdx.x;
    const bool row = r < A.n_seqs;
    const int parent = row ? A.parents[r] : -1;
    const int old_len = row ? A.lens[r] : 0;
    for (int p = r; p < A.n_pages; p += kThreads) s_refs[p] = A.refs[p];
    s_first[r] = kSmallSeqs;
    s_len[r] = old_len > 0 ? old_len : 0;
    s_pages[r] = pages_of(old_len, A.page_size, A.table_stride);     // once: the divisions would be half of the loop below
    s_parent[r] = parent >= 0 && parent < A.n_seqs ? parent : -1;
    __syncthreads();
    const bool has = s_parent[r] >= 0;
    const int len = has ? s_len[parent] : 0;
    const int new_pages = has ? s_pages[parent] : 0;
    const bool partial = len % A.page_size != 0;
    int last = -1;                         // the page to be copied, if the row is not its parent's first
    if (partial) {
        last = A.tables[(size_t)parent * A.table_stride + new_pages - 1];
        atomicMin(s_first + parent, r);
    }
    __syncthreads();
    const bool copied = partial && s_first[parent] != r;
    if (copied) s_page[r] = -2;            // not counted and not written below
    else s_page[r] = -1;
    __syncthreads();
    const unsigned total = (unsigned)A.n_seqs * A.by_vectors.d;
    for (unsigned i = r; i < total; i += kThreads) {
        unsigned c;
        const unsigned to = A.by_vectors.divmod(i, c);
        c *= VEC;
        const int from = s_parent[to];
        const int old_pages = s_pages[to];
        const int pages = from >= 0 ? s_pages[from] : 0;
        const int kept = s_page[to] == -2 ? pages - 1 : pages;
        int o[VEC], x[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            o[j] = -1;
            x[j] = -1;
        }
        const int* old_row = A.tables + (size_t)to * A.table_stride + c;
        const int* new_row = A.tables + (size_t)(from >= 0 ? from : 0) * A.table_stride + c;
        if constexpr (VEC == 4) {
            if ((int)c < old_pages) *reinterpret_cast<int4*>(o) = *reinterpret_cast<const int4*>(old_row);
            if ((int)c < pages) *reinterpret_cast<int4*>(x) = *reinterpret_cast<const int4*>(new_row);
        } else {
            if ((int)c < old_pages) o[0] = *old_row;
            if ((int)c < pages) x[0] = *new_row;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if ((int)c + j < old_pages && o[j] >= 0 && o[j] < A.n_pages) atomicSub(s_refs + o[j], 1);
            if ((int)c + j >= pages) x[j] = -1;
            if ((int)c + j < kept && x[j] >= 0 && x[j] < A.n_pages) atomicAdd(s_refs + x[j], 1);
        }
        int* out = A.tables_out + (size_t)to * A.table_stride + c;
        if constexpr (VEC == 4) *reinterpret_cast<int4*>(out) = *reinterpret_cast<int4*>(x);
        else *out = x[0];
    }
    __syncthreads();
    const bool wants = copied && last >= 0 && last < A.n_pages;
    int wanted, available;
    const int rank = block_scan(wants, &wanted);
    MyPages mine;
    mine.load(s_refs, A.n_pages);
    const int before = block_scan(mine.free_count(), &available);
    const bool enough = available >= wanted;
    if (enough) mine.take(before, wanted, [&](int k, int page) {
        s_page[k] = page;
        s_refs[page] = 1;
    });
    __syncthreads();
    if (r == 0) *A.missing = enough ? 0 : wanted - available;
    if (row) {
        const int page = wants && enough ? s_page[rank] : -1;
        if (page >= 0) A.tables_out[(size_t)r * A.table_stride + new_pages - 1] = page;
        A.copy_src[r] = page >= 0 ? last : -1;
        A.copy_dst[r] = page;
        A.lens_out[r] = enough ? len : old_len;
    }
    for (int p = r; p < A.n_pages; p += kThreads) A.refs_out[p] = enough ? s_refs[p] : A.refs[p];
    if (!enough)
        for (size_t i = r; i < (size_t)A.n_seqs * A.table_stride; i += kThreads) A.tables_out[i] = A.tables[i];
}

__global__ void __launch_bounds__(kThreads)
pages_extend_small_kernel(int* tables, int* lens, int* refs, const int* add, int* missing, int n_seqs, int table_stride, int n_pages, int page_size) {
    __shared__ int s_first[kSmallSeqs];   // number of pages wanted by the rows before
    const int r = threadIdx.x;
    const int len = r < n_seqs ? max(lens[r], 0) : 0;
    const long more = r < n_seqs ? max(add[r], 0) : 0;
    MyPages mine;
    mine.load(refs, n_pages);
    const long pages = (len + more + page_size - 1) / page_size;
    const bool fits = pages <= table_stride && len + more <= 0x7fffffffl;
    const int held = pages_of(len, page_size, table_stride);
    int wanted, available;
    s_first[r] = block_scan(fits ? (int)pages - held : 0, &wanted);
    const int before = block_scan(mine.free_count(), &available);
    const bool refused = __syncthreads_or(!fits);
    if (r == 0) *missing = refused ? -1 : available < wanted ? wanted - available : 0;
    if (refused || available < wanted) return;
    mine.take(before, wanted, [&](int k, int page) {
        int lo = 0, hi = n_seqs - 1;      // the last row whose first page is at most k
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (s_first[mid] <= k) lo = mid;
            else hi = mid - 1;
        }
        refs[page] = 1;
        tables[(size_t)lo * table_stride + pages_of(lens[lo], page_size, table_stride) + k - s_first[lo]] = page;
    });
    __syncthreads();                       // every length has been read
    if (r < n_seqs) lens[r] = len + (int)more;
}

// Plan and remap of a small pool.  s_new: a page's new id; the k-th mover and the k-th hole meet in the two lists.
__global__ void __launch_bounds__(kThreads)
pages_compact_small_kernel(const int* tables, const int* refs, int* tables_out, int* refs_out, int* remap, int* copy_src, int* copy_dst, int* count,
                           int n_pages, int n_entries) {
    __shared__ unsigned short s_mover[kSmallPages / 2], s_hole[kSmallPages / 2];
    extern __shared__ int s_new[];
    const int tid = threadIdx.x;
    MyPages mine;
    mine.load(refs, n_pages);
    int live, total, holes;
    block_scan(mine.count([&](int p, int ref) { return p < n_pages && ref > 0; }), &live);
    int m = block_scan(mine.count([&](int p, int ref) { return p < n_pages && p >= live && ref > 0; }), &total);
    int h = block_scan(mine.count([&](int p, int ref) { return p < live && ref <= 0; }), &holes);
    const int movers = total;              // as many as holes, at most half of the pages
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int p = mine.page(j);
        if (j < mine.per && p < n_pages) {
            if (p >= live && mine.ref[j] > 0) s_mover[m++] = (unsigned short)p;
            if (p < live && mine.ref[j] <= 0) s_hole[h++] = (unsigned short)p;
            s_new[p] = mine.ref[j] > 0 ? p : -1;
        }
    }
    __syncthreads();
    for (int k = tid; k < movers; k += kThreads) s_new[s_mover[k]] = s_hole[k];
    __syncthreads();
    for (int k = tid; k < n_pages; k += kThreads) {
        copy_src[k] = k < movers ? s_mover[k] : -1;
        copy_dst[k] = k < movers ? s_hole[k] : -1;
        const int to = s_new[k], ref = refs[k];
        remap[k] = to;
        if (k >= live) refs_out[k] = 0;
        if (to >= 0) refs_out[to] = ref;   // below the line: itself, or the hole that it fills
    }
    if (tid == 0) *count = movers;
    for (int i = tid; i < n_entries; i += kThreads) {
        const int p = tables[i];
        tables_out[i] = p >= 0 && p < n_pages ? s_new[p] : p;
    }
}

// ---- any size ----

__global__ void __launch_bounds__(256) pages_copy_ints_kernel(int* out, const int* in, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) out[i] = in[i];
}

// One workgroup per row: releases the row's old pages, takes its parent's, and notes the page to be copied for a child
// after the first of a parent with a partly filled page.
__global__ void __launch_bounds__(256) pages_fork_rows_kernel(ForkArgs A) {
    const int row = blockIdx.x;
    const int parent = A.parents[row];
    const bool has = parent >= 0 && parent < A.n_seqs;
    const int old_pages = pages_of(A.lens[row], A.page_size, A.table_stride);
    const int len = has ? max(A.lens[parent], 0) : 0;
    const int new_pages = pages_of(len, A.page_size, A.table_stride);
    int earlier = 0;
    if (has && len % A.page_size != 0)
        for (int i = threadIdx.x; i < row; i += 256) earlier |= A.parents[i] == parent;
    const bool copied = __syncthreads_or(earlier) != 0;
    const size_t stride = (size_t)A.table_stride;
    const int* old_row = A.tables + row * stride;
    const int* from = A.tables + (has ? parent : 0) * stride;
    int* to = A.tables_out + row * stride;
    for (int c = threadIdx.x; c < A.table_stride; c += 256) {
        if (c < old_pages) {
            const int p = old_row[c];
            if (p >= 0 && p < A.n_pages) atomicSub(A.refs_out + p, 1);
        }
        int p = -1;
        if (c < new_pages) {
            p = from[c];
            if (p >= 0 && p < A.n_pages && !(copied && c == new_pages - 1)) atomicAdd(A.refs_out + p, 1);
        }
        to[c] = p;
    }
    if (threadIdx.x == 0) {
        const int last = new_pages > 0 ? from[new_pages - 1] : -1;
        A.copy_src[row] = copied && last >= 0 && last < A.n_pages ? last : -1;
        A.copy_dst[row] = -1;
        A.lens_out[row] = len;
    }
}

// One workgroup: hands the lowest free pages to the rows that copy one; without enough of them, everything is put back.
__global__ void __launch_bounds__(kThreads) pages_fork_take_kernel(ForkArgs A) {
    int wanted = 0;
    for (int r0 = 0; r0 < A.n_seqs; r0 += kThreads) {
        const int r = r0 + (int)threadIdx.x;
        int total;
        const int k = wanted + block_scan(r < A.n_seqs && A.copy_src[r] >= 0, &total);
        if (r < A.n_seqs && A.copy_src[r] >= 0) A.copy_dst[k] = r;      // the k-th row that wants a page, for a moment
        wanted += total;
    }
    const int available = wanted ? count_free(A.refs_out, A.n_pages, wanted) : 0;
    if (threadIdx.x == 0) *A.missing = available < wanted ? wanted - available : 0;
    __syncthreads();
    if (available < wanted) {
        for (int i = threadIdx.x; i < A.n_pages; i += kThreads) A.refs_out[i] = A.refs[i];
        for (size_t i = threadIdx.x; i < (size_t)A.n_seqs * A.table_stride; i += kThreads) A.tables_out[i] = A.tables[i];
        for (int i = threadIdx.x; i < A.n_seqs; i += kThreads) {
            A.lens_out[i] = A.lens[i];
            A.copy_src[i] = A.copy_dst[i] = -1;
        }
        return;
    }
    if (wanted == 0) return;
    // The list sits in copy_dst[0, wanted); the pages go to the rows' tables, and copy_dst is filled from there.
    take_free(A.refs_out, A.n_pages, wanted, [&](int k, int page) {
        const int row = A.copy_dst[k];
        A.tables_out[(size_t)row * A.table_stride + pages_of(A.lens_out[row], A.page_size, A.table_stride) - 1] = page;
    });
    __syncthreads();
    for (int r = threadIdx.x; r < A.n_seqs; r += kThreads)
        A.copy_dst[r] = A.copy_src[r] >= 0 ? A.tables_out[(size_t)r * A.table_stride + pages_of(A.lens_out[r], A.page_size, A.table_stride) - 1] : -1;
}

// Room for add[r] more positions of every sequence, all or nothing (one workgroup).
__global__ void __launch_bounds__(kThreads)
pages_extend_kernel(int* tables, int* lens, int* refs, const int* add, int* missing, int n_seqs, int table_stride, int n_pages, int page_size) {
    extern __shared__ int s_first[];      // number of pages wanted by the rows before
    int wanted = 0, refused = 0;
    for (int r0 = 0; r0 < n_seqs; r0 += kThreads) {
        const int r = r0 + (int)threadIdx.x;
        int need = 0;
        if (r < n_seqs) {
            const int len = max(lens[r], 0);
            const long more = max(add[r], 0);
            const long pages = (len + more + page_size - 1) / page_size;
            if (pages > table_stride || len + more > 0x7fffffffl) refused = 1;
            else need = (int)pages - pages_of(len, page_size, table_stride);
        }
        int total;
        const int k = wanted + block_scan(need, &total);
        if (r < n_seqs) s_first[r] = k;
        wanted += total;
    }
    refused = __syncthreads_or(refused);
    const int available = count_free(refs, n_pages, wanted);
    if (threadIdx.x == 0) *missing = refused ? -1 : available < wanted ? wanted - available : 0;
    if (refused || available < wanted) return;
    __syncthreads();
    take_free(refs, n_pages, wanted, [&](int k, int page) {
        int lo = 0, hi = n_seqs - 1;      // the last row whose first page is at most k
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (s_first[mid] <= k) lo = mid;
            else hi = mid - 1;
        }
        tables[(size_t)lo * table_stride + pages_of(lens[lo], page_size, table_stride) + k - s_first[lo]] = page;
    });
    __syncthreads();
    for (int r = threadIdx.x; r < n_seqs; r += kThreads) lens[r] = max(lens[r], 0) + max(add[r], 0);
}

__global__ void __launch_bounds__(256)
pages_free_kernel(int* tables, int* lens, int* refs, const uint8_t* rows, int table_stride, int n_pages, int page_size) {
    const int row = blockIdx.x;
    if (!rows[row]) return;
    const int used = pages_of(lens[row], page_size, table_stride);
    __syncthreads();
    int* t = tables + (size_t)row * table_stride;
    for (int c = threadIdx.x; c < table_stride; c += 256) {
        const int p = t[c];
        if (c < used && p >= 0 && p < n_pages) atomicSub(refs + p, 1);
        t[c] = -1;
    }
    if (threadIdx.x == 0) lens[row] = 0;
}

// One workgroup: the live pages above the number of live pages move into the free ones below it, in page order.
__global__ void __launch_bounds__(kThreads)
pages_compact_plan_kernel(const int* refs, int* refs_out, int* remap, int* copy_src, int* copy_dst, int* count, int n_pages) {
    int live = 0;
    for (int p0 = 0; p0 < n_pages; p0 += 4 * kThreads) {
        int mine = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int p = p0 + (int)threadIdx.x * 4 + j;
            mine += p < n_pages && refs[p] > 0;
        }
        int total;
        block_scan(mine, &total);
        live += total;
    }
    int movers = 0, holes = 0;
    for (int p0 = 0; p0 < n_pages; p0 += kThreads) {
        const int p = p0 + (int)threadIdx.x;
        const int ref = p < n_pages ? refs[p] : 0;
        const bool mover = ref > 0 && p >= live, hole = p < live && ref <= 0;
        int total;
        const int k = movers + block_scan(mover, &total);
        movers += total;
        const int h = holes + block_scan(hole, &total);
        holes += total;
        if (mover) copy_src[k] = p;
        if (hole) copy_dst[h] = p;
        if (p < n_pages) {
            remap[p] = ref > 0 ? p : -1;
            refs_out[p] = p < live ? ref : 0;
        }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < n_pages; k += kThreads) {
        if (k < movers) {
            remap[copy_src[k]] = copy_dst[k];
            refs_out[copy_dst[k]] = refs[copy_src[k]];
        } else {
            copy_src[k] = copy_dst[k] = -1;
        }
    }
    if (threadIdx.x == 0) *count = movers;
}

__global__ void __launch_bounds__(256) pages_remap_kernel(int* out, const int* in, const int* remap, int n_pages, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const int p = in[i];
        out[i] = p >= 0 && p < n_pages ? remap[p] : p;
    }
}

// Piece `i` of all pieces of all planes of all pairs: 256 threads x 4 x 16 bytes.  STREAM: accesses that do not settle in the
// caches, for calls that may move more than fits there.
constexpr unsigned kPiece = 256 * 4 * 16;
template <bool STREAM>
__global__ void __launch_bounds__(256)
pages_copy_kernel(unsigned char* pool, size_t plane_stride, size_t page_stride, size_t page_bytes, unsigned pieces, int n_planes, int n_pages,
                  const int* src, const int* dst, const int* count, int max_pairs) {
    int pairs = max_pairs;
    if (count) pairs = min(max(*count, 0), max_pairs);
    const size_t per_pair = (size_t)pieces * n_planes, total = per_pair * pairs;
    for (size_t i = blockIdx.x; i < total; i += gridDim.x) {
        const size_t pair = i / per_pair, rest = i % per_pair;
        const int from = src[pair], to = dst[pair];
        if (from < 0 || from >= n_pages || to < 0 || to >= n_pages) continue;
        const size_t plane = rest / pieces, at = (rest % pieces) * kPiece;
        const unsigned char* s = pool + plane * plane_stride + from * page_stride + at;
        unsigned char* d = pool + plane * plane_stride + to * page_stride + at;
        const size_t left = page_bytes - at;
        float4_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned o = (j * 256 + threadIdx.x) * 16;
            const float4_t* from4 = reinterpret_cast<const float4_t*>(s + o);
            if (o < left) x[j] = STREAM ? __builtin_nontemporal_load(from4) : *from4;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned o = (j * 256 + threadIdx.x) * 16;
            float4_t* to4 = reinterpret_cast<float4_t*>(d + o);
            if (o >= left) continue;
            if (STREAM) __builtin_nontemporal_store(x[j], to4);
            else *to4 = x[j];
        }
    }
}

static int check_state(const char* what, int n_seqs, int table_stride, int n_pages, int page_size) {
    TL_REQUIRE(n_seqs >= 0 && table_stride >= 1 && n_pages >= 1 && page_size >= 1, "%s: sizes out of range", what);
    if (n_seqs > kMaxSeqs) return set_error(TL_ELIMIT, "%s: %d sequences, at most %d", what, n_seqs, kMaxSeqs);
    if ((size_t)n_seqs * (size_t)table_stride >= (1u << 31)) return set_error(TL_ELIMIT, "%s: tables of %d x %d entries are too large", what, n_seqs, table_stride);
    return TL_OK;
}

static bool small_state(int n_seqs, int table_stride, int n_pages) {
    return n_seqs <= kSmallSeqs && n_pages <= kSmallPages && (size_t)n_seqs * (size_t)table_stride <= kSmallEntries;
}

static unsigned ints_grid(size_t n) {
    const size_t b = (n + 255) / 256;
    return (unsigned)(b < 2048 ? b : 2048);
}

}  // namespace tl

extern "C" {

int tl_pages_fork(const int* tables, const int* lens, const int* refs, const int* parents, int* tables_out, int* lens_out, int* refs_out,
                  int* copy_src, int* copy_dst, int* missing, int n_seqs, int table_stride, int n_pages, int page_size) {
    using namespace tl;
    const char* what = "tl_pages_fork";
    int rc = check_state(what, n_seqs, table_stride, n_pages, page_size);
    if (rc != TL_OK) return rc;
    TL_REQUIRE(refs && refs_out && missing, "%s: null pointer", what);
    TL_REQUIRE(n_seqs == 0 || (tables && lens && parents && tables_out && lens_out && copy_src && copy_dst), "%s: null pointer", what);
    TL_REQUIRE((n_seqs == 0 || (tables_out != tables && lens_out != lens)) && refs_out != refs, "%s: the new state must not lie over the old one", what);
    TL_ENSURE_INIT();
    ForkArgs A{tables, lens, refs, parents, tables_out, lens_out, refs_out, copy_src, copy_dst, missing, n_seqs, table_stride, n_pages, page_size, {}};
    if (small_state(n_seqs, table_stride, n_pages)) {
        const bool vec = table_stride % 4 == 0 && aligned16(tables) && aligned16(tables_out);
        A.by_vectors = FastDiv((unsigned)(vec ? table_stride / 4 : table_stride));
        if (vec) pages_fork_small_kernel<4><<<1, kThreads, n_pages * sizeof(int), stream()>>>(A);
        else pages_fork_small_kernel<1><<<1, kThreads, n_pages * sizeof(int), stream()>>>(A);
        TL_CHECK_LAUNCH("pages_fork_small_kernel");
        return TL_OK;
    }
    pages_copy_ints_kernel<<<ints_grid(n_pages), 256, 0, stream()>>>(refs_out, refs, n_pages);
    TL_CHECK_LAUNCH("pages_copy_ints_kernel");
    if (n_seqs > 0) {
        pages_fork_rows_kernel<<<n_seqs, 256, 0, stream()>>>(A);
        TL_CHECK_LAUNCH("pages_fork_rows_kernel");
    }
    pages_fork_take_kernel<<<1, kThreads, 0, stream()>>>(A);
    TL_CHECK_LAUNCH("pages_fork_take_kernel");
    return TL_OK;
}

int tl_pages_extend(int* tables, int* lens, int* refs, const int* add, int* missing, int n_seqs, int table_stride, int n_pages, int page_size) {
    using namespace tl;
    const char* what = "tl_pages_extend";
    int rc = check_state(what, n_seqs, table_stride, n_pages, page_size);
    if (rc != TL_OK) return rc;
    TL_REQUIRE(refs && missing && (n_seqs == 0 || (tables && lens && add)), "%s: null pointer", what);
    TL_ENSURE_INIT();
    if (small_state(n_seqs, 1, n_pages)) {
        pages_extend_small_kernel<<<1, kThreads, 0, stream()>>>(tables, lens, refs, add, missing, n_seqs, table_stride, n_pages, page_size);
        TL_CHECK_LAUNCH("pages_extend_small_kernel");
        return TL_OK;
    }
    pages_extend_kernel<<<1, kThreads, (size_t)n_seqs * sizeof(int), stream()>>>(tables, lens, refs, add, missing, n_seqs, table_stride, n_pages, page_size);
    TL_CHECK_LAUNCH("pages_extend_kernel");
    return TL_OK;
}

int tl_pages_free(int* tables, int* lens, int* refs, const uint8_t* rows, int n_seqs, int table_stride, int n_pages, int page_size) {
    using namespace tl;
    const char* what = "tl_pages_free";
    int rc = check_state(what, n_seqs, table_stride, n_pages, page_size);
    if (rc != TL_OK) return rc;
    if (n_seqs == 0) return TL_OK;
    TL_REQUIRE(tables && lens && refs && rows, "%s: null pointer", what);
    TL_ENSURE_INIT();
    pages_free_kernel<<<n_seqs, 256, 0, stream()>>>(tables, lens, refs, rows, table_stride, n_pages, page_size);
    TL_CHECK_LAUNCH("pages_free_kernel");
    return TL_OK;
}

int tl_pages_compact(const int* tables, const int* refs, int* tables_out, int* refs_out, int* remap, int* copy_src, int* copy_dst, int* count,
                     int n_seqs, int table_stride, int n_pages) {
    using namespace tl;
    const char* what = "tl_pages_compact";
    TL_REQUIRE(n_seqs >= 0 && table_stride >= 1 && n_pages >= 1, "%s: sizes out of range", what);
    TL_REQUIRE(refs && refs_out && remap && copy_src && copy_dst && count && (n_seqs == 0 || (tables && tables_out)), "%s: null pointer", what);
    TL_REQUIRE(refs_out != refs, "%s: the new reference counts must not lie over the old ones", what);
    TL_ENSURE_INIT();
    if (small_state(0, 1, n_pages) && (size_t)n_seqs * (size_t)table_stride <= kSmallEntries) {
        pages_compact_small_kernel<<<1, kThreads, n_pages * sizeof(int), stream()>>>(tables, refs, tables_out, refs_out, remap, copy_src, copy_dst, count,
                                                                                    n_pages, n_seqs * table_stride);
        TL_CHECK_LAUNCH("pages_compact_small_kernel");
        return TL_OK;
    }
    pages_compact_plan_kernel<<<1, kThreads, 0, stream()>>>(refs, refs_out, remap, copy_src, copy_dst, count, n_pages);
    TL_CHECK_LAUNCH("pages_compact_plan_kernel");
    const size_t n = (size_t)n_seqs * table_stride;
    if (n > 0) {
        pages_remap_kernel<<<ints_grid(n), 256, 0, stream()>>>(tables_out, tables, remap, n_pages, n);
        TL_CHECK_LAUNCH("pages_remap_kernel");
    }
    return TL_OK;
}

int tl_pages_copy(void* pool, size_t plane_stride, size_t page_stride, size_t page_bytes, int n_planes, int n_pages, const int* src, const int* dst,
                  const int* count, int max_pairs) {
    using namespace tl;
    const char* what = "tl_pages_copy";
    TL_REQUIRE(n_planes >= 0 && n_pages >= 0 && max_pairs >= 0, "%s: negative size", what);
    if (n_planes == 0 || max_pairs == 0 || page_bytes == 0 || n_pages == 0) return TL_OK;
    TL_REQUIRE(pool && src && dst, "%s: null pointer", what);
    TL_REQUIRE(aligned16(pool) && plane_stride % 16 == 0 && page_stride % 16 == 0 && page_bytes % 16 == 0,
               "%s: the pool, its strides and the page size must be multiples of 16 bytes", what);
    TL_REQUIRE(page_stride >= page_bytes || n_pages == 1, "%s: pages overlap", what);
    const size_t pieces = (page_bytes + kPiece - 1) / kPiece;
    if (pieces > 0x7fffffffu) return set_error(TL_ELIMIT, "%s: pages of %zu bytes are too large", what, page_bytes);
    TL_ENSURE_INIT();
    // Past the caches from 256 MB of possible moves on (the host knows no more): packing 4096 pages of 16 x 32 KB, of which a
    // quarter moves, takes 210 us, 5.4 TB/s, against 237; 192 rows of which 48 copy 64 x 8 KB 28 against 29.5 the other way.
    // The workgroups share the possible pieces, about four each: with fewer of them the ones with work become too few.
    const double total = (double)pieces * n_planes * max_pairs;
    const bool past = (double)page_bytes * n_planes * max_pairs >= 268435456.0;
    double blocks = total / 4 < 4096.0 ? 4096.0 : total / 4 < 24576.0 ? total / 4 : 24576.0;
    if (!past) blocks = 4096.0;
    if (blocks > total) blocks = total;
    auto kernel = past ? pages_copy_kernel<true> : pages_copy_kernel<false>;
    kernel<<<(unsigned)blocks, 256, 0, stream()>>>(static_cast<unsigned char*>(pool), plane_stride, page_stride, page_bytes, (unsigned)pieces, n_planes,
                                                   n_pages, src, dst, count, max_pairs);
    TL_CHECK_LAUNCH("pages_copy_kernel");
    return TL_OK;
}

}  // extern "C"
