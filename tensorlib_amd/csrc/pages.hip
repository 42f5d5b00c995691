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
constexpr int kMaxPages = 1 << 30;         // page numbers are stepped through in int

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

// A workgroup of 1024 over the reference counts of any number of pages: each wavefront has a sixteenth of them to itself and
// goes through it in page order, 256 at a time, so that ranks come from ballots and the wavefronts meet only once.  The first
// 256 are read when the range is made, early where that hides the wait, and kept: up to 4096 pages there are no others.
constexpr int kWaves = kThreads / 64;
struct PageRange {
    const int* refs;
    int n_pages, begin, end;
    int4 first;
    __device__ PageRange(const int* refs_, int n_pages_) : refs(refs_), n_pages(n_pages_) {
        const long steps = ((long)n_pages + kWaves * 256 - 1) / (kWaves * 256), wave = threadIdx.x / 64;
        const long b = wave * steps * 256, e = b + steps * 256;
        begin = b < n_pages ? (int)b : n_pages;
        end = e < n_pages ? (int)e : n_pages;
        first = load(begin + (int)(threadIdx.x % 64) * 4);
    }
    // Four counts of the lane; behind the range's last page zeros, which f() never sees.
    __device__ __forceinline__ int4 load(int p) const {
        int4 r = {0, 0, 0, 0};
        if (p + 4 <= end) __builtin_memcpy(&r, refs + p, 16);
        else {
            if (p < end) r.x = refs[p];
            if (p + 1 < end) r.y = refs[p + 1];
            if (p + 2 < end) r.z = refs[p + 2];
        }
        return r;
    }
    // take(rank, page, count) for the pages of the wavefront's range that f(page, count) picks, ranks from `rank` on; returns
    // the rank behind the last one.  Stops at a rank of `most`.  Of the counts, take() may change the one it is given.
    template <class F, class T>
    __device__ __forceinline__ int visit(int rank, int most, F f, T take) const {
        const int lane = threadIdx.x % 64;
        const unsigned long long below = (1ull << lane) - 1;
        int4 next = first;
        for (int p0 = begin; p0 < end && rank < most; p0 += 256) {
            const int p = p0 + lane * 4;
            const int4 r = next;
            if (p0 + 256 < end) next = load(p + 256);
            const bool pick[4] = {p < end && f(p, r.x), p + 1 < end && f(p + 1, r.y), p + 2 < end && f(p + 2, r.z), p + 3 < end && f(p + 3, r.w)};
            const unsigned long long b[4] = {__ballot(pick[0]), __ballot(pick[1]), __ballot(pick[2]), __ballot(pick[3])};
            int mine = rank + (int)(__popcll(b[0] & below) + __popcll(b[1] & below) + __popcll(b[2] & below) + __popcll(b[3] & below));
            const int count[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (pick[j]) {
                    take(mine, p + j, count[j]);
                    ++mine;
                }
            rank += (int)(__popcll(b[0]) + __popcll(b[1]) + __popcll(b[2]) + __popcll(b[3]));
        }
        return rank;
    }
    // How many pages f picks in the whole pool; *before: in the ranges of the wavefronts before this one.  In the same meeting
    // the sum of another number of each wavefront, own(pages picked here): *all_own, and its part before this one, *own_before.
    template <class F, class G>
    __device__ int count(F f, int* before, G own, int* own_before, int* all_own) const {
        __shared__ int2 s_count[kWaves];
        const int n = visit(0, 0x7fffffff, f, [](int, int, int) {});
        const int also = own(n);
        __syncthreads();
        if (threadIdx.x % 64 == 0) s_count[threadIdx.x / 64] = {n, also};
        __syncthreads();
        int all = 0;
        *before = *own_before = *all_own = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const int2 c = s_count[w];
            if (w < (int)threadIdx.x / 64) {
                *before += c.x;
                *own_before += c.y;
            }
            all += c.x;
            *all_own += c.y;
        }
        return all;
    }
};
__device__ __forceinline__ bool is_free(int, int count) { return count == 0; }

constexpr int kSmallPages = 16384;         // a fork of at most this in one launch: the counts fit LDS,
constexpr int kSmallSeqs = kThreads;       // the rows a thread each,
constexpr size_t kSmallEntries = 65536;    // and the tables' entries are soon gone through

struct ForkArgs {
    const int *tables, *lens, *refs, *parents;
    int *tables_out, *lens_out, *refs_out, *copy_src, *copy_dst, *missing;
    int n_seqs, table_stride, n_pages, page_size;
    int row_shift;                         // log2 of the threads a row has
};

// A fork in one launch, one workgroup (192 x 128 entries of which 19 are pages 7.2 us, against 11 for the three launches
// below; 256 x 128 with 120 pages 15 against 23; 512 x 128 13 against 14.5 and 31 against 33; 1000 x 128 with 60 pages 63
// against 45).  A row has 1024 / n_seqs threads, rounded down to a power of two.  First the counts: an entry of an old row is
// named by the row's children instead of by the row, a partly filled last page by the first of them, so nothing changes for
// a row with one child and its table need not be read.  The new tables are written last, when all pages are known, since a
// barrier behind a store waits for it (1.4 us).  VEC: table entries a thread moves at a time, 4 where rows are 16-byte aligned.
template <int VEC>
__global__ void __launch_bounds__(kThreads) pages_fork_small_kernel(ForkArgs A) {
    __shared__ int s_len[kSmallSeqs], s_pages[kSmallSeqs], s_full[kSmallSeqs], s_parent[kSmallSeqs], s_first[kSmallSeqs], s_children[kSmallSeqs],
        s_page[kSmallSeqs], s_copy[kSmallSeqs];
    extern __shared__ int s_refs[];
    struct alignas(4 * VEC) Entries { int v[VEC]; };
    const int r = threadIdx.x;
    const bool row = r < A.n_seqs;
    const int parent = row ? A.parents[r] : -1;
    const int old_len = row ? A.lens[r] : 0;
    for (int p = r; p < A.n_pages; p += kThreads) s_refs[p] = A.refs[p];
    const int held = pages_of(old_len, A.page_size, A.table_stride);
    s_first[r] = kSmallSeqs;
    s_children[r] = 0;
    s_len[r] = old_len > 0 ? old_len : 0;
    s_pages[r] = held;
    s_full[r] = old_len > 0 && old_len % A.page_size != 0 ? held - 1 : held;
    s_parent[r] = parent >= 0 && parent < A.n_seqs ? parent : -1;
    __syncthreads();
    const bool has = s_parent[r] >= 0;
    const int len = has ? s_len[parent] : 0;
    const int new_pages = has ? s_pages[parent] : 0;
    const bool partial = has && s_full[parent] < new_pages;
    int last = -1;                         // the page to be copied, if the row is not its parent's first
    if (has) atomicAdd(s_children + parent, 1);
    if (partial) {
        last = A.tables[(size_t)parent * A.table_stride + new_pages - 1];
        atomicMin(s_first + parent, r);
    }
    __syncthreads();
    const bool wants = partial && s_first[parent] != r && last >= 0 && last < A.n_pages;
    const int to = r >> A.row_shift, step = VEC << A.row_shift, c0 = (r & ((1 << A.row_shift) - 1)) * VEC;
    if (to < A.n_seqs && s_children[to] != 1) {
        const int children = s_children[to], full = s_full[to], pages = s_pages[to];
        for (int c = c0; c < pages; c += step) {
            const Entries o = *reinterpret_cast<const Entries*>(A.tables + (size_t)to * A.table_stride + c);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int gained = (c + j < full ? children : children ? 1 : 0) - 1;
                if (c + j < pages && gained != 0 && o.v[j] >= 0 && o.v[j] < A.n_pages) atomicAdd(s_refs + o.v[j], gained);
            }
        }
    }
    __syncthreads();
    const unsigned long long wanting = __ballot(wants);
    int wanted, before, rank;
    const PageRange range(s_refs, A.n_pages);
    const int available = range.count(is_free, &before, [&](int) { return (int)__popcll(wanting); }, &rank, &wanted);
    rank += __popcll(wanting & ((1ull << (r % 64)) - 1));
    const bool enough = available >= wanted;
    if (enough) range.visit(before, wanted, is_free, [&](int k, int page, int) {
        if (k >= wanted) return;
        s_page[k] = page;
        s_refs[page] = 1;
    });
    __syncthreads();
    if (r == 0) *A.missing = enough ? 0 : wanted - available;
    if (row) {
        const int page = wants && enough ? s_page[rank] : -1;
        s_copy[r] = page;
        A.copy_src[r] = page >= 0 ? last : -1;
        A.copy_dst[r] = page;
        A.lens_out[r] = enough ? len : old_len;
    }
    for (int p = r; p < A.n_pages; p += kThreads) A.refs_out[p] = enough ? s_refs[p] : A.refs[p];
    __syncthreads();
    if (to >= A.n_seqs) return;
    const int from = enough ? s_parent[to] : to, page = s_copy[to];
    const int pages = !enough ? A.table_stride : from >= 0 ? s_pages[from] : 0;
    for (int c = c0; c < A.table_stride; c += step) {
        Entries x;
        if (c < pages) x = *reinterpret_cast<const Entries*>(A.tables + (size_t)from * A.table_stride + c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if (c + j >= pages) x.v[j] = -1;
            if (page >= 0 && c + j == pages - 1) x.v[j] = page;
        }
        *reinterpret_cast<Entries*>(A.tables_out + (size_t)to * A.table_stride + c) = x;
    }
}

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
    const PageRange range(A.refs_out, A.n_pages);
    int before, unused, none;
    const int available = range.count(is_free, &before, [](int) { return 0; }, &unused, &none);
    if (threadIdx.x == 0) *A.missing = available < wanted ? wanted - available : 0;
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
    range.visit(before, wanted, is_free, [&](int k, int page, int) {
        if (k >= wanted) return;
        A.refs_out[page] = 1;
        const int row = A.copy_dst[k];
        A.tables_out[(size_t)row * A.table_stride + pages_of(A.lens_out[row], A.page_size, A.table_stride) - 1] = page;
    });
    __syncthreads();
    for (int r = threadIdx.x; r < A.n_seqs; r += kThreads)
        A.copy_dst[r] = A.copy_src[r] >= 0 ? A.tables_out[(size_t)r * A.table_stride + pages_of(A.lens_out[r], A.page_size, A.table_stride) - 1] : -1;
}

// Room for add[r] more positions of every sequence, all or nothing (one workgroup).  Each wavefront has a sixteenth of the
// sequences and of the pages, and they meet once.  The pages go into a list first and from there to the rows, a thread each with the
// search for its row: 1.5 us for 192 rows that want a page each, against 3.6 where a lane's four neighbours were searched for in turn.
constexpr int kListPages = 8192;           // more are stored where they are found
__global__ void __launch_bounds__(kThreads)
pages_extend_kernel(int* tables, int* lens, int* refs, const int* add, int* missing, int n_seqs, int table_stride, int n_pages, int page_size) {
    __shared__ int s_page[kListPages];
    __shared__ int s_refused;
    extern __shared__ int s_first[];      // number of pages wanted by the rows before
    const PageRange range(refs, n_pages);
    const int lane = threadIdx.x % 64, steps = (n_seqs + kThreads - 1) / kThreads, r0 = (int)threadIdx.x / 64 * steps * 64 + lane;
    if (threadIdx.x == 0) s_refused = 0;
    int own = 0;
    bool refused = false;
    for (int i = 0; i < steps; ++i) {
        const int r = r0 + i * 64;
        int need = 0;
        if (r < n_seqs) {
            const int len = max(lens[r], 0);
            const unsigned target = (unsigned)len + (unsigned)max(add[r], 0);
            const unsigned pages = target ? (target - 1) / (unsigned)page_size + 1 : 0;
            if (target > 0x7fffffffu || pages > (unsigned)table_stride) refused = true;
            else need = (int)pages - pages_of(len, page_size, table_stride);
        }
        int x = need;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int y = __shfl_up(x, d, 64);
            if (lane >= d) x += y;
        }
        if (r < n_seqs) s_first[r] = own + x - need;
        own += __shfl(x, 63, 64);
    }
    int before, own_before, wanted;
    const int available = range.count(is_free, &before, [&](int) { return own; }, &own_before, &wanted);
    if (refused) s_refused = 1;
    for (int i = 0; i < steps; ++i)
        if (r0 + i * 64 < n_seqs) s_first[r0 + i * 64] += own_before;
    __syncthreads();
    refused = s_refused != 0;
    if (threadIdx.x == 0) *missing = refused ? -1 : available < wanted ? wanted - available : 0;
    if (refused || available < wanted) return;
    auto place = [&](int k, int page) {
        refs[page] = 1;
        int lo = 0, hi = n_seqs - 1;      // the last row whose first page is at most k
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (s_first[mid] <= k) lo = mid;
            else hi = mid - 1;
        }
        tables[(size_t)lo * table_stride + pages_of(lens[lo], page_size, table_stride) + k - s_first[lo]] = page;
    };
    const bool listed = wanted <= kListPages;
    range.visit(before, wanted, is_free, [&](int k, int page, int) {
        if (k >= wanted) return;
        if (listed) s_page[k] = page;
        else place(k, page);
    });
    __syncthreads();
    if (listed) {
        for (int k = threadIdx.x; k < wanted; k += kThreads) place(k, s_page[k]);
        __syncthreads();                   // lens have been read
    }
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

// New ids and counts, and the rest of the lists, for pages i, i + step, ..  The lists are in page order, so the first mover and
// the last hole tell a page's part: live and not below the first mover, it moves; free and not above the last hole, it is filled.
struct CompactArgs {
    const int* refs;
    int *refs_out, *remap, *copy_src, *copy_dst, *count;
    int n_pages;
    const int* tables;
    int* tables_out;
    size_t n_entries;
};
__device__ __forceinline__ void compact_apply(const CompactArgs& A, int movers, size_t i, size_t step) {
    const int first = movers ? A.copy_src[0] : A.n_pages, last = movers ? A.copy_dst[movers - 1] : -1;
    for (; i < (size_t)A.n_pages; i += step) {
        const int p = (int)i, ref = A.refs[p];
        if (ref <= 0) A.remap[p] = -1;
        else if (p < first) A.remap[p] = p;
        if (p < first && ref > 0) A.refs_out[p] = ref;
        else if (p > last || ref > 0) A.refs_out[p] = 0;
        if (p < movers) {
            const int from = A.copy_src[p], to = A.copy_dst[p];
            A.remap[from] = to;
            A.refs_out[to] = A.refs[from];
        } else {
            A.copy_src[p] = A.copy_dst[p] = -1;
        }
    }
}
// The tables' entries i, i + step, ..
__device__ __forceinline__ void compact_tables(const CompactArgs& A, size_t i, size_t step) {
    for (; i < A.n_entries; i += step) {
        const int p = A.tables[i];
        A.tables_out[i] = p >= 0 && p < A.n_pages ? A.remap[p] : p;
    }
}
__global__ void __launch_bounds__(256) pages_remap_kernel(CompactArgs A) {
    compact_tables(A, (size_t)blockIdx.x * 256 + threadIdx.x, (size_t)gridDim.x * 256);
}
__global__ void __launch_bounds__(256) pages_compact_apply_kernel(CompactArgs A) {
    compact_apply(A, *A.count, (size_t)blockIdx.x * 256 + threadIdx.x, (size_t)gridDim.x * 256);
}
// One workgroup: the live pages above the number of live pages move into the free ones below it, in page order.  PARTS: and all
// the rest for a pool that one workgroup is soon through with (2; 1000 pages 5.6 against 6.9 us and a launch, 4096 7.9 against
// 8.2, 8192 11.4 against 10.3), the tables too (3; 1000 pages and 100 entries 4.5 against 5.7 us and a launch, 4096 entries 5.6
// against 5.9, 16384 9.0 against 6.0).
constexpr int kWholePages = 4096;
constexpr size_t kWholeEntries = 4096;
template <int PARTS>
__global__ void __launch_bounds__(kThreads) pages_compact_plan_kernel(CompactArgs A) {
    const PageRange range(A.refs, A.n_pages);
    int before, mine = 0, holes_before, unused;
    const int live = range.count([](int, int ref) { return ref > 0; }, &before, [&](int n) { return mine = n; }, &holes_before, &unused);
    auto mover = [live](int p, int ref) { return ref > 0 && p >= live; };
    auto hole = [live](int p, int ref) { return ref <= 0 && p < live; };
    // of the range's pages below `live`, those that are not live
    const int below = live < range.begin ? 0 : (live < range.end ? live : range.end) - range.begin;
    const int movers = range.count(mover, &before, [&](int n) { return below - (mine - n); }, &holes_before, &unused);
    range.visit(before, 0x7fffffff, mover, [&](int k, int p, int) { A.copy_src[k] = p; });
    range.visit(holes_before, 0x7fffffff, hole, [&](int k, int p, int) { A.copy_dst[k] = p; });
    if (threadIdx.x == 0) *A.count = movers;
    if constexpr (PARTS >= 2) {
        __syncthreads();
        compact_apply(A, movers, threadIdx.x, kThreads);
    }
    if constexpr (PARTS >= 3) {
        __syncthreads();
        compact_tables(A, threadIdx.x, kThreads);
    }
}

// A piece is 256 threads x 4 x 16 bytes of a pair's page in all planes, one plane's after the other's: pages may be much
// smaller than a piece (16 planes of 1 KB, 1100 pairs: 29 -> 15 us with the numbering).  STREAM: accesses that do not settle in the caches, for calls that may move more than fits there.
constexpr unsigned kPiece = 256 * 4;       // in units of 16 bytes
template <bool STREAM>
__global__ void __launch_bounds__(256)
pages_copy_kernel(unsigned char* pool, size_t plane_stride, size_t page_stride, FastDiv by_page, FastDiv by_pieces, unsigned units, int n_pages, const int* src,
                  const int* dst, const int* count, int max_pairs) {
    const unsigned pairs = count ? (unsigned)min(max(*count, 0), max_pairs) : (unsigned)max_pairs;
    unsigned piece, step;
    unsigned pair = by_pieces.divmod(blockIdx.x, piece);
    const unsigned pair_step = by_pieces.divmod(gridDim.x, step);
    for (; pair < pairs; pair += pair_step + (piece + step >= by_pieces.d), piece = piece + step >= by_pieces.d ? piece + step - by_pieces.d : piece + step) {
        const unsigned first = piece * kPiece + threadIdx.x;
        const int from = src[pair], to = dst[pair];
        if (from < 0 || from >= n_pages || to < 0 || to >= n_pages) continue;
        float4_t x[4];
        size_t at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned u = first + j * 256;
            unsigned unit;
            const unsigned plane = by_page.divmod(u, unit);
            at[j] = plane * plane_stride + (size_t)unit * 16;
            const float4_t* from4 = reinterpret_cast<const float4_t*>(pool + from * page_stride + at[j]);
            if (u < units) x[j] = STREAM ? __builtin_nontemporal_load(from4) : *from4;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float4_t* to4 = reinterpret_cast<float4_t*>(pool + to * page_stride + at[j]);
            if (first + j * 256 >= units) continue;
            if (STREAM) __builtin_nontemporal_store(x[j], to4);
            else *to4 = x[j];
        }
    }
}

static int check_state(const char* what, int n_seqs, int table_stride, int n_pages, int page_size) {
    TL_REQUIRE(n_seqs >= 0 && table_stride >= 1 && n_pages >= 1 && page_size >= 1, "%s: sizes out of range", what);
    if (n_seqs > kMaxSeqs) return set_error(TL_ELIMIT, "%s: %d sequences, at most %d", what, n_seqs, kMaxSeqs);
    if (n_pages > kMaxPages) return set_error(TL_ELIMIT, "%s: %d pages, at most %d", what, n_pages, kMaxPages);
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
    ForkArgs A{tables, lens, refs, parents, tables_out, lens_out, refs_out, copy_src, copy_dst, missing, n_seqs, table_stride, n_pages, page_size, 0};
    if (small_state(n_seqs, table_stride, n_pages)) {
        const bool vec = table_stride % 4 == 0 && aligned16(tables) && aligned16(tables_out);
        while ((n_seqs << (A.row_shift + 1)) <= kThreads && A.row_shift < 10) ++A.row_shift;
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
    if (n_pages > kMaxPages) return set_error(TL_ELIMIT, "%s: %d pages, at most %d", what, n_pages, kMaxPages);
    TL_REQUIRE(refs && refs_out && remap && copy_src && copy_dst && count && (n_seqs == 0 || (tables && tables_out)), "%s: null pointer", what);
    TL_REQUIRE(refs_out != refs, "%s: the new reference counts must not lie over the old ones", what);
    TL_ENSURE_INIT();
    const size_t n = (size_t)n_seqs * table_stride;
    const CompactArgs A{refs, refs_out, remap, copy_src, copy_dst, count, n_pages, tables, tables_out, n};
    const int parts = n_pages > kWholePages ? 1 : n > kWholeEntries ? 2 : 3;
    auto plan = parts == 1 ? pages_compact_plan_kernel<1> : parts == 2 ? pages_compact_plan_kernel<2> : pages_compact_plan_kernel<3>;
    plan<<<1, kThreads, 0, stream()>>>(A);
    TL_CHECK_LAUNCH("pages_compact_plan_kernel");
    if (parts < 2) {
        pages_compact_apply_kernel<<<ints_grid(n_pages), 256, 0, stream()>>>(A);
        TL_CHECK_LAUNCH("pages_compact_apply_kernel");
    }
    if (parts < 3 && n > 0) {
        pages_remap_kernel<<<ints_grid(n), 256, 0, stream()>>>(A);
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
    const double all_units = (double)page_bytes / 16 * n_planes;
    if (all_units > 2147482624.0) return set_error(TL_ELIMIT, "%s: %d pages of %zu bytes are too much for one pair", what, n_planes, page_bytes);
    TL_ENSURE_INIT();
    const unsigned units = (unsigned)(page_bytes / 16 * n_planes), pieces = (units + kPiece - 1) / kPiece;
    // Past the caches from 256 MB of possible moves on (the host knows no more): packing 4096 pages of 16 x 32 KB, of which a
    // quarter moves, takes 206 us, 5.5 TB/s, against 237; 192 rows of which 48 copy 64 x 8 KB 22 against 24 the other way.
    // The workgroups share the possible pieces, about four each: with fewer of them the ones with work become too few.
    const double total = (double)pieces * max_pairs;
    const bool past = all_units * 16 * max_pairs >= 268435456.0;
    double blocks = total / 4 < 4096.0 ? 4096.0 : total / 4 < 24576.0 ? total / 4 : 24576.0;
    if (!past) blocks = 4096.0;
    if (blocks > total) blocks = total;
    auto kernel = past ? pages_copy_kernel<true> : pages_copy_kernel<false>;
    kernel<<<(unsigned)blocks, 256, 0, stream()>>>(static_cast<unsigned char*>(pool), plane_stride, page_stride, FastDiv((unsigned)(page_bytes / 16)), FastDiv(pieces), units,
                                                   n_pages, src, dst, count, max_pairs);
    TL_CHECK_LAUNCH("pages_copy_kernel");
    return TL_OK;
}

}  // extern "C"
