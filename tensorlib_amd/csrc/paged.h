// Helpers of the paged-cache translation units (rotary.hip, paged_attention.hip, pages.hip).
#pragma once
#include "tl_internal.h"

namespace tl {

// Division of n < 2^31 by a divisor that is only known at launch: one 32x32 -> 64 multiplication.  With
// s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1, n / d = (mulhi(n, m) + n) >> s (the sum stays below 2^32).
struct FastDiv {
    unsigned d, m, s;
    FastDiv() = default;
    explicit FastDiv(unsigned divisor) : d(divisor), m(0), s(0) {
        while ((1ull << s) < d) ++s;
        m = (unsigned)((((1ull << 32) * ((1ull << s) - d)) / d) + 1);
    }
#if defined(__HIPCC__)
    __device__ __forceinline__ unsigned div(unsigned n) const { return (__umulhi(n, m) + n) >> s; }
    __device__ __forceinline__ unsigned divmod(unsigned n, unsigned& rem) const {
        const unsigned q = div(n);
        rem = n - q * d;
        return q;
    }
#endif
};

// Host checks shared by the entry points that take a tl_kv_pages.
inline int check_kv_pages(const tl_kv_pages* c, const char* what) {
    TL_REQUIRE(c != nullptr, "%s: cache description is null", what);
    TL_REQUIRE(c->k && c->v, "%s: null cache pointer", what);
    TL_REQUIRE(c->n_pages >= 1 && c->page_size >= 1 && c->n_kv_heads >= 1, "%s: n_pages, page_size and n_kv_heads must be positive", what);
    TL_REQUIRE(c->head_dim >= 8 && c->head_dim <= 256 && c->head_dim % 8 == 0,
               "%s: head_dim %d is not a multiple of 8 in [8, 256]", what, c->head_dim);
    TL_REQUIRE(aligned16(c->k) && aligned16(c->v), "%s: cache pointers must be 16-byte aligned", what);
    TL_REQUIRE(c->page_stride % 8 == 0 && c->row_stride % 8 == 0 && c->head_stride % 8 == 0,
               "%s: cache strides must be multiples of 8 elements", what);
    return TL_OK;
}

}  // namespace tl
