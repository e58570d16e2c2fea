// Shared by the kernels that write, read and attend to the 8-bit token cache (VdaTokenCache in include/vda_hip.h).
#pragma once
#include "common.h"

// Bytes a row's codes occupy: hd codes, zero-padded so that every row starts on a 16-byte boundary.
__host__ __device__ __forceinline__ int cache_row_bytes(int hd) { return (hd + 15) & ~15; }

static inline int cache_check(const VdaTokenCache* c) {
    if (!c || !c->k || !c->v || !c->k_exp || !c->v_exp || c->pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->hd <= 0) return VDA_EINVAL;
    if (c->format != VDA_CACHE_E4M3 && c->format != VDA_CACHE_I8) return VDA_EINVAL;
    if (c->hd % 8 != 0 || c->hd > 128 || c->page_size % 16 != 0 || c->kv_heads > 65536) return VDA_ESHAPE;
    if ((((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_exp | (uintptr_t)c->v_exp) & 15) != 0) return VDA_ESHAPE;
    if ((long)c->pages * c->page_size > 0x7fffffffL || (long)c->pages * c->page_size * c->kv_heads > (1L << 40)) return VDA_ESHAPE;
    return VDA_OK;
}

// n / d for 0 <= n < 2^31 and a divisor known when the call is made: one high product and a shift.  With l = ceil(log2 d) and
// m = ceil(2^(31 + l) / d) < 2^32, n m / 2^(31 + l) exceeds n / d by less than n / 2^(31 + l) < 2^-l <= 1 / d: the same integer part.
struct Quick {
    unsigned d, m;
    int s;
    explicit Quick(unsigned n) : d(n) {
        int l = 0;
        while ((1ull << l) < n) ++l;
        m = (unsigned)(((1ull << (31 + l)) + n - 1) / n);
        s = l - 1;
    }
    __device__ __forceinline__ int over(int n) const { return d == 1 ? n : (int)(__umulhi((unsigned)n, m) >> s); }
};
