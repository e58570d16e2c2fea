// What the two attention kernels over the token cache share (cached_attention.hip).
#pragma once
#include "token_cache.h"

// One launch.  Query row `rho` of a sequence and key head is query token rho / group, head kvh * group + rho % group: the heads that
// share a key head share its tiles.
struct AttendJob {
    const uint8_t *k, *v, *k_exp, *v_exp;
    const int *page_table, *kv_len, *q_start, *visible;
    float* part;                // per (item, split): [rows of a block][hd padded] outputs, then their references and sums (outputs over sums are the
                                // part's result, both times 2^(127 + P_SHIFT - reference)); a part behind a sequence's last key is not written, a row
                                // without a key in a written part has sum 0.  Unused where splits == 1
    long rows, ldq, ldo;
    int pages, page_size, kv_heads, hd, row_bytes, max_pages, group, seqs;
    int row_blocks, splits;     // blocks of query rows per (sequence, key head); parts of the key axis,
    int chunk;                  // of `chunk` keys each: a short sequence has fewer parts, not smaller ones
    float scale_log2e;
    Quick by_splits, by_heads, by_blocks, by_group, by_page;
};

// The sequence's own numbers, cut to what the tensors hold.
struct Span {
    int q0, nq, n;              // first query row, query rows, keys
};
__device__ __forceinline__ Span span_of(const AttendJob& j, int s, int max_q) {
    const long a = max(0L, min((long)j.q_start[s], j.rows)), b = max(a, min((long)j.q_start[s + 1], j.rows));
    return Span{(int)a, (int)min(b - a, (long)max_q), max(0, min(j.kv_len[s], j.max_pages * j.page_size))};
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
constexpr float LOWEST = -1e30f;        // running maximum of a row that has seen no key: exp2(-inf - LOWEST) is 0, not NaN
constexpr float DEFER = 6.f;            // growth of the running maximum (in octaves) below which sums are not rescaled
// Probabilities of 16-bit rows are one half each, 11 bits: that adds a tenth to a quarter to the error of an fp16 result (2.07e-4 of the
// outputs becomes 2.2e-4 to 2.5e-4) and nothing to a bf16 one (1.6e-3).  Two pieces are what fp32 rows take, of q and of the
// probabilities: 94 us where 16-bit rows take 67 (1370 rows over 10960 keys, 8 heads of 64).
constexpr int P_SHIFT = 8;              // probabilities reach 2^DEFER; in IEEE halves they are kept times 2^P_SHIFT, far from subnormals

// 8-bit codes to IEEE halves, exactly.  Integers: the biased byte under the exponent of 1024, then minus 1024 + 128.
__device__ __forceinline__ f16x2 unbias(unsigned magic) {
    return __builtin_bit_cast(f16x2, magic) - f16x2{(f16)1152.f, (f16)1152.f};
}
template <int FMT>
__device__ __forceinline__ void codes4(unsigned w, f16x2& a, f16x2& b) {                 // bytes 0, 1 and 2, 3
    if (FMT == VDA_CACHE_I8) {
        w ^= 0x80808080u;
        a = unbias(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u));
        b = unbias(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u));
    } else {
        a = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
        b = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true));
    }
}
template <int FMT>
__device__ __forceinline__ f16x8 codes8(u32x2 w) {
    f16x2 a, b, c, d;
    codes4<FMT>(w[0], a, b);
    codes4<FMT>(w[1], c, d);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Eight query values as fp32 (zeros for a row that is not there).
template <typename T>
__device__ __forceinline__ void query8(const T* p, bool there, float* f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
    if (!there) return;
    if constexpr (sizeof(T) == 2) {
        const typename Vec<T>::v8 v = *reinterpret_cast<const typename Vec<T>::v8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)v[i];
    } else {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[i] = a[i]; f[4 + i] = b[i]; }
    }
}
// A query row is brought to magnitudes 2^13 .. 2^14 by a power of two before it becomes halves: 16-bit rows then convert exactly
// (down to 2^-38 of the row's largest value) and fp32 rows split into two halves of 22 bits, whatever their size.
__device__ __forceinline__ int query_shift(float amax) {
    if (!(amax > 0.f) || amax == INFINITY) return 0;
    int e;
    frexpf(amax, &e);
    return 14 - e;
}
template <int NP>
__device__ __forceinline__ void query_pieces(const float* f, int shift, f16x8* out) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = __builtin_amdgcn_ldexpf(f[i], shift);
        const f16 hi = (f16)v;
        out[0][i] = hi;
        if (NP == 2) out[NP - 1][i] = (f16)(v - (float)hi);
    }
}
template <typename T> struct Pieces { static constexpr int n = 1; };
template <> struct Pieces<float> { static constexpr int n = 2; };

__device__ __forceinline__ unsigned byte_of(unsigned w, int i) { return (w >> (8 * i)) & 255u; }
// not 0 if some byte of w is 0 or 255 (and now and then for 254 above a 255: a carry; the caller then looks at each byte)
__device__ __forceinline__ unsigned odd_bytes(unsigned w) {
    const unsigned x = (w + 0x01010101u) & 0xfefefefeu;
    return (x - 0x01010101u) & ~x & 0x80808080u;
}
__device__ __forceinline__ float power_of_byte(unsigned byte) { return __uint_as_float(byte << 23); }      // 2^(byte - 127), 1 <= byte <= 254

int attend_few(const AttendJob& j, const void* q, void* out, int dtype, int format, int max_q, int waves, hipStream_t st);
int attend_many(const AttendJob& j, const void* q, void* out, int dtype, int format, int max_q, hipStream_t st);
int attend_join(const AttendJob& j, void* out, int dtype, int max_q, int block_rows, int hd_pad, hipStream_t st);
