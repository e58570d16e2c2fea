// Rotary positions over three axes, and the 8-bit token cache's writer and reader (see vda_rotary_axes, vda_cache_write and
// vda_cache_read in include/vda_hip.h).  All three move every value once and compute little: memory bandwidth bounds them.
#include "token_cache.h"

namespace {

// Pair j of a head turns by pos[axis(j)] * freq[j].  Time positions of a long video reach millions, where an fp32 product is off
// by a tenth of a turn: the product and its reduction to within half a turn are formed in double, once per token and pair (every
// head of the token then uses it), and only the remainder goes to fp32.
struct Axes {
    const void* pos;
    const double* freq;
    int half, end_t, end_h, pos_float;
};
__device__ __forceinline__ float2 turn(const Axes& a, long row, int j) {
    const int axis = j < a.end_t ? 0 : j < a.end_h ? 1 : 2;
    const long at = row * 3 + axis;
    const double p = a.pos_float ? (double)reinterpret_cast<const float*>(a.pos)[at] : (double)reinterpret_cast<const int*>(a.pos)[at];
    double rev = p * a.freq[j] * 0.15915494309189533577;
    rev -= rint(rev);
    float2 cs;
    sincospif((float)(2.0 * rev), &cs.y, &cs.x);
    return cs;
}

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };
template <typename T, int N>
__device__ __forceinline__ void load_f32(const T* p, float* f) {
    const Pack<T, N> r = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = (float)r.v[i];
}
template <typename T, int N>
__device__ __forceinline__ void store_f32(T* p, const float* f) {
    Pack<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = (T)f[i];
    *reinterpret_cast<Pack<T, N>*>(p) = r;
}

// A workgroup turns `tb` tokens: first the angles of their tb * half pairs into LDS, then one unit of U pairs per thread.  A
// thread holds both members of its pairs, so the call may be in place.
template <typename T, int U, bool ADJ>
__global__ __launch_bounds__(256) void rotary_kernel(const T* x, T* out, Axes ax, long rows, long ldx, long ldo, int heads, int hd, int tb,
                                                     int copies) {
    extern __shared__ float2 cs[];
    const long r0 = (long)blockIdx.x * tb;
    const int nt = (int)min((long)tb, rows - r0);
    const int half = ax.half;
    for (int i = threadIdx.x; i < nt * half; i += 256) {
        const int t = i / half;
        cs[i] = turn(ax, r0 + t, i - t * half);
    }
    __syncthreads();
    constexpr int CU = U < 4 ? 4 : (sizeof(T) == 2 ? 8 : 4);         // channels of a unit that is only copied
    const unsigned units = half / U, per_head = units + copies, per_row = per_head * heads;
    for (unsigned i = threadIdx.x; i < nt * per_row; i += 256) {
        const unsigned t = i / per_row, in_row = i - t * per_row, head = in_row / per_head, u = in_row - head * per_head;
        const T* xr = x + (r0 + t) * ldx + head * hd;
        T* yr = out + (r0 + t) * ldo + head * hd;
        if (u >= units) {
            float f[CU];
            const int c = 2 * half + (u - units) * CU;
            load_f32<T, CU>(xr + c, f);
            store_f32<T, CU>(yr + c, f);
            continue;
        }
        const float2* w = cs + t * half + u * U;
        if (ADJ) {
            float f[2 * U], g[2 * U];
            load_f32<T, U>(xr + 2 * U * u, f);
            load_f32<T, U>(xr + 2 * U * u + U, f + U);
#pragma unroll
            for (int k = 0; k < U; ++k) {
                g[2 * k] = f[2 * k] * w[k].x - f[2 * k + 1] * w[k].y;
                g[2 * k + 1] = f[2 * k + 1] * w[k].x + f[2 * k] * w[k].y;
            }
            store_f32<T, U>(yr + 2 * U * u, g);
            store_f32<T, U>(yr + 2 * U * u + U, g + U);
        } else {
            float a[U], b[U], c[U], d[U];
            load_f32<T, U>(xr + U * u, a);
            load_f32<T, U>(xr + half + U * u, b);
#pragma unroll
            for (int k = 0; k < U; ++k) {
                c[k] = a[k] * w[k].x - b[k] * w[k].y;
                d[k] = b[k] * w[k].x + a[k] * w[k].y;
            }
            store_f32<T, U>(yr + U * u, c);
            store_f32<T, U>(yr + half + U * u, d);
        }
    }
}

// ---- the 8-bit cache -------------------------------------------------------------------------------------------------------
// Scales are powers of two, stored as the exponent plus 127: multiplying and dividing by them is exact, so a code is one rounding
// of the value and every implementation of the rule stores the same code.  The row's exponent is the smallest that brings its
// largest magnitude within the largest code (127 = 1.984375 * 2^6, 448 = 1.75 * 2^8); it follows from the bits of that magnitude.
__device__ __forceinline__ int exponent_byte(unsigned amax_bits, int format) {
    const int field = amax_bits >> 23;
    const unsigned mant = amax_bits & 0x7fffff;
    if (field == 255) return 255;                                  // the row holds an infinity or a NaN
    const int e = format == VDA_CACHE_I8 ? field - 6 + (mant > 0x7e0000) : field - 8 + (mant > 0x600000);
    return max(1, min(254, e));                                    // 0 marks an empty slot
}
__device__ __forceinline__ u32x2 encode8(const float* f, int byte, int format) {
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = __builtin_amdgcn_ldexpf(f[k], 127 - byte);
    u32x2 c = {0u, 0u};
    if (byte == 255) return c;
    if (format == VDA_CACHE_I8) {
#pragma unroll
        for (int k = 0; k < 8; ++k) c[k >> 2] |= ((unsigned)(int)rintf(y[k]) & 255u) << (8 * (k & 3));
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * k], y[4 * k + 1], 0, false);
            c[k] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * k + 2], y[4 * k + 3], w, true);
        }
    }
    return c;
}
__device__ __forceinline__ void decode8(u32x2 c, int byte, int format, float* f) {
    if (byte == 0 || byte == 255) {
        const float v = byte ? __builtin_nanf("") : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = v;
        return;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (format == VDA_CACHE_I8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[4 * k + i] = (float)(int)(signed char)(c[k] >> (8 * i));
        } else {
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(c[k], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c[k], true);
            f[4 * k] = lo[0]; f[4 * k + 1] = lo[1]; f[4 * k + 2] = hi[0]; f[4 * k + 3] = hi[1];
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = __builtin_amdgcn_ldexpf(f[k], byte - 127);
}

struct CacheDims {
    uint8_t *k, *v, *k_exp, *v_exp;
    int page_size, kv_heads, hd, row_bytes;
    long slots;
};
// Where a token's row of head 0 lies, in rows of a cache plane; -1: the token has no slot.  Head h's row lies h * page_size further.
__device__ __forceinline__ long plane_row(const CacheDims& c, long slot) {
    if (slot < 0 || slot >= c.slots) return -1;
    const unsigned page = (unsigned)slot / (unsigned)c.page_size;
    return (long)page * c.page_size * c.kv_heads + ((unsigned)slot - page * (unsigned)c.page_size);
}

// The rotated value of four channels e0..e0+3 of a row at p (e0 % 4 == 0, so that the four lie in one half).
template <typename T, bool ADJ>
__device__ __forceinline__ void rotated4(const T* p, int e0, int half, const float2* w, float* y) {
    float a[4], b[4];
    load_f32<T, 4>(p + e0, a);
    if (e0 >= 2 * half) {
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = a[k];
    } else if (ADJ) {
        const float2 w0 = w[e0 >> 1], w1 = w[(e0 >> 1) + 1];
        y[0] = a[0] * w0.x - a[1] * w0.y; y[1] = a[1] * w0.x + a[0] * w0.y;
        y[2] = a[2] * w1.x - a[3] * w1.y; y[3] = a[3] * w1.x + a[2] * w1.y;
    } else {
        const bool first = e0 < half;
        load_f32<T, 4>(p + (first ? e0 + half : e0 - half), b);
        const float2* wj = w + (first ? e0 : e0 - half);
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = a[k] * wj[k].x + (first ? -b[k] : b[k]) * wj[k].y;
    }
}

// A workgroup stores `tb` tokens (a power of two), LPH lanes of 8 channels for each (head, token), tokens fastest: the codes of a
// head's consecutive slots are neighbours in the cache.
enum { ROT_NONE = 0, ROT_HALVES = 1, ROT_ADJ = 2 };
template <typename T, int LPH, int ROT>
__global__ __launch_bounds__(256) void cache_write_kernel(const T* __restrict__ k, const T* __restrict__ v, CacheDims c, const long* __restrict__ slots,
                                                          Axes ax, long rows, long ldk, long ldv, int log_tb, int format) {
    extern __shared__ float2 cs[];
    __shared__ long at_row[32];
    const int tb = 1 << log_tb;
    const long r0 = (long)blockIdx.x << log_tb;
    const int nt = (int)min((long)tb, rows - r0), half = ax.half;
    if ((int)threadIdx.x < tb) at_row[threadIdx.x] = (int)threadIdx.x < nt ? plane_row(c, slots[r0 + threadIdx.x]) : -1;
    if (ROT != ROT_NONE)
        for (int i = threadIdx.x; i < nt * half; i += 256) {
            const int t = i / half;
            cs[i] = turn(ax, r0 + t, i - t * half);
        }
    __syncthreads();
    const int sub = threadIdx.x % LPH, e0 = sub * 8;
    for (int item = threadIdx.x / LPH; item < (c.kv_heads << log_tb); item += 256 / LPH) {
        const int t = item & (tb - 1), head = item >> log_tb;
        const long base = at_row[t];
        const bool has = base >= 0 && e0 < c.hd;
        float fk[8] = {}, fv[8] = {};
        if (has) {
            const T* kr = k + (r0 + t) * ldk + (long)head * c.hd;
            if (ROT == ROT_NONE) {
                load_f32<T, 8>(kr + e0, fk);
            } else {
                rotated4<T, ROT == ROT_ADJ>(kr, e0, half, cs + t * half, fk);
                rotated4<T, ROT == ROT_ADJ>(kr, e0 + 4, half, cs + t * half, fk + 4);
            }
            load_f32<T, 8>(v + (r0 + t) * ldv + (long)head * c.hd + e0, fv);
        }
        unsigned ak = 0, av = 0;             // magnitudes as bits: they order as integers do, with NaN above infinity
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            ak = max(ak, __float_as_uint(fk[i]) & 0x7fffffffu);
            av = max(av, __float_as_uint(fv[i]) & 0x7fffffffu);
        }
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) {
            ak = max(ak, (unsigned)__shfl_xor((int)ak, o));
            av = max(av, (unsigned)__shfl_xor((int)av, o));
        }
        const int bk = exponent_byte(ak, format), bv = exponent_byte(av, format);
        if (base < 0 || e0 >= c.row_bytes) continue;
        const long row = base + (long)head * c.page_size;
        *reinterpret_cast<u32x2*>(c.k + row * c.row_bytes + e0) = encode8(fk, bk, format);
        *reinterpret_cast<u32x2*>(c.v + row * c.row_bytes + e0) = encode8(fv, bv, format);
        if (sub == 0) {
            c.k_exp[row] = (uint8_t)bk;
            c.v_exp[row] = (uint8_t)bv;
        }
    }
}

template <typename T, int LPH>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheDims c, const long* __restrict__ slots, T* __restrict__ k, T* __restrict__ v, long rows,
                                                         long ldk, long ldv, int log_tb, int format) {
    __shared__ long at_row[32];
    const int tb = 1 << log_tb;
    const long r0 = (long)blockIdx.x << log_tb;
    const int nt = (int)min((long)tb, rows - r0);
    if ((int)threadIdx.x < tb) at_row[threadIdx.x] = (int)threadIdx.x < nt ? plane_row(c, slots[r0 + threadIdx.x]) : -1;
    __syncthreads();
    const int e0 = (threadIdx.x % LPH) * 8;
    if (e0 >= c.hd) return;
    for (int item = threadIdx.x / LPH; item < (c.kv_heads << log_tb); item += 256 / LPH) {
        const int t = item & (tb - 1), head = item >> log_tb;
        const long base = at_row[t];
        if (base < 0) continue;
        const long row = base + (long)head * c.page_size;
        float f[8];
        decode8(*reinterpret_cast<const u32x2*>(c.k + row * c.row_bytes + e0), c.k_exp[row], format, f);
        store_f32<T, 8>(k + (r0 + t) * ldk + (long)head * c.hd + e0, f);
        decode8(*reinterpret_cast<const u32x2*>(c.v + row * c.row_bytes + e0), c.v_exp[row], format, f);
        store_f32<T, 8>(v + (r0 + t) * ldv + (long)head * c.hd + e0, f);
    }
}

int axes_check(const void* pos, const double* freq, int n_t, int n_h, int n_w, int pairing, int hd) {
    if (!pos || !freq || n_t < 0 || n_h < 0 || n_w < 0) return VDA_EINVAL;
    if (pairing != VDA_PAIR_HALVES && pairing != VDA_PAIR_ADJACENT) return VDA_EINVAL;
    const long half = (long)n_t + n_h + n_w;
    if (half <= 0 || half % 4 != 0 || 2 * half > hd) return VDA_ESHAPE;
    return VDA_OK;
}
bool known_type(int t) { return t == VDA_T_F32 || t == VDA_T_BF16 || t == VDA_T_F16; }
bool aligned(const void* p, long ld, int bytes, int size) { return ((uintptr_t)p & (bytes - 1)) == 0 && (ld * size) % bytes == 0; }

// Tokens per workgroup: as many as give every CU several workgroups, at most `most` (a power of two)
int log_tokens(long rows, int most) {
    int l = 0;
    while ((1 << (l + 1)) <= most && (rows >> (l + 1)) >= 1024) ++l;
    return l;
}

template <typename T>
int launch_rotary(const T* x, T* out, const Axes& ax, long rows, long ldx, long ldo, int heads, int hd, int pairing, hipStream_t st) {
    const bool in_place = x == out && ldx == ldo;
    const bool wide = sizeof(T) == 2 && pairing == VDA_PAIR_HALVES && ax.half % 8 == 0 && aligned(x, ldx, 16, 2) && aligned(out, ldo, 16, 2);
    const int need = sizeof(T) == 2 ? (pairing == VDA_PAIR_HALVES && in_place ? 8 : 16) : 16;
    if (!wide && (!aligned(x, ldx, need, sizeof(T)) || !aligned(out, ldo, need, sizeof(T)))) return VDA_ESHAPE;
    const int copies = in_place ? 0 : (hd - 2 * ax.half) / (sizeof(T) == 2 ? 8 : 4);
    const int tb = 1 << log_tokens(rows, 16);
    const long grid = (rows + tb - 1) / tb;
    if (grid > 0x7fffffffL) return VDA_ESHAPE;
    const size_t lds = (size_t)tb * ax.half * sizeof(float2);
#define VDA_ROT(U, ADJ) hipLaunchKernelGGL((rotary_kernel<T, U, ADJ>), dim3(grid), dim3(256), lds, st, x, out, ax, rows, ldx, ldo, heads, hd, tb, copies)
    if (pairing == VDA_PAIR_ADJACENT) VDA_ROT(4, true);
    else if (wide) VDA_ROT(8, false);
    else VDA_ROT(4, false);
#undef VDA_ROT
    return hip_rc(hipGetLastError());
}

CacheDims dims_of(const VdaTokenCache* c) {
    return CacheDims{(uint8_t*)c->k, (uint8_t*)c->v, c->k_exp, c->v_exp, c->page_size, c->kv_heads, c->hd, cache_row_bytes(c->hd),
                     (long)c->pages * c->page_size};
}
int log_lanes(int hd) {
    const int lanes = cache_row_bytes(hd) / 8;
    return lanes <= 2 ? 1 : lanes <= 4 ? 2 : lanes <= 8 ? 3 : 4;
}

}  // namespace

extern "C" int vda_rotary_axes(const void* x, void* out, const void* pos, const double* freq, long rows, int heads, int hd, long ldx, long ldo,
                               int n_t, int n_h, int n_w, int pairing, int pos_float, int dtype, void* stream) {
    if (!x || !out || rows <= 0 || heads <= 0 || hd <= 0 || !known_type(dtype)) return VDA_EINVAL;
    if (const int rc = axes_check(pos, freq, n_t, n_h, n_w, pairing, hd)) return rc;
    if (x == out && ldx != ldo) return VDA_EINVAL;
    if (hd % 8 != 0 || hd > 256 || heads > 65536 || rows > (1L << 40) || ldx < (long)heads * hd || ldo < (long)heads * hd) return VDA_ESHAPE;
    const Axes ax{pos, freq, n_t + n_h + n_w, n_t, n_t + n_h, pos_float};
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (dtype == VDA_T_BF16) return launch_rotary((const bf16*)x, (bf16*)out, ax, rows, ldx, ldo, heads, hd, pairing, st);
    if (dtype == VDA_T_F16) return launch_rotary((const f16*)x, (f16*)out, ax, rows, ldx, ldo, heads, hd, pairing, st);
    return launch_rotary((const float*)x, (float*)out, ax, rows, ldx, ldo, heads, hd, pairing, st);
}

extern "C" int vda_cache_write(const VdaTokenCache* cache, const void* k, const void* v, const int64_t* slots, long rows, long ldk, long ldv,
                               int dtype, const void* pos, const double* freq, int n_t, int n_h, int n_w, int pairing, int pos_float, void* stream) {
    if (const int rc = cache_check(cache)) return rc;
    if (!k || !v || !slots || rows <= 0 || !known_type(dtype) || (!pos != !freq)) return VDA_EINVAL;
    if (rows > (1L << 40)) return VDA_ESHAPE;
    if (pos)
        if (const int rc = axes_check(pos, freq, n_t, n_h, n_w, pairing, cache->hd)) return rc;
    const int size = dtype == VDA_T_F32 ? 4 : 2;
    const long width = (long)cache->kv_heads * cache->hd;
    if (ldk < width || ldv < width || !aligned(k, ldk, 16, size) || !aligned(v, ldv, 16, size)) return VDA_ESHAPE;
    const Axes ax{pos, freq, pos ? n_t + n_h + n_w : 0, n_t, n_t + n_h, pos_float};
    const int log_tb = log_tokens(rows, 32);
    const long grid = (rows + (1L << log_tb) - 1) >> log_tb;
    if (grid > 0x7fffffffL) return VDA_ESHAPE;
    const size_t lds = ((size_t)ax.half << log_tb) * sizeof(float2);
    const int rot = !pos ? ROT_NONE : pairing == VDA_PAIR_HALVES ? ROT_HALVES : ROT_ADJ;
    const CacheDims c = dims_of(cache);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
#define VDA_CW3(T, L, R) hipLaunchKernelGGL((cache_write_kernel<T, L, R>), dim3(grid), dim3(256), lds, st, (const T*)k, (const T*)v, c, (const long*)slots, \
                                            ax, rows, ldk, ldv, log_tb, cache->format)
#define VDA_CW2(T, L) do { if (rot == ROT_NONE) VDA_CW3(T, L, ROT_NONE); else if (rot == ROT_HALVES) VDA_CW3(T, L, ROT_HALVES); else VDA_CW3(T, L, ROT_ADJ); } while (0)
#define VDA_CW(T) do { switch (log_lanes(cache->hd)) { case 1: VDA_CW2(T, 2); break; case 2: VDA_CW2(T, 4); break; case 3: VDA_CW2(T, 8); break; \
                       default: VDA_CW2(T, 16); } } while (0)
    if (dtype == VDA_T_BF16) VDA_CW(bf16);
    else if (dtype == VDA_T_F16) VDA_CW(f16);
    else VDA_CW(float);
#undef VDA_CW
#undef VDA_CW2
#undef VDA_CW3
    return hip_rc(hipGetLastError());
}

extern "C" int vda_cache_read(const VdaTokenCache* cache, const int64_t* slots, void* k, void* v, long rows, long ldk, long ldv, int dtype,
                              void* stream) {
    if (const int rc = cache_check(cache)) return rc;
    if (!k || !v || !slots || rows <= 0 || !known_type(dtype)) return VDA_EINVAL;
    if (rows > (1L << 40)) return VDA_ESHAPE;
    const int size = dtype == VDA_T_F32 ? 4 : 2;
    const long width = (long)cache->kv_heads * cache->hd;
    if (ldk < width || ldv < width || !aligned(k, ldk, 16, size) || !aligned(v, ldv, 16, size)) return VDA_ESHAPE;
    const int log_tb = log_tokens(rows, 32);
    const long grid = (rows + (1L << log_tb) - 1) >> log_tb;
    if (grid > 0x7fffffffL) return VDA_ESHAPE;
    const CacheDims c = dims_of(cache);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
#define VDA_CR2(T, L) hipLaunchKernelGGL((cache_read_kernel<T, L>), dim3(grid), dim3(256), 0, st, c, (const long*)slots, (T*)k, (T*)v, rows, ldk, ldv, \
                                         log_tb, cache->format)
#define VDA_CR(T) do { switch (log_lanes(cache->hd)) { case 1: VDA_CR2(T, 2); break; case 2: VDA_CR2(T, 4); break; case 3: VDA_CR2(T, 8); break; \
                       default: VDA_CR2(T, 16); } } while (0)
    if (dtype == VDA_T_BF16) VDA_CR(bf16);
    else if (dtype == VDA_T_F16) VDA_CR(f16);
    else VDA_CR(float);
#undef VDA_CR
#undef VDA_CR2
    return hip_rc(hipGetLastError());
}
