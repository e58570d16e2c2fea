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
    Quick by_half;
};
__device__ __forceinline__ float2 turn(const Axes& a, long row, int j) {
    const int axis = j < a.end_t ? 0 : j < a.end_h ? 1 : 2;
    const long at = row * 3 + axis;
    const double p = a.pos_float ? (double)reinterpret_cast<const float*>(a.pos)[at] : (double)reinterpret_cast<const int*>(a.pos)[at];
    double rev = p * a.freq[j] * 0.15915494309189533577;
    rev -= rint(rev);
    const float f = (float)(2.0 * rev);                           // in half turns; what its rounding leaves out turns the result a little further
    const float d = (float)((2.0 * rev - (double)f) * 3.14159265358979323846);
    float2 cs;
    sincospif(f, &cs.y, &cs.x);
    return float2{fmaf(-cs.y, d, cs.x), fmaf(cs.x, d, cs.y)};
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

// A workgroup turns `tb` tokens: first the angles of their tb * half pairs into LDS, then the rows, each thread keeping one piece of the
// row (or several 256 apart) and walking down the tokens, so that no address is divided out.
struct RotaryShape {
    long rows, ldx, ldo;
    int heads, hd, tb, per_head, far;       // pieces of a head; line form: lanes between the two channels of a pair
    Quick by_row, by_head;                  // pieces of a row, of a head
};
struct Walk {
    int piece, t, side;                     // first piece of this thread, first token, tokens side by side
};
__device__ __forceinline__ bool walk(const RotaryShape& s, Walk& w) {
    const int per_row = s.heads * s.per_head, tid = threadIdx.x;
    w = Walk{tid, 0, 1};
    if (per_row < 256) {
        w.side = s.by_row.over(256);
        w.t = s.by_row.over(tid);
        w.piece = tid - w.t * per_row;
    }
    return w.t < w.side;
}
__device__ __forceinline__ void angles(float2* cs, const Axes& ax, long r0, int nt) {
    for (int i = threadIdx.x; i < nt * ax.half; i += 256) {
        const int t = ax.by_half.over(i);
        cs[i] = turn(ax, r0 + t, i - t * ax.half);
    }
    __syncthreads();
}

// Line form: a lane moves 16 bytes of the row, neighbours moving neighbouring ones, and takes the other channels of its pairs from the
// lane `far` away (a power of two: both lie in one group of 2 far lanes, which hold one head's pieces or a part of them).  Reading
// both halves of a head in one thread instead touches every cache line twice, by halves: 101 against 75 us for q and k of 32
// frames of 1370 tokens (16 heads of 64, 16-bit, 359 MB moved: 4.8 TB/s).  All lanes of a group load before any of them stores: the call may be in place.
template <typename T, bool ADJ>
__global__ __launch_bounds__(256) void rotary_line_kernel(const T* x, T* out, Axes ax, RotaryShape s) {
    extern __shared__ float2 cs[];
    constexpr int N = 16 / sizeof(T);
    const long r0 = (long)blockIdx.x * s.tb;
    const int nt = (int)min((long)s.tb, s.rows - r0), half = ax.half;
    angles(cs, ax, r0, nt);
    Walk w;
    if (!walk(s, w)) return;
    for (int c = w.piece; c < s.heads * s.per_head; c += 256) {
        const int head = s.by_head.over(c), e0 = (c - head * s.per_head) * N;                   // first channel of the piece in its head
        const bool turned = e0 < 2 * half, second = e0 >= half;
        const T* xr = x + (r0 + w.t) * s.ldx + (long)c * N;
        T* yr = out + (r0 + w.t) * s.ldo + (long)c * N;
        const float2* a = cs + w.t * half + (ADJ ? e0 >> 1 : second ? e0 - half : e0);
        for (int t = w.t; t < nt; t += w.side) {
            const Pack<T, N> own = *reinterpret_cast<const Pack<T, N>*>(xr);
            Pack<T, N> res = own;
            if constexpr (ADJ) {
                if (turned) {
#pragma unroll
                    for (int k = 0; k < N; k += 2) {
                        const float p = (float)own.v[k], q = (float)own.v[k + 1];
                        res.v[k] = (T)(p * a[k >> 1].x - q * a[k >> 1].y);
                        res.v[k + 1] = (T)(q * a[k >> 1].x + p * a[k >> 1].y);
                    }
                }
            } else {
                const u32x4 mine = __builtin_bit_cast(u32x4, own);
                u32x4 their;
#pragma unroll
                for (int k = 0; k < 4; ++k) their[k] = (unsigned)__shfl_xor((int)mine[k], s.far);
                const Pack<T, N> other = __builtin_bit_cast(Pack<T, N>, their);
                if (turned) {
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        const float p = (float)own.v[k], q = (float)other.v[k];
                        res.v[k] = (T)(p * a[k].x + (second ? q : -q) * a[k].y);
                    }
                }
            }
            *reinterpret_cast<Pack<T, N>*>(yr) = res;
            xr += w.side * s.ldx;
            yr += w.side * s.ldo;
            a += w.side * half;
        }
    }
}

// The general form, for pairs in halves whose distance is no power of two pieces, and rows that are only 8-byte aligned: a
// thread holds four pairs, or CU channels that are only copied.  q and k of 32 x 1370 tokens, 16 + 16 heads of 64 of which 48 channels
// turn: 103 us in bf16 (3.5 TB/s), 202 in fp32, where the line form takes 75 and 147 for whole heads; 20 heads of 96, all of it, 77 and 139.
template <typename T>
__global__ __launch_bounds__(256) void rotary_pairs_kernel(const T* x, T* out, Axes ax, RotaryShape s) {
    extern __shared__ float2 cs[];
    constexpr int CU = sizeof(T) == 2 ? 8 : 4;
    const long r0 = (long)blockIdx.x * s.tb;
    const int nt = (int)min((long)s.tb, s.rows - r0), half = ax.half, units = half / 4;
    angles(cs, ax, r0, nt);
    Walk w;
    if (!walk(s, w)) return;
    for (int c = w.piece; c < s.heads * s.per_head; c += 256) {
        const int head = s.by_head.over(c), u = c - head * s.per_head;
        const bool copy = u >= units;
        const int at = head * s.hd + (copy ? 2 * half + (u - units) * CU : 4 * u);
        const T* xr = x + (r0 + w.t) * s.ldx + at;
        T* yr = out + (r0 + w.t) * s.ldo + at;
        const float2* a = cs + w.t * half + 4 * u;
        for (int t = w.t; t < nt; t += w.side) {
            if (copy) {
                *reinterpret_cast<Pack<T, CU>*>(yr) = *reinterpret_cast<const Pack<T, CU>*>(xr);
            } else {
                float p[4], q[4], y[4], z[4];
                load_f32<T, 4>(xr, p);
                load_f32<T, 4>(xr + half, q);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    y[k] = p[k] * a[k].x - q[k] * a[k].y;
                    z[k] = q[k] * a[k].x + p[k] * a[k].y;
                }
                store_f32<T, 4>(yr, y);
                store_f32<T, 4>(yr + half, z);
            }
            xr += w.side * s.ldx;
            yr += w.side * s.ldo;
            a += w.side * half;
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
    return max(1, e);                                              // 0 marks an empty slot; 249 at most (254 - 6 + 1)
}
__device__ __forceinline__ u32x2 encode8(const float* f, int byte, int format) {
    u32x2 c = {0u, 0u};
    if (byte == 255) return c;
    const float s = __uint_as_float((unsigned)(254 - byte) << 23);      // 2^(127 - byte)
    if (format == VDA_CACHE_I8) {
        // on 1.5 * 2^23 a unit in the last place is 1: the sum's one rounding, to nearest even, leaves the code in the low byte
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            unsigned w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(fmaf(f[4 * k + i], s, 12582912.f));
            c[k] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(w[3], w[2], 0x0c0c0400u), __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0400u), 0x05040100u);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k] * s, f[4 * k + 1] * s, 0, false);
            c[k] = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k + 2] * s, f[4 * k + 3] * s, w, true);
        }
    }
    return c;
}
__device__ __forceinline__ void decode8(u32x2 c, int byte, int format, float* f) {
    // 2^(byte - 127); an empty slot's factor is 0, a lost row's NaN (times any code)
    const float s = byte == 255 ? __builtin_nanf("") : __uint_as_float((unsigned)byte << 23);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (format == VDA_CACHE_I8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[4 * k + i] = (float)(int)(signed char)(c[k] >> (8 * i));
        } else {
            if (byte == 0) c[k] = 0;                                // (an empty slot may hold e4m3's NaN)
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(c[k], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c[k], true);
            f[4 * k] = lo[0]; f[4 * k + 1] = lo[1]; f[4 * k + 2] = hi[0]; f[4 * k + 3] = hi[1];
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = byte == 0 ? 0.f : f[k] * s;
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
// ROT_LINE takes the other channels of the pairs from the lane `far` away, as rotary_line_kernel does; ROT_HALVES reads them (eight
// frames of 1370 tokens written and read, 16 heads of 64: 39.7 us when all halves were read, 32.3 by lanes).  That writer moves 68 MB
// in 16.5 us and the reader as much in 12.4: 4.1 and 5.4 TB/s.
enum { ROT_NONE = 0, ROT_HALVES = 1, ROT_ADJ = 2, ROT_LINE = 3 };
template <typename T, int LPH, int ROT>
__global__ __launch_bounds__(256) void cache_write_kernel(const T* __restrict__ k, const T* __restrict__ v, CacheDims c, const long* __restrict__ slots,
                                                          Axes ax, long rows, long ldk, long ldv, int log_tb, int format, int far) {
    extern __shared__ float2 cs[];
    __shared__ long at_row[32];
    const int tb = 1 << log_tb;
    const long r0 = (long)blockIdx.x << log_tb;
    const int nt = (int)min((long)tb, rows - r0), half = ax.half;
    const int sub = threadIdx.x % LPH, e0 = sub * 8, items = c.kv_heads << log_tb;
    // the rows of the next (head, token) are in flight while one is stored, the first ones while the angles are formed
    Pack<T, 8> k_next = {}, v_next = {};
    auto fetch = [&](int item) {
        const int t = item & (tb - 1), head = item >> log_tb;
        if (item < items && t < nt && e0 < c.hd) {
            k_next = *reinterpret_cast<const Pack<T, 8>*>(k + (r0 + t) * ldk + (long)head * c.hd + e0);
            v_next = *reinterpret_cast<const Pack<T, 8>*>(v + (r0 + t) * ldv + (long)head * c.hd + e0);
        }
    };
    fetch(threadIdx.x / LPH);
    if ((int)threadIdx.x < tb) at_row[threadIdx.x] = (int)threadIdx.x < nt ? plane_row(c, slots[r0 + threadIdx.x]) : -1;
    if (ROT != ROT_NONE) angles(cs, ax, r0, nt);                   // (ends with a barrier)
    else __syncthreads();
    for (int item = threadIdx.x / LPH; item < items; item += 256 / LPH) {
        const int t = item & (tb - 1), head = item >> log_tb;
        const long base = at_row[t];
        float fk[8], fv[8];
        Pack<T, 8> far_k = k_next;
#pragma unroll
        for (int i = 0; i < 8; ++i) { fk[i] = (float)k_next.v[i]; fv[i] = (float)v_next.v[i]; }
        fetch(item + 256 / LPH);
        if (ROT == ROT_HALVES || ROT == ROT_ADJ) {
            if (t < nt && e0 < c.hd) {
                const T* kr = k + (r0 + t) * ldk + (long)head * c.hd;
                rotated4<T, ROT == ROT_ADJ>(kr, e0, half, cs + t * half, fk);
                rotated4<T, ROT == ROT_ADJ>(kr, e0 + 4, half, cs + t * half, fk + 4);
            }
        }
        if constexpr (ROT == ROT_LINE) {
            const bool second = e0 >= half;
            const float2* w = cs + t * half + (e0 < 2 * half ? (second ? e0 - half : e0) : 0);
            float y[8];
            struct Words { int w[2 * sizeof(T)]; } words = __builtin_bit_cast(Words, far_k);
#pragma unroll
            for (unsigned i = 0; i < 2 * sizeof(T); ++i) words.w[i] = __shfl_xor(words.w[i], far);
            far_k = __builtin_bit_cast(Pack<T, 8>, words);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float q = (float)far_k.v[i];
                y[i] = fk[i] * w[i].x + (second ? q : -q) * w[i].y;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) fk[i] = e0 < 2 * half ? y[i] : fk[i];
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
    constexpr int size = sizeof(T), N = 16 / size;
    const bool in_place = x == out, adjacent = pairing == VDA_PAIR_ADJACENT, wide = aligned(x, ldx, 16, size) && aligned(out, ldo, 16, size);
    const int far = ax.half / N;                                  // pieces between the channels of a pair
    const bool line = wide && (adjacent || (ax.half % N == 0 && (far & (far - 1)) == 0 && far <= 32 && (hd / N) % (2 * far) == 0));
    if (!wide && (size == 4 || adjacent || !in_place || !aligned(x, ldx, 8, size))) return VDA_ESHAPE;
    const int tb = 1 << log_tokens(rows, 16);
    const long grid = (rows + tb - 1) / tb;
    if (grid > 0x7fffffffL) return VDA_ESHAPE;
    const size_t lds = (size_t)tb * ax.half * sizeof(float2);
    const int per_head = line ? hd / N : ax.half / 4 + (in_place ? 0 : (hd - 2 * ax.half) / (size == 2 ? 8 : 4));
    const RotaryShape s{rows, ldx, ldo, heads, hd, tb, per_head, far, Quick(per_head * heads), Quick(per_head)};
    if (line && adjacent) hipLaunchKernelGGL((rotary_line_kernel<T, true>), dim3(grid), dim3(256), lds, st, x, out, ax, s);
    else if (line) hipLaunchKernelGGL((rotary_line_kernel<T, false>), dim3(grid), dim3(256), lds, st, x, out, ax, s);
    else hipLaunchKernelGGL((rotary_pairs_kernel<T>), dim3(grid), dim3(256), lds, st, x, out, ax, s);
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
    const Axes ax{pos, freq, n_t + n_h + n_w, n_t, n_t + n_h, pos_float, Quick(n_t + n_h + n_w)};
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
    const Axes ax{pos, freq, pos ? n_t + n_h + n_w : 0, n_t, n_t + n_h, pos_float, Quick(pos ? n_t + n_h + n_w : 1)};
    const int log_tb = log_tokens(rows, 32);
    const long grid = (rows + (1L << log_tb) - 1) >> log_tb;
    if (grid > 0x7fffffffL) return VDA_ESHAPE;
    const size_t lds = ((size_t)ax.half << log_tb) * sizeof(float2);
    const int far = ax.half / 8;
    const bool line = pos && ax.half % 8 == 0 && (far & (far - 1)) == 0 && (cache->hd / 8) % (2 * far) == 0;
    const int rot = !pos ? ROT_NONE : pairing == VDA_PAIR_ADJACENT ? ROT_ADJ : line ? ROT_LINE : ROT_HALVES;
    const CacheDims c = dims_of(cache);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
#define VDA_CW3(T, L, R) hipLaunchKernelGGL((cache_write_kernel<T, L, R>), dim3(grid), dim3(256), lds, st, (const T*)k, (const T*)v, c, (const long*)slots, \
                                            ax, rows, ldk, ldv, log_tb, cache->format, far)
#define VDA_CW2(T, L) do { if (rot == ROT_NONE) VDA_CW3(T, L, ROT_NONE); else if (rot == ROT_HALVES) VDA_CW3(T, L, ROT_HALVES); \
                           else if (rot == ROT_ADJ) VDA_CW3(T, L, ROT_ADJ); else VDA_CW3(T, L, ROT_LINE); } while (0)
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
