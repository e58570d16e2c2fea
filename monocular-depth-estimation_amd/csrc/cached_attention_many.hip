// Attention over the token cache for many query rows per key head (the tokens of a frame).
//
// One workgroup = 4 waves = 128 query rows of one (sequence, key head), 32 for each wave; tiles of 64 keys.  The codes of the next tile
// go from global memory to registers while this tile is multiplied, become IEEE halves times the power of two of their row, and
// are stored in LDS once for the four waves, in a second buffer: one barrier per tile.  Scores are S^T = K Q^T (mfma 32x32x16), so a
// query lives on a lane, the softmax needs one exchange (lane ^ 32) and only where a maximum grows, and the probabilities
// are as they stand the B operand of O^T += V^T P^T, whose V^T operand the transposed LDS read gathers in the same key order.
// What it spends its time on are vector instructions: about five per score, one of them the exponential, against two matrix
// instructions of 32 cycles per 1024 scores and 16 channels.  The 1370 tokens of a frame over 32 frames, 16 heads of 64: 382 us
// (433 where the clock is lower), 0.65 PFLOP/s, where a large library product of the type reaches 1.2.  Counters: a SIMD issues vector
// instructions in 55 % of the cycles and its matrix pipe works in 27 %; of the 2.1 waves that it holds on average each waits for
// memory or the barrier for 26 % of its time and for its turn to issue for 32 %.  A fourth wave per SIMD (32 keys per tile) gained nothing: 388 against 381 us.  Within a wave, the scores of one half of the
// tile formed between the exponentials of the other: 1 % less here, 3 % more for three clips of 5 x 380 tokens, not kept; the
// scores of the next tile between them: 204 registers, two waves, 607 us.  64 rows per wave: slower.
//
// Rows of the cache carry powers of two of any size, halves do not.  Where the exponents of a part's keys lie close enough together, and
// those of its values, tiles hold halves relative to the largest of each: the smallest and the largest are found by a pass over the
// exponent bytes (a 33rd of the codes' bytes) before the first tile.  Powers of two leave no trace in such products, so it does not
// matter whose the largest was.  Elsewhere a workgroup takes the form of single exponents, as the kernel for few rows does: tiles hold the
// codes as they are, a key's power of two multiplies its scores, and a value's is part of the exponent that becomes the probability,
// so that a row is taken relative to its own largest sum of score and value exponent, whatever others see.  With a value row of zeros
// in every part, which makes it so, the frame over 32 frames takes 21 % longer, clips 12 %.
#include "cached_attention.h"

#include <type_traits>

namespace {

constexpr int TK = 64;                                            // keys of a tile
// Spreads of exponents that common references take.  Keys: codes stay exact, the smallest one times 2^-32 (e4m3: 2^-21) and the shift of
// scaled16 being a half, 2^-24 at least.  Values: probabilities are halves down to 2^-33 of the row's largest, which is 2^-25 of it on
// a value 2^8 larger than another.
template <int FMT> constexpr int key_spread() { return FMT == VDA_CACHE_I8 ? 32 : 21; }
constexpr int VALUE_SPREAD = 8;
constexpr int V_MIN = 40;            // smaller value exponents count as this where they are part of a reference (see V_REF_MIN in the kernel for few rows)

__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// byte offset of 16-byte chunk `chunk` of key `row` in the K tile [64][HDP] of halves: the sixteen rows that are read together fall
// into the sixteen slots of a 256-byte bank row
template <int HDP>
__device__ __forceinline__ int ktile(int row, int chunk) {
    const int swz = HDP == 64 ? (row >> 1) & 7 : HDP == 128 ? row & 15 : (row >> 2) & 3;
    return row * (2 * HDP) + ((chunk ^ swz) << 4);
}
// byte offset of (key, byte column) in the V tile: four rows' 64-byte pieces, read transposed together, fall into different banks
template <int HDP>
__device__ __forceinline__ int vtile(int row, int col) {
    const int swz = HDP == 64 ? ((row >> 1) & 1) << 6 : HDP == 128 ? (row & 3) << 6 : 0;
    return row * (2 * HDP) + (col ^ swz);
}

// Sixteen codes times 2^e as halves; e <= 8, below -24 the factor is 0 for integers.
template <int FMT>
__device__ __forceinline__ void scaled16(u32x4 w, int e, f16x8& lo, f16x8& hi) {
    f16x2 h[8];
    if (FMT == VDA_CACHE_I8) {
        const f16 s = (f16)__builtin_amdgcn_ldexpf(1.f, e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            codes4<FMT>(w[i], h[2 * i], h[2 * i + 1]);
            h[2 * i] *= f16x2{s, s};
            h[2 * i + 1] *= f16x2{s, s};
        }
    } else {
        const float s = __builtin_amdgcn_ldexpf(1.f, e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h[2 * i] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], s, false));
            h[2 * i + 1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], s, true));
        }
    }
    lo = f16x8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
    hi = f16x8{h[4][0], h[4][1], h[5][0], h[5][1], h[6][0], h[6][1], h[7][0], h[7][1]};
}

// Waves per SIMD that the registers allow without spilling.
template <typename T, int HDP> constexpr int many_waves() { return HDP <= 64 ? 3 : HDP == 128 && Pieces<T>::n == 2 ? 1 : 2; }

// (out may be q: each row's queries are read by the workgroup that writes it, before it writes)
template <typename T, int HDP, int FMT>
__global__ __launch_bounds__(256, (many_waves<T, HDP>())) void attend_many_kernel(const T* q, T* out, AttendJob j, int max_q, int groups) {
    constexpr int NP = Pieces<T>::n, KS = HDP / 16, DB = HDP / 32, CPR = HDP / 16, NC = (HDP + 63) / 64, SHIFT = FMT == VDA_CACHE_I8 ? 8 : 6;
    constexpr int PLANE = TK * HDP * 2, BUF = 2 * PLANE;
    __shared__ __attribute__((aligned(16))) char smem[2 * BUF];
    __shared__ uint8_t hide[2][TK];
    // of the keys of a tile of single exponents: a key's power of two, a value's exponent less 127, the power of two that undoes it
    __shared__ __attribute__((aligned(16))) float single[2][3][TK];
    __shared__ int wave_top[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    // row blocks of one (sequence, key head, split) follow each other on one XCD and share its copy of the keys
    const int id = xcd_contiguous(blockIdx.x, groups);
    const int t0 = j.by_blocks.over(id), rb = id - t0 * j.row_blocks, t1 = j.by_splits.over(t0), split = t0 - t1 * j.splits;
    const int s = j.by_heads.over(t1), kvh = t1 - s * j.kv_heads;
    const Span sp = span_of(j, s, max_q);
    const int n_rho = sp.nq * j.group;
    if (rb * 128 >= n_rho || split * j.chunk >= max(sp.n, 1)) return;      // the whole workgroup
    const int rho = rb * 128 + wave * 32 + r, token = j.by_group.over(rho), head = kvh * j.group + (rho - token * j.group);
    const bool live = rho < n_rho;
    const long row = sp.q0 + (live ? token : 0);

    // keys that a row, the wave's rows, the workgroup's rows see
    int limit = live ? sp.n : 0, least = live ? sp.n : 0x7fffffff, most;
    if (j.visible && live) limit = least = max(0, min(limit, j.visible[row]));
    most = limit;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        most = max(most, __shfl_xor(most, o));
        least = min(least, __shfl_xor(least, o));
    }
    if (lane == 0) wave_top[wave] = most;
    least = __builtin_amdgcn_readfirstlane(least);
    __syncthreads();
    most = __builtin_amdgcn_readfirstlane(max(max(wave_top[0], wave_top[1]), max(wave_top[2], wave_top[3])));
    __syncthreads();
    const int k_begin = split * j.chunk, k_end = min(k_begin + j.chunk, most);

    const int* table = j.page_table + (long)s * j.max_pages;
    // the largest exponents of the part's keys and values
    int k_ref, v_ref;
    bool common;
    {
        int tk = 1, tv = 1, lk = 255, lv = 255;
        for (int b = (k_begin >> 4) + tid; b * 16 < k_end; b += 256) {
            const int key = b * 16, pi = j.by_page.over(key), page = table[pi];
            if (page < 0 || page >= j.pages) continue;
            const long at = ((long)page * j.kv_heads + kvh) * j.page_size + key - pi * j.page_size;
            const u32x4 e = *reinterpret_cast<const u32x4*>(j.k_exp + at), w = *reinterpret_cast<const u32x4*>(j.v_exp + at);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int be = (int)byte_of(e[i >> 2], i & 3), bw = (int)byte_of(w[i >> 2], i & 3);
                if (key + i < k_end && be != 0 && be != 255 && bw != 255) {
                    tk = max(tk, be);
                    tv = max(tv, bw);
                    lk = min(lk, be == 1 ? 255 : be);             // (keys of zeros are exact at any scale)
                    lv = min(lv, bw);
                }
            }
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            tk = max(tk, __shfl_xor(tk, o));
            tv = max(tv, __shfl_xor(tv, o));
            lk = min(lk, __shfl_xor(lk, o));
            lv = min(lv, __shfl_xor(lv, o));
        }
        if (lane == 0) { wave_top[wave] = tk; wave_top[4 + wave] = tv; wave_top[8 + wave] = lk; wave_top[12 + wave] = lv; }
        __syncthreads();
        k_ref = __builtin_amdgcn_readfirstlane(max(max(wave_top[0], wave_top[1]), max(wave_top[2], wave_top[3])));
        v_ref = __builtin_amdgcn_readfirstlane(max(max(wave_top[4], wave_top[5]), max(wave_top[6], wave_top[7])));
        lk = __builtin_amdgcn_readfirstlane(min(min(wave_top[8], wave_top[9]), min(wave_top[10], wave_top[11])));
        lv = __builtin_amdgcn_readfirstlane(min(min(wave_top[12], wave_top[13]), min(wave_top[14], wave_top[15])));
        common = k_ref - lk <= key_spread<FMT>() && v_ref - lv <= VALUE_SPREAD;
        if (!common) k_ref = v_ref = 127;
    }

    f16x8 qf[KS][NP];
    float c_row;                                                  // from products of halves to octaves
    {
        float f[KS][8], amax = 0.f;
        const T* qr = q + row * j.ldq + (long)head * j.hd;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const int e = 16 * i + 8 * h;
            query8<T>(qr + e, live && e < j.hd, f[i]);
#pragma unroll
            for (int x = 0; x < 8; ++x) amax = fmaxf(amax, fabsf(f[i][x]));
        }
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        const int shift = query_shift(amax);
#pragma unroll
        for (int i = 0; i < KS; ++i) query_pieces<NP>(f[i], shift, qf[i]);
        c_row = __builtin_amdgcn_ldexpf(j.scale_log2e, k_ref - 127 - SHIFT - shift);
    }

    // staging: wave w brings the sixteen keys 16 w .. 16 w + 15 of every tile, which lie in one page, part i of a lane being the codes
    // of one 16-byte chunk of one key (HDP 32: lanes 0 .. 31 bring K, the others V)
    int s_key[NC], s_col[NC], s_k[NC], s_v[NC];                   // key of the block, byte of its row, places in the K and V tiles
    bool s_on[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int idx = HDP == 32 ? lane & 31 : i * 64 + lane;
        s_on[i] = idx < 16 * CPR;
        s_key[i] = s_on[i] ? idx / CPR : 15;
        const int c = idx % CPR;
        s_col[i] = min(16 * c, j.row_bytes - 16);                 // padding channels meet zeros of q, or are not stored
        s_k[i] = ktile<HDP>(16 * wave + s_key[i], 2 * c);
        s_v[i] = PLANE + vtile<HDP>(16 * wave + s_key[i], 32 * c);
    }
    const bool do_k = HDP != 32 || lane < 32, do_v = HDP != 32 || lane >= 32;
    int pi = j.by_page.over(k_begin + 16 * wave), off = k_begin + 16 * wave - pi * j.page_size;
    const int step_pages = j.by_page.over(TK), step_off = TK - step_pages * j.page_size;
    // the page is asked for one tile ahead, from constant memory: a scalar load, which no other load has to be waited for
    typedef const int __attribute__((address_space(4)))* constant;
    const constant pages = (constant)table;
    int page = pages[min(pi, j.max_pages - 1)], k_next = k_begin + 16 * wave;
    u32x4 k_code[NC], v_code[NC];
    int k_exp[NC], v_exp[NC], in_block = 0;                       // in_block: keys of the block that are there
    auto fetch = [&]() {                                          // the next tile
        in_block = min(16, k_end - k_next);
        if (page < 0 || page >= j.pages) in_block = 0;
        const long a = in_block > 0 ? ((long)page * j.kv_heads + kvh) * j.page_size + off : 0L;      // (rows 0 .. 15 exist; they are read and not used)
        // (uniform: kept as scalar bases with 32-bit offsets, not summed into vector registers; global memory, said aloud, because a
        // pointer that passes through here otherwise becomes a flat one, whose loads the LDS waits would wait for)
        typedef const uint8_t __attribute__((address_space(1)))* global;
        global kr = (global)(j.k + a * j.row_bytes), vr = (global)(j.v + a * j.row_bytes), ke = (global)(j.k_exp + a), ve = (global)(j.v_exp + a);
        asm("" : "+s"(kr), "+s"(vr), "+s"(ke), "+s"(ve));
        typedef const u32x4 __attribute__((address_space(1)))* global16;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const unsigned o = s_key[i] * j.row_bytes + s_col[i];
            if (HDP == 32) {
                k_code[i] = v_code[i] = *(global16)((do_k ? kr : vr) + o);
            } else {
                k_code[i] = *(global16)(kr + o);
                v_code[i] = *(global16)(vr + o);
            }
            k_exp[i] = ke[(unsigned)s_key[i]];
            v_exp[i] = ve[(unsigned)s_key[i]];
        }
        pi += step_pages;
        off += step_off;
        if (off >= j.page_size) { off -= j.page_size; ++pi; }
        k_next += TK;
        page = pages[min(pi, j.max_pages - 1)];
    };
    auto store = [&](int buf, auto relative) {
        constexpr bool COMMON = decltype(relative)::value;
        char* b = smem + buf * BUF;
        bool odd = false;                                         // some key of the block is hidden or not a number
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (s_key[i] >= in_block) k_exp[i] = 0;
        }
#pragma unroll
        for (int i = 0; i < NC; ++i) odd |= k_exp[i] == 0 || k_exp[i] == 255 || v_exp[i] == 255;
        const bool any_odd = __builtin_amdgcn_ballot_w64(odd) != 0;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            f16x8 k_lo, k_hi, v_lo, v_hi;
            const int v_at = COMMON ? v_ref : max(v_exp[i], V_MIN);
            scaled16<FMT>(k_code[i], SHIFT + (COMMON ? k_exp[i] - k_ref : 0), k_lo, k_hi);
            scaled16<FMT>(v_code[i], SHIFT + v_exp[i] - v_at, v_lo, v_hi);
            if (do_k && s_on[i]) {
                *reinterpret_cast<f16x8*>(b + s_k[i]) = k_lo;
                *reinterpret_cast<f16x8*>(b + (s_k[i] ^ 16)) = k_hi;
            }
            if (do_v && s_on[i]) {
                *reinterpret_cast<f16x8*>(b + s_v[i]) = v_lo;     // (the V swizzle moves 64-byte pieces)
                *reinterpret_cast<f16x8*>(b + s_v[i] + 16) = v_hi;
            }
            if (any_odd && s_on[i]) {     // hidden: value 0 and a score that is not looked at; not a number: value 0, score NaN
                const bool nan = k_exp[i] == 255 || (v_exp[i] == 255 && k_exp[i] != 0);
                const f16 z = (f16)__builtin_nanf("");
                if (do_k && nan) {
                    *reinterpret_cast<f16x8*>(b + s_k[i]) = f16x8{z, z, z, z, z, z, z, z};
                    *reinterpret_cast<f16x8*>(b + (s_k[i] ^ 16)) = f16x8{z, z, z, z, z, z, z, z};
                }
                if (do_v && (nan || k_exp[i] == 0)) {
                    *reinterpret_cast<f16x8*>(b + s_v[i]) = f16x8{};
                    *reinterpret_cast<f16x8*>(b + s_v[i] + 16) = f16x8{};
                }
            }
            if (do_k && s_on[i] && s_col[i] == 0) {
                const int key = 16 * wave + s_key[i];
                hide[buf][key] = k_exp[i] == 0;
                if constexpr (!COMMON) {
                    single[buf][0][key] = __builtin_amdgcn_ldexpf(1.f, k_exp[i] - 127);
                    single[buf][1][key] = (float)(v_at - 127);
                    single[buf][2][key] = __builtin_amdgcn_ldexpf(1.f, 127 - v_at);
                }
            }
        }
    };

    // scores (of single exponents: plus the value's) are formed relative to their running maximum (0 until the row has seen a key: then it
    // moves there whatever its sign)
    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[i][x] = 0.f;
    float m_run = 0.f, l_run = 0.f;                               // l_run: of probabilities times 2^P_SHIFT
    bool unset = true;
    const int tq = (lane & 15) >> 2, tp = lane & 3, tcol = 2 * (16 * ((lane >> 4) & 1) + 4 * tp);

    auto walk = [&](auto relative) {
        constexpr bool COMMON = decltype(relative)::value;
        if (k_begin < k_end) {
            fetch();
            store(0, relative);
        }
        __syncthreads();
        int cur = 0;
        for (int k0 = k_begin; k0 < k_end; k0 += TK, cur ^= 1) {
            fetch();                                              // of the tile after this one, or of nothing
            const char* kb = smem + cur * BUF;
            const char* vb = kb + PLANE;
            const unsigned long hidden = __builtin_amdgcn_ballot_w64(hide[cur][lane] != 0);
            // 32 keys at a time: half the registers for scores and probabilities
            // (unrolled where the registers allow it without spilling: 3 waves per SIMD of 64 channels in two pieces)
            constexpr int UNROLL = COMMON && (NP == 1 || HDP != 64) ? 2 : 1;
#pragma unroll UNROLL
            for (int kh = 0; kh < 2; ++kh) {
                f32x16 sc;
#pragma unroll
                for (int x = 0; x < 16; ++x) sc[x] = 0.f;
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const f16x8 kf = *reinterpret_cast<const f16x8*>(kb + ktile<HDP>(32 * kh + r, 2 * i + h));
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) sc = mfma32(kf, qf[i][p], sc);
                }
                const unsigned gone = (unsigned)(kh ? hidden >> 32 : hidden);
                const float base = (float)P_SHIFT - m_run;
                const f32x4* mine4 = reinterpret_cast<const f32x4*>(&single[cur][0][32 * kh + 4 * h]);      // of this lane's keys: four at 0, 8, 16 and 24
                if constexpr (COMMON) {
#pragma unroll
                    for (int x = 0; x < 16; ++x) sc[x] = fmaf(sc[x], c_row, base);
                } else {
#pragma unroll
                    for (int x = 0; x < 16; ++x) sc[x] = fmaf(sc[x] * mine4[2 * (x >> 2)][x & 3], c_row, base + mine4[TK / 4 + 2 * (x >> 2)][x & 3]);
                }
                if (gone != 0 || k0 + 32 * kh + 32 > least) {
                    const unsigned mine = gone >> (4 * h);
                    const int left = limit - (k0 + 32 * kh + 4 * h);
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const int in32 = (x & 3) + 8 * (x >> 2);      // + 4 h
                        if ((mine >> in32 & 1) || in32 >= left) sc[x] = -INFINITY;
                    }
                }
                float mx = sc[0];
#pragma unroll
                for (int x = 1; x < 16; ++x) mx = fmaxf(mx, sc[x]);
                if (__builtin_amdgcn_ballot_w64(mx > DEFER + P_SHIFT || (unset && mx > -INFINITY)) != 0) {
                    mx = fmaxf(mx, __shfl_xor(mx, 32)) - P_SHIFT;
                    const float delta = !unset ? fmaxf(mx, 0.f) : mx == -INFINITY ? 0.f : mx, root = unset ? 1.f : __builtin_amdgcn_exp2f(-0.5f * delta), alpha = root * root;      // (in two steps: a value's exponent may have grown by more than 126)
                    unset = unset && mx == -INFINITY;
                    m_run += delta;
                    l_run = l_run * root * root;
#pragma unroll
                    for (int i = 0; i < DB; ++i)
#pragma unroll
                        for (int x = 0; x < 16; ++x) o[i][x] *= alpha;
#pragma unroll
                    for (int x = 0; x < 16; ++x) sc[x] -= delta;
                }
                float sum[2] = {0.f, 0.f};
                f16x8 pf[2][NP];
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const float p = __builtin_amdgcn_exp2f(sc[x]);
                    sum[x & 1] = COMMON ? sum[x & 1] + p : fmaf(p, mine4[2 * (TK / 4) + 2 * (x >> 2)][x & 3], sum[x & 1]);      // (without the value's exponent)
                    const f16 hi = (f16)p;                        // at most 2^(P_SHIFT + DEFER); rounded to 11 bits (22 in two pieces)
                    pf[x >> 3][0][x & 7] = hi;
                    if (NP == 2) pf[x >> 3][NP - 1][x & 7] = (f16)(p - (float)hi);
                }
                l_run += sum[0] + sum[1];
#pragma unroll
                for (int i = 0; i < DB; ++i)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int key = 32 * kh + 16 * x + 4 * h + tq;
                        const f16x4 lo = read_tr<f16>(vb + vtile<HDP>(key, 64 * i + tcol)), hi = read_tr<f16>(vb + vtile<HDP>(key + 8, 64 * i + tcol));
                        const f16x8 vf = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
                        for (int p2 = NP - 1; p2 >= 0; --p2) o[i] = mfma32(vf, pf[x][p2], o[i]);
                    }
            }
            store(cur ^ 1, relative);
            __syncthreads();
        }
    };
    if (common) walk(std::true_type{});
    else walk(std::false_type{});

    // lane (r, h) holds channels 32 i + 8 g + 4 h + 0..3 of query r in o[i][4 g + 0..3]
    const float l = l_run + __shfl_xor(l_run, 32);
    if (!live) return;
    if (j.splits > 1) {
        float* part = j.part + ((((long)s * j.row_blocks + rb) * j.kv_heads + kvh) * j.splits + split) * (128 * (HDP + 2));
        const int in_wg = wave * 32 + r;
        float* d = part + in_wg * HDP + 4 * h;
        // as the join expects them: outputs and sum relative to one power of two, which holds the value exponent; what its rounding leaves out
        // (a hundred thousandth) multiplies both
        const int v_in_m = max(v_ref, V_MIN);                     // (a smaller one would make the sum overflow)
        const float v = (float)v_in_m, m = unset ? LOWEST : m_run + v, v_in = m - m_run;
        const float left = unset ? 1.f : __builtin_amdgcn_exp2f((m_run - (m - v_in)) + (v - v_in));
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 y;
#pragma unroll
                for (int x = 0; x < 4; ++x) y[x] = __builtin_amdgcn_ldexpf(o[i][4 * g + x] * left, v_ref - v_in_m - SHIFT);
                *reinterpret_cast<f32x4*>(d + 32 * i + 8 * g) = y;
            }
        if (h == 0) {
            part[128 * HDP + in_wg] = m;
            part[128 * HDP + 128 + in_wg] = __builtin_amdgcn_ldexpf(l * left, 127 - v_in_m);
        }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* orow = out + row * j.ldo + (long)head * j.hd + 4 * h;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (32 * i + 8 * g >= j.hd) continue;
            typename Vec<T>::v4 v;
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] = (T)__builtin_amdgcn_ldexpf(o[i][4 * g + x] * inv, v_ref - 127 - SHIFT);
            *reinterpret_cast<typename Vec<T>::v4*>(orow + 32 * i + 8 * g) = v;
        }
}

template <typename T>
int many(const AttendJob& j, const T* q, T* out, int format, int max_q, hipStream_t st) {
    const int groups = j.seqs * j.kv_heads * j.row_blocks * j.splits;
#define VDA_M2(H, F) hipLaunchKernelGGL((attend_many_kernel<T, H, F>), dim3(groups), dim3(256), 0, st, q, out, j, max_q, groups)
#define VDA_M(H) do { if (format == VDA_CACHE_I8) VDA_M2(H, VDA_CACHE_I8); else VDA_M2(H, VDA_CACHE_E4M3); } while (0)
    if (j.hd <= 32) VDA_M(32);
    else if (j.hd <= 64) VDA_M(64);
    else if (j.hd <= 96) VDA_M(96);
    else VDA_M(128);
#undef VDA_M
#undef VDA_M2
    return hip_rc(hipGetLastError());
}

}  // namespace

int attend_many(const AttendJob& j, const void* q, void* out, int dtype, int format, int max_q, hipStream_t st) {
    if (dtype == VDA_T_BF16) return many(j, (const bf16*)q, (bf16*)out, format, max_q, st);
    if (dtype == VDA_T_F16) return many(j, (const f16*)q, (f16*)out, format, max_q, st);
    return many(j, (const float*)q, (float*)out, format, max_q, st);
}
