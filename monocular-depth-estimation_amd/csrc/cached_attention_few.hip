// Attention over the token cache for few query rows per key head (single tokens, a temporal module's positions).
//
// Memory bound: every cached byte is read once and meets at most 16 query rows, which all sit in one 16-wide matrix instruction.  A
// wave works on its own 32 keys at a time.  Scores are S^T = K Q^T (mfma 16x16x32 on IEEE halves): the keys' codes go from global
// memory to registers in the operand's order (the order of channels within a row is free as long as q uses the same), become
// halves there, and the exponent of a key multiplies its four scores.  A lane then holds one query's scores of keys
// 4g .. 4g+3 (g = lane / 16) of two blocks of 16, which, exponentiated, is the B operand of O^T = V^T P^T if the 8 keys of lane group g
// are taken in that order.  V^T needs 8 keys of one channel per lane: the codes pass through LDS, whose transposed
// 16-bit read delivers pairs of channels, even and odd channels becoming two operands.  A value's exponent multiplies its
// probability, so codes are never scaled.  Loads and products of different waves overlap.
//
// What becomes a half is the probability times the value's power of two, so what a row is taken relative to is the largest sum of
// score and value exponent, in octaves, of the keys that this row sees and weighs: large values of keys that it does not see, or
// gives no weight, cost it no bits.  A row's reference moves when its own scores ask for it, never for another row's sake: its bits do not
// depend on what its neighbours see.
//
// Measured: one token for each of 48 streams over one to eight frames of 1370 tokens, 16 query heads on 4 key heads of 64 (170 MB),
// 42 us here, 4.0 TB/s, and 4.6 us in the join; one token for each of 5476 positions over 32 keys, 8 heads of 32 (98 MB), 30 us,
// 3.3 TB/s: there a wave lives for one step and its chain of loads (arguments, page, keys) is what it lasts.
#include "cached_attention.h"

namespace {

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// byte offset of (key, byte column) in a wave's V tile: 32-byte segments of a row are permuted so that the eight rows which half a
// wave reads together start in different banks
template <int HDP>
__device__ __forceinline__ int vtile(int key, int col) {
    const int swz = HDP == 64 ? ((key >> 2) & 1) << 5 : HDP == 128 ? ((key >> 1) & 3) << 5 : 0;
    return key * HDP + (col ^ swz);
}

constexpr float V_REF_MIN = 40.f;    // a smaller value exponent counts as this one in the reference, or the sum of the probabilities would
                                     // overflow: values of 1e-31 and less lose bits

template <int HDP> struct Step {
    u32x4 k[2][HDP >= 64 ? HDP / 64 : 1];         // 64 channels of a key: 16 bytes per lane
    u32x2 k8[2];                                  // 32 channels of a key: 8 bytes per lane (HDP 32 and 96)
    u32x4 v[HDP / 32];
    unsigned ek[2], ev[2];
};

// Waves per SIMD that the registers allow without spilling.  (A second set of registers for the next keys' loads costs one or two
// of them and gains nothing: with it, 5476 sequences of 32 keys take 35 us, without 31; 48 streams of thousands of keys 54.4 either way.)
template <typename T, int HDP> constexpr int few_waves() {
    constexpr bool two = Pieces<T>::n == 2;
    return HDP == 32 ? (two ? 5 : 7) : HDP == 64 ? 4 : HDP == 96 ? (two ? 3 : 4) : (two ? 2 : 3);
}

// W waves share a (sequence, key head, row block, split) item, each with a part of its keys; W = 1: a wave per item.
// (out may be q: each row's queries are read by the workgroup that writes it, before it writes)
template <typename T, int HDP, int FMT, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W, (few_waves<T, HDP>())) void attend_few_kernel(const T* q, T* out,
                                                                                                       AttendJob j, int max_q, int items) {
    constexpr int NP = Pieces<T>::n, C64 = HDP / 64, TAIL32 = (HDP / 32) & 1, CB = HDP / 32;
    constexpr int LD = HDP + 4, JOIN = W == 1 ? 0 : W * (LD * 16 + 32) * 4, TILES = (W == 1 ? 4 : W) * 32 * HDP;
    __shared__ __attribute__((aligned(16))) char smem[JOIN > TILES ? JOIN : TILES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g = lane >> 4;
    const int id = W == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
    if (W == 1 && id >= items) return;
    const int item = j.by_splits.over(id), split = id - item * j.splits;
    const int t0 = j.by_heads.over(item), kvh = item - t0 * j.kv_heads, s = j.by_blocks.over(t0), rb = t0 - s * j.row_blocks;
    const int share = W == 1 ? j.chunk : j.chunk / W, k_begin = split * j.chunk + (W == 1 ? 0 : wave * share);

    // this lane's part of a V tile: it copies 16 bytes of HDP / 32 keys
    char* vt = smem + wave * (32 * HDP);
    int v_key[CB], v_lds[CB];
    int v_col[CB], k_col[C64 + TAIL32];                             // bytes of a row
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        const int idx = i * 64 + lane;
        v_key[i] = idx / (HDP / 16);
        const int col = (idx % (HDP / 16)) * 16;
        v_col[i] = min(col, j.row_bytes - 16);
        v_lds[i] = vtile<HDP>(v_key[i], col);
    }
#pragma unroll
    for (int i = 0; i < C64; ++i) k_col[i] = min(64 * i + 16 * g, j.row_bytes - 16);
    if (TAIL32) k_col[C64] = min(64 * C64 + 8 * g, j.row_bytes - 8);

    // A step has two blocks of 16 keys, each in one page (a page holds a multiple of 16 slots); a block without one reads as empty
    // slots.  Pages are asked for one step ahead, from constant memory: scalar loads, for which no other load has to be waited.
    typedef const int __attribute__((address_space(4)))* constant;
    typedef const uint8_t __attribute__((address_space(1)))* global;
    typedef const unsigned __attribute__((address_space(1)))* global4;
    typedef const u32x2 __attribute__((address_space(1)))* global8;
    typedef const u32x4 __attribute__((address_space(1)))* global16;
    const constant table = (constant)(j.page_table + (long)s * j.max_pages);
    int pi[2], off[2], page[2];
    pi[0] = j.by_page.over(k_begin);
    off[0] = k_begin - pi[0] * j.page_size;
    auto next_block = [&](int from, int to) {
        pi[to] = pi[from];
        off[to] = off[from] + 16;
        if (off[to] >= j.page_size) { off[to] = 0; ++pi[to]; }
    };
    auto ask = [&]() {
        next_block(0, 1);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int x = table[min(pi[b], j.max_pages - 1)];
            page[b] = pi[b] < j.max_pages ? x : -1;
        }
    };
    ask();
    const Span sp = span_of(j, s, max_q);
    auto fetch = [&](Step<HDP>& st, int k0) {
        long r[2];
        int last[2];                                                // of a block's rows; those behind the sequence's last key are not read from memory
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const bool any = page[b] >= 0 && page[b] < j.pages;
            r[b] = any ? ((long)page[b] * j.kv_heads + kvh) * j.page_size + off[b] : 0L;      // rows 0 .. 15 exist: they are read and not used
            // (global memory, said aloud, with scalar bases and 32-bit offsets of the lanes)
            global kr = (global)(j.k + r[b] * j.row_bytes), ke = (global)(j.k_exp + r[b]), ve = (global)(j.v_exp + r[b]);
            asm("" : "+s"(kr), "+s"(ke), "+s"(ve));
            last[b] = max(0, sp.n - 1 - k0 - 16 * b);
            const unsigned at = min(c16, last[b]) * j.row_bytes;
#pragma unroll
            for (int i = 0; i < C64; ++i) st.k[b][i] = *(global16)(kr + (at + k_col[i]));
            if (TAIL32) st.k8[b] = *(global8)(kr + (at + k_col[C64]));
            st.ek[b] = *(global4)(ke + 4u * g);
            st.ev[b] = *(global4)(ve + 4u * g);
            if (!any) st.ek[b] = 0u;
        }
        global vr[2] = {(global)(j.v + r[0] * j.row_bytes), (global)(j.v + r[1] * j.row_bytes)};
        asm("" : "+s"(vr[0]), "+s"(vr[1]));
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            const unsigned at = min(v_key[i] & 15, HDP % 64 == 0 ? last[2 * i / CB] : v_key[i] < 16 ? last[0] : last[1]) * j.row_bytes + v_col[i];
            if (HDP % 64 == 0) st.v[i] = *(global16)(vr[2 * i / CB] + at);       // (a block's keys fill whole chunks of 64 lanes)
            else st.v[i] = *(global16)((v_key[i] < 16 ? vr[0] : vr[1]) + at);
        }
        next_block(1, 0);
        ask();
    };
    // the first keys are asked for before it is known whether a row of the block sees them: the loads of keys, limits and query rows
    // are in flight together
    Step<HDP> now;
    fetch(now, k_begin);

    const int rho = rb * 16 + c16, n_rho = sp.nq * j.group;
    if (rb * 16 >= n_rho || split * j.chunk >= max(sp.n, 1)) return;      // the whole workgroup
    const int token = j.by_group.over(rho), head = kvh * j.group + (rho - token * j.group);
    const bool live = rho < n_rho;
    const long row = sp.q0 + (live ? token : 0);
    // what a row sees ends at `limit`; most: what any row of the block sees
    int limit = sp.n, most = sp.n;
    if (j.visible) {
        limit = most = live ? max(0, min(sp.n, j.visible[row])) : 0;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) most = max(most, __shfl_xor(most, o));
        if (!live) limit = most;                                    // (rows that are not there take no part in the tests below)
    }
    most = __builtin_amdgcn_readfirstlane(most);
    const int k_end = min(k_begin + share, most);
    limit = min(limit, k_end);

    f16x8 qf[2 * C64 + TAIL32][NP];
    float c_row;                                                    // from products of halves to octaves, not negative
    {
        float f[2 * C64 + TAIL32][8], amax = 0.f;
        const T* qr = q + row * j.ldq + (long)head * j.hd;
#pragma unroll
        for (int i = 0; i < 2 * C64 + TAIL32; ++i) {
            const int e = i < 2 * C64 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 64 * C64 + 8 * g;
            query8<T>(qr + e, live && e < j.hd, f[i]);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                amax = fmaxf(amax, fabsf(f[i][x]));
                f[i][x] = copysignf(1.f, j.scale_log2e) * f[i][x];
            }
        }
        amax = fmaxf(amax, __shfl_xor(amax, 16));
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        const int shift = query_shift(amax);
#pragma unroll
        for (int i = 0; i < 2 * C64 + TAIL32; ++i) query_pieces<NP>(f[i], shift, qf[i]);
        c_row = fmaxf(__builtin_amdgcn_ldexpf(fabsf(j.scale_log2e), -shift), 1e-36f);      // (0 times -infinity is no score)
    }

    f32x4 o[CB][2];
#pragma unroll
    for (int i = 0; i < CB; ++i) { o[i][0] = f32x4{0.f, 0.f, 0.f, 0.f}; o[i][1] = o[i][0]; }
    // m_run: largest score plus value exponent so far, in octaves.  Probabilities, their sum and the outputs all carry the factor
    // 2^(127 + P_SHIFT - m_run), which cancels in the end
    float m_run = LOWEST, l_run = 0.f;

    auto step = [&](Step<HDP>& st, int k0) {
        // V codes to LDS (in the order of the keys); the wave alone reads them, LDS operations of a wave stay in order
#pragma unroll
        for (int i = 0; i < CB; ++i) *reinterpret_cast<u32x4*>(vt + v_lds[i]) = st.v[i];
        asm volatile("" ::: "memory");

        float sc[2][4];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < C64; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f16x8 kf = codes8<FMT>(u32x2{st.k[b][i][2 * h], st.k[b][i][2 * h + 1]});
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) a = mfma16(kf, qf[2 * i + h][p], a);
                }
            if (TAIL32) {
                const f16x8 kf = codes8<FMT>(st.k8[b]);
#pragma unroll
                for (int p = NP - 1; p >= 0; --p) a = mfma16(kf, qf[2 * C64][p], a);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[b][i] = a[i] * power_of_byte(byte_of(st.ek[b], i));
        }
        // what is not seen: keys beyond the row's limit, empty slots; what is seen and not a number: rows with exponent 255
        unsigned keep[2] = {0xffffffffu, 0xffffffffu};
        if (__builtin_amdgcn_ballot_w64((odd_bytes(st.ek[0]) | odd_bytes(st.ek[1]) | odd_bytes(st.ev[0]) | odd_bytes(st.ev[1])) != 0 || k0 + 32 > limit) != 0) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                keep[b] = 0u;
                unsigned ev = 0u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = k0 + 16 * b + 4 * g + i;
                    const unsigned e = byte_of(st.ek[b], i), w = byte_of(st.ev[b], i);
                    const bool there = key < k_end && e != 0, nan = e == 255 || w == 255;
                    if (there && !nan) {
                        keep[b] |= 255u << (8 * i);
                        ev |= w << (8 * i);
                    }
                    if (!there || key >= limit) sc[b][i] = -INFINITY;
                    else if (nan) sc[b][i] = __builtin_nanf("");
                }
                st.ev[b] = ev;
            }
        }
        float mx = LOWEST;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fmaf(sc[b][i], c_row, fmaxf((float)byte_of(st.ev[b], i), V_REF_MIN)));
        if (__builtin_amdgcn_ballot_w64(mx > m_run + DEFER) != 0) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m_new = mx > m_run + DEFER ? mx : m_run;
            // in two steps: where a value exponent grew by more than 126, the factor's square is below the smallest number and the sum is not
            const float root = __builtin_amdgcn_exp2f(0.5f * (m_run - m_new)), alpha = root * root;
            l_run = l_run * root * root;
#pragma unroll
            for (int i = 0; i < CB; ++i) { o[i][0] *= alpha; o[i][1] *= alpha; }
            m_run = m_new;
        }
        const float base = (float)(127 + P_SHIFT) - m_run;
        f16x8 pf[NP];
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = __builtin_amdgcn_exp2f(fmaf(sc[b][i], c_row, base));
                sum += p;
                const float w = p * power_of_byte(byte_of(st.ev[b], i));         // at most 2^(P_SHIFT + DEFER), rounded to 11 bits (22 in two pieces)
                const f16 hi = (f16)w;
                pf[0][4 * b + i] = hi;
                if (NP == 2) pf[NP - 1][4 * b + i] = (f16)(w - (float)hi);
            }
        l_run += sum;

        // (a hidden key's value codes may be anything, e4m3's NaN too: 0 times them has to be 0)
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            const int q4 = c16 >> 2, p4 = c16 & 3;
            const u32x2 r0 = __builtin_bit_cast(u32x2, read_tr<f16>(vt + vtile<HDP>(4 * g + q4, 32 * i + 8 * p4)));
            const u32x2 r1 = __builtin_bit_cast(u32x2, read_tr<f16>(vt + vtile<HDP>(16 + 4 * g + q4, 32 * i + 8 * p4)));
#pragma unroll
            for (int par = 0; par < 2; ++par) {
                const unsigned sel = par ? 0x07050301u : 0x06040200u;
                u32x2 w = {__builtin_amdgcn_perm(r0[1], r0[0], sel), __builtin_amdgcn_perm(r1[1], r1[0], sel)};
                if (FMT == VDA_CACHE_E4M3) { w[0] &= keep[0]; w[1] &= keep[1]; }
                const f16x8 vf = codes8<FMT>(w);
#pragma unroll
                for (int p = NP - 1; p >= 0; --p) o[i][par] = mfma16(vf, pf[p], o[i][par]);
            }
        }
    };
    for (int k0 = k_begin; k0 < k_end; k0 += 32) {
        if (k0 > k_begin) fetch(now, k0);
        step(now, k0);
    }

    // lane (c16, g) holds channels 32 i + 8 g + 0..7 of query c16, even ones in o[i][0], odd ones in o[i][1]
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
    if constexpr (W > 1) {        // join the waves' parts: [wave][16 rows][LD] outputs, then [wave][16] maxima and sums
        __syncthreads();                                            // the V tiles are done with
        float* jo = reinterpret_cast<float*>(smem);
        float* jm = jo + W * 16 * LD;
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            float* p = jo + (wave * 16 + c16) * LD + 32 * i + 8 * g;
            *reinterpret_cast<f32x4*>(p) = f32x4{o[i][0][0], o[i][1][0], o[i][0][1], o[i][1][1]};
            *reinterpret_cast<f32x4*>(p + 4) = f32x4{o[i][0][2], o[i][1][2], o[i][0][3], o[i][1][3]};
        }
        if (g == 0) { jm[wave * 16 + c16] = m_run; jm[W * 16 + wave * 16 + c16] = l_run; }
        __syncthreads();
        float* part = j.part + ((long)item * j.splits + split) * (16 * (HDP + 2));
        for (int x = threadIdx.x; x < 16 * (HDP / 4); x += 64 * W) {       // a row and four channels per thread
            const int r = x / (HDP / 4), d = (x % (HDP / 4)) * 4, rho_r = rb * 16 + r;
            if (rho_r >= n_rho) continue;
            float m = LOWEST, l = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) m = fmaxf(m, jm[w * 16 + r]);
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float root = __builtin_amdgcn_exp2f(0.5f * (jm[w * 16 + r] - m));
                l += jm[W * 16 + w * 16 + r] * root * root;
                v += root * root * *reinterpret_cast<const f32x4*>(jo + (w * 16 + r) * LD + d);
            }
            if (j.splits > 1) {
                *reinterpret_cast<f32x4*>(part + r * HDP + d) = v;
                if (d == 0) { part[16 * HDP + r] = m; part[16 * HDP + 16 + r] = l; }
            } else if (d < j.hd) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const int tok = j.by_group.over(rho_r);
                const typename Vec<T>::v4 y = {(T)(v[0] * inv), (T)(v[1] * inv), (T)(v[2] * inv), (T)(v[3] * inv)};
                *reinterpret_cast<typename Vec<T>::v4*>(out + (sp.q0 + tok) * j.ldo + (long)(kvh * j.group + rho_r - tok * j.group) * j.hd + d) = y;
            }
        }
    } else {
        if (!live) return;
        const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
        T* orow = out + row * j.ldo + (long)head * j.hd;
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            const int d = 32 * i + 8 * g;
            if (d >= j.hd) continue;
            typename Vec<T>::v8 r;
#pragma unroll
            for (int x = 0; x < 4; ++x) { r[2 * x] = (T)(o[i][0][x] * inv); r[2 * x + 1] = (T)(o[i][1][x] * inv); }
            *reinterpret_cast<typename Vec<T>::v8*>(orow + d) = r;
        }
    }
}

// The parts of a row block joined in their order: out = sum 2^(m_s - m) o_s / sum 2^(m_s - m) l_s, m the largest reference, found on the way.
// A thread per row and four channels; grid (item, run of rows).  Latency bound: with one part's loads at a time 42 parts took 14 us longer.
template <typename T>
__global__ __launch_bounds__(256) void attend_join_kernel(T* __restrict__ out, AttendJob j, int max_q, int block_rows, int hdp) {
    const int item = blockIdx.x, t0 = j.by_heads.over(item), kvh = item - t0 * j.kv_heads, s = j.by_blocks.over(t0), rb = t0 - s * j.row_blocks;
    const Span sp = span_of(j, s, max_q);
    const int rows = min(block_rows, sp.nq * j.group - rb * block_rows), quads = j.hd / 4, per = 256 / quads;
    const int r0 = threadIdx.x / quads, r = blockIdx.y * per + r0, d = (threadIdx.x - r0 * quads) * 4;
    if (r0 >= per || r >= rows) return;
    const long stride = (long)block_rows * (hdp + 2);
    const float* p = j.part + (long)item * j.splits * stride;
    const int parts = max(1, (sp.n + j.chunk - 1) / j.chunk);
    float m = LOWEST, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int x0 = 0; x0 < parts; x0 += 4) {                         // four parts' loads in flight together
        float mx[4], lx[4];
        f32x4 ox[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float* px = p + min(x0 + i, parts - 1) * stride;
            mx[i] = px[block_rows * hdp + r];
            lx[i] = x0 + i < parts ? px[block_rows * hdp + block_rows + r] : 0.f;
            ox[i] = *reinterpret_cast<const f32x4*>(px + r * hdp + d);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {                               // (a part without a key of the row does not move the reference)
            const bool none = lx[i] == 0.f;
            const float mn = none ? m : fmaxf(m, mx[i]), ra = __builtin_amdgcn_exp2f(0.5f * (m - mn)), rb = none ? 0.f : __builtin_amdgcn_exp2f(0.5f * (mx[i] - mn));
            m = mn;
            l = l * ra * ra + lx[i] * rb * rb;
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = ra * ra * o[k] + (none ? 0.f : rb * rb * ox[i][k]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int rho = rb * block_rows + r, token = j.by_group.over(rho);
    const typename Vec<T>::v4 y = {(T)(o[0] * inv), (T)(o[1] * inv), (T)(o[2] * inv), (T)(o[3] * inv)};
    *reinterpret_cast<typename Vec<T>::v4*>(out + (sp.q0 + token) * j.ldo + (long)(kvh * j.group + rho - token * j.group) * j.hd + d) = y;
}

template <typename T>
int few(const AttendJob& j, const T* q, T* out, int format, int max_q, int waves, hipStream_t st) {
    const int items = j.seqs * j.kv_heads * j.row_blocks * j.splits;
    const int grid = waves == 1 ? (items + 3) / 4 : items;
#define VDA_F3(H, F, W) hipLaunchKernelGGL((attend_few_kernel<T, H, F, W>), dim3(grid), dim3(W == 1 ? 256 : 64 * W), 0, st, q, out, j, max_q, items)
#define VDA_F2(H, F) do { if (waves == 1) VDA_F3(H, F, 1); else VDA_F3(H, F, 8); } while (0)
#define VDA_F(H) do { if (format == VDA_CACHE_I8) VDA_F2(H, VDA_CACHE_I8); else VDA_F2(H, VDA_CACHE_E4M3); } while (0)
    if (j.hd <= 32) VDA_F(32);
    else if (j.hd <= 64) VDA_F(64);
    else if (j.hd <= 96) VDA_F(96);
    else VDA_F(128);
#undef VDA_F
#undef VDA_F2
#undef VDA_F3
    return hip_rc(hipGetLastError());
}

}  // namespace

int attend_few(const AttendJob& j, const void* q, void* out, int dtype, int format, int max_q, int waves, hipStream_t st) {
    if (dtype == VDA_T_BF16) return few(j, (const bf16*)q, (bf16*)out, format, max_q, waves, st);
    if (dtype == VDA_T_F16) return few(j, (const f16*)q, (f16*)out, format, max_q, waves, st);
    return few(j, (const float*)q, (float*)out, format, max_q, waves, st);
}

int attend_join(const AttendJob& j, void* out, int dtype, int max_q, int block_rows, int hd_pad, hipStream_t st) {
    const int per = 256 / (j.hd / 4);
    const dim3 grid(j.seqs * j.kv_heads * j.row_blocks, (block_rows + per - 1) / per);
    if (dtype == VDA_T_BF16) hipLaunchKernelGGL((attend_join_kernel<bf16>), grid, dim3(256), 0, st, (bf16*)out, j, max_q, block_rows, hd_pad);
    else if (dtype == VDA_T_F16) hipLaunchKernelGGL((attend_join_kernel<f16>), grid, dim3(256), 0, st, (f16*)out, j, max_q, block_rows, hd_pad);
    else hipLaunchKernelGGL((attend_join_kernel<float>), grid, dim3(256), 0, st, (float*)out, j, max_q, block_rows, hd_pad);
    return hip_rc(hipGetLastError());
}
