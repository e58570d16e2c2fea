// The step between two blocks of a transformer in one pass over the residual stream (see vda_gated_norm in include/vda_hip.h):
//     x' = resid_scale * x + gate * post(b),   y = pre(x') * (1 + mod_scale) + mod_shift
// Bound by memory bandwidth: 4 + 4 bytes of x and 2 + 2 of b and y per channel, each moved once; a row stays in registers between
// the two norms.  Statistics are two-pass in fp32.  32 frames of 1370 tokens, 1024 channels in bf16 (539 MB), norms before and after:
// 124 us, 4.35 TB/s; a copy of 4 GiB reaches 4.7.  One wave holds a row of up to 1024 channels (no barrier), four share one of up to 4096, eight a longer one.
#include "common.h"

namespace {

struct NormArgs {
    const float *x, *post_w, *post_b, *gate, *pre_w, *pre_b, *mod_scale, *mod_shift;
    float* x_out;
    long rows, ldx, ldb, ldxo, ldy;
    float resid_scale, eps;
    int C, post, pre;
    unsigned per_group;
};

// Sum over the W waves of a workgroup that share a row (W = 1: the wave's own sum).
template <int W>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
    v = wave_sum(v);
    if (W > 1) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) v += scratch[i];
    }
    return v;
}

// v -> its norm's (v - mean) * rstd, kind VDA_NORM_LAYER or VDA_NORM_RMS.  Channels beyond C hold 0 and stay 0.
template <int N, int W>
__device__ __forceinline__ void normalise(f32x4 (&v)[N], int kind, int lane0, int C, float eps, float* scratch) {
    if (kind == VDA_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s += (v[i][0] + v[i][1]) + (v[i][2] + v[i][3]);
        const float mean = row_sum<W>(s, scratch) / C;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((i * 64 * W + lane0) * 4 < C) v[i] -= mean;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) q += (v[i][0] * v[i][0] + v[i][1] * v[i][1]) + (v[i][2] * v[i][2] + v[i][3] * v[i][3]);
    const float rstd = rsqrtf(row_sum<W>(q, scratch) / C + eps);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= rstd;
}

// W waves share a row of up to 256 N W channels: a workgroup holds four rows of one wave each, or one row.  N = 8 takes 190 registers, two
// waves per SIMD: 20000 rows of 2048 channels, norms before and after, 243 us with one wave to a row, 114 with four and N = 2.
template <typename TB, typename TY, int N, int W>
__global__ __launch_bounds__(W == 8 ? 512 : 256) void gated_norm_kernel(NormArgs a, const TB* __restrict__ b, TY* __restrict__ y) {
    __shared__ float scratch[W];
    const int lane0 = W == 1 ? (threadIdx.x & 63) : threadIdx.x;
    const long row = W == 1 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long)blockIdx.x;
    if (row >= a.rows) return;
    const size_t group = (size_t)((unsigned long)row / a.per_group) * a.C;
    f32x4 v[N];
    if (b) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (i * 64 * W + lane0) * 4;
            v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (c < a.C) {
                const typename Vec<TB>::v4 r = *reinterpret_cast<const typename Vec<TB>::v4*>(b + row * a.ldb + c);
                v[i] = f32x4{(float)r[0], (float)r[1], (float)r[2], (float)r[3]};
            }
        }
        if (a.post != VDA_NORM_NONE) normalise<N, W>(v, a.post, lane0, a.C, a.eps, scratch);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * 64 * W + lane0) * 4;
        if (c >= a.C) { v[i] = f32x4{0.f, 0.f, 0.f, 0.f}; continue; }
        f32x4 x = *reinterpret_cast<const f32x4*>(a.x + row * a.ldx + c);
        if (b) {
            if (a.post_w) v[i] *= *reinterpret_cast<const f32x4*>(a.post_w + c);
            if (a.post_b) v[i] += *reinterpret_cast<const f32x4*>(a.post_b + c);
            if (a.gate) v[i] *= *reinterpret_cast<const f32x4*>(a.gate + group + c);
            x = x * a.resid_scale + v[i];
            *reinterpret_cast<f32x4*>(a.x_out + row * a.ldxo + c) = x;
        }
        v[i] = x;
    }
    if (!y) return;
    if (a.pre != VDA_NORM_NONE) normalise<N, W>(v, a.pre, lane0, a.C, a.eps, scratch);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * 64 * W + lane0) * 4;
        if (c >= a.C) continue;
        f32x4 r = v[i];
        if (a.pre_w) r *= *reinterpret_cast<const f32x4*>(a.pre_w + c);
        if (a.pre_b) r += *reinterpret_cast<const f32x4*>(a.pre_b + c);
        if (a.mod_scale) r *= 1.f + *reinterpret_cast<const f32x4*>(a.mod_scale + group + c);
        if (a.mod_shift) r += *reinterpret_cast<const f32x4*>(a.mod_shift + group + c);
        const typename Vec<TY>::v4 o = {(TY)r[0], (TY)r[1], (TY)r[2], (TY)r[3]};
        *reinterpret_cast<typename Vec<TY>::v4*>(y + row * a.ldy + c) = o;
    }
}

template <typename TB, typename TY>
int launch(const NormArgs& a, const void* b, void* y, hipStream_t st) {
    const int wave_row = a.C <= 1024;
    const long grid = wave_row ? (a.rows + 3) / 4 : a.rows;
    if (grid > 0x7fffffffL) return VDA_ESHAPE;
#define VDA_GN(N, W) hipLaunchKernelGGL((gated_norm_kernel<TB, TY, N, W>), dim3(grid), dim3(W == 8 ? 512 : 256), 0, st, a, (const TB*)b, (TY*)y)
    if (a.C <= 256) VDA_GN(1, 1);
    else if (a.C <= 512) VDA_GN(2, 1);
    else if (a.C <= 1024) VDA_GN(4, 1);
    else if (a.C <= 2048) VDA_GN(2, 4);
    else if (a.C <= 4096) VDA_GN(4, 4);
    else VDA_GN(4, 8);
#undef VDA_GN
    return hip_rc(hipGetLastError());
}

bool norm_kind(int k) { return k == VDA_NORM_NONE || k == VDA_NORM_LAYER || k == VDA_NORM_RMS; }
bool rows16(const void* p, long ld, int size) { return ((uintptr_t)p & (4 * size - 1)) == 0 && ld % 4 == 0; }

}  // namespace

extern "C" int vda_gated_norm(const VdaGatedNormArgs* g, void* stream) {
    if (!g || !g->x || g->rows <= 0 || g->C <= 0 || g->rows_per_group <= 0 || !norm_kind(g->post) || !norm_kind(g->pre)) return VDA_EINVAL;
    if (!g->b != !g->x_out || (!g->b && !g->y)) return VDA_EINVAL;                   // a block's output makes a new stream; something is written
    if (!g->b && (g->post != VDA_NORM_NONE || g->gate || g->post_w || g->post_b)) return VDA_EINVAL;
    if (!g->y && (g->pre != VDA_NORM_NONE || g->pre_w || g->pre_b || g->mod_scale || g->mod_shift)) return VDA_EINVAL;
    auto type = [](int t) { return t == VDA_T_F32 || t == VDA_T_BF16 || t == VDA_T_F16; };
    if ((g->b && !type(g->b_type)) || (g->y && !type(g->y_type))) return VDA_EINVAL;
    if (g->C % 4 != 0 || g->C > 8192 || g->ldx < g->C || (g->b && (g->ldb < g->C || g->ldxo < g->C)) || (g->y && g->ldy < g->C)) return VDA_ESHAPE;
    const int bs = g->b_type == VDA_T_F32 ? 4 : 2, ys = g->y_type == VDA_T_F32 ? 4 : 2;
    if (!rows16(g->x, g->ldx, 4) || (g->b && (!rows16(g->b, g->ldb, bs) || !rows16(g->x_out, g->ldxo, 4))) || (g->y && !rows16(g->y, g->ldy, ys))) return VDA_ESHAPE;
    if ((((uintptr_t)g->post_w | (uintptr_t)g->post_b | (uintptr_t)g->gate | (uintptr_t)g->pre_w | (uintptr_t)g->pre_b | (uintptr_t)g->mod_scale |
          (uintptr_t)g->mod_shift) & 15) != 0) return VDA_ESHAPE;
    if (g->x_out == g->x && g->ldxo != g->ldx) return VDA_EINVAL;
    const NormArgs a{g->x, g->post_w, g->post_b, g->gate, g->pre_w, g->pre_b, g->mod_scale, g->mod_shift, g->x_out, g->rows, g->ldx, g->ldb, g->ldxo,
                     g->ldy, g->resid_scale, g->eps, g->C, g->post, g->pre, (unsigned)g->rows_per_group};
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int tb = g->b ? g->b_type : g->y_type, ty = g->y ? g->y_type : g->b_type;
#define VDA_GNT(TB) (ty == VDA_T_F32 ? launch<TB, float>(a, g->b, g->y, st) : ty == VDA_T_F16 ? launch<TB, f16>(a, g->b, g->y, st) : launch<TB, bf16>(a, g->b, g->y, st))
    return tb == VDA_T_F32 ? VDA_GNT(float) : tb == VDA_T_F16 ? VDA_GNT(f16) : VDA_GNT(bf16);
#undef VDA_GNT
}
