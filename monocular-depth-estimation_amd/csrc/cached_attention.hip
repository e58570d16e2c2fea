// Attention of new tokens over the 8-bit token cache (see vda_cached_attention in include/vda_hip.h).
#include "token_cache.h"

namespace {

struct Job {
    const uint8_t *k, *v, *k_exp, *v_exp;
    const int *page_table, *kv_len, *q_start, *visible;
    int pages, page_size, kv_heads, hd, row_bytes, format, max_pages, group;
    long rows, ldq, ldo;
    float scale_log2e;
};

__device__ __forceinline__ float code_value(unsigned byte, int format) {
    return format == VDA_CACHE_I8 ? (float)(int)(signed char)byte : __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
}
__device__ __forceinline__ float power(int byte) { return byte == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(1.f, byte - 127); }

// One wave per (row, head): lanes are keys for the scores, channels for the output.
template <typename T>
__global__ __launch_bounds__(64) void attend_kernel(const T* __restrict__ q, T* __restrict__ out, Job j, int max_q) {
    __shared__ float qs[128];
    const int s = blockIdx.y, head = blockIdx.z, lane = threadIdx.x;
    const long q0 = max(0L, min((long)j.q_start[s], j.rows)), q1 = max(q0, min((long)j.q_start[s + 1], j.rows));
    const long row = q0 + blockIdx.x;
    if (row >= q1) return;
    const int kvh = head / j.group;
    int n = max(0, min(j.kv_len[s], j.max_pages * j.page_size));
    if (j.visible) n = max(0, min(n, j.visible[row]));
    for (int d = lane; d < j.hd; d += 64) qs[d] = (float)q[row * j.ldq + (long)head * j.hd + d] * j.scale_log2e;
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
    for (int k0 = 0; k0 < n; k0 += 64) {
        const int key = k0 + lane;
        float sc = -INFINITY;
        long at = -1;
        if (key < n) {
            const int page = j.page_table[(long)s * j.max_pages + key / j.page_size];
            if (page >= 0 && page < j.pages) {
                at = ((long)page * j.kv_heads + kvh) * j.page_size + key % j.page_size;
                const int e = j.k_exp[at];
                if (e == 0) at = -1;
                else {
                    float acc = 0.f;
                    for (int d = 0; d < j.hd; ++d) acc += qs[d] * code_value(j.k[at * j.row_bytes + d], j.format);
                    sc = acc * power(e);
                }
            }
        }
        float mx = isnan(sc) ? 0.f : sc;
        for (int x = 32; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
        if (mx == -INFINITY && !__any(isnan(sc))) continue;
        const float mn = fmaxf(m, mx), alpha = m == -INFINITY ? 0.f : exp2f(m - mn), p = sc == -INFINITY ? 0.f : exp2f(sc - mn);
        l = l * alpha + wave_sum(p);
        o[0] *= alpha;
        o[1] *= alpha;
        m = mn;
        for (int i = 0; i < 64; ++i) {
            const float pi = __shfl(p, i);
            const long ai = __shfl(at, i);
            if (ai < 0) continue;
            const float w = power(j.v_exp[ai]);
            for (int c = 0; c < 2; ++c)
                if (lane + 64 * c < j.hd) o[c] += pi * (w * code_value(j.v[ai * j.row_bytes + lane + 64 * c], j.format));
        }
    }
    for (int c = 0; c < 2; ++c)
        if (lane + 64 * c < j.hd) out[row * j.ldo + (long)head * j.hd + lane + 64 * c] = (T)(l == 0.f ? 0.f : o[c] / l);
}

}  // namespace

extern "C" long vda_cached_attention_work(const VdaTokenCache* cache, int seqs, int max_pages, int max_q, int heads) {
    if (const int rc = cache_check(cache)) return rc;
    if (seqs <= 0 || max_pages <= 0 || max_q <= 0 || heads <= 0) return VDA_EINVAL;
    if (heads % cache->kv_heads != 0 || (long)max_pages * cache->page_size > 0x7fffffffL) return VDA_ESHAPE;
    return 0;                                                      // nothing is split
}

extern "C" int vda_cached_attention(const VdaTokenCache* cache, const VdaCachedAttentionArgs* a, void* stream) {
    if (const int rc = cache_check(cache)) return rc;
    if (!a || !a->q || !a->out || !a->page_table || !a->kv_len || !a->q_start || a->seqs <= 0 || a->max_pages <= 0 || a->max_q <= 0 || a->heads <= 0 ||
        a->rows <= 0) return VDA_EINVAL;
    if (a->dtype != VDA_T_BF16 && a->dtype != VDA_T_F16 && a->dtype != VDA_T_F32) return VDA_EINVAL;
    const int size = a->dtype == VDA_T_F32 ? 4 : 2;
    if (a->heads % cache->kv_heads != 0 || a->ldq < (long)a->heads * cache->hd || a->ldo < (long)a->heads * cache->hd) return VDA_ESHAPE;
    if ((((uintptr_t)a->q | (uintptr_t)a->out) & 15) != 0 || (a->ldq * size) % 16 != 0 || (a->ldo * size) % 16 != 0) return VDA_ESHAPE;
    if ((long)a->max_pages * cache->page_size > 0x7fffffffL || a->seqs > 65535 || a->heads > 65535) return VDA_ESHAPE;
    const Job j{(const uint8_t*)cache->k, (const uint8_t*)cache->v, cache->k_exp, cache->v_exp, a->page_table, a->kv_len, a->q_start, a->visible,
                cache->pages, cache->page_size, cache->kv_heads, cache->hd, cache_row_bytes(cache->hd), cache->format, a->max_pages,
                a->heads / cache->kv_heads, a->rows, a->ldq, a->ldo, a->scale * 1.4426950408889634f};
    dim3 grid(a->max_q, a->seqs, a->heads);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (a->dtype == VDA_T_BF16) hipLaunchKernelGGL((attend_kernel<bf16>), grid, dim3(64), 0, st, (const bf16*)a->q, (bf16*)a->out, j, a->max_q);
    else if (a->dtype == VDA_T_F16) hipLaunchKernelGGL((attend_kernel<f16>), grid, dim3(64), 0, st, (const f16*)a->q, (f16*)a->out, j, a->max_q);
    else hipLaunchKernelGGL((attend_kernel<float>), grid, dim3(64), 0, st, (const float*)a->q, (float*)a->out, j, a->max_q);
    return hip_rc(hipGetLastError());
}
