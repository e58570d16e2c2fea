// Attention of new tokens over the 8-bit token cache: argument checks, the choice of kernel and of how the key axis is split
// (see vda_cached_attention in include/vda_hip.h).
#include "cached_attention.h"

namespace {

struct Plan {
    int row_blocks, splits, chunk, waves, block_rows, hd_pad;
    long work;
};

// Up to 32 rows per key head, or few rows of work in all (blocks of 16 rows times keys, fewer for wide heads): the kernel whose waves
// hold 16 rows each and read the cache straight into registers.  It wants enough waves in flight to draw the full memory bandwidth:
// where there are fewer than 4096 (sequence, key head, row block) items, eight waves share an item, and beyond 2048 keys the key
// axis is split over workgroups too, down to 64 keys for each wave.
// More rows: the kernel whose workgroups of 128 rows share decoded tiles; the key axis is split, down to 512 keys, until the
// workgroups that a CU holds at once (three, two for wide heads) are there.
// Measured, us of the first kernel / the second, 8 heads of 64 in IEEE half: 32 rows over 8192 keys 20 / 25, 96 rows 27 / 26; 384 rows
// over 2048 keys 16 / 23; 8 sequences over 2048 keys, 96 rows 23 / 26, 256 rows 40 / 38; 64 sequences over 512 keys, 32 rows
// 18 / 22, 64 rows 30 / 23.  Heads of 128, in half and in fp32: 8 sequences over 2048 keys, 64 rows 21 / 32 and 26 / 41, 96 rows
// 37 / 34 and 46 / 44; over 512 keys, 384 rows 46 / 25 and 58 / 38.
constexpr int FEW_ROWS = 32, FEW_KEYS = 4096;
constexpr int ONE_FEW = 2048, MIN_FEW = 512, MIN_MANY = 512;
int plan_of(const VdaTokenCache* c, int seqs, int max_pages, int max_q, int heads, Plan* p) {
    if (const int rc = cache_check(c)) return rc;
    if (seqs <= 0 || max_pages <= 0 || max_q <= 0 || heads <= 0) return VDA_EINVAL;
    if (heads % c->kv_heads != 0 || (long)max_pages * c->page_size > 0x40000000L) return VDA_ESHAPE;
    const long rows = (long)max_q * (heads / c->kv_heads), keys = (long)max_pages * c->page_size;
    if (rows > 0x3fffffffL || (long)seqs * c->kv_heads > 0x3fffffffL) return VDA_ESHAPE;
    const long few_items = (rows + 15) / 16 * seqs * c->kv_heads;
    const bool few = rows <= FEW_ROWS || (keys <= FEW_KEYS && few_items <= ((c->hd <= 64 ? 6L : 5L) << 17) / keys);
    p->block_rows = few ? 16 : 128;
    p->hd_pad = (c->hd + 31) & ~31;
    const long blocks = (rows + p->block_rows - 1) / p->block_rows, items = blocks * seqs * c->kv_heads;
    if (items > 0x3fffffffL) return VDA_ESHAPE;
    long chunk = keys;                                            // keys of a part, a multiple of 32 for each of eight waves
    if (few) {
        p->waves = items >= 4096 || keys <= 64 ? 1 : 8;
        if (p->waves == 8 && keys > ONE_FEW) {
            const long wanted = 2048 / items;                     // parts, if there are keys enough
            chunk = wanted <= 1 ? keys : (keys + wanted - 1) / wanted;
            chunk = chunk < MIN_FEW ? MIN_FEW : chunk;
        }
    } else {
        p->waves = 0;
        const long wanted = 256 * (c->hd <= 64 ? 3 : 2) / items;
        chunk = wanted <= 1 ? keys : (keys + wanted - 1) / wanted;
        chunk = chunk < MIN_MANY ? MIN_MANY : chunk;
    }
    chunk = (chunk + 255) & ~255L;
    const long splits = (keys + chunk - 1) / chunk;
    if (items * splits > 0x7fffffffL) return VDA_ESHAPE;
    p->chunk = (int)chunk;
    p->splits = (int)splits;
    p->row_blocks = (int)blocks;
    p->work = p->splits == 1 ? 0 : items * p->splits * p->block_rows * (p->hd_pad + 2) * (long)sizeof(float);
    return VDA_OK;
}

}  // namespace

extern "C" long vda_cached_attention_work(const VdaTokenCache* cache, int seqs, int max_pages, int max_q, int heads) {
    Plan p;
    const int rc = plan_of(cache, seqs, max_pages, max_q, heads, &p);
    return rc ? rc : p.work;
}

extern "C" int vda_cached_attention(const VdaTokenCache* cache, const VdaCachedAttentionArgs* a, void* stream) {
    if (!a || !a->q || !a->out || !a->page_table || !a->kv_len || !a->q_start || a->rows <= 0) return VDA_EINVAL;
    if (a->dtype != VDA_T_BF16 && a->dtype != VDA_T_F16 && a->dtype != VDA_T_F32) return VDA_EINVAL;
    Plan p;
    if (const int rc = plan_of(cache, a->seqs, a->max_pages, a->max_q, a->heads, &p)) return rc;
    const int size = a->dtype == VDA_T_F32 ? 4 : 2;
    if (a->ldq < (long)a->heads * cache->hd || a->ldo < (long)a->heads * cache->hd || a->rows > 0x7fffffffL) return VDA_ESHAPE;
    if ((((uintptr_t)a->q | (uintptr_t)a->out) & 15) != 0 || (a->ldq * size) % 16 != 0 || (a->ldo * size) % 16 != 0) return VDA_ESHAPE;
    if (p.work > 0) {
        if (!a->work) return VDA_EINVAL;
        if (a->work_bytes < p.work || ((uintptr_t)a->work & 15) != 0) return VDA_ESHAPE;
    }
    const AttendJob j{(const uint8_t*)cache->k, (const uint8_t*)cache->v, cache->k_exp, cache->v_exp, a->page_table, a->kv_len, a->q_start, a->visible,
                      (float*)a->work, a->rows, a->ldq, a->ldo, cache->pages, cache->page_size, cache->kv_heads, cache->hd, cache_row_bytes(cache->hd),
                      a->max_pages, a->heads / cache->kv_heads, a->seqs, p.row_blocks, p.splits, p.chunk, a->scale * 1.4426950408889634f,
                      Quick(p.splits), Quick(cache->kv_heads), Quick(p.row_blocks), Quick(a->heads / cache->kv_heads), Quick(cache->page_size)};
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int rc = p.waves ? attend_few(j, a->q, a->out, a->dtype, cache->format, a->max_q, p.waves, st)
                           : attend_many(j, a->q, a->out, a->dtype, cache->format, a->max_q, st);
    if (rc) return rc;
    return p.splits > 1 ? attend_join(j, a->out, a->dtype, a->max_q, p.block_rows, p.hd_pad, st) : VDA_OK;
}
