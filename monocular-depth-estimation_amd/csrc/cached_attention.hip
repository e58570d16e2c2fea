// Attention of new tokens over the 8-bit token cache: argument checks, the choice of kernel and of how the key axis is split
// (see vda_cached_attention in include/vda_hip.h).
#include "cached_attention.h"

#include <cmath>

namespace {

struct Plan {
    int row_blocks, splits, chunk, waves, block_rows, hd_pad;
    long work;
};

// Up to 32 rows per key head, or few rows of work in all (blocks of 16 rows times keys, fewer for wide heads): the kernel whose waves
// hold 16 rows each and read the cache straight into registers.  Where there are fewer than 4096 (sequence, key head, row block)
// items, eight waves share an item, and the key axis is split over workgroups where part_of finds that it pays.
// More rows: the kernel whose workgroups of 128 rows share decoded tiles; the key axis is split, down to 512 keys, until the
// workgroups that a CU holds at once (three, two for wide heads) are there.
// Measured, us of the first kernel / the second, 8 heads of 64 in IEEE half: 32 rows over 8192 keys 20 / 25, 96 rows 27 / 26; 384 rows
// over 2048 keys 16 / 23; 8 sequences over 2048 keys, 96 rows 23 / 26, 256 rows 40 / 38; 64 sequences over 512 keys, 32 rows
// 18 / 22, 64 rows 30 / 23.  Heads of 128, in half and in fp32: 8 sequences over 2048 keys, 64 rows 21 / 32 and 26 / 41, 96 rows
// 37 / 34 and 46 / 44; over 512 keys, 384 rows 46 / 25 and 58 / 38.
constexpr int FEW_ROWS = 32, FEW_KEYS = 4096;
constexpr int MIN_PART = 512;        // keys of a part at least

// Keys of a part, for workgroups of eight waves and `items` of them per part.  A workgroup costs its keys and what 700 more would
// (first loads, join of the waves); up to 256 run side by side, one on each CU, and 512 take half as long again (wide heads, whose
// registers leave room for one on a CU: twice as long).  The join of the parts costs as 2000 keys: 4 us on the device, and a second launch.
// Tried: parts that make 256, 512, ... 2048 workgroups.  Measured, us of 1 part / 512 / 1024 / 2048 workgroups on the device, heads of 64:
// 64 items of 10960 keys 60 / 28 / 35 / 40, 192 items 71 / 61 / 58 / 62, 256 items of 4096 keys 29 / 31 / 34 / 41, 512 items of 10960
// keys 147 / - / 155 / 159; 6 items of 3000 keys 18.8, in six parts 10.1; heads of 128: 192 items of 10960 keys 114 / 132 / 126 / 137.
// The rule does not know how many bytes a key has: at 32 channels it leaves 384 items of 10960 keys in one part, 83 us, where parts
// took 72.  It goes by the keys that the table can hold, as the workspace does: a table wider than its sequences may cost a join.
long part_of(long keys, long items, bool wide) {
    long best = 0, part = keys;
    for (int j = 0; j <= 8; ++j) {
        const long wanted = j ? 256L * j / items : 1;
        if (wanted < 1) continue;
        long each = (keys + wanted - 1) / wanted;
        each = wanted > 1 && each < MIN_PART ? MIN_PART : each;
        each = (each + 255) & ~255L;
        const long parts = (keys + each - 1) / each, groups = parts * items, pair = wide ? 4 : 3;
        const long cost = (groups <= 256 ? 2 : (groups + 511) / 512 * pair) * (each + 700) + (parts > 1 ? 2 * 2000 : 0);      // in halves
        if (j == 0 || cost < best) { best = cost; part = each; }
    }
    return part;
}
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
        if (p->waves == 8) chunk = part_of(keys, items, c->hd > 64);
    } else {
        p->waves = 0;
        const long wanted = 256 * (c->hd <= 64 ? 3 : 2) / items;
        chunk = wanted <= 1 ? keys : (keys + wanted - 1) / wanted;
        chunk = chunk < MIN_PART ? MIN_PART : chunk;
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
    const float octaves = a->scale * 1.4426950408889634f;
    if (!std::isfinite(octaves)) return VDA_EINVAL;
    Plan p;
    if (const int rc = plan_of(cache, a->seqs, a->max_pages, a->max_q, a->heads, &p)) return rc;
    const int size = a->dtype == VDA_T_F32 ? 4 : 2;
    if (a->ldq < (long)a->heads * cache->hd || a->ldo < (long)a->heads * cache->hd || a->rows > 0x7fffffffL) return VDA_ESHAPE;
    if ((((uintptr_t)a->q | (uintptr_t)a->out) & 15) != 0 || (a->ldq * size) % 16 != 0 || (a->ldo * size) % 16 != 0) return VDA_ESHAPE;
    if (a->q == a->out && a->ldq != a->ldo) return VDA_EINVAL;
    if (p.work > 0) {
        if (!a->work) return VDA_EINVAL;
        if (a->work_bytes < p.work || ((uintptr_t)a->work & 15) != 0) return VDA_ESHAPE;
    }
    const AttendJob j{(const uint8_t*)cache->k, (const uint8_t*)cache->v, cache->k_exp, cache->v_exp, a->page_table, a->kv_len, a->q_start, a->visible,
                      (float*)a->work, a->rows, a->ldq, a->ldo, cache->pages, cache->page_size, cache->kv_heads, cache->hd, cache_row_bytes(cache->hd),
                      a->max_pages, a->heads / cache->kv_heads, a->seqs, p.row_blocks, p.splits, p.chunk, octaves,
                      Quick(p.splits), Quick(cache->kv_heads), Quick(p.row_blocks), Quick(a->heads / cache->kv_heads), Quick(cache->page_size)};
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int rc = p.waves ? attend_few(j, a->q, a->out, a->dtype, cache->format, a->max_q, p.waves, st)
                           : attend_many(j, a->q, a->out, a->dtype, cache->format, a->max_q, st);
    if (rc) return rc;
    return p.splits > 1 ? attend_join(j, a->out, a->dtype, a->max_q, p.block_rows, p.hd_pad, st) : VDA_OK;
}
