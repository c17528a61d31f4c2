// C ABI of the 4-bit cache: argument checking and launch geometry.  The interface is documented in include/homcomp_cache.h.
#include "../../include/homcomp_cache.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>

#include "homcomp_cache.hpp"

namespace {

constexpr int64_t kMostSlots = (int64_t)INT32_MAX - 64;
constexpr int64_t kMostWorkgroups = UINT32_MAX / 256;   // a launch has fewer than 2^32 threads

constexpr int kComputeUnits = 256;

int launched(hipError_t e)
{
    if (e == hipSuccess) return HOMCOMP_OK;
    hc::note_hip_error((int)e);
    return HOMCOMP_ERR_HIP;
}

inline bool aligned(const void *p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
inline uintptr_t bytes_of(int type) { return type == HOMCOMP_F32 ? 4 : 2; }
inline bool eights_aligned(const void *p, int type, size_t row_stride, size_t head_stride)
{
    return aligned(p, 16) && (row_stride | head_stride) % (16 / bytes_of(type)) == 0;
}
inline bool type_ok(int type) { return type == HOMCOMP_BF16 || type == HOMCOMP_F16 || type == HOMCOMP_F32; }

// Blocks of a row, 0 where the shape is not supported.
int blocks_of(int kv_heads, int head_dim, int page_tokens)
{
    if (kv_heads < 1 || kv_heads > 1024) return 0;
    if (page_tokens < 32 || page_tokens > 65536 || (page_tokens & (page_tokens - 1))) return 0;
    return head_dim == 64 || head_dim == 128 || head_dim == 256 ? head_dim / 32 : 0;
}

// The shape alone: what a size query can look at.
int shape_of(const homcomp_cache *c, int *nb, int64_t *slots)
{
    if (!c) return HOMCOMP_ERR_INVALID_ARG;
    *nb = blocks_of(c->kv_heads, c->head_dim, c->page_tokens);
    if (!*nb || c->n_seqs < 0 || c->n_seqs > 65535 || c->n_pages > (size_t)INT32_MAX) return HOMCOMP_ERR_INVALID_ARG;
    if (c->table_stride > (size_t)kMostSlots / (size_t)c->page_tokens) return HOMCOMP_ERR_INVALID_ARG;
    *slots = (int64_t)c->table_stride * c->page_tokens;
    return HOMCOMP_OK;
}

int cache_args(const homcomp_cache *c, size_t max_length, hc::CacheArgs *a, int *nb)
{
    int64_t slots = 0;
    const int rc = shape_of(c, nb, &slots);
    if (rc) return rc;
    std::memset(a, 0, sizeof *a);
    a->n_seqs = c->n_seqs;
    if (c->n_seqs == 0) return HOMCOMP_OK;
    if ((c->n_pages && !c->d_pages) || !c->d_lengths || (c->table_stride && !c->d_table)) return HOMCOMP_ERR_INVALID_ARG;
    if (!aligned(c->d_pages, 16) || !aligned(c->d_table, 4) || !aligned(c->d_lengths, 4)) return HOMCOMP_ERR_ALIGNMENT;
    a->pages = (uint8_t *)c->d_pages;
    a->table = c->d_table;
    a->lengths = c->d_lengths;
    a->n_pages = (uint32_t)c->n_pages;
    a->table_stride = (uint32_t)c->table_stride;
    a->kv_heads = c->kv_heads;
    while ((1 << a->page_shift) < c->page_tokens) ++a->page_shift;
    a->max_slots = (int32_t)((int64_t)max_length < 0 || (int64_t)max_length > slots ? slots : (int64_t)max_length);
    return HOMCOMP_OK;
}

// `k`, `v`: what the store reads or the load writes.
int rows_call(bool store, const homcomp_cache *cache, void *k, void *v, int type, size_t row_stride, size_t head_stride,
              const int32_t *starts, size_t n_rows, void *stream)
{
    hc::CacheArgs c;
    int nb = 0;
    const int rc = cache_args(cache, SIZE_MAX, &c, &nb);
    if (rc) return rc;
    if (!type_ok(type)) return HOMCOMP_ERR_INVALID_ARG;
    if (n_rows > (size_t)INT32_MAX || ((int64_t)n_rows / 16 + 2 * (int64_t)cache->n_seqs) * cache->kv_heads > 4 * (kMostWorkgroups - 1)) return HOMCOMP_ERR_INVALID_ARG;
    if (c.n_seqs == 0 || n_rows == 0) return HOMCOMP_OK;
    if (!k || !v || !starts) return HOMCOMP_ERR_INVALID_ARG;
    if (!aligned(k, bytes_of(type)) || !aligned(v, bytes_of(type)) || !aligned(starts, 4)) return HOMCOMP_ERR_ALIGNMENT;
    if (!store && k == v) return HOMCOMP_ERR_INVALID_ARG;
    const bool eights = eights_aligned(k, type, row_stride, head_stride) && aligned(v, 16);
    const hc::RowsArgs r = {k, v, row_stride, head_stride, starts, (int32_t)n_rows, eights ? 1 : 0};
    return launched(store ? hc::launch_cache_store(c, r, nb, type, (hipStream_t)stream) : hc::launch_cache_load(c, r, nb, type, (hipStream_t)stream));
}

// Shapes of an attention call: column tiles, parts, scratch memory.
struct AttendPlan {
    int tiles, columns, splits, split_records, wide_tiles, tiles_in_wide;
    size_t partial_bytes, sums_bytes, lse_bytes, left_bytes;
};

int plan_attention(const homcomp_cache *c, const homcomp_attention *t, int nb, int64_t slots, AttendPlan *p)
{
    std::memset(p, 0, sizeof *p);
    p->splits = 1;
    if (!type_ok(t->type) || t->q_heads < 1 || t->q_heads % c->kv_heads || t->q_heads / c->kv_heads > 256) return HOMCOMP_ERR_INVALID_ARG;
    if (t->n_rows > (size_t)(INT32_MAX / t->q_heads) || t->max_rows > t->n_rows || !std::isfinite(t->scale)) return HOMCOMP_ERR_INVALID_ARG;
    if ((t->d_weights && t->weight_stride < t->max_length) || (t->d_prior && !t->d_weights)) return HOMCOMP_ERR_INVALID_ARG;
    const int group = t->q_heads / c->kv_heads;
    const int64_t most = (int64_t)t->max_length < 0 || (int64_t)t->max_length > slots ? slots : (int64_t)t->max_length;
    p->tiles = (int)(((int64_t)t->max_rows * group + hc::kColumns - 1) / hc::kColumns);
    p->columns = p->tiles == 1 ? (int)((int64_t)t->max_rows * group) : hc::kColumns;
    int64_t span = most;
    if (t->window && t->window < (size_t)most && (int64_t)(t->window + t->max_rows) < most) span = (int64_t)(t->window + t->max_rows);
    int64_t records = (span + 31) / 32 + 1;   // a window can begin inside a record
    if (records > (most + 31) / 32) records = (most + 31) / 32;
    if (records < 1) records = 1;
    const int64_t units = (int64_t)c->n_seqs * c->kv_heads * p->tiles;
    // more columns than a tile: records are unpacked once for up to 4, 8 or 16 tiles (rows of 256 values leave no room for two tiles
    // a wave); 32-bit results need more than float16 values
    if (p->tiles > 1 && t->type != HOMCOMP_F32) {
        p->tiles_in_wide = p->tiles <= 4 ? 4 : (p->tiles <= 8 || nb == 8 ? 8 : 16);
        p->wide_tiles = (p->tiles + p->tiles_in_wide - 1) / p->tiles_in_wide;
    }
    const int64_t groups = p->wide_tiles ? (int64_t)c->n_seqs * c->kv_heads * p->wide_tiles : units;   // workgroups without parts
    // Two workgroups for every compute unit, which is what one holds at once, as far as that leaves a wave two records (a short sequence: 1 x 4000 slots takes
    // 11 us, with eight a wave 17).  Where that makes parts of more than 128 records of several sequences: up to eight a unit, of 64 records at least, as
    // units would be idle behind the shorter ones (a single sequence has none: 1 x 524288 takes 125 us whole, 151 cut).
    // 8 heads of 128 values, four columns, us:
    //                          1 x 131072   2 x 131072   4 x 65536   16 x 16384*   64 x 4096*   128 x 4096   32 x 16384*   64 x 8192*   64 x 8192
    //   two a unit, or cut         45           70          69           61            51           126           84          107          140
    //   two a unit                 45           69          69           61            51           127          108          105          124
    //   four                       51           75          75           57            57           129           89          112          134
    //   eight                      53           87          83           63            56           145           84          107          141
    // (* lengths from a tenth to all of it.)
    int64_t splits = groups ? (2 * kComputeUnits + groups - 1) / groups : 1;
    const int64_t fine = (records + 2 * hc::kAttendWaves - 1) / (2 * hc::kAttendWaves);
    if (splits > fine) splits = fine;
    int64_t each = (records + splits - 1) / splits;
    if (!p->wide_tiles && c->n_seqs > 1 && groups > 0 && each > 128) {
        int64_t more = (8 * kComputeUnits + groups - 1) / groups;
        if (more > records / 64) more = records / 64;
        each = (records + more - 1) / more;
    }
    each = (each + hc::kAttendWaves - 1) / hc::kAttendWaves * hc::kAttendWaves;
    p->split_records = (int)each;
    p->splits = (int)((records + each - 1) / each);
    // (k_cache_attend, k_cache_join; of k_cache_weights, which takes a few batches for every sequence and head, the batches' number)
    if (units * p->splits > kMostWorkgroups || units * p->columns > kMostWorkgroups) return HOMCOMP_ERR_INVALID_ARG;
    if ((int64_t)c->n_seqs * c->kv_heads > kMostWorkgroups / 2 || (int64_t)c->n_seqs * c->kv_heads * ((most + 31) / 32) > INT32_MAX) return HOMCOMP_ERR_INVALID_ARG;
    if (p->splits > 1) {
        const size_t parts = (size_t)units * (size_t)p->splits * hc::kColumns;
        p->partial_bytes = parts * (size_t)(32 * nb) * sizeof(float);
        p->sums_bytes = parts * 2 * sizeof(float);
    }
    if (p->wide_tiles) p->left_bytes = (size_t)groups * (size_t)p->splits * sizeof(uint32_t);
    if (t->d_weights && !t->d_lse) p->lse_bytes = (t->n_rows * (size_t)t->q_heads * sizeof(float) + 15) / 16 * 16;
    return HOMCOMP_OK;
}

}  // namespace

extern "C" {

size_t homcomp_cache_page_bytes(int kv_heads, int head_dim, int page_tokens)
{
    const int nb = blocks_of(kv_heads, head_dim, page_tokens);
    return (size_t)hc::record_bytes(nb) * (size_t)(page_tokens / 32) * (size_t)kv_heads * (nb ? 1 : 0);
}

int homcomp_cache_store(const homcomp_cache *cache, const void *d_k, const void *d_v, int type, size_t row_stride, size_t head_stride,
                        const int32_t *d_starts, size_t n_rows, void *stream)
{
    return rows_call(true, cache, (void *)d_k, (void *)d_v, type, row_stride, head_stride, d_starts, n_rows, stream);
}

int homcomp_cache_load(const homcomp_cache *cache, void *d_k, void *d_v, int type, size_t row_stride, size_t head_stride,
                       const int32_t *d_starts, size_t n_rows, void *stream)
{
    return rows_call(false, cache, d_k, d_v, type, row_stride, head_stride, d_starts, n_rows, stream);
}

size_t homcomp_cache_attend_scratch(const homcomp_cache *cache, const homcomp_attention *attention)
{
    int nb = 0;
    int64_t slots = 0;
    AttendPlan p;
    if (!attention || shape_of(cache, &nb, &slots) || plan_attention(cache, attention, nb, slots, &p)) return 0;
    return p.partial_bytes + p.sums_bytes + p.lse_bytes + p.left_bytes;
}

int homcomp_cache_attend(const homcomp_cache *cache, const homcomp_attention *t, void *stream)
{
    if (!t) return HOMCOMP_ERR_INVALID_ARG;
    hc::AttendArgs a;
    std::memset(&a, 0, sizeof a);
    int nb = 0;
    int64_t slots = 0;
    AttendPlan p;
    int rc = shape_of(cache, &nb, &slots);
    if (!rc) rc = cache_args(cache, t->max_length, &a.c, &nb);
    if (!rc) rc = plan_attention(cache, t, nb, slots, &p);
    if (rc) return rc;
    if (a.c.n_seqs == 0) return HOMCOMP_OK;
    if (!t->d_starts || !aligned(t->d_starts, 4)) return t->d_starts ? HOMCOMP_ERR_ALIGNMENT : HOMCOMP_ERR_INVALID_ARG;
    if (!aligned(t->d_lse, 4) || !aligned(t->d_prior, 4) || !aligned(t->d_weights, 4) || !aligned(t->d_scratch, 16)) return HOMCOMP_ERR_ALIGNMENT;
    if (p.tiles > 0) {
        if (!t->d_q || !t->d_out || t->d_q == t->d_out) return HOMCOMP_ERR_INVALID_ARG;
        if (t->d_lse && (t->d_lse == t->d_weights || t->d_lse == t->d_out)) return HOMCOMP_ERR_INVALID_ARG;
        if (!aligned(t->d_q, bytes_of(t->type)) || !aligned(t->d_out, bytes_of(t->type))) return HOMCOMP_ERR_ALIGNMENT;
    }
    const size_t need = p.partial_bytes + p.sums_bytes + p.lse_bytes + p.left_bytes;
    if (need && (!t->d_scratch || t->scratch_bytes < need)) return HOMCOMP_ERR_INVALID_ARG;
    a.q = t->d_q;
    a.out = t->d_out;
    a.q_row_stride = t->q_row_stride;
    a.q_head_stride = t->q_head_stride;
    a.out_row_stride = t->out_row_stride;
    a.out_head_stride = t->out_head_stride;
    a.starts = t->d_starts;
    a.n_rows = (int32_t)t->n_rows;
    a.max_rows = (int32_t)t->max_rows;
    a.group = t->q_heads / cache->kv_heads;
    a.tiles = p.tiles;
    a.splits = p.splits;
    a.split_records = p.split_records;
    a.q_aligned = eights_aligned(t->d_q, t->type, t->q_row_stride, t->q_head_stride) ? 1 : 0;
    a.causal = t->causal ? 1 : 0;
    a.window = t->window > (size_t)kMostSlots ? 0 : (int32_t)t->window;   // (no slot is that far away)
    a.scale = std::frexp(t->scale, &a.scale_exponent) * 1.4426950408889634f;
    a.lse = p.lse_bytes ? (float *)((uint8_t *)t->d_scratch + p.partial_bytes + p.sums_bytes) : t->d_lse;
    a.partial = (float *)t->d_scratch;
    a.partial_sums = (float *)((uint8_t *)t->d_scratch + p.partial_bytes);
    a.columns = p.columns;
    a.wide_tiles = p.wide_tiles;
    a.tiles_in_wide = p.tiles_in_wide;
    if (p.wide_tiles) a.left_over = (uint32_t *)((uint8_t *)t->d_scratch + p.partial_bytes + p.sums_bytes + p.lse_bytes);
    a.prior = t->d_prior;
    a.weights = t->d_weights;
    a.weight_stride = t->weight_stride;
    return launched(hc::launch_cache_attend(a, nb, t->type, (hipStream_t)stream));
}

int homcomp_cache_evict(const homcomp_cache *cache, const homcomp_eviction *t, void *stream)
{
    if (!t) return HOMCOMP_ERR_INVALID_ARG;
    hc::EvictArgs a;
    std::memset(&a, 0, sizeof a);
    int nb = 0;
    const int rc = cache_args(cache, t->max_length, &a.c, &nb);
    if (rc) return rc;
    if (t->keep < 1 || t->keep > (size_t)kMostSlots || t->first > t->keep || t->recent > t->keep - t->first) return HOMCOMP_ERR_INVALID_ARG;
    if (t->to_table_stride > (size_t)kMostSlots / (size_t)cache->page_tokens || t->keep > t->to_table_stride * (size_t)cache->page_tokens)
        return HOMCOMP_ERR_INVALID_ARG;
    if (t->weight_stride < t->max_length || (int64_t)cache->n_seqs * cache->kv_heads * (int64_t)((t->keep + 127) / 128) > kMostWorkgroups ||
        (int64_t)cache->n_seqs * cache->kv_heads > kMostWorkgroups / 4)
        return HOMCOMP_ERR_INVALID_ARG;
    if (a.c.n_seqs == 0) return HOMCOMP_OK;
    if (!t->d_weights || !t->d_to_table || !t->d_to_lengths || !t->d_to_weights || !t->d_kept) return HOMCOMP_ERR_INVALID_ARG;
    if (t->d_to_lengths == cache->d_lengths || t->d_to_weights == t->d_weights || t->d_to_table == cache->d_table ||
        (const void *)t->d_kept == t->d_weights || (const void *)t->d_kept == t->d_to_weights)
        return HOMCOMP_ERR_INVALID_ARG;
    if (!aligned(t->d_weights, 4) || !aligned(t->d_to_table, 4) || !aligned(t->d_to_lengths, 4) || !aligned(t->d_to_weights, 4) || !aligned(t->d_kept, 4))
        return HOMCOMP_ERR_ALIGNMENT;
    a.weights = t->d_weights;
    a.weight_stride = t->weight_stride;
    a.keep = (int32_t)t->keep;
    a.first = (int32_t)t->first;
    a.recent = (int32_t)t->recent;
    a.to_table = t->d_to_table;
    a.to_table_stride = (uint32_t)t->to_table_stride;
    a.to_lengths = t->d_to_lengths;
    a.to_weights = t->d_to_weights;
    a.kept = t->d_kept;
    return launched(hc::launch_cache_evict(a, nb, (hipStream_t)stream));
}

}  // extern "C"
