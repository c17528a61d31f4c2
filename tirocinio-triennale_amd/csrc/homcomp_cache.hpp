// Host-visible launch interface of the 4-bit cache kernels, and the geometry both sides share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hc {

void note_hip_error(int error);   // for homcomp_last_hip_error

constexpr int kRecordSlots = 32;        // slots of a record (include/homcomp_cache.h)
constexpr int kColumns = 16;            // query columns (row, head of the group) of one tile of the attention kernel
constexpr int kAttendWaves = 4;         // waves of its workgroup; the records of a split are dealt out to them in turn

constexpr uint32_t record_bytes(int nb) { return 1280u * (uint32_t)nb; }

struct CacheArgs {
    uint8_t *pages;
    const int32_t *table;
    const int32_t *lengths;
    uint32_t n_pages;
    uint32_t table_stride;
    uint32_t page_shift;        // log2 of page_tokens
    int32_t kv_heads;
    int32_t n_seqs;
    int32_t max_slots;          // lengths are cut to this
};

struct RowsArgs {
    void *k, *v;                // read by the store, written by the load
    uint64_t row_stride, head_stride;
    const int32_t *starts;
    int32_t n_rows;
    int32_t aligned;            // every eight numbers lie at a multiple of 16 bytes
};

struct AttendArgs {
    CacheArgs c;
    const void *q;
    void *out;
    uint64_t q_row_stride, q_head_stride, out_row_stride, out_head_stride;
    const int32_t *starts;
    int32_t n_rows, max_rows;
    int32_t group;              // query heads of a key/value head
    int32_t tiles;              // column tiles a sequence's rows can take
    int32_t splits;             // parts the records are cut into, and
    int32_t split_records;      // records of a part, a multiple of kAttendWaves
    int32_t q_aligned;          // every eight numbers of q lie at a multiple of 16 bytes
    int32_t causal, window;     // window 0: none
    float scale;                // of the scores, times log2 e: scale 2^scale_exponent
    int32_t scale_exponent;
    float *lse;                 // null: not wanted
    float *partial;             // of more than one split: [tile][kColumns][split][head_dim], means
    float *partial_sums;        // [tile][kColumns][split][2]: exponent the part is relative to, sum
    int32_t columns;            // columns that a tile can have
    int32_t wide_tiles;         // tiles of many columns that a sequence's rows can take, 0: not that kernel
    int32_t tiles_in_wide;      // of kColumns: 4, 8 or 16
    uint32_t *left_over;        // [sequence, head, wide tile][split]: 1 where the columns are left to the other kernel
    const float *prior;
    float *weights;
    uint64_t weight_stride;
};

struct EvictArgs {
    CacheArgs c;
    const float *weights;
    uint64_t weight_stride;
    int32_t keep, first, recent;
    const int32_t *to_table;
    uint32_t to_table_stride;
    int32_t *to_lengths;
    float *to_weights;
    int32_t *kept;
};

// nb: blocks of a row (head_dim / 32: 2, 4 or 8); type: HOMCOMP_BF16, HOMCOMP_F16 or HOMCOMP_F32.
hipError_t launch_cache_store(const CacheArgs &c, const RowsArgs &r, int nb, int type, hipStream_t s);
hipError_t launch_cache_load(const CacheArgs &c, const RowsArgs &r, int nb, int type, hipStream_t s);
hipError_t launch_cache_attend(const AttendArgs &a, int nb, int type, hipStream_t s);
hipError_t launch_cache_evict(const EvictArgs &e, int nb, hipStream_t s);

}  // namespace hc
