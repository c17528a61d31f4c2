/*
 * homcomp_cache.h -- key/value rows held in 4 bits, and the operators that work on them
 * (libhomcomp_amd.so, beside homcomp.h).
 *
 * A stream of homcomp.h has blocks of varying length behind one global scan; no row of it can be written
 * or read alone.  This is the codec's other form: blocks of 32 values again, quantised to integers, with an error bound that
 * holds, but of one size each, in pages that sequences own, so that a decoder's keys and values can
 * be appended to, attended to and evicted one row at a time without leaving their 4 bits.  The
 * reference has no counterpart.
 *
 * A block of 32 values x of one row:
 *   lo  the largest bfloat16 not above min x
 *   s   the smallest float16 not below (max x - lo) / 15
 *   c   how many of the fifteen borders lo + (j + 1/2) s, j = 0..14, are <= x   (0 where s = 0)
 *   the block stands for x' = lo + s c, and |x - x'| <= s / 2 for every value of it.
 *   A block that holds a NaN or an infinity, or needs s > 65504, reads back as 32 NaNs (s = NaN, lo = 0, c = 0).
 * Five bits a value: 4 for c, 1/2 each for s and lo.
 *
 * A record holds the keys and values of 32 consecutive slots of one head, nb = head_dim / 32 blocks each, 1280 nb bytes:
 *   at 0         keys' codes    slot t, then group g = 0..3, then block b: a 32-bit word whose bits 4 p + 16 h hold the code of value
 *                               32 b + 8 g + 2 p + h        (p = 0..3, h = 0..1)
 *   512 nb       values' codes  slots 8 o .. 8 o + 7 together, then unit u = 0 .. 16 nb / 2 - 1, then slot: a 16-bit word
 *                               whose bits 4 p hold the code of value 64 (u / 16) + 16 p + u % 16
 *   1024 nb      keys' s        slots 8 o .. 8 o + 7 together, then block, then slot: float16
 *   1088 nb      values' s      likewise
 *   1152 nb      keys' lo       slot, then block: bfloat16
 *   1216 nb      values' lo     slots 8 o .. 8 o + 7 together, then block, then slot: bfloat16
 * A page holds, for every head in turn, page_tokens / 32 records.  Slot j of sequence s lies in page
 * d_table[s * table_stride + j / page_tokens].
 *
 * Conventions
 *   - All data pointers are device pointers of the current device; d_pages is 16-byte aligned, numbers
 *     are aligned to their size.  `stream` is a hipStream_t passed as void*.  Nothing blocks, allocates or synchronises, so
 *     every call can be recorded into a graph.  Every function returns HOMCOMP_OK or a negative HOMCOMP_ERR_* code (homcomp.h);
 *     arguments are checked before anything is enqueued.
 *   - Rows of a batch are packed: those of sequence s are starts[s] .. starts[s + 1] - 1, and they are the LAST ones of the d_lengths[s]
 *     slots it holds (store first, with the lengths that count the new rows).  starts does not fall.  Rows at and behind
 *     starts[n_seqs] are padding: neither read nor written.
 *   - Table entries outside 0 .. n_pages - 1 name no page: their slots are not stored, load as zeros, are not attended
 *     to and are evicted as zeros.  A length is cut to what a row of the table can hold, a negative one is 0.  What lies behind a
 *     sequence's last slot is never part of a result.
 *   - Two calls that touch the same slots or the same scratch memory have to be ordered by the caller (one stream, or events).
 *     Sequences may have pages in common; rows that one call writes must have slots of their own.
 *   - Rows of numbers that a call writes (of out, or of the arrays that a load fills) share no memory, with one another or with what it reads.
 *   - A call of more workgroups than a launch can have (2^24 - 1 of 256 threads) is refused.
 *   - A row in front of a sequence's first slot (more rows than slots) has none: it is not stored, a load leaves it as it was, and it sees what its
 *     place says (nothing where `causal`).
 */
#ifndef HOMCOMP_CACHE_H
#define HOMCOMP_CACHE_H

#include "homcomp.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of the numbers outside the cache. */
#define HOMCOMP_BF16 0
#define HOMCOMP_F16 1
#define HOMCOMP_F32 2

typedef struct homcomp_cache {
    void *d_pages;            /* n_pages * homcomp_cache_page_bytes(...) bytes */
    size_t n_pages;           /* below 2^31 */
    int kv_heads;             /* 1 .. 1024 */
    int head_dim;             /* 64, 128 or 256 */
    int page_tokens;          /* a power of two, 32 .. 65536 */
    int n_seqs;               /* 0 .. 65535; with 0 a call does nothing */
    const int32_t *d_table;   /* [n_seqs][table_stride] */
    size_t table_stride;      /* pages a sequence can have; times page_tokens below 2^31 - 64 */
    const int32_t *d_lengths; /* [n_seqs] */
} homcomp_cache;

/* Bytes of a page, 0 where the shape is not supported. */
size_t homcomp_cache_page_bytes(int kv_heads, int head_dim, int page_tokens);

/* Quantises rows into their slots, and reads rows back as numbers.  Row r, head h of the keys begins at element
 * r * row_stride + h * head_stride of d_k, its head_dim values are adjacent; the values' rows likewise.  n_rows:
 * rows the arrays hold (rows at and behind it are taken as padding whatever d_starts says). */
int homcomp_cache_store(const homcomp_cache *cache, const void *d_k, const void *d_v, int type, size_t row_stride, size_t head_stride,
                        const int32_t *d_starts, size_t n_rows, void *stream);
int homcomp_cache_load(const homcomp_cache *cache, void *d_k, void *d_v, int type, size_t row_stride, size_t head_stride,
                       const int32_t *d_starts, size_t n_rows, void *stream);

/* Attention over the cache.  Row i of the n rows of a sequence that holds L slots is at slot a = L - n + i.  It sees the slots j < L,
 * with `causal` those j <= a, with a window w > 0 those j > a - w.  With S_j = scale * <q, k_j>:
 *   lse = log sum_j exp S_j      out = sum_j exp(S_j - lse) v_j
 * A row that sees no slot gets out = 0 and lse = -infinity.  Scores have to stay below 2^127 in size.  Query head g reads the keys and values of head
 * g / (q_heads / kv_heads).
 * d_weights (optional): weights[s][h][j] = prior[s][h][j] + the sum of exp(S_j - lse) over the sequence's rows and the query heads of
 * head h, for the slots j < L; what lies behind is left as it was.  d_prior NULL: 0; d_prior may be d_weights.  The sum is
 * taken in a fixed order: the same inputs give the same bits.  A weight is exp(S_j - lse) with lse in 32 bits, at most 1: it loses digits where scores
 * exceed 2^16. */
typedef struct homcomp_attention {
    const void *d_q;          /* row r, query head g at element r * q_row_stride + g * q_head_stride */
    size_t q_row_stride, q_head_stride;
    void *d_out;              /* the same, of out's strides; not d_q */
    size_t out_row_stride, out_head_stride;
    int type;                 /* of q and out */
    int q_heads;              /* a multiple of kv_heads; q_heads / kv_heads at most 256 */
    const int32_t *d_starts;  /* [n_seqs + 1] */
    size_t n_rows;            /* rows the arrays hold; below 2^31 / q_heads */
    size_t max_rows;          /* no sequence has more rows than this (those beyond it are left out), at most n_rows */
    size_t max_length;        /* no sequence holds more slots than this (a longer one is cut to its first max_length) */
    float scale;              /* finite */
    int causal;
    size_t window;            /* 0: none.  Slots are counted, not positions: of evicted sequences it is that many of the slots left */
    float *d_lse;             /* [n_rows][q_heads], optional; memory of its own */
    const float *d_prior;     /* [n_seqs][kv_heads][weight_stride], optional */
    float *d_weights;         /* the same, optional */
    size_t weight_stride;     /* at least max_length where weights are asked for */
    void *d_scratch;          /* 16-byte aligned, homcomp_cache_attend_scratch bytes; of one call at a time */
    size_t scratch_bytes;
} homcomp_attention;

/* Scratch bytes that homcomp_cache_attend needs for these shapes (pointers are not looked at); 0 where the arguments are refused or
 * none is needed. */
size_t homcomp_cache_attend_scratch(const homcomp_cache *cache, const homcomp_attention *attention);
int homcomp_cache_attend(const homcomp_cache *cache, const homcomp_attention *attention, void *stream);

/* Eviction by the weights that homcomp_cache_attend gathers.  Of a sequence that holds L > keep slots every head keeps `keep` of its own
 * choice: the first `first`, the last `recent`, and of those between the keep - first - recent of the largest weight (of equal
 * ones those in front; a NaN counts as the smallest).  They go, in their order and as the bits they are, to the first slots of the pages
 * that d_to_table names.  A sequence of at most `keep` slots is moved whole.  The pages moved to must not be pages of any sequence's slots,
 * nor named twice; the old pages are left as they were.  n = min(L, keep):
 *   to_lengths[s] = n     kept[s][h][i] = the old slot of row i < n, -1 for i >= n       to_weights[s][h][i] = its weight, 0 for i >= n
 */
typedef struct homcomp_eviction {
    const float *d_weights;   /* [n_seqs][kv_heads][weight_stride] */
    size_t weight_stride;     /* at least max_length */
    size_t max_length;        /* as above */
    size_t keep;              /* 1 .. to_table_stride * page_tokens */
    size_t first, recent;     /* together at most keep */
    const int32_t *d_to_table; /* [n_seqs][to_table_stride] */
    size_t to_table_stride;
    int32_t *d_to_lengths;    /* [n_seqs]; not d_lengths */
    float *d_to_weights;      /* [n_seqs][kv_heads][keep]; not d_weights */
    int32_t *d_kept;          /* [n_seqs][kv_heads][keep]; neither of the two */
} homcomp_eviction;

int homcomp_cache_evict(const homcomp_cache *cache, const homcomp_eviction *eviction, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* HOMCOMP_CACHE_H */
