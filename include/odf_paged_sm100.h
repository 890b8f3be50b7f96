/*
 * odf_paged_sm100.h -- C ABI of the paged key-value cache: attention of one new token,
 * appending tokens, copying pages, and the host-side page pool.
 *
 * A cache is a pool of `num_pages` pages per layer; a page holds `page_size` consecutive tokens
 * of one sequence for every kv-head.  A sequence's page table lists its pages in order: token j
 * is slot j % page_size of page table[j / page_size].  The serving counterpart of the forward
 * pass in odf_sm100.h: same statuses, score mods, GQA rule (kv_head = q_head / group), softmax and
 * LSE definition, and the same rules for calls: plain pointers and sizes, nothing throws, device
 * calls are asynchronous on `stream` (a cudaStream_t; NULL = legacy default stream), allocate
 * no device memory and read nothing back, so they can be captured into a CUDA graph after a first call.
 * The reference has no key-value cache; there is no counterpart to cite.
 *
 * Page ids and lengths live on the device, where the host cannot check them.  The kernels check
 * them themselves: an entry outside [0, num_pages) or a length beyond max_pages * page_size leads to no
 * access out of range; it sets ODF_ERR_BAD_PAGE in the status word (odf_device_status).
 */
#ifndef ODF_PAGED_SM100_H
#define ODF_PAGED_SM100_H

#include "odf_sm100.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ODF_ERR_BAD_PAGE 7  /* status word: a page id or a length was out of range (see above) */
#define ODF_ERR_NO_PAGES 8  /* page pool: not enough free pages; nothing was changed */

/* Element type of a cache besides ODF_DTYPE_BF16: 8-bit floats with 4 exponent and 3 mantissa
   bits (finite range +-448, one NaN), times the scale of their kv-head.  Not an
   onednn_flash::DataType. */
#define ODF_DTYPE_E4M3 16

typedef struct odf_paged_cache {
    void* k_pages;              /* [num_pages, heads_kv, page_size, head_dim], element strides below */
    void* v_pages;
    int32_t kv_dtype;           /* ODF_DTYPE_BF16 or ODF_DTYPE_E4M3 */
    int64_t num_pages, heads_kv, page_size, head_dim;  /* head_dim 64 or 128; page_size 1 .. 65536 */
    /* Element strides {page, head, slot}, positive multiples of 16 bytes; all zero = contiguous.
       {H*S*D, D, H*D} is the [page, slot, head] layout. */
    int64_t k_strides[3], v_strides[3];
    /* E4M3: device arrays [heads_kv], what one unit of a stored value is worth; NULL = 1. */
    const float* k_scale;
    const float* v_scale;
    const int32_t* page_table;  /* device [batch, max_pages]; entries past a sequence's length are not read */
    int64_t table_stride;       /* elements from one sequence's row to the next; 0 = max_pages */
    int64_t max_pages;
} odf_paged_cache;

/*
 * Attention of one new token per sequence.  Sequence b has lens[b] keys in the cache, the new
 * token's own included (append first), and the token sits at position p = lens[b] - 1:
 *   s_j = mod(q . k_j * scale), key j < lens[b] visible iff window == 0, or p - j < window, or
 *   j < sinks;   o = sum_j softmax(s)_j v_j,   lse = log sum_j exp(s_j)
 * with mod the ALiBi term slope[h] * (j - p) and the soft-cap of odf_fwd_params.  lens[b] <= 0
 * writes o = 0, lse = -inf.  K and V of keys that are not visible, and slots past a sequence's
 * end, may hold anything, NaN included.  Accumulation and softmax are fp32.
 * Limits (ODF_ERR_UNSUPPORTED past them): K pages, and V pages, of one layer span at most 64 GB; 256 explicit
 * slopes; batch below 2^23, heads_q below 2^16, batch x heads_q below 2^31; and
 *   (ceil(keys / S) + 12) x batch x heads_kv x ceil(heads_q / heads_kv / T)  is below 2^31,
 * with keys = max_pages * page_size (with a window at most window + sinks), S = 16 where a row of the cache has 256
 * bytes and 32 where it has fewer, T = 8 up to eight query heads to a kv-head and 16 from nine on.  Lengths must not
 * change while a call runs.  Results do not depend on timing: the same call gives the same bits.
 */
typedef struct odf_decode_params {
    const void* q;              /* bf16 [batch, heads_q, head_dim] */
    void* o;                    /* [batch, heads_q, head_dim] */
    float* lse;                 /* [batch, heads_q] contiguous, natural log; NULL = not wanted */
    int32_t o_dtype;            /* ODF_DTYPE_F32 or ODF_DTYPE_BF16 */
    int64_t batch, heads_q;
    int64_t q_strides[2], o_strides[2];  /* elements {batch, head}, multiples of 16 bytes; all zero = contiguous */
    const int32_t* lens;        /* device [batch] */
    odf_paged_cache cache;
    float scale;
    int64_t window, sinks;      /* window 0 = every key (sinks is then not read) */
    int32_t bias_kind;          /* ODF_BIAS_NONE or ODF_BIAS_ALIBI */
    const float* alibi_slopes;  /* as in odf_fwd_params (HOST array or NULL) */
    float softcap;
    /* Device scratch of odf_paged_decode_workspace_size() bytes, 16-byte aligned, zeroed by the
       caller once before its first use; every call leaves it ready for the next.  Calls that share
       one must not overlap on the GPU. */
    void* workspace;
    size_t workspace_bytes;
} odf_decode_params;

int odf_paged_decode_sm100(const odf_decode_params* p, void* stream);

/* Scratch bytes for these params: the same for every batch size and length. */
size_t odf_paged_decode_workspace_size(const odf_decode_params* p);

/*
 * Writes new keys and values into the cache: token t < counts[b] (every t < tokens when counts is
 * NULL) of sequence b goes to position starts[b] + t.  A bf16 cache gets them bit for bit; an E4M3
 * cache gets round-to-nearest-even of x / scale, saturated at +-448 (NaN stays NaN).  Rows t at or
 * past counts[b] are not read (a padded batch), other slots are left as they are.  No two tokens of
 * one call may go to the same slot.  Tokens whose page id is out of range are dropped.
 */
typedef struct odf_append_params {
    const void* k;              /* bf16 [batch, heads_kv, tokens, head_dim] */
    const void* v;
    int64_t batch, tokens;
    int64_t k_strides[3], v_strides[3];  /* elements {batch, head, token}, multiples of 16 bytes; all zero = contiguous */
    const int32_t* starts;      /* device [batch], >= 0 */
    const int32_t* counts;      /* device [batch] or NULL */
    odf_paged_cache cache;
} odf_append_params;

int odf_paged_append_sm100(const odf_append_params* p, void* stream);

/*
 * Copies pages pairs[2i] -> pairs[2i + 1] (HOST array of n_pairs pairs, copied into the launch) of
 * K and V in every one of `layers` layers, layer l at k_pages + l * k_layer_stride elements.  Every
 * id must be in [0, num_pages), no page may be written twice, and no written page may also be read
 * (ODF_ERR_INVALID_ARG otherwise; the check of more than 32 pairs takes num_pages bytes of host memory, which are
 * freed before the call returns).  n_pairs == 0 does nothing.  The cache's tables, scales and
 * page contents outside the written pages are not touched.
 */
typedef struct odf_page_copy_params {
    odf_paged_cache cache;
    int64_t layers, k_layer_stride, v_layer_stride;  /* strides are not read for one layer */
    const int32_t* pairs;
    int64_t n_pairs;
} odf_page_copy_params;

int odf_page_copy_sm100(const odf_page_copy_params* p, void* stream);

/*
 * Host-side page pool: which pages are free, how many sequences share each, and every sequence's
 * table.  No CUDA calls.  Not thread-safe: one pool is used by one thread at a time.  Copies that a
 * call asks for come back as (source, destination) pairs, which the caller hands to
 * odf_page_copy_sm100 before it writes the cache again.  The pairs of consecutive calls of extend may be
 * gathered into one copy; it has to run before any other call that changes the pool (fork, truncate, free, compact),
 * which may hand out a page that a pair still reads.
 */
typedef struct odf_page_pool odf_page_pool;

int odf_page_pool_create(int64_t num_pages, int64_t page_size, odf_page_pool** out);
void odf_page_pool_destroy(odf_page_pool* pool);
/* A new, empty sequence. */
int odf_page_pool_add(odf_page_pool* pool, int64_t* seq);
/* A new sequence with the same tokens, sharing every page of `seq`. */
int odf_page_pool_fork(odf_page_pool* pool, int64_t seq, int64_t* child);
/* Makes room for `tokens` more tokens.  A partly filled last page that is shared is replaced by a
   page of its own, and pair[0..1] says what to copy (*n_pairs 0 or 1). */
int odf_page_pool_extend(odf_page_pool* pool, int64_t seq, int64_t tokens, int32_t pair[2], int64_t* n_pairs);
/* Drops tokens past `length` (rejected drafts) and the pages that then hold none. */
int odf_page_pool_truncate(odf_page_pool* pool, int64_t seq, int64_t length);
/* Ends a sequence; its pages become free once no other sequence shares them. */
int odf_page_pool_free(odf_page_pool* pool, int64_t seq);
/* Moves pages so that the used ones are 0 .. used - 1 and rewrites the tables.  `pairs` has room for
   `room` pairs; at most min(used, free) are needed (ODF_ERR_INVALID_ARG, nothing changed, if it is less). */
int odf_page_pool_compact(odf_page_pool* pool, int32_t* pairs, int64_t room, int64_t* n_pairs);
/* Number of tokens of a sequence and of its pages. */
int odf_page_pool_length(const odf_page_pool* pool, int64_t seq, int64_t* tokens, int64_t* pages);
/* Writes the sequence's page ids, then -1 up to `max_pages` entries. */
int odf_page_pool_table(const odf_page_pool* pool, int64_t seq, int32_t* out, int64_t max_pages);
int64_t odf_page_pool_free_pages(const odf_page_pool* pool);

#ifdef __cplusplus
}
#endif

#endif /* ODF_PAGED_SM100_H */
