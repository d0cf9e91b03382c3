/* forge_kv4.h — a KV cache held in 4 bits, and the flash-decode that reads it.
 *
 * The int4 weights' format (stdlib/flame/quant_lib.hexa:33-129, codes q + 7)
 * applied to cached K and V rows: every 64 dims of a row share one bf16
 * scale s = amax / 7 (1 for a group of zeros), a code is x / s rounded to the
 * nearest integer (halves away from zero, -7..7) plus 7, and a byte holds two
 * codes, the even dim in its low nibble: the codes and scales that
 * forge_q4_quantize_bf16 gives with group 64. A group that holds a NaN or an
 * infinity gets a NaN scale, so it reads back as NaN. 4.25 bits a value: a
 * quarter of the bf16 cache's bytes. The reference has no cache in 4 bits
 * (its decode keeps f32 rows, tool/decode_eager_baseline.cu).
 *
 * Layout: codes [slab][n_kv_head][rows][head_dim / 2] bytes and scales
 * [slab][n_kv_head][rows][head_dim / 64] bf16, for K and for V. A slab is a
 * sequence of lmax rows (contiguous, table NULL) or a page of page_tokens
 * rows of a pool of num_pages (row r of a sequence is row r % page_tokens of
 * page table[seq][r / page_tokens]; the page ids come from forge_paged_kv.h's
 * allocator). All arrays are the caller's, in memory of the current device,
 * 16-byte aligned. lmax and page_tokens are multiples of 8.
 *
 * Every entry is asynchronous on `stream` and returns 0 or a FORGE_* code. A
 * position, sequence or page id that only the device can see to be out of
 * range sets the error word that forge_ops_check() reads; such a row is not
 * written by append and reads as NaN. Every call may be captured into a graph
 * (the descriptor is copied, the arrays it names are not); the first call of
 * any per-op entry on a device allocates that word and comes before a
 * capture. */
#ifndef FORGE_KV4_H
#define FORGE_KV4_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FORGE_KV4_GROUP 64

typedef struct ForgeKv4 {
    uint8_t *k, *v;        /* codes                                          */
    uint16_t *ks, *vs;     /* scales, bf16                                   */
    const int32_t* table;  /* [n_seq][max_pages] page ids, NULL: contiguous  */
    int32_t n_seq;         /* sequences (slabs, or rows of the table)        */
    int32_t n_kv_head, head_dim; /* head_dim 64 or 128                       */
    int32_t lmax;          /* contiguous: rows a sequence can hold           */
    int32_t page_tokens, max_pages, num_pages; /* paged                      */
} ForgeKv4;

/* Quantises n_rows rows and writes them to the cache: row r of k and v
 * (bf16, ld elements from row to row, head h at h * head_dim) becomes
 * position pos[r] of sequence seq[r] (seq NULL: sequence r). A negative
 * pos[r] leaves row r out (padding). k and v are 16-byte aligned, ld a
 * multiple of 8. Two rows of one call may not name the same position. */
int forge_kv4_append(const ForgeKv4* cache, const uint16_t* k, const uint16_t* v, int64_t ld, const int32_t* seq,
                     const int32_t* pos, int n_rows, void* stream);

/* The values of n_rows cached rows, named as for append, into k_out and v_out
 * (fp32, ld elements from row to row, 16-byte aligned, ld a multiple of 4):
 * exact, code - 7 times the scale. Rows left out (pos[r] < 0) stay as they
 * were. */
int forge_kv4_read(const ForgeKv4* cache, const int32_t* seq, const int32_t* pos, int n_rows, float* k_out,
                   float* v_out, int64_t ld, void* stream);

/* Flash-decode over the cache: out[b] = softmax(q[b] K^T / sqrt(head_dim)) V
 * over positions 0..pos[b] of sequence seq[b] (seq NULL: sequence b), query
 * head h reading KV head h / (H / n_kv_head). q and out [B][H * head_dim]
 * fp32, 16-byte aligned; H a multiple of n_kv_head; scores, softmax and sums
 * in fp32. The products are on the tensor cores in integers, exactly: q is
 * rounded to 23 bits of its head's largest channel, and the weights (a key's
 * probability times its V's scale) of 64 keys to 23 bits of their largest for a
 * head and group of 64 dims, so an output's error is relative to the sum of the
 * weighted rows' largest values in the group (or to 2^-100 where that is less).
 * A probability below 2^-126 of the largest counts as 0.
 * A scale of V that is NaN or negative, which append does not write, makes the
 * group's output NaN. pos[b] < 0: an
 * empty sequence, its output is zeros (a padded batch). A position beyond the
 * cache, or a page outside the pool, sets the error word and makes the
 * sequence's output NaN.
 * workspace: forge_flash_decode_kv4_workspace_bytes(...) bytes, 16-byte
 * aligned, zeroed once before first use (every call leaves its counters at
 * zero, unless a wait ran out, which forge_ops_check() reports: zero it again
 * then); one for the largest batch serves smaller ones of the same heads and
 * head_dim. Calls that may overlap on the GPU, captured graphs among them,
 * need a workspace each. */
int64_t forge_flash_decode_kv4_workspace_bytes(int B, int H, int n_kv_head, int head_dim);
int forge_flash_decode_kv4(const float* q, const ForgeKv4* cache, const int32_t* seq, const int32_t* pos, int B, int H,
                           float* out, void* workspace, void* stream);

#ifdef __cplusplus
}
#endif
#endif
