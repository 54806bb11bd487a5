/*
 * C ABI of libattn_b200_kv.so: a quantised, paged KV cache for decoding on NVIDIA B200 (sm_100a). Conventions as in attn_b200.h:
 * device pointers owned by the caller, launches on `stream`, 0 or an error code, the text of the calling thread's last error from
 * attn_b200_kv_last_error(); no device memory is allocated. No counterpart in the reference, whose operators take dense tensors.
 *
 * A position of a head of K or V is held as head_dim whole numbers n of 4 or 8 bits with a scale and a zero of the cache's type:
 *     zero = min x,  scale = round16((max x - min x) / N),  n = min(rint((x - zero) / scale), N),  N = 2^bits - 1
 * and stands for zero + scale n. scale = 0: n = 0. A row that holds an infinity or a NaN (or whose range exceeds fp32) stands
 * for NaN. Memory: data[num_pages][heads][page_size / 16][attn_b200_kv_block_bytes(bits, head_dim)], uninitialised memory is
 * fine: nothing is read that was not written, but for blocks of 16 positions of which some were (the rest has no influence).
 *
 * Sequences are rows of a table: entry i of row b is the page of positions [i page_size, (i + 1) page_size). Entries behind the
 * positions in use are never read and may hold anything. Tables, starts, counts and lengths are read on the device when the
 * kernels run: a captured launch sees their values at replay. What is out of range there (a page that does not exist, positions
 * behind the last entry, negative numbers) is left out: not written, read back as zeros, not attended to; and it sets a status
 * that makes later calls fail with ATTN_B200_KV_ERR_DEVICE until attn_b200_kv_status(1) has cleared it.
 * A page may stand in several rows for reading. Two rows that write the same position leave a mixture of both.
 */
#ifndef ATTN_B200_KV_H_
#define ATTN_B200_KV_H_

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ATTN_B200_KV_F16 0
#define ATTN_B200_KV_BF16 1
#define ATTN_B200_KV_ERR_DEVICE 4     /* the other codes are those of attn_b200.h as well */
#define ATTN_B200_KV_MAX_QUERIES 64   /* new positions of a sequence in one attn_b200_kv_attn call */

typedef struct {
  void* data;       /* 16-byte aligned */
  int num_pages, heads, page_size; /* page_size: a power of two from 16 on */
  int head_dim;     /* 64, 128 or 256 */
  int bits;         /* 4 or 8 */
  int dtype;        /* of k, v, q and o, and of the scales and zeros */
} attn_b200_kv_cache;

const char* attn_b200_kv_last_error(void);
/* Synchronises the current device. 0, 1 (a bounded wait expired), 3 (a page that does not exist), 4 (a length, start or count out
 * of range), -1 (the read failed). clear != 0 resets it. */
int attn_b200_kv_status(int clear);
/* Sets up the status words of the current device; the first launch does it too, but not inside a stream capture. */
int attn_b200_kv_prepare(void);
/* Bytes of a block of 16 positions of one head, K and V together; 0 for sizes that are not supported. */
int attn_b200_kv_block_bytes(int bits, int head_dim);

/* Writes positions start[b] + i, i < count[b] (count NULL: L), of every head from k, v [B, heads, L, head_dim]. Strides in elements
 * for batch, head and position, multiples of 8; channels are dense; pointers 16-byte aligned. B and heads up to 65535. */
int attn_b200_kv_write(const attn_b200_kv_cache* cache, const int* table, int table_stride, int table_width, const int* start,
                       const int* count, const void* k, const long long* k_strides, const void* v, const long long* v_strides, int B,
                       int L, void* stream);

/* Reads positions start[b] + i (start NULL: 0) back into dense k, v [B, heads, L, head_dim]; rows i >= count[b] are zeros. */
int attn_b200_kv_read(const attn_b200_kv_cache* cache, const int* table, int table_stride, int table_width, const int* start,
                      const int* count, void* k, void* v, int B, int L, void* stream);

/* o = softmax(q K^T scale) V over the first lengths[b] positions (the values before any rounding to 16 bits). q, o
 * [B, heads * group, Lq, head_dim] dense, query heads h * group ... of head h; lse [B, heads * group, Lq] or NULL. causal: query i
 * sees position j <= i + lengths[b] - Lq. A query that sees none gets 0 and -inf. Lq up to ATTN_B200_KV_MAX_QUERIES, B up to 4096.
 * workspace: attn_b200_kv_attn_workspace_bytes() bytes (0 where tables hold few positions; then NULL will do), 16-byte aligned,
 * contents undefined before and after; two calls that may run at the same time need one each. One or two launches, or that for each
 * part of a batch whose tables could hold more than 2^31 units of work (32 or 16 positions of a head for up to 16 rows); a single
 * sequence whose table could hold more is refused. The same call gives the same bits. */
size_t attn_b200_kv_attn_workspace_bytes(const attn_b200_kv_cache* cache, int table_width, int B, int group, int Lq);
int attn_b200_kv_attn(const void* q, const attn_b200_kv_cache* cache, const int* table, int table_stride, int table_width,
                      const int* lengths, void* o, float* lse, void* workspace, size_t workspace_bytes, int B, int group, int Lq,
                      float scale, int causal, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ATTN_B200_KV_H_ */
