/* C ABI of the operators around a growing cache: rotary positions, the append to a paged cache and attention over it.
 *
 * The conventions are those of sage_b200.h (libsage_b200.so exports both): device pointers on the current CUDA device,
 * sizes and strides in elements, work enqueued on `stream`, no allocation, no synchronisation, SAGE_OK or a SAGE_ERR_*
 * code with sage_last_error().  Base pointers are 16-byte aligned and strides multiples of 8 elements.
 * The reference has no counterpart of anything in this file.
 */
#ifndef SAGE_PAGED_B200_H_
#define SAGE_PAGED_B200_H_

#include <stdint.h>

#include "sage_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SAGE_DTYPE_F32 2             /* sage_apply_rotary only */

/* Status codes that the kernels of this file write, next to those of sage_b200.h: arguments of one call.  Unlike those they
 * stop neither the call nor one behind it, and give way to them in the word; otherwise the first code stays. */
#define SAGE_STATUS_BAD_PAGE 3       /* a page index outside the cache */
#define SAGE_STATUS_BAD_LENGTH 4     /* more keys than the row of the page table holds, or more new tokens than keys */

#define SAGE_MAX_ROTARY_AXES 4

/* Rotary positions.  The pairs of a head, (x[i], x[i + pairs]) or, interleaved, (x[2i], x[2i+1]), are turned by
 * freq[i] * positions[token][axis[i]].  freq is the angle per position in turns, as a fraction of 2^64: the product with
 * an integer position wraps at whole turns and is exact, so that only the rounding of freq itself (half of 2^-64 turns at best)
 * grows with the position.  pairs is a multiple of 8;
 * what a head has behind its pairs is copied. */
typedef struct sage_rotary {
  const uint64_t* freq;              /* [pairs], 16-byte aligned */
  const int32_t* axis;               /* [pairs], each below n_axes; 16-byte aligned */
  int pairs, n_axes, interleaved;
  const void* positions;             /* n_axes neighbouring integers per token */
  int positions_64;                  /* 0: int32, 1: int64 */
  int64_t stride_b, stride_s;        /* of positions */
} sage_rotary_t;

/* q_out = q turned, k_out = k turned ([B,H,S,D] in any strides; k and k_out may both be NULL, Hkv is 0 then).  inverse != 0
 * turns the other way: the gradient.  Outputs must not overlap inputs unless they are the same tensors.
 * dtype: fp16, bf16 or fp32.  D: 64 or 128, at least 2 * pairs. */
int sage_apply_rotary(const sage_strided_t* q, const sage_strided_t* q_out, const sage_strided_t* k, const sage_strided_t* k_out,
                      const sage_rotary_t* rotary, int dtype, int B, int Hq, int Hkv, int S, int D, int inverse, void* stream);

/* Keys and values in pages of page_size tokens, in any strides (head_dim contiguous).  page_size: 16, 32, 64, 128 or 256.
 * D: 64 or 128.  dtype: fp16 or bf16. */
typedef struct sage_paged_kv {
  void* k;
  void* v;
  int64_t k_stride_page, k_stride_slot, k_stride_head;
  int64_t v_stride_page, v_stride_slot, v_stride_head;
  int num_pages, page_size, Hkv, D, dtype;
} sage_paged_kv_t;

/* A batch of B sequences whose T new tokens lie one behind the other: those of sequence b are rows
 * [cu_q[b], cu_q[b+1]), or row b alone if cu_q is NULL (then T == B).  kv_lens[b] counts all keys of the sequence, the
 * new tokens included: new token i of n has position kv_lens[b] - n + i, and key j stands in slot j % page_size of page
 * page_table[b * table_stride + j / page_size].  All four arrays are int32 on the device and stay as they are until the call has completed.  Entries of the table behind the
 * last key are not looked at.  cu_q that leaves [0, T] or falls is clipped; rows that belong to no sequence are not written
 * (by sage_paged_append: zeroed).  Without cu_q a kv_lens of 0 is a slot that is not in use: nothing is stored for it, and
 * its rows are zero. */
typedef struct sage_paged_batch {
  const int32_t* page_table;
  int64_t table_stride;
  int table_width;
  const int32_t* kv_lens;
  const int32_t* cu_q;
  int B, T;
} sage_paged_batch_t;

/* Rows [T, H, D]. */
typedef struct sage_rows {
  const void* ptr;
  int64_t stride_t, stride_h;
} sage_rows_t;

/* Puts k and v of the new tokens into their slots; with `rotary` k is turned on the way, and so is q into q_out (q and q_out
 * may both be NULL, Hq is 0 then).  rotary->positions == NULL: the position in the sequence, for every axis.  A token whose
 * page or position is out of range is not stored, and `status` (optional) gets a code. */
int sage_paged_append(const sage_paged_kv_t* cache, const sage_paged_batch_t* batch, const sage_rows_t* k, const sage_rows_t* v,
                      const sage_rows_t* q, const sage_rows_t* q_out, int Hq, const sage_rotary_t* rotary, int* status, void* stream);

/* Attention of the new tokens over the cache: row t, head h of `o` = softmax(sm_scale q.k) v over the visible keys of the
 * token's sequence - all of them, or with is_causal those up to the token's own position - and of kv head h / (Hq / Hkv).
 * A row that sees no key is 0, its log-sum-exp -inf.
 * o: 16-bit rows like q, in any strides.  lse (optional): [T, Hq] fp32, contiguous, natural log.
 * Hq: a multiple of Hkv, at most 128 times it.  max_q: an upper bound of the new tokens of a sequence, 0 if not known (it
 * chooses the kernel; a wrong one costs time only).
 * shared_pages (optional): n_shared page indices on the device.  The first n_shared * page_size keys of EVERY sequence are
 * in these pages; the first n_shared columns of page_table are not looked at.  The result is the same as with them in
 * the table, but these keys and values are read once for all sequences.
 * zero_rest: rows of o (lse) that belong to no sequence are set to 0 (-inf); 0: they are left as they are.
 * workspace: sage_paged_workspace_bytes() bytes, 16-byte aligned; it belongs to the call until that has completed. */
int64_t sage_paged_workspace_bytes(const sage_paged_kv_t* cache, const sage_paged_batch_t* batch, int Hq, int max_q, int n_shared);
int sage_paged_attn(const sage_paged_kv_t* cache, const sage_paged_batch_t* batch, const sage_rows_t* q, const sage_rows_t* o, int Hq,
                    int max_q, int is_causal, float sm_scale, float* lse, const int32_t* shared_pages, int n_shared, int zero_rest,
                    int* status, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SAGE_PAGED_B200_H_ */
