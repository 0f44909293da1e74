/*
 * kvdec_paged8.h -- C ABI of the paged 8-bit KV cache (libkvdec.so): rows of
 * K and V quantized as they are written, read back, and attended over.
 *
 * No counterpart in the reference, whose caches are contiguous and built once
 * (quant_kernel.py:584-622).  Conventions, error codes and element types as in
 * kvdec.h; nothing allocates, synchronises or keeps state.
 *
 * The cache.  Tokens live in pages shared by all sequences; token t of
 * sequence b is row t % page_size of page block_table[b * max_blocks +
 * t / page_size].  A row of a KV head is D = 128 one-byte codes; the codes of
 * `block_size` consecutive tokens of a KV head share one fp32 scale, and a
 * code stands for code * scale.
 */
#ifndef KVDEC_PAGED8_H_
#define KVDEC_PAGED8_H_

#include "kvdec.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- code types ------------------------------------------------------- */
#define KVDEC_I8 3               /* int8, written in -127..127                */
#define KVDEC_E4M3 4             /* OCP fp8 e4m3 (largest 448, NaN, no inf)   */

/*
 * A cache as the entry points take it (host memory, read during the call).
 *   k_pages, v_pages : codes; row r of page p, KV head h starts at byte
 *     p * page_stride + r * row_stride + h * head_stride; pointers and strides
 *     are multiples of 16, the strides shared by K and V, 16 rows within 2 GiB
 *   k_scales, v_scales : [num_pages, KVH, page_size / block_size] fp32
 *   block_table : [B, max_blocks] int32; an entry outside [0, num_pages) is no
 *     page: its tokens are not written, read as zeros, and weigh in attention
 *     as keys and values of zero
 *   seq_lens : [B] int32, the tokens of each sequence with its new ones (below
 *     0: 0).  Positions past the table have no page; attention has no keys there
 *   page_size : a power of two, 16 or more; block_size 16, 32, 64 or 128 and
 *     at most page_size; max_blocks * page_size < 2^30
 */
typedef struct kvdec_paged8_cache {
  void* k_pages;
  void* v_pages;
  float* k_scales;
  float* v_scales;
  const int32_t* block_table;
  const int32_t* seq_lens;
  int64_t num_pages, page_stride, row_stride, head_stride;
  int32_t code, KVH, D, page_size, block_size, max_blocks;
} kvdec_paged8_cache;

/*
 * New tokens.  cu_seqlens [B + 1] int32 on the device: the new tokens of
 * sequence b are rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 of the T rows that
 * a call takes or gives, and the last tokens of the sequence (positions
 * seq_lens[b] - n .. seq_lens[b] - 1; positions below 0 do not exist).  NULL:
 * one new token a sequence, T == B.  cu_seqlens[0] counts as 0, the others are
 * clamped into [0, T]; rows at and past cu_seqlens[B] belong to no sequence.
 */

/*
 * Quantize the new tokens' rows into the cache.
 *   k, v : [T, KVH, D] of dtype (KVDEC_F16, KVDEC_BF16, KVDEC_F32), strides in
 *     elements, the last dimension contiguous, rows on 16-byte boundaries.
 * With M the largest finite |x| of the call's rows of a block and head, need is
 * the least power of two >= 2^-100 with M <= need * (448 for e4m3, 127 for
 * int8).  A block whose first token is among the call's takes scale = need;
 * any other takes max(old scale, need), and where that grows the codes of its
 * earlier tokens become round(code * old / scale).  code = round(x / scale),
 * ties to even.  Since scales are powers of two the quotients are exact, and a
 * token's codes are off by less than one step however often its block grows.
 * A NaN or infinite x becomes the NaN code of e4m3; int8 has none, so there
 * the scale of its block becomes NaN, until the block is written from its
 * first token again (codes of the call's tokens in it: 0).
 * Rows of the cache that no new token names are left as they are.  Pages that
 * two sequences of the call write to hold neither's tokens for certain.
 */
int kvdec_paged8_write(const kvdec_paged8_cache* cache, const void* k, const void* v, int dtype,
                       int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                       int64_t v_head_stride, const int32_t* cu_seqlens, int64_t B, int64_t T,
                       void* stream);

/*
 * The new tokens' rows read back: k_out, v_out [T, KVH, D] of dtype,
 * code * scale rounded once; zeros for rows of no sequence or no page.
 */
int kvdec_paged8_read(const kvdec_paged8_cache* cache, const int32_t* cu_seqlens, int64_t B, int64_t T,
                      void* k_out, void* v_out, int dtype, void* stream);

/*
 * Causal GQA attention of the new tokens over the cache, which holds them
 * already: query head h of the token at position i attends with KV head
 * h / (H / KVH) to the positions p <= i, and with window > 0 only to
 * p > i - window and p < sink.
 *   q, o : [T, H, D] of dtype (KVDEC_F16 or KVDEC_BF16); q's strides in
 *     elements, rows on 16-byte boundaries; o contiguous
 *   o = softmax(q k^T * sm_scale) v, fp32 softmax and accumulation; zeros for
 *     tokens that attend to nothing and for rows of no sequence
 *   ws : kvdec_paged8_workspace_bytes() bytes of device memory, 16-byte
 *     aligned, whose contents do not matter; calls that overlap need their own
 */
int kvdec_paged8_attention(const kvdec_paged8_cache* cache, const void* q, void* o, int dtype,
                           int64_t q_token_stride, int64_t q_head_stride, const int32_t* cu_seqlens,
                           int64_t B, int64_t T, int32_t H, int32_t window, int32_t sink, float sm_scale,
                           void* ws, size_t ws_bytes, void* stream);

/* Workspace bytes of kvdec_paged8_attention (0 for arguments it refuses).
 * max_len = max_blocks * page_size.  Pure arithmetic, no HIP call. */
size_t kvdec_paged8_workspace_bytes(int64_t B, int64_t T, int32_t H, int32_t KVH, int64_t max_len);

#ifdef __cplusplus
}
#endif

#endif /* KVDEC_PAGED8_H_ */
