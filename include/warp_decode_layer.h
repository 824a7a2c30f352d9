/*
 * warp_decode_b200 — C ABI of the operators around the MoE FFN in a decoder
 * layer's step (libwarp_decode_layer_b200.so): queries and keys made ready,
 * the FP8 paged key/value cache, attention over it, and the expert choice.
 * None of them has a counterpart in the reference, which covers the two FFN
 * kernels of warp_decode.h only.
 *
 * The rules of warp_decode.h hold here too: plain device pointers, sizes and
 * a CUDA stream handle; nothing synchronises or allocates device memory;
 * arguments are checked on the host before anything is launched; a failing
 * call returns a wd_error_t code and wd_layer_last_error_message() says why
 * (thread-local).  What only the device can see is OR-ed into a 32-bit status
 * word: the caller's `status`, or a word of this library when that is NULL
 * (wd_layer_status_read).  Strides are in elements.
 *
 * One step of a layer:
 *   wd_qk_norm_rope -> wd_kv_cache_write_fp8 -> wd_attn_decode_fp8 ->
 *   (output projection, norm, router product) -> wd_moe_router_scored_topk ->
 *   wd_moe_ffn_3d_batched
 *
 * FP8 paged cache (keys and values alike):
 *   cache  [pages, Hkv, page, D]  uint8, E4M3 codes (OCP FP8: no infinities,
 *                                 0x7f / 0xff are NaN)
 *   scale  [pages, Hkv]           uint8, UE8M0: value = e4m3(code) * 2^(scale - 127),
 *                                 NaN where the scale is 255
 *   table  [B, table_stride]      int32, page of the tokens [n * page, (n + 1) * page)
 *                                 of sequence b at table[b][n]
 * page is 16, 32, 64 or 128 tokens; D is a multiple of 16 up to 256, Hkv at
 * most 1024; the caches are 16-byte aligned.  A call writes or reads at most
 * 65534 pages of tokens of each sequence.
 */
#ifndef WARP_DECODE_LAYER_B200_H_
#define WARP_DECODE_LAYER_B200_H_

#include "warp_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bits of the device status word (with WD_STATUS_WAIT_TIMEOUT). */
#define WD_STATUS_BAD_PAGE     0x10u /* a needed page id was outside [0, pages), or a
                                        token lies past the table's last column    */
#define WD_STATUS_BAD_POSITION 0x20u /* a position was outside the table of angles,
                                        or a start was negative                    */

/* Detail message of the last failing call on this host thread ("" if none). */
WD_API const char* wd_layer_last_error_message(void);

/* As wd_status_read, for this library's word of the current device. */
WD_API int wd_layer_status_read(uint32_t* value, int clear);

/* As wd_launch_count, for this library's kernels. */
WD_API unsigned long long wd_layer_launch_count(void);

/*
 * Expert choice of T tokens from router logits [T, E] (bf16, or fp32 when
 * logits_fp32 != 0):
 *   s = softmax(logits) (scoring 0) or sigmoid(logits) (scoring 1), in fp32
 *   c = s + bias; without a bias, and with group_top 1, c = logits (the same
 *       order, without the ties that rounding a score would make)
 *   the n_group groups of E / n_group consecutive experts are ranked by the
 *   sum of their group_top (1 or 2) largest c; experts of the topk_group best
 *   groups stand for choice
 *   topk_ids     [T, topk] int32: the topk largest c among them, descending
 *   topk_weights [T, topk] fp32:  s at those ids, over their sum when
 *                renormalize, times weight_scale
 * Ties go to the lowest index, of experts and of groups.  A NaN logit scores
 * 0 and ranks below every number.  A logit of +infinity leaves a softmax without
 * scores: its token's weights are NaN.  Renormalised softmax weights are the
 * softmax of the chosen logits, which does not underflow; where the chosen scores
 * sum to 0 (all -infinity or NaN, or sigmoids that underflow), renormalised
 * weights are weight_scale / topk.
 * bias: [E] fp32 or NULL.  1 <= topk <= min(32, topk_group * E / n_group),
 * E <= 1024, n_group <= 32 a divisor of E.
 */
WD_API int wd_moe_router_scored_topk(const void* logits, int logits_fp32, const float* bias,
                                     int32_t* topk_ids, float* topk_weights, int T, int E, int topk,
                                     int scoring, int n_group, int topk_group, int group_top,
                                     int renormalize, float weight_scale, void* stream);

/*
 * RMS norm of every query and key head, then the position rotation:
 *   y = x * rsqrt(mean(x^2) + eps) * weight            (over the head's D values)
 *   for the pairs (y[a], y[b]) of the first `rot` values, with angle i of pair i:
 *   (y[a] cos - y[b] sin, y[b] cos + y[a] sin)
 * interleaved 0: pair i is (i, i + rot/2); 1: (2i, 2i + 1).  fp32 arithmetic,
 * one rounding to bf16.
 *   q [T, Hq, D], k [T, Hkv, D] bf16 with the given token and head strides
 *   q_weight, k_weight [D], bf16, or fp32 when weight_fp32 != 0
 *   positions [T] int32; cos_sin [max_pos, rot] fp32: rot/2 cosines, then the sines
 *   q_out [T, Hq, D], k_out [T, Hkv, D] bf16 with their strides; they may be q
 *   and k themselves (same strides)
 * A position outside [0, max_pos) gives zeros and WD_STATUS_BAD_POSITION.
 * D a multiple of 2 up to 256, rot even, 0 <= rot <= D.  Hq or Hkv may be 0.
 */
WD_API int wd_qk_norm_rope(const void* q, long long q_token_stride, long long q_head_stride,
                           const void* k, long long k_token_stride, long long k_head_stride,
                           const void* q_weight, const void* k_weight, int weight_fp32,
                           const int32_t* positions, const float* cos_sin, int max_pos,
                           void* q_out, long long qo_token_stride, long long qo_head_stride,
                           void* k_out, long long ko_token_stride, long long ko_head_stride, int T,
                           int Hq, int Hkv, int D, int rot, int interleaved, float eps,
                           uint32_t* status, void* stream);

/*
 * Quantise new keys and values as they are written: token i < lens[b] (S
 * without lens) of sequence b goes to position start[b] + i.
 *   k, v [B, S, Hkv, D] bf16 with the given batch, token and head strides
 * Scale of a page and head: 2^e, e the least integer with |x| <= 448 * 2^e for
 * all finite x of the page.  A page that holds earlier tokens of the sequence
 * keeps a scale that is larger; where the new tokens need a larger one its
 * earlier codes are rounded again to the new scale.  Tokens past the new ones
 * are not kept: the next write of the sequence starts there.  Codes round to
 * nearest even; infinities become the largest code, NaN becomes NaN.
 * A page is written by one sequence of a call at most.  Tokens whose page is
 * invalid are skipped (WD_STATUS_BAD_PAGE).
 */
WD_API int wd_kv_cache_write_fp8(const void* k, long long k_batch_stride, long long k_token_stride,
                                 long long k_head_stride, const void* v, long long v_batch_stride,
                                 long long v_token_stride, long long v_head_stride,
                                 uint8_t* k_cache, uint8_t* k_scale, uint8_t* v_cache,
                                 uint8_t* v_scale, const int32_t* table, int table_stride,
                                 const int32_t* start, const int32_t* lens, int B, int S, int Hkv,
                                 int D, int page, int pages, uint32_t* status, void* stream);

/*
 * Read back: positions start[b] + i, i < lens[b] (R without lens), of sequence
 * b to k_out, v_out [B, R, Hkv, D] bf16 (contiguous); rows past lens[b], and
 * rows whose page is invalid (WD_STATUS_BAD_PAGE), are zeros.
 */
WD_API int wd_kv_cache_read_fp8(const uint8_t* k_cache, const uint8_t* k_scale,
                                const uint8_t* v_cache, const uint8_t* v_scale,
                                const int32_t* table, int table_stride, const int32_t* start,
                                const int32_t* lens, void* k_out, void* v_out, int B, int R,
                                int Hkv, int D, int page, int pages, uint32_t* status,
                                void* stream);

/*
 * Attention of the last Sq tokens of each sequence over its cache (negative
 * lengths count as 0):
 *   out[b, i, h] = sum_t p[t] v[t] / sum_t p[t],  p[t] = exp(softmax_scale * q[b, i, h] . k[t])
 * over the tokens t <= seq_lens[b] - Sq + i of key head h / (Hq / Hkv), and
 * t > seq_lens[b] - Sq + i - window where window > 0.  Rows without such a
 * token are zeros (lse -infinity).  What lies in the cache past seq_lens[b],
 * or in a page of an invalid id (WD_STATUS_BAD_PAGE, as if masked), has no
 * influence.
 *   q   [B, Sq, Hq, D] bf16 with the given strides; out [B, Sq, Hq, D] bf16
 *   lse [B, Sq, Hq] fp32 (natural log of sum_t p[t]) or NULL
 *   out 16-byte aligned
 * workspace: device memory of at least wd_attn_decode_fp8_workspace bytes
 * (none for head sizes other than 64 and 128), 16-byte aligned, zeroed once
 * before its first use; every call leaves it ready for the next, except one
 * that raised WD_STATUS_WAIT_TIMEOUT (zero it again).  Calls that share it must
 * not overlap in time.
 * D = 64 and 128 run on the tensor cores, one cooperative launch of a CTA per
 * SM; other head sizes, and caches of 2^31 token rows (pages * Hkv * page) or
 * more, on the CUDA cores.  On the tensor cores each weight p, times the scale
 * of its page of V, is rounded to two E4M3 terms: within 2^-9 of itself or, where
 * that is more, within 2^-16 of the row's largest and without bias over the
 * tokens (for V scales of 2^-90 or more).  Sums are fp32.
 */
WD_API int wd_attn_decode_fp8(const void* q, long long q_batch_stride, long long q_token_stride,
                              long long q_head_stride, const uint8_t* k_cache,
                              const uint8_t* k_scale, const uint8_t* v_cache,
                              const uint8_t* v_scale, const int32_t* table, int table_stride,
                              const int32_t* seq_lens, void* out, float* lse, float softmax_scale,
                              int window, int B, int Sq, int Hq, int Hkv, int D, int page,
                              int pages, void* workspace, size_t workspace_bytes, uint32_t* status,
                              void* stream);

/* Bytes of workspace that wd_attn_decode_fp8 needs for these sizes on the current device. */
WD_API int wd_attn_decode_fp8_workspace(int B, int Sq, int Hq, int Hkv, int D, size_t* bytes);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* WARP_DECODE_LAYER_B200_H_ */
