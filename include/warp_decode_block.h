/*
 * warp_decode_b200 — C ABI of the operators that complete a decoder layer's step
 * (libwarp_decode_block_b200.so): the norms between two blocks with gate and
 * residual, projections with 4-bit weights, and attention over the FP8 paged
 * cache of a batch whose sequences begin with the same tokens.  None of them has
 * a counterpart in the reference.
 *
 * The rules of warp_decode.h and warp_decode_layer.h hold here too (strides in
 * elements, a status word, nothing synchronises or allocates); a failing call
 * returns a wd_error_t code and wd_block_last_error_message() says why.
 *
 * One step of a layer:
 *   wd_linear_w4 (queries, keys, values) -> wd_qk_norm_rope -> wd_kv_cache_write_fp8
 *   -> wd_attn_decode_fp8_prefix -> wd_linear_w4 (output) -> wd_block_norm ->
 *   (router product) -> wd_moe_router_scored_topk -> wd_moe_ffn_3d_batched -> wd_block_norm
 */
#ifndef WARP_DECODE_BLOCK_B200_H_
#define WARP_DECODE_BLOCK_B200_H_

#include "warp_decode_layer.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Detail message of the last failing call on this host thread ("" if none). */
WD_API const char* wd_block_last_error_message(void);

/* As wd_status_read, for this library's word of the current device. */
WD_API int wd_block_status_read(uint32_t* value, int clear);

/* As wd_launch_count, for this library's kernels. */
WD_API unsigned long long wd_block_launch_count(void);

/*
 * Between two blocks, for T rows of H values:
 *   z  = y, or with post_weight  y * rsqrt(mean(y^2) + eps) * post_weight
 *   r' = residual_scale * r + gate * z
 *   x  = r' * rsqrt(mean(r'^2) + eps) * norm_weight
 * in fp32, each output rounded once (x is of r' before its rounding); of a gate that
 * all tokens share, gate * post_weight may be taken first.
 *   y, x [T, H] bf16; r, residual_out [T, H] bf16, or fp32 when residual_fp32 != 0;
 *   rows contiguous, with the given token strides.  residual_out may be r itself
 *   (same stride); otherwise no output may share memory with an input or an output.
 *   norm_weight, post_weight [H] bf16, or fp32 when weight_fp32 != 0; post_weight
 *   may be NULL
 *   gate bf16, or fp32 when gate_fp32 != 0, or NULL (1): of token t and channel h
 *   at gate[t * gate_token_stride + h * gate_channel_stride], gate_channel_stride 0
 *   or 1
 * 1 <= H <= 16384.
 */
WD_API int wd_block_norm(const void* y, long long y_token_stride, const void* r,
                         long long r_token_stride, int residual_fp32, const void* norm_weight,
                         const void* post_weight, int weight_fp32, const void* gate,
                         long long gate_token_stride, int gate_channel_stride, int gate_fp32,
                         float residual_scale, float eps, void* x, long long x_token_stride,
                         void* residual_out, long long ro_token_stride, int T, int H, void* stream);

/* Types of the scales of wd_linear_w4. */
#define WD_W4_SCALE_BF16 0
#define WD_W4_SCALE_FP16 1
#define WD_W4_SCALE_FP32 2

/*
 * out[t, n] = sum_k x[t, k] * (code[n, k] - zero[n, k / group]) * scale[n, k / group]
 * with 4-bit codes.
 *   x [T, K] bf16, rows contiguous, with its token stride
 *   w [N, ceil(K / 128) * 64] uint8: rows of blocks of 128 codes, 64 bytes each; as
 *     little-endian 32-bit words, word 4 t + s of a block holds the codes of
 *     k = 32 s + 8 t + 0..7 of it, k = 2 i in bits 4 i, k = 2 i + 1 in bits 16 + 4 i
 *     (the codes past K are not used)
 *   scale [N, K / group] of scale_type; zero [N, K / group] uint8, 0 to 127 (larger
 *     ones count as 127), or NULL (8)
 *   out [T, N] bf16, rows contiguous, with its token stride
 * A group's products and their sum, and the sum of the groups, are fp32; one
 * rounding.  group 32, 64 or 128, K a multiple of it; w 16-byte aligned.
 */
WD_API int wd_linear_w4(const void* x, long long x_token_stride, const uint8_t* w,
                        const void* scale, int scale_type, const uint8_t* zero, void* out,
                        long long out_token_stride, int T, int N, int K, int group, void* stream);

/*
 * wd_attn_decode_fp8 for sequences that begin with the same tokens in the same
 * pages: the first prefix_len[0] tokens (device memory; whole pages of them count)
 * of every sequence lie in the pages that the table of the longest sequence shows.
 * The result is wd_attn_decode_fp8's, and so are the arguments; those pages are
 * read once for all sequences, and only they: a sequence's own table is not read
 * for them.  A prefix_len of 0 is allowed, and sequences that end within it (or are
 * empty) too.
 * It is for large batches behind long prompts: where B * prefix_len * Hkv passes about
 * a million.  Below, and with a window that hides most of the prefix, wd_attn_decode_fp8
 * on full tables is faster (D 128, 4 key heads of 8 rows, cold, us, that one and this: 4
 * sequences behind 1024 tokens 16 and 36; 16 behind 16384 53 and 53; 64 behind 4096 57
 * and 59; 128 behind 4096 100 and 77; 64 behind 16384 169 and 74; 128 behind 16384 322
 * and 117).
 * workspace: as wd_attn_decode_fp8's, of wd_attn_decode_fp8_prefix_workspace bytes; one
 * that is large enough for both may serve calls of both, one after the other.
 * Head sizes other than 64 and 128, and caches of 2^31 token rows or more, run on the
 * CUDA cores, where each sequence reads the shared pages (of the same table) by itself.
 * Head sizes 64 and 128, prefix and own tokens alike: each weight p, times the scale of
 * its page of V, is rounded to fp16, within 2^-11 of itself or, where that is more, within
 * 2^-31 of the row's largest; q is taken within 2^-18 of its row's largest value.  Sums
 * are fp32.
 */
WD_API int wd_attn_decode_fp8_prefix(const void* q, long long q_batch_stride,
                                     long long q_token_stride, long long q_head_stride,
                                     const uint8_t* k_cache, const uint8_t* k_scale,
                                     const uint8_t* v_cache, const uint8_t* v_scale,
                                     const int32_t* table, int table_stride,
                                     const int32_t* seq_lens, const int32_t* prefix_len, void* out,
                                     float* lse, float softmax_scale, int window, int B, int Sq,
                                     int Hq, int Hkv, int D, int page, int pages, void* workspace,
                                     size_t workspace_bytes, uint32_t* status, void* stream);

/* Bytes of workspace that wd_attn_decode_fp8_prefix needs for these sizes on the current device. */
WD_API int wd_attn_decode_fp8_prefix_workspace(int B, int Sq, int Hq, int Hkv, int D, size_t* bytes);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* WARP_DECODE_BLOCK_B200_H_ */
