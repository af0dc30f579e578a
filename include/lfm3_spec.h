/* lfm3_spec.h -- C ABI of the model-side operators of a step whose rows bring several new tokens each (drafted tokens to
 * verify, short prompt chunks), in the same library as the 800h path (lfm3-kv800_amd/_lib/libkv800_hip.so).
 *
 * No counterpart in the reference's own code: its model (vllm_model.py:327-431) leaves prompt chunks of the short conv to
 * vLLM's causal-conv op, and sampling and drafts to vLLM's sampler. Conventions as include/kv800_hip.h: device pointers,
 * `stream` a hipStream_t as void*, asynchronous launches, 0 on success or a negative status with kv800_hip_last_error().
 * The tokens of a step lie row after row: row r's are [qsl[r], qsl[r + 1]) (qsl (R + 1) int64 on the device, ascending from
 * 0, as kv800_hip_chunk_meta makes it); tokens [qsl[R], T) are padding. A qsl that reaches past T is cut at T.
 */
#ifndef LFM3_SPEC_H
#define LFM3_SPEC_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Short conv over each row's new tokens: token t of row r has tap_t = bf16(B_t x_t) per channel (bcx (T, >= 3H; row stride
 * `stride`) = [B | C | x]) and out_t = bf16(C_t sum_k conv_w[c, k] window_k), the window being the last 7 of
 * [state[r] (6 taps, the oldest first) | the row's taps up to t], products and sum in fp32 (lfm3_hip_conv_step rounds
 * each to bf16). out, taps (T, H) bf16; padding tokens get zeros. state (R, H, 6) is read only: lfm3_hip_conv_commit moves it
 * on. H a multiple of 8; stride a multiple of 8; all pointers 16-byte aligned. */
int lfm3_hip_conv_chunk(const uint16_t* bcx, int64_t stride, const uint16_t* conv_w, const uint16_t* state,
                        const int64_t* qsl, int64_t R, int64_t T, int64_t H, uint16_t* out, uint16_t* taps, void* stream);

/* The conv state behind the kept tokens: state[r] <- the last 6 of [state[r] | the row's first kept[r] taps], kept (R) int32
 * clamped to [0, the row's tokens]. In place; taps as lfm3_hip_conv_chunk wrote them. */
int lfm3_hip_conv_commit(uint16_t* state, const uint16_t* taps, const int64_t* qsl, const int32_t* kept, int64_t R,
                         int64_t T, int64_t H, void* stream);

/* Workspace bytes of lfm3_hip_verify_drafts for R rows with T tokens in all and V logits each. */
int64_t lfm3_hip_verify_workspace(int64_t R, int64_t T, int64_t V);

/* Verification of drafted tokens. logits (T, V) bf16 (row stride ld): row t holds the target's logits behind token t; within a
 * row's tokens, token t + 1 is the draft that logits row t judges. p = softmax(logits / temp[r]) in 64 bits. A draft d is
 * kept iff u[t] q(d) < p(d), q = row t of draft_probs ((T, V) fp32, row stride ldq; NULL: all of it on d). At the first
 * draft that is not kept the row ends with a token of max(p - q, 0) (of p without d if NULL; of p where that is empty), a
 * row whose drafts are all kept with a token of p behind its last one: the first index whose running sum exceeds
 * u_next[r] times the whole. temp[r] not in (0, 1e30], or a largest logit that is not finite: a draft is kept iff it is the
 * largest logit (the first of equal ones; the first NaN ranks above every number) and the row ends with that one.
 * Drafts outside [0, V) are never kept. out (T) int64: row r's kept drafts and its last token at qsl[r] .., -1 in the rest
 * and in the padding; count (R) int32: how many (0 for a row without tokens). u (T), u_next (R) fp32 in [0, 1). Sums run in
 * a fixed order. ws: lfm3_hip_verify_workspace bytes, 16-byte aligned; 0 < V < 2^31, any strides >= V; R, T <= 65,535. */
int lfm3_hip_verify_drafts(const uint16_t* logits, int64_t ld, const int64_t* tokens, const int64_t* qsl, const float* temp,
                           const float* u, const float* u_next, const float* draft_probs, int64_t ldq, int64_t R,
                           int64_t T, int64_t V, int64_t* out, int32_t* count, void* ws, int64_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LFM3_SPEC_H */
