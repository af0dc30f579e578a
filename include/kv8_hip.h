/* kv8_hip.h -- C ABI of the paged 8-bit cache of keys and values (lfm3-kv800_amd/csrc/kv8_cache.hip, kv8_attn.hip), in the
 * same library as the 800h path (lfm3-kv800_amd/_lib/libkv800_hip.so).
 *
 * No counterpart in the reference, whose caches are bf16 or 800h. Conventions as include/kv800_hip.h: device pointers, bf16 as
 * uint16_t, `stream` a hipStream_t as void*, asynchronous launches without allocation, 0 on success or a negative status with
 * kv800_hip_last_error(), arguments checked on the host before any launch.
 *
 * Format. A block is 64 tokens of one KV head: 64 D e4m3 codes of its keys, 64 D of its values, an exponent byte b (e8m0) for
 * each: value = code 2^(b - 127), b in [27, 247] (others are taken as the nearer end). Codes lie in the order in which a wave
 * takes them as operands of the matrix instructions, 16 bytes a lane, so that nothing rearranges them:
 *   keys   [D / 16][64 slots][16 dims], token t = 16 g + 4 a + i (i, a < 4) of the block in slot 16 a + 4 g + i;
 *   values [t / 16][D][t % 16].
 * Page p, head h, block u of the page: data + p page_stride + ((h blocks + u) 2 + (0 keys, 1 values)) 64 D, exponents at
 * exps + p exp_stride + (h blocks + u) 2 + (0, 1). Row r's position x is token x % 64 of block x / 64 % blocks of page
 * bt[r, x / (64 blocks)]; entries outside [0, pages) and positions past the table hold no tokens. kv8_hip_attend reads a pair of
 * exponents as the 4-byte aligned word around it: up to 2 bytes before and behind exps, which go into nothing.
 *
 * A step's tokens lie row after row: row r's qsl[r] .. qsl[r + 1] (qsl (R + 1) int64, as kv800_hip_chunk_meta makes it) at the
 * positions lens[r] - (qsl[r + 1] - qsl[r]) + i, lens (R) int64 the lengths with the new tokens. */
#ifndef KV8_HIP_H
#define KV8_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct kv8_cache {
  uint8_t* data;
  uint8_t* exps;
  int64_t pages, kv_heads, blocks, dim;   /* blocks of 64 tokens a page; dim D: 64 or 128 */
  int64_t page_stride, exp_stride;        /* bytes from page to page (a multiple of 16 and of 2; data 16-byte aligned, exps 2) */
} kv8_cache_t;

/* Append the step's tokens: k, v rows of kv_heads x D bf16, token and head strides in elements (multiples of 8, 16-byte
 * aligned). With cos_t / sin_t ((rope_rows, freqs) bf16, freqs a multiple of 8 up to D / 2) the key pairs (f, f + D / 2),
 * f < freqs, are rotated by the angle at the token's position (clamped into the tables) in fp32 and not rounded before their
 * encoding; NULL: as they come. A block's exponent is the least e in [-100, 120] whose 448 2^e holds the largest finite
 * magnitude of the call's tokens in it, and not below the present one where the block holds earlier tokens of the row; when it
 * grows, their codes are rounded again. Codes are rounded to nearest even; infinities and NaN become the NaN code. Codes of
 * tokens behind the row's last one stay. Two rows of a call may not append to one block. */
int kv8_hip_append(const kv8_cache_t* cache, const uint16_t* k, int64_t k_ts, int64_t k_hs, const uint16_t* v, int64_t v_ts,
                   int64_t v_hs, const int32_t* bt, int64_t bt_stride, int64_t bt_cols, const int64_t* lens,
                   const int64_t* qsl, int64_t R, int64_t T, const uint16_t* cos_t, const uint16_t* sin_t,
                   int64_t rope_rows, int64_t freqs, void* stream);

/* What the cache stands for: k, v (pages, kv_heads, 64 blocks, D) bf16 (exact, but for magnitudes of 2^128, which become infinite). */
int kv8_hip_dequantize(const kv8_cache_t* cache, uint16_t* k, uint16_t* v, void* stream);

/* Attention of the step's tokens over the cache, which holds them already: q (T, heads, D) bf16, heads = G kv_heads with G up to
 * 16, query head h on KV head h / G; out (T, heads, D) bf16 = softmax(scale q . k) v over positions <= the query's and, with
 * window > 0, > position - window. A query without keys and the padding [qsl[R], T) get zeros; what a query does not see does not
 * reach it, NaN included. An infinity or NaN in a query gives NaN where it sees a key. Scores are fp32 (finite ones have to stay in its
 * range), weights are rounded to bf16 and summed as rounded. ws: kv8_hip_attend_workspace(...) bytes, 16-byte aligned, of this
 * call alone. bt_cols blocks 64 < 2^31.
 *
 * How a call runs goes by what the host knows, T tokens over R rows and the positions of bt_cols pages, not by the rows themselves.
 * A table wider than its rows costs little (one row of 1,000 positions 9.9 us, 13.8 in a table of 8,192 and of 65,536), a first chunk in one
 * more (64 tokens 9.8, 17.8, 26.6). A prompt beside single tokens over long rows is quicker in a call of its own (a prompt of
 * 2,048 and 63 tokens over 16,384 positions each: 396, in two calls 253; one token over 131,072 positions: 2,919, 87). */
int64_t kv8_hip_attend_workspace(const kv8_cache_t* cache, int64_t heads, int64_t R, int64_t T, int64_t bt_cols, int64_t window);
int kv8_hip_attend(const kv8_cache_t* cache, const uint16_t* q, int64_t heads, const int32_t* bt, int64_t bt_stride,
                   int64_t bt_cols, const int64_t* lens, const int64_t* qsl, int64_t R, int64_t T, int64_t window,
                   float scale, uint16_t* out, void* ws, int64_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KV8_HIP_H */
