/* lfm3_int8.h -- C ABI of the engine loop's products in 8-bit integers (lfm3-kv800_amd/csrc/lfm3_int8.hip), in the same library as
 * the 800h path (lfm3-kv800_amd/_lib/libkv800_hip.so).
 *
 * No counterpart in the reference, whose weights are bf16. Conventions as include/kv800_hip.h: device pointers, bf16 as uint16_t,
 * `stream` a hipStream_t as void*, asynchronous launches without allocation, 0 on success or a negative status with
 * kv800_hip_last_error(), arguments checked on the host before any launch.
 *
 * A weight W (N, K) int8 with a scale for each row is stored once in the operand order of the 32 x 32 x 32 int8 matrix
 * instruction: Npad / 32 x Kpad / 32 blocks of 1,024 bytes, block (nt, ks) lane l = W[32 nt + l % 32][32 ks + 16 (l / 32) .. + 16],
 * Npad a multiple of 64, Kpad of 128, zeros behind N and K. gated: W = [g | u], N = 2 F: tiles 2 j and 2 j + 1 hold rows
 * 32 j .. of g and of u (F padded to 32 for itself). */
#ifndef LFM3_INT8_H
#define LFM3_INT8_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* W (N, K; row stride ld, any alignment) and its scales (N) fp32 into that order: wsh Npad Kpad bytes, ssh Npad floats (Npad for a
 * gated weight: 2 ceil(F / 32) 32). */
int lfm3_hip_int8_layout(const int8_t* w, int64_t ld, const float* scale, int64_t N, int64_t K, int gated, int8_t* wsh, float* ssh,
                         void* stream);

/* A bf16 weight (N, K; row stride ld) quantized by rows: with t = max(max |w|, 2^-100) of a row, scale = t / 127 and w8 (N, K) = w (127 / t)
 * rounded to nearest even, quotient and product rounded to fp32 before. */
int lfm3_hip_int8_quantize(const uint16_t* w, int64_t ld, int64_t N, int64_t K, int8_t* w8, float* scale, void* stream);

/* y (R, N, or R, N / 2 for a gated weight; row stride ldy) bf16 = s_r s_n sum_k x8 w8, x8 and s_r of a token as w8 and scale of
 * a weight's row (above); the sums are exact, and a scale above 1 of a token is multiplied behind the row's, so that what is finite stays
 * finite. gated: silu(y_g) y_u in fp32, rounded once. A token with an
 * infinity or NaN gives NaN. x (R, K; row stride ldx, a multiple of 8, 16-byte aligned) bf16, K a multiple of 8 up to 65,536.
 * ws: lfm3_hip_linear8_workspace bytes, 16-byte aligned, of this call alone. */
int64_t lfm3_hip_linear8_workspace(int64_t R, int64_t N, int64_t K, int gated);
int lfm3_hip_linear8(const uint16_t* x, int64_t ldx, const int8_t* wsh, const float* ssh, int64_t R, int64_t N, int64_t K,
                     int gated, uint16_t* y, int64_t ldy, void* ws, int64_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LFM3_INT8_H */
