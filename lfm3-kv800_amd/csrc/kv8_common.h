// kv8_common.h -- what the kernels of the paged 8-bit cache share (include/kv8_hip.h): the block layout, exponents, e4m3
// conversions.
#pragma once
#include "kv800_common.h"
#include "../../include/kv800_hip.h"
#include "../../include/kv8_hip.h"

namespace kv8 {
namespace {

constexpr int BLK = 64;               // tokens per block (one exponent for its keys, one for its values)
constexpr int E_MIN = -100, E_MAX = 120;

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // e in [-126, 127]
// The least e in [E_MIN, E_MAX] with top <= 448 2^e (448 = 1.75 2^8 is the largest e4m3 number), top >= 0 and finite.
__device__ __forceinline__ int exponent_for(float top) {
  const uint32_t u = __float_as_uint(top);
  return min(max((int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0), E_MIN), E_MAX);
}
__device__ __forceinline__ int held_exponent(uint8_t b) { return min(max((int)b - 127, E_MIN), E_MAX); }
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}
// four floats -> e4m3 codes, round to nearest even; infinities and NaN -> a NaN code
__device__ __forceinline__ uint32_t enc4(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
__device__ __forceinline__ void dec4(uint32_t w, float (&o)[4]) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  o[0] = a[0]; o[1] = a[1]; o[2] = b[0]; o[3] = b[1];
}
// codes rounded again to code * f, f a power of two below 1
__device__ __forceinline__ uint32_t down4(uint32_t w, float f) {
  float x[4];
  dec4(w, x);
  return enc4(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
}
// slot of token t of a block's keys
__device__ __forceinline__ int slot_of(int t) { return ((t >> 2) & 3) * 16 + (t >> 4) * 4 + (t & 3); }

// The last i in [0, n) with below(i), for a predicate that holds up to some index, 0 among them, looked for around a guess first: one
// load where it is within 31 of it, else as kv800::last_at. By a whole wave, the same result in every lane.
template <typename F>
__device__ __forceinline__ int64_t row_near(int64_t n, int64_t guess, F below) {
  const int lane = threadIdx.x & 63;
  const int64_t lo = max(min(guess - 31, n - 64), (int64_t)0), i = lo + lane;
  const uint64_t yes = __ballot(i < n && below(i < n ? i : 0));
  const int c = __popcll(yes);                                          // lanes 0 .. c - 1
  if (c > 0 && (c < 64 || lo + 64 >= n)) return lo + c - 1;
  return kv800::last_at(n, below);
}

struct Cache {
  uint8_t* data;
  uint8_t* exps;
  int pages, heads, blocks;
  int64_t page_stride, exp_stride;
};
// block u of head h of page p: its keys (values 64 D bytes behind)
template <int D>
__device__ __forceinline__ uint8_t* block_of(const Cache& c, int64_t p, int h, int u) {
  return c.data + p * c.page_stride + (int64_t)(h * c.blocks + u) * (2 * BLK * D);
}
__device__ __forceinline__ uint8_t* exps_of(const Cache& c, int64_t p, int h, int u) {
  return c.exps + p * c.exp_stride + (h * c.blocks + u) * 2;
}

// host: the descriptor's checks, and the form that kernels take
inline bool valid(const kv8_cache_t* c) {
  return c && c->data && c->exps && (uintptr_t)c->data % 16 == 0 && c->pages > 0 && c->pages < INT32_MAX && c->kv_heads > 0 &&
         c->blocks > 0 && (c->dim == 64 || c->dim == 128) && c->kv_heads <= 65535 / 2 && c->blocks <= (1 << 20) &&
         c->kv_heads * c->blocks < (1 << 24) && c->page_stride % 16 == 0 &&
         c->page_stride >= c->kv_heads * c->blocks * 2 * BLK * c->dim && c->exp_stride >= c->kv_heads * c->blocks * 2 &&
         c->exp_stride % 2 == 0 && (uintptr_t)c->exps % 2 == 0;
}
inline Cache device_form(const kv8_cache_t* c) {
  return {c->data, c->exps, (int)c->pages, (int)c->kv_heads, (int)c->blocks, c->page_stride, c->exp_stride};
}

}  // namespace
}  // namespace kv8
