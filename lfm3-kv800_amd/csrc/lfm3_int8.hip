// lfm3_int8.hip -- the engine loop's products in 8-bit integers (include/lfm3_int8.h), gfx950: y = s_r s_n sum_k x8 w8.
//
//   layout_kernel    a weight into operand order, once
//   quantize_kernel  tokens (or a weight's rows) to 8 bits, a scale for each
//   product_kernel   the products, 4 waves of 64 x 64 outputs each
//
// Sums of up to 65,536 products of 8-bit integers fit 32 bits, so they are exact and any split of K gives the same result; the
// scales are applied once, in fp32.
#include "kv800_common.h"
#include "../../include/kv800_hip.h"
#include "../../include/lfm3_int8.h"

namespace lfm3 {
namespace {

typedef int i4v __attribute__((ext_vector_type(4)));
typedef int i16v __attribute__((ext_vector_type(16)));

constexpr float LEAST = 0x1p-100f;     // of a token's largest magnitude: 127 / t stays finite

__device__ __forceinline__ i16v mfma(i4v a, i4v b, i16v c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }

// row of W that padded row n of the layout holds, -1: none
__device__ __forceinline__ int64_t source_row(int64_t n, int64_t N, int gated) {
  if (!gated) return n < N ? n : -1;
  const int64_t t = n >> 5, f = (t >> 1) * 32 + (n & 31), F = N / 2;
  return f < F ? (t & 1) * F + f : -1;
}

__global__ void __launch_bounds__(256) layout_kernel(const int8_t* __restrict__ w, int64_t ld, const float* __restrict__ scale,
                                                     int64_t N, int64_t K, int64_t Npad, int64_t nks, int gated,
                                                     int8_t* __restrict__ wsh, float* __restrict__ ssh) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;             // (block, lane)
  if (i < Npad) {
    const int64_t r = source_row(i, N, gated);
    ssh[i] = r < 0 ? 0.f : scale[r];
  }
  if (i >= Npad / 32 * nks * 64) return;
  const int64_t blk = i >> 6, l = i & 63, nt = blk / nks, ks = blk % nks;
  const int64_t r = source_row(32 * nt + (l & 31), N, gated), k = 32 * ks + 16 * (l >> 5);
  uint32_t v[4] = {0u, 0u, 0u, 0u};
  if (r >= 0)
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (k + e < K) v[e >> 2] |= (uint32_t)(uint8_t)w[r * ld + k + e] << (8 * (e & 3));
  *reinterpret_cast<uint4*>(wsh + i * 16) = make_uint4(v[0], v[1], v[2], v[3]);
}

// One wave per row. Up to 16 pieces of 512 channels stay in registers between the maximum and the codes; a longer row is read again.
// OPERAND: codes in operand order of tiles of 32 rows (nks blocks each), else row by row.
template <bool OPERAND>
__global__ void __launch_bounds__(256) quantize_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t R, int64_t K, int64_t nks,
                                                       int8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int HELD = 16;
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= R) return;
  const uint16_t* src = x + r * ldx;
  uint4 held[HELD];
  uint32_t top = 0;                                                      // magnitudes of bf16 order as integers; NaN above infinity
  auto take = [&](const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
  };
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    const int64_t k = j * 512 + lane * 8;
    held[j] = make_uint4(0, 0, 0, 0);
    if (k < K) held[j] = *reinterpret_cast<const uint4*>(src + k);
  }
#pragma unroll
  for (int j = 0; j < HELD; ++j) take(held[j]);
  for (int64_t k = HELD * 512 + lane * 8; k < K; k += 512) take(*reinterpret_cast<const uint4*>(src + k));
#pragma unroll
  for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  const float t = fmaxf(kv800::bf2f(top), LEAST), inv = 127.f / t;
  if (lane == 0) scale[r] = top < 0x7F80u ? t / 127.f : __uint_as_float(0x7FC00000u);
  auto put = [&](int64_t k, const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t o[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t b = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float f = e & 1 ? kv800::bf2f_hi(w[2 * i + (e >> 1)]) : kv800::bf2f_lo(w[2 * i + (e >> 1)]);
        b |= ((uint32_t)(int)rintf(f * inv) & 0xFFu) << (8 * e);
      }
      o[i] = b;
    }
    int8_t* dst;
    if (OPERAND) dst = q + (((r >> 5) * nks + (k >> 5)) * 64 + (r & 31) + 32 * ((k >> 4) & 1)) * 16 + (k & 15);
    else dst = q + r * K + k;
    *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
  };
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    const int64_t k = j * 512 + lane * 8;
    if (k < K) put(k, held[j]);
  }
  for (int64_t k = HELD * 512 + lane * 8; k < K; k += 512) put(k, *reinterpret_cast<const uint4*>(src + k));
}

// One workgroup: 128 rows of the weight x 128 tokens, a wave 64 x 64, operands straight from memory (both lie in operand order).
// Output of the instruction (weight rows x tokens): lane l holds token l % 32, rows 8 b + 4 (l / 32) + i.
template <bool GATED>
__global__ void __launch_bounds__(256) product_kernel(const int8_t* __restrict__ xq, const float* __restrict__ sx,
                                                      const int8_t* __restrict__ wsh, const float* __restrict__ ssh, int64_t R,
                                                      int64_t N, int64_t nt, int64_t mt, int64_t nks, uint16_t* __restrict__ y, int64_t ldy) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int64_t n0 = (int64_t)blockIdx.x * 4 + 2 * (wv & 1), m0 = (int64_t)blockIdx.y * 4 + 2 * (wv >> 1);
  if (n0 >= nt || m0 >= mt) return;
  const int8_t* wp[2];
  const int8_t* xp[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    wp[j] = wsh + (n0 + j) * nks * 1024 + lane * 16;                     // nt is even
    xp[j] = xq + min(m0 + j, mt - 1) * nks * 1024 + lane * 16;           // a tile past the last is computed again, not stored
  }
  i16v acc[2][2];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[a][b][v] = 0;
  for (int64_t ks = 0; ks < nks; ++ks) {
    i4v a[2], b[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) { a[j] = *reinterpret_cast<const i4v*>(wp[j] + ks * 1024); b[j] = *reinterpret_cast<const i4v*>(xp[j] + ks * 1024); }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mfma(a[i], b[j], acc[i][j]);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t r = (m0 + j) * 32 + (lane & 31);
    if (m0 + j >= mt || r >= R) continue;
    const float s = sx[r];
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 8 * b + 4 * (lane >> 5) + i;
        const float y0 = (float)acc[0][j][4 * b + i] * s * ssh[n0 * 32 + row], y1 = (float)acc[1][j][4 * b + i] * s * ssh[n0 * 32 + 32 + row];
        if (GATED) {
          const int64_t f = n0 * 16 + row;
          if (f < N / 2) y[r * ldy + f] = (uint16_t)kv800::f2bf(y0 / (1.f + __expf(-y0)) * y1);
        } else {
          if (n0 * 32 + row < N) y[r * ldy + n0 * 32 + row] = (uint16_t)kv800::f2bf(y0);
          if (n0 * 32 + 32 + row < N) y[r * ldy + n0 * 32 + 32 + row] = (uint16_t)kv800::f2bf(y1);
        }
      }
  }
}

// ---------------------------------------------------------------- host
constexpr int64_t K_MOST = 65536;      // 127^2 K below 2^31
int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
int64_t padded_rows(int64_t N, int gated) { return gated ? 2 * round_up(N / 2, 32) : round_up(N, 64); }
bool sizes(int64_t R, int64_t N, int64_t K, int gated) {
  return R >= 0 && R <= (1 << 24) && N > 0 && N <= (1 << 24) && K > 0 && K <= K_MOST && K % 8 == 0 && (gated == 0 || (gated == 1 && N % 2 == 0));
}

}  // namespace
}  // namespace lfm3

extern "C" {

int lfm3_hip_int8_layout(const int8_t* w, int64_t ld, const float* scale, int64_t N, int64_t K, int gated, int8_t* wsh, float* ssh,
                         void* stream) {
  KV800_REQUIRE(lfm3::sizes(0, N, K, gated) && ld >= 0, "int8_layout: N up to 2^24 (even for a gated weight), K a multiple of 8 up to 65536");
  KV800_REQUIRE(w && scale && wsh && ssh && (uintptr_t)wsh % 16 == 0, "int8_layout: null or unaligned pointer");
  const int64_t Npad = lfm3::padded_rows(N, gated), nks = lfm3::round_up(K, 128) / 32, n = Npad / 32 * nks * 64;
  hipLaunchKernelGGL(lfm3::layout_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, w, ld, scale, N, K,
                     Npad, nks, gated, wsh, ssh);
  return kv800::check_launch("int8_layout");
}

int lfm3_hip_int8_quantize(const uint16_t* w, int64_t ld, int64_t N, int64_t K, int8_t* w8, float* scale, void* stream) {
  KV800_REQUIRE(lfm3::sizes(0, N, K, 0) && ld % 8 == 0, "int8_quantize: N up to 2^24, K a multiple of 8 up to 65536, ld a multiple of 8");
  KV800_REQUIRE(w && w8 && scale && (uintptr_t)w % 16 == 0 && (uintptr_t)w8 % 8 == 0, "int8_quantize: null or unaligned pointer");
  hipLaunchKernelGGL(lfm3::quantize_kernel<false>, dim3((unsigned)((N + 3) / 4)), dim3(256), 0, (hipStream_t)stream, w, ld, N, K, 0,
                     w8, scale);
  return kv800::check_launch("int8_quantize");
}

int64_t lfm3_hip_linear8_workspace(int64_t R, int64_t N, int64_t K, int gated) {
  if (!lfm3::sizes(R, N, K, gated) || R == 0) return 0;
  const int64_t mpad = lfm3::round_up(R, 32);
  return mpad * lfm3::round_up(K, 128) + mpad * 4;
}

int lfm3_hip_linear8(const uint16_t* x, int64_t ldx, const int8_t* wsh, const float* ssh, int64_t R, int64_t N, int64_t K,
                     int gated, uint16_t* y, int64_t ldy, void* ws, int64_t ws_bytes, void* stream) {
  KV800_REQUIRE(lfm3::sizes(R, N, K, gated),
                "linear8: R and N up to 2^24 (N even for a gated weight), K a multiple of 8 up to 65536, gated 0 or 1");
  KV800_REQUIRE(ldx % 8 == 0 && ldy >= 0, "linear8: ldx must be a multiple of 8 and ldy >= 0");
  if (R == 0) return KV800_OK;
  KV800_REQUIRE(x && wsh && ssh && y && (uintptr_t)x % 16 == 0 && (uintptr_t)wsh % 16 == 0, "linear8: null or unaligned pointer");
  const int64_t need = lfm3_hip_linear8_workspace(R, N, K, gated);
  KV800_REQUIRE(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need, "linear8: %lld bytes of 16-byte aligned workspace needed", (long long)need);
  const int64_t mt = lfm3::round_up(R, 32) / 32, nt = lfm3::padded_rows(N, gated) / 32, nks = lfm3::round_up(K, 128) / 32;
  int8_t* xq = (int8_t*)ws;
  float* sx = (float*)(xq + mt * nks * 1024);
  hipLaunchKernelGGL(lfm3::quantize_kernel<true>, dim3((unsigned)((R + 3) / 4)), dim3(256), 0, (hipStream_t)stream, x, ldx, R, K, nks,
                     xq, sx);
  int rc = kv800::check_launch("linear8 quantize");
  if (rc != KV800_OK) return rc;
  const dim3 grid((unsigned)((nt + 3) / 4), (unsigned)((mt + 3) / 4));
  KV800_REQUIRE(grid.y <= 65535, "linear8: too many tokens");
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, xq, sx, wsh, ssh, R, N, nt, mt, nks, y, ldy);
  };
  if (gated) go(lfm3::product_kernel<true>);
  else go(lfm3::product_kernel<false>);
  return kv800::check_launch("linear8");
}

}  // extern "C"
