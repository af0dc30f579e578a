// lfm3_int8.hip -- the engine loop's products in 8-bit integers (include/lfm3_int8.h), gfx950: y = s_r s_n sum_k x8 w8.
//
//   layout_kernel    a weight into operand order, once
//   quantize_kernel  tokens (or a weight's rows) to 8 bits, a scale for each
//   few_kernel       products of few tokens: weights streamed, K split over a workgroup's waves
//   many_kernel      products of many: 256 x 128 outputs a workgroup through LDS
//
// Sums of up to 65,536 products of 8-bit integers fit 32 bits, so they are exact and any split of K gives the same result; the
// scales are applied once, in fp32.
#include "kv800_attn.h"
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

// 16 channels to codes: the product with inv = 127 / t rounds to 32 bits first, so that a channel on the border between two codes (half
// of t, say) may go to either
__device__ __forceinline__ uint4 codes16(const uint4 (&u)[2], float inv) {
  const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[i] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float f = e & 1 ? kv800::bf2f_hi(w[2 * i + (e >> 1)]) : kv800::bf2f_lo(w[2 * i + (e >> 1)]);
      o[i] |= ((uint32_t)(int)rintf(f * inv) & 0xFFu) << (8 * e);
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
// largest magnitude of 16 channels as an integer: of bf16 they order as their bits do, NaN above infinity
__device__ __forceinline__ uint32_t top16(const uint4 (&u)[2]) {
  const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) t = max(t, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
  return t;
}

// WAVES waves of the workgroup's 4 per row. Up to 2 pieces of 16 channels a lane stay in registers between the maximum and the codes;
// a longer row is read again. OPERAND: codes in operand order of tiles of 32 rows (nks blocks each), else row by row.
template <bool OPERAND, int WAVES>
__global__ void __launch_bounds__(256) quantize_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t R, int64_t K, int64_t nks,
                                                       int8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int HELD = 2, LANES = 64 * WAVES;
  __shared__ uint32_t tops[4];
  const int tid = threadIdx.x, lt = tid % LANES;
  const int64_t r = (int64_t)blockIdx.x * (4 / WAVES) + tid / LANES;
  if (WAVES == 1 && r >= R) return;
  const uint16_t* src = x + r * ldx;
  auto take = [&](int64_t k, uint4 (&u)[2]) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      u[p] = make_uint4(0, 0, 0, 0);
      if (k + 8 * p < K) u[p] = *reinterpret_cast<const uint4*>(src + k + 8 * p);
    }
  };
  uint4 held[HELD][2];
#pragma unroll
  for (int j = 0; j < HELD; ++j) take((j * LANES + lt) * 16, held[j]);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < HELD; ++j) top = max(top, top16(held[j]));
  for (int64_t k = (HELD * LANES + lt) * 16; k < K; k += LANES * 16) {
    uint4 u[2];
    take(k, u);
    top = max(top, top16(u));
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  if (WAVES > 1) {
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  }
  const float t = fmaxf(kv800::bf2f(top), LEAST), inv = 127.f / t;
  if (lt == 0) scale[r] = top < 0x7F80u ? t / 127.f : __uint_as_float(0x7FC00000u);
  auto put = [&](int64_t k, const uint4 (&u)[2]) {
    const uint4 o = codes16(u, inv);
    if (OPERAND) {       // the row's padding to whole blocks meets zeros of the weight
      *reinterpret_cast<uint4*>(q + (((r >> 5) * nks + (k >> 5)) * 64 + (r & 31) + 32 * ((k >> 4) & 1)) * 16) = o;
    } else {
      *reinterpret_cast<uint2*>(q + r * K + k) = make_uint2(o.x, o.y);
      if (k + 8 < K) *reinterpret_cast<uint2*>(q + r * K + k + 8) = make_uint2(o.z, o.w);
    }
  };
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    const int64_t k = (j * LANES + lt) * 16;
    if (k < K) put(k, held[j]);
  }
  for (int64_t k = (HELD * LANES + lt) * 16; k < K; k += LANES * 16) {
    uint4 u[2];
    take(k, u);
    put(k, u);
  }
}

// tokens to 8 bits inside a product: the lane's 16 channels from k on (zeros past K), token row src
__device__ __forceinline__ i4v quantized16(const uint16_t* src, int64_t k, int64_t K, float inv) {
  uint4 u[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    u[p] = make_uint4(0, 0, 0, 0);
    if (k + 8 * p < K) u[p] = *reinterpret_cast<const uint4*>(src + k + 8 * p);
  }
  return __builtin_bit_cast(i4v, codes16(u, inv));
}

// A sum by its token's and its row's scale, of which the token's comes last where it is above 1: sum s would leave the range of 32 bits
// from tokens of about 2^97 on, whatever the row's scale makes of it. {before, after}: one of them is 1.
__device__ __forceinline__ float2 scales(float s) { return s > 1.f ? make_float2(1.f, s) : make_float2(s, 1.f); }
__device__ __forceinline__ float scaled(int sum, float2 s, float row) { return (float)sum * s.x * row * s.y; }

// silu(g) u. With e = 2^(-|g| log2(e) / 2) the sigmoid is 1 / (1 + e^2), of a negative g e^2 / (1 + e^2), whose two factors e go in one
// by one: their product leaves the normal numbers at g = -87, where g u may yet be large. The reciprocal and the exponential are
// within an ulp, which the rounding to bf16 behind them does not show.
__device__ __forceinline__ float gate(float g, float u) {
  const float e = __builtin_amdgcn_exp2f(fabsf(g) * -0.7213475204444817f), f = g < 0.f ? e : 1.f;
  return g * f * u * f * __builtin_amdgcn_rcpf(__builtin_fmaf(e, e, 1.f));
}
struct Out {
  uint16_t* y;
  int64_t ldy, R, N;
  bool wide;                 // rows on 16-byte boundaries
};
// Four outputs of token r from row n of the (padded) weight on; gated: g and u of output f on.
__device__ __forceinline__ void put4(const Out& o, int64_t r, int64_t n, int64_t width, const float (&v)[4]) {
  uint16_t* dst = o.y + r * o.ldy + n;
  if (o.wide && n + 4 <= width) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(kv800::bfpk(v[0], v[1]), kv800::bfpk(v[2], v[3]));
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < width) dst[i] = (uint16_t)kv800::bfpk(v[i], 0.f);
}
// Few tokens: one workgroup takes 32 NT rows of the weight x 32 WM tokens, its 16 / NT waves a part of K each, so that every wave has
// blocks of 1 KB in flight from its first instruction on; their sums meet in LDS, 32 tokens at a time. Output of the instruction
// (weight rows x tokens): lane l holds token l % 32, rows 8 b + 4 (l / 32) + i.
// FUSED (one tile of tokens; how() takes it up to 4): the tokens are rounded to 8 bits by every workgroup for itself, while its first weights are on their way.
template <int NT, int WM, bool GATED, bool FUSED>
__global__ void __launch_bounds__(64 * 16 / NT) few_kernel(const uint16_t* __restrict__ x, int64_t ldx, const int8_t* __restrict__ xq,
                                                       const float* __restrict__ sx, const int8_t* __restrict__ wsh,
                                                       const float* __restrict__ ssh, int64_t K, int64_t nks, Out o) {
  constexpr int FEW = 16 / NT, U = WM == 1 && NT == 2 ? 8 : 4;   // waves; k-steps in flight
  __shared__ int4 part[FEW][NT][4][64];
  __shared__ int tops[32];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t n0 = (int64_t)blockIdx.x * NT, m0 = (int64_t)blockIdx.y * WM;
  const int per = (int)((nks + FEW - 1) / FEW), k0 = wv * per, k1 = min((int)nks, k0 + per);
  const int8_t* wp = wsh + n0 * nks * 1024 + lane * 16;
  const int tok = lane & 31;
  i16v acc[NT][WM];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int b = 0; b < WM; ++b)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[a][b][v] = 0;
  i4v wr[NT][U];
  auto weights = [&](int ks) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int a = 0; a < NT; ++a) wr[a][u] = *reinterpret_cast<const i4v*>(wp + (a * nks + min(ks + u, k1 - 1)) * 1024);
  };
  if (k0 < k1) weights(k0);
  float inv = 0.f;
  if (FUSED) {
    if (tid < 32) tops[tid] = 0;
    __syncthreads();
    const int R = (int)o.R;
    for (int r = 0; r < R; ++r) {
      uint32_t top = 0;
      for (int64_t k = tid * 8; k < K; k += 8 * 64 * FEW) {
        const uint4 u = *reinterpret_cast<const uint4*>(x + r * ldx + k);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
      }
#pragma unroll
      for (int d = 32; d; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
      if (lane == 0) atomicMax(&tops[r], (int)top);
    }
    __syncthreads();
    inv = 127.f / fmaxf(kv800::bf2f((uint32_t)tops[tok]), LEAST);
  }
  for (int ks = k0; ks < k1; ks += U) {
    i4v xr[WM][U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int b = 0; b < WM; ++b) {
        xr[b][u] = i4v{0, 0, 0, 0};
        const int64_t r = (m0 + b) * 32 + tok;
        if (r < o.R && ks + u < k1) {
          if (FUSED) xr[b][u] = quantized16(x + r * ldx, 32 * (int64_t)(ks + u) + 16 * (lane >> 5), K, inv);
          else xr[b][u] = *reinterpret_cast<const i4v*>(xq + ((m0 + b) * nks + ks + u) * 1024 + lane * 16);
        }
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < WM; ++b) acc[a][b] = mfma(wr[a][u], xr[b][u], acc[a][b]);
    if (ks + U < k1) weights(ks + U);
  }
#pragma unroll
  for (int b = 0; b < WM; ++b) {
    if (b) __syncthreads();
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int q = 0; q < 4; ++q) part[wv][a][q][lane] = make_int4(acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]);
    __syncthreads();
    // thread: 4 rows of one token, of tile wv / 4 (gated: waves 0 .. 3, both tiles)
    const int q = wv & 3, row = 8 * q + 4 * (lane >> 5);
    const int64_t r = (m0 + b) * 32 + tok;
    if (r >= o.R || wv >= (GATED ? 4 : 4 * NT)) continue;
    float token;
    if (FUSED) token = tops[tok] < 0x7F80 ? fmaxf(kv800::bf2f((uint32_t)tops[tok]), LEAST) / 127.f : __uint_as_float(0x7FC00000u);
    else token = sx[r];
    const float2 s = scales(token);
    auto sums = [&](int a, float (&f)[4]) {
      int4 t = part[0][a][q][lane];
#pragma unroll
      for (int w = 1; w < FEW; ++w) {
        const int4 p = part[w][a][q][lane];
        t.x += p.x; t.y += p.y; t.z += p.z; t.w += p.w;
      }
      const float4 sc = *reinterpret_cast<const float4*>(ssh + (n0 + a) * 32 + row);
      f[0] = scaled(t.x, s, sc.x); f[1] = scaled(t.y, s, sc.y); f[2] = scaled(t.z, s, sc.z); f[3] = scaled(t.w, s, sc.w);
    };
    float f[4];
    if (GATED) {
      float u[4];
      sums(0, f);
      sums(NT - 1, u);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = gate(f[i], u[i]);
      put4(o, r, n0 * 16 + row, o.N / 2, f);
    } else {
      sums(wv >> 2, f);
      put4(o, r, (n0 + (wv >> 2)) * 32 + row, o.N, f);
    }
  }
}

// Many tokens: one workgroup of 4 waves takes 256 rows of the weight x 128 tokens, 64 channels a stage, three stages in LDS: a stage's
// blocks are loaded straight into LDS two stages ahead, one barrier a stage. A block lies in LDS as it does in memory, in operand
// order, so that loads and reads go over consecutive addresses. A wave has 128 rows x 64 tokens: 6 blocks read from LDS for 8 products.
// Two workgroups share a CU, so that one's epilogue and barriers pass under the other's products: 8192 x 16384 x 2048 gated 300 us
// (310 with the gate that keeps small results); one workgroup of 8 waves for 256 x 256 with two stages of 128 channels 336.
constexpr int TN = 8, TM = 4, STAGE = 2, MANY = 4;       // tiles of 32 of the weight and of tokens, k-steps a stage, waves
constexpr int LOADS = (TN + TM) * STAGE / MANY;          // loads of a wave a stage
struct alignas(16) Stage {
  int8_t b[(TN + TM) * STAGE * 1024];                    // (tile, k-step): the weight's tiles, then the tokens'
};
template <bool GATED>
__global__ void __launch_bounds__(64 * MANY, 2) many_kernel(const int8_t* __restrict__ xq, const float* __restrict__ sx,
                                                            const int8_t* __restrict__ wsh, const float* __restrict__ ssh, int64_t nt,
                                                            int64_t mt, int64_t nks, Out o) {
  __shared__ Stage A, B, C;  // three objects: a read of one is not held for the others' loads
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wv & 1, wm = wv >> 1;
  // workgroup b runs on XCD b % 8, which takes a contiguous run of the order (group of 8 token tiles, weight tile, token tile):
  // the 64 workgroups that run there together share 8 weight tiles and 8 token tiles in its L2
  const int nb = (int)gridDim.x, xcd = (int)blockIdx.x & 7, per = nb >> 3, rem = nb & 7;
  const int L = xcd * per + min(xcd, rem) + ((int)blockIdx.x >> 3);
  const int tn = (int)((nt + TN - 1) / TN), tm = (int)((mt + TM - 1) / TM);
  const int grp = L / (8 * tn), gm = min(8, tm - 8 * grp), in = L - grp * 8 * tn;
  const int64_t n0 = (int64_t)(in / gm) * TN, m0 = (int64_t)(8 * grp + in % gm) * TM;
  // the wave's loads: tiles wv, wv + MANY, ... of the stage; a tile past the last is the last one again, not stored
  const int8_t* src[LOADS / STAGE];
#pragma unroll
  for (int i = 0; i < LOADS / STAGE; ++i) {
    const int t = wv + i * MANY;
    src[i] = (t < TN ? wsh + min(n0 + t, nt - 1) * nks * 1024 : xq + min(m0 + t - TN, mt - 1) * nks * 1024) + lane * 16;
  }
  auto load = [&](int64_t ks, Stage& S) {
#pragma unroll
    for (int i = 0; i < LOADS / STAGE; ++i)
#pragma unroll
      for (int k = 0; k < STAGE; ++k)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src[i] + (ks + k) * 1024),
                                         (__attribute__((address_space(3))) void*)&S.b[((wv + i * MANY) * STAGE + k) * 1024], 16, 0, 0);
    asm volatile("" ::"s"((uint32_t)(uintptr_t)&S) : "memory");   // the loads write S behind the compiler's view of it
  };
  // the wave's LDS reads are done and its loads, but for those of the last stage asked for; then all waves' are
  auto meet = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | LOADS);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  i16v acc[4][2];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[a][b][v] = 0;
  // stage i from S, whose loads have arrived; those of stage i + 2 go out into `later`, whose reads ended at the last barrier (behind
  // the last stage the last one again, so that the number of loads on their way is always the same)
  const int n = (int)(nks / STAGE);
  auto step = [&](int i, const Stage& S, Stage& later) {
    load((int64_t)min(i + 2, n - 1) * STAGE, later);
    i4v a[STAGE][4], b[STAGE][2];
#pragma unroll
    for (int k = 0; k < STAGE; ++k) {
#pragma unroll
      for (int j = 0; j < 2; ++j) b[k][j] = *reinterpret_cast<const i4v*>(&S.b[((TN + 2 * wm + j) * STAGE + k) * 1024 + lane * 16]);
#pragma unroll
      for (int i = 0; i < 4; ++i) a[k][i] = *reinterpret_cast<const i4v*>(&S.b[((4 * wn + i) * STAGE + k) * 1024 + lane * 16]);
    }
#pragma unroll
    for (int k = 0; k < STAGE; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma(a[k][i], b[k][j], acc[i][j]);
    // all of the stage's reads before its products: read one by one, each pair of products waited for its operand
    __builtin_amdgcn_sched_group_barrier(0x100, 6 * STAGE, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, 8 * STAGE, 0);
    meet();
  };
  load(0, A);
  load((int64_t)min(1, n - 1) * STAGE, B);
  meet();
  for (int i = 0;;) {
    step(i, A, C);
    if (++i == n) break;
    step(i, B, A);
    if (++i == n) break;
    step(i, C, B);
    if (++i == n) break;
  }
  __builtin_amdgcn_s_waitcnt(0x0070);                    // nothing is on its way to LDS any more
  __syncthreads();
  // The outputs leave through LDS, so that a row's go out side by side (straight from the registers they are 16 bytes a line and store:
  // 325 us): 64 tokens x 64 outputs a wave and pass, rows of 144 bytes.
  constexpr int ROW = 144;
  uint8_t* buf = reinterpret_cast<uint8_t*>(wv < 2 ? A.b : B.b) + (wv & 1) * 64 * ROW;
  static_assert(2 * 64 * ROW <= (int)sizeof(Stage), "two waves' outputs fit a stage");
  const int64_t width = GATED ? o.N / 2 : o.N, t0 = (m0 + 2 * wm) * 32;
  float2 s[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) s[j] = scales(sx[min(t0 + 32 * j + (lane & 31), o.R - 1)]);
#pragma unroll
  for (int pass = 0; pass < (GATED ? 1 : 2); ++pass) {
    if (pass) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int c = 0; c < 2; ++c)                          // 32 outputs: of tiles 2 c and 2 c + 1, or of tile 2 pass + c
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = GATED ? 2 * c : 2 * pass + c, row = 8 * q + 4 * (lane >> 5);
        const float4 k0 = *reinterpret_cast<const float4*>(ssh + min(n0 + 4 * wn + i, nt - 1) * 32 + row);
        const float4 k1 = GATED ? *reinterpret_cast<const float4*>(ssh + min(n0 + 4 * wn + i + 1, nt - 1) * 32 + row) : k0;
        const float ka[4] = {k0.x, k0.y, k0.z, k0.w}, kb[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[e] = scaled(acc[i][j][4 * q + e], s[j], ka[e]);
            if (GATED) f[e] = gate(f[e], scaled(acc[i + (GATED ? 1 : 0)][j][4 * q + e], s[j], kb[e]));
          }
          *reinterpret_cast<uint2*>(buf + (32 * j + (lane & 31)) * ROW + (32 * c + row) * 2) = make_uint2(kv800::bfpk(f[0], f[1]), kv800::bfpk(f[2], f[3]));
        }
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int64_t n = (GATED ? (n0 + 4 * wn) * 16 : (n0 + 4 * wn + 2 * pass) * 32) + (lane & 7) * 8;
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int tr = it * 8 + (lane >> 3);
      const int64_t r = t0 + tr;
      if (r >= o.R || n >= width) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(buf + tr * ROW + (lane & 7) * 16);
      uint16_t* dst = o.y + r * o.ldy + n;
      if (o.wide && n + 8 <= width) {
        *reinterpret_cast<uint4*>(dst) = v;
      } else {
        const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (n + i < width) dst[i] = (uint16_t)(e[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
}

// ---------------------------------------------------------------- host
constexpr int64_t K_MOST = 65536;      // 127^2 K below 2^31
int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
int64_t padded_rows(int64_t N, int gated) { return gated ? 2 * round_up(N / 2, 32) : round_up(N, 64); }
bool sizes(int64_t R, int64_t N, int64_t K, int gated) {
  return R >= 0 && R < (1 << 24) && N > 0 && N < (1 << 24) && K > 0 && K <= K_MOST && K % 8 == 0 && (gated == 0 || (gated == 1 && N % 2 == 0));
}

// How a product runs: in 256 x 128 tiles, or on few_kernel with nt tiles of the weight and wm of the tokens a workgroup, which rounds
// the tokens itself or not. Times of whole calls on both sides of each rule, us (tokens x rows of the weight x K):
//   tiles, from 112 on: 256 x 16384 x 2048 gated (128) 25.7, few 29.7; 512 x 6144 x 2048 (96) 26.9, few 21.2; 1024 x 2048 x 8192 (64) 80, few 40
//   rounding inside, one round of workgroups (256) of up to 8 steps of 32 channels a wave, on one tile of the weight up to 256 tiles
//     and on two up to 512. Weight rows on the border and behind it, 1 / 4 tokens: x 2048, 8192 8.0 / 9.3, apart 12.5 / 12.7; 10240 on
//     two tiles 8.9 / 11.0, on one 12.7 / 16.0, apart 12.4 / 12.5; 14336 10.6 / 12.1, apart 12.6 / 12.8; 16512 17.9 / 20.3, apart 12.8 / 13.1.
//     Channels: 6144 on one tile, x 4096 11.3 / 13.4, apart 12.6 / 12.7, x 8192 20.5 / 21.5, apart 15.1 / 15.0; 8192 gated on two, x 2048
//     9.3 / 10.5, apart 12.5 / 12.7, x 2560 12.2 / 13.8, apart 12.7 / 12.8, x 4096 16.1 / 17.3, apart 12.5 / 12.7. 16 x 16384 x 2048
//     19.2, apart 12.8.
//   16 waves on one tile of the weight: 256 x 2048 x 8192 18.6, 8 waves on two 21.8; 1024 x 2048 x 8192 50.6, 40.2
//   32 tokens a workgroup: 64 x 2048 x 8192 13.2, 64 tokens 15.2; 256 x 2048 x 8192 19.1, 18.6
struct How {
  bool tiles, fused;
  int nt, wm;
};
How how(int64_t R, int64_t N, int64_t K, int gated) {
  const int64_t nt = padded_rows(N, gated) / 32, mt = (R + 31) / 32;
  How h = {false, false, 2, mt > 1 ? 2 : 1};
  h.tiles = ((nt + TN - 1) / TN) * ((mt + TM - 1) / TM) >= 112;
  const bool one = !gated && nt <= 256;
  if (!h.tiles && R <= 4 && nt <= 512 && K <= (one ? 4096 : 2048)) {
    h.fused = true;
    h.nt = one ? 1 : 2;
  } else if (!gated && (nt / 2) * ((mt + 1) / 2) < 256) {
    h.nt = 1;
    h.wm = nt * mt <= 256 ? 1 : 2;
  }
  return h;
}

}  // namespace
}  // namespace lfm3

extern "C" {

int lfm3_hip_int8_layout(const int8_t* w, int64_t ld, const float* scale, int64_t N, int64_t K, int gated, int8_t* wsh, float* ssh,
                         void* stream) {
  KV800_REQUIRE(lfm3::sizes(0, N, K, gated) && ld >= 0, "int8_layout: N below 2^24 (even for a gated weight), K a multiple of 8 up to 65536");
  KV800_REQUIRE(w && scale && wsh && ssh && (uintptr_t)wsh % 16 == 0 && (uintptr_t)ssh % 16 == 0, "int8_layout: null or unaligned pointer");
  const int64_t Npad = lfm3::padded_rows(N, gated), nks = lfm3::round_up(K, 128) / 32, n = Npad / 32 * nks * 64;
  KV800_REQUIRE(n < (int64_t)1 << 32, "int8_layout: a weight of 64 GiB or more");   // 2^32 threads a launch
  hipLaunchKernelGGL(lfm3::layout_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, w, ld, scale, N, K,
                     Npad, nks, gated, wsh, ssh);
  return kv800::check_launch("int8_layout");
}

int lfm3_hip_int8_quantize(const uint16_t* w, int64_t ld, int64_t N, int64_t K, int8_t* w8, float* scale, void* stream) {
  KV800_REQUIRE(lfm3::sizes(0, N, K, 0) && ld % 8 == 0, "int8_quantize: N below 2^24, K a multiple of 8 up to 65536, ld a multiple of 8");
  KV800_REQUIRE(w && w8 && scale && (uintptr_t)w % 16 == 0 && (uintptr_t)w8 % 8 == 0, "int8_quantize: null or unaligned pointer");
  hipLaunchKernelGGL((lfm3::quantize_kernel<false, 4>), dim3((unsigned)N), dim3(256), 0, (hipStream_t)stream, w, ld, N, K, 0,
                     w8, scale);
  return kv800::check_launch("int8_quantize");
}

int64_t lfm3_hip_linear8_workspace(int64_t R, int64_t N, int64_t K, int gated) {
  if (!lfm3::sizes(R, N, K, gated) || R == 0) return 0;
  if (lfm3::how(R, N, K, gated).fused) return 0;
  const int64_t mpad = lfm3::round_up(R, 32);
  return mpad * lfm3::round_up(K, 128) + mpad * 4;
}

int lfm3_hip_linear8(const uint16_t* x, int64_t ldx, const int8_t* wsh, const float* ssh, int64_t R, int64_t N, int64_t K,
                     int gated, uint16_t* y, int64_t ldy, void* ws, int64_t ws_bytes, void* stream) {
  KV800_REQUIRE(lfm3::sizes(R, N, K, gated),
                "linear8: R and N below 2^24 (N even for a gated weight), K a multiple of 8 up to 65536, gated 0 or 1");
  KV800_REQUIRE(ldx % 8 == 0 && ldy >= 0, "linear8: ldx must be a multiple of 8 and ldy >= 0");
  if (R == 0) return KV800_OK;
  KV800_REQUIRE(x && wsh && ssh && y && (uintptr_t)x % 16 == 0 && (uintptr_t)wsh % 16 == 0 && (uintptr_t)ssh % 16 == 0, "linear8: null or unaligned pointer");
  const int64_t need = lfm3_hip_linear8_workspace(R, N, K, gated);
  KV800_REQUIRE(need == 0 || (ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need), "linear8: %lld bytes of 16-byte aligned workspace needed", (long long)need);
  const int64_t mt = lfm3::round_up(R, 32) / 32, nt = lfm3::padded_rows(N, gated) / 32, nks = lfm3::round_up(K, 128) / 32;
  const lfm3::Out o = {y, ldy, R, N, ldy % 8 == 0 && (uintptr_t)y % 16 == 0};
  const lfm3::How h = lfm3::how(R, N, K, gated);
  hipStream_t st = (hipStream_t)stream;
  int8_t* xq = (int8_t*)ws;
  float* sx = (float*)(xq + mt * nks * 1024);
  if (!h.fused) {
    // a wave a row: 8192 x 2048 x 2048 49.4 us, a workgroup a row 56; 1024 x 2048 x 8192 41.7, 40.4
    if (R >= 1024 && K <= 2048)
      hipLaunchKernelGGL((lfm3::quantize_kernel<true, 1>), dim3((unsigned)((R + 3) / 4)), dim3(256), 0, st, x, ldx, R, K, nks, xq, sx);
    else
      hipLaunchKernelGGL((lfm3::quantize_kernel<true, 4>), dim3((unsigned)R), dim3(256), 0, st, x, ldx, R, K, nks, xq, sx);
    const int rc = kv800::check_launch("linear8 quantize");
    if (rc != KV800_OK) return rc;
  }
  auto few = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(nt / h.nt), (unsigned)((mt + h.wm - 1) / h.wm)), dim3((unsigned)(1024 / h.nt)), 0, st, x, ldx, xq,
                       sx, wsh, ssh, K, nks, o);
  };
  if (h.fused) {
    if (gated) few(lfm3::few_kernel<2, 1, true, true>);
    else if (h.nt == 1) few(lfm3::few_kernel<1, 1, false, true>);
    else few(lfm3::few_kernel<2, 1, false, true>);
  } else if (!h.tiles && h.wm == 1) {
    if (gated) few(lfm3::few_kernel<2, 1, true, false>);
    else if (h.nt == 1) few(lfm3::few_kernel<1, 1, false, false>);
    else few(lfm3::few_kernel<2, 1, false, false>);
  } else if (!h.tiles) {
    if (gated) few(lfm3::few_kernel<2, 2, true, false>);
    else if (h.nt == 1) few(lfm3::few_kernel<1, 2, false, false>);
    else few(lfm3::few_kernel<2, 2, false, false>);
  } else {
    const dim3 grid((unsigned)((nt + lfm3::TN - 1) / lfm3::TN * ((mt + lfm3::TM - 1) / lfm3::TM)));
    if (gated) hipLaunchKernelGGL(lfm3::many_kernel<true>, grid, dim3(64 * lfm3::MANY), 0, st, xq, sx, wsh, ssh, nt, mt, nks, o);
    else hipLaunchKernelGGL(lfm3::many_kernel<false>, grid, dim3(64 * lfm3::MANY), 0, st, xq, sx, wsh, ssh, nt, mt, nks, o);
  }
  return kv800::check_launch("linear8");
}

}  // extern "C"
