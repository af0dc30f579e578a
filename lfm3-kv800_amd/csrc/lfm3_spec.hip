// lfm3_spec.hip -- model-side operators of a step whose rows bring several new tokens each (include/lfm3_spec.h), gfx950.
//
//   conv_chunk_kernel     the gated short conv over each row's new tokens, from the row's 6-tap state
//   conv_commit_kernel    that state moved on over the tokens that were kept
//   verify_stats_kernel     per piece of a logits row: largest value, its index, sum of exponentials
//   verify_residual_kernel  per piece of the logits row that ends a batch row: what p has over q
//   verify_pick_kernel      per batch row: which drafts are kept, and the token behind them
#include <type_traits>

#include "kv800_common.h"
#include "../../include/kv800_hip.h"
#include "../../include/lfm3_spec.h"

namespace lfm3 {
namespace {

using kv800::bf2f;
using kv800::f2bf;
using kv800::ranks_before;
using kv800::row_of;

__device__ __forceinline__ void load8(const uint16_t* p, float (&f)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = kv800::bf2f_lo(w[i]); f[2 * i + 1] = kv800::bf2f_hi(w[i]); }
}
__device__ __forceinline__ void store8(uint16_t* p, const float (&f)[8]) {
  uint4 u;
  u.x = f2bf(f[0]) | (f2bf(f[1]) << 16); u.y = f2bf(f[2]) | (f2bf(f[3]) << 16);
  u.z = f2bf(f[4]) | (f2bf(f[5]) << 16); u.w = f2bf(f[6]) | (f2bf(f[7]) << 16);
  *reinterpret_cast<uint4*>(p) = u;
}

// ---------------------------------------------------------------- short conv over a row's new tokens
// One workgroup per (TT consecutive tokens, 2048 channels); a thread holds 8 channels' window of 7 taps in registers and
// slides it over the tokens, so each token's B, C and x are read once (the 6 taps before the first token again).
// The tokens may lie in several rows: at a row's first token the window is its state.
// TAPS are rounded to bf16, the type of the state, before the products, so that a window does not depend on which of its
// taps have been committed; the products and the sum stay in fp32 and the output is rounded once.
template <int TT>
__global__ void __launch_bounds__(256)
conv_chunk_kernel(const uint16_t* __restrict__ bcx, int64_t stride, const uint16_t* __restrict__ cw,
                  const uint16_t* __restrict__ state, const int64_t* __restrict__ qsl, int64_t R, int64_t T, int64_t H,
                  uint16_t* __restrict__ out, uint16_t* __restrict__ taps) {
  // workgroups go round the 8 XCDs: four tiles in a row to one of them, so that three of them may find their first taps in its
  // L2 (2,048 tokens 12.5 -> 11.0 us, 4,096 18.3 -> 17.0; 16,384 the same: 300 MB fetched, which is every such tap again; a
  // whole eighth to each: 69 -> 73)
  const int64_t t0 = ((int64_t)((blockIdx.x >> 5) * 8 + (blockIdx.x & 7)) * 4 + ((blockIdx.x >> 3) & 3)) * TT;
  const int64_t c0 = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8;
  if (t0 >= T) return;                                 // uniform
  const int64_t total = min(qsl[R], T);
  int64_t r = row_of(qsl, R, t0);                      // by whole waves: before any lane leaves
  if (c0 >= H) return;
  float win[6][8];                                     // the 6 taps before the current token, the oldest first
  auto from_state = [&](int64_t row) {
    const uint4* s = reinterpret_cast<const uint4*>(state + (row * H + c0) * 6);   // 8 channels x 6 taps
    uint32_t x[24];
#pragma unroll
    for (int i = 0; i < 6; ++i) { const uint4 v = s[i]; x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w; }
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int k = 0; k < 6; ++k) win[k][c] = ((c * 6 + k) & 1) ? kv800::bf2f_hi(x[(c * 6 + k) / 2]) : kv800::bf2f_lo(x[(c * 6 + k) / 2]);
  };
  auto tap = [&](int64_t t, float (&f)[8]) {
    float b[8];
    load8(bcx + t * stride + c0, b);
    load8(bcx + t * stride + 2 * H + c0, f);
#pragma unroll
    for (int c = 0; c < 8; ++c) f[c] = kv800::bfround(b[c] * f[c]);
  };
  uint32_t cwp[28];                                    // the 8 channels' 7 weights, two a register
  {
    const uint4* s = reinterpret_cast<const uint4*>(cw + c0 * 7);
#pragma unroll
    for (int i = 0; i < 7; ++i) { const uint4 v = s[i]; cwp[4 * i] = v.x; cwp[4 * i + 1] = v.y; cwp[4 * i + 2] = v.z; cwp[4 * i + 3] = v.w; }
  }
  auto wt = [&](int k, int c) { const int e = c * 7 + k; return (e & 1) ? kv800::bf2f_hi(cwp[e / 2]) : kv800::bf2f_lo(cwp[e / 2]); };
  if (t0 < total) {
    const int64_t s0 = qsl[r];
    if (t0 - s0 < 6) from_state(r);
    // the window behind the row's i = t0 - s0 first tokens: state taps i .., then the tokens' own
    const int64_t i0 = t0 - s0;
    if (i0 > 0) {
      if (i0 < 6) {
        for (int64_t i = 0; i < i0; ++i) {
          float f[8];
          tap(s0 + i, f);
#pragma unroll
          for (int k = 0; k < 5; ++k)
#pragma unroll
            for (int c = 0; c < 8; ++c) win[k][c] = win[k + 1][c];
#pragma unroll
          for (int c = 0; c < 8; ++c) win[5][c] = f[c];
        }
      } else {
#pragma unroll
        for (int k = 0; k < 6; ++k) tap(t0 - 6 + k, win[k]);
      }
    }
  }
#pragma unroll 4
  for (int j = 0; j < TT; ++j) {
    const int64_t t = t0 + j;
    if (t >= T) break;
    float y[8] = {0, 0, 0, 0, 0, 0, 0, 0}, f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (t < total) {
      if (j > 0 && t >= qsl[r + 1]) {                  // the next row that has tokens
        do ++r; while (t >= qsl[r + 1]);
        from_state(r);
      }
      float g[8];
      load8(bcx + t * stride + H + c0, g);
      tap(t, f);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
#pragma unroll
        for (int k = 0; k < 6; ++k) y[c] = fmaf(win[k][c], wt(k, c), y[c]);
        y[c] = fmaf(f[c], wt(6, c), y[c]) * g[c];
      }
#pragma unroll
      for (int k = 0; k < 5; ++k)
#pragma unroll
        for (int c = 0; c < 8; ++c) win[k][c] = win[k + 1][c];
#pragma unroll
      for (int c = 0; c < 8; ++c) win[5][c] = f[c];
    }
    store8(out + t * H + c0, y);
    store8(taps + t * H + c0, f);
  }
}

// One thread per (row, 8 channels): the last 6 of the state and the row's first a taps.
__global__ void __launch_bounds__(256)
conv_commit_kernel(uint16_t* __restrict__ state, const uint16_t* __restrict__ taps, const int64_t* __restrict__ qsl,
                   const int32_t* __restrict__ kept, int64_t R, int64_t T, int64_t H) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= R * (H / 8)) return;
  const int64_t r = i / (H / 8), c0 = i % (H / 8) * 8;
  const int64_t s0 = min(qsl[r], T), n = min(qsl[r + 1], T) - s0, a = min(max((int64_t)kept[r], (int64_t)0), n);
  if (a <= 0) return;
  uint4* sp = reinterpret_cast<uint4*>(state + (r * H + c0) * 6);
  uint32_t x[24], y[24];
  uint16_t old[8][6], z[8][6];
#pragma unroll
  for (int k = 0; k < 6; ++k) { const uint4 v = sp[k]; x[4 * k] = v.x; x[4 * k + 1] = v.y; x[4 * k + 2] = v.z; x[4 * k + 3] = v.w; }
#pragma unroll
  for (int c = 0; c < 8; ++c)
#pragma unroll
    for (int k = 0; k < 6; ++k) old[c][k] = (uint16_t)(x[(c * 6 + k) / 2] >> (16 * ((c * 6 + k) & 1)));
#pragma unroll
  for (int k = 0; k < 6; ++k) {                        // new tap k = tap a - 6 + k of the row, or state tap a + k
    const int64_t j = a - 6 + k;
    uint4 v = {0, 0, 0, 0};
    if (j >= 0) v = *reinterpret_cast<const uint4*>(taps + (s0 + j) * H + c0);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      uint16_t o = 0;
#pragma unroll
      for (int q = 0; q < 6; ++q)
        if (q == a + k) o = old[c][q];
      z[c][k] = j >= 0 ? (uint16_t)(u[c / 2] >> (16 * (c & 1))) : o;
    }
  }
#pragma unroll
  for (int e = 0; e < 24; ++e) y[e] = (uint32_t)z[2 * e / 6][2 * e % 6] | ((uint32_t)z[(2 * e + 1) / 6][(2 * e + 1) % 6] << 16);
#pragma unroll
  for (int k = 0; k < 6; ++k) sp[k] = make_uint4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
}

// ---------------------------------------------------------------- verification of drafts
// A logits row is cut into pieces; verify_stats gives each piece's largest value m, its index and s = sum exp((x - m) / temp).
// verify_residual (drafts with a distribution), else verify_pick, derives from these which row of logits ends a batch row, each
// workgroup for itself; the first sums max(p - q, 0) over its piece of that row, the second picks the piece in which the
// running sum passes u W and scans it. So every row of logits is read once, the deciding one of each batch row (and its
// q) once more, and one piece of it again.
// All in 64 bits: the running sums of neighbours among 65,536 tokens lie 1e-5 apart where 32-bit exponentials are
// 1e-7 off, and the choice has to be the same whatever way a row is cut. Bound: the logits' bytes and the exponentials'
// instructions: about 30 per value, half of them of 64 bits, take longer than the bytes. 256 rows, 722 logits rows of 65,536 with
// the drafts' distributions (162 MB): stats 37, residual 16, pick 10 us; one row of 5: 3.4, 0 and 8 us, chains of dependent
// loads and of 64-bit sums over lanes.
constexpr int VT = 256;                                // threads; a piece holds VT x VE values, VE = 8 or 32 a thread
struct Stat { double s; float m; int32_t at; };        // 16 bytes

// whether a row with largest logit m is sampled: a temperature in (0, 1e30] and a finite m; else its choice is m's index
__device__ __forceinline__ bool sampled(float tp, float m) { return tp > 0.f && tp <= 1e30f && m - m == 0.f; }
// Reductions over a wave, the same in every lane: partners within rows of 16 by DPP (neighbours 1 and 2 apart, then mirrored
// halves and rows, whose lanes are alike by then), across the rows by lane swaps, which return the values of both sides.
// (By __shfl_xor, through the LDS, and with the deciding token combined twice: 256 rows 73 us of kernels instead of 68, one
// row 14 instead of 11.6.)
constexpr int DPP_STEP[4] = {0xB1, 0x4E, 0x141, 0x140};   // quad_perm [1 0 3 2], [2 3 0 1], row_half_mirror, row_mirror
template <int K>
__device__ __forceinline__ uint32_t dpp(uint32_t x) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, DPP_STEP[K], 0xF, 0xF, false); }
struct Pair32 { uint32_t a, b; };
template <int K>
__device__ __forceinline__ Pair32 both_sides(uint32_t x) {   // step K: this lane's value and its partner's, or the two in lane order
  if constexpr (K < 4) return {x, dpp<K>(x)};
  else if constexpr (K == 4) { const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false); return {r[0], r[1]}; }
  else { const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false); return {r[0], r[1]}; }
}
template <int K = 0>
__device__ __forceinline__ double wave_sumd(double v) {
  const uint64_t x = __builtin_bit_cast(uint64_t, v);
  const Pair32 lo = both_sides<K>((uint32_t)x), hi = both_sides<K>((uint32_t)(x >> 32));
  v = __builtin_bit_cast(double, ((uint64_t)hi.a << 32) | lo.a) + __builtin_bit_cast(double, ((uint64_t)hi.b << 32) | lo.b);
  if constexpr (K < 5) return wave_sumd<K + 1>(v);
  else return v;
}
template <int K = 0>
__device__ __forceinline__ float wave_maxn(float v) {        // NaN wins
  const Pair32 x = both_sides<K>(__float_as_uint(v));
  v = __builtin_elementwise_maximum(__uint_as_float(x.a), __uint_as_float(x.b));
  if constexpr (K < 5) return wave_maxn<K + 1>(v);
  else return v;
}
template <int K = 0>
__device__ __forceinline__ void wave_first(float& m, int& at) {   // the first in rank of the lanes' (m, at)
  const Pair32 x = both_sides<K>(__float_as_uint(m)), i = both_sides<K>((uint32_t)at);
  const bool second = ranks_before(__uint_as_float(x.b), (int)i.b, __uint_as_float(x.a), (int)i.a);
  m = __uint_as_float(second ? x.b : x.a);
  at = (int)(second ? i.b : i.a);
  if constexpr (K < 5) wave_first<K + 1>(m, at);
}
// exp((x - m) / temp) for x <= m, within 2^-42, by a table of powers of two and a short series (Tang's table-driven
// exponential): y = (x - m) / temp with the difference exact, so that a small temperature does
// not enlarge its rounding, = (16 e + j) ln2 / 16 + r, |r| <= ln2 / 32; 16 e + j is the low word of 16 y / ln2 + 1.5 2^52; 2^(j / 16)
// from a table of 16 in LDS (32 banks: any lanes at once), exp(r) as its series to r^5 / 120 (the next term is 1.4e-13). What
// lies 800 temp below m, -inf among it, is 2^-1154 and comes out as 0.
__device__ const double POW16[16] = {1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916, 1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927, 1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543, 1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};
struct Expo { double m, it; };
__device__ __forceinline__ double expo(float x, const Expo& E, const double* pow16) {
  const double magic = 6755399441055744.0;             // 1.5 2^52
  const double y = __builtin_elementwise_max(((double)x - E.m) * E.it, -800.0);
  const double zz = fma(y, 23.083120654223414, magic);   // 16 / ln2
  const double r = fma(zz - magic, -0.043321698784996581, y);   // ln2 / 16
  const int k = (int)(uint32_t)__double_as_longlong(zz);
  double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(r, p, 1.0 / 6.0);
  p = fma(r, p, 0.5);
  p = fma(r, p, 1.0);
  p = fma(r, p, 1.0);
  return ldexp(p * pow16[k & 15], k >> 4);
}

// Eight values from index i of a piece of n on: 16-byte loads where they are all there and aligned, else one by one; what
// lies past n is `fill`.
__device__ __forceinline__ void load_group(const uint16_t* p, int i, int n, float fill, float (&x)[8]) {
  if (((uintptr_t)p & 15) == 0 && i + 8 <= n) load8(p + i, x);
  else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = i + e < n ? bf2f(p[i + e]) : fill;
  }
}
__device__ __forceinline__ void load_group(const float* p, int i, int n, float fill, float (&x)[8]) {
  if (((uintptr_t)p & 15) == 0 && i + 8 <= n) {
    const float4 a = *reinterpret_cast<const float4*>(p + i), b = *reinterpret_cast<const float4*>(p + i + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = i + e < n ? p[i + e] : fill;
  }
}
// a thread's group k of a piece: the 8 values from here on
__device__ __forceinline__ int group_at(int k) { return 8 * (VT * k + (int)threadIdx.x); }

// What a batch row comes to, the same in every thread of the workgroup.
struct Verdict {
  int64_t s0, s1, t;   // the row's tokens; the logits row that ends it
  float m;             // that row's largest logit,
  int at;              // where it is,
  double s;            // sum of exp((x - m) / temp)
  double it;           // 1 / temp
  bool sample, full;   // sampled; all drafts kept
};
struct VerifyArgs {
  const uint16_t* logits;
  int64_t ld;
  const int64_t *tokens, *qsl;
  const float *temp, *u, *u_next, *q;
  int64_t ldq, R, T, V, pieces;
  Stat* st;            // (T, pieces)
  double* left;        // (R, pieces): sums of max(p - q, 0) over the deciding rows' pieces
  Verdict* verdicts;   // (R): of the rows with drafts, where these have a distribution
  int64_t* out;
  int32_t* count;
};

template <int VE>
__global__ void __launch_bounds__(VT) verify_stats_kernel(VerifyArgs A) {
  __shared__ double pow16[16], rs[4];
  __shared__ float rm[4];
  __shared__ int at;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int64_t t = blockIdx.y, v0 = (int64_t)blockIdx.x * (VT * VE);
  if (t >= min(A.qsl[A.R], A.T)) return;               // uniform
  const int n = (int)min((int64_t)(VT * VE), A.V - v0);
  float x[VE / 8][8];
#pragma unroll
  for (int k = 0; k < VE / 8; ++k) load_group(A.logits + t * A.ld + v0, group_at(k), n, -INFINITY, x[k]);
  if (tid < 16) pow16[tid] = POW16[tid];
  const float tp = A.temp[row_of(A.qsl, A.R, t)];
  // the piece's largest value first (NaN wins), then the first index that has it, by the threads whose own largest it is: about
  // 35 instructions a value in all are what the kernel takes its time for, six of them fewer than with an index along
  float own = -INFINITY;
#pragma unroll
  for (int k = 0; k < VE / 8; ++k)
#pragma unroll
    for (int e = 0; e < 8; e += 2) own = __builtin_elementwise_maximum(own, __builtin_elementwise_maximum(x[k][e], x[k][e + 1]));
  float bm = wave_maxn(own);
  if (lane == 0) rm[w] = bm;
  if (tid == 0) at = 0x7FFFFFFF;
  __syncthreads();
  bm = __builtin_elementwise_maximum(__builtin_elementwise_maximum(rm[0], rm[1]), __builtin_elementwise_maximum(rm[2], rm[3]));
  if (own == bm || own != own) {
    int bi = 0x7FFFFFFF;
#pragma unroll
    for (int k = VE / 8 - 1; k >= 0; --k)
#pragma unroll
      for (int e = 7; e >= 0; --e) {
        const int i = group_at(k) + e;
        bi = (x[k][e] == bm || x[k][e] != x[k][e]) && i < n ? i : bi;
      }
    atomicMin(&at, bi);                                // the smallest index, whatever the order
  }
  double s = 0.0;
  if (sampled(tp, bm)) {
    const Expo E = {(double)bm, 1.0 / (double)tp};
#pragma unroll
    for (int k = 0; k < VE / 8; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += expo(x[k][e], E, pow16);        // 0 for what lies past the row
  }
  s = wave_sumd(s);
  if (lane == 0) rs[w] = s;
  __syncthreads();
  if (tid == 0) A.st[t * A.pieces + blockIdx.x] = Stat{(rs[0] + rs[1]) + (rs[2] + rs[3]), bm, (int32_t)(v0 + at)};
}

struct VerdictLds { long long stop; double pow16[16], s; float m; int at; };
__device__ __forceinline__ Verdict decide(const VerifyArgs& A, int64_t r, VerdictLds& L) {
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  Verdict d;
  d.s0 = min(A.qsl[r], A.T);
  d.s1 = min(A.qsl[r + 1], A.T);
  const float tp = A.temp[r];
  d.it = 1.0 / (double)tp;
  if (tid < 16) L.pow16[tid] = POW16[tid];
  if (tid == 0) L.stop = d.s1 - 1;
  __syncthreads();
  // a logits row's pieces combined, by a wave: the same result in every lane
  auto combine = [&](int64_t t, float& M, int& at, double& S) {
    M = -INFINITY;
    at = 0x7FFFFFFF;
    for (int64_t p = lane; p < A.pieces; p += 64) {
      const Stat a = A.st[t * A.pieces + p];
      if (ranks_before(a.m, a.at, M, at)) { M = a.m; at = a.at; }
    }
    wave_first(M, at);
    S = 0.0;
    if (sampled(tp, M))
      for (int64_t p = lane; p < A.pieces; p += 64) {
        const Stat a = A.st[t * A.pieces + p];
        S += a.s * expo(a.m, Expo{(double)M, d.it}, L.pow16);
      }
    S = wave_sumd(S);
  };
  // the wave that looks at the row's deciding token leaves what it found: the token breaks its loop, or is the row's last
  float M = -INFINITY;
  int at = 0x7FFFFFFF;
  double S = 0.0;
  int64_t mine = -1;
  for (int64_t t = d.s0 + w; t < d.s1; t += VT / 64) {
    const bool draft = t < d.s1 - 1;
    const int64_t k = draft ? A.tokens[t + 1] : -1;
    const bool in = k >= 0 && k < A.V;
    const float xk = in ? bf2f(A.logits[t * A.ld + k]) : -INFINITY, ut = draft ? A.u[t] : 0.f;
    const double qk = A.q ? (in ? (double)A.q[t * A.ldq + k] : 0.0) : 1.0;
    combine(t, M, at, S);
    mine = t;
    if (!draft) break;
    const bool keep = sampled(tp, M) ? in && (double)ut * qk < expo(xk, Expo{(double)M, d.it}, L.pow16) / S : k == at;
    if (!keep) {
      if (lane == 0) atomicMin(&L.stop, (long long)t);
      break;
    }
  }
  __syncthreads();
  d.t = L.stop;
  if (mine == d.t && lane == 0) { L.m = M; L.at = at; L.s = S; }
  __syncthreads();
  d.m = L.m;
  d.at = L.at;
  d.s = L.s;
  d.sample = sampled(tp, d.m);
  d.full = d.t == d.s1 - 1;
  return d;
}

// Weights of group k of a piece of the deciding row: mode 0: exp((x - m) / temp); 1: the same without token `skip`; 2:
// max(p - q, 0).
template <int VE>
__device__ __forceinline__ void group_weights(const VerifyArgs& A, const Verdict& d, const double* pow16, int64_t piece, int k, int mode,
                                              int64_t skip, double (&g)[8]) {
  const int64_t v0 = piece * (VT * VE);
  const int n = (int)min((int64_t)(VT * VE), A.V - v0), i = group_at(k);
  float x[8], q[8];
  load_group(A.logits + d.t * A.ld + v0, i, n, -INFINITY, x);
  if (mode == 2) load_group(A.q + d.t * A.ldq + v0, i, n, 0.f, q);
  const double inv = 1.0 / d.s;
  const Expo E = {(double)d.m, d.it};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    double y = expo(x[e], E, pow16);
    if (mode == 1) y = v0 + i + e == skip ? 0.0 : y;
    if (mode == 2) {
      y = y * inv - (double)q[e];
      y = y > 0.0 ? y : 0.0;                           // and for a q that is NaN
    }
    g[e] = y;
  }
}
__device__ __forceinline__ double sum8(const double (&g)[8]) {
  return ((g[0] + g[1]) + (g[2] + g[3])) + ((g[4] + g[5]) + (g[6] + g[7]));
}
// The sum of a piece's weights, in the order in which pick_kernel takes it apart; group(k, g) gives a thread's weights of
// group k. The same in every thread.
template <int VE, typename F>
__device__ __forceinline__ double piece_sum(double* seg, F group) {
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  __syncthreads();                                     // seg's last readers are done
#pragma unroll
  for (int k = 0; k < VE / 8; ++k) {
    double g[8];
    group(k, g);
    const double s = wave_sumd(sum8(g));
    if (lane == 0) seg[4 * k + w] = s;                 // 64 lanes x 8 values from index 512 (4 k + w) on
  }
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < VE / 2; ++k) s += seg[k];
  return s;
}

template <int VE>
__global__ void __launch_bounds__(VT, 8) verify_residual_kernel(VerifyArgs A) {
  __shared__ VerdictLds L;
  __shared__ double seg[VE / 2];
  const int64_t r = blockIdx.y;
  if (min(A.qsl[r + 1], A.T) - min(A.qsl[r], A.T) < 2) return;   // no drafts
  const Verdict d = decide(A, r, L);
  if (blockIdx.x == 0 && threadIdx.x == 0) A.verdicts[r] = d;    // for verify_pick
  if (!d.sample || d.full) return;
  const double s = piece_sum<VE>(seg, [&](int k, double (&g)[8]) { group_weights<VE>(A, d, L.pow16, blockIdx.x, k, 2, -1, g); });
  if (threadIdx.x == 0) A.left[r * A.pieces + blockIdx.x] = s;
}

template <int VE>
__global__ void __launch_bounds__(VT) verify_pick_kernel(VerifyArgs A) {
  __shared__ VerdictLds L;
  __shared__ double seg[VE / 2], total;
  __shared__ int piece, where;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int64_t r = blockIdx.x;
  {
    const int64_t s0 = min(A.qsl[r], A.T), s1 = min(A.qsl[r + 1], A.T);
    if (r == A.R - 1)
      for (int64_t t = s1 + tid; t < A.T; t += VT) A.out[t] = -1;   // the padding
    if (s1 <= s0) {
      if (tid == 0) A.count[r] = 0;
      return;
    }
  }
  Verdict d;
  if (A.q && min(A.qsl[r + 1], A.T) - min(A.qsl[r], A.T) >= 2) {   // verify_residual has it
    d = A.verdicts[r];
    if (tid < 16) L.pow16[tid] = POW16[tid];
    __syncthreads();
  } else {
    d = decide(A, r, L);
  }
  int64_t pick = d.at;
  if (d.sample) {                                      // uniform, like all of the branches below
    const int64_t skip = d.full || A.q ? -1 : A.tokens[d.t + 1];
    int mode = d.full ? 0 : A.q ? 2 : 1;
    double g[VE / 8][8];
    // first the piece that lacks a token, whose sum is taken anew and not by subtraction; then the piece picked
    const int64_t sp = mode == 1 && skip >= 0 && skip < A.V ? skip / (VT * VE) : -1;
    int64_t look = sp;
    double own = 0.0;
    for (bool picked = false;;) {
      if (look >= 0) {
        own = piece_sum<VE>(seg, [&](int k, double (&gk)[8]) {
          group_weights<VE>(A, d, L.pow16, look, k, mode, skip, gk);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[k][e] = gk[e];
        });
      }
      if (picked) break;
      if (w == 0) {                                    // the pieces' running sum passes u W in piece `piece`
        auto weight = [&](int64_t p) -> double {
          if (p >= A.pieces) return 0.0;
          if (mode == 2) return A.left[r * A.pieces + p];
          if (mode == 1 && p == sp) return own;
          const Stat a = A.st[d.t * A.pieces + p];
          return a.s * expo(a.m, Expo{(double)d.m, d.it}, L.pow16);
        };
        double W = 0.0;
        for (int64_t p0 = 0; p0 < A.pieces; p0 += 64) W += wave_sumd(weight(p0 + lane));
        const double gl = fmax((double)A.u_next[r] * W, 0.0);
        double c = 0.0, before = 0.0;
        int64_t at = -1, lastp = -1;
        double lastc = 0.0;
        for (int64_t p0 = 0; p0 < A.pieces && at < 0; p0 += 64) {
          const double x = weight(p0 + lane);
          double y = x;
#pragma unroll
          for (int o = 1; o < 64; o <<= 1) {
            const double z = __shfl_up(y, o, 64);
            if (lane >= o) y += z;
          }
          const uint64_t over = __ballot(x > 0.0 && c + y > gl), any = __ballot(x > 0.0);
          if (any) {
            const int k = 63 - __clzll(any);
            lastp = p0 + k;
            lastc = c + __shfl(y - x, k, 64);
          }
          if (over) {
            const int k = __ffsll((unsigned long long)over) - 1;
            at = p0 + k;
            before = c + __shfl(y - x, k, 64);
          }
          c += __shfl(y, 63, 64);
        }
        if (at < 0) { at = lastp; before = lastc; }    // u at 1 or past it: the last one with any weight
        if (lane == 0) { total = W > 0.0 ? fmax(gl - before, 0.0) : -1.0; piece = (int)at; where = -1; }
      }
      __syncthreads();
      if (total < 0.0 && mode != 0) {                  // nothing is left of p: p itself
        mode = 0;
        look = -1;
        __syncthreads();
        continue;
      }
      look = piece;
      picked = true;
      if (look < 0) break;
    }
    if (look >= 0) {
      const double gl = total;
      double c = 0.0;
      int hit = -1, lasts = -1;                        // the segment of 512 in which it passes; the last one with any weight
#pragma unroll
      for (int k = 0; k < VE / 2; ++k) {
        if (seg[k] > 0.0) {
          lasts = k;
          if (hit < 0 && c + seg[k] > gl) hit = k;
        }
        if (hit < 0) c += seg[k];
      }
      if (hit < 0) {
        hit = lasts;
        c = INFINITY;                                  // any weight: the last one
      }
      if (hit >= 0 && (hit & 3) == w) {
        double y[8];
#pragma unroll
        for (int k = 0; k < VE / 8; ++k)
          if (k == hit >> 2) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = g[k][e];
          }
        const double x = sum8(y);
        double pre = x;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const double z = __shfl_up(pre, o, 64);
          if (lane >= o) pre += z;
        }
        double run = c == INFINITY ? -INFINITY : c + (pre - x);
        int at = -1, lastw = -1;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          run += y[e];
          if (y[e] > 0.0) lastw = e;
          if (at < 0 && y[e] > 0.0 && run > gl) at = e;
        }
        const uint64_t over = __ballot(at >= 0), any = __ballot(lastw >= 0);
        const int from = over ? __ffsll((unsigned long long)over) - 1 : any ? 63 - __clzll(any) : -1;
        if (lane == from) where = 512 * hit + 8 * lane + (over ? at : lastw);
      }
      __syncthreads();
      if (where >= 0) pick = look * (VT * VE) + where;
    }
  }
  for (int64_t t = d.s0 + tid; t < d.s1; t += VT) A.out[t] = t < d.t ? A.tokens[t + 1] : t == d.t ? pick : -1;
  if (tid == 0) A.count[r] = (int32_t)(d.t - d.s0 + 1);
}

// Pieces of 2,048 values while all rows in them make up to 9,216 workgroups, else of 8,192, whose sums and lookups of a piece's
// row are fewer. All kernels, us in small / large pieces, 65,536 logits, drafts without a distribution: 4 rows of logits 11.3 / 18.3,
// 48 14.3 / 20.2, 128 20.0 / 24.2, 256 (8,192 workgroups) 30.2 / 34.1, 320 37.1 / 39.8, 448 46.2 / 46.6, 640 60.7 / 57.5, 1,280 106 / 91;
// with one: 4 13.4 / 20.2, 128 24.5 / 26.4, 256 37.9 / 39.4, 320 (10,240) 46.9 / 45.1, 640 77 / 67, 1,280 139 / 107.
int verify_ve(int64_t T, int64_t V) { return T * ((V + 8 * VT - 1) / (8 * VT)) <= 9216 ? 8 : 32; }
int64_t verify_pieces(int64_t T, int64_t V) { const int64_t n = VT * verify_ve(T, V); return (V + n - 1) / n; }

template <int VE>
int verify_launch(const VerifyArgs& A, hipStream_t s) {
  int rc;
  if (A.T > 0) {
    hipLaunchKernelGGL(verify_stats_kernel<VE>, dim3((unsigned)A.pieces, (unsigned)A.T), dim3(VT), 0, s, A);
    if ((rc = kv800::check_launch("verify_stats")) != KV800_OK) return rc;
    if (A.q) {
      hipLaunchKernelGGL(verify_residual_kernel<VE>, dim3((unsigned)A.pieces, (unsigned)A.R), dim3(VT), 0, s, A);
      if ((rc = kv800::check_launch("verify_residual")) != KV800_OK) return rc;
    }
  }
  hipLaunchKernelGGL(verify_pick_kernel<VE>, dim3((unsigned)A.R), dim3(VT), 0, s, A);
  return kv800::check_launch("verify_pick");
}

}  // namespace
}  // namespace lfm3

extern "C" {

int lfm3_hip_conv_chunk(const uint16_t* bcx, int64_t stride, const uint16_t* conv_w, const uint16_t* state,
                        const int64_t* qsl, int64_t R, int64_t T, int64_t H, uint16_t* out, uint16_t* taps, void* stream) {
  KV800_REQUIRE(R >= 1 && T >= 0 && H > 0 && H % 8 == 0 && stride >= 3 * H && stride % 8 == 0,
                "conv_chunk: needs R >= 1, H a positive multiple of 8 and a row stride >= 3H that is a multiple of 8");
  if (T == 0) return KV800_OK;
  KV800_REQUIRE(bcx && conv_w && state && qsl && out && taps, "conv_chunk: null pointer");
  KV800_REQUIRE(((uintptr_t)bcx | (uintptr_t)conv_w | (uintptr_t)state | (uintptr_t)out | (uintptr_t)taps) % 16 == 0,
                "conv_chunk: pointers must be 16-byte aligned");
  const int64_t ny = (H / 8 + 255) / 256;
  KV800_REQUIRE(T <= 0x7FFFFFFF && ny <= 65535, "conv_chunk: too large");
  const hipStream_t s = (hipStream_t)stream;
  // Tokens per workgroup, by the workgroups that one each would make: few, so that every CU has one and a token's taps are
  // not formed again by its successors' workgroups more often than that costs; 16 where 8 make more than three rounds of the
  // CUs and less than six.
  // H = 2048, us with 1 / 2 / 4 / 8 / 16 / 32, the commit's 4.6 among them: T = 256: 9.0 9.2 10.5 11.3 17 26; 512: 10.3 9.7 10.8
  // 12.4 16 27; 1,024: 13.9 11.3 11.5 13.1 17 26; 1,280: 15.8 13.3 13.5 14.0 18 33; 4,096: 31 26 25.0 21.9 23.6 35; 6,144: 41 34 31 29.7
  // 27.9 36; 7,168: 46 38 36 37.3 30.6 37; 10,240: 62 50 46 45.8 41.7 42; 12,288: 72 58 54 52.3 48.1 46; 13,312: 83 71 61 61.9 64.1 61;
  // 16,384: 123 101 82 72.0 77.6 70; 32,768: 252 194 156 147 149 158.
  const int64_t n = T * ny;
  const auto go = [&](auto tt) {
    constexpr int TT = decltype(tt)::value;
    hipLaunchKernelGGL(lfm3::conv_chunk_kernel<TT>, dim3((unsigned)((T + 32 * TT - 1) / (32 * TT) * 32), (unsigned)ny), dim3(256), 0, s, bcx, stride,
                       conv_w, state, qsl, R, T, H, out, taps);
  };
  if (n <= 256) go(std::integral_constant<int, 1>());
  else if (n <= 512) go(std::integral_constant<int, 2>());
  else if (n <= 1024) go(std::integral_constant<int, 4>());
  else if (n > 6144 && n <= 12288) go(std::integral_constant<int, 16>());
  else go(std::integral_constant<int, 8>());
  return kv800::check_launch("conv_chunk");
}

int lfm3_hip_conv_commit(uint16_t* state, const uint16_t* taps, const int64_t* qsl, const int32_t* kept, int64_t R,
                         int64_t T, int64_t H, void* stream) {
  KV800_REQUIRE(R >= 1 && T >= 0 && H > 0 && H % 8 == 0, "conv_commit: needs R >= 1 and H a positive multiple of 8");
  if (T == 0) return KV800_OK;
  KV800_REQUIRE(state && taps && qsl && kept, "conv_commit: null pointer");
  KV800_REQUIRE(((uintptr_t)state | (uintptr_t)taps) % 16 == 0, "conv_commit: state and taps must be 16-byte aligned");
  const int64_t n = R * (H / 8), nb = (n + 255) / 256;
  KV800_REQUIRE(nb <= 0x7FFFFFFF, "conv_commit: too large");
  hipLaunchKernelGGL(lfm3::conv_commit_kernel, dim3((unsigned)nb), dim3(256), 0, (hipStream_t)stream, state, taps, qsl, kept,
                     R, T, H);
  return kv800::check_launch("conv_commit");
}

int64_t lfm3_hip_verify_workspace(int64_t R, int64_t T, int64_t V) {
  if (R <= 0 || T <= 0 || V <= 0) return 0;
  return lfm3::verify_pieces(T, V) * (T * (int64_t)sizeof(lfm3::Stat) + R * (int64_t)sizeof(double)) + R * (int64_t)sizeof(lfm3::Verdict);
}

int lfm3_hip_verify_drafts(const uint16_t* logits, int64_t ld, const int64_t* tokens, const int64_t* qsl, const float* temp,
                           const float* u, const float* u_next, const float* draft_probs, int64_t ldq, int64_t R,
                           int64_t T, int64_t V, int64_t* out, int32_t* count, void* ws, int64_t ws_bytes, void* stream) {
  KV800_REQUIRE(R >= 1 && T >= 0 && V > 0 && V < (1LL << 31) && ld >= V && (!draft_probs || ldq >= V),
                "verify_drafts: needs R >= 1, 0 < V < 2^31 and row strides of at least V");
  KV800_REQUIRE(R <= 65535 && T <= 65535, "verify_drafts: at most 65,535 rows and tokens a call");
  KV800_REQUIRE(qsl && count && (T == 0 || (logits && tokens && temp && u && u_next && out)), "verify_drafts: null pointer");
  KV800_REQUIRE(ws_bytes >= lfm3_hip_verify_workspace(R, T, V) && (T == 0 || (ws && (uintptr_t)ws % 16 == 0)),
                "verify_drafts: the workspace is too small or not 16-byte aligned");
  lfm3::VerifyArgs A = {logits, ld, tokens, qsl, temp, u, u_next, draft_probs, ldq, R, T, V, lfm3::verify_pieces(T, V),
                        reinterpret_cast<lfm3::Stat*>(ws), nullptr, nullptr, out, count};
  A.left = reinterpret_cast<double*>(A.st + T * A.pieces);
  A.verdicts = reinterpret_cast<lfm3::Verdict*>(A.left + R * A.pieces);
  const hipStream_t s = (hipStream_t)stream;
  return lfm3::verify_ve(T, V) == 8 ? lfm3::verify_launch<8>(A, s) : lfm3::verify_launch<32>(A, s);
}

}  // extern "C"
