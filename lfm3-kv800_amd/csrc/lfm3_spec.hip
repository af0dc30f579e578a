// lfm3_spec.hip -- model-side operators of a step whose rows bring several new tokens each (include/lfm3_spec.h), gfx950.
//
//   conv_chunk_kernel     the gated short conv over each row's new tokens, from the row's 6-tap state
//   conv_commit_kernel    that state moved on over the tokens that were kept
//   verify_stats_kernel   per piece of a logits row: largest value, its index, sum of exponentials
//   verify_pick_kernel    per row of the batch: which drafts are kept, and the token behind them
#include "kv800_common.h"
#include "../../include/kv800_hip.h"
#include "../../include/lfm3_spec.h"

namespace lfm3 {
namespace {

using kv800::bf2f;
using kv800::f2bf;

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

// The row that holds token t: the last r < R with qsl[r] <= t (qsl[0] = 0). 64-way search by the whole wave, the same
// result in every lane: R of a few hundred takes two dependent loads.
__device__ __forceinline__ int64_t row_of(const int64_t* __restrict__ qsl, int64_t R, int64_t t) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, hi = R;                              // qsl[lo] <= t; qsl[hi] > t, or hi = R
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 63) / 64, i = lo + lane * step;
    const int c = __popcll(__ballot(i < hi && qsl[i < hi ? i : lo] <= t));   // lane 0 probes lo
    lo += (c > 0 ? c - 1 : 0) * step;
    hi = min(hi, lo + step);
  }
  return lo;
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
  const int64_t t0 = (int64_t)blockIdx.x * TT, c0 = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8;
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
  float w[7][8];
  {
    const uint4* s = reinterpret_cast<const uint4*>(cw + c0 * 7);                  // 8 channels x 7 taps
    uint32_t x[28];
#pragma unroll
    for (int i = 0; i < 7; ++i) { const uint4 v = s[i]; x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w; }
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int k = 0; k < 7; ++k) w[k][c] = ((c * 7 + k) & 1) ? kv800::bf2f_hi(x[(c * 7 + k) / 2]) : kv800::bf2f_lo(x[(c * 7 + k) / 2]);
  }
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
        for (int k = 0; k < 6; ++k) y[c] = fmaf(win[k][c], w[k][c], y[c]);
        y[c] = fmaf(f[c], w[6][c], y[c]) * g[c];
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
// A logits row is cut into pieces of VP; a piece gives its largest value m, its index and s = sum exp((x - m) / temp) in
// 64 bits. Why 64: the token behind a rejection is found by the running sum passing u W, and among 65,536 tokens the sums
// of neighbours lie 1e-5 apart where 32-bit exponentials are 1e-7 off; and the choice has to be the same whatever
// way the row is cut.
constexpr int VT = 256, VE = 32, VP = VT * VE;         // threads, values a thread, values a piece
struct Stat { double s; float m; int32_t at; };        // 16 bytes

// (a, ia) ranks before (b, ib): larger first, the smaller index among equals, the first NaN before every number
__device__ __forceinline__ bool ranks_before(float a, int ia, float b, int ib) {
  const bool na = a != a, nb = b != b;
  if (na || nb) return na && (!nb || ia < ib);
  return a > b || (a == b && ia < ib);
}
// whether a row with largest logit m is sampled: a positive finite temperature and a finite m; else its choice is m's index
__device__ __forceinline__ bool sampled(float tp, float m) { return tp > 0.f && tp < INFINITY && m - m == 0.f; }
__device__ __forceinline__ double wave_sumd(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ double expo(float x, float m, double it) { return exp(((double)x - (double)m) * it); }

__global__ void __launch_bounds__(VT)
verify_stats_kernel(const uint16_t* __restrict__ logits, int64_t ld, const int64_t* __restrict__ qsl,
                    const float* __restrict__ temp, int64_t R, int64_t T, int64_t V, int64_t pieces, Stat* __restrict__ st) {
  __shared__ float rm[4];
  __shared__ int ri[4];
  __shared__ double rs[4];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int64_t t = blockIdx.y, v0 = (int64_t)blockIdx.x * VP;
  if (t >= min(qsl[R], T)) return;                     // uniform
  const float tp = temp[row_of(qsl, R, t)];
  const int n = (int)min((int64_t)VP, V - v0);
  const uint16_t* row = logits + t * ld + v0;
  float x[VE];
  float bm = -INFINITY;
  int bi = 0x7FFFFFFF;
#pragma unroll
  for (int k = 0; k < VE; ++k) {
    const int i = tid + VT * k;
    x[k] = i < n ? bf2f(row[i]) : -INFINITY;
    if (i < n && ranks_before(x[k], i, bm, bi)) { bm = x[k]; bi = i; }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(bm, o, 64);
    const int i2 = __shfl_xor(bi, o, 64);
    if (ranks_before(m2, i2, bm, bi)) { bm = m2; bi = i2; }
  }
  if (lane == 0) { rm[w] = bm; ri[w] = bi; }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (ranks_before(rm[k], ri[k], bm, bi)) { bm = rm[k]; bi = ri[k]; }
  double s = 0.0;
  if (sampled(tp, bm)) {
    const double it = 1.0 / (double)tp;
#pragma unroll
    for (int k = 0; k < VE; ++k)
      if (tid + VT * k < n) s += expo(x[k], bm, it);
  }
  s = wave_sumd(s);
  if (lane == 0) rs[w] = s;
  __syncthreads();
  if (tid == 0) st[t * pieces + blockIdx.x] = Stat{(rs[0] + rs[1]) + (rs[2] + rs[3]), bm, (int32_t)(v0 + bi)};
}

// One workgroup of 1,024 threads per row of the batch.
constexpr int PT = 1024, PW = PT / 64;
__global__ void __launch_bounds__(PT)
verify_pick_kernel(const uint16_t* __restrict__ logits, int64_t ld, const int64_t* __restrict__ tokens,
                   const int64_t* __restrict__ qsl, const float* __restrict__ temp, const float* __restrict__ u,
                   const float* __restrict__ u_next, const float* __restrict__ q, int64_t ldq, int64_t R, int64_t T,
                   int64_t V, int64_t pieces, const Stat* __restrict__ st, int64_t* __restrict__ out,
                   int32_t* __restrict__ count) {
  __shared__ long long stop;                           // the first logits row that ends the batch row
  __shared__ double seg[PW], top_s;
  __shared__ float top_m;
  __shared__ int top_at, found, part;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int64_t r = blockIdx.x;
  const int64_t s0 = min(qsl[r], T), s1 = min(qsl[r + 1], T);
  if (r == R - 1)
    for (int64_t t = s1 + tid; t < T; t += PT) out[t] = -1;   // the padding
  if (s1 <= s0) {
    if (tid == 0) count[r] = 0;
    return;
  }
  const float tp = temp[r];
  const double it = 1.0 / (double)tp;
  if (tid == 0) { stop = s1 - 1; found = -1; }
  __syncthreads();
  // a logits row's pieces combined: largest value, its index and the sum about it, the same in every lane
  auto combine = [&](int64_t t, float& M, int& at, double& S) {
    M = -INFINITY;
    at = 0x7FFFFFFF;
    for (int64_t p = lane; p < pieces; p += 64) {
      const Stat a = st[t * pieces + p];
      if (ranks_before(a.m, a.at, M, at)) { M = a.m; at = a.at; }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float m2 = __shfl_xor(M, o, 64);
      const int i2 = __shfl_xor(at, o, 64);
      if (ranks_before(m2, i2, M, at)) { M = m2; at = i2; }
    }
    S = 0.0;
    if (sampled(tp, M))
      for (int64_t p = lane; p < pieces; p += 64) {
        const Stat a = st[t * pieces + p];
        if (a.m > -INFINITY) S += a.s * expo(a.m, M, it);
      }
    S = wave_sumd(S);
  };
  for (int64_t t = s0 + w; t < s1 - 1; t += PW) {
    float M;
    int at;
    double S;
    combine(t, M, at, S);
    const int64_t d = tokens[t + 1];
    bool keep;
    if (!sampled(tp, M)) keep = d == at;
    else {
      keep = d >= 0 && d < V;
      if (keep) {
        const double pd = expo(bf2f(logits[t * ld + d]), M, it) / S;
        keep = (double)u[t] * (q ? (double)q[t * ldq + d] : 1.0) < pd;
      }
    }
    if (!keep) {
      if (lane == 0) atomicMin((long long*)&stop, (long long)t);
      break;
    }
  }
  __syncthreads();
  const int64_t tt = stop;
  if (w == 0) {
    float M;
    int at;
    double S;
    combine(tt, M, at, S);
    if (lane == 0) { top_m = M; top_at = at; top_s = S; }
  }
  __syncthreads();
  const float M = top_m;
  int64_t pick = top_at;
  if (sampled(tp, M)) {                                // uniform over the workgroup
    const double S = top_s;
    const bool full = tt == s1 - 1;
    const int64_t d = full ? -1 : tokens[tt + 1];
    const uint16_t* row = logits + tt * ld;
    const float* qr = (q && !full) ? q + tt * ldq : nullptr;
    // mode 0: the row's distribution; 1: what p has over q; either way the weight of token i
    auto weight = [&](int64_t i, bool plain) -> double {
      const double p = expo(bf2f(row[i]), M, it) / S;
      if (plain || full) return p;
      if (!qr) return i == d ? 0.0 : p;
      const double x = p - (double)qr[i];
      return x > 0.0 ? x : 0.0;
    };
    for (int plain = 0; plain < 2; ++plain) {
      // wave w sums its 1/16 of the row
      const int64_t per = (V + PW - 1) / PW, a = min(V, w * per), b = min(V, a + per);
      double s = 0.0;
      for (int64_t i = a + lane; i < b; i += 64) s += weight(i, plain);
      s = wave_sumd(s);
      if (lane == 0) seg[w] = s;
      __syncthreads();
      double W = 0.0;
      for (int k = 0; k < PW; ++k) W += seg[k];
      if (W > 0.0 || plain) {
        const double goal = fmax((double)u_next[r] * W, 0.0);
        if (tid == 0) {                                // the wave in whose part the sum passes the goal
          double c = 0.0;
          int k = 0, lastk = 0;
          for (; k < PW; ++k) {
            if (seg[k] > 0.0) lastk = k;
            if (c + seg[k] > goal) break;
            c += seg[k];
          }
          part = k < PW ? k : lastk;
        }
        __syncthreads();
        if (w == part) {
          double c = 0.0;
          for (int k = 0; k < w; ++k) c += seg[k];
          int64_t at = -1, some = -1;                  // the token found; the last one with any weight
          for (int64_t i0 = a; i0 < b && at < 0; i0 += 64) {
            const int64_t i = i0 + lane;
            const double x = i < b ? weight(i, plain) : 0.0;
            double y = x;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
              const double z = __shfl_up(y, o, 64);
              if (lane >= o) y += z;
            }
            const uint64_t over = __ballot(i < b && c + y > goal), any = __ballot(x > 0.0);
            if (any) some = i0 + 63 - __clzll(any);
            if (over) at = i0 + __ffsll((unsigned long long)over) - 1;
            c += __shfl(y, 63, 64);
          }
          if (lane == 0) found = (int)(at >= 0 ? at : some);
        }
        __syncthreads();
        break;
      }
      __syncthreads();
    }
    if (found >= 0) pick = found;
  }
  for (int64_t t = s0 + tid; t < s1; t += PT) out[t] = t < tt ? tokens[t + 1] : t == tt ? pick : -1;
  if (tid == 0) count[r] = (int32_t)(tt - s0 + 1);
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
  if (T * ny <= 4096)
    hipLaunchKernelGGL(lfm3::conv_chunk_kernel<1>, dim3((unsigned)T, (unsigned)ny), dim3(256), 0, s, bcx, stride, conv_w, state,
                       qsl, R, T, H, out, taps);
  else
    hipLaunchKernelGGL(lfm3::conv_chunk_kernel<16>, dim3((unsigned)((T + 15) / 16), (unsigned)ny), dim3(256), 0, s, bcx, stride,
                       conv_w, state, qsl, R, T, H, out, taps);
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

int64_t lfm3_hip_verify_workspace(int64_t T, int64_t V) {
  if (T <= 0 || V <= 0) return 0;
  return T * ((V + lfm3::VP - 1) / lfm3::VP) * (int64_t)sizeof(lfm3::Stat);
}

int lfm3_hip_verify_drafts(const uint16_t* logits, int64_t ld, const int64_t* tokens, const int64_t* qsl, const float* temp,
                           const float* u, const float* u_next, const float* draft_probs, int64_t ldq, int64_t R,
                           int64_t T, int64_t V, int64_t* out, int32_t* count, void* ws, int64_t ws_bytes, void* stream) {
  KV800_REQUIRE(R >= 1 && T >= 0 && V > 0 && V < (1LL << 31) && ld >= V && (!draft_probs || ldq >= V),
                "verify_drafts: needs R >= 1, 0 < V < 2^31 and row strides of at least V");
  KV800_REQUIRE(R <= 0x7FFFFFFF && T <= 65535, "verify_drafts: at most 65,535 tokens a call");
  KV800_REQUIRE(qsl && count && (T == 0 || (logits && tokens && temp && u && u_next && out)), "verify_drafts: null pointer");
  KV800_REQUIRE(ws_bytes >= lfm3_hip_verify_workspace(T, V) && (T == 0 || (ws && (uintptr_t)ws % 16 == 0)),
                "verify_drafts: the workspace is too small or not 16-byte aligned");
  const int64_t pieces = (V + lfm3::VP - 1) / lfm3::VP;
  const hipStream_t s = (hipStream_t)stream;
  lfm3::Stat* st = reinterpret_cast<lfm3::Stat*>(ws);
  if (T > 0) {
    hipLaunchKernelGGL(lfm3::verify_stats_kernel, dim3((unsigned)pieces, (unsigned)T), dim3(lfm3::VT), 0, s, logits, ld, qsl, temp,
                       R, T, V, pieces, st);
    const int rc = kv800::check_launch("verify_stats");
    if (rc != KV800_OK) return rc;
  }
  hipLaunchKernelGGL(lfm3::verify_pick_kernel, dim3((unsigned)R), dim3(lfm3::PT), 0, s, logits, ld, tokens, qsl, temp, u, u_next,
                     draft_probs, ldq, R, T, V, pieces, st, out, count);
  return kv800::check_launch("verify_pick");
}

}  // extern "C"
