// kv8_cache.hip -- writing and reading back the paged 8-bit cache (include/kv8_hip.h), gfx950.
//
//   append_kernel      a step's keys (rotated on the way) and values into their blocks
//   dequantize_kernel  the values that the blocks stand for
#include "kv8_common.h"

namespace kv8 {
namespace {

using kv800::bf2f_hi;
using kv800::bf2f_lo;

// WHOLE: one workgroup per (block that a row's new tokens touch, head, keys or values), wave g its tokens 16 g .. 16 g + 15; else one
// wave, which goes through the groups of 16 that hold new tokens, once for the maximum and once for the codes. Row r's blocks
// have the numbers from (qsl[r] + 126 r) / 64 on: c tokens touch at most (c + 126) / 64 blocks, so no list is needed, and few
// workgroups find nothing. D / 16 lanes take a token, 8 channels of each half a lane: f and f + D / 2, the pairs that are rotated
// together. Bound: memory for long prompts (8 x 8,191 tokens 57 us; one wave a block with all its tokens in registers 66), else a chain
// of five loads and the number of waves (256 rows of up to 5 tokens 13 us; a workgroup a block 16.8).
template <int D, bool WHOLE>
__global__ void __launch_bounds__(256)
append_kernel(Cache C, const uint16_t* __restrict__ k, int64_t k_ts, int64_t k_hs, const uint16_t* __restrict__ v, int64_t v_ts,
              int64_t v_hs, const int32_t* __restrict__ bt, int64_t bt_stride, int64_t bt_cols, const int64_t* __restrict__ lens,
              const int64_t* __restrict__ qsl, int64_t R, int64_t T, const uint16_t* __restrict__ cos_t,
              const uint16_t* __restrict__ sin_t, int64_t rope_rows, int F, float rows_per_block) {
  constexpr int LT = D / 16, TP = 64 / LT, NP = 16 / TP;   // lanes a token, tokens a pass, passes of a wave
  __shared__ __align__(16) uint8_t turn[4][18 * D];        // a group's new values by channel: 16 bytes each, 16 more every 8 channels
  __shared__ float tops[4];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int hk = WHOLE ? blockIdx.y : blockIdx.y * 4 + wv, h = hk >> 1, kind = hk & 1;
  if (!WHOLE && h >= C.heads) return;
  const int64_t u = blockIdx.x;
  const int64_t r = row_near(R, (int64_t)((float)u * rows_per_block), [&](int64_t i) { return (qsl[i] + 126 * i) / BLK <= u; });
  const int64_t q0 = qsl[r], n = lens[r], p0 = n - (qsl[r + 1] - q0);   // the first new token's position
  const int64_t b = max(p0, (int64_t)0) / BLK + (u - (q0 + 126 * r) / BLK);
  if (b * BLK >= n || b < 0 || b > INT32_MAX || q0 < 0) return;         // uniform, as every return before the last barrier
  const int col = (int)((uint32_t)b / (uint32_t)C.blocks);
  if (col >= bt_cols) return;
  const int first = (int)(max(p0, b * BLK) - b * BLK);                  // new tokens of the block: [first, last)
  const int last = (int)max(min(min((int64_t)BLK, n - b * BLK), p0 - q0 + T - b * BLK), (int64_t)0);
  if (first >= last) return;
  const int64_t page = bt[r * bt_stride + col];

  // token of a pass and channels of the lane: the pairs of lanes that exchange keys' codes lie side by side, so do the fours that
  // exchange values' codes
  const int tl = kind ? lane % TP : lane / LT, c = kind ? lane / TP : lane % LT;
  const int64_t ts = kind ? v_ts : k_ts;
  const uint16_t* src = (kind ? v + h * v_hs : k + h * k_hs) + (q0 + b * BLK - p0) * ts + c * 8;
  const bool turns = !kind && c * 8 < F;
  uint4 w[NP][2], cw[NP], sw[NP];
  auto load = [&](int g) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int t = 16 * g + i * TP + tl;
      w[i][0] = w[i][1] = cw[i] = sw[i] = make_uint4(0, 0, 0, 0);
      if (t >= first && t < last) {
        w[i][0] = *reinterpret_cast<const uint4*>(src + t * ts);
        w[i][1] = *reinterpret_cast<const uint4*>(src + t * ts + D / 2);
        if (turns) {
          const int64_t at = min(max(b * BLK + t, (int64_t)0), rope_rows - 1) * F + c * 8;
          cw[i] = *reinterpret_cast<const uint4*>(cos_t + at);
          sw[i] = *reinterpret_cast<const uint4*>(sin_t + at);
        }
      }
    }
  };
  float x[NP][2][8], top = 0.f;
  auto channels = [&]() {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const uint32_t a[4] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w}, d[4] = {w[i][1].x, w[i][1].y, w[i][1].z, w[i][1].w};
      const uint32_t cs[4] = {cw[i].x, cw[i].y, cw[i].z, cw[i].w}, ss[4] = {sw[i].x, sw[i].y, sw[i].z, sw[i].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f0 = e & 1 ? bf2f_hi(a[e >> 1]) : bf2f_lo(a[e >> 1]), f1 = e & 1 ? bf2f_hi(d[e >> 1]) : bf2f_lo(d[e >> 1]);
        const float co = e & 1 ? bf2f_hi(cs[e >> 1]) : bf2f_lo(cs[e >> 1]), si = e & 1 ? bf2f_hi(ss[e >> 1]) : bf2f_lo(ss[e >> 1]);
        // products of two bf16 are exact in fp32, so a rotated channel is rounded once, by the sum (fused or not)
        x[i][0][e] = turns ? f0 * co - f1 * si : f0;
        x[i][1][e] = turns ? f1 * co + f0 * si : f1;
        top = fmaxf(top, fmaxf(finite_abs(x[i][0][e]), finite_abs(x[i][1][e])));
      }
    }
  };
  const int g0 = WHOLE ? wv : first >> 4, g1 = WHOLE ? wv : (last - 1) >> 4;   // groups with new tokens (WHOLE: the wave's)
  load(g0);
  if (page < 0 || page >= C.pages) return;
  const int ub = (int)b - col * C.blocks;
  uint8_t* blk = block_of<D>(C, page, h, ub) + kind * (BLK * D);
  uint8_t* ex = exps_of(C, page, h, ub) + kind;
  const int old = first > 0 ? held_exponent(*ex) : E_MIN;               // a block's first token starts it anew
  channels();
  for (int g = g0 + 1; g <= g1; ++g) {
    load(g);
    channels();
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (WHOLE) {
    if (lane == 0) tops[wv] = top;
    __syncthreads();                                                    // also: every thread has read the old exponent
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  }
  const int ne = max(exponent_for(top), old);
  const bool grown = first > 0 && ne > old;
  const float inv = pow2(-ne), down = pow2(max(old - ne, -40));         // any code times 2^-40 rounds to 0
  if (WHOLE ? threadIdx.x == 0 : lane == 0) *ex = (uint8_t)(ne + 127);
  // no barriers from here on: a wave goes through its groups with new tokens, and those with codes to round again
  for (int g = WHOLE ? wv : grown ? 0 : g0; g <= g1; ++g) {
    const int t0 = 16 * g;
    if (WHOLE && !(t0 < last && t0 + 16 > first) && !(grown && t0 < first)) return;
    if (!WHOLE && g0 != g1) {
      load(g);
      channels();
    }
    uint8_t* vb = turn[wv];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int t = t0 + i * TP + tl;
      const bool fresh = t >= first && t < last, again = grown && t < first;
      uint32_t code[2][2];
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          code[half][e] = enc4(x[i][half][4 * e] * inv, x[i][half][4 * e + 1] * inv, x[i][half][4 * e + 2] * inv, x[i][half][4 * e + 3] * inv);
      if (kind) {      // 4 tokens of a channel lie in four lanes: lane i of them takes channel i of each four
        const uint32_t sel = 0x0400u + 0x0101u * (lane & 3);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int w0 = __builtin_amdgcn_mov_dpp((int)code[half][e], 0x00, 0xF, 0xF, true), w1 = __builtin_amdgcn_mov_dpp((int)code[half][e], 0x55, 0xF, 0xF, true);
            const int w2 = __builtin_amdgcn_mov_dpp((int)code[half][e], 0xAA, 0xF, 0xF, true), w3 = __builtin_amdgcn_mov_dpp((int)code[half][e], 0xFF, 0xF, 0xF, true);
            const uint32_t lo = __builtin_amdgcn_perm((uint32_t)w1, (uint32_t)w0, sel), hi = __builtin_amdgcn_perm((uint32_t)w3, (uint32_t)w2, sel);
            const int d = half * (D / 2) + c * 8 + e * 4 + (lane & 3);
            *reinterpret_cast<uint32_t*>(vb + (d + (d >> 3)) * 16 + ((t - t0) & 12)) = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
          }
        continue;
      }
      // 16 channels of a slot lie in two lanes: the even one takes those of the lower half, the odd one of the upper
      const bool odd = c & 1;
      const int s0 = __builtin_amdgcn_mov_dpp((int)(odd ? code[0][0] : code[1][0]), 0xB1, 0xF, 0xF, true);   // of lane ^ 1
      const int s1 = __builtin_amdgcn_mov_dpp((int)(odd ? code[0][1] : code[1][1]), 0xB1, 0xF, 0xF, true);
      uint4 y = odd ? make_uint4((uint32_t)s0, (uint32_t)s1, code[1][0], code[1][1]) : make_uint4(code[0][0], code[0][1], (uint32_t)s0, (uint32_t)s1);
      uint4* dst = reinterpret_cast<uint4*>(blk + (((odd ? D / 32 : 0) + (c >> 1)) * BLK + slot_of(t)) * 16);
      if (again) {
        const uint4 o = *dst;
        y = make_uint4(down4(o.x, down), down4(o.y, down), down4(o.z, down), down4(o.w, down));
      }
      if (fresh || again) *dst = y;
    }
    if (!kind) continue;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const bool mixed = t0 < first || t0 + 16 > last;
#pragma unroll
    for (int p = 0; p < D / 64; ++p) {                                  // piece: the group's tokens of one channel
      const int d = p * 64 + lane;
      uint4* dst = reinterpret_cast<uint4*>(blk + (g * D + d) * 16);
      const uint4 y = *reinterpret_cast<const uint4*>(vb + (d + (d >> 3)) * 16);
      uint32_t out[4] = {y.x, y.y, y.z, y.w};
      if (mixed) {
        const uint4 o4 = *dst;
        const uint32_t o[4] = {o4.x, o4.y, o4.z, o4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // bytes of tokens [first, last) are new; behind them the codes stay, before them they are as they were or rounded again
          const int lo = min(max(first - t0 - 4 * i, 0), 4), hi = min(max(last - t0 - 4 * i, 0), 4);
          const uint32_t below = (uint32_t)((1ull << (8 * lo)) - 1), upto = (uint32_t)((1ull << (8 * hi)) - 1);
          const uint32_t was = grown ? down4(o[i], down) : o[i];
          out[i] = (out[i] & upto & ~below) | (was & below) | (o[i] & ~(upto | below));
        }
      }
      *dst = make_uint4(out[0], out[1], out[2], out[3]);
    }
    if (!WHOLE) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the next group's values come behind these reads
  }
}

// One workgroup per (block, head, page); both directions of the layouts in 16-byte pieces, the values turned through LDS.
template <int D>
__global__ void __launch_bounds__(256)
dequantize_kernel(Cache C, uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
  constexpr int ROW = D + 4;                       // bytes of a token in LDS (rows on different banks)
  __shared__ __align__(16) uint8_t vb[BLK * ROW];
  const int tid = threadIdx.x, u = blockIdx.x % C.blocks, h = blockIdx.x / C.blocks;
  const int64_t page = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (page >= C.pages) return;                     // uniform
  const uint8_t* kb = block_of<D>(C, page, h, u);
  const uint8_t* ex = exps_of(C, page, h, u);
  const float ks = pow2(held_exponent(ex[0])), vs = pow2(held_exponent(ex[1]));
  const int64_t row0 = ((page * C.heads + h) * C.blocks + u) * BLK;
  auto put = [](uint16_t* dst, const uint32_t (&w)[4], float s) {       // 16 codes -> 16 bf16
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[4];
      dec4(w[i], f);
      o[2 * i] = kv800::f2bf(f[0] * s) | (kv800::f2bf(f[1] * s) << 16);
      o[2 * i + 1] = kv800::f2bf(f[2] * s) | (kv800::f2bf(f[3] * s) << 16);
    }
    reinterpret_cast<uint4*>(dst)[0] = make_uint4(o[0], o[1], o[2], o[3]);
    reinterpret_cast<uint4*>(dst)[1] = make_uint4(o[4], o[5], o[6], o[7]);
  };
  for (int p = tid; p < 4 * D; p += 256) {         // piece: 16 tokens of channel p % D
    const uint4 w = *reinterpret_cast<const uint4*>(kb + BLK * D + p * 16);
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
    const int t0 = p / D * 16, d = p % D;
#pragma unroll
    for (int j = 0; j < 16; ++j) vb[(t0 + j) * ROW + d] = (uint8_t)(a[j >> 2] >> (8 * (j & 3)));
  }
  for (int p = tid; p < BLK * D / 16; p += 256) {  // piece: 16 channels of token t
    const int t = p / (D / 16), dg = p % (D / 16);
    const uint4 w = *reinterpret_cast<const uint4*>(kb + (dg * BLK + slot_of(t)) * 16);
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
    put(k + (row0 + t) * D + dg * 16, a, ks);
  }
  __syncthreads();
  for (int p = tid; p < BLK * D / 16; p += 256) {
    const int t = p / (D / 16), dg = p % (D / 16);
    const uint32_t* s = reinterpret_cast<const uint32_t*>(vb + t * ROW + dg * 16);
    const uint32_t a[4] = {s[0], s[1], s[2], s[3]};
    put(v + (row0 + t) * D + dg * 16, a, vs);
  }
}

}  // namespace
}  // namespace kv8

extern "C" {

int kv8_hip_append(const kv8_cache_t* cache, const uint16_t* k, int64_t k_ts, int64_t k_hs, const uint16_t* v, int64_t v_ts,
                   int64_t v_hs, const int32_t* bt, int64_t bt_stride, int64_t bt_cols, const int64_t* lens,
                   const int64_t* qsl, int64_t R, int64_t T, const uint16_t* cos_t, const uint16_t* sin_t,
                   int64_t rope_rows, int64_t freqs, void* stream) {
  KV800_REQUIRE(kv8::valid(cache), "kv8_append: bad cache descriptor");
  KV800_REQUIRE(R >= 0 && T >= 0 && bt_cols >= 0 && bt_stride >= 0, "kv8_append: negative size");
  if (R == 0 || T == 0 || bt_cols == 0) return KV800_OK;
  KV800_REQUIRE(k && v && bt && lens && qsl, "kv8_append: null pointer");
  KV800_REQUIRE(k_ts % 8 == 0 && k_hs % 8 == 0 && v_ts % 8 == 0 && v_hs % 8 == 0 && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0,
                "kv8_append: k and v need 16-byte aligned rows (strides multiples of 8)");
  KV800_REQUIRE(R < (1 << 30) && T < (1 << 30) && T + 126 * R < (1 << 30), "kv8_append: too many tokens or rows");   // 2^32 threads a launch
  KV800_REQUIRE((cos_t == nullptr) == (sin_t == nullptr), "kv8_append: cos_t and sin_t go together");
  KV800_REQUIRE(!cos_t || (freqs > 0 && freqs % 8 == 0 && freqs <= cache->dim / 2 && rope_rows > 0 && (uintptr_t)cos_t % 16 == 0 &&
                           (uintptr_t)sin_t % 16 == 0),
                "kv8_append: tables need freqs a multiple of 8 up to D / 2, rows, and 16-byte alignment");
  // 256 rows of 16 / 32 / 64 tokens, appended and read back: a wave a block 27.2 / 32.4 / 42.9 us, a workgroup 35.3 / 37.0 / 39.8
  const bool whole = T >= 48 * R;
  const dim3 grid((unsigned)((T + 126 * R) / kv8::BLK), (unsigned)(whole ? 2 * cache->kv_heads : (2 * cache->kv_heads + 3) / 4));
  const int F = cos_t ? (int)freqs : 0;
  const kv8::Cache C = kv8::device_form(cache);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, C, k, k_ts, k_hs, v, v_ts, v_hs, bt, bt_stride, bt_cols,
                       lens, qsl, R, T, cos_t, sin_t, rope_rows, F, 64.f / (126.f + (float)T / (float)R));
  };
  if (cache->dim == 128) whole ? go(kv8::append_kernel<128, true>) : go(kv8::append_kernel<128, false>);
  else whole ? go(kv8::append_kernel<64, true>) : go(kv8::append_kernel<64, false>);
  return kv800::check_launch("kv8_append");
}

int kv8_hip_dequantize(const kv8_cache_t* cache, uint16_t* k, uint16_t* v, void* stream) {
  KV800_REQUIRE(kv8::valid(cache), "kv8_dequantize: bad cache descriptor");
  KV800_REQUIRE(k && v && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, "kv8_dequantize: k and v must be 16-byte aligned");
  const int64_t py = cache->pages < 32768 ? cache->pages : 32768;
  const dim3 grid((unsigned)(cache->kv_heads * cache->blocks), (unsigned)py, (unsigned)((cache->pages + py - 1) / py));
  const kv8::Cache C = kv8::device_form(cache);
  if (cache->dim == 128) hipLaunchKernelGGL(kv8::dequantize_kernel<128>, grid, dim3(256), 0, (hipStream_t)stream, C, k, v);
  else hipLaunchKernelGGL(kv8::dequantize_kernel<64>, grid, dim3(256), 0, (hipStream_t)stream, C, k, v);
  return kv800::check_launch("kv8_dequantize");
}

}  // extern "C"
