// kv8_cache.hip -- writing and reading back the paged 8-bit cache (include/kv8_hip.h), gfx950.
//
//   append_kernel      a step's keys (rotated on the way) and values into their blocks
//   dequantize_kernel  the values that the blocks stand for
#include "kv8_common.h"

namespace kv8 {
namespace {

using kv800::bf2f_hi;
using kv800::bf2f_lo;

// One wave per (block that a row's new tokens touch, head, keys or values). Row r's blocks have the numbers from
// (qsl[r] + 126 r) / 64 on: c tokens touch at most (c + 126) / 64 blocks, so no list is needed, and few waves find nothing. A lane
// holds 2 x D / 8 channels of a token of each group of 16: channels f and f + D / 2, the pairs that are rotated together. The
// block's tokens stay in registers between the maximum and the encoding, so they are read once; groups without new tokens are passed over.
template <int D>
__global__ void __launch_bounds__(256)
append_kernel(Cache C, const uint16_t* __restrict__ k, int64_t k_ts, int64_t k_hs, const uint16_t* __restrict__ v, int64_t v_ts,
              int64_t v_hs, const int32_t* __restrict__ bt, int64_t bt_stride, int64_t bt_cols, const int64_t* __restrict__ lens,
              const int64_t* __restrict__ qsl, int64_t R, int64_t T, const uint16_t* __restrict__ cos_t,
              const uint16_t* __restrict__ sin_t, int64_t rope_rows, int F) {
  constexpr int E = D / 8;                         // channels of each half that a lane holds: 16 or 8
  __shared__ __align__(16) uint8_t turn[4][16 * D];   // a group's new values, transposed
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int hk = blockIdx.y * 4 + wv, h = hk >> 1, kind = hk & 1;
  if (h >= C.heads) return;                        // the whole wave, as every return: no workgroup barriers here
  const int64_t u = blockIdx.x;
  const int64_t r = kv800::last_at(R, [&](int64_t i) { return (qsl[i] + 126 * i) / BLK <= u; });
  const int64_t q0 = qsl[r], n = lens[r], p0 = n - (qsl[r + 1] - q0);   // the first new token's position
  const int64_t b = max(p0, (int64_t)0) / BLK + (u - (q0 + 126 * r) / BLK);
  if (b * BLK >= n || b < 0 || q0 < 0) return;
  const int64_t col = b / C.blocks;
  if (col >= bt_cols) return;
  const int64_t page = bt[r * bt_stride + col];
  if (page < 0 || page >= C.pages) return;
  const int first = (int)(max(p0, b * BLK) - b * BLK);                  // new tokens of the block: [first, last)
  const int last = (int)max(min(min((int64_t)BLK, n - b * BLK), p0 - q0 + T - b * BLK), (int64_t)0);
  if (first >= last) return;
  const int ub = (int)(b % C.blocks);
  uint8_t* blk = block_of<D>(C, page, h, ub) + kind * (BLK * D);
  uint8_t* ex = exps_of(C, page, h, ub) + kind;
  const int old = first > 0 ? held_exponent(*ex) : E_MIN;               // a block's first token starts it anew

  const int tl = lane >> 2, c = lane & 3;
  float x[4][2][E], top = 0.f;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int t = 16 * g + tl;
    if (16 * g >= last || 16 * g + 16 <= first) continue;
    const bool fresh = t >= first && t < last;
    const int64_t pos = b * BLK + t, row = q0 + (pos - p0);
    const uint16_t* src = kind ? v + row * v_ts + h * v_hs : k + row * k_ts + h * k_hs;
    const int64_t at = min(max(pos, (int64_t)0), rope_rows - 1) * F + c * E;
#pragma unroll
    for (int e = 0; e < E; e += 8) {
      uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)}, cw = w[0], sw = w[0];
      const bool turned = fresh && !kind && c * E + e < F;
      if (fresh) {
        w[0] = *reinterpret_cast<const uint4*>(src + c * E + e);
        w[1] = *reinterpret_cast<const uint4*>(src + D / 2 + c * E + e);
      }
      if (turned) {
        cw = *reinterpret_cast<const uint4*>(cos_t + at + e);
        sw = *reinterpret_cast<const uint4*>(sin_t + at + e);
      }
      const uint32_t a[4] = {w[0].x, w[0].y, w[0].z, w[0].w}, d[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
      const uint32_t cs[4] = {cw.x, cw.y, cw.z, cw.w}, ss[4] = {sw.x, sw.y, sw.z, sw.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f0 = i & 1 ? bf2f_hi(a[i >> 1]) : bf2f_lo(a[i >> 1]), f1 = i & 1 ? bf2f_hi(d[i >> 1]) : bf2f_lo(d[i >> 1]);
        const float co = i & 1 ? bf2f_hi(cs[i >> 1]) : bf2f_lo(cs[i >> 1]), si = i & 1 ? bf2f_hi(ss[i >> 1]) : bf2f_lo(ss[i >> 1]);
        // products of two bf16 are exact in fp32, so a rotated channel is rounded once, by the sum (fused or not)
        x[g][0][e + i] = turned ? f0 * co - f1 * si : f0;
        x[g][1][e + i] = turned ? f1 * co + f0 * si : f1;
        top = fmaxf(top, fmaxf(finite_abs(x[g][0][e + i]), finite_abs(x[g][1][e + i])));
      }
    }
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  const int ne = max(exponent_for(top), old);
  const bool grown = first > 0 && ne > old;
  const float inv = pow2(-ne), down = pow2(max(old - ne, -40));         // any code times 2^-40 rounds to 0
  if (lane == 0) *ex = (uint8_t)(ne + 127);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int t0 = 16 * g, t = t0 + tl;
    const bool news = t0 < last && t0 + 16 > first;
    if (!news && !(grown && t0 < first)) continue;
    const bool fresh = t >= first && t < last;
    uint32_t code[2][E / 4];
    if (news)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < E; e += 4)
          code[j][e / 4] = enc4(x[g][j][e] * inv, x[g][j][e + 1] * inv, x[g][j][e + 2] * inv, x[g][j][e + 3] * inv);
    if (!kind) {
      if (!fresh && !(grown && t < first)) continue;
      const int slot = slot_of(t);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int d = j * (D / 2) + c * E;
        uint32_t* dst = reinterpret_cast<uint32_t*>(blk + ((d >> 4) * BLK + slot) * 16 + (d & 15));
        if (!fresh)
#pragma unroll
          for (int e = 0; e < E / 4; ++e) code[j][e] = down4(dst[e], down);
        if (E == 16) *reinterpret_cast<uint4*>(dst) = make_uint4(code[j][0], code[j][1], code[j][E / 4 - 2], code[j][E / 4 - 1]);
        else *reinterpret_cast<uint2*>(dst) = make_uint2(code[j][0], code[j][1]);
      }
      continue;
    }
    uint8_t* vb = turn[wv];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");              // the group before has been read
    if (fresh)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) vb[(j * (D / 2) + c * E + e) * 16 + tl] = (uint8_t)(code[j][e / 4] >> (8 * (e & 3)));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const bool mixed = t0 < first || t0 + 16 > last;
    uint32_t m[4], s[4];                                                // bytes of new tokens; of tokens behind the last
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = s[i] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int tt = t0 + 4 * i + j;
        m[i] |= tt >= first && tt < last ? 0xFFu << (8 * j) : 0u;
        s[i] |= tt >= last ? 0xFFu << (8 * j) : 0u;
      }
    }
#pragma unroll
    for (int p = 0; p < D / 64; ++p) {                                  // piece: 16 tokens of one channel
      const int d = p * 64 + lane;
      uint4* dst = reinterpret_cast<uint4*>(blk + (g * D + d) * 16);
      uint4 w = *reinterpret_cast<const uint4*>(vb + d * 16);
      if (mixed) {
        uint32_t a[4] = {w.x, w.y, w.z, w.w};
        const uint4 o4 = *dst;
        const uint32_t o[4] = {o4.x, o4.y, o4.z, o4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t was = grown ? down4(o[i], down) : o[i];
          a[i] = (a[i] & m[i]) | (o[i] & s[i]) | (was & ~(m[i] | s[i]));
        }
        w = make_uint4(a[0], a[1], a[2], a[3]);
      }
      *dst = w;
    }
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
  KV800_REQUIRE(R <= INT32_MAX / 4 && T <= (int64_t)INT32_MAX * 32, "kv8_append: too many tokens or rows");
  KV800_REQUIRE((cos_t == nullptr) == (sin_t == nullptr), "kv8_append: cos_t and sin_t go together");
  KV800_REQUIRE(!cos_t || (freqs > 0 && freqs % 8 == 0 && freqs <= cache->dim / 2 && rope_rows > 0 && (uintptr_t)cos_t % 16 == 0 &&
                           (uintptr_t)sin_t % 16 == 0),
                "kv8_append: tables need freqs a multiple of 8 up to D / 2, rows, and 16-byte alignment");
  const dim3 grid((unsigned)((T + 126 * R) / kv8::BLK), (unsigned)((2 * cache->kv_heads + 3) / 4));
  const int F = cos_t ? (int)freqs : 0;
  const kv8::Cache C = kv8::device_form(cache);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, C, k, k_ts, k_hs, v, v_ts, v_hs, bt, bt_stride, bt_cols,
                       lens, qsl, R, T, cos_t, sin_t, rope_rows, F);
  };
  if (cache->dim == 128) go(kv8::append_kernel<128>);
  else go(kv8::append_kernel<64>);
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
