// kv800_attn.h -- device helpers shared by the attention kernels over the 800h cache (kv800_decode.hip,
// kv800_chunk.hip): vector types, MFMA wrappers, cross-lane reductions, conversions, the RoPE of dequantized key pairs and
// buffer resources.
#pragma once
#include "kv800_common.h"

namespace kv800 {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef int i2v __attribute__((ext_vector_type(2)));

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

constexpr float NEG_BIG = -1e30f;

__device__ __forceinline__ uint32_t hbits(h2 x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ h8 pack8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  u4v v = {a, b, c, d};
  return __builtin_bit_cast(h8, v);
}
__device__ __forceinline__ f4 mfma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ uint32_t pk2(float a, float b) {   // two floats -> packed fp16 (round to nearest even)
  h2 v = {(_Float16)a, (_Float16)b};
  return hbits(v);
}

// Values of the lanes 16 (32) apart without an LDS round trip: v_permlane16_swap (v_permlane32_swap) on two copies of
// x leaves the even 16-lane row (lower half) in .x and the odd row (upper half) in .y, in both lanes of each pair, so
// combining .x and .y gives the pair the same result. All 64 lanes must be active.
__device__ __forceinline__ float2 rows16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float2 halves32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum4rows(float x) {   // sum over lanes l, l ^ 16, l ^ 32, l ^ 48
  float2 p = rows16(x);
  p = halves32(p.x + p.y);
  return p.x + p.y;
}
__device__ __forceinline__ float max4rows(float x) {
  float2 p = rows16(x);
  p = halves32(vmax(p.x, p.y));
  return vmax(p.x, p.y);
}

// Four fp8 e4m3fn bytes of w -> floats (byte i -> o[i]) with the hardware conversion: gfx950 converts the OCP e4m3
// format, the same as torch's float8_e4m3fn, exactly; the NaN bytes 0x7F / 0xFF give NaN as torch's .float() does
// (kv800.py:84-91; the quantizer writes them only for scales beyond +-464).
__device__ __forceinline__ void f8x4(uint32_t w, float* o) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  o[0] = a[0]; o[1] = a[1]; o[2] = b[0]; o[3] = b[1];
}

__device__ __forceinline__ float bf_elem(const u4v& x, int e) {   // bf16 element e < 8 of x as a float
  const uint32_t w = x[e >> 1];
  return __uint_as_float((e & 1) ? (w & 0xFFFF0000u) : (w << 16));
}
__device__ __forceinline__ uint32_t bfpk(float a, float b) {   // two floats -> packed bf16 (round to nearest even)
  const bf2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ b8 as_b8(const u4v& x) { return __builtin_bit_cast(b8, x); }
__device__ __forceinline__ f4 mfma_bf(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Slot of chunk token t in the staged vb rows: slot 8 g + k holds token 4 g + k (k < 4) or 16 + 4 g + k - 4, the 8
// tokens of lane group g in the K order of the PV MFMA (the tokens whose scores the group's lanes hold).
__device__ __forceinline__ int vb_slot(int t) { return 8 * ((t >> 2) & 3) + 4 * (t >> 4) + (t & 3); }

// RoPE of four channels' dequantized key pairs k[e] = (k0, k2) (bf16 lo / hi) against cs[e] = (cos, sin) and
// sw[e] = (sin, cos): r[e] = (bf16(k0 cos - k2 sin), bf16(k2 cos + k0 sin)), torch_decode.py:22-24. Each sum comes from
// one v_dot2_f32_bf16 (exact bf16 products; the hardware sum is within one fp32 ulp of the rounded exact sum, which
// changes the bf16 rounding that follows only for values within that ulp of a bf16 rounding boundary) and the pair is
// rounded by v_cvt_pk_bf16_f32 (RNE). The compiler does not see inside the block, so the block keeps the hazards of the
// dot instructions itself: every v_cvt reads dot results written at least three instructions earlier, and the
// leading / trailing s_nop cover a VALU write of an input just before and an MFMA read of an output just after.
__device__ __forceinline__ void rope4(const uint32_t (&k)[4], const uint32_t (&cs)[4], const uint32_t (&sw)[4],
                                      uint32_t (&r)[4]) {
  uint32_t t0, t1, t2, t3;
  asm("s_nop 1\n"
      "v_dot2_f32_bf16 %0, %8, %12, 0 neg_hi:[0,1,0]\n"
      "v_dot2_f32_bf16 %4, %8, %16, 0\n"
      "v_dot2_f32_bf16 %1, %9, %13, 0 neg_hi:[0,1,0]\n"
      "v_dot2_f32_bf16 %5, %9, %17, 0\n"
      "v_dot2_f32_bf16 %2, %10, %14, 0 neg_hi:[0,1,0]\n"
      "v_dot2_f32_bf16 %6, %10, %18, 0\n"
      "v_dot2_f32_bf16 %3, %11, %15, 0 neg_hi:[0,1,0]\n"
      "v_dot2_f32_bf16 %7, %11, %19, 0\n"
      "v_cvt_pk_bf16_f32 %0, %0, %4\n"
      "v_cvt_pk_bf16_f32 %1, %1, %5\n"
      "v_cvt_pk_bf16_f32 %2, %2, %6\n"
      "v_cvt_pk_bf16_f32 %3, %3, %7\n"
      "s_nop 1"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(t0), "=&v"(t1), "=&v"(t2), "=&v"(t3)
      : "v"(k[0]), "v"(k[1]), "v"(k[2]), "v"(k[3]), "v"(cs[0]), "v"(cs[1]), "v"(cs[2]), "v"(cs[3]), "v"(sw[0]),
        "v"(sw[1]), "v"(sw[2]), "v"(sw[3]));
}
__device__ __forceinline__ b8 pack8b(const uint32_t (&x)[4]) { return as_b8(u4v{x[0], x[1], x[2], x[3]}); }

// Sub-block reads go through a buffer resource of the sub-block (base and size in SGPRs, built per sub-block by
// scalar instructions): each load's address is a lane constant plus a wave-uniform SGPR offset plus its immediate, so
// no per-lane address arithmetic runs per chunk, and a read past the 51,200 bytes returns zeros.
typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr int RSRC_WORD3 = 0x00020000;   // raw (untyped, unswizzled) buffer access on gfx9-family parts
__device__ __forceinline__ rsrc_t sub_rsrc(const uint8_t* sb) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(sb), (short)0, SUB, RSRC_WORD3);
}

// Byte E of x, zero-extended, or'ed with base: one v_or_b32_sdwa (the compiler forms it from two instructions).
template <int E>
__device__ __forceinline__ uint32_t byte_or(uint32_t x, uint32_t base) {
  uint32_t r;
  asm("v_or_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_%c3 src1_sel:DWORD"
      : "=v"(r) : "v"(x), "v"(base), "n"(E));
  return r;
}

}  // namespace
}  // namespace kv800
