// kv800_chunk.hip -- attention of a few new tokens per row over the paged 800h cache for gfx950 (decode_chunk): the rows of a
// step that verifies drafted tokens, or brings a short prompt chunk. The reference attends such rows by assembling
// their whole history as bf16 keys first (vllm_attn.py:351-402); here the compressed blocks and pages are read as they are.
//
// Row r has c = qsl[r + 1] - qsl[r] queries at positions N[r] - c + i, 16 query heads over 4 KV heads (head 4 h + e reads KV
// head h), head_dim 128. Its keys: positions below 256 NQ[r] from the quantized sub-blocks (K = bf16(code ksc + klo),
// V = (bit vsc + vlo) H), the others from the exact pages, or its sinks; K rotated in fp32 and rounded to bf16 as the model
// does; scores q . K / sqrt(128), softmax over the positions that the query may see, in fp32.
//
// A tile is QT = 4 CT queries of one row; for one KV head they are 16 CT columns (query, query head) of a matrix product,
// so that the 16 columns of an MFMA, of which a single token fills 4, are all of use: the keys of a chunk are
// unpacked and rotated once for all of a tile's queries. Tile k of row r has the number r + qsl[r] / QT + k (ascending over
// the rows without a scan; at most R + T / QT numbers, of which some stay without a tile).
//
//   quant_part           the sub-blocks, one workgroup of 4 waves per equal share of the list of (tile, 64 tokens), wave = KV
//                        head; writes a partial (m, l, acc) per tile that it enters
//   exact_part           exact rows and sinks, one workgroup per (tile, KV head); writes a partial, or for layers without
//                        sub-blocks the output
//   chunk_both_kernel    the two in one launch; chunk_quant_kernel, chunk_exact_kernel: in a launch each
//   chunk_merge_kernel   partials of a (tile, KV head) joined, Hadamard transform of the quantized part, bf16 output
//
// What bounds it (rates of a large copy 5.1 TB/s, of a large read 6.0 TB/s): long lists of tiles of 4 take about twice the
// time of their bytes (64 rows x 32768 x 4 tokens, 451 MB: 156 us of quant_part in a long run of calls, up to 230 from an idle
// card, whose clock is low), VALU instructions in 69 % of the cycles, which are table lookups and rotation of the keys; it reads
// 677 MB, for rows out of step need every position of the rope table at once, 4 MB beside the stream in each L2. Each column's
// share of the instructions falls with the tile: tiles of 8 take 1.4 times as long for twice the queries. Window layers
// read at 4.1 TB/s (398 rows x 5 tokens, 223 MB: 55 us). One row takes 17 + 6 us for 5 tokens at 16384 positions: the latency
// of exact chunks and of lookups one after the other, and of a second launch.
#include <mutex>

#include "kv800_attn.h"
#include "../../include/kv800_hip.h"

namespace kv800 {
namespace {

// v_maximum3_f32, which needs no operand quieted first (fmaxf does, for operands straight from an MFMA); NaN wins
__device__ __forceinline__ float maxn(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ int64_t uniform64(int64_t x) {   // a value that all lanes share, as a scalar
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), CTRL, 0xF, 0xF, false));
}
// over a wave, the same in every lane: within rows of 16 by DPP (lanes 1 and 2 apart, mirrored halves, mirrored rows), then
// across the rows
__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp<0xB1>(x)); x = fmaxf(x, dpp<0x4E>(x)); x = fmaxf(x, dpp<0x141>(x)); x = fmaxf(x, dpp<0x140>(x));
  return max4rows(x);
}

struct ChunkArgs {
  kv800_paged_t P;
  const uint16_t* q;
  const int64_t* qsl;
  int64_t R, T;
  const uint16_t *cos_t, *sin_t;   // null: keys as stored
  const uint32_t* cs2;
  int64_t rope_rows, qpool_bytes, epool_elems, sink_elems;
  int64_t G, I;                    // workgroups of the quantized list; tile numbers
  int32_t* pre;                    // R + 1: the quantized list's entries before each row; then entries per workgroup
  float *mo, *lo, *ao;             // partial slots: [slot][4 heads][16 CT columns] and, for ao, [128]
  uint16_t* out;
  float scale;                     // log2(e) / sqrt(128)
  int nsink;
  int held;                        // positions that the page and rope tables hold
  bool xfirst;                     // one launch: the exact part's workgroups come first
};

// A tile: its row, the row's first token, length and queries, the tile's first query and queries
struct Tile { int64_t row, t0; int n, c, q0, nq; };
template <int QT>
__device__ __forceinline__ int64_t tile_number(const int64_t* qsl, int64_t T, int64_t r) { return r + min(qsl[r], T) / QT; }
// Tile `it`: 64-way search for the last row whose first tile number is <= it, by a whole wave; false if the number has none.
template <int QT>
__device__ __forceinline__ bool find_tile(const ChunkArgs& A, int64_t it, Tile& t) {
  const int64_t lo = last_at(A.R, [&](int64_t i) { return tile_number<QT>(A.qsl, A.T, i) <= it; });
  const int64_t a = A.qsl[lo], b = A.qsl[lo + 1];
  const int n = A.P.N[lo];                             // asked for along with them
  t.row = lo;
  t.t0 = uniform64(min(a, A.T));
  t.c = (int)(uniform64(min(b, A.T)) - t.t0);
  t.n = __builtin_amdgcn_readfirstlane(n);
  t.q0 = (int)min((it - (lo + t.t0 / QT)) * QT, (int64_t)0x7FFFFFFF);
  t.nq = min(QT, t.c - t.q0);
  return t.nq > 0;
}

// ---------------------------------------------------------------- quantized sub-blocks
// Log2 units by which a score may exceed the running max before the state is rescaled; with the exact max a quarter of the
// chunks rescaled (52 instructions).
constexpr float QLAZY = 4.f;
// Weights p vsc go to the matrix product as fp16, held as p vsc 2^(WEXP - ve), 2^ve above every vsc of the span so far: 2^(QLAZY
// + WEXP) = 2^15 at most, and 11 bits down to 2^-14, 2^-25 of a weight of 1 at the largest scale; what is below is off by
// 2^-36 of that at most. fp16(p vsc) itself lost bits from 2^-14 on and all of them from 2^-25 on: behind one key 12 to 17 above the
// others whose value is near zero, outputs were off by 6 to 700 %. Following the largest scale costs 0.4 % (192 ragged rows).
constexpr int WEXP = 11;
constexpr int VE_MIN = -9;     // the least e4m3 number
constexpr int QCH = 32;        // tokens per stage
// A stage as it lies in LDS: kc, (cos, sin) and vb rows of 32 tokens, all heads, in pieces of 16 bytes. Pieces are permuted
// within a row so that the reads of one piece of 16 rows spread over the banks: piece p of token t at p ^ (t % 8), of vb rows
// (4 pieces) at p ^ (t / 2 % 4).
struct alignas(16) ChunkStage {
  uint8_t kc[QCH * 128], cs[QCH * 128], vb[QCH * 64];
};
struct QLutWords { uint32_t la, lb, sa, sb; };   // klo / ksc bytes of the table that the lane builds
struct ListRow { int t0, c, n, nu; };                  // first token, queries, length, entries per tile
struct alignas(16) ChunkQLds {
  uint32_t lut[4][1024];       // each wave's code tables of the sub-block it is in
  float vs[4][64], vl[4][64];  // decoded vsc / vlo of 64 tokens
  int ws[4], row, pre;
  ListRow at;
};

// 16 tables of 4 groups: block (kind, d, e) of 256 bytes holds the tables of channels 8 g + 4 d + e, g = 0..3, entry (ca, cb)
// of group g at byte 64 cb + 16 g + 4 ca. Lane l builds the table of g = l % 4, block l / 4.
__device__ __forceinline__ QLutWords lut_words(rsrc_t rs, int h, int lane) {
  const int kind = lane >> 5, j = 8 * (lane & 3) + 4 * ((lane >> 4) & 1) + ((lane >> 2) & 3);
  const int o = 128 * h + 32 * kind + j;
  return QLutWords{__builtin_amdgcn_raw_buffer_load_b8(rs, o, KLO_O, 0), __builtin_amdgcn_raw_buffer_load_b8(rs, o + 64, KLO_O, 0),
                   __builtin_amdgcn_raw_buffer_load_b8(rs, o, KSC_O, 0), __builtin_amdgcn_raw_buffer_load_b8(rs, o + 64, KSC_O, 0)};
}
__device__ __forceinline__ void lut_build(uint32_t* lut, int lane, const QLutWords& b) {
  float v[4];
  f8x4(b.la | (b.lb << 8) | (b.sa << 16) | (b.sb << 24), v);   // klo_a, klo_b, ksc_a, ksc_b
  uint32_t pa[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) pa[c] = bfpk(fmaf((float)c, v[2], v[0]), fmaf((float)c, v[3], v[1]));
  uint32_t* tab = lut + 64 * (lane >> 2) + 4 * (lane & 3);
#pragma unroll
  for (int k = 0; k < 4; ++k) {                                // lanes 4 i .. 4 i + 3 start at row i % 4: all banks at once
    const int cb = (k + (lane >> 2)) & 3;
    const uint32_t hi = (cb & 2 ? (cb & 1 ? pa[3] : pa[2]) : (cb & 1 ? pa[1] : pa[0])) & 0xFFFF0000u;
    *reinterpret_cast<u4v*>(tab + 16 * cb) =
        u4v{(pa[0] & 0xFFFFu) | hi, (pa[1] & 0xFFFFu) | hi, (pa[2] & 0xFFFFu) | hi, (pa[3] & 0xFFFFu) | hi};
  }
}
// Wave w's part of a stage, straight into LDS: tokens 8 w .. + 7 of kc and cs, and (waves 0, 1) tokens 16 w .. + 15 of vb. Lane l
// writes bytes 16 l .. + 15 of the wave's kilobyte and fetches the piece that belongs there, so that a load reads whole
// lines: rows fetched straight into the operand layout (lane = token, 128 bytes apart) cost the L1 one line per lane, 460
// per chunk and head, and held it busy 86 % of the time (64 rows x 32768 x 4: 242 us; staged 174 us).
__device__ __forceinline__ void stage_load(ChunkStage& S, rsrc_t rs, rsrc_t rc, int cpos, int t0, int w, int lane) {
  typedef __attribute__((address_space(3))) void lds_v;
  const int o = (lane >> 3) * 128 + 16 * ((lane & 7) ^ (lane >> 3));
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_v*)&S.kc[1024 * w], 16, o, KC_O + (t0 + 8 * w) * 128, 0, 0);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rc, (lds_v*)&S.cs[1024 * w], 16, o, (cpos + t0 + 8 * w) * 128, 0, 0);
  if (w < 2)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_v*)&S.vb[1024 * w], 16,
                                             (lane >> 2) * 64 + 16 * ((lane & 3) ^ ((lane >> 3) & 3)),
                                             VB_O + (t0 + 16 * w) * 64, 0, 0);
  asm volatile("" ::"s"((uint32_t)(uintptr_t)&S) : "memory");   // the loads write S behind the compiler's view
}
__device__ __forceinline__ uint32_t chunk_scales(rsrc_t rs, int t0, int h, int lane) {   // vlo | vsc << 8 of token t0 + lane
  const int o = 2 * lane + (h >> 1);
  return (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(rs, o, VLO_O + 2 * t0, 0) |
         ((uint32_t)__builtin_amdgcn_raw_buffer_load_b8(rs, o, VSC_O + 2 * t0, 0) << 8);
}

// The list of (tile, 64 tokens) pairs, tile by tile: row r has tiles x sub-blocks x 4 of them.
// Sub-blocks past the host's bound, the offset table or the rope table are not read: P.nqmax is the least of the three.
__device__ __forceinline__ int row_nq(const ChunkArgs& A, int64_t r) { return min(max(A.P.NQ[r], 0), 1 << 22); }
__device__ __forceinline__ int row_blocks(const ChunkArgs& A, int64_t r) {
  return (int)min((int64_t)row_nq(A, r), A.P.nqmax);
}
// Attention of one tile's columns of KV head h (the wave's) over tokens [64 u0, 64 u1) of its row, into partial slot `slot`.
// As in decode_quant_kernel, with the wave's one head: K pairs by table lookup, RoPE by v_dot2_f32_bf16, Q K^T on bf16 MFMA
// with exact products; fp32 online softmax; P V on fp16 MFMA over the bit planes, weights of 11 bits, an eighth of the output's own
// rounding.
// NC: columns of a slot, of which the tile has 16 CT at most.
template <int CT, int NC>
__device__ __forceinline__ void chunk_span(ChunkQLds& L, ChunkStage& SA, ChunkStage& SB, const ChunkArgs& A, const Tile& t, int u0, int u1, int64_t slot) {
  const int h = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, n = lane & 15;
  const char* lutc = reinterpret_cast<const char*>(&L.lut[0][0]);
  const int pbase = t.n - t.c + t.q0;                 // position of the tile's first query
  int pcol[CT];
  b8 bq[CT][4];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int qi = 4 * ct + (n >> 2);
    pcol[ct] = pbase + qi;
    const uint16_t* qr = A.q + ((t.t0 + t.q0 + min(qi, t.nq - 1)) * 16 + 4 * h + (n & 3)) * 128 + 8 * g;
    const u4v Q0 = *reinterpret_cast<const u4v*>(qr), Q1 = *reinterpret_cast<const u4v*>(qr + 32);
    const u4v Q2 = *reinterpret_cast<const u4v*>(qr + 64), Q3 = *reinterpret_cast<const u4v*>(qr + 96);
    auto el = [](const u4v& Q, int i) -> uint32_t { return (Q[i >> 1] >> (16 * (i & 1))) & 0xFFFFu; };
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      uint32_t r[4], p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        r[e] = el(Q0, 4 * d + e) | (el(Q2, 4 * d + e) << 16);
        p[e] = el(Q1, 4 * d + e) | (el(Q3, 4 * d + e) << 16);
      }
      bq[ct][d] = pack8b(r);
      bq[ct][2 + d] = pack8b(p);
    }
  }
  float m[CT], lsum[CT], lvs[CT];
  f4 acc[CT][8];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = NEG_BIG; lsum[ct] = 0.f; lvs[ct] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[ct][i] = f4{0.f, 0.f, 0.f, 0.f};
  }
  const float scale = A.scale;
  // 2^ve and what the scales are multiplied by before P V; the sums follow when ve grows. The fp32 sum of vlo needs none of it
  int ve = VE_MIN;
  float cap = 0x1p-9f, fac = 0x1p20f;                  // 2^ve, 2^(WEXP - ve)
  auto stage_scales = [&](uint32_t x) {
    float v[4];
    f8x4(x, v);
    const float a = fabsf(v[1]);
    if (__builtin_expect(__any(a > cap), 0)) {
      const float top = wave_max(a);                   // a NaN scale is not among them
      const int e = __builtin_amdgcn_readfirstlane((int)(__float_as_uint(top) >> 23) - 126);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[ct][i] *= ldexpf(1.f, ve - e);
      ve = e;
      cap = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(ldexpf(1.f, e))));
      fac = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(ldexpf(1.f, WEXP - e))));
    }
    L.vl[h][lane] = v[0];
    L.vs[h][lane] = v[1] * fac;
  };
  const uint32_t kg = (uint32_t)h * 4096u + 16u * (uint32_t)g;
  // one 32-token chunk, tokens 32 cc .. of the staged 64; kpos: position of its first token
  const int okc = n * 128 + 16 * ((2 * h + (g >> 1)) ^ (n & 7)) + 8 * (g & 1);   // kc bytes of channels 8 g .. of token n
  const int ocs = n * 128 + 16 * ((2 * g) ^ (n & 7));                            // its pairs of channels 8 g .. + 3; the next
                                                                                 // four in the piece beside it (^ 16)
  // the transposed vb read: lane n of group g gives row n / 2 of the group's 8 tokens 4 g .., 16 + 4 g .. (the tokens whose
  // scores its lanes hold), half n % 2
  const int tvb = 4 * g + ((n >> 1) & 3) + 16 * (n >> 3);
  const int ovb = tvb * 64 + 16 * (h ^ ((tvb >> 1) & 3)) + 8 * (n & 1);
  auto chunk = [&](const ChunkStage& S, int cc, int kpos) {
    f4 sc[2][CT];
    __builtin_amdgcn_s_setprio(3);
    // 4 steps (tile u, kc dword d); a step's table reads are issued two steps ahead of their use, all operands of the
    // stage before the first
    uint2 kc[2];
    u4v cs[2][2];
    uint32_t kk[3][4], an[3][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) kc[u] = *reinterpret_cast<const uint2*>(&S.kc[okc + 2048 * u]);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int d = 0; d < 2; ++d) cs[u][d] = *reinterpret_cast<const u4v*>(&S.cs[(ocs ^ (16 * d)) + 2048 * u]);
    auto lookup = [&](const int st) {
      const int u = st >> 1, d = st & 1, b = st % 3;
      const uint32_t x = d ? kc[u].y : kc[u].x;
      const uint32_t xr = (x << 2) & 0xCCCCCCCCu, xn = x & 0xCCCCCCCCu;
      const char *br = lutc + 256 * (4 * d), *bn = lutc + 256 * (8 + 4 * d);
      kk[b][0] = *reinterpret_cast<const uint32_t*>(br + byte_or<0>(xr, kg));
      kk[b][1] = *reinterpret_cast<const uint32_t*>(br + 256 + byte_or<1>(xr, kg));
      kk[b][2] = *reinterpret_cast<const uint32_t*>(br + 512 + byte_or<2>(xr, kg));
      kk[b][3] = *reinterpret_cast<const uint32_t*>(br + 768 + byte_or<3>(xr, kg));
      an[b][0] = *reinterpret_cast<const uint32_t*>(bn + byte_or<0>(xn, kg));
      an[b][1] = *reinterpret_cast<const uint32_t*>(bn + 256 + byte_or<1>(xn, kg));
      an[b][2] = *reinterpret_cast<const uint32_t*>(bn + 512 + byte_or<2>(xn, kg));
      an[b][3] = *reinterpret_cast<const uint32_t*>(bn + 768 + byte_or<3>(xn, kg));
      __builtin_amdgcn_sched_barrier(0);
    };
    __builtin_amdgcn_sched_barrier(0);
    lookup(0);
    lookup(1);
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      if (st + 2 < 4) lookup(st + 2);
      const int u = st >> 1, d = st & 1, b = st % 3;
      uint32_t c4[4], s4[4], ar[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c4[e] = cs[u][d][e];
        s4[e] = __builtin_amdgcn_alignbit(cs[u][d][e], cs[u][d][e], 16);
      }
      rope4(kk[b], c4, s4, ar);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        sc[u][ct] = mfma_bf(pack8b(ar), bq[ct][d], d == 0 ? f4{0.f, 0.f, 0.f, 0.f} : sc[u][ct]);
        sc[u][ct] = mfma_bf(pack8b(an[b]), bq[ct][2 + d], sc[u][ct]);
      }
    }
    // A weight of 0 does not take out a NaN scale: where queries do not see all of the chunk, such a token's scales become 0 and
    // its scores NaN, for the queries that see it.
    uint32_t odd = 0;
    if (kpos + 31 > pbase) {
      const int tk = 32 * cc + (lane & 31);
      const bool bad = __builtin_isnan(L.vs[h][tk]) || __builtin_isnan(L.vl[h][tk]);
      odd = (uint32_t)__ballot(bad);
      if (bad) L.vs[h][tk] = L.vl[h][tk] = 0.f;
    }
    // what the softmax and P V read, issued under the last products
    float4 vs4[2], vl4[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int tk = 32 * cc + 16 * u + 4 * g;
      vs4[u] = *reinterpret_cast<const float4*>(&L.vs[h][tk]);
      vl4[u] = *reinterpret_cast<const float4*>(&L.vl[h][tk]);
    }
    typedef __attribute__((address_space(3))) i2v lds_i2;
    const i2v X = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2*)(const_cast<uint8_t*>(S.vb) + ovb));
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(2);
    if (kpos + 31 > pbase) {                           // a caller's NQ that reaches into the new tokens: mask by position
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (kpos + 16 * u + 4 * g + i > pcol[ct]) sc[u][ct][i] = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((odd >> (16 * u + 4 * g + i)) & 1u && kpos + 16 * u + 4 * g + i <= pcol[ct]) sc[u][ct][i] = __builtin_nanf("");
    }
    h8 Bw[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const f4 s0 = sc[0][ct], s1 = sc[1][ct];
      float tmax = maxn(maxn(maxn(s0[0], s0[1]), maxn(s0[2], s0[3])), maxn(maxn(s1[0], s1[1]), maxn(s1[2], s1[3])));
      if (__any(tmax * scale > m[ct] + QLAZY)) {       // a lane's own scores; the column's maximum only where it matters
        const float mn = fmaxf(m[ct], max4rows(tmax + 0.f) * scale);
        const float al = __builtin_amdgcn_exp2f(m[ct] - mn);
        m[ct] = mn; lsum[ct] *= al; lvs[ct] *= al;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[ct][i] *= al;
      }
      float wt[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[u][ct][0], scale, -m[ct]));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[u][ct][1], scale, -m[ct]));
        const float p2 = __builtin_amdgcn_exp2f(fmaf(sc[u][ct][2], scale, -m[ct]));
        const float p3 = __builtin_amdgcn_exp2f(fmaf(sc[u][ct][3], scale, -m[ct]));
        lsum[ct] += (p0 + p1) + (p2 + p3);
        lvs[ct] = fmaf(p3, vl4[u].w, fmaf(p2, vl4[u].z, fmaf(p1, vl4[u].y, fmaf(p0, vl4[u].x, lvs[ct]))));
        wt[u][0] = p0 * vs4[u].x; wt[u][1] = p1 * vs4[u].y; wt[u][2] = p2 * vs4[u].z; wt[u][3] = p3 * vs4[u].w;
      }
      Bw[ct] = pack8(pk2(wt[0][0], wt[0][2]), pk2(wt[0][1], wt[0][3]), pk2(wt[1][0], wt[1][2]), pk2(wt[1][1], wt[1][3]));
    }
    __builtin_amdgcn_s_setprio(0);
    const uint32_t x0 = (uint32_t)X.x, x1 = (uint32_t)X.x >> 8, x2 = (uint32_t)X.y, x3 = (uint32_t)X.y >> 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t msk = (1u << i) | (1u << (16 + i));
      const h8 a = pack8(x0 & msk, x1 & msk, x2 & msk, x3 & msk);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) acc[ct][i] = mfma16(a, Bw[ct], acc[ct][i]);
    }
    asm volatile("" ::: "memory");
  };

  // the span's u1 - u0 pairs of 32-token stages, one after the other; loads one stage ahead, tables and scales one pair
  const int64_t* brow = A.P.boff + t.row * A.P.boff_stride;
  auto sanitize = [&](int64_t x, int jb) -> int64_t {
    const int64_t raw = uniform64(x);
    return (raw < 0 || raw > A.qpool_bytes - SUB || (int64_t)(jb + 1) * BLK > A.rope_rows) ? -1 : raw;
  };
  const rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t*>(A.cs2), (short)0,
                                                      (int)min(A.rope_rows * 128, (int64_t)INT32_MAX), RSRC_WORD3);
  const int np = u1 - u0, jl = (u1 - 1) >> 2;          // pairs; the last sub-block
  int jb = u0 >> 2, pin = u0 & 3;
  int64_t base = sanitize(brow[jb], jb), nraw = brow[min(jb + 1, jl)];
  rsrc_t rs = sub_rsrc(A.P.qpool + (base < 0 ? 0 : base));
  int cpos = base < 0 ? 0 : jb * BLK;
  stage_load(SA, rs, rc, cpos, 64 * pin, h, lane);
  lut_build(L.lut[h], lane, lut_words(rs, h, lane));
  stage_scales(chunk_scales(rs, 64 * pin, h, lane));
  __syncthreads();
  for (int p = 0; p < np; ++p) {
    const bool more = p + 1 < np, cross = more && pin == 3;
    const int njb = cross ? jb + 1 : jb, npin = cross ? 0 : (pin + 1) & 3;
    int64_t nbase = base;
    rsrc_t nrs = rs;
    int ncpos = cpos;
    stage_load(SB, rs, rc, cpos, 64 * pin + 32, h, lane);
    if (cross) {
      nbase = sanitize(nraw, njb);
      nrs = sub_rsrc(A.P.qpool + (nbase < 0 ? 0 : nbase));
      ncpos = nbase < 0 ? 0 : njb * BLK;
      nraw = brow[min(njb + 1, jl)];
    }
    const QLutWords nlw = lut_words(nrs, h, lane);
    const uint32_t nsc = chunk_scales(nrs, 64 * npin, h, lane);
    if (base >= 0) chunk(SA, 0, cpos + 64 * pin);
    __syncthreads();                                   // SB is whole, and everyone is done with SA
    if (more) stage_load(SA, nrs, rc, ncpos, 64 * npin, h, lane);
    if (base >= 0) chunk(SB, 1, cpos + 64 * pin + 32);
    if (more) {
      if (cross) lut_build(L.lut[h], lane, nlw);
      stage_scales(nsc);
    }
    __syncthreads();
    jb = njb; pin = npin; base = nbase; rs = nrs; cpos = ncpos;
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const float ls = sum4rows(lsum[ct]), lv = sum4rows(lvs[ct]);
    if (4 * ct + (n >> 2) < t.nq) {
      const int64_t col = (slot * 4 + h) * NC + 16 * ct + n;
      if (g == 0) { A.mo[col] = m[ct]; A.lo[col] = ls; }
#pragma unroll
      for (int i = 0; i < 8; ++i) {                    // plane i: dims 16 i + 4 g + r, bits worth 2^(i - 24)
        const float ps = __uint_as_float((uint32_t)(127 + 24 - WEXP + ve - i) << 23);
        const f4 o = acc[ct][i];
        *reinterpret_cast<float4*>(A.ao + col * 128 + 16 * i + 4 * g) =
            make_float4(o[0] * ps + lv, o[1] * ps + lv, o[2] * ps + lv, o[3] * ps + lv);
      }
    }
  }
}

// Workgroup w takes entries [w C, (w + 1) C) of the list, C = ceil(total / G): equal shares, whatever the rows' lengths. Two
// stages of loads, one ahead: three, two ahead, took 186 us against 167 (64 rows x 32768 x 4), their barriers and addresses
// costing more than the waits that they saved. The part of a tile that it begins with goes
// to slot w; a tile that starts inside its range goes to slot G + the tile's number (nobody else enters that tile from an
// earlier entry).
__device__ __forceinline__ ListRow list_row(const ChunkArgs& A, int64_t r) {
  const int64_t a = A.qsl[r], b = A.qsl[r + 1];
  const int n = A.P.N[r], nb = row_blocks(A, r);
  ListRow x;
  x.t0 = (int)min(a, A.T);
  x.c = max((int)min(b, A.T) - x.t0, 0);
  x.n = n;
  x.nu = 4 * nb;
  return x;
}
template <int QT>
__device__ __forceinline__ int list_size(const ListRow& x) { return (x.c + QT - 1) / QT * x.nu; }

template <int CT>
__device__ __forceinline__ void quant_part(ChunkQLds& L, ChunkStage& SA, ChunkStage& SB, const ChunkArgs& A, const unsigned wg) {
  constexpr int QT = 4 * CT;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  // every workgroup sums the rows' entries itself: thread i takes the rows [i k, i k + k). The list's entries, and a
  // workgroup's end past them, are below 2^31 (the host's check).
  const int R = (int)A.R, k = (R + 255) / 256, ra = min(tid * k, R), rb = min(ra + k, R);
  ListRow first = {0, 0, 0, 0};
  int mine = 0;
  if (ra < rb) {
    first = list_row(A, ra);
    mine = list_size<QT>(first);
  }
  for (int r = ra + 1; r < rb; ++r) mine += list_size<QT>(list_row(A, r));
  int inc = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(inc, o, 64);
    if (lane >= o) inc += x;
  }
  if (lane == 63) L.ws[w] = inc;
  __syncthreads();
  int pre = inc - mine;
  for (int i = 0; i < w; ++i) pre += L.ws[i];
  const int total = __builtin_amdgcn_readfirstlane(L.ws[0] + L.ws[1] + L.ws[2] + L.ws[3]), G = (int)A.G, C = (total + G - 1) / G;
  if (wg == 0) {                               // for the merge
    int x = pre;
    for (int r = ra; r < rb; ++r) {
      A.pre[r] = x;
      if (r + 1 < rb) x += list_size<QT>(list_row(A, r));
    }
    if (tid == 0) A.pre[R] = C;
  }
  int v = (int)wg * C;
  const int v1 = min(v + C, total);
  if (v >= v1) return;                                 // uniform
  if (v >= pre && v < pre + mine) {                    // one thread: the row of the workgroup's first entry
    ListRow y = first;
    int x = pre, r = ra;
    while (v >= x + list_size<QT>(y)) {
      x += list_size<QT>(y);
      y = list_row(A, ++r);
    }
    L.row = r;
    L.pre = x;
    L.at = y;
  }
  __syncthreads();
  // the walk over the list in scalars: the sub-blocks' buffer resources, offsets and loop bounds stay in SGPRs
  auto scalar = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  int r = scalar(L.row), x = scalar(L.pre);
  ListRow y = L.at;
  for (bool head = true;; head = false) {
    const int c = scalar(y.c), nu = scalar(y.nu), sz = (c + QT - 1) / QT * nu;
    while (v < v1 && v < x + sz) {
      const int tile = (int)((unsigned)(v - x) / (unsigned)nu), u0 = v - x - tile * nu, u1 = min(nu, u0 + (v1 - v));
      Tile t;
      t.row = r;
      t.t0 = scalar(y.t0);
      t.n = scalar(y.n);
      t.c = c;
      t.q0 = tile * QT;
      t.nq = min(QT, c - t.q0);
      const int64_t slot = head ? (int64_t)wg : A.G + r + (unsigned)t.t0 / QT + tile;
      // a tile of up to 4 queries in one column tile (192 rows with 1 to 8: 238 against 254 us, both with the exact part; shares
      // weighted by the tiles' queries gave nothing more)
      if (CT == 1 || t.nq > 4)
        chunk_span<CT, 16 * CT>(L, SA, SB, A, t, u0, u1, slot);
      else
        chunk_span<1, 16 * CT>(L, SA, SB, A, t, u0, u1, slot);
      head = false;
      v += u1 - u0;
    }
    if (v >= v1) return;
    x += sz;
    y = list_row(A, ++r);
  }
}

__global__ void __launch_bounds__(256, 3) chunk_quant_kernel(ChunkArgs A) {
  __shared__ ChunkQLds L;
  __shared__ ChunkStage SA, SB;   // two objects: a read of one is not held for the other's loads
  quant_part<1>(L, SA, SB, A, blockIdx.x);
}

// ---------------------------------------------------------------- exact rows and sinks
// NW waves per (tile, KV head) take the 32-token chunks of the tile's keys in turn and join their states at the end. The keys
// in order: the row's sinks, exact positions below the sink count (kept out of the window too), exact positions from the
// first one in a query's window up to the last query. As decode_exact_kernel otherwise: Q K^T and P V on bf16 MFMA, weights
// as hi + lo bf16 pairs (16 bits), V^T by transposed reads.
// K and V rows of a chunk go straight into LDS, whole 256-byte rows by 16 lanes each (fetched in the operand layout, lane =
// token, every lane is a cache line of its own: 1,280 line requests per chunk, and 398 rows of a window layer took
// 80 us), in pieces of 16 bytes permuted within the row so that operand reads spread over the banks. One buffer for each: the
// next chunk's K is requested when this one's scores are formed, its V when this one's V is read, so that each is
// in flight for about half a chunk, and 16 KB a wave leave room for the eight waves that 256 registers allow on a CU.
// Window layers, 398 rows x 5: 55 us (223 MB); sliding 64 x 16: 21 us, the latency of five chunks in a row.
constexpr int XCH = 32;
template <int NW>
struct alignas(16) ChunkXRows { uint16_t r[NW][XCH * 128]; };
template <int CT, int NW>
struct alignas(16) ChunkXLds {
  float m[NW][16 * CT], l[NW][16 * CT];
  int odd[NW];
};
__device__ const uint4 chunk_zeros[16] = {};           // a row for tokens without a key: a zero weight needs a finite value

// 16 bytes per lane from p to LDS address dst + 16 lane (dst the same for all lanes). The compiler does not see the load:
// whoever reads it waits by the memory counter (vm_wait), which retires loads in order; the compiler's own waits only come
// out longer. As a builtin, every read of LDS waited for every such load, whichever array it fills.
typedef __attribute__((address_space(3))) uint16_t lds_u16;
__device__ __forceinline__ uint32_t lds_addr(const uint16_t* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const lds_u16*)p);
}
__device__ __forceinline__ void load_lds(const uint16_t* p, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(dst) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void vm_wait() {            // all but the N youngest loads are done
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Queries [qa, qa + nq) of tile t, KV head h. Returns whether an infinity or NaN stands among values that not all of them see:
// a weight of 0 does not take it out of a product, so the caller then has the queries one by one, whose lists hold no other
// keys.
template <int CT, int NW, bool DIRECT>
__device__ __forceinline__ bool exact_tile(ChunkXRows<NW>& Ks, ChunkXRows<NW>& Vs, ChunkXLds<CT, NW>& L, const ChunkArgs& A,
                                           const Tile& t, int64_t it, int h, int qa, int nq) {
  constexpr int NC = 16 * CT, XROW = 132;
  static_assert((NW - 1) * 16 * XROW * 4 <= (int)sizeof(Ks) || NW == 1, "the join must fit");
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));                        // nothing that hangs on it is kept in registers for the next call
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, n = lane & 15;
  const int N = t.n, win = (int)A.P.win;
  const int pbase = N - t.c + t.q0 + qa, plast = pbase + nq - 1;
  const bool wide = CT > 1 && nq > 4;                // a tile of up to 4 queries leaves the second column tile out
  // key list: sinks [0, cnt), exact positions lo_row .. + cnt2, then lo_tile ..
  int lo_row, lo_tile;
  if (win > 0) {
    lo_row = max(0, N - t.c - (win - 1));
    lo_tile = max(lo_row, pbase - (win - 1));
  } else {
    lo_row = lo_tile = A.P.NQ ? __builtin_amdgcn_readfirstlane(row_nq(A, t.row)) * BLK : 0;
  }
  const int cnt = max(0, min(min(A.nsink, lo_row), min(N, plast + 1)));
  const int hi = min(min(N, plast + 1), A.held);       // what the tables do not hold is not walked through
  const int cnt2 = win > 0 ? max(0, min(min(A.nsink, hi) - lo_row, lo_tile - lo_row)) : 0;
  const int rest = lo_tile - cnt - cnt2;               // list index i >= cnt + cnt2 is position rest + i
  const int nk = cnt + cnt2 + max(0, hi - lo_tile);
  const int64_t* et = A.P.eoff + t.row * A.P.eoff_stride;
  const int64_t sko = cnt ? A.P.skoff[t.row] : 0, svo = cnt ? A.P.svoff[t.row] : 0;
  const bool rot = A.cos_t != nullptr;
  const int ebs = (int)A.P.ebs;
  const double iebs = 1.0 / (double)ebs;
  const int64_t hoff = h * A.P.e_hs;
  const int ets = (int)A.P.e_ts;
  const uint16_t* const zeros = reinterpret_cast<const uint16_t*>(chunk_zeros);
  auto posof = [&](int i) {
    const int x = i < cnt + cnt2 ? lo_row - cnt : rest;
    return i + (i < cnt ? 0 : x);
  };
  // Lane l (and l ^ 32) looks after token l % 32 of a chunk. page(): its page's offset, asked for two chunks ahead, before the
  // rows of the chunk between: loads retire in order. locate(): its K and V row of head h.
  auto split = [&](int pos, int& pg, int& in) {        // pos = pg ebs + in
    pg = (int)((double)pos * iebs);                    // within one of the quotient
    in = pos - pg * ebs;
    if (in < 0) { --pg; in += ebs; }
    if (in >= ebs) { ++pg; in -= ebs; }
  };
  auto page = [&](int c0) -> int64_t {
    const int i = c0 + (lane & 31);
    int pg = 0, in;
    if (i >= cnt && i < nk) split(posof(i), pg, in);
    return et[pg];                                     // of a position below A.held, or the first
  };
  struct Where { const uint16_t *k, *v; uint32_t ok; };   // bit t of ok: token t of the chunk has a key
  auto locate = [&](int c0, int64_t base) {
    const int i = c0 + (lane & 31);
    Where r = {zeros, zeros, 0u};
    bool ok = false;
    if (i < nk) {
      const int pos = posof(i);
      int64_t ko, vo;
      const uint16_t *kb = A.P.epool, *vb = A.P.epool;
      if (i < cnt) {
        ko = sko + ((int64_t)i * 4 + h) * 128;
        vo = svo + ((int64_t)i * 4 + h) * 128;
        ok = sko >= 0 && svo >= 0 && ko + 128 <= A.sink_elems && vo + 128 <= A.sink_elems;
        kb = A.P.sk; vb = A.P.sv;
      } else {
        int pg, in;
        split(pos, pg, in);
        ko = base + hoff + (int64_t)in * ets;
        vo = ko + A.P.e_v;
        ok = base >= 0 && ko >= 0 && vo >= 0 && ko + 128 <= A.epool_elems && vo + 128 <= A.epool_elems;
      }
      ok = ok && (!rot || pos < A.rope_rows);
      if (ok) { r.k = kb + ko; r.v = vb + vo; }
    }
    r.ok = (uint32_t)__ballot(ok);
    return r;
  };
  auto key_at = [&](int c0, uint32_t ok, int e) {      // position of token e of the chunk; past every query if it has no key
    const int kp = c0 >= cnt + cnt2 ? rest + c0 + e : posof(c0 + e);
    return (ok >> e) & 1u ? kp : 0x7FFFFFFF;
  };
  auto sees = [&](int qp, int kp) { return (kp <= qp) & ((kp > (win > 0 ? qp - win : -1)) | (kp < A.nsink)); };
  const uint32_t kl = lds_addr(Ks.r[w]), vl = lds_addr(Vs.r[w]);
  const int r4 = lane >> 4, pc = lane & 15;            // an instruction fills 4 rows: row r4, piece pc
  auto row_at = [&](const uint16_t* p, int t) {        // token t's pointer
    const uint64_t x = (uint64_t)p;
    const uint32_t lo = __shfl((uint32_t)x, t, 64), hi = __shfl((uint32_t)(x >> 32), t, 64);
    return (const uint16_t*)(((uint64_t)hi << 32) | lo);
  };
  auto load_k = [&](const uint16_t* p) {               // piece p of token t at p ^ (t % 16)
    const uint16_t* src[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) src[i] = row_at(p, 4 * i + r4) + 8 * (pc ^ ((4 * i + r4) & 15));
#pragma unroll
    for (int i = 0; i < 8; ++i) load_lds(src[i], kl + 1024 * i);
  };
  auto load_v = [&](const uint16_t* p) {               // at p ^ 2 (t % 8): pairs of pieces stay together
    const uint16_t* src[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) src[i] = row_at(p, 4 * i + r4) + 8 * (pc ^ (2 * ((4 * i + r4) & 7)));
#pragma unroll
    for (int i = 0; i < 8; ++i) load_lds(src[i], vl + 1024 * i);
  };
  struct Rope { u4v c[2], s[2]; };                     // cos / sin of channels 8 g .. + 7 at token 16 u + n
  auto load_rope = [&](int c0, Rope& r) {
    if (!rot) return;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = c0 + 16 * u + n;
      const int64_t p = i < nk ? min((int64_t)posof(i), A.rope_rows - 1) : 0;
      r.c[u] = *reinterpret_cast<const u4v*>(A.cos_t + p * 32 + 8 * g);
      r.s[u] = *reinterpret_cast<const u4v*>(A.sin_t + p * 32 + 8 * g);
    }
  };
  b8 bq[CT][4];
  int pcol[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int qi = 4 * ct + (n >> 2);
    pcol[ct] = pbase + qi;
    const uint16_t* qr = A.q + ((t.t0 + t.q0 + qa + min(qi, nq - 1)) * 16 + 4 * h + (n & 3)) * 128 + 8 * g;
#pragma unroll
    for (int s = 0; s < 4; ++s) bq[ct][s] = as_b8(*reinterpret_cast<const u4v*>(qr + 32 * s));
  }
  bool odd = false;                                    // an infinity or NaN among values that not every query sees
  float m[CT], lsum[CT];
  f4 acc[CT][8];                                       // dims 16 j + 4 g + i of column n
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = NEG_BIG; lsum[ct] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[ct][j] = f4{0.f, 0.f, 0.f, 0.f};
  }
  constexpr int STEP = NW * XCH;
  if (w * XCH < nk) {
    Rope rp = {};
    int64_t pg = page(w * XCH), pgn = page(w * XCH + STEP);
    Where at = locate(w * XCH, pg);
    load_rope(w * XCH, rp);
    asm volatile("" ::"v"(rp.c[0]), "v"(rp.c[1]), "v"(rp.s[0]), "v"(rp.s[1]), "v"(pgn) : "memory");   // waited for here
    load_k(at.k);
    load_v(at.v);
    vm_wait<8>();                                      // K is there, V under way
    for (int c0 = w * XCH; c0 < nk; c0 += STEP) {
      const bool more = c0 + STEP < nk;                // uniform
      const Where nx = locate(c0 + STEP, pgn);
      const uint16_t* kw = Ks.r[w];
      f4 sc[2][CT];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        u4v k[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) k[s] = *reinterpret_cast<const u4v*>(kw + (16 * u + n) * 128 + 8 * ((4 * s + g) ^ n));
        if (rot) {
          u4v a0, a2;
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            float r0[2], r2[2];
#pragma unroll
            for (int d = 0; d < 2; ++d) {
#pragma clang fp contract(off)   // products rounded before the sum, as torch_decode.py:22-23 evaluates them
              const float k0 = bf_elem(k[0], e + d), k2 = bf_elem(k[2], e + d);
              const float cs = bf_elem(rp.c[u], e + d), sn = bf_elem(rp.s[u], e + d);
              r0[d] = k0 * cs - k2 * sn;
              r2[d] = k2 * cs + k0 * sn;
            }
            a0[e >> 1] = bfpk(r0[0], r0[1]);
            a2[e >> 1] = bfpk(r2[0], r2[1]);
          }
          k[0] = a0;
          k[2] = a2;
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          if (ct > 0 && !wide) continue;
          f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < 4; ++s) x = mfma_bf(as_b8(k[s]), bq[ct][s], x);
          sc[u][ct] = x;
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // K is read: its rows may be overwritten
      if (more) {
        pgn = page(c0 + 2 * STEP);
        load_rope(c0 + STEP, rp);
        load_k(nx.k);
      }
      // a chunk whose keys are all there and seen by every query of the tile needs no mask
      const int p0 = rest + c0;                        // position of the chunk's first key, behind the sinks
      const bool all = (c0 >= cnt + cnt2) & (at.ok == 0xFFFFFFFFu) & (p0 + 31 <= pbase) & ((win == 0) | (p0 > plast - win));
      if (!all) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kp = key_at(c0, at.ok, 16 * u + 4 * g + i);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) sc[u][ct][i] = sees(pcol[ct], kp) ? sc[u][ct][i] : -INFINITY;
          }
      }
      u4v bh[CT], bl[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        if (ct > 0 && !wide) continue;
        const f4 s0 = sc[0][ct], s1 = sc[1][ct];
        const float cm = maxn(maxn(maxn(s0[0], s0[1]), maxn(s0[2], s0[3])), maxn(maxn(s1[0], s1[1]), maxn(s1[2], s1[3])));
        if (__any(cm * A.scale > m[ct])) {             // a lane's own scores; the column's maximum only where it matters
          const float mn = fmaxf(m[ct], max4rows(cm + 0.f) * A.scale), al = __builtin_amdgcn_exp2f(m[ct] - mn);
          m[ct] = mn;
          lsum[ct] *= al;
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[ct][j] *= al;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int u = k >> 1, i = 2 * (k & 1);
          const float pa = __builtin_amdgcn_exp2f(fmaf(sc[u][ct][i], A.scale, -m[ct]));
          const float pb = __builtin_amdgcn_exp2f(fmaf(sc[u][ct][i + 1], A.scale, -m[ct]));
          lsum[ct] += pa + pb;
          bh[ct][k] = bfpk(pa, pb);
          bl[ct][k] = bfpk(pa - __uint_as_float(bh[ct][k] << 16), pb - __uint_as_float(bh[ct][k] & 0xFFFF0000u));
        }
      }
      if (more) vm_wait<8>(); else vm_wait<0>();       // V is there, the next K under way
      // V^T: lane (g, n) gives 4 values of row 4 g + n / 4 from dim 16 j + 4 (n % 4) on
      uint16_t* vw = Vs.r[w];
      const int vrow = 4 * g + (n >> 2);
      // A weight of 0 does not take out an infinity or NaN. Where a chunk has a mask, its values are looked over: the largest
      // exponent of each half, all ones in infinities and NaN.
      if (!all && !odd && nq > 1) {
        typedef unsigned short us2 __attribute__((ext_vector_type(2)));
        us2 z = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const u4v x = *reinterpret_cast<const u4v*>(vw + 512 * i + 8 * lane);
#pragma unroll
          for (int k = 0; k < 4; ++k) z = __builtin_elementwise_max(z, __builtin_bit_cast(us2, x[k] & 0x7F807F80u));
        }
        odd = __any((z.x == 0x7F80) | (z.y == 0x7F80));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int o = vrow * 128 + 8 * ((2 * j + ((n & 3) >> 1)) ^ (2 * (vrow & 7))) + 4 * (n & 1);
        const s4 t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)&vw[o]);
        const s4 t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)&vw[o + 16 * 128]);
        const u4v av = {__builtin_bit_cast(uint32_t, __builtin_shufflevector(t0, t0, 0, 1)),
                        __builtin_bit_cast(uint32_t, __builtin_shufflevector(t0, t0, 2, 3)),
                        __builtin_bit_cast(uint32_t, __builtin_shufflevector(t1, t1, 0, 1)),
                        __builtin_bit_cast(uint32_t, __builtin_shufflevector(t1, t1, 2, 3))};
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          if (ct > 0 && !wide) continue;
          acc[ct][j] = mfma_bf(as_b8(av), as_b8(bh[ct]), acc[ct][j]);
          acc[ct][j] = mfma_bf(as_b8(av), as_b8(bl[ct]), acc[ct][j]);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // V is read
      // the register loads are waited for here, before loads that a later wait would include
      asm volatile("" ::"v"(rp.c[0]), "v"(rp.c[1]), "v"(rp.s[0]), "v"(rp.s[1]), "v"(pgn) : "memory");
      if (more) {
        load_v(nx.v);
        vm_wait<8>();
      }
      at = nx;
    }
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) lsum[ct] = sum4rows(lsum[ct]);
  bool any = odd;
  if constexpr (NW > 1) {
    float (*O)[16][XROW] = reinterpret_cast<float (*)[16][XROW]>(Ks.r[0]);   // the other waves' accumulators, scaled alike
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
      if (g == 0) { L.m[w][16 * ct + n] = m[ct]; L.l[w][16 * ct + n] = lsum[ct]; }
    L.odd[w] = odd;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      if (ct > 0 && !wide) break;                      // uniform
      __syncthreads();                                 // the chunks, and the last column tile's join, are done
      if (ct == 0)
        for (int k = 0; k < NW; ++k) any |= L.odd[k] != 0;
      float M = NEG_BIG, l = 0.f;
      for (int k = 0; k < NW; ++k) M = fmaxf(M, L.m[k][16 * ct + n]);
      for (int k = 0; k < NW; ++k) l += L.l[k][16 * ct + n] * __builtin_amdgcn_exp2f(L.m[k][16 * ct + n] - M);
      const float f = __builtin_amdgcn_exp2f(m[ct] - M);
      m[ct] = M;
      lsum[ct] = l;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[ct][j] *= f;
        if (w > 0) *reinterpret_cast<f4*>(&O[w - 1][n][16 * j + 4 * g]) = acc[ct][j];
      }
      __syncthreads();
      if (w == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          for (int k = 0; k < NW - 1; ++k) acc[ct][j] += *reinterpret_cast<const f4*>(&O[k][n][16 * j + 4 * g]);
      }
    }
    if (w > 0) return any;
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int qi = 4 * ct + (n >> 2);
    if (qi >= nq) continue;
    if (DIRECT) {
      const float inv = lsum[ct] > 0.f ? 1.0f / lsum[ct] : 0.f;
      uint16_t* o = A.out + ((t.t0 + t.q0 + qa + qi) * 16 + 4 * h + (n & 3)) * 128 + 4 * g;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const f4 a = acc[ct][j];
        *reinterpret_cast<uint2*>(o + 16 * j) = make_uint2(bfpk(a[0] * inv, a[1] * inv), bfpk(a[2] * inv, a[3] * inv));
      }
    } else {
      const int64_t col = ((A.G + A.I + it) * 4 + h) * NC + 4 * (qa + qi) + (n & 3);
      if (g == 0) { A.mo[col] = m[ct]; A.lo[col] = lsum[ct]; }
#pragma unroll
      for (int j = 0; j < 8; ++j) *reinterpret_cast<f4*>(A.ao + col * 128 + 16 * j + 4 * g) = acc[ct][j];
    }
  }
  return any;
}

template <int CT, int NW, bool DIRECT>
__device__ __forceinline__ void exact_part(ChunkXRows<NW>& Ks, ChunkXRows<NW>& Vs, ChunkXLds<CT, NW>& L, const ChunkArgs& A,
                                           const unsigned wg) {
  const int64_t it = wg >> 2;
  Tile t;
  if (!find_tile<4 * CT>(A, it, t)) return;
  for (int k = -1; k < t.nq; ++k) {                    // all queries, or after them one by one
    const bool odd = exact_tile<CT, NW, DIRECT>(Ks, Vs, L, A, t, it, wg & 3, max(k, 0), k < 0 ? t.nq : 1);
    if (k < 0 && !odd) return;                         // uniform
    __syncthreads();
  }
}
template <int CT, int NW, bool DIRECT>
__global__ void __launch_bounds__(64 * NW, 2) chunk_exact_kernel(ChunkArgs A) {
  __shared__ ChunkXRows<NW> Ks, Vs;                    // two objects: a read of one is not held for the other's loads
  __shared__ ChunkXLds<CT, NW> L;
  if (DIRECT && (int64_t)blockIdx.x == 4 * A.I) {      // the padding's output rows
    const int64_t e0 = min(A.qsl[A.R], A.T) * 256;
    for (int64_t i = e0 + threadIdx.x; i < A.T * 256; i += 64 * NW) reinterpret_cast<u4v*>(A.out)[i] = u4v{0u, 0u, 0u, 0u};
    return;
  }
  exact_part<CT, NW, DIRECT>(Ks, Vs, L, A, blockIdx.x);
}
// Both in one launch: three of four waves per (tile, KV head), whose LDS (48 KB) lets two workgroups stay on a CU beside the tables.
// The exact part's workgroups come first while the quantized ones have up to three entries each, for they are the longer
// chain then; behind them they fill the end. In us, exact first / last: 1 row x 5 tokens at 16384 (half an entry) 23.5 / 26.9,
// 16 x 8 at 4096 (1.9) 37.8 / 40.6, 32 x 8 at 4096 (3.8) 52.3 / 47.5, 16 x 8 at 16384 (7.9) 64.9 / 60.6, 16 x 33 at 16384 173 / 166.
constexpr int BNW = 3;
union ChunkBoth { ChunkStage s; ChunkXRows<BNW> x; };
template <int CT>
__global__ void __launch_bounds__(256, 2) chunk_both_kernel(ChunkArgs A) {
  __shared__ ChunkQLds L;
  __shared__ ChunkBoth a, b;
  __shared__ ChunkXLds<CT, BNW> X;
  const unsigned nx = 4 * (unsigned)A.I, nq = (unsigned)A.G, wg = blockIdx.x, q0 = A.xfirst ? nx : 0;
  if (wg - q0 < nq)
    quant_part<CT>(L, a.s, b.s, A, wg - q0);
  else if (threadIdx.x < 64 * BNW)
    exact_part<CT, BNW, false>(a.x, b.x, X, A, A.xfirst ? wg : wg - nq);
}

// ---------------------------------------------------------------- merge
__device__ __forceinline__ float wave_sum(float x) {
  x += dpp<0xB1>(x); x += dpp<0x4E>(x); x += dpp<0x141>(x); x += dpp<0x140>(x);
  return sum4rows(x);
}
// Walsh-Hadamard transform over the 64 lanes: lanes 1, 2, 4 (7 apart, then 3), 8 apart by DPP; 16 and 32 apart by swaps,
// which return the lower lane's value first
__device__ __forceinline__ float lane_hadamard(float x) {
  const int lane = threadIdx.x & 63;
  float p;
  p = dpp<0xB1>(x); x = lane & 1 ? p - x : x + p;
  p = dpp<0x4E>(x); x = lane & 2 ? p - x : x + p;
  p = dpp<0x1B>(dpp<0x141>(x)); x = lane & 4 ? p - x : x + p;
  p = dpp<0x128>(x); x = lane & 8 ? p - x : x + p;
  float2 r = rows16(x);
  x = lane & 16 ? r.x - r.y : r.x + r.y;
  r = halves32(x);
  return lane & 32 ? r.x - r.y : r.x + r.y;
}
// WPC waves per (token, query head), the four heads of a KV head (WPC = 1) or one head (8) per workgroup: 8 for few tokens,
// whose partials are many (the whole call with 8 / 1: 1 x 16384 x 5 tokens 23.2 / 37.9 us, 8 x 16384 x 4 36.8 / 38.2, 8 x 16384 x 8
// 48.8 / 48.0, 16 x 1024 x 8 29.5 / 25.4). Lanes take the partials' m and l side by side, then the wave adds up the partials'
// accumulators, lane = dims 2 lane, 2 lane + 1, eight loads in flight.
template <int CT, int WPC>
__global__ void __launch_bounds__(WPC == 1 ? 256 : 64 * WPC) chunk_merge_kernel(ChunkArgs A) {
  constexpr int QT = 4 * CT, NC = 16 * CT;
  __shared__ float jm[WPC], jl[WPC], jx[WPC][128];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, dd = 2 * lane;
  const int64_t tok = blockIdx.x / (WPC == 1 ? 4 : 16);
  const int q = WPC == 1 ? 4 * (int)(blockIdx.x & 3) + w : (int)(blockIdx.x & 15), h = q >> 2;
  const int part = WPC == 1 ? 0 : w;                   // this wave's share of the partials
  uint32_t* dst = reinterpret_cast<uint32_t*>(A.out + (tok * 16 + q) * 128 + dd);
  if (tok >= min(A.qsl[A.R], A.T)) {                   // padding
    if (part == 0) *dst = 0u;
    return;
  }
  const int64_t row = row_of(A.qsl, A.R, tok), i = tok - A.qsl[row];
  const int64_t it = tile_number<QT>(A.qsl, A.T, row) + i / QT;
  const int c = 4 * (int)(i % QT) + (q & 3);
  const unsigned C = A.pre[A.R], nu = 4 * row_blocks(A, row);
  const unsigned s = A.pre[row] + (unsigned)i / QT * nu, e = s + nu;   // the tile's entries of the list
  const unsigned w0 = nu ? s / C : 0;
  const int n = nu ? (int)((e - 1) / C - w0) + 1 : 0;            // partials of the quantized list
  const bool mid = nu && w0 * C < s;                             // the first of them starts inside its workgroup's range
  auto slot = [&](int k) { return ((k == 0 && mid ? A.G + it : w0 + k) * 4 + h) * NC + c; };
  const int64_t cx = ((A.G + A.I + it) * 4 + h) * NC + c;
  const float mx = A.mo[cx], lx = A.lo[cx];
  const float2 ax = *reinterpret_cast<const float2*>(A.ao + cx * 128 + dd);
  float M = mx, l = 0.f, x0 = 0.f, x1 = 0.f;
  const int share = WPC == 1 ? 64 : min(64, max(8, (n + WPC - 1) / WPC));   // partials of a wave at a time
  for (int k0 = share * part; k0 < n; k0 += share * WPC) {
    const int kn = min(share, n - k0);
    const bool in = lane < kn;
    const int64_t p = slot(in ? k0 + lane : 0);
    const float mk = in ? A.mo[p] : NEG_BIG, lk = in ? A.lo[p] : 0.f;
    const float m2 = fmaxf(wave_max(mk), M);
    const float al = __builtin_amdgcn_exp2f(M - m2), f = __builtin_amdgcn_exp2f(mk - m2);
    M = m2;
    l = l * al + f * lk;                               // the lane's own share; M starts at the exact part's m
    x0 *= al;
    x1 *= al;
    for (int k = 0; k < kn; k += 8) {
      float2 a[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = *reinterpret_cast<const float2*>(A.ao + slot(k0 + min(k + j, kn - 1)) * 128 + dd);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float fk = k + j < kn ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), min(k + j, 63))) : 0.f;
        x0 += fk * a[j].x;
        x1 += fk * a[j].y;
      }
    }
  }
  l = wave_sum(l);
  if constexpr (WPC > 1) {                             // the waves' shares, in wave order
    if (lane == 0) { jm[w] = M; jl[w] = l; }
    *reinterpret_cast<float2*>(&jx[w][dd]) = make_float2(x0, x1);
    __syncthreads();
    if (w > 0) return;
    float m2 = M;
    for (int k = 1; k < WPC; ++k) m2 = fmaxf(m2, jm[k]);
    l = x0 = x1 = 0.f;
    for (int k = 0; k < WPC; ++k) {
      const float f = __builtin_amdgcn_exp2f(jm[k] - m2);
      l += f * jl[k];
      x0 += f * jx[k][dd];
      x1 += f * jx[k][dd + 1];
    }
    M = m2;
  }
  const float fx = __builtin_amdgcn_exp2f(mx - M);
  l += fx * lx;
  {                                                    // H x: bit 0 of the dim in the lane, bits 1..6 across the lanes
    const float a = x0, b = x1;
    x0 = a + b;
    x1 = a - b;
  }
  x0 = lane_hadamard(x0);
  x1 = lane_hadamard(x1);
  const float hn = __uint_as_float(0x3DB504F3u);       // 1 / sqrt(128)
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  *dst = bfpk((x0 * hn + fx * ax.x) * inv, (x1 * hn + fx * ax.y) * inv);
}

// Queries per tile: 4 (one MFMA column tile) while the rows bring up to 4 tokens on average, else 8, whose keys are unpacked once
// for twice the queries. All kernels, us in tiles of 4 / 8: 16 rows x 4096 with 4 tokens each 29.8 / 30.8, with 5 35.4 / 37.1; 32 x
// 16384 72.4 / 71.6, 117 / 88; 64 x 8192 79.4 / 76.7, 121 / 93; 192 x 4096 with 2, 4, 5, 8 102 / 109, 115 / 119, 181 / 145, 192 /
// 179. Ragged rows about the border, 1 .. 5, 7, 8 tokens: 16 x 4096 24.2 / 30.0, 33.4 / 33.1, 36.0 / 34.7; 32 x 16384 81 / 76, 88 / 81,
// 100 / 86; 192 x 4096 120 / 123, 128 / 128, 148 / 137: of tiles of 8, those of up to 4 queries take one column tile.
// Layers without sub-blocks: 4 only while every row brings one token; their kernel passes over an empty second half
// (window, 398 rows x 5: 66 us in tiles of 4, 55 in tiles of 8).
int chunk_ct(int64_t R, int64_t T, bool quant) { return T <= (quant ? 4 * R : R) ? 1 : 2; }

int64_t chunk_cus() {
  static std::mutex mu;
  static int64_t cache[64] = {0};
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) { (void)hipGetLastError(); return 256; }
  std::lock_guard<std::mutex> lock(mu);
  if (cache[dev] == 0) {
    int cu = 0;
    if (hipDeviceGetAttribute(&cu, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cu <= 0) {
      (void)hipGetLastError();
      cu = 256;
    }
    cache[dev] = cu;
  }
  return cache[dev];
}

struct ChunkPlan { int ct; bool both; int64_t G, I, cols, pre; };   // cols: partial columns; pre: entries
ChunkPlan chunk_plan(int64_t R, int64_t T, int64_t nqmax) {
  ChunkPlan p;
  p.ct = chunk_ct(R, T, nqmax > 0);
  p.I = R + T / (4 * p.ct);
  // One launch for both parts, except where tiles of 4 have long lists: alone, their quantized part has three workgroups on a
  // CU instead of two. In us, one launch / two: 1 row x 5 at 16K tokens 25 / 35, 16 x 8 at 4K 39 / 45, 128 x 8 at 16K 266 / 270;
  // tiles of 4: 1 x 1 at 4K 19 / 25, 64 x 1 at 1K 26 / 34, 64 x 4 at 4K 53 / 53, 32 x 4 at 16K 71 / 70, 64 x 4 at 16K 117 / 106.
  p.both = nqmax > 0 && (p.ct == 2 || R * nqmax <= 8 * chunk_cus());
  p.G = nqmax > 0 ? chunk_cus() * (p.both ? 2 : 3) : 0;   // what is resident: 256 registers and 68 KB, or 168 and 39 KB
  p.cols = nqmax > 0 ? (p.G + 2 * p.I) * 64 * p.ct : 0;
  p.pre = nqmax > 0 ? (R + 4) / 4 * 4 : 0;
  return p;
}

template <int CT, int NW, bool DIRECT>
int chunk_exact(const ChunkArgs& A, hipStream_t s) {
  hipLaunchKernelGGL((chunk_exact_kernel<CT, NW, DIRECT>), dim3((unsigned)(4 * A.I + DIRECT)), dim3(64 * NW), 0, s, A);
  return check_launch("chunk_exact");
}
// Waves per (tile, KV head): as many as are resident at once (66, 33 and 16 KB of LDS), by the workgroups, of which those
// without a tile leave soon. In us with 4 / 2 / 1 waves, window layers: 64 rows x 5 tokens (416 workgroups) 16.8 / 19.2 / 23.5,
// 64 x 16 (768) 29.1 / 21.8 / 25.1, 128 x 1 (640) 18.4 / 15.8 / 16.6, 256 x 5 (1,664) 43.5 / 38.8 / 32.0.
template <int CT, bool DIRECT>
int chunk_exact_all(const ChunkArgs& A, hipStream_t s) {
  const int64_t cu = chunk_cus(), wgs = 4 * A.I;
  return wgs <= 2 * cu ? chunk_exact<CT, 4, DIRECT>(A, s)
                       : wgs <= 4 * cu ? chunk_exact<CT, 2, DIRECT>(A, s) : chunk_exact<CT, 1, DIRECT>(A, s);
}
template <int CT>
int chunk_launch(const ChunkArgs& A, bool quant, bool both, hipStream_t s) {
  if (!quant) return chunk_exact_all<CT, true>(A, s);
  int rc = KV800_OK;
  if (both) {
    hipLaunchKernelGGL(chunk_both_kernel<CT>, dim3((unsigned)(4 * A.I + A.G)), dim3(256), 0, s, A);
    rc = check_launch("chunk_both");
  } else if constexpr (CT == 1) {
    hipLaunchKernelGGL(chunk_quant_kernel, dim3((unsigned)A.G), dim3(256), 0, s, A);
    rc = check_launch("chunk_quant");
    if (rc == KV800_OK) rc = chunk_exact_all<1, false>(A, s);
  }
  if (rc != KV800_OK) return rc;
  if (8 * A.T <= chunk_cus())
    hipLaunchKernelGGL((chunk_merge_kernel<CT, 8>), dim3((unsigned)(16 * A.T)), dim3(64 * 8), 0, s, A);
  else
    hipLaunchKernelGGL((chunk_merge_kernel<CT, 1>), dim3((unsigned)(4 * A.T)), dim3(256), 0, s, A);
  return check_launch("chunk_merge");
}

}  // namespace
}  // namespace kv800

using namespace kv800;

extern "C" {

int64_t kv800_hip_decode_chunk_workspace(int64_t R, int64_t T, int64_t nqmax) {
  if (R <= 0 || T <= 0 || nqmax <= 0) return 0;
  const ChunkPlan p = chunk_plan(R, T, nqmax);
  return p.pre * 4 + p.cols * 130 * 4;
}

int kv800_hip_decode_chunk(const kv800_paged_t* P, const uint16_t* q, const int64_t* qsl, int64_t R, int64_t T,
                           const uint16_t* cos_t, const uint16_t* sin_t, int64_t rope_rows, const uint32_t* cs2,
                           int64_t qpool_bytes, int64_t epool_elems, int64_t sink_elems, uint16_t* out, void* ws,
                           int64_t ws_bytes, void* stream) {
  KV800_REQUIRE(P, "decode_chunk: null pointer");
  return kv800_hip_decode_chunk_sized(P, P->boff_stride, P->eoff_stride, q, qsl, R, T, cos_t, sin_t, rope_rows, cs2, qpool_bytes,
                                      epool_elems, sink_elems, out, ws, ws_bytes, stream);
}

int kv800_hip_decode_chunk_sized(const kv800_paged_t* P, int64_t boff_cols, int64_t eoff_cols, const uint16_t* q, const int64_t* qsl,
                                 int64_t R, int64_t T, const uint16_t* cos_t, const uint16_t* sin_t, int64_t rope_rows,
                                 const uint32_t* cs2, int64_t qpool_bytes, int64_t epool_elems, int64_t sink_elems, uint16_t* out,
                                 void* ws, int64_t ws_bytes, void* stream) {
  KV800_REQUIRE(P && R >= 0 && T >= 0 && (R > 0 || T == 0), "decode_chunk: bad row or token count");
  if (T == 0) return KV800_OK;
  KV800_REQUIRE(q && qsl && out && P->epool && P->eoff && P->N, "decode_chunk: null pointer");
  KV800_REQUIRE(P->ebs > 0 && eoff_cols > 0 && P->eoff_stride >= 0 && P->win >= 0 && P->win < (1LL << 31) && P->nqmax >= 0,
                "decode_chunk: bad page geometry, window or nqmax");
  KV800_REQUIRE(P->e_hs % 8 == 0 && P->e_ts % 8 == 0 && P->e_v % 8 == 0 && P->e_ts < (1LL << 31) &&
                    P->e_ts > -(1LL << 31),
                "decode_chunk: strides must be multiples of 8 elements, the token stride below 2^31");
  KV800_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)P->epool) % 16 == 0, "decode_chunk: q, out and epool must be 16-byte aligned");
  KV800_REQUIRE((cos_t == nullptr) == (sin_t == nullptr), "decode_chunk: cos and sin tables go together");
  KV800_REQUIRE(!cos_t || ((((uintptr_t)cos_t | (uintptr_t)sin_t) % 16) == 0 && rope_rows > 0),
                "decode_chunk: rope tables must be 16-byte aligned and not empty");
  const bool quant = P->win == 0 && P->nqmax > 0;
  if (quant)
    KV800_REQUIRE(P->qpool && P->boff && boff_cols > 0 && P->boff_stride >= 0 && P->NQ && cos_t && cs2 && qpool_bytes >= SUB && (uintptr_t)cs2 % 16 == 0 &&
                      (uintptr_t)P->qpool % 16 == 0,
                  "decode_chunk: quantized layers need NQ, the quant pool (16-byte aligned, one sub-block at least), its offsets and the rope tables");
  KV800_REQUIRE(!quant || rope_rows < (1LL << 24), "decode_chunk: rope tables of 2^24 rows or more are not addressed");   // 128 bytes a row of cs2
  const bool sinks = P->win > 0 && P->sk;
  KV800_REQUIRE(!sinks || (P->sv && P->skoff && P->svoff && (((uintptr_t)P->sk | (uintptr_t)P->sv) % 16) == 0),
                "decode_chunk: sinks need sv, skoff, svoff and 16-byte aligned buffers");
  const ChunkPlan p = chunk_plan(R, T, quant ? P->nqmax : 0);
  KV800_REQUIRE(p.I <= (1LL << 28) && T <= (1LL << 28) && P->ebs < (1LL << 30) && eoff_cols < (1LL << 32), "decode_chunk: too many rows, tokens or pages");
  KV800_REQUIRE(!quant || p.I <= (int64_t)0x7F000000 / 4 / P->nqmax, "decode_chunk: too many rows and sub-blocks");
  KV800_REQUIRE(!quant || (ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= kv800_hip_decode_chunk_workspace(R, T, P->nqmax)),
                "decode_chunk: the workspace is too small or not 16-byte aligned");
  ChunkArgs A;
  A.P = *P;
  A.q = q; A.qsl = qsl; A.R = R; A.T = T;
  A.cos_t = cos_t; A.sin_t = sin_t; A.cs2 = cs2;
  A.rope_rows = rope_rows; A.qpool_bytes = qpool_bytes; A.epool_elems = epool_elems; A.sink_elems = sink_elems;
  A.P.nqmax = quant ? min(min(P->nqmax, boff_cols), rope_rows / BLK) : 0;   // of the kernels; the plan goes by the caller's
  A.G = p.G; A.I = p.I;
  A.pre = reinterpret_cast<int32_t*>(ws);
  A.ao = quant ? reinterpret_cast<float*>(A.pre + p.pre) : nullptr;
  A.mo = quant ? A.ao + p.cols * 128 : nullptr;
  A.lo = quant ? A.mo + p.cols : nullptr;
  A.out = out;
  A.scale = 1.4426950408889634f * 0.08838834764831845f;
  A.nsink = sinks ? NSINK : 0;
  const int64_t pages = min(eoff_cols * P->ebs, (int64_t)0x7FFFFFFF - 4096);   // the chunks asked for ahead stay below 2^31
  A.held = (int)(cos_t ? min(pages, rope_rows) : pages);
  A.xfirst = 4 * P->nqmax * max(R, T / (4 * p.ct)) <= 3 * p.G;
  const hipStream_t s = (hipStream_t)stream;
  return p.ct == 1 ? chunk_launch<1>(A, quant, p.both, s) : chunk_launch<2>(A, quant, p.both, s);
}

}  // extern "C"
