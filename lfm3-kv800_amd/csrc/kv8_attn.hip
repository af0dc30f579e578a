// kv8_attn.hip -- attention over the paged 8-bit cache (include/kv8_hip.h), gfx950.
//
//   attend_kernel      softmax(scale q . k) v of a step's tokens, a list of (query tile, KV head, positions) in equal shares
//   merge_kernel       joins what several workgroups have of one (query tile, KV head)
//   prompt_kernel      the same for many new tokens a row: tiles of 128 (query, query head), each block's values once through LDS
//   merge_rows_kernel  joins what several workgroups have of one (token, head)
//
// With m the running maximum of a query's scores, l the sum of its weights and o that of the weighted values, a step of keys is
//   m' = max(m, max s),  p = 2^(s - m'),  l' = 2^(m - m') l + sum p,  o' = 2^(m - m') o + p V;  o / l at the end,
// in log2 units; parts of a row join by the same rule. All of m, l and o are fp32.
//
// Both products run on the bf16 matrix instruction: a code times its power of two is exact in bf16, two codes an instruction, so
// that scores are those of the held keys in fp32 and a weight is rounded to 8 bits once, in the product and in l alike (count below).
// Error against 64 bits 0.00173 on 1 x 16384, 0.00175 with a window of 256, where a 32-bit form rounded to bf16 has 0.00172 and 0.00167
// (l of weights not rounded and whole maxima: 0.0024, 0.0024). The fp8 instructions with block scales
// would take the codes as they are, but drop products below about 2^-13 of the largest one of a sum: next to a strong channel,
// scores of 300 were 0.02 off.
// Operands of 16 x 16 x 32 (lane l: row or column l % 16, g = l / 16): k = 8 g + j. Output: column l % 16, rows 4 g + i. Scores are
// taken transposed (keys x queries): with the keys of a tile in the cache's slot order the lane's scores are those of the 16
// tokens 16 g .. of a block, in order, and the lane reads the values of the same: weights never leave their lane.
#include <cfloat>
#include <type_traits>

#include "kv8_common.h"
#include "kv800_attn.h"

namespace kv8 {
namespace {

using kv800::f4;

constexpr int GROUP = 16;             // query heads a KV head may have
constexpr float LAZY = 8.f;           // log2 units by which a prompt's running maximum may lag: the top weight is then rounded, too (2
                                      // prompts of 1,500: error 0.00184, 0.00176 without a lag; of 8,192: 558 us, 568)

struct Desc {                         // of a workgroup whose last item others finish: where that item's outputs go
  int token, queries, head, last;     // first token, its queries, KV head, last workgroup; last -1: none
};
struct Attend {
  Cache C;
  const uint16_t* q;
  const int32_t* bt;
  int64_t bt_stride;
  int bt_cols;
  const int64_t* lens;
  const int64_t* qsl;
  int R;
  int64_t T;
  int G, TQ;                          // query heads per KV head, queries per tile of 16 or 32 columns (query, query head)
  int64_t window;
  int shift;                          // log2 of the positions of a wave's step
  float sl2;                          // |scale| log2(e)
  uint32_t flip;                      // sign bits of two bf16 for a negative scale: q changes its sign
  uint16_t* out;
  float* part;                        // 2 slots per workgroup of a tile's parts: of an item that others began, of one that others finish
  Desc* desc;                         // one per workgroup
};

// What is the same for a whole wave and not written by the kernel: through the scalar cache, so that its arrival is not waited for in
// the order of the vector loads.
template <typename T>
__device__ __forceinline__ T scalar_load(const T* p) { return *(const __attribute__((address_space(4))) T*)p; }
__device__ __forceinline__ int64_t same(int64_t x) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) | (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}
// the exponent bytes of keys and values at p (an even address): the low and high byte. The load is of the aligned word around them, two
// bytes of which may lie before the first or behind the last pair of exps (the header says so).
__device__ __forceinline__ uint32_t exps_load(const uint8_t* p) {
  const uintptr_t a = (uintptr_t)p;
  return scalar_load((const uint32_t*)(a & ~(uintptr_t)3)) >> (8 * (a & 2));
}

struct Row {
  int64_t q0, p0, n;                  // first token, its position, positions (those the table covers)
  int64_t b0;                         // first block that its first query sees
  int c, tiles, steps;                // new tokens, query tiles, steps from that block on
};
__device__ __forceinline__ Row row_at(const Attend& A, int r) {
  Row w;
  w.q0 = max(A.qsl[r], (int64_t)0);
  const int64_t q1 = A.qsl[r + 1], n = A.lens[r];
  w.c = (int)max(min(q1, A.T) - w.q0, (int64_t)0);
  w.p0 = n - max(q1 - w.q0, (int64_t)0);   // of tokens past T too, which are not there
  w.n = max(min(n, (int64_t)A.bt_cols * A.C.blocks * BLK), (int64_t)0);
  w.tiles = (w.c + A.TQ - 1) / A.TQ;
  const int64_t lo = A.window > 0 ? max(w.p0 + 1 - A.window, (int64_t)0) : 0;
  w.b0 = min(lo, w.n) / BLK;
  w.steps = max((int)((w.n - w.b0 * BLK + (1 << A.shift) - 1) >> A.shift), 1);   // 1 also without keys: the outputs are written
  return w;
}
// The same with r and all results in scalar registers.
__device__ __forceinline__ Row uniform_row(const Attend& A, int r) {
  Row w = row_at(A, r);
  w.q0 = same(w.q0); w.p0 = same(w.p0); w.n = same(w.n); w.b0 = same(w.b0);
  w.c = __builtin_amdgcn_readfirstlane(w.c); w.tiles = __builtin_amdgcn_readfirstlane(w.tiles); w.steps = __builtin_amdgcn_readfirstlane(w.steps);
  return w;
}
__device__ __forceinline__ int64_t cost_of(const Attend& A, const Row& w) { return (int64_t)w.tiles * A.C.heads * w.steps; }

// Prefix sums of what the rows count for: pre[i] of those before thread i's `per` rows, pre[256] all.
struct List {
  int64_t pre[257];
  int64_t wave[4];
};
template <typename F>
__device__ __forceinline__ void scan_rows(const Attend& A, List& L, int per, F cost) {
  const int tid = threadIdx.x;
  int64_t s = 0;
  for (int r = tid * per; r < min((tid + 1) * per, A.R); ++r) s += cost(row_at(A, r));
  int64_t x = s;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(x, o);
    if ((tid & 63) >= o) x += y;
  }
  if ((tid & 63) == 63) L.wave[tid >> 6] = x;
  __syncthreads();
  int64_t before = 0;
  for (int w = 0; w < (tid >> 6); ++w) before += L.wave[w];
  L.pre[tid + 1] = before + x;
  if (tid == 0) L.pre[0] = 0;
  __syncthreads();
}
// Row that holds number x of what was summed, and the sum before that row.
template <typename F>
__device__ __forceinline__ int find_row(const Attend& A, const List& L, int per, int64_t x, int64_t& before, F cost) {
  int lo = 0, hi = 256;
  while (hi - lo > 1) {
    const int m = (lo + hi) / 2;
    if (L.pre[m] <= x) lo = m;
    else hi = m;
  }
  int r = lo * per;
  before = L.pre[lo];
  for (; r + 1 < A.R; ++r) {
    const int64_t c = cost(row_at(A, r));
    if (x < before + c) break;
    before += c;
  }
  return r;
}

// 1 in each byte of w that is a NaN code (0x7F, 0xFF)
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7; }
// eight codes in bf16, times the power of two f; exact
__device__ __forceinline__ kv800::b8 wide8(uint32_t a, uint32_t b, float f) {
  const kv800::bf2 x[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, f, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, f, true),
                    __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, f, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, f, true)};
  return kv800::b8{x[0][0], x[0][1], x[1][0], x[1][1], x[2][0], x[2][1], x[3][0], x[3][1]};
}

// two bf16 of a query, their signs flipped for a negative scale; an infinity becomes NaN, since no softmax has scores that are infinite,
// while a maximum of minus infinity means that no key was seen
__device__ __forceinline__ uint32_t query(uint32_t u, uint32_t flip) {
  return (u ^ flip) | (((u & 0x7F807F80u) + 0x00800080u) & 0x80008000u) >> 9;
}
__device__ __forceinline__ kv800::u4v query(uint4 u, uint32_t flip) {
  return kv800::u4v{query(u.x, flip), query(u.y, flip), query(u.z, flip), query(u.w, flip)};
}

// sum + the two rounded weights of w: what the values are multiplied by is what the sum counts, so that equal values come back as they
// are and a dominant weight's rounding cancels
__device__ __forceinline__ float count(uint32_t w, float sum) {
  const kv800::bf2 ones = {(__bf16)1.f, (__bf16)1.f};
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(kv800::bf2, w), ones, sum, false);
}

// Zeros for the tokens behind the last row's, by all workgroups.
template <int D>
__device__ __forceinline__ void clear_padding(const Attend& A) {
  for (int64_t t = max(A.qsl[A.R], (int64_t)0) + blockIdx.x; t < A.T; t += gridDim.x)
    for (int i = threadIdx.x; i < A.C.heads * A.G * D / 8; i += blockDim.x)
      reinterpret_cast<uint4*>(A.out + t * A.C.heads * A.G * D)[i] = make_uint4(0, 0, 0, 0);
}

// A part of one column: D sums of weighted values, the maximum (log2 units), the sum of weights, relative to it; PART floats.
template <int D>
constexpr int PART = D + 4;

// LIST: one workgroup takes its share of the W entries of the list (row, query tile, head, step); else workgroup w is one
// (query tile, head), found by the tiles' numbers: row r's begin at (qsl[r] + r (TQ - 1)) / TQ, which leaves none out for rows of one
// token. The four waves take every fourth step of an item, each with its own maximum, sum and output, and are joined in LDS.
// Bound: HBM for large batches (32 rows of 32,768 188 us: 5.7 TB/s of
// the cache), else the chain lengths - table - page - codes - join, 8 us, and the merge.
// NB, NC: blocks of 64 positions a step, column tiles. A list by steps of 128 positions (1 x 32768 18.5 us, by 64 22.5; 8 x 4096 20.2,
// 17.8); with 32 columns by 64, for the registers.
template <int D, bool LIST, int NB, int NC>
__global__ void __launch_bounds__(256, NB * NC == 1 ? 3 : 2) attend_kernel(Attend A, int per) {
  constexpr int STEP = NB * BLK, COLS = 16 * NC;   // positions of a wave's step; columns of a tile
  constexpr int NT = D / 16, NK = D / 32, LD = D + 4;
  __shared__ typename std::conditional<LIST, List, int>::type L;
  __shared__ __align__(16) float so[4][COLS][LD];
  __shared__ float sm[4][COLS], sl[4][COLS];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), rr = lane & 15, g = lane >> 4;
  const int64_t w = blockIdx.x;

  clear_padding<D>(A);

  int64_t x = 0, end = 1, before = 0, W = 0, NG = 1, share = 1;
  int r, tile0 = 0;
  Row row;
  if constexpr (LIST) {
    if (tid == 0) A.desc[w].last = -1;
    const auto cost = [&](const Row& w) { return cost_of(A, w); };
    int64_t incl = 0;                              // up to 64 rows: every wave for itself, lane r the sum to row r
    if (A.R <= 64) {
      incl = lane < A.R ? cost(row_at(A, lane)) : 0;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(incl, o);
        if (lane >= o) incl += y;
      }
      W = __shfl(incl, 63);
    } else {
      scan_rows(A, L, per, cost);
      W = L.pre[256];
    }
    W = same(W);
    if (W == 0) return;                            // no row has tokens
    // Up to 4 entries each, which run at once: as many for each, so that most items begin with a workgroup (1 x 16384, 4 tokens: 17.2 us,
    // 20.8 in proportion); else in proportion, no two differing by more than one (16 x 4096, 8 tokens: 25.4, 29.2 with as many for each).
    NG = min((int64_t)gridDim.x, W);
    share = W <= 4 * (int64_t)gridDim.x ? (W + gridDim.x - 1) / gridDim.x : 0;
    x = share ? w * share : w * W / NG;
    if (w >= NG || x >= W) return;                 // no workgroup between two others is without entries
    end = share ? min(x + share, W) : (w + 1) * W / NG;
    if (A.R <= 64) {
      r = __popcll(__ballot(incl <= x));
      before = r ? __shfl(incl, r - 1) : 0;
    } else {
      r = find_row(A, L, per, x, before, cost);
    }
    r = __builtin_amdgcn_readfirstlane(r);
    before = same(before);
    x = same(x);
    end = same(end);
    row = uniform_row(A, r);
  } else {
    const int64_t ti = (uint32_t)w / (uint32_t)A.C.heads;
    const auto from = [&](int64_t i) { return (A.qsl[i] + i * (A.TQ - 1)) / A.TQ; };
    r = (int)min(ti, (int64_t)A.R - 1);            // so it is where every row before has one tile
    if (from(r) > ti || (r + 1 < A.R && from(r + 1) <= ti)) r = (int)kv800::last_at(A.R, [&](int64_t i) { return from(i) <= ti; });
    r = __builtin_amdgcn_readfirstlane(r);
    row = uniform_row(A, r);
    tile0 = (int)((row.q0 + (int64_t)r * (A.TQ - 1)) / A.TQ);
    if (ti - tile0 >= row.tiles) return;
  }
  while (x < end) {
    int64_t at = 0;
    int s0 = 0, s1 = row.steps, h, tile;
    if constexpr (LIST) {
      while (x >= before + cost_of(A, row)) {
        before += cost_of(A, row);
        row = uniform_row(A, ++r);
      }
      const int64_t item = (x - before) / row.steps;
      at = before + item * row.steps;
      s0 = (int)(x - at);
      s1 = (int)min((int64_t)row.steps, end - at);
      h = (int)(item % A.C.heads);
      tile = (int)(item / A.C.heads);
    } else {
      h = (int)((uint32_t)w % (uint32_t)A.C.heads);
      tile = (int)((uint32_t)w / (uint32_t)A.C.heads) - tile0;
    }

    // ---- the queries of the lane's columns
    int64_t qp[NC], qlo[NC];     // the query sees positions (qlo, qp]
    kv800::b8 qr[NC][NK];        // dims 16 g .. of the lower and (D = 128) upper 64, 8 an instruction
    f4 o[NC][NT];
    float M[NC], l[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int c = 16 * n + rr, i = tile * A.TQ + c / A.G, hq = h * A.G + c % A.G;
      const bool have = c < A.TQ * A.G && i < row.c;
      qp[n] = row.p0 + i;
      qlo[n] = A.window > 0 ? qp[n] - A.window : -1;
#pragma unroll
      for (int e = 0; e < NK; ++e) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (have) u = *reinterpret_cast<const uint4*>(A.q + ((row.q0 + i) * A.C.heads * A.G + hq) * D + (e >> 1) * 64 + 16 * g + 8 * (e & 1));
        qr[n][e] = kv800::as_b8(query(u, A.flip));
      }
#pragma unroll
      for (int d = 0; d < NT; ++d) o[n][d] = f4{0.f, 0.f, 0.f, 0.f};
      M[n] = -INFINITY;
      l[n] = 0.f;
    }

    // positions that some query of the tile sees, (tlo, thi], and those that all of them see, [alo, ahi)
    const int ilast = min(row.c, (tile + 1) * A.TQ) - 1;
    const int64_t thi = min(row.p0 + ilast, row.n - 1), tlo = A.window > 0 ? row.p0 + tile * A.TQ - A.window : -1;
    const int64_t ahi = min(row.p0 + tile * A.TQ + 1, row.n), alo = A.window > 0 ? row.p0 + ilast - A.window + 1 : 0;

    for (int st = s0 + wv; st < s1; st += 4) {
      const int64_t pos = row.b0 * BLK + (int64_t)st * STEP;
      if (pos > thi || pos + STEP <= tlo + 1) continue;
      // ---- codes of the step's blocks; a block that no query sees, or without a page, is not read
      uint4 kk[4 * NB][D / 64], vv[NT][NB];
      float sc[NB][2];
      bool on[NB];
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        const int64_t bp = pos + u * BLK;
        on[u] = bp <= thi && bp + BLK > tlo + 1;                           // then below 2^31, which a division in 64 bits is too long for
        const uint32_t bi = (uint32_t)(bp / BLK), col = bi / (uint32_t)A.C.blocks;
        on[u] = on[u] && col < (uint32_t)A.bt_cols;
        int64_t page = 0;
        if (on[u]) {
          page = scalar_load(A.bt + (int64_t)r * A.bt_stride + col);
          on[u] = page >= 0 && page < A.C.pages;
        }
        if (on[u]) {
          const int ub = (int)(bi - col * (uint32_t)A.C.blocks);
          const uint8_t* base = block_of<D>(A.C, page, h, ub);
          const uint32_t ex = exps_load(exps_of(A.C, page, h, ub));
          sc[u][0] = pow2(held_exponent((uint8_t)ex));
          sc[u][1] = pow2(held_exponent((uint8_t)(ex >> 8)));
#pragma unroll
          for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int e = 0; e < D / 64; ++e)
              kk[4 * u + a][e] = *reinterpret_cast<const uint4*>(base + ((4 * e + g) * BLK + 16 * a + rr) * 16);
#pragma unroll
          for (int d = 0; d < NT; ++d) vv[d][u] = *reinterpret_cast<const uint4*>(base + BLK * D + (g * D + 16 * d + rr) * 16);
        } else {
          sc[u][0] = sc[u][1] = 1.f;
#pragma unroll
          for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int e = 0; e < D / 64; ++e) kk[4 * u + a][e] = make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int d = 0; d < NT; ++d) vv[d][u] = make_uint4(0, 0, 0, 0);
        }
      }
      // ---- scores of the lane's columns: tile a holds tokens 64 (a / 4) + 16 g + 4 (a % 4) + j
      float s[NC][16 * NB];
#pragma unroll
      for (int a = 0; a < 4 * NB; ++a) {
        f4 c[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) c[n] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < D / 64; ++e) {
          const kv800::b8 k0 = wide8(kk[a][e].x, kk[a][e].y, sc[a >> 2][0]), k1 = wide8(kk[a][e].z, kk[a][e].w, sc[a >> 2][0]);
#pragma unroll
          for (int n = 0; n < NC; ++n) c[n] = kv800::mfma_bf(k1, qr[n][2 * e + 1], kv800::mfma_bf(k0, qr[n][2 * e], c[n]));
        }
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[n][4 * a + j] = c[n][j] * A.sl2;
      }
      const bool edge = pos < alo || pos + STEP > ahi || !on[0] || !on[NB - 1];
      uint32_t pw[NC][8 * NB];
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        if (edge) {        // tokens of the step that the column's query sees: [lo, hi)
          int lo = (int)min(max(qlo[n] + 1 - pos, (int64_t)0), (int64_t)STEP), hi = (int)min(max(min(qp[n] + 1, row.n) - pos, (int64_t)0), (int64_t)STEP);
          if (!on[0]) lo = max(lo, BLK);
          if (!on[NB - 1]) hi = min(hi, STEP - BLK);
          const int see0 = lo - 16 * g;
          const uint32_t seen = (uint32_t)max(hi - lo, 0);
#pragma unroll
          for (int a = 0; a < 4 * NB; ++a)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if ((uint32_t)(64 * (a >> 2) + 4 * (a & 3) + j - see0) >= seen) s[n][4 * a + j] = -INFINITY;
        }
        float mt = s[n][0];
#pragma unroll
        for (int j = 1; j < 16 * NB; ++j) mt = fmaxf(mt, s[n][j]);
        mt = kv800::max4rows(mt);
        const float Mn = fmaxf(M[n], mt);
        if (__any(Mn > M[n])) {
          const float alpha = Mn > M[n] ? __builtin_amdgcn_exp2f(M[n] - Mn) : 1.f;    // M = -inf: 0
          l[n] *= alpha;
#pragma unroll
          for (int d = 0; d < NT; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[n][d][j] *= alpha;
          M[n] = Mn;
        }
        // ---- weights
        const float M0 = M[n] > -INFINITY ? M[n] : 0.f;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8 * NB; ++j) {
          const float p0 = __builtin_amdgcn_exp2f(s[n][2 * j] - M0), p1 = __builtin_amdgcn_exp2f(s[n][2 * j + 1] - M0);
          pw[n][j] = kv800::bfpk(p0, p1);
          sum = count(pw[n][j], sum);
        }
        if (__any(sum != sum)) {   // a column whose every key so far is NaN has no maximum, yet its sum counts
          if (kv800::max4rows(sum != sum ? 1.f : 0.f) > 0.f && M[n] == -INFINITY) M[n] = 0.f;
        }
        l[n] += sum;
      }
      // ---- in a step with a mask, codes that not every query sees: a weight of 0 does not take out a NaN
      bool poison = false;
      if (edge) {
        uint32_t top = 0;  // bit 7 of a byte: some value there is a NaN code
        auto look = [&](const uint4& x) {
          top |= ((x.x & 0x7F7F7F7Fu) + 0x01010101u) | ((x.y & 0x7F7F7F7Fu) + 0x01010101u);
          top |= ((x.z & 0x7F7F7F7Fu) + 0x01010101u) | ((x.w & 0x7F7F7F7Fu) + 0x01010101u);
        };
#pragma unroll
        for (int d = 0; d < NT; ++d)
#pragma unroll
          for (int u = 0; u < NB; ++u) look(vv[d][u]);
        poison = __any((top & 0x80808080u) != 0);
        if (poison) {
          auto clean = [&](uint32_t& x) { x &= ~(nan_bytes(x) * 255u); };
#pragma unroll
          for (int d = 0; d < NT; ++d)
#pragma unroll
            for (int u = 0; u < NB; ++u) { clean(vv[d][u].x); clean(vv[d][u].y); clean(vv[d][u].z); clean(vv[d][u].w); }
        }
      }
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        kv800::b8 pa[NC], pb[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          pa[n] = kv800::as_b8(kv800::u4v{pw[n][8 * u], pw[n][8 * u + 1], pw[n][8 * u + 2], pw[n][8 * u + 3]});
          pb[n] = kv800::as_b8(kv800::u4v{pw[n][8 * u + 4], pw[n][8 * u + 5], pw[n][8 * u + 6], pw[n][8 * u + 7]});
        }
#pragma unroll
        for (int d = 0; d < NT; ++d) {
          const kv800::b8 v0 = wide8(vv[d][u].x, vv[d][u].y, sc[u][1]), v1 = wide8(vv[d][u].z, vv[d][u].w, sc[u][1]);
#pragma unroll
          for (int n = 0; n < NC; ++n) o[n][d] = kv800::mfma_bf(v1, pb[n], kv800::mfma_bf(v0, pa[n], o[n][d]));
        }
      }
      if (poison) {        // NaN values taken out above go to the queries that see them
        for (int t = 0; t < STEP; ++t) {
          const int64_t tp = pos + t;
          if (!on[t >> 6] || tp > thi) continue;
          const int64_t bi = tp / BLK;
          const uint8_t* base = block_of<D>(A.C, A.bt[(int64_t)r * A.bt_stride + bi / A.C.blocks], h, (int)(bi % A.C.blocks)) + BLK * D;
#pragma unroll
          for (int n = 0; n < NC; ++n)
            if (tp <= qp[n] && tp > qlo[n] && tp < row.n)
#pragma unroll
              for (int d = 0; d < NT; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  if ((base[((t >> 4 & 3) * D + 16 * d + 4 * g + j) * 16 + (t & 15)] & 0x7F) == 0x7F) o[n][d][j] = NAN;
        }
      }
    }
    // ---- the four waves' parts
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const float ls = kv800::sum4rows(l[n]);
      if (g == 0) { sm[wv][16 * n + rr] = M[n]; sl[wv][16 * n + rr] = ls; }
#pragma unroll
      for (int d = 0; d < NT; ++d) *reinterpret_cast<f4*>(&so[wv][16 * n + rr][16 * d + 4 * g]) = o[n][d];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int c = 16 * n + (tid >> 4), d0 = (tid & 15) * (D / 16);
      float m = sm[0][c];
#pragma unroll
      for (int k = 1; k < 4; ++k) m = fmaxf(m, sm[k][c]);
      float ls = 0.f, acc[D / 16];
#pragma unroll
      for (int e = 0; e < D / 16; ++e) acc[e] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = sm[k][c] > -INFINITY ? __builtin_amdgcn_exp2f(sm[k][c] - m) : 0.f;
        if (sm[k][c] > -INFINITY) {
          ls += f * sl[k][c];
#pragma unroll
          for (int e = 0; e < D / 16; ++e) acc[e] += f * so[k][c][d0 + e];
        }
      }
      if (s0 == 0 && s1 == row.steps) {
        const int ic = tile * A.TQ + c / A.G;
        if (c < A.TQ * A.G && ic < row.c) {
          const float inv = ls == 0.f ? 0.f : 1.f / ls;
          uint16_t* dst = A.out + ((row.q0 + ic) * A.C.heads * A.G + h * A.G + c % A.G) * D + d0;
          uint32_t y[D / 32];
#pragma unroll
          for (int e = 0; e < D / 32; ++e) y[e] = kv800::bfpk(acc[2 * e] * inv, acc[2 * e + 1] * inv);
          if (D == 128) *reinterpret_cast<uint4*>(dst) = make_uint4(y[0], y[1], y[D / 32 - 2], y[D / 32 - 1]);
          else *reinterpret_cast<uint2*>(dst) = make_uint2(y[0], y[1]);
        }
      } else {
        float* pt = A.part + ((2 * w + (s0 == 0 ? 1 : 0)) * COLS + c) * PART<D>;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) pt[d0 + e] = acc[e];
        if (d0 == 0) { pt[D] = m; pt[D + 1] = ls; }
        // the item's last workgroup; in proportion: the least w' with (w' + 1) W / NG at or behind its end
        if (s0 == 0 && tid == 0 && n == 0)
          A.desc[w] = {(int)row.q0 + tile * A.TQ, min(A.TQ, row.c - tile * A.TQ), h, (int)(share ? (at + row.steps - 1) / share : ((at + row.steps) * NG + W - 1) / W - 1)};
      }
    }
    if constexpr (!LIST) return;
    __syncthreads();
    x = at + s1;
  }
}

// ---------------------------------------------------------------- joining parts
// A wave joins `count` parts, 64 at a time: their maxima and factors side by side, then two parts a load, D / 32 channels a lane, 16
// parts on their way while the maxima are. The sums' order is that of the parts. Writes the column's output. (A part a load, 4 on
// their way: 1 x 65536 positions, 128 parts an item, 35.7 us the whole call, 27.0 so.)
template <int D, typename Slot>
__device__ __forceinline__ void join(int count, Slot slot, uint16_t* __restrict__ out) {
  constexpr int C = D / 32, AHEAD = 8;
  typedef float fc __attribute__((ext_vector_type(C)));
  const int lane = threadIdx.x & 63, half = lane >> 5, li = lane & 31;
  fc acc = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int k0 = 0; k0 < count; k0 += 64) {
    const int n = min(64, count - k0);
    fc v[AHEAD];
    auto load = [&](int j) {                       // behind the last part: that one again, times 0
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) v[i] = *reinterpret_cast<const fc*>(slot(k0 + min(j + 2 * i + half, n - 1)) + C * li);
    };
    const float2 ml = *reinterpret_cast<const float2*>(slot(k0 + min(lane, n - 1)) + D);
    load(0);
    float top = ml.x;
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    top = fmaxf(m, top);
    const float M0 = top > -INFINITY ? top : 0.f;  // no part has keys: all sums are 0
    const float f = lane < n ? __builtin_amdgcn_exp2f(ml.x - M0) : 0.f, old = __builtin_amdgcn_exp2f(m - M0);
    m = top;
    l = l * old + f * ml.y;
    acc *= old;
    for (int j = 0;;) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) acc += __shfl(f, j + 2 * i + half) * v[i];
      j += 2 * AHEAD;
      if (j >= n) break;
      load(j);
    }
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o);
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] += __shfl_xor(acc[c], 32);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint32_t y[C / 2];
#pragma unroll
  for (int c = 0; c < C / 2; ++c) y[c] = kv800::bfpk(acc[2 * c] * inv, acc[2 * c + 1] * inv);
  if (half) return;
  if (D == 128) reinterpret_cast<uint2*>(out)[li] = make_uint2(y[0], y[C / 2 - 1]);
  else reinterpret_cast<uint32_t*>(out)[li] = y[0];
}

// One wave per (workgroup of the list, column): where that workgroup began an item that others finish, its part and theirs.
template <int D, int NC>
__global__ void __launch_bounds__(256) merge_kernel(Attend A) {
  constexpr int COLS = 16 * NC;
  const int64_t w = blockIdx.x;
  const Desc d = A.desc[w];
  const int c = blockIdx.y * 4 + (threadIdx.x >> 6), i = c / A.G;
  asm volatile("" ::"s"(d.token), "s"(d.queries), "s"(d.head));          // all of it in one load
  if (d.last < 0 || i >= d.queries) return;
  const int Hq = A.C.heads * A.G;
  join<D>(d.last - (int)w + 1, [&](int k) { return A.part + ((2 * (w + k) + (k == 0 ? 1 : 0)) * COLS + c) * PART<D>; },
          A.out + ((int64_t)(d.token + i) * Hq + d.head * A.G + c % A.G) * D);
}

// One wave per (token, head) of the split prompt kernel.
template <int D>
__global__ void __launch_bounds__(256) merge_rows_kernel(const float* __restrict__ part, int splits, const int64_t* __restrict__ total, int heads,
                                                         int64_t T, uint16_t* __restrict__ out) {
  const int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (c >= min(*total, T) * heads) return;         // the padding has no parts
  join<D>(splits, [&](int k) { return part + (c * splits + k) * PART<D>; }, out + c * D);
}

// ---------------------------------------------------------------- many new tokens a row
typedef float f16v __attribute__((ext_vector_type(16)));
typedef __amdgpu_buffer_rsrc_t rsrc_t;
__device__ __forceinline__ f16v mfma32(kv800::u4v a, kv800::u4v b, f16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(kv800::as_b8(a), kv800::as_b8(b), c, 0, 0, 0);
}
__device__ __forceinline__ float halves_max(float x) {
  const float2 p = kv800::halves32(x);
  return fmaxf(p.x, p.y);
}

// One workgroup: NW waves of 32 columns ((query, query head) of one KV head), all over the same blocks of 64 tokens, which go
// through LDS in bf16, two buffers: the next block's codes, loaded a block earlier, are widened and stored while the present
// one is multiplied, one barrier a block. S^T = K Q^T and O^T += V^T P^T on 32 x 32 x 16 (lane l: row or column l % 32, k = 8 (l / 32) + j;
// output column l % 32, rows 8 b + 4 (l / 32) + i), so a column's weights and sums stay in its two lanes. Row 8 b + 4 h + i of
// key tile a is token 32 a + 16 (b / 2) + 8 h + 4 (b % 2) + i: the lane's weights are then those of 8 tokens side by side, half
// of a piece of the values. Two prompts of 8,192 tokens, 16 heads: 558 us, 1 PFLOP/s, bound by the issue of both vector and matrix
// instructions (46 and 44 % busy), of which two waves a SIMD overlap little.
template <int D, int NW>
__global__ void __launch_bounds__(64 * NW, 2) prompt_kernel(Attend A, int TQ, int per, int splits, float* __restrict__ part) {
  constexpr int NT = D / 32, NK = D / 16, NP = 4 * D / (64 * NW);          // dim tiles, k-steps, pieces of K (and V) a thread stages
  constexpr int KB = BLK * D * 2;                                          // bytes of a block's keys in bf16
  __shared__ __align__(16) uint8_t lds[2][2 * KB];
  __shared__ int flag[2];
  __shared__ List L;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, cl = lane & 31, hf = lane >> 5;
  const int H = A.C.heads, Hq = H * A.G;
  clear_padding<D>(A);
  // The rows' tiles side by side: idle workgroups are the last ones (at every other place they would leave half the chip's
  // engines without work: 64 rows of 32 tokens over 4K 165 us). Workgroup b runs on XCD b % 8: where the heads divide 8, an XCD has
  // one head and every (8 / heads)-th tile of it, so that its L2 holds one head's blocks; the last tiles first, which see the most.
  const auto tiles = [&](const Row& w) { return (int64_t)((w.c + TQ - 1) / TQ); };
  scan_rows(A, L, per, tiles);
  const int64_t ntiles = same(L.pre[256]);
  int64_t b = blockIdx.x;
  const int sp = (int)(b % splits);
  b /= splits;
  int h;
  int64_t ti;
  if (8 % H == 0 && splits == 1) {
    const int xs = 8 / H, x = (int)(b & 7);
    h = x / xs;
    ti = (b >> 3) * xs + x % xs;
  } else {
    h = (int)(b % H);
    ti = b / H;
  }
  if (ti >= ntiles) return;                                               // uniform, as every return
  ti = ntiles - 1 - ti;
  int64_t before;
  const int64_t r = same(find_row(A, L, per, ti, before, tiles));
  const Row row = uniform_row(A, (int)r);
  const int64_t tile = ti - same(before);
  const int i0 = (int)tile * TQ, ilast = min(row.c, i0 + TQ) - 1;         // queries [i0, ilast] of the row
  const int cc = wv * 32 + cl, iq = i0 + cc / A.G, hq = h * A.G + cc % A.G;
  const bool have = cc < TQ * A.G && iq <= ilast;
  const int64_t qp = row.p0 + iq, qlo = A.window > 0 ? qp - A.window : -1;

  kv800::u4v qr[NK];
#pragma unroll
  for (int s = 0; s < NK; ++s) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (have) u = *reinterpret_cast<const uint4*>(A.q + ((row.q0 + iq) * Hq + hq) * D + 16 * s + 8 * hf);
    qr[s] = query(u, A.flip);
  }
  // blocks that some query sees, and positions that all of them see
  const int64_t thi = min(row.p0 + ilast, row.n - 1), tlo = A.window > 0 ? max(row.p0 + i0 - A.window + 1, (int64_t)0) : 0;
  const int64_t ahi = min(row.p0 + i0 + 1, row.n), alo = A.window > 0 ? row.p0 + ilast - A.window + 1 : 0;
  int b0 = (int)(tlo / BLK), b1 = thi < tlo ? b0 : (int)(thi / BLK) + 1;
  {
    const int share = (b1 - b0 + splits - 1) / splits;
    b0 = min(b1, b0 + sp * share);
    b1 = min(b1, b0 + share);
  }

  // ---- staging: the codes of block bi into registers, later widened into LDS
  uint4 rk[NP], rv[NP];
  uint32_t re = 0;
  // Places of blocks are counted on, not divided for: the loop's scalar instructions stand between the wave's products (562 -> 550 us
  // for two prompts of 8,192).
  struct Place { int col, u; };  // table column, block of the page
  auto place = [&](int bi) { return Place{bi / A.C.blocks, bi % A.C.blocks}; };
  auto onward = [&](Place& x) {
    if (++x.u == A.C.blocks) { x.u = 0; ++x.col; }
  };
  const int32_t* table = A.bt + r * A.bt_stride;
  auto page_of = [&](const Place& x) { return scalar_load(table + min(x.col, A.bt_cols - 1)); };   // looked at a block later, when it has arrived
  auto valid = [&](int page, int bi) { return page >= 0 && page < A.C.pages && bi < b1; };
  auto load = [&](int bi, int page, int u) {
    if (valid(page, bi)) {
      const uint8_t* base = block_of<D>(A.C, page, h, u);
      const uint8_t* ex = exps_of(A.C, page, h, u);
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        rk[j] = *reinterpret_cast<const uint4*>(base + (tid + j * 64 * NW) * 16);
        rv[j] = *reinterpret_cast<const uint4*>(base + BLK * D + (tid + j * 64 * NW) * 16);
      }
      re = exps_load(ex);
    } else {
#pragma unroll
      for (int j = 0; j < NP; ++j) rk[j] = rv[j] = make_uint4(0, 0, 0, 0);
      re = 0;
    }
  };
  const int in0 = (int)min((max(alo, (int64_t)0) + BLK - 1) / BLK, (int64_t)INT32_MAX), in1 = (int)min(max(ahi, (int64_t)0) / BLK, (int64_t)INT32_MAX);
  auto is_edge = [&](int bi) { return bi < in0 || bi >= in1; };           // not every query sees all of the block
  auto store = [&](int bi, int buf) {
    if (is_edge(bi)) {      // a weight of 0 does not take out a NaN: NaN values leave the block, and are dealt out afterwards
      bool any = false;
      auto clean = [&](uint32_t& x) {
        const uint32_t nb = nan_bytes(x);
        any |= nb != 0;
        x &= ~(nb * 255u);
      };
#pragma unroll
      for (int j = 0; j < NP; ++j) { clean(rv[j].x); clean(rv[j].y); clean(rv[j].z); clean(rv[j].w); }
      if (any) flag[buf] = bi;
    }
    const float sk = pow2(held_exponent((uint8_t)re)), sv = pow2(held_exponent((uint8_t)(re >> 8)));
    uint8_t* kd = lds[buf];
    uint8_t* vd = lds[buf] + KB;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int p = tid + j * 64 * NW;
      const int dg = p >> 6, slot = p & 63, a4 = slot >> 4, g = (slot >> 2) & 3;
      const int at = 32 * (g >> 1) + 8 * (2 * (g & 1) + (a4 & 1)) + 4 * (a4 >> 1) + (slot & 3);
      *reinterpret_cast<kv800::b8*>(kd + ((dg * 2) * BLK + at) * 16) = wide8(rk[j].x, rk[j].y, sk);
      *reinterpret_cast<kv800::b8*>(kd + ((dg * 2 + 1) * BLK + at) * 16) = wide8(rk[j].z, rk[j].w, sk);
      const int tg = p / D, d = p % D;
      *reinterpret_cast<kv800::b8*>(vd + ((tg * 2) * D + d) * 16) = wide8(rv[j].x, rv[j].y, sv);
      *reinterpret_cast<kv800::b8*>(vd + ((tg * 2 + 1) * D + d) * 16) = wide8(rv[j].z, rv[j].w, sv);
    }
  };

  f16v o[NT];
#pragma unroll
  for (int d = 0; d < NT; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.f;
  float m = have ? -FLT_MAX : FLT_MAX, l = 0.f;   // columns without a query never ask for a rescale
  const float lazy = part || A.window > 0 ? 0.f : LAZY;

  if (tid < 2) flag[tid] = -1;
  int now = 0, next = 0, next2 = 0;               // pages of blocks bi, bi + 1, bi + 2
  if (b0 < b1) {                                   // then the table has columns
    now = page_of(place(b0));
    next = page_of(place(b0 + 1));
    next2 = page_of(place(b0 + 2));
    load(b0, now, place(b0).u);
  }
  __syncthreads();
  if (b0 < b1) {
    store(b0, b0 & 1);
    load(b0 + 1, next, place(b0 + 1).u);
  }
  __syncthreads();
  Place ahead = place(b0 + 3);
  int u2 = place(b0 + 2).u;                        // of block bi + 2
  for (int bi = b0; bi < b1; ++bi) {
    const int buf = bi & 1;
    const int after = page_of(ahead), u3 = ahead.u;
    onward(ahead);
    const bool held = valid(now, bi);
    {
      const uint8_t* kd = lds[buf] + (hf * BLK + cl) * 16;
      f16v s[2];
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const kv800::u4v x = *reinterpret_cast<const kv800::u4v*>(kd + (2 * k * BLK + 32 * a) * 16);
          const f16v zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          s[a] = mfma32(x, qr[k], k == 0 ? zero : s[a]);
        }
      store(bi + 1, buf ^ 1);
      load(bi + 2, next2, u2);
      u2 = u3;
      const bool edge = !held || is_edge(bi);
      if (edge) {
        // tokens of the block that the lane's query sees: [lo, hi)
        const int64_t bp = (int64_t)bi * BLK;
        const int lo = (int)min(max(qlo + 1 - bp, (int64_t)0), (int64_t)BLK), hi = held ? (int)min(max(min(qp + 1, row.n) - bp, (int64_t)0), (int64_t)BLK) : 0;
        const int see0 = lo - 8 * hf;
        const uint32_t seen = (uint32_t)max(hi - lo, 0);
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            if ((uint32_t)(32 * a + 16 * (v >> 3) + (v & 7) - see0) >= seen) s[a][v] = -INFINITY;
          }
      }
      float mt = -INFINITY;
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int v = 0; v < 16; v += 2) mt = fmaxf(fmaxf(mt, s[a][v]), s[a][v + 1]);
      mt = halves_max(mt) * A.sl2;
      if (__any(mt > m + lazy)) {
        const float mn = fmaxf(m, mt), alpha = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < NT; ++d) o[d] *= alpha;
      }
      // A weight is 2^(s sl2 - m) in one instruction, whose product is not rounded, while m is a rounded one: their difference, up to half
      // a step of m, is the same for all of the column's weights and goes out in o / l, but from scores of 2^31 on it passes what
      // exponents reach. Large scores go by the rounded products.
      float by = A.sl2, from = m;
      if (__any(fabsf(m) >= 0x1p20f && fabsf(m) < FLT_MAX)) {
#pragma clang fp contract(off)
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const float x = s[a][v] * A.sl2;
            s[a][v] = x - m;
          }
        by = 1.f;
        from = 0.f;
      }
      const uint8_t* vd = lds[buf] + KB + (hf * D + cl) * 16;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k >> 1][8 * (k & 1) + e], by, -from));
        const kv800::u4v pw = {kv800::bfpk(p[0], p[1]), kv800::bfpk(p[2], p[3]), kv800::bfpk(p[4], p[5]), kv800::bfpk(p[6], p[7])};
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = count(pw[e], sum);
#pragma unroll
        for (int d = 0; d < NT; ++d) {
          const kv800::u4v x = *reinterpret_cast<const kv800::u4v*>(vd + (2 * k * D + 32 * d) * 16);
          o[d] = mfma32(x, pw, o[d]);
        }
      }
      l += sum;
      if (edge && held && flag[buf] == bi) {
        const uint8_t* base = block_of<D>(A.C, now, h, bi % A.C.blocks) + BLK * D;
        for (int t = 0; t < BLK; ++t) {
          const int64_t tp = (int64_t)bi * BLK + t;
          if (tp <= qp && tp > qlo && tp < row.n)
#pragma unroll
            for (int d = 0; d < NT; ++d)
#pragma unroll
              for (int v = 0; v < 16; ++v)
                if ((base[((t >> 4) * D + 32 * d + 8 * (v >> 2) + 4 * hf + (v & 3)) * 16 + (t & 15)] & 0x7F) == 0x7F) o[d][v] = NAN;
        }
      }
    }
    now = next;
    next = next2;
    next2 = after;
    __syncthreads();
  }
  const float2 ls = kv800::halves32(l);
  l = ls.x + ls.y;
  if (!have) return;
  if (part) {
    float* pp = part + (((row.q0 + iq) * Hq + hq) * splits + sp) * PART<D>;
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<f4*>(pp + 32 * d + 8 * c + 4 * hf) = f4{o[d][4 * c], o[d][4 * c + 1], o[d][4 * c + 2], o[d][4 * c + 3]};
    if (hf == 0) { pp[D] = m; pp[D + 1] = l; }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* dst = A.out + ((row.q0 + iq) * Hq + hq) * D + 4 * hf;
#pragma unroll
  for (int d = 0; d < NT; ++d)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<uint2*>(dst + 32 * d + 8 * c) =
          make_uint2(kv800::bfpk(o[d][4 * c] * inv, o[d][4 * c + 1] * inv), kv800::bfpk(o[d][4 * c + 2] * inv, o[d][4 * c + 3] * inv));
}

// ---------------------------------------------------------------- host
// How a call runs. PROMPT: rows bring a third of a tile of the prompt kernel or more on average. DIRECT: few steps an item. A row that is
// not as the mean has it is right all the same.
enum Kind { LISTED, DIRECT, PROMPT };
struct Plan {
  Kind kind;
  int TQ, G, splits, step, cols;
  int64_t tiles, groups;              // query tiles of all rows at most; workgroups (LISTED)
  int64_t bytes;                      // workspace
};
constexpr int NW = 4;                 // waves of the prompt kernel
// Sizes whose sums and products stay in 64 bits below.
bool fits(const kv8_cache_t* c, int64_t heads, int64_t R, int64_t T, int64_t bt_cols) {
  return R <= INT32_MAX / 512 && T <= INT32_MAX / 512 && R * c->kv_heads < (1 << 24) && T * heads < (int64_t)1 << 32 &&
         bt_cols <= INT32_MAX / (c->blocks * BLK);
}
Plan plan(const kv8_cache_t* c, int64_t heads, int64_t R, int64_t T, int64_t bt_cols, int64_t window) {
  Plan p;
  p.G = (int)(heads / c->kv_heads);
  p.splits = 1;
  p.groups = 0;
  p.bytes = 0;
  const int64_t positions = bt_cols * c->blocks * BLK, mean = (T + R - 1) / R;
  const int64_t seen = window > 0 && window < positions - mean ? window + mean : positions;   // of a row, or so
  // Columns of a row and KV head, on average: the prompt kernel's tile has 128, the list's 16 or 32 (`wide`). Times, us, by tiles of 16, of
  // 32, and as prompts; 4 columns a token, 4 KV heads of 128:
  //   every row with the same tokens  columns 24          36             48             64             80
  //     1 x 16384                     17.3 23.2 19.7   22.7 20.4 20.7   22.7 21.5 21.5  18.1 23.6 22.5  25.6 26.1 23.2
  //     16 x 4096                     24.5 25.1 30.4   41.0 31.2 32.0   40.8 31.6 33.0  32.0 32.0 34.5  60.5 45.6 36.3
  //     64 x 4096                     86.3 56.1 106.6  131 90.2 107     131 90.6 108    160 92.0 108    208 137 109
  //     48 x 12000                    200 119 203      297 213 206      297 213 208     348 215 211     440 313 217
  //   rows with 1 to so many          up to 16            20               24               28               32
  //     5 x 3000                      19.4 20.6 18.3   18.7 21.6 18.5   25.5 23.9 21.4  26.4 21.2 22.0  21.5 24.1 21.4
  //     16 x 4097                     24.4 30.4 31.5   34.3 33.6 32.3   52.4 39.9 34.9  46.7 39.4 33.5  60.2 42.2 36.6
  //     32 x 4096                     58.4 48.5 49.8   66.8 52.5 51.0   81.2 59.0 53.7  98.4 70.7 57.1  98.3 71.1 56.9
  //     32 x 9000                     116 87.1 93.1    135 92.5 96.0    170 105 99.7    202 130 104     184 125 102
  // Uniform rows would go by tiles of 32 up to 64 columns; in steps whose rows differ, as a server's do, prompts draw level at a mean of 40
  // (up to 20 tokens) and are ahead behind it. Neither can be told from the other here.
  const int64_t cols = T * p.G / R, items = R * c->kv_heads;
  const bool wide = items * seen >= 1 << 19;
  // A workgroup an item without a list: short rows (1 x 1000 10.5 us, listed 14.9; 256 x 1000 51, 60), and of many rows with a token each
  // longer ones (40 x 1800 18, 23; 100 x 4000 76, 93; 100 x 8000 145, 164; 32 x 8000 58, 56.5). With more tokens a row some of the items'
  // numbers are idle workgroups: 128 x 4000 with 2 tokens 106, 102.5.
  p.kind = cols >= 40 ? PROMPT : seen <= (T <= R && items >= 128 ? 8192 : 1024) ? DIRECT : LISTED;
  p.cols = p.kind == PROMPT ? 32 * NW : p.kind == LISTED && wide && cols > 16 ? 32 : 16;
  p.TQ = p.cols / p.G;
  p.step = p.kind == LISTED && p.cols == 16 ? 2 * BLK : BLK;
  p.tiles = (T + R * (p.TQ - 1)) / p.TQ;
  if (p.kind == PROMPT) {
    // Few tiles: each split over its blocks, down to 4, for two workgroups a CU. Times, us, so / unsplit: 64 new tokens of one row of 16,384
    // 30 / 368, 24 of each of 16 of 4,096 38 / 103; 256 tiles, split in two, 45 / 32 (2 prompts of 1,024). Down to 8 blocks: one row of 2,048
    // 23.5, 19.4 down to 4.
    const int64_t wgs = (mean + p.TQ - 1) / p.TQ * R * c->kv_heads, most = seen / (4 * BLK);
    int64_t s = wgs > 0 && wgs < 256 ? 512 / wgs : 1;
    if (s > most) s = most;
    p.splits = (int)(s < 1 ? 1 : s);
    if (p.splits > 1) p.bytes = T * heads * p.splits * (c->dim + 4) * 4;
  } else if (p.kind == LISTED) {
    // One workgroup a CU, fewer rather than with less than 2 entries; two where all entries then run at once and the items are not so few
    // that each has many parts. Times, us, with up to 256 / 512: 1 x 65536 22.4 / 27.3, 64 x 4096 with 4 tokens 58 / 65, 32 x 32768 190 / 194;
    // 24 x 2500 23.4 / 19.7; 1 x 32768 18.8 / 22.3. Two also for many items, so that one's joins pass under the
    // other's steps: 128 x 2048 with 4 tokens 63.8 / 62.0, 192 rows of up to 32768 186.2 / 183.7.
    const int64_t entries = p.tiles * c->kv_heads * ((seen + p.step - 1) / p.step + (seen < positions ? 1 : 0));
    p.groups = entries <= 1024 ? (entries + 1) / 2 : entries < 2048 ? (entries + 3) / 4 : items > 256 ? 512 : 256;
    if (p.groups > 256 && items < 32) p.groups = 256;
    p.bytes = p.groups * (2 * p.cols * (c->dim + 4) * 4 + (int64_t)sizeof(Desc));
  }
  return p;
}

template <int D>
int run(const Attend& A0, const Plan& p, int64_t heads, void* ws, hipStream_t s) {
  Attend A = A0;
  const int64_t H = A.C.heads;
  if (p.kind == PROMPT) {
    const int64_t xs = 8 % H == 0 && p.splits == 1 ? 8 / H : 1;
    float* part = p.splits > 1 ? (float*)ws : nullptr;
    hipLaunchKernelGGL((prompt_kernel<D, NW>), dim3((unsigned)((p.tiles + xs - 1) / xs * xs * H * p.splits)), dim3(64 * NW), 0, s, A, p.TQ,
                       (A.R + 255) / 256, p.splits, part);
    if (part)
      hipLaunchKernelGGL(merge_rows_kernel<D>, dim3((unsigned)((A.T * heads + 3) / 4)), dim3(256), 0, s, part, p.splits, A.qsl + A.R,
                         (int)heads, A.T, A.out);
    return kv800::check_launch("kv8_attend prompt");
  }
  if (p.kind == DIRECT) {
    hipLaunchKernelGGL((attend_kernel<D, false, 1, 1>), dim3((unsigned)(p.tiles * H)), dim3(256), 0, s, A, 0);
    return kv800::check_launch("kv8_attend");
  }
  A.part = (float*)ws;
  A.desc = (Desc*)(A.part + p.groups * 2 * p.cols * PART<D>);
  const dim3 grid((unsigned)p.groups), mg((unsigned)p.groups, (unsigned)(p.cols / 4));
  const int per = (A.R + 255) / 256;
  if (p.cols == 32) hipLaunchKernelGGL((attend_kernel<D, true, 1, 2>), grid, dim3(256), 0, s, A, per);
  else hipLaunchKernelGGL((attend_kernel<D, true, 2, 1>), grid, dim3(256), 0, s, A, per);
  const int rc = kv800::check_launch("kv8_attend");
  if (rc != KV800_OK) return rc;
  if (p.cols == 32) hipLaunchKernelGGL((merge_kernel<D, 2>), mg, dim3(256), 0, s, A);
  else hipLaunchKernelGGL((merge_kernel<D, 1>), mg, dim3(256), 0, s, A);
  return kv800::check_launch("kv8_attend merge");
}

}  // namespace
}  // namespace kv8

extern "C" {

int64_t kv8_hip_attend_workspace(const kv8_cache_t* cache, int64_t heads, int64_t R, int64_t T, int64_t bt_cols, int64_t window) {
  if (!kv8::valid(cache) || heads <= 0 || heads % cache->kv_heads || heads / cache->kv_heads > kv8::GROUP || R <= 0 || T <= 0 || bt_cols < 0 ||
      window < 0 || !kv8::fits(cache, heads, R, T, bt_cols))
    return 0;
  return kv8::plan(cache, heads, R, T, bt_cols, window >= (int64_t)1 << 40 ? 0 : window).bytes;
}

int kv8_hip_attend(const kv8_cache_t* cache, const uint16_t* q, int64_t heads, const int32_t* bt, int64_t bt_stride,
                   int64_t bt_cols, const int64_t* lens, const int64_t* qsl, int64_t R, int64_t T, int64_t window,
                   float scale, uint16_t* out, void* ws, int64_t ws_bytes, void* stream) {
  KV800_REQUIRE(kv8::valid(cache), "kv8_attend: bad cache descriptor");
  KV800_REQUIRE(R >= 0 && T >= 0 && bt_cols >= 0 && bt_stride >= 0 && window >= 0, "kv8_attend: negative size");
  KV800_REQUIRE(heads > 0 && heads % cache->kv_heads == 0 && heads / cache->kv_heads <= kv8::GROUP,
                "kv8_attend: heads must be a multiple of the cache's, up to 16 times");
  KV800_REQUIRE(fabsf(scale) > 0.f && fabsf(scale) < INFINITY, "kv8_attend: scale must be finite and not 0");
  KV800_REQUIRE(bt_cols <= INT32_MAX / (cache->blocks * kv8::BLK), "kv8_attend: the table covers 2^31 positions or more");
  KV800_REQUIRE(kv8::fits(cache, heads, R, T, bt_cols), "kv8_attend: too many tokens or rows");
  if (T == 0) return KV800_OK;
  if (window >= (int64_t)1 << 40) window = 0;      // more than any row has; sums with positions stay in 64 bits
  KV800_REQUIRE(R > 0, "kv8_attend: tokens without rows");
  KV800_REQUIRE(q && lens && qsl && out && (bt || bt_cols == 0), "kv8_attend: null pointer");
  KV800_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0, "kv8_attend: q and out must be 16-byte aligned");
  const kv8::Plan p = kv8::plan(cache, heads, R, T, bt_cols, window);
  KV800_REQUIRE(p.tiles * cache->kv_heads * p.splits < (1 << 24) - 64, "kv8_attend: too many tokens or rows");   // 2^32 threads a launch
  KV800_REQUIRE(p.bytes == 0 || (ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= p.bytes), "kv8_attend: %lld bytes of 16-byte aligned workspace needed",
                (long long)p.bytes);
  const kv8::Attend A = {kv8::device_form(cache), q, bt, bt_stride, (int)bt_cols, lens, qsl, (int)R, T, p.G, p.TQ, window, p.step == 2 * kv8::BLK ? 7 : 6,
                         fabsf(scale) * 1.4426950408889634f, scale < 0.f ? 0x80008000u : 0u, out, nullptr, nullptr};
  return cache->dim == 128 ? kv8::run<128>(A, p, heads, ws, (hipStream_t)stream) : kv8::run<64>(A, p, heads, ws, (hipStream_t)stream);
}

}  // extern "C"
