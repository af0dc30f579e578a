// kv800_cache.hip -- per-step cache bookkeeping of the 800h path in vLLM's page geometry, for gfx950.
//
//   write_exact_kernel   the step's K / V rows into the exact pages through the slot mapping (vllm_attn.py:263-272),
//                        and, for tokens at positions < 4 of a window layer, into the sink aux area of the host
//                        layers' first quant page (vllm_attn.py:276-291).
//   step_tables_kernel   per row of the quant KV group: NQ = max(N - 128, 0) / 256 flushed sub-blocks and the byte
//                        offsets of its first nqmax sub-blocks in the quant pool, qbt[r, 256 j / bsq] * qs0 +
//                        (256 j % bsq) / 256 * 51200 (vllm_attn.py:332-340); optionally the sub-blocks flushed before
//                        the step's nnew tokens (the flush range's start, vllm_attn.py:297-317), the block table as
//                        int64 and the offsets of the sink aux areas (vllm_attn.py:276-291).
//   step_meta_kernel     per row of a decode step: the new token's slot, its position and the int32 length
//   chunk_meta_kernel    per new token of a step whose rows bring any number of them: slot, position and row, their prefix
//                        sums over the rows, and the pages that rows outgrow their block table by, from a list of free ones.
//   page_offsets_kernel  off[r, p] = bt[r, p] * scale + add: an exact group's block table as element offsets of its
//                        pages (the eoff table of the decode and flush kernels).
// All are plain data movement: one thread per 16-byte piece or per table entry, coalesced along the row.
#include "kv800_common.h"
#include "../../include/kv800_hip.h"

namespace kv800 {
namespace {

// thread -> (row r, piece): 4 heads x 128 dims = 64 pieces of 8 bf16 per K row and as many per V row
__global__ void __launch_bounds__(256)
write_exact_kernel(uint16_t* __restrict__ ep, int64_t s0, int64_t s1, int64_t s2, int64_t e_v, int64_t ebs,
                   const int64_t* __restrict__ slot, const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                   int64_t R, const int64_t* __restrict__ pos, uint16_t* __restrict__ skp, uint16_t* __restrict__ svp,
                   const int64_t* __restrict__ skoff, const int64_t* __restrict__ svoff, int nsink) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= R * 128) return;
  const int64_t r = i >> 7;
  const int piece = (int)(i & 127), isv = piece >> 6, h = (piece >> 4) & 3, d0 = 8 * (piece & 15);
  const uint4 x = *reinterpret_cast<const uint4*>((isv ? v : k) + (r * 4 + h) * 128 + d0);
  const int64_t sl = slot[r];
  if (sl >= 0) {   // slot < 0: padding token, not written (vllm_attn.py:265)
    const int64_t o = (sl / ebs) * s0 + h * s1 + (sl % ebs) * s2 + (isv ? e_v : 0) + d0;
    *reinterpret_cast<uint4*>(ep + o) = x;
  }
  if (nsink > 0 && pos[r] >= 0 && pos[r] < nsink) {   // sink rows of a window layer
    uint16_t* dst = isv ? svp : skp;
    const int64_t base = isv ? svoff[r] : skoff[r];
    *reinterpret_cast<uint4*>(dst + base + (pos[r] * 4 + h) * 128 + d0) = x;
  }
}

__global__ void __launch_bounds__(256)
step_tables_kernel(const int32_t* __restrict__ qbt, int64_t qbt_stride, int64_t bsq, int64_t qs0,
                   const int32_t* __restrict__ N, int64_t R, int64_t nqmax, int64_t nnew,
                   const int32_t* __restrict__ nnew_rows, int64_t* __restrict__ boff,
                   int32_t* __restrict__ NQ, int32_t* __restrict__ NP, int64_t* __restrict__ qbt64,
                   int64_t* __restrict__ aux, int64_t aux_scale, int64_t aux_add) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t w = max(max(nqmax, (int64_t)1), qbt64 ? qbt_stride : (int64_t)1);   // entries per row
  if (i >= R * w) return;
  const int64_t r = i / w, j = i % w;
  if (j == 0) {
    NQ[r] = max(N[r] - LAG, 0) / BLK;
    if (NP) NP[r] = max(N[r] - (nnew_rows ? max(nnew_rows[r], 0) : (int)nnew) - LAG, 0) / BLK;
    if (aux) aux[r] = (int64_t)qbt[r * qbt_stride] * aux_scale + aux_add;
  }
  if (j < nqmax) {
    const int64_t tok0 = j * BLK;
    boff[r * nqmax + j] = (int64_t)qbt[r * qbt_stride + tok0 / bsq] * qs0 + ((tok0 % bsq) / BLK) * SUB;
  }
  if (qbt64 && j < qbt_stride) qbt64[r * qbt_stride + j] = qbt[r * qbt_stride + j];
}

__global__ void __launch_bounds__(256)
page_offsets_kernel(const int32_t* __restrict__ bt, int64_t bt_stride, int64_t R, int64_t npages, int64_t scale,
                    int64_t add, int64_t* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= R * npages) return;
  const int64_t r = i / npages, p = i % npages;
  out[i] = (int64_t)bt[r * bt_stride + p] * scale + add;
}

// One decode step's slot, position and int32 length of row r (every row appends one token at position len - 1): the
// slot is the token's page bt[r, pos / ebs] times ebs plus pos % ebs; a row of length 0 gets slot and position -1
// (a padding token, which write_exact skips); a position past the row's npages pages gets slot -1 as well.
__global__ void __launch_bounds__(256)
step_meta_kernel(const int32_t* __restrict__ bt, int64_t bt_stride, int64_t npages, const int64_t* __restrict__ lens,
                 int64_t R, int64_t ebs, int64_t* __restrict__ slot, int64_t* __restrict__ pos,
                 int32_t* __restrict__ lens32) {
  const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= R) return;
  const int64_t n = lens[r], p = n - 1, pg = p >= 0 ? p / ebs : -1;
  slot[r] = (pg >= 0 && pg < npages) ? (int64_t)bt[r * bt_stride + pg] * ebs + p % ebs : -1;
  pos[r] = p >= 0 ? p : -1;
  lens32[r] = (int32_t)n;
}

// Slots, positions and rows of a step's new tokens, and the growth of the block tables, from the rows' lengths on the
// device. Row r has n = lens[r] positions of which c = min(max(qlens[r], 0), n) are new: its tokens are
// qsl[r] .. qsl[r] + c - 1 (qsl the exclusive prefix sum of c), token qsl[r] + i at position n - c + i. With `held` it
// takes max(0, ceil(n / ebs) - held[r]) further pages (as many as its table has room for), consecutive entries of the free
// list behind the earlier rows' ones.
// No workgroup waits for another: workgroup (x, y) takes the rows [256 x, 256 x + 256) and, of their tokens, every
// gridDim.y-th piece of 256. It sums the earlier rows' counts itself (12 bytes a row, from the L2) and scans its own in
// LDS; a token finds its row by 8 steps of a binary search there. Fresh table entries are read from the free list, not
// from the table, so the order in which workgroups write the table does not matter.
// Bound: launch and two dependent rounds of loads. 1 row: 3.4 us; 398 rows x 8 tokens
// with growth: 6.4 us (59 KB).
struct MetaArgs {
  int32_t* bt;
  int64_t bt_stride, npages;
  const int64_t* lens;
  const int32_t* qlens;
  int64_t R, ebs, tokens;
  const int32_t* held;      // null: no growth
  const int32_t* freep;
  int64_t nfree;
  const int64_t* taken;
  int32_t* held_out;
  int64_t* taken_out;
  int64_t *qsl, *slot, *pos, *row;
  int32_t* lens32;
};
constexpr int MROWS = 256;   // rows and threads per workgroup
__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// a row's length, new tokens and (with held) pages before the step and to add; everything is clamped to what is possible
struct MetaRow { int64_t n, c, have, add; };
__device__ __forceinline__ MetaRow meta_row(const MetaArgs& A, int64_t r) {
  MetaRow m;
  m.n = min(max(A.lens[r], (int64_t)0), (int64_t)0x7FFFFFFF);
  m.c = min(max((int64_t)A.qlens[r], (int64_t)0), m.n);
  m.have = A.npages;
  m.add = 0;
  if (A.held) {
    m.have = min(max((int64_t)A.held[r], (int64_t)0), A.npages);
    m.add = max(min((m.n + A.ebs - 1) / A.ebs, A.npages) - m.have, (int64_t)0);
  }
  return m;
}
__global__ void __launch_bounds__(MROWS) chunk_meta_kernel(MetaArgs A) {
  __shared__ int64_t first[MROWS + 1];                 // first token of each of the rows, and the next workgroup's
  __shared__ int64_t pos0[MROWS], page0[MROWS];        // position of a row's first token; its first fresh free-list entry
  __shared__ int32_t have[MROWS], all[MROWS];          // pages held before the step, and after it
  __shared__ int64_t wc[4], wa[4], bc[4], ba[4];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int64_t r0 = (int64_t)blockIdx.x * MROWS, r = r0 + tid;
  const bool last = blockIdx.x == gridDim.x - 1;
  int64_t ec = 0, ea = 0;                              // the earlier rows' tokens and fresh pages
  for (int64_t i = tid; i < r0; i += MROWS) {
    const MetaRow m = meta_row(A, i);
    ec += m.c;
    ea += m.add;
  }
  MetaRow m = {0, 0, 0, 0};
  if (r < A.R) m = meta_row(A, r);
  int64_t sc = m.c, sa = m.add;                        // inclusive scan over the wave
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t pc = __shfl_up(sc, o, 64), pa = __shfl_up(sa, o, 64);
    if (lane >= o) { sc += pc; sa += pa; }
  }
  ec = wave_sum64(ec);
  ea = wave_sum64(ea);
  if (lane == 63) { wc[w] = sc; wa[w] = sa; }
  if (lane == 0) { bc[w] = ec; ba[w] = ea; }
  __syncthreads();
  int64_t basec = bc[0] + bc[1] + bc[2] + bc[3], basea = ba[0] + ba[1] + ba[2] + ba[3];
  for (int k = 0; k < w; ++k) { basec += wc[k]; basea += wa[k]; }
  const int64_t f = basec + sc - m.c;                  // the row's first token
  const int64_t tk = A.held ? min(max(A.taken[0], (int64_t)0), A.nfree) : 0;
  const int64_t at = tk + basea + sa - m.add;          // its first fresh page in the free list
  const int64_t got = m.have + max(min(m.add, A.nfree - at), (int64_t)0);
  first[tid] = f;
  if (tid == MROWS - 1) first[MROWS] = f + m.c;
  pos0[tid] = m.n - m.c;
  page0[tid] = at - m.have;
  have[tid] = (int32_t)m.have;
  all[tid] = (int32_t)(A.held ? got : A.npages);
  if (blockIdx.y == 0 && r < A.R) {
    A.qsl[r] = min(f, A.tokens);
    A.lens32[r] = (int32_t)m.n;
    if (r == A.R - 1) A.qsl[A.R] = min(f + m.c, A.tokens);
    if (A.held) {
      A.held_out[r] = (int32_t)got;
      if (r == A.R - 1) A.taken_out[0] = min(at + m.add, A.nfree);
      for (int64_t p = m.have; p < got; ++p) A.bt[r * A.bt_stride + p] = A.freep[at + p - m.have];
    }
  }
  __syncthreads();
  // ---- the tokens of these rows; behind the last row's, the padding
  const int64_t end = min(first[MROWS], A.tokens), stop = last ? A.tokens : end;
  for (int64_t t = first[0] + (int64_t)blockIdx.y * MROWS + tid; t < stop; t += (int64_t)gridDim.y * MROWS) {
    int64_t sl = -1, ps = -1, rw = 0;
    if (t < end) {
      int lo = 0;                                      // the last row with first[row] <= t: it holds t
#pragma unroll
      for (int s = MROWS / 2; s > 0; s >>= 1)
        if (first[lo + s] <= t) lo += s;
      rw = r0 + lo;
      ps = pos0[lo] + (t - first[lo]);
      const int64_t pg = ps / A.ebs;
      int64_t page = -1;
      if (pg < have[lo]) page = A.bt[rw * A.bt_stride + pg];
      else if (pg < all[lo]) page = A.freep[page0[lo] + pg];
      if (page >= 0) sl = page * A.ebs + ps % A.ebs;
    }
    A.slot[t] = sl;
    A.pos[t] = ps;
    A.row[t] = rw;
  }
}

// Streaming-read probe (a measurement aid of bench.py, not part of the cache path): workgroup g reads the 16-byte
// units g * 2048 + tid + 256 k (k < 8) of the buffer and every gridDim.x * 2048 units after, xor-folds them and writes
// one word; with 8 loads in flight per lane and two workgroups per CU it reads at what the part sustains for
// plain (cached) loads.
typedef uint32_t pv4 __attribute__((ext_vector_type(4)));
__global__ void __launch_bounds__(256) read_probe_kernel(const pv4* __restrict__ p, int64_t n16,
                                                         uint32_t* __restrict__ out) {
  constexpr int U = 8;
  const int64_t stride = (int64_t)gridDim.x * 256 * U;
  pv4 acc = {0u, 0u, 0u, 0u};
  for (int64_t i = (int64_t)blockIdx.x * 256 * U + threadIdx.x; i < n16; i += stride) {
    pv4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = (i + 256 * u < n16) ? p[i + 256 * u] : pv4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int u = 0; u < U; ++u) acc ^= v[u];
  }
  __shared__ uint32_t red[256];
  red[threadIdx.x] = acc[0] ^ acc[1] ^ acc[2] ^ acc[3];
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t x = 0;
    for (int k = 0; k < 256; ++k) x ^= red[k];
    out[blockIdx.x] = x;
  }
}

}  // namespace
}  // namespace kv800

using namespace kv800;

extern "C" {

int kv800_hip_write_exact(uint16_t* epool, int64_t s0, int64_t s1, int64_t s2, int64_t e_v, int64_t ebs,
                          const int64_t* slot, const uint16_t* k, const uint16_t* v, int64_t R, const int64_t* pos,
                          uint16_t* sk, uint16_t* sv, const int64_t* skoff, const int64_t* svoff, void* stream) {
  KV800_REQUIRE(R >= 0, "write_exact: R < 0");
  if (R == 0) return KV800_OK;
  KV800_REQUIRE(epool && slot && k && v, "write_exact: null pointer");
  KV800_REQUIRE(ebs > 0 && s0 % 8 == 0 && s1 % 8 == 0 && s2 % 8 == 0 && e_v % 8 == 0,
                "write_exact: strides must be multiples of 8 elements and ebs > 0");
  KV800_REQUIRE(((uintptr_t)epool % 16) == 0 && ((uintptr_t)k % 16) == 0 && ((uintptr_t)v % 16) == 0,
                "write_exact: epool, k and v must be 16-byte aligned");
  const int nsink = sk ? NSINK : 0;
  KV800_REQUIRE(!nsink || (sv && pos && skoff && svoff && ((uintptr_t)sk % 16) == 0 && ((uintptr_t)sv % 16) == 0),
                "write_exact: sinks need sv, pos, skoff, svoff and 16-byte aligned sink buffers");
  KV800_REQUIRE(R * 128 <= 0x7FFFFFFFLL * 256, "write_exact: R too large");
  hipLaunchKernelGGL(write_exact_kernel, dim3((unsigned)((R * 128 + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                     epool, s0, s1, s2, e_v, ebs, slot, k, v, R, pos, sk, sv, skoff, svoff, nsink);
  return check_launch("write_exact");
}

int kv800_hip_step_tables(const int32_t* qbt, int64_t qbt_stride, int64_t bsq, int64_t qs0, const int32_t* N,
                          int64_t R, int64_t nqmax, int64_t nnew, const int32_t* nnew_rows, int64_t* boff,
                          int32_t* NQ, int32_t* NP, int64_t* qbt64, int64_t* aux, int64_t aux_scale, int64_t aux_add,
                          void* stream) {
  KV800_REQUIRE(R >= 0 && nqmax >= 0 && nnew >= 0, "step_tables: R, nqmax and nnew must be >= 0");
  if (R == 0) return KV800_OK;
  KV800_REQUIRE(N && NQ && (!nqmax || boff) && ((!nqmax && !qbt64 && !aux) || (qbt && qbt_stride > 0)),
                "step_tables: null pointer");
  KV800_REQUIRE(bsq > 0 && bsq % BLK == 0, "step_tables: bsq must be a positive multiple of 256");
  KV800_REQUIRE(!nqmax || (nqmax - 1) * BLK / bsq < qbt_stride, "step_tables: nqmax exceeds the quant block table");
  KV800_REQUIRE(nnew <= 0x7FFFFFFF, "step_tables: nnew too large");
  int64_t w = nqmax > 0 ? nqmax : 1;
  if (qbt64 && qbt_stride > w) w = qbt_stride;
  const int64_t n = R * w;
  KV800_REQUIRE(n <= 0x7FFFFFFFLL * 256, "step_tables: table too large");
  hipLaunchKernelGGL(step_tables_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, qbt,
                     qbt_stride, bsq, qs0, N, R, nqmax, nnew, nnew_rows, boff, NQ, NP, qbt64, aux, aux_scale,
                     aux_add);
  return check_launch("step_tables");
}

int kv800_hip_decode_tables(const int32_t* qbt, int64_t qbt_stride, int64_t bsq, int64_t qs0, const int32_t* N,
                            int64_t R, int64_t nqmax, int64_t* boff, int32_t* NQ, void* stream) {
  return kv800_hip_step_tables(qbt, qbt_stride, bsq, qs0, N, R, nqmax, 0, nullptr, boff, NQ, nullptr, nullptr, nullptr,
                               0, 0, stream);
}

int kv800_hip_page_offsets(const int32_t* bt, int64_t bt_stride, int64_t R, int64_t npages, int64_t scale, int64_t add,
                           int64_t* out, void* stream) {
  KV800_REQUIRE(R >= 0 && npages >= 0 && bt_stride >= npages, "page_offsets: need R, npages >= 0, bt_stride >= npages");
  if (R == 0 || npages == 0) return KV800_OK;
  KV800_REQUIRE(bt && out, "page_offsets: null pointer");
  const int64_t n = R * npages;
  KV800_REQUIRE(n <= 0x7FFFFFFFLL * 256, "page_offsets: table too large");
  hipLaunchKernelGGL(page_offsets_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, bt,
                     bt_stride, R, npages, scale, add, out);
  return check_launch("page_offsets");
}

int kv800_hip_step_meta(const int32_t* bt, int64_t bt_stride, int64_t npages, const int64_t* lens, int64_t R,
                        int64_t ebs, int64_t* slot, int64_t* pos, int32_t* lens32, void* stream) {
  KV800_REQUIRE(R >= 0 && ebs > 0 && npages >= 0 && bt_stride >= npages, "step_meta: need R >= 0, ebs > 0, "
                "bt_stride >= npages >= 0");
  if (R == 0) return KV800_OK;
  KV800_REQUIRE((bt || npages == 0) && lens && slot && pos && lens32, "step_meta: null pointer");
  hipLaunchKernelGGL(step_meta_kernel, dim3((unsigned)((R + 255) / 256)), dim3(256), 0, (hipStream_t)stream, bt,
                     bt_stride, npages, lens, R, ebs, slot, pos, lens32);
  return check_launch("step_meta");
}

int kv800_hip_chunk_meta(int32_t* bt, int64_t bt_stride, int64_t npages, const int64_t* lens, const int32_t* qlens,
                         int64_t R, int64_t ebs, int64_t tokens, const int32_t* held, const int32_t* free_pages,
                         int64_t nfree, const int64_t* taken, int32_t* held_out, int64_t* taken_out, int64_t* qsl,
                         int64_t* slot, int64_t* pos, int64_t* row, int32_t* lens32, void* stream) {
  KV800_REQUIRE(R >= 1 && ebs > 0 && npages >= 0 && npages <= 0x7FFFFFFF && bt_stride >= npages && tokens >= 0,
                "chunk_meta: need R >= 1, ebs > 0, bt_stride >= npages >= 0 and tokens >= 0");
  KV800_REQUIRE((bt || npages == 0) && lens && qlens && qsl && lens32 && (tokens == 0 || (slot && pos && row)),
                "chunk_meta: null pointer");
  KV800_REQUIRE(!held || (taken && held_out && taken_out && nfree >= 0 && (free_pages || nfree == 0)),
                "chunk_meta: a growing table needs the free list, taken, held_out and taken_out");
  KV800_REQUIRE(!held || (held != held_out && taken != taken_out), "chunk_meta: held and taken are not updated in place");
  const int64_t nb = (R + MROWS - 1) / MROWS;
  KV800_REQUIRE(nb <= 0x7FFFFFFF, "chunk_meta: R too large");
  const int64_t ny = (tokens + nb * 4 * MROWS - 1) / (nb * 4 * MROWS);   // about four tokens a thread
  const MetaArgs A = {bt, bt_stride, npages, lens, qlens, R, ebs, tokens, held, free_pages, held ? nfree : 0, taken,
                      held_out, taken_out, qsl, slot, pos, row, lens32};
  hipLaunchKernelGGL(chunk_meta_kernel, dim3((unsigned)nb, (unsigned)(ny < 1 ? 1 : ny > 256 ? 256 : ny)), dim3(MROWS), 0,
                     (hipStream_t)stream, A);
  return check_launch("chunk_meta");
}

int kv800_hip_capture_id(void* stream, uint64_t* id) {
  KV800_REQUIRE(id, "capture_id: null pointer");
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  unsigned long long n = 0;
  if (hipStreamGetCaptureInfo((hipStream_t)stream, &st, &n) != hipSuccess) {
    (void)hipGetLastError();
    kv800::set_error("capture_id: no such stream");
    return KV800_EHIP;
  }
  id[0] = st == hipStreamCaptureStatusActive ? n : 0;
  return KV800_OK;
}

int kv800_hip_read_probe(const void* buf, int64_t bytes, uint32_t* out, int64_t groups, void* stream) {
  KV800_REQUIRE(buf && out, "read_probe: null pointer");
  KV800_REQUIRE(bytes >= 16 && bytes % 16 == 0 && ((uintptr_t)buf % 16) == 0,
                "read_probe: bytes must be a positive multiple of 16 and buf 16-byte aligned");
  KV800_REQUIRE(groups >= 1 && groups <= 65536, "read_probe: groups must be in [1, 65536]");
  hipLaunchKernelGGL(read_probe_kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream,
                     reinterpret_cast<const pv4*>(buf), bytes / 16, out);
  return check_launch("read_probe");
}

}  // extern "C"
