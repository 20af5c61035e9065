// Losses of the vocabulary decoder with their gradients, the scores never kept:
//   z = h W^T + b       h [n, H] hidden rows, W [V, H] decoder weight, b [V] (CrossEntropyLoss over the LM head's scores,
//                       sentclf/bert_model.py:165,175-179; V 30 522, H 768 for BERT-base)
//   cross entropy       loss_i = lse(z_i) - z_i[y_i]                             dz_i = g_i (softmax(z_i) - onehot(y_i))
//   distillation        loss_i = T^2 sum_j p_ij (log p_ij - log q_ij)            dz_i = g_i T (q_i - p_i),  q_i = softmax(z_i / T)
//   gradients           dh = dz W,   dW = dz^T h,   db = sum_i dz_i
// Forward: one pass over W; every 128-column tile of scores lives in MFMA accumulators only and leaves one (max, sum of
// exp2) pair per row and 64 columns; a second kernel joins the pairs and forms the target scores as k dot products per row.
// Backward: the scores are formed once more, piece by piece of the vocabulary, and leave as the 16-bit operand
// G = c (softmax - targets) of two products, dh += G W and dW = G^T h.  G holds c = g_i / max|g|, |c| <= 1, so that fp16's
// range holds it (times 2^15 there: c q down to 2e-9 stays a normal number, and 2^-40 is its smallest half step: dh rows with c of 2^-20
// and more are as exact as the largest one's, V 30 522; the factor is common to all rows because dW sums over them); it is put back
// in fp32 when the products are stored.
// What G's rounding costs: most of a row's gradient sits in few entries (its targets), whose rounding errors do not average
// out.  dh gets them back in fp32: the residuals of a row's largest entries times their rows of W, added where the partials are
// joined.  dW of few rows (at most 64) is a product of G's high AND low parts, k twice as long under an output that is the
// bound; with more rows its errors average out like those of the operands, but where an entry's gradient comes from a row or two
// they are a second rounding beside the result's (4096 distilled rows: 2.3e-3 off, 1.7e-3 without G's rounding).
// Rows that take no part (ignored label, empty teacher list) are dropped first: the live rows are copied side by side, so
// their products cost nothing and whatever a dropped row holds (NaN included) reaches no gradient.
// Times below: one MI355X, V 30 522, H 768, bf16, unless said otherwise; the card copies at 4.7 TB/s and multiplies large
// matrices at 1.29 PF (2.5 is the matrix cores' peak).
#include <type_traits>

#include "vocab.h"

#define TRY(...)                           \
  do {                                     \
    hipError_t _e = (__VA_ARGS__);         \
    if (_e != hipSuccess) return _e;       \
  } while (0)

namespace {

// ---- LDS image of a K tile of one operand, R rows (of the output's M or N) by 64 k:
//   K-major (the operand is [R, K] in memory): [R][128 B], 16-byte chunks swizzled by swz128, read by ds_read_b128
//   R-major (the operand is [K, R] in memory): [64][2R B], 32-byte slots swizzled so that the 4 rows x 32 bytes that each
//     16-lane group of ds_read_b64_tr_b16 takes, and those of its neighbour group 8 rows on, fall into different banks
template <int R, bool TR, int NW>
struct Operand {
  static constexpr int BYTES = R * BK * 2, PIECES = BYTES / 1024 / NW;   // per wave
  static_assert(BYTES % (1024 * NW) == 0, "whole pieces per wave");
  u32x4_t rsrc;
  uint32_t off[PIECES], step;
  // base: the tile's first element; ld in elements; bytes: what may be read from base on
  __device__ __forceinline__ void init(const bf16_t* base, int64_t bytes, int64_t ld, int w, int lane) {
    rsrc = make_rsrc(base, bytes);
    step = TR ? (uint32_t)(BK * ld * 2) : BK * 2;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int at = (w * PIECES + p) * 1024 + lane * 16;   // byte of the image this lane fills
      if constexpr (TR) {
        const int k = at / (2 * R), c = (at % (2 * R)) >> 4;
        off[p] = (uint32_t)(k * ld * 2) + ((((c >> 1) ^ tr_swz<R>(k)) << 1) | (c & 1)) * 16;
      } else {
        const int r = at >> 7, c = (at >> 4) & 7;
        off[p] = (uint32_t)(r * ld * 2) + swz128(r, c) * 16;
      }
    }
  }
  // rows base[map[r]] (K-major); a row that is not there (-1) lies past the end: zeros.  bytes < 2^31
  __device__ __forceinline__ void init_rows(const bf16_t* base, int64_t bytes, int64_t ld, const int* map, int w, int lane) {
    rsrc = make_rsrc(base, bytes);
    step = BK * 2;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int at = (w * PIECES + p) * 1024 + lane * 16, r = at >> 7, from = map[r];
      off[p] = from < 0 ? 0x80000000u : (uint32_t)(from * ld * 2) + swz128(r, (at >> 4) & 7) * 16;
    }
  }
  __device__ __forceinline__ void stage(uint32_t kt, uint32_t lds, int w) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) dma16(rsrc, off[p] + kt * step, lds + (w * PIECES + p) * 1024);
  }
  // MFMA operand of 16 rows starting at r0 (a multiple of 16), k 32 ks + 8 (lane >> 4) .. + 7
  static __device__ __forceinline__ opx8_t frag(const char* img, int r0, int ks, int lane) {
    const int fr = lane & 15, fq = lane >> 4;
    if constexpr (!TR) {
      const int r = r0 + fr;
      return *reinterpret_cast<const opx8_t*>(img + r * 128 + swz128(r, ks * 4 + fq) * 16);
    } else {
      const int qq = fr >> 2, pp = fr & 3, k = ks * 32 + fq * 8 + qq;   // (k + 4 has the same swizzle)
      const char* a = img + k * (2 * R) + ((r0 >> 4) ^ tr_swz<R>(k)) * 32 + pp * 8;
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(a));
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(a + 4 * 2 * R));
      const s16x8_t v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return *reinterpret_cast<const opx8_t*>(&v);
    }
  }
};

// ---- block-wide sums (256 threads) through LDS, every thread gets the result; fixed order
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- how the two products of a piece share the workgroups (one wave; result in lane 0).  Time is counted in pairs of K
// tiles: a dW tile takes rows / 128 of them, a dh tile 2 x (vocabulary tiles) / splits, and an epilogue some more (dW: 128 KB
// leave the CU; partials: 256 KB leave it and are read again by the last kernel).  Lane s tries s + 1 splits of dh's tiles, and
// for each some of dW's (where the vocabulary is so short that its tiles do not fill the workgroups: dw_room).
__device__ VocabSchedule choose_schedule(const VocabRows& a, int total, int vocab_tiles, int max_splits, int lane) {
  const int rows_t = (total + 255) >> 8, tiles = a.dh ? rows_t * a.tiles_h : 0, wgs = a.wgs;
  if (tiles > 0) {   // partials that there is room for
    const int64_t room = a.dh_room / ((int64_t)tiles * 65536);
    if (room < max_splits) max_splits = (int)room;
  }
  const int dw_tiles = a.with_dw ? vocab_tiles * a.tiles_h : 0, pairs = (total + 127) / 128, splits = lane + 1;
  const int n_dh = tiles * splits, len_dh = (vocab_tiles * 2 + splits - 1) / splits + 6;
  VocabSchedule r = {splits, 1, 0, {0, 0}, {0, 0}, 0};
  int best = 0x7fffffff;
  if (splits <= max_splits && splits <= vocab_tiles)
    for (int d = 1; d <= 16; d += d < 4 ? 1 : d) {   // 1 2 3 4 8 16
      if (d > 1 && (d > pairs || (int64_t)dw_tiles * d * 65536 > a.dw_room)) break;
      const int n_dw = dw_tiles * d, len_dw = (pairs + d - 1) / d + (d > 1 ? 6 : 3);
      // one product dealt evenly, so that some workgroups are behind by one tile; those take more of the other's
#pragma unroll
      for (int even_dh = 0; even_dh < 2; ++even_dh) {
        const int n0 = even_dh ? n_dh : n_dw, l0 = even_dh ? len_dh : len_dw, n1 = even_dh ? n_dw : n_dh, l1 = even_dh ? len_dw : len_dh;
        const int full = n0 / wgs, rest = n0 - full * wgs;
        for (int less = 0; less < 3; ++less) {
          const int left = n1 - less * rest, more = left > 0 ? (left + wgs - rest - 1) / (wgs - rest) : 0;
          const int cost = max(rest ? (full + 1) * l0 + less * l1 : 0, full * l0 + more * l1);
          if (cost < best) {
            best = cost;
            r.dw_splits = d;
            r.first = rest;
            r.dw[0] = even_dh ? less : full + 1;
            r.dw[1] = even_dh ? more : full;
            r.dh[0] = even_dh ? full + 1 : less;
            r.dh[1] = even_dh ? full : more;
          }
        }
      }
    }
  const int low = best;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) best = min(best, __shfl_xor(best, o, 64));
  const int win = __ffsll(__ballot(low == best)) - 1;
  r.dh_splits = win + 1;
  r.dw_splits = __shfl(r.dw_splits, win, 64);
  r.first = __shfl(r.first, win, 64);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    r.dw[i] = __shfl(r.dw[i], win, 64);
    r.dh[i] = __shfl(r.dh[i], win, 64);
  }
  return r;
}

// 0 takes no part, 1 live, 2 live with a target outside the vocabulary
__device__ __forceinline__ int row_state(const VocabRows& a, int r) {
  if (a.state) return a.state[r];
  const int64_t y = a.labels[r];
  return y == a.ignore ? 0 : (y < 0 || y >= a.vocab ? 2 : 1);
}
__device__ __forceinline__ float finite_abs(float g) {
  g = fabsf(g);
  return g < INFINITY ? g : 0.f;
}

// what the whole call needs to know: by one wave, once
template <bool GRAD>
__device__ void write_head(const VocabRows& a, int total, float grad_max, int lane) {
  // (every piece sums into the first's partials: the last must not have more of them)
  VocabSchedule s0 = {a.max_splits, 1, 0, {0, 0}, {0, 0}, 0}, s1 = s0;
  if (GRAD && a.wgs) {
    s0 = choose_schedule(a, total, a.piece_tiles[0], 64, lane);
    s1 = a.piece_tiles[1] == a.piece_tiles[0] ? s0 : choose_schedule(a, total, a.piece_tiles[1], s0.dh_splits, lane);
  }
  if (lane != 0) return;
  *a.count = total;
  if (!GRAD) a.head->done = 0;
  if (GRAD) {
    // the factor common to all rows; what is left of a row's gradient is c, |c| <= 1.  No live row: zeros, not 0 / 0
    const float f = (a.grad_rows ? grad_max : a.grad[0]) * a.grad_factor / (a.mean ? (float)max(total, 1) : 1.f);
    *a.grad_max = grad_max;
    a.out_scale[0] = f / G_SCALE;
    a.out_scale[1] = f;
    a.schedule[0] = s0;
    a.schedule[1] = s1;
  }
}

// what V_GRAD needs of a live row: (x, y, label, t), G = y exp2(z log2(e) / T - x) but t at the label; lc: (x, 1 / sum, c).  x is the
// row's largest score and not its logsumexp: where q is large the exponent is small, and so is its rounding
__device__ __forceinline__ float4 row_info_of(const VocabRows& a, int r, int st, float grad_max, float4& lc) {
  float c = 1.f;
  if (a.grad_rows) {
    const float g = a.grad[r];
    c = fabsf(g) < INFINITY ? (grad_max > 0.f ? g / grad_max : 0.f) : g;
  }
  if (st == 2) c = __builtin_nanf("");   // the target is outside the vocabulary
  const float2 lse = a.lse[r];
  const float x = lse.x == -INFINITY ? 0.f : lse.x, inv = 1.f / lse.y;
  lc = make_float4(x, inv, c, 0.f);
  float4 info = make_float4(x, c * G_SCALE * inv, __int_as_float(-1), 0.f);
  if (!a.state && st == 1) {
    info.z = __int_as_float((int)a.labels[r]);
    info.w = c * (__builtin_amdgcn_exp2f(fmaf(a.target_in[r], LOG2E * a.inv_t, -x)) * inv - 1.f) * G_SCALE;
  }
  return info;
}
__device__ __forceinline__ float4 no_row() { return make_float4(INFINITY, 1.f, __int_as_float(-1), 0.f); }   // G = 0

// Calls of at most 64 rows: what vocab_pack_kernel does otherwise, by the product kernel itself (a launch of 4 us less; the
// one-row loss 21 -> 18 us).  Every workgroup finds the
// live rows for itself (map, in LDS; and info); workgroup 0 notes them down for the kernels that follow, and all of them share
// the copies.  Returns the number of live rows.
template <bool GRAD>
__device__ __forceinline__ int gather_few(const VocabRows& a, bool first_piece, int* map, float4* info) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, groups = gridDim.x;
  const int st = lane < a.n ? row_state(a, lane) : 0;
  const unsigned long long live = __ballot(st != 0);
  const int count = __popcll(live), rank = __popcll(live & ((1ull << lane) - 1));
  const float gm = GRAD && a.grad_rows ? wave_max(st != 0 ? finite_abs(a.grad[lane]) : 0.f) : 0.f;
  if (w == 0) {
    if (GRAD && lane >= count) info[lane] = no_row();
    if (lane >= count) map[lane] = -1;
    if (st != 0) {
      map[rank] = lane;
      float4 lc;
      if (GRAD) info[rank] = row_info_of(a, lane, st, gm, lc);
      if (blockIdx.x == 0) {
        a.row_map[rank] = st == 2 ? ~lane : lane;
        if (GRAD) a.row_info[rank] = info[rank];
        if (GRAD && a.state) a.row_lc[rank] = lc;
      }
    } else if (!GRAD && blockIdx.x == 0 && lane < a.n) {
      a.row_loss[lane] = 0.f;
      a.lse_out[lane] = make_float2(0.f, 1.f);
    }
    if (blockIdx.x == 0) write_head<GRAD>(a, count, gm, lane);
  }
  __syncthreads();
  if (GRAD) {
    // dW reads the rows k by k: side by side, and zeros up to 64
    for (int q = blockIdx.x * 4 + w; q < 64; q += groups * 4) {
      const int r = map[q];
      for (int c = lane * 8; c < a.hidden; c += 512) {   // twice: beside G's high and its low part
        const uint4 v = r < 0 ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(a.h + (int64_t)r * a.ldh + c);
        *reinterpret_cast<uint4*>(a.x + (int64_t)q * a.hidden + c) = v;
        *reinterpret_cast<uint4*>(a.x + (int64_t)(q + 64) * a.hidden + c) = v;
      }
      if (a.dh && q < a.n && !(live >> q & 1))
        for (int c = lane; c < a.hidden; c += 64) a.dh[(int64_t)q * a.ld_dh + c] = 0;
    }
    if (a.fix && first_piece)
      for (int64_t v = (int64_t)blockIdx.x * 256 + tid; v < a.vocab * FIX_COPIES; v += (int64_t)groups * 256) a.fix[v] = 0;
  }
  return count;
}

struct NoRows {};

// what rounding to the operand type leaves of x (0 of what is not finite)
__device__ __forceinline__ float residual(float x) {
  const float r = x - op_to_f32(f32_to_op(x));
  return fabsf(r) < INFINITY ? r : 0.f;
}

// waits until at most N of this wave's loads are in flight
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N <= 63, "counted");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// One output tile of BM x BN per workgroup of WM x WN waves, 64 columns per wave, through a ring of NST K tiles (few rows: many
// small tiles and a deep ring, the weight's bytes are the bound; vocab8.hip takes the large calls).
// FEW: calls of at most 64 rows, whose live rows this kernel finds and reads in place (gather_few).
template <int EPI, int BM, int BN, int WM, int WN, int NST, bool FEW>
__device__ __forceinline__ void vocab_tile(const VocabGemm& a, const std::conditional_t<FEW, VocabRows, NoRows>& rows, char* smem, int tn,
                                           int tm, int split, int splits) {
  constexpr int NW = WM * WN, MB = BM / WM / 16, NB = BN / WN / 16;
  static_assert(NB == 4, "64 columns per wave");
  constexpr bool A_TR = EPI == V_DW, B_TR = EPI == V_DH || EPI == V_DW;
  typedef Operand<BM, A_TR, NW> OA;
  typedef Operand<BN, B_TR, NW> OB;
  constexpr int STAGE = OA::BYTES + OB::BYTES;   // of NST in smem

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w / WN, wn = w % WN, fr = lane & 15, fq = lane >> 4;
  __shared__ int map_s[FEW ? 64 : 1];
  __shared__ float4 info_s[FEW ? 64 : 1];
  int count;                                        // live rows
  if constexpr (FEW) count = gather_few<EPI == V_GRAD>(rows, a.v0 == 0, map_s, info_s);
  else count = *a.count;
  if (EPI != V_DW && tm * BM >= count) return;      // workgroup-uniform

  int nt, kt0 = 0;
  OA oa;
  OB ob;
  if (EPI == V_STATS || EPI == V_GRAD) {
    nt = a.hidden / BK;
    if constexpr (FEW) oa.init_rows(rows.h, ((int64_t)(rows.n - 1) * rows.ldh + a.hidden) * 2, rows.ldh, map_s, w, lane);
    else oa.init(a.x + (int64_t)tm * BM * a.hidden, (int64_t)BM * a.hidden * 2, a.hidden, w, lane);
    const int64_t v0 = a.v0 + (int64_t)tn * BN;
    ob.init(a.w + v0 * a.ldw, ((a.vocab - 1 - v0) * a.ldw + a.hidden) * 2, a.ldw, w, lane);
  } else if (EPI == V_DH) {
    const int all = a.ldg / BK;
    kt0 = (int)((int64_t)all * split / splits);
    nt = (int)((int64_t)all * (split + 1) / splits) - kt0;
    oa.init(a.g + (int64_t)tm * BM * a.ldg + (int64_t)kt0 * BK, (int64_t)BM * a.ldg * 2, a.ldg, w, lane);
    const int64_t v0 = a.v0 + (int64_t)kt0 * BK;
    ob.init(a.w + v0 * a.ldw + tn * BN, ((a.vocab - 1 - v0) * a.ldw + a.hidden - tn * BN) * 2, a.ldw, w, lane);
  } else {
    nt = (count + BK - 1) / BK * (a.low ? 2 : 1);
    oa.init(a.g + (int64_t)tm * BM, ((int64_t)nt * BK * a.ldg - (int64_t)tm * BM) * 2, a.ldg, w, lane);
    ob.init(a.x + tn * BN, ((int64_t)nt * BK * a.hidden - tn * BN) * 2, a.hidden, w, lane);
  }
  // acc[m][n][e]: row fr of the 16-row block m, column 4 fq + e of the 16-column block n
  const int row0 = tm * BM + wm * (BM / WM) + fr, col0 = tn * BN + wn * (BN / WN) + fq * 4;
  f32x4_t acc[MB][NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    f32x4_t start = {0.f, 0.f, 0.f, 0.f};
    if (EPI == V_STATS || EPI == V_GRAD)   // the bias; -inf past the vocabulary
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t v = a.v0 + col0 + n * 16 + e;
        start[e] = v < a.vocab ? (a.bias ? a.bias[v] : 0.f) : -INFINITY;
      }
#pragma unroll
    for (int m = 0; m < MB; ++m) acc[m][n] = start;
  }

  const uint32_t lds0 = (uint32_t)(uintptr_t)LDS_PTR(smem);
#pragma unroll
  for (int i = 0; i < NST - 1; ++i)
    if (i < nt) {
      oa.stage(i, lds0 + i * STAGE, w);
      ob.stage(i, lds0 + i * STAGE + OA::BYTES, w);
    }
  int slot = 0;
  for (int kt = 0; kt < nt; ++kt) {
    // K tile kt has landed; behind it NST - 2 tiles are in flight, until the last ones
    if (kt + NST - 1 <= nt) wait_loads<(NST - 2) * (OA::PIECES + OB::PIECES)>();
    else wait_loads<0>();
    __syncthreads();   // ... for every wave; and every wave has read the buffer that is filled next
    const char* buf = smem + slot * STAGE;
    if (kt + NST - 1 < nt) {
      const uint32_t nxt = lds0 + (slot == 0 ? NST - 1 : slot - 1) * STAGE;
      oa.stage(kt + NST - 1, nxt, w);
      ob.stage(kt + NST - 1, nxt + OA::BYTES, w);
    }
    slot = slot + 1 == NST ? 0 : slot + 1;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      opx8_t af[MB], bf[NB];
#pragma unroll
      for (int m = 0; m < MB; ++m) af[m] = OA::frag(buf, wm * (BM / WM) + m * 16, ks, lane);
#pragma unroll
      for (int n = 0; n < NB; ++n) bf[n] = OB::frag(buf + OA::BYTES, wn * (BN / WN) + n * 16, ks, lane);
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[m][n] = MFMA_16x16x32(bf[n], af[m], acc[m][n]);
    }
  }

  // 16-bit results leave as whole 128-byte row segments, by way of this wave's [16 rows][128 B] in the ring's LDS
  if (EPI == V_GRAD || EPI == V_DW) __syncthreads();
  char* scr = smem + w * 2048;
  auto put = [&](int n, uint2 v) { *reinterpret_cast<uint2*>(scr + fr * 128 + ((n * 4 + fq) ^ ((fr & 7) << 1)) * 8) = v; };
  auto flush = [&](auto&& store) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int row = p * 8 + (lane >> 3), c16 = lane & 7;
      store(row, c16 * 8, *reinterpret_cast<const u32x4_t*>(scr + row * 128 + ((c16 ^ (row & 7)) * 16)));
    }
  };
  if (EPI == V_STATS) {
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      float mx = -INFINITY, t = 0.f;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, acc[m][n][e]);
      mx = fq_max(mx) * a.scale2;
      const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) t += __builtin_amdgcn_exp2f(fmaf(acc[m][n][e], a.scale2, -ref));
      t = fq_sum(t);
      if (fq == 0) a.part[(int64_t)(row0 + m * 16) * a.n_part + tn * WN + wn] = make_float2(mx, t);
    }
  } else if (EPI == V_GRAD) {
    float cs[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) cs[n][e] = 0.f;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const int r = row0 + m * 16;
      const float4 ri = FEW ? info_s[r & 63] : a.row_info[r];
      const int at = __float_as_int(ri.z) - (int)a.v0 - col0;   // the label, counted from this lane's first column
      float low[NB][4];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float g[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          g[e] = at == n * 16 + e ? ri.w : __builtin_amdgcn_exp2f(fmaf(acc[m][n][e], a.scale2, -ri.x)) * ri.y;
          cs[n][e] += g[e];
        }
        put(n, make_uint2(pack_op2(g[0], g[1]), pack_op2(g[2], g[3])));
        if (FEW) {
#pragma unroll
          for (int e = 0; e < 4; ++e) low[n][e] = residual(g[e]);
        }
      }
      auto store = [&](int row, int c, const u32x4_t& v) {
        *reinterpret_cast<u32x4_t*>(a.g + (int64_t)(row0 - fr + m * 16 + row) * a.ldg + tn * BN + wn * 64 + c) = v;
      };
      flush(store);
      if (FEW) {   // G's rows 64 .. 127
#pragma unroll
        for (int n = 0; n < NB; ++n) put(n, make_uint2(pack_op2(low[n][0], low[n][1]), pack_op2(low[n][2], low[n][3])));
        flush([&](int row, int c, const u32x4_t& v) { store(row + 64, c, v); });
      }
    }
    if (a.colsum) {   // fp32 column sums of what was rounded above: db is not made of rounded values
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        f32x4_t t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = fr_sum(cs[n][e]);
        if (fr == 0)
          *reinterpret_cast<f32x4_t*>(a.colsum + (int64_t)(tm * WM + wm) * a.ld_colsum + col0 + n * 16) = t;
      }
    }
  } else if (EPI == V_DH) {
    float* out = a.out32 + (int64_t)split * a.slot_stride;
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n)
        if (col0 + n * 16 < a.hidden) {
          f32x4_t* o = reinterpret_cast<f32x4_t*>(out + (int64_t)(row0 + m * 16) * a.hidden + col0 + n * 16);
          *o = a.accumulate ? *o + acc[m][n] : acc[m][n];
        }
  } else {
    const float s = a.out_scale[0];
#pragma unroll
    for (int m = 0; m < MB; ++m) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
        put(n, make_uint2(pack_op2(acc[m][n][0] * s, acc[m][n][1] * s), pack_op2(acc[m][n][2] * s, acc[m][n][3] * s)));
      flush([&](int row, int c, const u32x4_t& v) {
        const int at = row0 - fr + m * 16 + row, h = tn * BN + wn * 64 + c;
        if (at < a.ldg && a.v0 + at < a.vocab && h < a.hidden) store_dw(a.out16 + (a.v0 + at) * a.ldo + h, v, a.wide);
      });
    }
  }
}

// Scores (V_STATS, V_GRAD), a tile per workgroup.  Few rows: bound by W's bytes, one row 10.9 - 11.8 us for 47 MB (4.0 - 4.3 TB/s).  Rings that
// leave room for two workgroups on a CU, so that 257 tiles and more are not two rounds (us of a loss, one 4-deep ring a CU / two
// 3-deep: V 30 522, H 768 18.0 / 17.8; V 33 000 25 / 20; V 40 000, H 1024 30 / 26; 128-row tiles, one 3-deep / two 2-deep: 128 rows of
// V 30 522 27.5 / 28.6, V 50 257 38 / 32; 4096 rows, H 704 314 / 229).  G with its low part (19 rows) 15 us for 47 MB read and
// 15.6 MB written.
template <int EPI, int BM, int NST, bool FEW>
__global__ __launch_bounds__(256) void vocab_scores_kernel(VocabGemm a, std::conditional_t<FEW, VocabRows, NoRows> rows) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  vocab_tile<EPI, BM, 128, 2, 2, NST, FEW>(a, rows, smem, blockIdx.x % a.tiles_n, blockIdx.x / a.tiles_n, 0, 1);
}
// Both products with G in one launch, which need nothing of each other: dh's tiles of BM rows first (few, with a long k in
// `splits` parts), then dW's of 128 vocabulary entries.  Rings short enough that a CU holds a workgroup of each.  19 rows:
// 27 us for W read, dW written and G (110 MB, 4.1 TB/s); as two launches 14 + 19 us, and 4 us more of host time.
template <int BM, int NST>
__global__ __launch_bounds__(256) void vocab_products_kernel(VocabGemm a, int tiles_m, int splits) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int id = blockIdx.x, tiles = tiles_m * a.tiles_n, n_dh = tiles * splits;
  if (id < n_dh) {
    const int split = id / tiles, t = id - split * tiles;
    vocab_tile<V_DH, BM, 128, 2, 2, NST, false>(a, {}, smem, t % a.tiles_n, t / a.tiles_n, split, splits);
  } else {
    vocab_tile<V_DW, 128, 128, 2, 2, 2, false>(a, {}, smem, (id - n_dh) % a.tiles_n, (id - n_dh) / a.tiles_n, 0, 1);
  }
}

// Teacher lists of a distillation: p = softmax(values / T) over a row's entries with index >= 0 and a value above -inf
// (0 elsewhere), log_p beside it, state[row] = 0 no entry, 1 live, 2 an index beyond the vocabulary or a value that is
// NaN or +inf.  One wave per row.  4096 x 64 entries: 5.5 us (3 MB read; latency).
template <int EACH>   // entries per lane
__global__ __launch_bounds__(256) void vocab_teacher_kernel(VocabRows a) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= a.n) return;
  float t[EACH];
  int64_t id[EACH];
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    t[u] = -INFINITY;
    id[u] = -1;
    if (u * 64 < a.k) {   // (clamped, not skipped: all loads in flight)
      const int j = min(u * 64 + lane, a.k - 1);
      t[u] = a.t_values[(int64_t)row * a.ld_t + j];
      id[u] = a.t_index[(int64_t)row * a.ld_ti + j];
    }
  }
  float mx = -INFINITY;
  int n_in = 0, bad = 0;
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    if (u * 64 + lane >= a.k || id[u] < 0) t[u] = -INFINITY;   // not in the list
    if (t[u] != -INFINITY) {
      mx = fmaxf(mx, t[u] * a.inv_t);
      ++n_in;
      bad |= id[u] >= a.vocab;
    }
  }
  mx = wave_max(mx);
  const float ref = mx == -INFINITY ? 0.f : mx;
  float s = 0.f;
#pragma unroll
  for (int u = 0; u < EACH; ++u)
    if (u * 64 < a.k && t[u] != -INFINITY) s += expf(t[u] * a.inv_t - ref);
  s = wave_sum(s);
  bad |= !(s < INFINITY);   // a NaN or +inf among the teacher's values
  const float log_s = logf(s);
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    const int j = u * 64 + lane;
    if (j >= a.k) continue;
    const float x = t[u] * a.inv_t - ref;
    a.t_p[(int64_t)row * a.k + j] = t[u] != -INFINITY ? expf(x) / s : 0.f;
    a.t_logp[(int64_t)row * a.k + j] = x - log_s;
  }
  const bool any_in = __any(n_in), any_bad = __any(bad);
  if (lane == 0) a.state[row] = any_bad ? 2 : (any_in ? 1 : 0);
}

// Calls of many rows (PACK_COUNTS and more): the live rows before every 16th row, by one workgroup (a thread reads 16 rows' states at
// a time); 131 072 labels in 76 us, latency
template <bool GRAD>
__global__ __launch_bounds__(1024) void vocab_scan_kernel(VocabRows a) {
  __shared__ int sums[16];
  __shared__ float maxs[16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int before = 0;
  float gm = 0.f;
  for (int r0 = 0; r0 < a.n; r0 += 16384) {
    const int r = r0 + tid * 16;
    int live = 0;
    int s[16];   // (clamped, not skipped: all loads in flight)
    if (a.state) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = a.state[min(r + i, a.n - 1)];
    } else {
      int64_t y[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = a.labels[min(r + i, a.n - 1)];
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = y[i] != a.ignore;
    }
    float g[16];
    if (GRAD && a.grad_rows)
#pragma unroll
      for (int i = 0; i < 16; ++i) g[i] = a.grad[min(r + i, a.n - 1)];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const bool takes_part = r + i < a.n && s[i] != 0;
      live += takes_part;
      if (GRAD && a.grad_rows && takes_part) gm = fmaxf(gm, finite_abs(g[i]));
    }
    int up = live;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(up, o, 64);
      if (lane >= o) up += t;
    }
    __syncthreads();
    if (lane == 63) sums[w] = up;
    __syncthreads();
    int base = before, all = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i < w) base += sums[i];
      all += sums[i];
    }
    if (r < a.n) a.block_base[r >> 4] = base + up - live;
    before += all;
  }
  if (GRAD) {
    gm = wave_max(gm);
    if (lane == 0) maxs[w] = gm;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) gm = fmaxf(gm, maxs[i]);
  }
  if (w == 0) write_head<GRAD>(a, before, gm, lane);
}

// Live rows side by side: x[r] = hidden[row_map[r]], zero rows up to the end of their last tile.  A workgroup per NT / 16 rows,
// four to a wave; without a scan before it each counts all rows' states itself.  Backward: also what V_GRAD needs of every row,
// zero gradients of the dropped rows, and a zeroed table of target sums.  16 384 rows 25 us (50 MB), 4096 rows 14 us (12.6 MB).
template <bool GRAD, int NT>
__global__ __launch_bounds__(NT) void vocab_pack_kernel(VocabRows a) {
  constexpr int NW = NT / 64, ROWS = NT / 16;
  __shared__ int before_s[NW], total_s[NW];
  __shared__ float max_s[NW];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, r0 = blockIdx.x * ROWS, r = r0 + lane;
  const int H = a.hidden;
  // this wave's four rows are on their way before it is known which of them are live
  uint4 held[4][2];
  if (a.h_aligned && a.n > 0)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c)
        held[i][c] = *reinterpret_cast<const uint4*>(a.h + (int64_t)min(r0 + w * 4 + i, a.n - 1) * a.ldh + min(lane * 8 + c * 512, H - 8));
  const int st = lane < ROWS && r < a.n ? row_state(a, r) : 0;
  int before, total;
  float gm = 0.f;
  if (a.block_base) {
    before = a.block_base[r0 >> 4];
    total = *a.count;
    if (GRAD) gm = *a.grad_max;
  } else {
    before = total = 0;
    auto count = [&]<int U>(int q0) {   // U loads in flight: clamped, not skipped
      int s[U];
      if (a.state) {
#pragma unroll
        for (int i = 0; i < U; ++i) s[i] = a.state[min(q0 + i * NT + tid, a.n - 1)];
      } else {
        int64_t y[U];
#pragma unroll
        for (int i = 0; i < U; ++i) y[i] = a.labels[min(q0 + i * NT + tid, a.n - 1)];
#pragma unroll
        for (int i = 0; i < U; ++i) s[i] = y[i] != a.ignore;
      }
      float g[U];
      if (GRAD && a.grad_rows)
#pragma unroll
        for (int i = 0; i < U; ++i) g[i] = a.grad[min(q0 + i * NT + tid, a.n - 1)];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int q = q0 + i * NT + tid;
        const bool live = q < a.n && s[i] != 0;
        total += live;
        before += live && q < r0;
        if (GRAD && a.grad_rows && live) gm = fmaxf(gm, finite_abs(g[i]));
      }
    };
    int q0 = 0;
    for (; q0 + 2 * NT < a.n; q0 += NT * 8) count.template operator()<8>(q0);
    for (; q0 < a.n; q0 += NT) count.template operator()<1>(q0);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      before += __shfl_xor(before, o, 64);
      total += __shfl_xor(total, o, 64);
    }
    if (GRAD) gm = wave_max(gm);
    if (lane == 0) { before_s[w] = before; total_s[w] = total; if (GRAD) max_s[w] = gm; }
    __syncthreads();
    before = total = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      before += before_s[i];
      total += total_s[i];
      if (GRAD) gm = fmaxf(gm, max_s[i]);
    }
    if (blockIdx.x == 0 && w == 0) write_head<GRAD>(a, total, gm, lane);
  }
  // every wave ranks its workgroup's rows, wave 0 notes them down, wave w copies rows 4 w .. 4 w + 3
  const unsigned long long live = __ballot(st != 0);
  {
    int64_t rank = before + __popcll(live & ((1ull << (w * 4)) - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int q = w * 4 + i;
      if (live >> q & 1) {
        bf16_t* dst = a.x + rank++ * H;
        const bf16_t* src = a.h + (int64_t)(r0 + q) * a.ldh;
        if (a.h_aligned) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (lane * 8 + c * 512 < H) *reinterpret_cast<uint4*>(dst + lane * 8 + c * 512) = held[i][c];
          for (int c = lane * 8 + 1024; c < H; c += 512) *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
        } else {
          for (int c = lane; c < H; c += 64) dst[c] = src[c];
        }
      } else if (GRAD && a.dh && r0 + q < a.n) {
        for (int c = lane; c < H; c += 64) a.dh[(int64_t)(r0 + q) * a.ld_dh + c] = 0;
      }
    }
  }
  if (w == 0 && lane < ROWS && r < a.n) {
    if (st != 0) {
      const int rank = before + __popcll(live & ((1ull << lane) - 1));
      a.row_map[rank] = st == 2 ? ~r : r;    // a row whose target is outside the vocabulary: NaN loss and gradients
      if (GRAD) {
        float4 lc;
        a.row_info[rank] = row_info_of(a, r, st, gm, lc);
        if (a.state) a.row_lc[rank] = lc;
      }
    } else if (!GRAD) {
      a.row_loss[r] = 0.f;
      a.lse_out[r] = make_float2(0.f, 1.f);
    }
  }
  const int pad = (total + a.tile_rows - 1) / a.tile_rows * a.tile_rows;
  for (int q = total + blockIdx.x * NW + w; q < pad; q += gridDim.x * NW) {
    for (int c = lane * 8; c < H; c += 512) *reinterpret_cast<uint4*>(a.x + (int64_t)q * H + c) = make_uint4(0, 0, 0, 0);
    if (GRAD && lane == 0) a.row_info[q] = no_row();
  }
  if (GRAD && a.fix)
    for (int64_t v = (int64_t)blockIdx.x * NT + tid; v < a.vocab * FIX_COPIES; v += (int64_t)gridDim.x * NT) a.fix[v] = 0;
}

// few rows that 16-byte loads with 31-bit offsets cannot read where they are, a row a workgroup
__global__ __launch_bounds__(256) void vocab_copy_kernel(const bf16_t* __restrict__ from, int64_t ld, bf16_t* __restrict__ to, int hidden) {
  for (int c = threadIdx.x; c < hidden; c += 256) to[(int64_t)blockIdx.x * hidden + c] = from[blockIdx.x * ld + c];
}

// Scores of 16 vocabulary entries for one hidden row x, acc = their bias to begin with: by the same instruction as the tiles of
// scores, in the same order of k, so that they have the bits that the row's softmax is made of (in any other order they would be off
// from these by fp32's rounding of a score, which a small temperature or large scores make a wrong probability).  x passes through
// this wave's KB of LDS, every entry's row of W (lane & 15: which) comes in pieces of 64 bytes; the result is acc[e] = the score of
// entry 4 (lane >> 4) + e.  ONE: all entries are the same, and its row passes through a second KB of LDS.  `p`: the first KB of either
// (a lane's 16 bytes), loaded by the caller before it waits for anything else.
struct RowPieces { uint4 x, w; };
template <bool ONE>
__device__ __forceinline__ RowPieces row_pieces(const bf16_t* x, const bf16_t* wrow, int c0, int H, int lane) {
  RowPieces p = {};
  const int at = min(c0 + lane * 8, H - 8);
  p.x = *reinterpret_cast<const uint4*>(x + at);
  if (ONE) p.w = *reinterpret_cast<const uint4*>(wrow + at);
  return p;
}
template <bool ONE>
__device__ __forceinline__ f32x4_t tile_scores(RowPieces p, const bf16_t* x, const bf16_t* wrow, f32x4_t acc, int H, int lane, char* lds) {
  const int fq = lane >> 4;
  for (int c0 = 0; c0 < H; c0 += 512) {
    const int steps = min(H - c0, 512) / 32;
    *reinterpret_cast<uint4*>(lds + lane * 16) = p.x;
    if (ONE) *reinterpret_cast<uint4*>(lds + 1024 + lane * 16) = p.w;
    if (c0 + 512 < H) p = row_pieces<ONE>(x, wrow, c0 + 512, H, lane);
    for (int s0 = 0; s0 < steps; s0 += 8) {   // eight pieces of every row in flight
      uint4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int s = min(s0 + u, steps - 1);
        v[u] = ONE ? *reinterpret_cast<const uint4*>(lds + 1024 + s * 64 + fq * 16)
                   : *reinterpret_cast<const uint4*>(wrow + c0 + s * 32 + fq * 8);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (s0 + u < steps)   // (uniform)
          acc = MFMA_16x16x32(*reinterpret_cast<const opx8_t*>(&v[u]), *reinterpret_cast<const opx8_t*>(lds + (s0 + u) * 64 + fq * 16), acc);
    }
  }
  return acc;
}

// what a row's exponentials over 64 columns at a time come to: (largest score, sum) of a wave's share of the pairs
__device__ __forceinline__ float2 wave_pairs(const float2* p, int n_part, int lane, int step) {
  float2 v[8];
  float mx = -INFINITY, s = 0.f;
  for (int i0 = lane; i0 < n_part; i0 += 8 * step) {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = i0 + u * step < n_part ? p[i0 + u * step] : make_float2(-INFINITY, 0.f);
    float m = mx;
#pragma unroll
    for (int u = 0; u < 8; ++u) m = fmaxf(m, v[u].x);
    const float ref = m == -INFINITY ? 0.f : m;
    s *= __builtin_amdgcn_exp2f(mx - ref);
#pragma unroll
    for (int u = 0; u < 8; ++u) s += v[u].y * __builtin_amdgcn_exp2f(v[u].x - ref);
    mx = m;
  }
  const float m = wave_max(mx), ref = m == -INFINITY ? 0.f : m;
  return make_float2(m, wave_sum(s * __builtin_amdgcn_exp2f(mx - ref)));
}
__device__ __forceinline__ float2 join_pairs(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x), ref = m == -INFINITY ? 0.f : m;
  return make_float2(m, a.y * __builtin_amdgcn_exp2f(a.x - ref) + b.y * __builtin_amdgcn_exp2f(b.x - ref));
}
// logsumexp(z / T) - z / T of one score, p the row's pair: the difference is taken next to the exponentials' own arithmetic
__device__ __forceinline__ float minus_log_q(float2 p, float z, float scale2) {
  return LN2 * (log2f(p.y) - fmaf(z, scale2, p.x == -INFINITY ? 0.f : -p.x));
}

// Forward over several pieces of the vocabulary: a piece's n pairs of every live row (rows n_part apart), and what the pieces before
// it (`more`) came to, in one pair.  One wave per row; bound by the pairs' bytes.  A loss in one piece / several: 131 072 rows (H 128),
// V 70 001 (2 pieces) 4.17 / 4.25 ms, V 262 221 (5) 13.6 / 13.8; 2^20 rows (H 64), V 262 221 (33) 129 / 138
__global__ __launch_bounds__(256) void vocab_join_kernel(const int32_t* __restrict__ count, const float2* __restrict__ part, int n_part, int n,
                                                         float2* __restrict__ joined, int more) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= *count) return;
  float2 all = wave_pairs(part + (int64_t)r * n_part, n, lane, 64);
  if (more) all = join_pairs(joined[r], all);
  if (lane == 0) joined[r] = all;
}

// The rows' losses are summed by the last of few workgroups to finish (the others' results are stored to where every XCD
// reads, and acknowledged, before they count themselves), or by a kernel of its own where there are many.
__device__ __forceinline__ void finish_rows(const VocabRows& a, int groups, float* red) {
  __shared__ int last_s;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    last_s = __hip_atomic_fetch_add(a.done, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == groups - 1;
  __syncthreads();
  if (!last_s) return;
  float s = 0.f;
  for (int i = threadIdx.x; i < a.n; i += 256) s += __hip_atomic_load(a.row_loss + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  s = block_sum(s, red);
  if (threadIdx.x == 0) a.loss[0] = a.mean ? s / (float)*a.count : s;
}

// Cross entropy, one wave per live row: lse from the tiles' (max, sum) pairs, the label's score, the row's loss.  16 384 rows
// 21 us for 63 MB of pairs and 50 MB of rows; 4096 rows 10 us; one row 4.4, the chain of 24 MFMAs and its LDS passes 0.6 of it.
__global__ __launch_bounds__(256) void vocab_ce_kernel(VocabRows a, const float2* __restrict__ part, int n_part) {
  __shared__ float red[4];
  __shared__ __attribute__((aligned(16))) char stage[4][2048];
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r < *a.count) {
    const int mapped = a.row_map[r], row = mapped < 0 ? ~mapped : mapped;
    float loss = __builtin_nanf(""), z = 0.f, b = 0.f;
    const bf16_t *x = a.x ? a.x + (int64_t)r * a.hidden : a.h + (int64_t)row * a.ldh, *wrow = a.w;
    if (mapped >= 0) {
      const int64_t v = a.labels[row];
      wrow += v * a.ldw;
      if (a.bias) b = a.bias[v];
    }
    const RowPieces first = row_pieces<true>(x, wrow, 0, a.hidden, lane);
    const float2 all = wave_pairs(part + (int64_t)r * n_part, n_part, lane, 64);
    if (mapped >= 0) {
      z = tile_scores<true>(first, x, wrow, (f32x4_t){b, b, b, b}, a.hidden, lane, stage[threadIdx.x >> 6])[0];
      loss = minus_log_q(all, z, LOG2E * a.inv_t);
      loss = loss < 0.f ? 0.f : loss;   // (the sum holds the label's own term: what is below zero is exp2's and log2's rounding; NaN stays)
    }
    if (lane == 0) {
      a.target[row] = z;
      a.lse_out[row] = all;
      __hip_atomic_store(a.row_loss + row, loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (a.done) finish_rows(a, gridDim.x, red);
}

// Distillation, WPR waves per live row sharing the teacher's entries: one for short lists, four for long ones.  Bound: the
// gather of k rows of W per row, which the caches serve: 4096 rows, k 64, H 512: 44 us for 268 MB (6.1 TB/s).
template <int WPR>
__global__ __launch_bounds__(256) void vocab_distill_kernel(VocabRows a, const float2* __restrict__ part, int n_part) {
  __shared__ float red[4];
  __shared__ float2 pair[4];
  __shared__ __attribute__((aligned(16))) char stage[4][1024];
  const int tid = threadIdx.x, lane = tid & 63, w = WPR == 4 ? tid >> 6 : 0;
  const int r = WPR == 4 ? blockIdx.x : blockIdx.x * 4 + (tid >> 6);
  if (r < *a.count) {   // (WPR 4: the same for the whole workgroup)
    const int mapped = a.row_map[r], row = mapped < 0 ? ~mapped : mapped;
    float2 all = wave_pairs(part + (int64_t)r * n_part, n_part, WPR == 4 ? tid : lane, 64 * WPR);
    if (WPR == 4) {
      if (lane == 0) pair[w] = all;
      __syncthreads();
      all = pair[0];
#pragma unroll
      for (int i = 1; i < 4; ++i) all = join_pairs(all, pair[i]);
    }
    const bf16_t* x = a.x ? a.x + (int64_t)r * a.hidden : a.h + (int64_t)row * a.ldh;
    const float scale2 = LOG2E * a.inv_t;
    const int fr = lane & 15, fq = lane >> 4;
    float loss = 0.f;
    if (mapped >= 0)
      for (int j0 = w * 16; j0 < a.k; j0 += 16 * WPR) {
        const int64_t mine = j0 + fr < a.k ? a.t_index[(int64_t)row * a.ld_ti + j0 + fr] : -1;
        const int v = mine >= 0 && mine < a.vocab ? (int)mine : -1;   // (beyond only where the value is -inf)
        f32x4_t z;
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = a.bias ? a.bias[max(__shfl(v, fq * 4 + e, 64), 0)] : 0.f;
        z = tile_scores<false>(row_pieces<false>(x, x, 0, a.hidden, lane), x, a.w + (int64_t)max(v, 0) * a.ldw, z, a.hidden, lane, stage[tid >> 6]);
        // entry 4 fq + fr is this lane's, fr < 4
        const int j = j0 + fq * 4 + fr, vj = __shfl(v, fq * 4 + (fr & 3), 64);
        if (fr < 4 && j < a.k) {
          const float zj = fr == 0 ? z[0] : fr == 1 ? z[1] : fr == 2 ? z[2] : z[3];
          a.target[(int64_t)row * a.k + j] = vj >= 0 ? zj : 0.f;
          const float pj = vj >= 0 ? a.t_p[(int64_t)row * a.k + j] : 0.f;
          if (pj != 0.f) loss += pj * (a.t_logp[(int64_t)row * a.k + j] + minus_log_q(all, zj, scale2));
        }
      }
    loss = wave_sum(loss);
    if (WPR == 4) {
      if (lane == 0) red[w] = loss;
      __syncthreads();
      loss = (red[0] + red[1]) + (red[2] + red[3]);
    }
    if (w == 0 && lane == 0) {
      loss = mapped < 0 ? __builtin_nanf("") : loss * a.loss_factor;
      a.lse_out[row] = all;
      __hip_atomic_store(a.row_loss + row, loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (a.done) finish_rows(a, gridDim.x, red);
}

// loss[0] = sum of the rows' losses, over the live rows' count for the mean (0 / 0 = NaN as torch's mean over none);
// one workgroup, fixed order
__global__ __launch_bounds__(1024) void vocab_reduce_kernel(VocabRows a) {
  __shared__ float red[16];
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = threadIdx.x; i < a.n; i += 4096)
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * 1024 < a.n) s[u] += a.row_loss[i + u * 1024];
  const float t = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    float sum = 0.f;
    for (int i = 0; i < 16; ++i) sum += red[i];
    a.loss[0] = a.mean ? sum / (float)*a.count : sum;
  }
}

// The teacher's part of G: G[r, v] = c (q_v - sum of p over the entries that name v), from the forward's fp32 score of v (a
// difference of the rounded q would lose what is left where q is near p).  (A label's part is set by V_GRAD itself.)  The sums
// of c p per vocabulary entry, which db needs, go to a table of 64-bit fixed point: integer adds commute, so their order does
// not show (2^-38 a unit; |c| p <= 1, n <= 2^24 rows); in FIX_COPIES copies by row, since a teacher's frequent entries are the
// same in most rows.
// `first`: this entry is the first of its row to name v (0 <= v), `p` what they add up to, `own` its own part.  Returns whether
// the entry is a sixteenth or more of the row, and what rounding leaves of it.
__device__ __forceinline__ bool teacher_entry(const VocabRows& a, const float4& lc, int r, int row, int j, int v, float own, float p, bool first,
                                              bf16_t* g, int64_t ldg, int64_t v0, int64_t v1, int table, float& rest) {
  if (a.fix && table && v >= 0 && fabsf(lc.z * own) <= 1.f)
    atomicAdd(reinterpret_cast<unsigned long long*>(a.fix + (r & (FIX_COPIES - 1)) * a.vocab + v), (unsigned long long)__double2ll_rn((double)(lc.z * own) * FIX));
  if (!first) return false;
  const float q = __builtin_amdgcn_exp2f(fmaf(a.target_in[(int64_t)row * a.k + j], LOG2E * a.inv_t, -lc.x)) * lc.y;
  const float e = lc.z * (q - p) * G_SCALE;
  if (v >= v0 && v < v1) {
    g[(int64_t)r * ldg + (v - v0)] = f32_to_op(e);
    if (a.low) g[(int64_t)(r + 64) * ldg + (v - v0)] = f32_to_op(residual(e));
  }
  rest = residual(e);
  return fabsf(q - p) >= 0.0625f;
}
__device__ __forceinline__ void teacher_list(const VocabRows& a, int row, int j, int& v, float& own) {
  // (not listed, or beyond the vocabulary, which only an entry of value -inf may be: -1)
  const int64_t t = j < a.k ? a.t_index[(int64_t)row * a.ld_ti + j] : -1;
  v = t >= 0 && t < a.vocab ? (int)t : -1;
  own = j < a.k ? a.t_p[(int64_t)row * a.k + j] : 0.f;
}
// up to 64 entries a row: one wave per live row, every entry against every other.  4096 x 64 entries: 23 us, mostly the table's
// adds (262 k of them)
__global__ __launch_bounds__(256) void vocab_teacher_grad_kernel(VocabRows a, bf16_t* __restrict__ g, int64_t ldg, int64_t v0, int64_t v1,
                                                                 int table) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= *a.count) return;
  const int row = a.row_map[r];
  unsigned long long big = 0;
  float rest = 0.f;
  int v = -1;
  if (row >= 0) {   // (else a row of NaN: nothing to put in or to correct)
    int earlier = 0;
    float own, p = 0.f;
    teacher_list(a, row, lane, v, own);
    for (int i = 0; i < a.k; ++i) {   // every entry that names v
      const int ui = __builtin_amdgcn_readlane(v, i);
      const float qi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(own), i));
      p += ui == v ? qi : 0.f;
      earlier += ui == v && i < lane;
    }
    big = __ballot(teacher_entry(a, a.row_lc[r], r, row, lane, v, own, p, v >= 0 && earlier == 0, g, ldg, v0, v1, table, rest));
  }
  if (table && a.dh) {   // the row's first ROW_FIX large entries
    float2* fix = a.row_fix + (int64_t)r * ROW_FIX;
    const int at = __popcll(big & ((1ull << lane) - 1));
    if ((big >> lane & 1) && at < ROW_FIX) fix[at] = make_float2(__int_as_float(v), rest);
    if (lane < ROW_FIX && lane >= __popcll(big)) fix[lane] = make_float2(__int_as_float(-1), 0.f);
  }
}
// more entries: a workgroup per live row, the sums by way of a hash table in LDS that is at most half full (64-bit fixed point
// again, of 2^-62 a unit).  4096 rows: 128 entries 35 us, 1024 200 us (every entry against every other: 51 us, 1530 us)
__global__ __launch_bounds__(256) void vocab_teacher_hash_kernel(VocabRows a, bf16_t* __restrict__ g, int64_t ldg, int64_t v0, int64_t v1,
                                                                 int table) {
  constexpr int SIZE = 2048, EACH = 4;   // 1024 entries
  constexpr double UNIT = 4611686018427387904.0;
  __shared__ int id_s[SIZE], first_s[SIZE];
  __shared__ unsigned long long sum_s[SIZE], big_s[EACH][4];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  if (r >= *a.count) return;
  const int row = a.row_map[r];
  float2* fix = table && a.dh ? a.row_fix + (int64_t)r * ROW_FIX : nullptr;
  if (row < 0) {
    if (fix && tid < ROW_FIX) fix[tid] = make_float2(__int_as_float(-1), 0.f);
    return;
  }
  const float4 lc = a.row_lc[r];
  int v[EACH], slot[EACH];
  float own[EACH], rest[EACH];
#pragma unroll
  for (int u = 0; u < EACH; ++u) teacher_list(a, row, u * 256 + tid, v[u], own[u]);
  for (int i = tid; i < SIZE; i += 256) {
    id_s[i] = -1;
    first_s[i] = 1 << 30;
    sum_s[i] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    slot[u] = 0;
    if (v[u] < 0) continue;
    int h = (int)((uint32_t)v[u] * 2654435761u >> 21);
    for (int at; (at = atomicCAS(&id_s[h], -1, v[u])) != -1 && at != v[u];) h = (h + 1) & (SIZE - 1);
    slot[u] = h;
    atomicAdd(&sum_s[h], (unsigned long long)__double2ull_rn((double)own[u] * UNIT));
    atomicMin(&first_s[h], u * 256 + tid);
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    const int j = u * 256 + tid;
    const bool first = v[u] >= 0 && first_s[slot[u]] == j;
    const float p = (float)((double)sum_s[slot[u]] / UNIT);
    const unsigned long long big = __ballot(teacher_entry(a, lc, r, row, j, v[u], own[u], p, first, g, ldg, v0, v1, table, rest[u]));
    if (lane == 0) big_s[u][w] = big;
  }
  if (!fix) return;
  __syncthreads();
  int before = 0;   // large entries ahead, in the list's order
#pragma unroll
  for (int u = 0; u < EACH; ++u)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const unsigned long long big = big_s[u][q];
      const int at = before + __popcll(big & ((1ull << lane) - 1));
      if (q == w && (big >> lane & 1) && at < ROW_FIX) fix[at] = make_float2(__int_as_float(v[u]), rest[u]);
      before += __popcll(big);
    }
  if (tid < ROW_FIX && tid >= before) fix[tid] = make_float2(__int_as_float(-1), 0.f);
}

// dh of the live rows from the fp32 partials (fixed order), and db of the entries v0 .. v1 (a piece of the vocabulary) from its column
// sums and the targets' table; dW from its partials where its k was split.  Bound: the partials' bytes; 16 384 rows 48 us, 4096 rows 15 us
__global__ __launch_bounds__(256) void vocab_finish_kernel(VocabRows a, VocabPlan p, const float* __restrict__ part,
                                                           const float* __restrict__ colsum, const float* __restrict__ dw_part,
                                                           bf16_t* __restrict__ dw, int64_t ld_dw, int row_blocks, int dw_blocks, int64_t v0, int64_t v1) {
  const int count = *a.count;
  const int b_blocks = gridDim.x - row_blocks - dw_blocks;
  // the sum of n slots' partials, four of them in flight, in order; rounded: times the common factor
  const float s = a.out_scale[0];
  auto sum_slots = [&](const float* q, int n, int64_t slot) -> f32x4_t {
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    int k = 0;
    for (; k + 4 <= n; k += 4) {
      f32x4_t t[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) t[u] = *reinterpret_cast<const f32x4_t*>(q + (k + u) * slot);
#pragma unroll
      for (int u = 0; u < 4; ++u) v += t[u];
    }
    for (; k < n; ++k) v += *reinterpret_cast<const f32x4_t*>(q + k * slot);
    return v;
  };
  auto rounded = [&](const f32x4_t& v) { return make_uint2(pack_op2(v[0] * s, v[1] * s), pack_op2(v[2] * s, v[3] * s)); };
  if ((int)blockIdx.x >= b_blocks + dw_blocks) {
    const int n = a.schedule[0].dh_splits;
    const int tiles_r = (count + 255) >> 8, h4 = a.hidden / 4;
    const int64_t total = p.large ? (int64_t)tiles_r * a.tiles_h * 16384 : (int64_t)count * h4;
    const int64_t slot = p.large ? total * 4 : p.dh_slot;
    for (int64_t i = (int64_t)(blockIdx.x - b_blocks - dw_blocks) * 256 + threadIdx.x; i < total; i += (int64_t)row_blocks * 256) {
      int r, c;
      if (p.large) {
        const int tile = (int)(i >> 14);
        dh_partial_at((int)(i & 16383), r, c);
        r += tile / a.tiles_h * 256;
        c += tile % a.tiles_h * 256;
        if (r >= count || c >= a.hidden) continue;
      } else {
        r = (int)(i / h4);
        c = (int)(i - (int64_t)r * h4) * 4;
      }
      f32x4_t v = sum_slots(part + i * 4, n, slot);
      // what G's rounding left of the row's largest entries
      auto correct = [&](int id, float rest) {
        const uint2 wv = *reinterpret_cast<const uint2*>(a.w + (int64_t)id * a.ldw + c);
        v[0] = fmaf(rest, op2_lo(wv.x), v[0]); v[1] = fmaf(rest, op2_hi(wv.x), v[1]);
        v[2] = fmaf(rest, op2_lo(wv.y), v[2]); v[3] = fmaf(rest, op2_hi(wv.y), v[3]);
      };
      if (a.row_fix) {
        for (int k = 0; k < ROW_FIX; ++k) {
          const float2 f = a.row_fix[(int64_t)r * ROW_FIX + k];
          if (__float_as_int(f.x) < 0) break;
          correct(__float_as_int(f.x), f.y);
        }
      } else {
        const float4 ri = a.row_info[r];
        if (__float_as_int(ri.z) >= 0) correct(__float_as_int(ri.z), residual(ri.w));
      }
      const uint2 packed = rounded(v);
      const int m = a.row_map[r];
      bf16_t* o = a.dh + (int64_t)(m < 0 ? ~m : m) * a.ld_dh + c;
      if (a.dh_aligned) {
        *reinterpret_cast<uint2*>(o) = packed;
      } else {
        o[0] = (bf16_t)packed.x; o[1] = (bf16_t)(packed.x >> 16);
        o[2] = (bf16_t)packed.y; o[3] = (bf16_t)(packed.y >> 16);
      }
    }
  } else if ((int)blockIdx.x >= b_blocks) {
    const int n = a.schedule[0].dw_splits, tiles = a.piece_tiles[0] * a.tiles_h;
    if (n == 1) return;   // written whole
    for (int64_t i = (int64_t)(blockIdx.x - b_blocks) * 256 + threadIdx.x; i < (int64_t)tiles * 16384; i += (int64_t)dw_blocks * 256) {
      const int tile = (int)(i >> 14);
      int r, c;
      dh_partial_at((int)(i & 16383), r, c);
      const int64_t v = (int64_t)(tile / a.tiles_h) * 256 + r;
      c += tile % a.tiles_h * 256;
      if (v < a.vocab && c < a.hidden) *reinterpret_cast<uint2*>(dw + v * ld_dw + c) = rounded(sum_slots(dw_part + i * 4, n, (int64_t)tiles * 65536));
    }
  } else {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, v = v0 + at;
    if (v >= v1) return;
    const int n_sums = (count + p.tile_rows - 1) / p.tile_rows * 2;   // one per half tile of rows
    float sum = 0.f;
    int k = 0;
    for (; k + 8 <= n_sums; k += 8) {
      float t[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) t[u] = colsum[(int64_t)(k + u) * p.ld_colsum + at];
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += t[u];
    }
    for (; k < n_sums; ++k) sum += colsum[(int64_t)k * p.ld_colsum + at];
    if (a.fix) {   // (the sum is in units of G, the table in units of c)
      int64_t t = 0;
#pragma unroll
      for (int u = 0; u < FIX_COPIES; ++u) t += a.fix[u * a.vocab + v];
      a.dbias[v] = (float)((double)sum / G_SCALE - (double)t / FIX) * a.out_scale[1];
    } else {
      a.dbias[v] = sum * s;
    }
  }
}

template <auto KERNEL, typename... Args>
hipError_t launch_tiles(int lds, int64_t groups, hipStream_t st, const Args&... args) {
  static DeviceOnce once;
  int unused;
  TRY(once.get([&](int, int*) {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  }, &unused));
  hipLaunchKernelGGL(KERNEL, dim3((uint32_t)groups), dim3(256), lds, st, args...);
  return hipGetLastError();
}
// up to 64 rows: 64-row tiles of scores and dh, (its k) of dW; more: 128-row tiles
constexpr int ring_bytes(int rows, int stages) { return stages * (rows + 128) * BK * 2; }
template <int EPI>
hipError_t launch_scores(const VocabGemm& g, const VocabRows& a, bool few, hipStream_t st) {
  if (few) return launch_tiles<vocab_scores_kernel<EPI, 64, 3, true>>(ring_bytes(64, 3), g.tiles_n, st, g, a);
  return launch_tiles<vocab_scores_kernel<EPI, 128, 2, false>>(ring_bytes(128, 2), (a.n + 127) / 128 * (int64_t)g.tiles_n, st, g, NoRows());
}
hipError_t launch_products(const VocabGemm& g, const VocabPlan& p, int n, hipStream_t st) {
  const int tiles_m = g.with_dh ? (n + p.tile_rows - 1) / p.tile_rows : 0;
  const int64_t groups = (int64_t)g.tiles_n * (tiles_m * p.splits + (g.with_dw ? g.ldg / 128 : 0));
  if (groups == 0) return hipSuccess;
  return p.tile_rows == 64 ? launch_tiles<vocab_products_kernel<64, 3>>(ring_bytes(64, 3), groups, st, g, tiles_m, (int)p.splits)
                           : launch_tiles<vocab_products_kernel<128, 2>>(ring_bytes(128, 2), groups, st, g, tiles_m, (int)p.splits);
}

}  // namespace

#if !CLIP_OPERAND_F16
// G of one piece of the vocabulary may take this much in the backward pass, (max, sum) pairs in the forward: the pieces are as few
// as that allows
constexpr int64_t PIECE_BYTES = (int64_t)1 << 30;
// Which calls run on the 256 x 256 tiles of vocab8.hip: up to 128 rows none (the small tiles read W once per 128 rows).
// The loss alone from 192 tiles, in us, these / the small ones:  V 30 522, H 768: n 256 (120 tiles) 35 / 32, 300 (240) 38 / 42;
//   H 128: n 257 (240) 22 / 25;   V 8 000, H 256: n 1024 (128) 26 / 24, 2048 (256) 26 / 32;   V 2 000, H 768: n 4096 (128) 42 / 40
// Loss and gradients from 500 blocks of 256^3:  V 30 522, H 768: n 256 (360 blocks) 119 / 116, 300 (720) 136 / 155, 1024 230 / 305;
//   H 128: n 1024 (240) 117 / 114, 2048 (480) 176 / 171, 8192 571 / 623;   V 8 000, H 768: n 1024 (384) 115 / 112, 2048 148 / 174;
//   H 256: n 2048 (256) 101 / 99, 4096 (512) 142 / 160;   V 2 000, H 768: n 4096 (384) 132 / 126
// and beyond 4096 rows, where the small tiles' unsplit k makes dW late:  V 2 000, H 256: n 4096 (128) 92 / 103, but 75 / 56 if 15 % of
//   the rows are live, 6000 (192) 104 / 138
bool large_tiles(int32_t n, int64_t vocab, int32_t hidden, bool grad) {
  if (hidden % 128 || n <= 128) return false;
  const int64_t tiles = ((int64_t)n + 255) / 256 * ((vocab + 255) / 256);
  return grad ? n > 4096 || tiles * hidden >= 500 * 256 : tiles >= 192;
}

VocabPlan vocab_plan(int32_t n, int64_t vocab, int32_t hidden, int64_t ldw, int32_t k, bool distill, bool grad) {
  VocabPlan p = {};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) & ~(size_t)255;
    return o;
  };
  p.large = large_tiles(n, vocab, hidden, grad);
  p.tile_rows = p.large ? 256 : (n <= 64 ? 64 : 128);
  const int64_t rows = ((int64_t)n + 255) / 256 * 256, vp = (vocab + 255) / 256 * 256;
  p.head = take(sizeof(VocabHead));
  p.row_map = take(rows * 4);
  p.block_base = take(rows / 16 * 4);
  if (distill && !grad) p.t_logp = take((size_t)n * k * 4);
  p.x = take(rows * hidden * 2);
  // pieces of whole 256-column tiles, at most `most` columns each, of about the same size
  auto cut = [&](int64_t most) {
    const int64_t piece = max((int64_t)256, min(most / 256 * 256, vp));
    p.pieces = (vp + piece - 1) / piece;
    p.piece = ((vp / 256 + p.pieces - 1) / p.pieces) * 256;
    p.pieces = (vp + p.piece - 1) / p.piece;
  };
  if (!grad) {
    const int64_t pair_rows = p.tile_rows == 64 ? (n > 0 ? 64 : 0) : rows;   // 8 bytes per row and 64 columns
    cut(pair_rows > 0 ? PIECE_BYTES / (pair_rows * 8) * 64 : vp);
    p.part = take(pair_rows * (p.piece / 64) * 8);
    if (p.pieces > 1) p.joined = take(pair_rows * 8);
  } else {
    p.row_info = take(rows * 16);
    if (distill) {
      p.row_lc = take(rows * 16);
      p.row_fix = take(rows * 8 * ROW_FIX);
      p.fix = take(vocab * 8 * FIX_COPIES);
    }
    // G within its bound, 32-bit byte offsets into the piece of W
    cut(min(rows > 0 ? PIECE_BYTES / (rows * 2) : vp, ((int64_t)1 << 30) / ldw));
    p.g = take(rows * p.piece * 2);
    p.ld_colsum = p.piece;
    p.colsum = take((rows / 64) * p.piece * 4);
    // dh = G W has few tiles and a long k, which is split: so that half of the CUs have a workgroup (dW's take the rest of them) or,
    // where its parts would be longer than 64 K tiles, up to all; (large) as the schedule on the device finds best, within this many
    // fp32 partials of the rows.  A step, us, all CUs / half: 19 rows of V 30 522 68 / 65, 64 rows (V 40 000, H 1024) 102 / 97, 1000 rows
    // (V 2 000, H 512) 68 / 64; 4000 rows (V 30 522, H 192) 421 / 473
    const int64_t tiles = ((int64_t)n + p.tile_rows - 1) / p.tile_rows * ((hidden + 127) / 128), parts = p.piece / BK / 64;
    int64_t s = tiles > 0 ? (p.large ? 256 : 128) / tiles : 1;
    if (!p.large && tiles > 0 && s < parts) s = parts < 256 / tiles ? parts : 256 / tiles;
    if (s > p.piece / 256) s = p.piece / 256;
    p.splits = (int32_t)(s < 1 ? 1 : s);
    p.dh_slot = rows * hidden;
    int64_t room = p.splits * p.dh_slot;
    if (p.large) {
      const int64_t tiles8 = (rows / 256) * ((hidden + 255) / 256);
      room = (tiles8 > 256 ? 2 * tiles8 : 512) * 65536;
    }
    p.dh_part = take((size_t)room * 4);
    p.dh_room = room;
    if (p.large && n >= 1024 && p.pieces == 1 && vp / 256 * ((hidden + 255) / 256) <= 256) {
      p.dw_room = 512 * 65536;
      p.dw_part = take((size_t)p.dw_room * 4);
    }
  }
  p.bytes = at;
  return p;
}
#endif

namespace {

hipError_t device_cus(int* out) {
  static DeviceOnce once;
  return once.get([](int dev, int* val) { return hipDeviceGetAttribute(val, hipDeviceAttributeMultiprocessorCount, dev); }, out);
}

// More rows than this: copied by workgroups of 64 rows, each of which counts all rows' states, instead of 16; and more than this
// are counted by a kernel of their own.  A forward of 15 % live rows (V 2 000, H 256), us, 16 rows / 64 rows / 64 rows and a
// counting kernel: n 4096 17 / 21 / -, 8192 25 / 26 / -, 16 384 36 / 30 / -, 32 768 64 / 41 / 53, 65 536 172 / 85 / 96
constexpr int PACK_WIDE = 8192, PACK_COUNTS = 65536;
// what the forward and the backward begin with: the teacher's lists, and the live rows side by side
template <bool GRAD>
hipError_t gather_rows(VocabRows& a, const VocabPlan& p, char* base, bool& few, hipStream_t st) {
  VocabHead* head = reinterpret_cast<VocabHead*>(base + p.head);
  a.head = head;
  a.tile_rows = p.tile_rows;
  a.count = &head->count;
  a.grad_max = &head->grad_max;
  a.out_scale = head->out_scale;
  a.schedule = head->schedule;
  a.row_map = reinterpret_cast<int32_t*>(base + p.row_map);
  a.x = reinterpret_cast<bf16_t*>(base + p.x);
  if (a.t_index) {
    // kept by the forward for the backward: scores [n, k], p [n, k], states [n]
    float* kept = GRAD ? const_cast<float*>(a.target_in) : a.target;
    a.t_p = kept + (int64_t)a.n * a.k;
    a.state = reinterpret_cast<int32_t*>(kept + (int64_t)a.n * a.k * 2);
    if (!GRAD && a.n > 0) {
      a.t_logp = reinterpret_cast<float*>(base + p.t_logp);
      const auto kfn = a.k > 64 ? vocab_teacher_kernel<16> : vocab_teacher_kernel<1>;
      hipLaunchKernelGGL(kfn, dim3((a.n + 3) / 4), dim3(256), 0, st, a);
      TRY(hipGetLastError());
    }
  }
  // few rows, read in place by the product kernel (16-byte loads, 31-bit offsets): no kernel of their own
  few = p.tile_rows == 64 && a.n > 0;
  if (few) {
    if (!a.h_aligned || ((int64_t)(a.n - 1) * a.ldh + a.hidden) * 2 >= (1ll << 31)) {   // ... but these, copied to where they can be
      bf16_t* to = a.x + (int64_t)128 * a.hidden;   // (x has room for 256 rows, of which the products of few rows use 128)
      hipLaunchKernelGGL(vocab_copy_kernel, dim3(a.n), dim3(256), 0, st, a.h, a.ldh, to, a.hidden);
      TRY(hipGetLastError());
      a.h = to;
      a.ldh = a.hidden;
    }
    return hipSuccess;
  }
  if (a.n > PACK_COUNTS) {
    a.block_base = reinterpret_cast<int32_t*>(base + p.block_base);
    hipLaunchKernelGGL(vocab_scan_kernel<GRAD>, dim3(1), dim3(1024), 0, st, a);
    TRY(hipGetLastError());
  }
  if (a.n > PACK_WIDE) {
    hipLaunchKernelGGL((vocab_pack_kernel<GRAD, 1024>), dim3((a.n + 63) / 64), dim3(1024), 0, st, a);
    return hipGetLastError();
  }
  int groups = a.n > 0 ? (a.n + 15) / 16 : 1;
  if (GRAD && a.fix && groups < 64) groups = 64;   // (they clear its table, too)
  hipLaunchKernelGGL((vocab_pack_kernel<GRAD, 256>), dim3(groups), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace

hipError_t KSET::launch_vocab_loss(const VocabRows& rows, const VocabPlan& p, void* work, hipStream_t st) {
  VocabRows a = rows;
  char* base = static_cast<char*>(work);
  float2 *part = reinterpret_cast<float2*>(base + p.part), *joined = reinterpret_cast<float2*>(base + p.joined);
  bool few;
  TRY(gather_rows<false>(a, p, base, few, st));
  if (a.n > 0) {
    VocabGemm g = {};
    g.x = a.x; g.w = a.w; g.bias = a.bias; g.ldw = a.ldw; g.vocab = a.vocab; g.hidden = a.hidden; g.count = a.count;
    g.scale2 = LOG2E * a.inv_t;
    g.part = part;
    g.n_part = (int)(p.piece / 64);
    for (int64_t v0 = 0; v0 < a.vocab; v0 += p.piece) {   // (one piece: as a rule)
      const int cols = (int)((min(p.piece, a.vocab - v0) + 255) / 256 * 256);
      g.v0 = v0;
      g.tiles_n = cols / (p.large ? 256 : 128);
      TRY(p.large ? launch_vocab8(V_STATS, g, st) : launch_scores<V_STATS>(g, a, few, st));
      if (p.pieces > 1) {
        hipLaunchKernelGGL(vocab_join_kernel, dim3((a.n + 3) / 4), dim3(256), 0, st, a.count, part, g.n_part, cols / 64, joined, v0 > 0 ? 1 : 0);
        TRY(hipGetLastError());
      }
    }
    if (p.pieces > 1) {
      part = joined;
      g.n_part = 1;
    }
    if (few) a.x = nullptr;   // rows stay where they are
    // (a loss of 15 % live rows, us, summed by the last workgroup / by a kernel more: n 1100 23.8 / 24.8, 1500 24.9 / 24.9,
    // 2048 27.0 / 25.4: every workgroup's count is an atomic on one word)
    if (a.loss && a.n <= 1024) a.done = &reinterpret_cast<VocabHead*>(base + p.head)->done;
    if (a.t_index && a.k > 16) hipLaunchKernelGGL(vocab_distill_kernel<4>, dim3(a.n), dim3(256), 0, st, a, part, g.n_part);
    else if (a.t_index) hipLaunchKernelGGL(vocab_distill_kernel<1>, dim3((a.n + 3) / 4), dim3(256), 0, st, a, part, g.n_part);
    else hipLaunchKernelGGL(vocab_ce_kernel, dim3((a.n + 3) / 4), dim3(256), 0, st, a, part, g.n_part);
    TRY(hipGetLastError());
  }
  if (a.loss && !a.done) {
    hipLaunchKernelGGL(vocab_reduce_kernel, dim3(1), dim3(1024), 0, st, a);
    TRY(hipGetLastError());
  }
  return hipSuccess;
}

hipError_t KSET::launch_vocab_grad(const VocabRows& rows, const VocabPlan& p, bf16_t* dw, int64_t ld_dw, void* work, hipStream_t st) {
  VocabRows a = rows;
  char* base = static_cast<char*>(work);
  a.row_info = reinterpret_cast<float4*>(base + p.row_info);
  if (a.t_index) {
    a.row_lc = reinterpret_cast<float4*>(base + p.row_lc);
    a.row_fix = reinterpret_cast<float2*>(base + p.row_fix);
    a.fix = a.dbias ? reinterpret_cast<int64_t*>(base + p.fix) : nullptr;
  }
  a.with_dw = dw != nullptr;
  a.dh_aligned = ((uintptr_t)a.dh & 7) == 0 && a.ld_dh % 4 == 0;
  a.max_splits = p.splits;
  a.tiles_h = p.large ? (a.hidden + 255) / 256 : (a.hidden + 127) / 128;
  if (p.large) {
    TRY(device_cus(&a.wgs));
    a.wgs &= ~7;
    a.dh_room = p.dh_room;
    a.dw_room = p.dw_room;
    a.piece_tiles[0] = (int32_t)(p.piece / 256);
    a.piece_tiles[1] = (int32_t)((a.vocab - (p.pieces - 1) * p.piece + 255) / 256);
  }
  bool few;
  TRY(gather_rows<true>(a, p, base, few, st));
  a.low = few;
  VocabGemm g = {};
  g.x = a.x; g.w = a.w; g.bias = a.bias; g.ldw = a.ldw; g.vocab = a.vocab; g.hidden = a.hidden; g.count = a.count;
  g.scale2 = LOG2E * a.inv_t;
  g.g = reinterpret_cast<bf16_t*>(base + p.g);
  g.row_info = a.row_info;
  g.colsum = a.dbias ? reinterpret_cast<float*>(base + p.colsum) : nullptr;
  g.ld_colsum = p.ld_colsum;
  g.out32 = reinterpret_cast<float*>(base + p.dh_part);
  g.dw32 = reinterpret_cast<float*>(base + p.dw_part);
  g.slot_stride = p.dh_slot;
  g.out16 = dw; g.ldo = ld_dw;
  g.wide = ((uintptr_t)dw & 15) == 0 && ld_dw % 8 == 0;
  g.out_scale = a.out_scale;
  g.with_dw = dw != nullptr;
  g.low = few;
  g.with_dh = a.dh && a.n > 0;
  auto finish = [&](int row_blocks, int dw_blocks, int64_t v0, int64_t v1) -> hipError_t {
    const int b_blocks = a.dbias ? (int)((v1 - v0 + 255) / 256) : 0;
    if (row_blocks + b_blocks + dw_blocks == 0) return hipSuccess;
    hipLaunchKernelGGL(vocab_finish_kernel, dim3(row_blocks + b_blocks + dw_blocks), dim3(256), 0, st, a, p, g.out32, g.colsum, g.dw32, dw,
                       ld_dw, row_blocks, dw_blocks, v0, v1);
    return hipGetLastError();
  };
  int64_t v0 = 0;
  for (int64_t piece = 0;; ++piece, v0 += p.piece) {
    const int64_t v1 = v0 + p.piece < a.vocab ? v0 + p.piece : a.vocab;
    g.v0 = v0;
    g.ldg = (int)((v1 - v0 + 255) / 256 * 256);
    g.schedule = a.schedule + (piece == p.pieces - 1 && piece > 0);
    g.accumulate = piece > 0;
    if (a.n > 0) {
      g.tiles_n = g.ldg / (p.large ? 256 : 128);
      TRY(p.large ? launch_vocab8(V_GRAD, g, st) : launch_scores<V_GRAD>(g, a, few, st));
      if (a.t_index) {
        const auto kfn = a.k > 64 ? vocab_teacher_hash_kernel : vocab_teacher_grad_kernel;
        hipLaunchKernelGGL(kfn, dim3(a.k > 64 ? a.n : (a.n + 3) / 4), dim3(256), 0, st, a, g.g, (int64_t)g.ldg, v0, v1, piece == 0 ? 1 : 0);
        TRY(hipGetLastError());
      }
    }
    g.tiles_n = a.tiles_h;
    TRY(p.large ? launch_vocab8(V_PROD, g, st) : launch_products(g, p, a.n, st));
    if (v1 == a.vocab) break;
    TRY(finish(0, 0, v0, v1));   // db of this piece: the next one's column sums take the place of its own
  }
  const int row_blocks = g.with_dh ? (int)min((int64_t)2048, ((int64_t)a.n * (a.hidden / 4) + 255) / 256) : 0;
  TRY(finish(row_blocks, dw && p.dw_room > 0 ? 1024 : 0, v0, a.vocab));
  return hipSuccess;
}
