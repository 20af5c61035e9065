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
// range holds it (times 2^15 there: softmax values down to 2e-9 stay normal numbers); the factor is put back in fp32 when
// the products are stored.
// Rows that take no part (ignored label, empty teacher list) are dropped first: the live rows are copied side by side, so
// their products cost nothing and whatever a dropped row holds (NaN included) reaches no gradient.
#include "vocab.h"

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
      if (TR) {
        const int k = at / (2 * R), c = (at % (2 * R)) >> 4;
        off[p] = (uint32_t)(k * ld * 2) + ((((c >> 1) ^ tr_swz<R>(k)) << 1) | (c & 1)) * 16;
      } else {
        const int r = at >> 7, c = (at >> 4) & 7;
        off[p] = (uint32_t)(r * ld * 2) + swz128(r, c) * 16;
      }
    }
  }
  __device__ __forceinline__ void stage(uint32_t kt, uint32_t lds, int w) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) dma16(rsrc, off[p] + kt * step, lds + (w * PIECES + p) * 1024);
  }
  // MFMA operand of 16 rows starting at r0 (a multiple of 16), k 32 ks + 8 (lane >> 4) .. + 7
  static __device__ __forceinline__ opx8_t frag(const char* img, int r0, int ks, int lane) {
    const int fr = lane & 15, fq = lane >> 4;
    if (!TR) {
      const int r = r0 + fr;
      return *reinterpret_cast<const opx8_t*>(img + r * 128 + swz128(r, ks * 4 + fq) * 16);
    }
    const int qq = fr >> 2, pp = fr & 3, k = ks * 32 + fq * 8 + qq;   // (k + 4 has the same swizzle)
    const char* a = img + k * (2 * R) + ((r0 >> 4) ^ tr_swz<R>(k)) * 32 + pp * 8;
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(a));
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(a + 4 * 2 * R));
    const s16x8_t v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return *reinterpret_cast<const opx8_t*>(&v);
  }
};

// One output tile of BM x BN per workgroup of WM x WN waves (few rows: many small tiles; vocab8.hip takes the large calls).
template <int EPI, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void vocab_gemm_kernel(VocabGemm a) {
  constexpr int NW = WM * WN, MB = BM / WM / 16, NB = BN / WN / 16;
  constexpr bool A_TR = EPI == V_DW, B_TR = EPI == V_DH || EPI == V_DW;
  typedef Operand<BM, A_TR, NW> OA;
  typedef Operand<BN, B_TR, NW> OB;
  constexpr int STAGE = OA::BYTES + OB::BYTES;
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w / WN, wn = w % WN, fr = lane & 15, fq = lane >> 4;
  const int count = *a.count;                       // live rows
  const int tn = blockIdx.x % a.tiles_n, tm = blockIdx.x / a.tiles_n, split = blockIdx.y;
  if (EPI != V_DW && tm * BM >= count) return;      // workgroup-uniform

  int nt, kt0 = 0;
  OA oa;
  OB ob;
  if (EPI == V_STATS || EPI == V_GRAD) {
    nt = a.hidden / BK;
    oa.init(a.x + (int64_t)tm * BM * a.hidden, (int64_t)BM * a.hidden * 2, a.hidden, w, lane);
    const int64_t v0 = a.v0 + (int64_t)tn * BN;
    ob.init(a.w + v0 * a.ldw, ((a.vocab - 1 - v0) * a.ldw + a.hidden) * 2, a.ldw, w, lane);
  } else if (EPI == V_DH) {
    const int all = a.ldg / BK;
    kt0 = (int)((int64_t)all * split / gridDim.y);
    nt = (int)((int64_t)all * (split + 1) / gridDim.y) - kt0;
    oa.init(a.g + (int64_t)tm * BM * a.ldg + (int64_t)kt0 * BK, (int64_t)BM * a.ldg * 2, a.ldg, w, lane);
    const int64_t v0 = a.v0 + (int64_t)kt0 * BK;
    ob.init(a.w + v0 * a.ldw + tn * BN, ((a.vocab - 1 - v0) * a.ldw + a.hidden - tn * BN) * 2, a.ldw, w, lane);
  } else {
    nt = (count + BK - 1) / BK;
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
  if (nt > 0) {
    oa.stage(0, lds0, w);
    ob.stage(0, lds0 + OA::BYTES, w);
  }
  for (int kt = 0; kt < nt; ++kt) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();   // the tile is in LDS; every wave has read the buffer that is filled next
    const char* buf = smem + (kt & 1) * STAGE;
    if (kt + 1 < nt) {
      const uint32_t nxt = lds0 + ((kt + 1) & 1) * STAGE;
      oa.stage(kt + 1, nxt, w);
      ob.stage(kt + 1, nxt + OA::BYTES, w);
    }
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
      const float4 rc = a.row_coef[r];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float g[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          g[e] = __builtin_amdgcn_exp2f(fmaf(acc[m][n][e], a.scale2, -rc.x)) * rc.y;
          cs[n][e] += g[e];
        }
        *reinterpret_cast<uint2*>(a.g + (int64_t)r * a.ldg + col0 + n * 16) = make_uint2(pack_op2(g[0], g[1]), pack_op2(g[2], g[3]));
      }
    }
    if (a.colsum) {   // fp32 column sums of what was rounded above: db is not made of rounded values
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        f32x4_t t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = fr_sum(cs[n][e]);
        if (fr == 0)
          *reinterpret_cast<f32x4_t*>(a.colsum + (int64_t)(tm * WM + wm) * a.ld_colsum + a.v0 + col0 + n * 16) = t;
      }
    }
  } else if (EPI == V_DH) {
    float* out = a.out32 + (int64_t)split * a.slot_stride;
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n)
        if (col0 + n * 16 < a.hidden)
          *reinterpret_cast<f32x4_t*>(out + (int64_t)(row0 + m * 16) * a.hidden + col0 + n * 16) = acc[m][n];
  } else {
    const float s = a.out_scale[0];
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const int64_t v = a.v0 + row0 + m * 16;
      if (v < a.vocab && row0 + m * 16 < a.ldg) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
          if (col0 + n * 16 < a.hidden)
            *reinterpret_cast<uint2*>(a.out16 + v * a.ldo + col0 + n * 16) =
                make_uint2(pack_op2(acc[m][n][0] * s, acc[m][n][1] * s), pack_op2(acc[m][n][2] * s, acc[m][n][3] * s));
      }
    }
  }
}

// ---- block-wide sums (256 threads) through LDS, every thread gets the result; fixed order
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}
__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// Teacher lists of a distillation: p = softmax(values / T) over a row's entries with index >= 0 and a value above -inf
// (0 elsewhere), log_p beside it, state[row] = 0 no entry, 1 live, 2 an index beyond the vocabulary or a value that is
// NaN or +inf.  One wave per row.
__global__ __launch_bounds__(256) void vocab_teacher_kernel(VocabRows a) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= a.n) return;
  const float* t = a.t_values + (int64_t)row * a.ld_t;
  const int64_t* ix = a.t_index + (int64_t)row * a.ld_ti;
  float mx = -INFINITY;
  int n_in = 0, bad = 0;
  auto in_list = [&](int j) { return ix[j] >= 0 && t[j] != -INFINITY; };
  for (int j = lane; j < a.k; j += 64)
    if (in_list(j)) {
      mx = fmaxf(mx, t[j] * a.inv_t);
      ++n_in;
      bad |= ix[j] >= a.vocab;
    }
  mx = wave_max(mx);
  const float ref = mx == -INFINITY ? 0.f : mx;
  float s = 0.f;
  for (int j = lane; j < a.k; j += 64)
    if (in_list(j)) s += expf(t[j] * a.inv_t - ref);
  s = wave_sum(s);
  bad |= !(s < INFINITY);   // a NaN or +inf among the teacher's values
  const float log_s = logf(s);
  for (int j = lane; j < a.k; j += 64) {
    const bool in = in_list(j);
    const float lp = t[j] * a.inv_t - ref - log_s;
    a.t_p[(int64_t)row * a.k + j] = in ? expf(t[j] * a.inv_t - ref) / s : 0.f;
    if (a.t_logp) a.t_logp[(int64_t)row * a.k + j] = lp;
  }
  const bool any_in = __any(n_in), any_bad = __any(bad);
  if (lane == 0) a.state[row] = any_bad ? 2 : (any_in ? 1 : 0);
}

// dh = G W over one piece has (rows / 256)(hidden / 256) tiles and a long k of `pairs` x 128: it is cut into the number of
// splits that fills the persistent workgroups best, a round of them costing its k plus about 8 pairs' time for the fp32
// partials (256 KiB a tile, written here and read by the last kernel).
__device__ int choose_splits(const VocabRows& a, int total, int pairs) {
  const int rows = (total + 255) & ~255, tiles = (rows >> 8) * a.split_tiles_n;
  if (tiles == 0) return 1;
  int64_t most = (int64_t)a.split_cap * 65536 / ((int64_t)rows * a.hidden);   // split_cap: 65536 floats of room each
  if (most > 64) most = 64;
  if (most > pairs) most = pairs;
  int best = 1, best_cost = 0x7fffffff;
  for (int s = 1; s <= (int)most; ++s) {
    const int cost = ((tiles * s + a.split_wgs - 1) / a.split_wgs) * ((pairs + s - 1) / s + 8);
    if (cost < best_cost) { best_cost = cost; best = s; }
  }
  return best;
}

// Live rows side by side: x[r] = hidden[row_map[r]], zero rows up to the next multiple of 256, count = how many.  One
// workgroup per 64 rows; each counts all rows' states itself (8 bytes a row from L2), so there is no scan kernel.
// Backward: also every live row's (lse, c), the common factor, zeroed gradients of the dropped rows and a zeroed table.
template <bool GRAD>
__global__ __launch_bounds__(256) void vocab_pack_kernel(VocabRows a) {
  __shared__ float red[4];
  __shared__ int rows[64], n_rows, before_s[4], total_s[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, r0 = blockIdx.x * 64;
  auto state_of = [&](int r) -> int {
    if (a.state) return a.state[r];
    const int64_t y = a.labels[r];
    return y == a.ignore ? 0 : (y < 0 || y >= a.vocab ? 2 : 1);
  };
  int before = 0, total = 0;
  float gm = 0.f;
  for (int r = tid; r < a.n; r += 256) {
    const int live = state_of(r) != 0;
    total += live;
    before += live && r < r0;
    if (GRAD && a.grad_rows && live) {
      const float g = fabsf(a.grad[r]);
      if (g < INFINITY) gm = fmaxf(gm, g);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    before += __shfl_xor(before, o, 64);
    total += __shfl_xor(total, o, 64);
  }
  if (lane == 0) { before_s[w] = before; total_s[w] = total; }
  if (GRAD && a.grad_rows) gm = block_max(gm, red);
  __syncthreads();
  before = before_s[0] + before_s[1] + before_s[2] + before_s[3];
  total = total_s[0] + total_s[1] + total_s[2] + total_s[3];
  // the factor common to all rows; c = what is left of a row's gradient, |c| <= 1
  float common = 1.f;
  if (GRAD) {
    if (a.grad_rows) {
      common = gm;
    } else {
      common = a.grad[0];
    }
  }
  if (blockIdx.x == 0 && tid == 0) {
    *a.count = total;
    if (GRAD) {
      const float f = common * a.grad_factor / (a.mean ? (float)max(total, 1) : 1.f);   // no live row: zeros, not 0 / 0
      a.out_scale[0] = f / G_SCALE;
      a.out_scale[1] = f;
      for (int i = 0; i < 2; ++i) a.splits[i] = a.split_wgs ? choose_splits(a, total, a.split_pairs[i]) : a.split_cap;
    }
  }
  if (w == 0) {
    const int r = r0 + lane;
    const int st = r < a.n ? state_of(r) : 0;
    const unsigned long long m = __ballot(st != 0);
    const int local = __popcll(m & ((1ull << lane) - 1)), rank = before + local;
    if (st != 0) {
      rows[local] = r;
      a.row_map[rank] = st == 2 ? ~r : r;    // a row whose target is outside the vocabulary: NaN loss and gradients
      if (GRAD) {
        float c = 1.f;
        if (a.grad_rows) {
          const float g = a.grad[r];
          c = fabsf(g) < INFINITY ? (common > 0.f ? g / common : 0.f) : g;
        }
        if (st == 2) c = __builtin_nanf("");
        const float l2 = a.lse[r] * LOG2E;
        // G = y exp2(z log2(e) / T - x): x takes |c| (and G's scale), y its sign
        a.row_coef[rank] = make_float4(l2 - log2f(fabsf(c) * G_SCALE), c < 0.f ? -1.f : 1.f, l2, c);
      }
    } else if (r < a.n && !GRAD) {
      a.row_loss[r] = 0.f;
      a.lse_out[r] = 0.f;
    }
    if (lane == 0) n_rows = __popcll(m);
  }
  __syncthreads();
  const int H = a.hidden;
  for (int i = w; i < n_rows; i += 4) {
    const bf16_t* src = a.h + (int64_t)rows[i] * a.ldh;
    bf16_t* dst = a.x + (int64_t)(before + i) * H;
    if (a.h_aligned)
      for (int c = lane * 8; c < H; c += 512) *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
    else
      for (int c = lane; c < H; c += 64) dst[c] = src[c];
  }
  const int pad = (total + 255) & ~255;
  for (int r = total + blockIdx.x * 4 + w; r < pad; r += gridDim.x * 4) {
    for (int c = lane * 8; c < H; c += 512) *reinterpret_cast<uint4*>(a.x + (int64_t)r * H + c) = make_uint4(0, 0, 0, 0);
    if (GRAD && lane == 0) a.row_coef[r] = make_float4(INFINITY, 1.f, 0.f, 0.f);   // G = 0
  }
  if (GRAD) {
    if (a.dh)
      for (int i = w; i < 64 && r0 + i < a.n; i += 4)
        if (state_of(r0 + i) == 0)
          for (int c = lane; c < H; c += 64) a.dh[(int64_t)(r0 + i) * a.ld_dh + c] = 0;
    if (a.fix)
      for (int64_t v = (int64_t)blockIdx.x * 256 + tid; v < a.vocab; v += (int64_t)gridDim.x * 256) a.fix[v] = 0;
  }
}

// score (times 1/T) of one vocabulary entry for the hidden row x: a wave's dot product, fp32
__device__ __forceinline__ float wave_score(const bf16_t* x, const bf16_t* wrow, int H, int lane) {
  float s = 0.f;
  for (int c = lane * 8; c < H; c += 512) {
    const uint4 xv = *reinterpret_cast<const uint4*>(x + c), wv = *reinterpret_cast<const uint4*>(wrow + c);
    const uint32_t* xp = reinterpret_cast<const uint32_t*>(&xv);
    const uint32_t* wp = reinterpret_cast<const uint32_t*>(&wv);
#pragma unroll
    for (int i = 0; i < 4; ++i) s = fmaf(op2_lo(xp[i]), op2_lo(wp[i]), fmaf(op2_hi(xp[i]), op2_hi(wp[i]), s));
  }
  return wave_sum(s);
}

// One workgroup per live row: lse from the tiles' (max, sum) pairs, the targets' scores, the row's loss.
__global__ __launch_bounds__(256) void vocab_loss_kernel(VocabRows a, const float2* __restrict__ part, int n_part) {
  __shared__ float red[4];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  if (r >= *a.count) return;
  const int mapped = a.row_map[r], row = mapped < 0 ? ~mapped : mapped;
  const float2* p = part + (int64_t)r * n_part;
  float mx = -INFINITY;
  for (int i = tid; i < n_part; i += 256) mx = fmaxf(mx, p[i].x);
  mx = block_max(mx, red);
  const float ref = mx == -INFINITY ? 0.f : mx;
  float s = 0.f;
  for (int i = tid; i < n_part; i += 256) s += p[i].y * __builtin_amdgcn_exp2f(p[i].x - ref);
  s = block_sum(s, red);
  const float lse = LN2 * (ref + log2f(s));
  const bf16_t* x = a.x + (int64_t)r * a.hidden;
  float loss = 0.f;
  if (mapped < 0) {
    loss = __builtin_nanf("");
  } else if (a.state) {
    for (int j = w; j < a.k; j += 4) {
      const int64_t v = a.t_index[(int64_t)row * a.ld_ti + j];
      float z = 0.f;
      if (v >= 0) {
        z = (wave_score(x, a.w + v * a.ldw, a.hidden, lane) + (a.bias ? a.bias[v] : 0.f)) * a.inv_t;
        const float pj = a.t_p[(int64_t)row * a.k + j];
        if (pj != 0.f) loss += pj * (a.t_logp[(int64_t)row * a.k + j] - z + lse);
      }
      if (lane == 0) a.target[(int64_t)row * a.k + j] = z;
    }
    __syncthreads();
    if (lane == 0) red[w] = loss;
    __syncthreads();
    loss = ((red[0] + red[1]) + (red[2] + red[3])) * a.loss_factor;
  } else if (w == 0) {
    const int64_t v = a.labels[row];
    const float z = wave_score(x, a.w + v * a.ldw, a.hidden, lane) + (a.bias ? a.bias[v] : 0.f);
    if (lane == 0) a.target[row] = z;
    loss = lse - z;
  }
  if (tid == 0) {
    a.row_loss[row] = loss;
    a.lse_out[row] = lse;
  }
}

// loss[0] = sum of the rows' losses, over the live rows' count for the mean (0 / 0 = NaN as torch's mean over none);
// one workgroup, fixed order
__global__ __launch_bounds__(256) void vocab_reduce_kernel(VocabRows a) {
  __shared__ float red[4];
  float s = 0.f;
  for (int i = threadIdx.x; i < a.n; i += 256) s += a.row_loss[i];
  s = block_sum(s, red);
  if (threadIdx.x == 0) a.loss[0] = a.mean ? s / (float)*a.count : s;
}

// The targets' part of G, one wave per live row: G[r, v] = c (q_v - sum of p over the entries that name v), from the
// forward's fp32 score of v (a difference of the rounded q would lose what is left where q is near p).  The sums of the
// targets per vocabulary entry, which db needs, go to a table of 64-bit fixed point: integer adds commute, so their
// order does not show (2^-38 a unit; p <= 1, n <= 2^24 rows).
__global__ __launch_bounds__(256) void vocab_targets_kernel(VocabRows a, bf16_t* __restrict__ g, int64_t ldg, int64_t v0, int64_t v1,
                                                            int table) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= *a.count) return;
  const int row = a.row_map[r];
  if (row < 0) return;
  const float4 rc = a.row_coef[r];
  for (int j = lane; j < a.k; j += 64) {
    const int64_t v = a.state ? a.t_index[(int64_t)row * a.ld_ti + j] : a.labels[row];
    if (v < 0) continue;
    float p = 1.f;
    if (a.state) {
      const float own = a.t_p[(int64_t)row * a.k + j];
      p = 0.f;
      for (int i = 0; i < a.k; ++i)
        if (a.t_index[(int64_t)row * a.ld_ti + i] == v) p += a.t_p[(int64_t)row * a.k + i];
      if (table && fabsf(rc.w * own) <= 1.f)
        atomicAdd(reinterpret_cast<unsigned long long*>(a.fix + v), (unsigned long long)__double2ll_rn((double)(rc.w * own) * FIX));
    } else if (table && fabsf(rc.w) <= 1.f) {
      atomicAdd(reinterpret_cast<unsigned long long*>(a.fix + v), (unsigned long long)__double2ll_rn((double)rc.w * FIX));
    }
    if (v < v0 || v >= v1) continue;
    const float q = __builtin_amdgcn_exp2f(a.target_in[(int64_t)row * a.k + j] * LOG2E - rc.z);
    g[(int64_t)r * ldg + (v - v0)] = f32_to_op(rc.w * (q - p) * G_SCALE);
  }
}

// dh of the live rows from the fp32 partials (fixed order), and db from the column sums and the targets' table
__global__ __launch_bounds__(256) void vocab_finish_kernel(VocabRows a, VocabPlan p, const float* __restrict__ part,
                                                           const float* __restrict__ colsum, int row_blocks) {
  const int count = *a.count;
  if ((int)blockIdx.x < row_blocks) {
    const int64_t total = (int64_t)count * (a.hidden / 4);
    const int64_t slot = p.large ? (int64_t)((count + 255) & ~255) * a.hidden : p.dh_slot;
    const float s = a.out_scale[0];
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)row_blocks * 256) {
      const int r = (int)(i / (a.hidden / 4)), c = (int)(i % (a.hidden / 4)) * 4;
      f32x4_t v = {0.f, 0.f, 0.f, 0.f};
      for (int64_t piece = 0; piece < p.pieces; ++piece) {
        const int n = a.splits[piece == p.pieces - 1];
        const float* q = part + piece * p.dh_piece + (int64_t)r * a.hidden + c;
        for (int k = 0; k < n; ++k) v += *reinterpret_cast<const f32x4_t*>(q + k * slot);
      }
      const int m = a.row_map[r];
      bf16_t* o = a.dh + (int64_t)(m < 0 ? ~m : m) * a.ld_dh + c;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = f32_to_op(v[e] * s);
    }
  } else {
    const int64_t v = (int64_t)(blockIdx.x - row_blocks) * 256 + threadIdx.x;
    if (v >= a.vocab) return;
    const int n_sums = p.large ? (count + 255) / 256 * 2 : (count + 127) / 128 * 2;
    float s = 0.f;
    for (int k = 0; k < n_sums; ++k) s += colsum[(int64_t)k * p.ld_colsum + v];
    // (s is in units of G, the table in units of c)
    a.dbias[v] = (float)((double)s / G_SCALE - (double)a.fix[v] / FIX) * a.out_scale[1];
  }
}

constexpr int T_BM = 128, T_BN = 128;

template <int EPI>
hipError_t launch_tiles(const VocabGemm& g, int tiles_m, int splits, hipStream_t st) {
  hipLaunchKernelGGL((vocab_gemm_kernel<EPI, T_BM, T_BN, 2, 2>), dim3(tiles_m * g.tiles_n, splits), dim3(256), 0, st, g);
  return hipGetLastError();
}

}  // namespace

#if !CLIP_OPERAND_F16
// G of one piece of the vocabulary may take this much: the pieces are as few as that allows
constexpr int64_t G_BYTES = 512ll << 20;

// From here on the 256 x 256 tiles
constexpr int LARGE_ROWS = 256;

VocabPlan vocab_plan(int32_t n, int64_t vocab, int32_t hidden, int64_t ldw, int32_t k, bool distill, bool grad) {
  VocabPlan p = {};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) & ~(size_t)255;
    return o;
  };
  p.large = n > LARGE_ROWS && hidden % 128 == 0;
  const int64_t rows = ((int64_t)n + 255) / 256 * 256, vp = (vocab + 255) / 256 * 256;
  p.count = take(4);
  p.out_scale = take(16);   // and V_DH's splits
  p.row_map = take(rows * 4);
  if (distill) {
    p.state = take(rows * 4);
    p.t_p = take((size_t)n * k * 4);
    if (!grad) p.t_logp = take((size_t)n * k * 4);
  }
  p.x = take(rows * hidden * 2);
  if (!grad) {
    p.part = take(rows * (vp / 64) * 8);
  } else {
    p.row_coef = take(rows * 16);
    p.fix = take(vocab * 8);
    // a piece: whole 256-column tiles, G within its bound, 32-bit byte offsets into the piece of W
    int64_t piece = rows > 0 ? G_BYTES / (rows * 2) : vp;
    if (piece > (1ll << 30) / ldw) piece = (1ll << 30) / ldw;
    piece = piece / 256 * 256;
    if (piece < 256) piece = 256;
    if (piece > vp) piece = vp;
    p.pieces = (vp + piece - 1) / piece;
    p.piece = ((vp / 256 + p.pieces - 1) / p.pieces) * 256;   // of about the same size
    p.pieces = (vp + p.piece - 1) / p.piece;
    p.g = take(rows * p.piece * 2);
    p.ld_colsum = vp;
    p.colsum = take((rows / 64) * vp * 4);
    // dh = G W has few tiles and a long k: the vocabulary is split until every CU has two workgroups
    const int64_t tiles = (rows / 128) * ((hidden + 127) / 128);
    int64_t s = tiles > 0 ? (512 + tiles - 1) / tiles : 1;
    if (s > p.piece / 256) s = p.piece / 256;
    p.splits = (int32_t)(s < 1 ? 1 : s);
    p.dh_slot = rows * hidden;
    p.dh_piece = p.splits * p.dh_slot;
    if (p.large) {   // room for the splits that few live rows call for
      const int64_t tiles8 = (rows / 256) * ((hidden + 255) / 256);
      p.dh_piece = (tiles8 > 256 ? 2 * tiles8 : 512) * 65536;
      if (p.dh_piece < p.dh_slot) p.dh_piece = p.dh_slot;
    }
    p.dh_part = take((size_t)p.pieces * p.dh_piece * 4);
  }
  p.bytes = at;
  return p;
}
#endif

#define TRY(expr)                          \
  do {                                     \
    hipError_t _e = (expr);                \
    if (_e != hipSuccess) return _e;       \
  } while (0)

hipError_t KSET::launch_vocab_loss(const VocabRows& rows, const VocabPlan& p, void* work, hipStream_t st) {
  VocabRows a = rows;
  char* base = static_cast<char*>(work);
  a.count = reinterpret_cast<int32_t*>(base + p.count);
  a.row_map = reinterpret_cast<int32_t*>(base + p.row_map);
  a.x = reinterpret_cast<bf16_t*>(base + p.x);
  float2* part = reinterpret_cast<float2*>(base + p.part);
  if (a.t_index) {
    a.state = reinterpret_cast<int32_t*>(base + p.state);
    a.t_p = reinterpret_cast<float*>(base + p.t_p);
    a.t_logp = reinterpret_cast<float*>(base + p.t_logp);
    if (a.n > 0) {
      hipLaunchKernelGGL(vocab_teacher_kernel, dim3((a.n + 3) / 4), dim3(256), 0, st, a);
      TRY(hipGetLastError());
    }
  }
  hipLaunchKernelGGL(vocab_pack_kernel<false>, dim3(a.n > 0 ? (a.n + 63) / 64 : 1), dim3(256), 0, st, a);
  TRY(hipGetLastError());
  if (a.n > 0) {
    VocabGemm g = {};
    g.x = a.x; g.w = a.w; g.bias = a.bias; g.ldw = a.ldw; g.vocab = a.vocab; g.hidden = a.hidden; g.count = a.count;
    g.scale2 = LOG2E * a.inv_t;
    g.part = part;
    g.n_part = (int)((a.vocab + 255) / 256 * 4);   // 64 columns each
    if (p.large) {
      g.tiles_n = (int)((a.vocab + 255) / 256);
      TRY(launch_vocab8(V_STATS, g, st));
    } else {
      g.tiles_n = g.n_part / 2;
      TRY(launch_tiles<V_STATS>(g, (a.n + T_BM - 1) / T_BM, 1, st));
    }
    hipLaunchKernelGGL(vocab_loss_kernel, dim3(a.n), dim3(256), 0, st, a, part, g.n_part);
    TRY(hipGetLastError());
  }
  if (a.loss) {
    hipLaunchKernelGGL(vocab_reduce_kernel, dim3(1), dim3(256), 0, st, a);
    TRY(hipGetLastError());
  }
  return hipSuccess;
}

hipError_t KSET::launch_vocab_grad(const VocabRows& rows, const VocabPlan& p, bf16_t* dw, int64_t ld_dw, void* work, hipStream_t st) {
  VocabRows a = rows;
  char* base = static_cast<char*>(work);
  a.count = reinterpret_cast<int32_t*>(base + p.count);
  a.out_scale = reinterpret_cast<float*>(base + p.out_scale);
  a.row_map = reinterpret_cast<int32_t*>(base + p.row_map);
  a.row_coef = reinterpret_cast<float4*>(base + p.row_coef);
  a.x = reinterpret_cast<bf16_t*>(base + p.x);
  a.fix = a.dbias ? reinterpret_cast<int64_t*>(base + p.fix) : nullptr;
  if (a.t_index) {
    a.state = reinterpret_cast<int32_t*>(base + p.state);
    a.t_p = reinterpret_cast<float*>(base + p.t_p);
    if (a.n > 0) {
      hipLaunchKernelGGL(vocab_teacher_kernel, dim3((a.n + 3) / 4), dim3(256), 0, st, a);
      TRY(hipGetLastError());
    }
  }
  a.splits = reinterpret_cast<int32_t*>(base + p.out_scale + 8);
  a.split_cap = p.splits;
  if (p.large) {
    static DeviceOnce once;
    TRY(once.get([](int dev, int* val) { return hipDeviceGetAttribute(val, hipDeviceAttributeMultiprocessorCount, dev); }, &a.split_wgs));
    a.split_wgs &= ~7;
    a.split_tiles_n = (a.hidden + 255) / 256;
    a.split_cap = (int32_t)(p.dh_piece / 65536);
    a.split_pairs[0] = (int32_t)(p.piece / 128);
    a.split_pairs[1] = (int32_t)((a.vocab - (p.pieces - 1) * p.piece + 255) / 256 * 2);
  }
  hipLaunchKernelGGL(vocab_pack_kernel<true>, dim3(a.n > 0 ? (a.n + 63) / 64 : 1), dim3(256), 0, st, a);
  TRY(hipGetLastError());
  VocabGemm g = {};
  g.x = a.x; g.w = a.w; g.bias = a.bias; g.ldw = a.ldw; g.vocab = a.vocab; g.hidden = a.hidden; g.count = a.count;
  g.scale2 = LOG2E * a.inv_t;
  g.g = reinterpret_cast<bf16_t*>(base + p.g);
  g.row_coef = a.row_coef;
  g.colsum = a.dbias ? reinterpret_cast<float*>(base + p.colsum) : nullptr;
  g.ld_colsum = p.ld_colsum;
  float* dh_part = reinterpret_cast<float*>(base + p.dh_part);
  g.slot_stride = p.dh_slot;
  g.out16 = dw; g.ldo = ld_dw;
  g.out_scale = a.out_scale;
  const int tiles_r = (a.n + T_BM - 1) / T_BM, tiles_h = (int)((a.hidden + (p.large ? 255 : T_BN - 1)) / (p.large ? 256 : T_BN));
  for (int64_t v0 = 0, piece = 0; v0 < a.vocab; v0 += p.piece, ++piece) {
    const int64_t v1 = v0 + p.piece < a.vocab ? v0 + p.piece : a.vocab;
    g.v0 = v0;
    g.ldg = (int)((v1 - v0 + 255) / 256 * 256);
    if (a.n > 0) {
      g.tiles_n = g.ldg / (p.large ? 256 : T_BN);
      TRY(p.large ? launch_vocab8(V_GRAD, g, st) : launch_tiles<V_GRAD>(g, tiles_r, 1, st));
      hipLaunchKernelGGL(vocab_targets_kernel, dim3((a.n + 3) / 4), dim3(256), 0, st, a, g.g, (int64_t)g.ldg, v0, v1,
                         (a.fix && piece == 0) ? 1 : 0);
      TRY(hipGetLastError());
    }
    g.tiles_n = tiles_h;
    if (a.dh && a.n > 0) {
      g.out32 = dh_part + piece * p.dh_piece;
      g.splits = a.splits + (piece == p.pieces - 1);
      TRY(p.large ? launch_vocab8(V_DH, g, st) : launch_tiles<V_DH>(g, tiles_r, p.splits, st));
    }
    if (dw) TRY(p.large ? launch_vocab8(V_DW, g, st) : launch_tiles<V_DW>(g, (g.ldg + T_BM - 1) / T_BM, 1, st));
  }
  const int row_blocks = a.dh && a.n > 0 ? (int)min((int64_t)2048, ((int64_t)a.n * (a.hidden / 4) + 255) / 256) : 0;
  const int b_blocks = a.dbias ? (int)((a.vocab + 255) / 256) : 0;
  if (row_blocks + b_blocks > 0) {
    hipLaunchKernelGGL(vocab_finish_kernel, dim3(row_blocks + b_blocks), dim3(256), 0, st, a, p, dh_part, g.colsum, row_blocks);
    TRY(hipGetLastError());
  }
  return hipSuccess;
}
