// The products of the decoder losses for large calls: 256 x 256 x 64 tiles on 8 waves, persistent workgroups, the ping-pong
// schedule of gemm8.hip (a K tile = four 16-KiB half-tiles by LDS-DMA into an 8-slot ring, two phases of 32 MFMAs per K tile,
// waves 4..7 one barrier behind waves 0..3, counted vmcnt waits) with what these products need beside it:
//  * either operand may lie R-major in memory ([K, R]: W in dh = G W, both in dW = G^T h).  Its half-tile is the same 16 KiB,
//    [64 k][128 x 2 B], read by ds_read_b64_tr_b16 in place of ds_read_b128: no transposed copy of W, h or G is ever made;
//  * loads go through a buffer descriptor, so the vocabulary may end anywhere (rows past the end read as zero);
//  * the number of live rows is read on the device: tiles past it are never visited;
//  * epilogues: (max, sum of exp2) per row and 64 columns; the 16-bit score gradients with their column sums; fp32 partials;
//    16-bit weight gradients;
//  * dW tiles and dh tiles share one launch: either alone leaves a last round of workgroups mostly idle.
// Bound: the matrix cores at the clock that the card's power limit leaves them (1.55 - 1.7 GHz in these loops, busy 68 % of the
// cycles); 256 x 256 tiles because each byte that a CU takes in feeds twice the MFMAs that it does in a 128 x 128 tile (of which
// two fit: 16 384 rows 4.6 ms instead of 2.7).  bf16, V 30 522, H 768, us (2 n V H, twice that for the pair; 1.29 PF is the rate
// of a large library product):
//   4096 rows:   scores 160 - 181 (1.06 - 1.20 PF), G 180 - 205 (0.94 - 1.07 PF; 250 MB leave it), dW + dh 339 - 382 (1.01 - 1.13 PF)
//   16 384 rows: scores 590 - 662 (1.16 - 1.30 PF), G 649 - 732 (1.05 - 1.18 PF; 1 GB leaves it), dW + dh 1220 - 1330 (1.15 - 1.26 PF)
// (averages on different boards; the first calls after a pause run slower)
#include "vocab.h"

namespace {

constexpr int BM = 256, BN = 256;
constexpr int HT = 16384;              // half-tile
constexpr int RING = 8 * HT;           // 2 K tiles
constexpr int SCR = 2048;              // epilogue scratch per wave
constexpr int SIDE = 1024 + 4096;      // of the next tile, by LDS-DMA: bias[256], row_info[256]
constexpr int LDS8 = RING + 8 * SCR + 2 * SIDE;

// where a staging cursor stands: the bytes from `at` on that may be read (saturated; every walk is shorter than 2^31)
struct Cursor {
  uint64_t at;
  uint32_t left;
  __device__ __forceinline__ void set(const void* p, int64_t bytes) {
    at = (uint64_t)p;
    left = bytes <= 0 ? 0u : (bytes > 0xfffffff0ll ? 0xfffffff0u : (uint32_t)bytes);
  }
  __device__ __forceinline__ void step(uint32_t by) {
    at += by;
    left = left > by ? left - by : 0u;
  }
  __device__ __forceinline__ u32x4_t rsrc(uint32_t ahead) const {
    const uint64_t p = at + ahead;
    u32x4_t r;
    r[0] = __builtin_amdgcn_readfirstlane((uint32_t)p);
    r[1] = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32) & 0xffffu);
    r[2] = __builtin_amdgcn_readfirstlane(left > ahead ? left - ahead : 0u);
    r[3] = 0x00020000u;
    return r;
  }
};

template <int EPI>
__global__ __launch_bounds__(512) void vocab8_kernel(VocabGemm a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr bool ROWS = EPI == V_STATS || EPI == V_GRAD;   // else V_PROD: dW tiles, then dh tiles

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = w >> 2, wc = w & 3;   // wr: barrier group AND 64-row block inside each A half
  char* scr = smem + RING + w * SCR;
  char* side = smem + RING + 8 * SCR;
  // What the K loop does not need is computed again, from the arguments in memory, where it is needed (at a change of tile
  // and in the epilogue): kept in registers it would be spilled, and the reloads wait for every staged half-tile
  typedef const __attribute__((address_space(4))) VocabGemm* Args;
  auto args = [&]() -> Args {
    Args p = (Args)__builtin_amdgcn_kernarg_segment_ptr();   // = &a: the only argument
    asm volatile("" : "+s"(p));
    return p;
  };
  const int count = __builtin_amdgcn_readfirstlane(*a.count);
  typedef const __attribute__((address_space(4))) VocabSchedule* Schedule;   // (scalar loads, where it is needed)
  const int G = gridDim.x;
  const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
  const int lin = xcd * (G >> 3) + slot;   // neighbours share an XCD
  const uint32_t ld_x = (uint32_t)a.hidden * 2, ld_g = (uint32_t)a.ldg * 2, ld_w = (uint32_t)a.ldw * 2;

  // ---- items of this workgroup: a dW or dh tile or one of scores (panel tm, column tile tn), K tiles kt0 .. kt0 + nt
  struct Item { bool dh, whole; int tm, tn, kt0, nt, split; };   // whole: a dW tile of all rows
  auto item = [&](int i, Item& o) -> bool {
    const auto& a = *args();
    const int tiles_r = (count + 255) >> 8, tiles_n = a.tiles_n;
    o.kt0 = o.split = 0;
    o.dh = o.whole = false;
    if (ROWS) {
      // the 8 XCDs take contiguous runs of the vocabulary's tiles, each its own part of W; within it column groups of 4 tiles
      // (their slice of W stays in this XCD's L2), all row panels of one before the next
      const int run = (tiles_n >> 3) + (xcd < (tiles_n & 7) ? 1 : 0), run0 = xcd * (tiles_n >> 3) + min(xcd, tiles_n & 7);
      const int q = slot + (G >> 3) * i;
      if (q >= run * tiles_r) return false;
      const int per_group = 4 * tiles_r, g = q / per_group, r = q - g * per_group;
      const int wide = min(4, run - g * 4), m = r / wide;
      o.tm = m;
      o.tn = run0 + g * 4 + (r - m * wide);
      o.nt = a.hidden / BK;
      return true;
    }
    // dW tiles, then dh tiles, dealt as the schedule says: workgroups < first, then the others
    const Schedule sc = (Schedule)a.schedule;
    const int dw_splits = sc->dw_splits, dh_splits = sc->dh_splits, first = sc->first;
    const int dw_tiles = a.with_dw ? (a.ldg >> 8) * tiles_n : 0, dh_tiles = a.with_dh ? tiles_r * tiles_n : 0;
    const bool front = lin < first;
    const int step = front ? first : G - first;
    const int dw_at = front ? lin : first * sc->dw[0] + lin - first, dw_left = dw_tiles * dw_splits - dw_at;
    const int my_dw = dw_left <= 0 ? 0 : min((dw_left + step - 1) / step, front ? sc->dw[0] : sc->dw[1]);
    if (i < my_dw) {
      o.whole = dw_splits == 1;
      const int q = dw_at + i * step, s = q / dw_tiles, u = q - s * dw_tiles, all = (count + 127) >> 7;
      o.split = s;
      o.tm = u / tiles_n;
      o.tn = u - o.tm * tiles_n;
      o.kt0 = all * s / dw_splits * 2;
      o.nt = all * (s + 1) / dw_splits * 2 - o.kt0;
      return true;
    }
    const int t = i - my_dw, q = (front ? lin : first * sc->dh[0] + lin - first) + t * step;
    if (t >= (front ? sc->dh[0] : sc->dh[1]) || q >= dh_tiles * dh_splits) return false;
    const int s = q / dh_tiles, u = q - s * dh_tiles, all = a.ldg >> 7;
    o.dh = true;
    o.split = s;
    o.tm = u / tiles_n;
    o.tn = u - o.tm * tiles_n;
    o.kt0 = all * s / dh_splits * 2;
    o.nt = all * (s + 1) / dh_splits * 2 - o.kt0;
    return true;
  };
  Item cur;
  if (!item(0, cur)) return;   // workgroup-uniform

  // ---- LDS-DMA: this wave's two 1-KiB pieces of a half-tile.  K-major image [128 rows][128 B]: rows 8 w .. and 64 + 8 w ..;
  // R-major image [64 k][256 B]: k 4 w .. and 32 + 4 w ..; the source chunk carries the swizzle
  const int rk = w * 8 + (lane >> 3), rr = w * 4 + (lane >> 4), cc = lane & 15;
  const uint32_t chunk_k = swz128(rk, lane & 7) * 16, chunk_r = ((((cc >> 1) ^ tr_swz<128>(rr)) << 1) | (cc & 1)) << 4;
  // A: x K-major (ROWS), G R-major (dW), G K-major (dh);  B: W K-major, x R-major, W R-major
  const uint32_t a_off0 = ROWS ? rk * ld_x + chunk_k : rr * ld_g + chunk_r, a_off1 = rk * ld_g + chunk_k;
  const uint32_t b_off0 = ROWS ? rk * ld_w + chunk_k : rr * ld_x + chunk_r, b_off1 = rr * ld_w + chunk_r;
  const uint32_t lds0 = (uint32_t)(uintptr_t)LDS_PTR(smem);
  auto stage_a = [&](const Cursor& c, bool is_dh, int half, int slot_idx) {
    const uint32_t dst = lds0 + slot_idx * HT + w * 1024;
    const uint32_t ld = ROWS ? ld_x : ld_g;
    const bool tr = !ROWS && !is_dh;
    const uint32_t off = ROWS || !is_dh ? a_off0 : a_off1;
    const u32x4_t r = c.rsrc(half ? (tr ? 256 : 128 * ld) : 0);
    dma16(r, off, dst);
    dma16(r, off + (tr ? 32 : 64) * ld, dst + 8192);
  };
  auto stage_b = [&](const Cursor& c, bool is_dh, int half, int slot_idx) {
    const uint32_t dst = lds0 + slot_idx * HT + w * 1024;
    const uint32_t ld = ROWS || is_dh ? ld_w : ld_x;
    const uint32_t off = ROWS || !is_dh ? b_off0 : b_off1;
    const u32x4_t r = c.rsrc(half ? (ROWS ? 128 * ld : 256) : 0);
    dma16(r, off, dst);
    dma16(r, off + (ROWS ? 64 : 32) * ld, dst + 8192);
  };
  // every wave fetches the bias slice and a quarter of the rows' info (waves 4..7 the same quarters): uniform counts
  auto stage_side = [&](int tm_x, int tn_x, int buf) {
    const auto& a = *args();
    const uint32_t dst = lds0 + RING + 8 * SCR + buf * SIDE;
    const int64_t v0 = a.v0 + (int64_t)tn_x * BN;
    dma16(make_rsrc(a.bias ? a.bias + v0 : nullptr, a.bias ? (a.vocab - v0) * 4 : 0), lane * 16, dst);
    if (EPI == V_GRAD) dma16(make_rsrc(a.row_info + tm_x * BM, BM * 16), (w & 3) * 1024 + lane * 16, dst + 1024 + (w & 3) * 1024);
  };
  auto start_of = [&](const Item& o, Cursor& ca, Cursor& cb) {
    const auto& a = *args();
    const int rows_pad = (count + 255) & ~255;
    if (ROWS) {
      ca.set(a.x + (int64_t)o.tm * BM * a.hidden, (int64_t)BM * a.hidden * 2);
      const int64_t v0 = a.v0 + (int64_t)o.tn * BN;
      cb.set(a.w + v0 * a.ldw, ((a.vocab - 1 - v0) * a.ldw + a.hidden) * 2);
    } else if (o.dh) {
      ca.set(a.g + (int64_t)o.tm * BM * a.ldg + (int64_t)o.kt0 * BK, ((int64_t)BM * a.ldg - (int64_t)o.kt0 * BK) * 2);
      const int64_t v0 = a.v0 + (int64_t)o.kt0 * BK;
      cb.set(a.w + v0 * a.ldw + o.tn * BN, ((a.vocab - 1 - v0) * a.ldw + a.hidden - o.tn * BN) * 2);
    } else {
      const int64_t k0 = (int64_t)o.kt0 * BK;
      ca.set(a.g + k0 * a.ldg + (int64_t)o.tm * BM, ((rows_pad - k0) * a.ldg - (int64_t)o.tm * BM) * 2);
      cb.set(a.x + k0 * a.hidden + o.tn * BN, ((rows_pad - k0) * a.hidden - o.tn * BN) * 2);
    }
  };

  // staging cursors: K tile t + 1 (c1) and t + 2 (c2) of the flattened (item, k) stream
  Cursor a1, b1, a2, b2;
  bool v1, v2, d1, d2;
  int s_it = 0, s_left = cur.nt;   // c2's item, and its K tiles from c2 on
  auto advance = [&]() {
    a1 = a2; b1 = b2; v1 = v2; d1 = d2;
    if (!v2) return;
    if (--s_left == 0) {
      Item o;
      v2 = item(++s_it, o);
      if (!v2) return;
      s_left = o.nt;
      d2 = o.dh;
      start_of(o, a2, b2);
    } else {
      // a K tile on: 128 bytes along a K-major row, 64 rows of an R-major operand
      a2.step(ROWS || d2 ? BK * 2 : BK * ld_g);
      b2.step(ROWS ? BK * 2 : BK * (d2 ? ld_w : ld_x));
    }
  };
  f32x4_t acc[2][2][4][2];
  if (cur.nt > 0) {   // (a dW tile without live rows has no K tile; then no item has one)
    start_of(cur, a2, b2);
    v2 = true;
    d2 = cur.dh;
    stage_a(a2, d2, 0, 0);
    stage_b(b2, d2, 0, 1);
    stage_b(b2, d2, 1, 2);
    stage_a(a2, d2, 1, 3);
    if (ROWS) stage_side(cur.tm, cur.tn, 0);
    advance();   // c2 = K tile 1
    advance();   // c1 = K tile 1, c2 = K tile 2 (or the next item's first)
    stage_a(a1, d1, 0, 4);
    stage_b(b1, d1, 0, 5);
    asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    __builtin_amdgcn_s_barrier();
  }

  const int fr = lane & 15, fq = lane >> 4;
  const int lsw = (fr >> 1) & 7, qq = fr >> 2, pp = fr & 3, trg = qq | (fq & 1) << 2;   // trg = tr_swz of k = 8 fq + qq
  const int c0 = (fq ^ lsw) * 16, c1 = ((4 + fq) ^ lsw) * 16;   // K-major: chunk of k-step 0 / 1
  const int tr_row = (fq * 8 + qq) * 256 + pp * 8;
  int a_tr[4], b_tr[4];   // R-major: 16-column block of m / (nh, i)
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    a_tr[m] = tr_row + (((wr * 4 + m) ^ trg) << 5);
    b_tr[m] = (1 + (wc >> 1)) * HT + tr_row + ((((wc & 1) * 4 + m) ^ trg) << 5);
  }
  const int a_rd = (wr * 64 + fr) * 128;                                  // within an A half-tile
  const int b_rd = (1 + (wc >> 1)) * HT + ((wc & 1) * 64 + fr) * 128;     // B half slot + row
  auto tr_frag = [&](const char* p) -> opx8_t {   // k and k + 4 rows of 256 B
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(p));
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(p + 1024));
    const s16x8_t v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return *reinterpret_cast<const opx8_t*>(&v);
  };
  auto a_frag = [&]<bool TR>(const char* half, int m, int ks) -> opx8_t {
    if (TR) return tr_frag(half + a_tr[m] + ks * 8192);
    return *reinterpret_cast<const opx8_t*>(half + a_rd + m * 2048 + (ks ? c1 : c0));
  };
  auto b_frag = [&](const char* buf, int nh, int i, int ks) -> opx8_t {
    if (!ROWS) return tr_frag(buf + b_tr[nh * 2 + i] + ks * 8192);
    return *reinterpret_cast<const opx8_t*>(buf + b_rd + nh * 4096 + i * 2048 + (ks ? c1 : c0));
  };

  int it = 0;
  // acc[mh][nh][m][i]: lane holds n = 4 fq .. +3 of 16-column block (nh, i), row fr of 16-row block (mh, m)
  auto epilogue = [&](int le) {
    const auto& a = *args();
    const int fr = le & 15, fq = le >> 4, tm = cur.tm, tn = cur.tn;
    const int row0 = tm * BM + wr * 64 + fr, col0 = tn * BN + wc * 64 + fq * 4;
    if (ROWS && a.v0 + (int64_t)(tn + 1) * BN > a.vocab) {   // the last tile: nothing past the vocabulary
#pragma unroll
      for (int nh = 0; nh < 2; ++nh)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (a.v0 + col0 + nh * 32 + i * 16 + e >= a.vocab) {
#pragma unroll
              for (int mh = 0; mh < 2; ++mh)
#pragma unroll
                for (int m = 0; m < 4; ++m) acc[mh][nh][m][i][e] = -INFINITY;
            }
    }
    if (EPI == V_STATS) {
#pragma unroll
      for (int mh = 0; mh < 2; ++mh)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          float mx = -INFINITY, t = 0.f;
#pragma unroll
          for (int nh = 0; nh < 2; ++nh)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) mx = fmaxf(mx, acc[mh][nh][m][i][e]);
          mx = xor32_max(xor16_max(mx)) * a.scale2;
          const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
          for (int nh = 0; nh < 2; ++nh)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) t += __builtin_amdgcn_exp2f(fmaf(acc[mh][nh][m][i][e], a.scale2, -ref));
          t = xor32_sum(xor16_sum(t));
          if (fq == 0) a.part[(int64_t)(row0 + mh * 128 + m * 16) * a.n_part + tn * 4 + wc] = make_float2(mx, t);
        }
    } else if (EPI == V_GRAD) {
      float cs[2][2][4];
#pragma unroll
      for (int nh = 0; nh < 2; ++nh)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) cs[nh][i][e] = 0.f;
#pragma unroll
      for (int mh = 0; mh < 2; ++mh)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const float4 ri = *reinterpret_cast<const float4*>(side + (it & 1) * SIDE + 1024 + (mh * 128 + wr * 64 + m * 16 + fr) * 16);
          // image [16 rows][128 B] in this wave's scratch, whole 128-byte row segments out
          float g[2][2][4];
#pragma unroll
          for (int nh = 0; nh < 2; ++nh)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                g[nh][i][e] = __builtin_amdgcn_exp2f(fmaf(acc[mh][nh][m][i][e], a.scale2, -ri.x)) * ri.y;
          // a label among these 64 columns: seldom
          const int at = __float_as_int(ri.z) - (int)a.v0 - tn * BN - wc * 64;
          if (__any((unsigned)at < 64u)) {
#pragma unroll
            for (int nh = 0; nh < 2; ++nh)
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (at == nh * 32 + i * 16 + fq * 4 + e) g[nh][i][e] = ri.w;
          }
#pragma unroll
          for (int nh = 0; nh < 2; ++nh)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
              for (int e = 0; e < 4; ++e) cs[nh][i][e] += g[nh][i][e];
              const int sl = ((nh * 2 + i) * 4 + fq) ^ ((fr & 7) << 1);
              *reinterpret_cast<uint2*>(scr + fr * 128 + sl * 8) =
                  make_uint2(pack_op2(g[nh][i][0], g[nh][i][1]), pack_op2(g[nh][i][2], g[nh][i][3]));
            }
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const int row = p * 8 + (le >> 3), c16 = le & 7;
            const u32x4_t v = *reinterpret_cast<const u32x4_t*>(scr + row * 128 + ((c16 ^ (row & 7)) * 16));
            __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t*>(a.g + (int64_t)(tm * BM + mh * 128 + wr * 64 + m * 16 + row) * a.ldg + tn * BN +
                                                  wc * 64 + c16 * 8));
          }
        }
      if (a.colsum) {
#pragma unroll
        for (int nh = 0; nh < 2; ++nh)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            f32x4_t t;
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = fr_sum(cs[nh][i][e]);
            if (fr == 0)
              *reinterpret_cast<f32x4_t*>(a.colsum + (int64_t)(tm * 2 + wr) * a.ld_colsum + col0 + nh * 32 + i * 16) = t;
          }
      }
    } else if (!cur.whole) {
      // fp32 partials in the accumulators' order (dh_partial_at): every store of a wave is 1 KiB contiguous
      const int panels = cur.dh ? (count + 255) >> 8 : a.ldg >> 8;
      float* out = (cur.dh ? a.out32 : a.dw32) + ((int64_t)(cur.split * panels + tm) * a.tiles_n + tn) * 65536 + w * 8192 + le * 4;
      auto each = [&](auto&& f) {
#pragma unroll
        for (int mh = 0; mh < 2; ++mh)
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int nh = 0; nh < 2; ++nh)
#pragma unroll
              for (int i = 0; i < 2; ++i) f(reinterpret_cast<f32x4_t*>(out + (((mh * 4 + m) * 2 + nh) * 2 + i) * 256), acc[mh][nh][m][i]);
      };
      if (cur.dh && a.accumulate) each([](f32x4_t* o, const f32x4_t& v) { *o += v; });
      else each([](f32x4_t* o, const f32x4_t& v) { *o = v; });
    } else {
      const float s = a.out_scale[0];
#pragma unroll
      for (int mh = 0; mh < 2; ++mh)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
#pragma unroll
          for (int nh = 0; nh < 2; ++nh)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const f32x4_t v = acc[mh][nh][m][i];
              const int sl = ((nh * 2 + i) * 4 + fq) ^ ((fr & 7) << 1);
              *reinterpret_cast<uint2*>(scr + fr * 128 + sl * 8) = make_uint2(pack_op2(v[0] * s, v[1] * s), pack_op2(v[2] * s, v[3] * s));
            }
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const int row = p * 8 + (le >> 3), c16 = le & 7;
            const u32x4_t v = *reinterpret_cast<const u32x4_t*>(scr + row * 128 + ((c16 ^ (row & 7)) * 16));
            const int64_t vocab_row = a.v0 + tm * BM + mh * 128 + wr * 64 + m * 16 + row;
            const int c = tn * BN + wc * 64 + c16 * 8;
            if (vocab_row < a.vocab && c < a.hidden) store_dw(a.out16 + vocab_row * a.ldo + c, v, a.wide);
          }
        }
    }
  };

  while (true) {
#pragma unroll
    for (int nh = 0; nh < 2; ++nh)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x4_t start = {0.f, 0.f, 0.f, 0.f};
        if (ROWS) start = *reinterpret_cast<const f32x4_t*>(side + (it & 1) * SIDE + (wc * 64 + fq * 4 + nh * 32 + i * 16) * 4);
#pragma unroll
        for (int mh = 0; mh < 2; ++mh)
#pragma unroll
          for (int m = 0; m < 4; ++m) acc[mh][nh][m][i] = start;
      }
    if (wr == 1) __builtin_amdgcn_s_barrier();   // waves 4..7 run one barrier behind

    opx8_t af[4][2], bf0[2][2], bf1[2][2];
    auto ktile = [&]<bool A_TR, int B>(int kk) {
        const char* buf = smem + B * 4 * HT;
        // ---------------- phase A: A0, both B halves -> acc[0][*]; stage (t+1).B1, (t+1).A1
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          bf0[i][0] = b_frag(buf, 0, i, 0);
          bf0[i][1] = b_frag(buf, 0, i, 1);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          af[m][0] = a_frag.template operator()<A_TR>(buf, m, 0);
          af[m][1] = a_frag.template operator()<A_TR>(buf, m, 1);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          bf1[i][0] = b_frag(buf, 1, i, 0);
          bf1[i][1] = b_frag(buf, 1, i, 1);
        }
        if (v1) {
          stage_b(b1, d1, 1, (B ^ 1) * 4 + 2);
          stage_a(a1, d1, 1, (B ^ 1) * 4 + 3);
          // in flight behind this wait: (t+1).A0/B0 from the previous phase and the four just issued
          asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        } else {
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        if (ROWS && B == 1 && kk == 0) {
          Item o;
          if (item(it + 1, o)) stage_side(o.tm, o.tn, (it + 1) & 1);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              acc[0][0][m][i] = MFMA_16x16x32(bf0[i][ks], af[m][ks], acc[0][0][m][i]);
              acc[0][1][m][i] = MFMA_16x16x32(bf1[i][ks], af[m][ks], acc[0][1][m][i]);
            }
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        // ---------------- phase B: A1 -> acc[1][*]; stage (t+2).A0, (t+2).B0; K tile t+1 retired
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          af[m][0] = a_frag.template operator()<A_TR>(buf + 3 * HT, m, 0);
          af[m][1] = a_frag.template operator()<A_TR>(buf + 3 * HT, m, 1);
        }
        const bool staged2 = v2;
        if (v2) {
          stage_a(a2, d2, 0, B * 4 + 0);
          stage_b(b2, d2, 0, B * 4 + 1);
        }
        advance();
        if (staged2) {
          asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        } else {
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              acc[1][1][m][i] = MFMA_16x16x32(bf1[i][ks], af[m][ks], acc[1][1][m][i]);
              acc[1][0][m][i] = MFMA_16x16x32(bf0[i][ks], af[m][ks], acc[1][0][m][i]);
            }
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
    };
    const int nt = cur.nt;
    if (ROWS || cur.dh) {
      for (int kk = 0; kk < nt; kk += 2) {
        ktile.template operator()<false, 0>(kk);
        ktile.template operator()<false, 1>(kk);
      }
    } else {
      for (int kk = 0; kk < nt; kk += 2) {
        ktile.template operator()<true, 0>(kk);
        ktile.template operator()<true, 1>(kk);
      }
    }
    if (wr == 0) __builtin_amdgcn_s_barrier();   // balances the extra barrier of waves 4..7

    // ---- epilogue.  Lane's rows: mh * 128 + wr * 64 + m * 16 + fr; its columns: wc * 64 + nh * 32 + i * 16 + 4 fq + e.
    // (lane id formed anew, too: see args())
    int le;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(le));
    epilogue(le);
    ++it;
    if (!item(it, cur)) break;
  }
}

template <int EPI>
hipError_t launch_8(const VocabGemm& g, hipStream_t st) {
  auto kfn = vocab8_kernel<EPI>;
  static DeviceOnce once;
  int n_cu = 0;
  hipError_t e0 = once.get([&](int dev, int* val) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kfn), hipFuncAttributeMaxDynamicSharedMemorySize, LDS8);
    if (e != hipSuccess) return e;
    int cus = 0;
    if ((e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev)) != hipSuccess) return e;
    *val = cus & ~7;
    return *val < 8 ? hipErrorInvalidValue : hipSuccess;
  }, &n_cu);
  if (e0 != hipSuccess) return e0;
  hipLaunchKernelGGL(kfn, dim3(n_cu), dim3(512), LDS8, st, g);
  return hipGetLastError();
}

}  // namespace

hipError_t KSET::launch_vocab8(int what, const VocabGemm& g, hipStream_t st) {
  if (g.hidden % 128 || g.ldg % 256) return hipErrorInvalidValue;
  switch (what) {
    case V_STATS: return launch_8<V_STATS>(g, st);
    case V_GRAD: return launch_8<V_GRAD>(g, st);
    case V_PROD: return launch_8<V_PROD>(g, st);
    default: return hipErrorInvalidValue;
  }
}
