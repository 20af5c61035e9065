// A row's k largest scores with their ids, ties to the lowest id: what a teacher hands to the distillation loss
// (clip_linear_distill).  Scores are ordered as torch orders them: NaN above everything, -0 equal to +0.
// One workgroup per row; a chunk of 64 KB (16 384 fp32 scores or 32 768 of 16 bits) is read at once into registers, 64 per
// thread.  A threshold that the k largest all reach and few others do is found to 16 bits by bisection on ballots:
// for k <= 128 the k-th largest of the 256 threads' maxima (177 random scores reach it at k = 128, 74 at k = 64), beyond that
// the k-th largest of the maxima of 16 bytes, and the k-th largest score itself where a row has not twice k of these.  Each wave notes what reaches it,
// one comparison per 16 bytes read, in its own part of LDS as 64-bit keys (order-preserving bits of the score above the inverted id: all keys differ, a larger key comes first), and
// the few keys noted are sorted by counting, for each, how many are larger.  Where too many reach the threshold (equal
// scores) the chunk is gone through again, a list being cut back to its k largest whenever it is full.
// Bound: reading the scores; 8192 x 30 522 with k 64: fp32 178 - 202 us (5.0 - 5.6 TB/s), bf16 114 - 138 us (3.6 - 4.4), fp16 107 -
// 119 us (4.2 - 4.7); five rows 8.4 - 10.4 us; k 300 on 4096 rows: fp32 360 us, bf16 290 - 300 us, fp16 242 us (the search's 16
// barriers, then every noted key against every other; 540 and 940 us, fp32 and bf16, with every score searched).
#include "common.h"
#include "kernels.h"

namespace {

typedef unsigned long long u64;

__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;   // any NaN
  if ((u << 1) == 0) return 0x80000000u;                     // -0 as +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_score(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);   // 0xffffffff: a NaN
}

// (maximum: NaN if either is)
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

struct F32 {
  static constexpr int VEC = 4;
  typedef float elem;
  static __device__ __forceinline__ float top(const uint4& v) {
    return max_nan(max_nan(get(v, 0), get(v, 1)), max_nan(get(v, 2), get(v, 3)));
  }
  static __device__ __forceinline__ float get(const uint4& v, int i) { return __uint_as_float(reinterpret_cast<const uint32_t*>(&v)[i]); }
  static __device__ __forceinline__ float one(const elem* p) { return *p; }
  static constexpr uint32_t one_inf_bits = 0;
};
struct Bf16 {
  static constexpr int VEC = 8;
  typedef uint16_t elem;
  static __device__ __forceinline__ float top(const uint4& v) {
    float m = max_nan(get(v, 0), get(v, 1));
#pragma unroll
    for (int i = 2; i < 8; i += 2) m = max_nan(max_nan(m, get(v, i)), get(v, i + 1));
    return m;
  }
  static __device__ __forceinline__ float bits(uint32_t h) { return __uint_as_float(h << 16); }
  static __device__ __forceinline__ float get(const uint4& v, int i) {
    const uint32_t d = reinterpret_cast<const uint32_t*>(&v)[i >> 1];
    return i & 1 ? __uint_as_float(d & 0xffff0000u) : __uint_as_float(d << 16);
  }
  static __device__ __forceinline__ float one(const elem* p) { return bits(*p); }
  static constexpr uint32_t one_inf_bits = 0xff80;
};
struct F16 {
  static constexpr int VEC = 8;
  typedef uint16_t elem;
  static __device__ __forceinline__ float top(const uint4& v) {
    typedef __attribute__((ext_vector_type(2))) _Float16 h2;
    h2 h[4];
    __builtin_memcpy(h, &v, 16);
    const h2 m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(h[0], h[1]), __builtin_elementwise_maximum(h[2], h[3]));
    return max_nan((float)m[0], (float)m[1]);
  }
  static __device__ __forceinline__ float half_bits(uint16_t h) { _Float16 f; __builtin_memcpy(&f, &h, 2); return (float)f; }
  static __device__ __forceinline__ float get(const uint4& v, int i) {
    const uint32_t d = reinterpret_cast<const uint32_t*>(&v)[i >> 1];
    return half_bits((uint16_t)(i & 1 ? d >> 16 : d));
  }
  static __device__ __forceinline__ float one(const elem* p) { return half_bits(*p); }
  static constexpr uint32_t one_inf_bits = 0xfc00;
};

constexpr int NT = 256;   // threads
// 16-byte loads per thread and chunk.  8192 rows of 30 522, k 64, in us (fp32 / bf16 / fp16): 8: 234 / 137 / 118, 12: 229 / 162 /
// 136, 16: 200 / 138 / 119, 24: 282 / 175 / 158, 32 (a whole fp32 row): 295.  16 leave room for four workgroups per CU: their
// loads and their searches overlap
constexpr int NV = 16;
constexpr uint32_t KEY_LOWEST = 0x007fffffu;   // order_key(-inf)

// KMAX: the largest k; MAXIMA: the threshold from the threads' maxima (k <= 128), else from all scores; WCAP: keys a wave may note
template <class T, int KMAX, bool MAXIMA, int WCAP>
__global__ __launch_bounds__(NT) void topk_rows_kernel(const typename T::elem* __restrict__ logits, int64_t ld, int vocab, int k,
                                                       typename T::elem* __restrict__ values, int64_t* __restrict__ index) {
  constexpr int CAP = KMAX + 4 * WCAP;           // cand[0 .. KMAX): kept so far; then the waves' notes
  __shared__ u64 cand[CAP];
  __shared__ uint32_t max_s[MAXIMA ? NT : 1];
  __shared__ uint32_t threshold_s;
  __shared__ int wave_s[2][4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const typename T::elem* row = logits + (int64_t)blockIdx.x * ld;

  int have = 0, turn = 0;            // uniform: keys kept
  u64 kth = 0;                       // uniform: a smaller key is not among the k largest
  float kth_f = -INFINITY;           // its score; !(x < kth_f) is the cheap test (NaN passes)
  auto key64 = [](float x, int id) { return ((u64)order_key(x) << 32) | (uint32_t)~id; };
  auto score_of = [](uint32_t key) { return key <= KEY_LOWEST ? -INFINITY : key_score(key); };

  // the k largest of the kept keys and n[w] notes of each wave, sorted, become the kept ones
  auto cut = [&](const int (&n)[4]) {
    constexpr int MINE = (CAP + NT - 1) / NT;
    const int total = have + n[0] + n[1] + n[2] + n[3];
    u64 mine[MINE];
    int rank[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      int at = tid + i * NT;
      if (at >= have) {
        at -= have;
        int seg = 0;
#pragma unroll
        for (int q = 0; q < 3; ++q)
          if (seg == q && at >= n[q]) { at -= n[q]; seg = q + 1; }
        at += KMAX + seg * WCAP;
      }
      mine[i] = tid + i * NT < total ? cand[at] : 0;
      rank[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < MINE; ++i)
      if (i * NT + w * 64 < total) {   // (wave-uniform)
        for (int j = 0; j < have; ++j) rank[i] += cand[j] > mine[i];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          for (int j = 0; j < n[q]; ++j) rank[i] += cand[KMAX + q * WCAP + j] > mine[i];
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MINE; ++i)
      if (tid + i * NT < total && rank[i] < k) cand[rank[i]] = mine[i];
    have = min(total, k);
    __syncthreads();
    if (have == k) {
      kth = cand[k - 1];
      kth_f = score_of((uint32_t)(kth >> 32));
    }
  };
  // where this thread's key goes if `p`; false = no room (the list, taken as one behind the kept keys, is full)
  int noted = 0;
  auto reserve = [&](bool p, int& at) -> bool {
    const unsigned long long m = __ballot(p);
    turn ^= 1;
    if (lane == 0) wave_s[turn][w] = __popcll(m);
    __syncthreads();
    const int t0 = wave_s[turn][0], t1 = wave_s[turn][1], t2 = wave_s[turn][2], t3 = wave_s[turn][3];
    at = KMAX + noted + __popcll(m & ((1ull << lane) - 1)) + (w > 0 ? t0 : 0) + (w > 1 ? t1 : 0) + (w > 2 ? t2 : 0);
    const int sum = t0 + t1 + t2 + t3;
    if (noted + sum > 4 * WCAP) return false;
    noted += sum;
    return true;
  };
  // the list as one segment: split over the waves' parts for cut()
  auto cut_list = [&]() {
    __syncthreads();
    int n[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) n[q] = min(max(noted - q * WCAP, 0), WCAP);
    cut(n);
    noted = 0;
  };

  // the largest threshold, to 16 bits, that k scores reach; count(reaches) = how many of this wave's do
  auto search = [&](auto&& count) -> uint32_t {
    uint32_t t = 0;
    for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1) {
      const float f = score_of(t | bit);
      const int n = (t | bit) <= 0xff800000u ? count([&](float x) { return !(x < f); }) : count([](float x) { return x != x; });
      turn ^= 1;
      if (lane == 0) wave_s[turn][w] = n;
      __syncthreads();
      if (wave_s[turn][0] + wave_s[turn][1] + wave_s[turn][2] + wave_s[turn][3] >= k) t |= bit;
    }
    return t;
  };

  // ---- the scores before the first and after the last whole 16 bytes are kept to begin with (at most 14)
  const int head = min((int)(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(typename T::elem)), vocab);
  const int body = (vocab - head) / T::VEC;   // whole vectors
  {
    const int rest = vocab - head - body * T::VEC;
    const int id = tid < head ? tid : head + body * T::VEC + (tid - head);
    if (tid < head + rest) cand[tid] = key64(T::one(row + id), id);
    have = head + rest;
  }
  const uint4* vec = reinterpret_cast<const uint4*>(row + head);
  for (int c0 = 0; c0 < body; c0 += NV * NT) {
    uint4 v[NV];
    const uint32_t neg = sizeof(typename T::elem) == 4 ? 0xff800000u : (T::one_inf_bits * 0x10001u);   // -inf
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = vec[min(c0 + i * NT + tid, body - 1)];   // (no branches: all loads in flight)
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (c0 + (i + 1) * NT > body && c0 + i * NT + tid >= body) v[i] = make_uint4(neg, neg, neg, neg);
    if (kth == 0) {   // no threshold yet
      uint32_t t = 0;
      const int left = min(body - c0, NV * NT);
      if (MAXIMA && left >= min(NT, 2 * k)) {
        float mx = T::top(v[0]);
#pragma unroll
        for (int i = 1; i < NV; ++i) mx = max_nan(mx, T::top(v[i]));
        max_s[tid] = order_key(mx);
        __syncthreads();
        if (w == 0) {
          uint32_t m[NT / 64];
#pragma unroll
          for (int i = 0; i < NT / 64; ++i) m[i] = max_s[i * 64 + lane];
          for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < NT / 64; ++i) n += __popcll(__ballot(m[i] >= (t | bit)));
            if (n >= k) t |= bit;
          }
          if (lane == 0) threshold_s = t;
        }
        __syncthreads();
        t = threshold_s;
      } else if (!MAXIMA && left >= 2 * k) {
        float mx[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) mx[i] = T::top(v[i]);
        t = search([&](auto&& reaches) {
          int n = 0;
#pragma unroll
          for (int i = 0; i < NV; ++i) n += __popcll(__ballot(reaches(mx[i])));
          return n;
        });
      } else {
        constexpr int FEW = MAXIMA ? 1 : 2 * KMAX / NT;   // 16-byte pieces per thread
        t = search([&](auto&& reaches) {
          int n = 0;
#pragma unroll
          for (int i = 0; i < FEW; ++i)
            if (i * NT < left)
#pragma unroll
              for (int e = 0; e < T::VEC; ++e) n += __popcll(__ballot(reaches(T::get(v[i], e))));
          return n;
        });
      }
      kth = (u64)t << 32;
      kth_f = score_of(t);
    }
    // every wave notes what reaches the threshold
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      // (what the threshold's pass formed of v is formed again: kept, it would take the registers of another workgroup)
      asm volatile("" : "+v"(v[i].x), "+v"(v[i].y), "+v"(v[i].z), "+v"(v[i].w));
      if (__any(!(T::top(v[i]) < kth_f)) && cnt <= WCAP) {
        const int at = c0 + i * NT + tid;
#pragma unroll
        for (int e = 0; e < T::VEC; ++e) {
          const float x = T::get(v[i], e);
          if (__any(!(x < kth_f))) {
            const int id = head + at * T::VEC + e;
            const u64 key = key64(x, id);
            const bool p = at < body && key >= kth;
            const unsigned long long m = __ballot(p);
            const int to = cnt + __popcll(m & ((1ull << lane) - 1));
            if (p && to < WCAP) cand[KMAX + w * WCAP + to] = key;
            cnt += __popcll(m);
          }
        }
      }
    }
    turn ^= 1;
    if (lane == 0) wave_s[turn][w] = cnt;
    __syncthreads();
    int n[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) n[q] = __builtin_amdgcn_readfirstlane(wave_s[turn][q]);
    if (n[0] <= WCAP && n[1] <= WCAP && n[2] <= WCAP && n[3] <= WCAP) {
      cut(n);
    } else {
      // crowded: read again, one score per thread at a time
      noted = 0;
#pragma unroll 1
      for (int q = 0; q < NV * T::VEC && c0 + q / T::VEC * NT < body; ++q) {
        const int at = c0 + q / T::VEC * NT + tid, id = head + at * T::VEC + q % T::VEC;
        const u64 key = at < body ? key64(T::one(row + id), id) : 0;
        bool p = at < body && key >= kth;
        int to;
        if (!reserve(p, to)) {
          cut_list();
          p = p && key >= kth;
          reserve(p, to);        // 256 always fit an empty list
        }
        if (p) cand[to] = key;
      }
      cut_list();
    }
  }
  if (body == 0) {
    __syncthreads();
    const int none[4] = {0, 0, 0, 0};
    cut(none);
  }
  for (int j = tid; j < k; j += NT) {
    const int id = (int)~(uint32_t)cand[j];
    values[(int64_t)blockIdx.x * k + j] = row[id];
    index[(int64_t)blockIdx.x * k + j] = id;
  }
}

template <class T>
hipError_t launch_t(const void* logits, int64_t ld, int n, int vocab, int k, void* values, int64_t* index, hipStream_t st) {
  const auto* in = static_cast<const typename T::elem*>(logits);
  auto* out = static_cast<typename T::elem*>(values);
  constexpr int MOST = 1 << 22;   // (a grid may have 2^32 threads)
  for (int r0 = 0; r0 < n; r0 += n - r0 < MOST ? n - r0 : MOST) {
    const dim3 rows(n - r0 < MOST ? n - r0 : MOST);
    const auto* from = in + r0 * ld;
    auto* to = out + (int64_t)r0 * k;
    if (k <= 128) hipLaunchKernelGGL((topk_rows_kernel<T, 128, true, 256>), rows, dim3(NT), 0, st, from, ld, vocab, k, to, index + (int64_t)r0 * k);
    else hipLaunchKernelGGL((topk_rows_kernel<T, 1024, false, 512>), rows, dim3(NT), 0, st, from, ld, vocab, k, to, index + (int64_t)r0 * k);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_topk_rows(const void* logits, int type, int64_t ld, int n, int vocab, int k, void* values, int64_t* index,
                            hipStream_t st) {
  if (n <= 0) return hipSuccess;
  switch (type) {
    case 0: return launch_t<Bf16>(logits, ld, n, vocab, k, values, index, st);
    case 1: return launch_t<F32>(logits, ld, n, vocab, k, values, index, st);
    case 2: return launch_t<F16>(logits, ld, n, vocab, k, values, index, st);
    default: return hipErrorInvalidValue;
  }
}
