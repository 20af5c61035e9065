// A row's k largest scores with their ids, ties to the lowest id: what a teacher hands to the distillation loss
// (clip_linear_distill).  Scores are ordered as torch orders them: NaN above everything, -0 equal to +0.
// One workgroup streams a row once.  What reaches the running threshold goes, as a 64-bit key (order-preserving bits of
// the score above the inverted id: all keys differ, a larger key comes first), to a candidate list in LDS; the list is cut
// back to its k largest by counting, for every candidate, how many are larger.  The first threshold is the k-th largest of
// the 256 threads' maxima over the first chunk, at most the true one, so that few candidates are ever written.
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

struct F32 {
  static constexpr int VEC = 4;
  typedef float elem;
  static __device__ __forceinline__ float get(const uint4& v, int i) { return __uint_as_float(reinterpret_cast<const uint32_t*>(&v)[i]); }
  static __device__ __forceinline__ float one(const elem* p) { return *p; }
};
struct Bf16 {
  static constexpr int VEC = 8;
  typedef uint16_t elem;
  static __device__ __forceinline__ float bits(uint32_t h) { return __uint_as_float(h << 16); }
  static __device__ __forceinline__ float get(const uint4& v, int i) {
    const uint32_t d = reinterpret_cast<const uint32_t*>(&v)[i >> 1];
    return i & 1 ? __uint_as_float(d & 0xffff0000u) : __uint_as_float(d << 16);
  }
  static __device__ __forceinline__ float one(const elem* p) { return bits(*p); }
};
struct F16 {
  static constexpr int VEC = 8;
  typedef uint16_t elem;
  static __device__ __forceinline__ float half_bits(uint16_t h) { _Float16 f; __builtin_memcpy(&f, &h, 2); return (float)f; }
  static __device__ __forceinline__ float get(const uint4& v, int i) {
    const uint32_t d = reinterpret_cast<const uint32_t*>(&v)[i >> 1];
    return half_bits((uint16_t)(i & 1 ? d >> 16 : d));
  }
  static __device__ __forceinline__ float one(const elem* p) { return half_bits(*p); }
};

constexpr int NT = 256, PER = 16;   // threads; scores per thread and chunk

// CAP: room for candidates, at least k + 256
template <class T, int CAP>
__global__ __launch_bounds__(NT) void topk_rows_kernel(const typename T::elem* __restrict__ logits, int64_t ld, int vocab, int k,
                                                       typename T::elem* __restrict__ values, int64_t* __restrict__ index) {
  constexpr int NV = PER / T::VEC;   // 16-byte loads per thread and chunk
  __shared__ u64 cand[CAP];
  __shared__ u64 kth_s;
  __shared__ float max_s[NT];
  __shared__ int wave_s[2][4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const typename T::elem* row = logits + (int64_t)blockIdx.x * ld;

  int have = 0, turn = 0;            // uniform: candidates in the list
  u64 kth = 0;                       // uniform: a key below the threshold does not count
  float kth_f = -INFINITY;           // its score; !(x < kth_f) is the cheap test (NaN passes)
  auto key64 = [](float x, int id) { return ((u64)order_key(x) << 32) | (uint32_t)~id; };

  // the list's k largest, sorted, to its front
  auto cut = [&]() {
    __syncthreads();
    // (the list is rarely longer than one or two scores per thread: those keep their scores in registers)
    u64 mine[CAP / NT];
    int rank[CAP / NT];
#pragma unroll
    for (int i = 0; i < CAP / NT; ++i) {
      mine[i] = tid + i * NT < have ? cand[tid + i * NT] : 0;
      rank[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < CAP / NT; ++i)
      if (i * NT < have)
        for (int j = 0; j < have; ++j) rank[i] += cand[j] > mine[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CAP / NT; ++i)
      if (tid + i * NT < have && rank[i] < k) cand[rank[i]] = mine[i];
    if (have > k) have = k;
    __syncthreads();
    if (have == k) {
      kth = cand[k - 1];
      kth_f = key_score((uint32_t)(kth >> 32));
    }
  };
  // `n` of this thread's scores pass: where its first one goes; false = no room, nothing reserved
  auto reserve = [&](int n, int& at) -> bool {
    int before = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(before, o, 64);
      if (lane >= o) before += up;
    }
    turn ^= 1;
    if (lane == 63) wave_s[turn][w] = before;
    __syncthreads();
    const int t0 = wave_s[turn][0], t1 = wave_s[turn][1], t2 = wave_s[turn][2], t3 = wave_s[turn][3];
    at = have + before - n + (w > 0 ? t0 : 0) + (w > 1 ? t1 : 0) + (w > 2 ? t2 : 0);
    const int sum = t0 + t1 + t2 + t3;
    if (have + sum > CAP) return false;
    have += sum;
    return true;
  };
  auto passes = [&](float x, int id) { return !(x < kth_f) && key64(x, id) >= kth; };

  // ---- the scores before the first and after the last whole 16 bytes
  const int head = min((int)(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(typename T::elem)), vocab);
  const int body = (vocab - head) / T::VEC;   // whole vectors
  {
    const int rest = vocab - head - body * T::VEC;
    const int id = tid < head ? tid : head + body * T::VEC + (tid - head);
    const bool in = tid < head + rest;
    int at;
    reserve(in ? 1 : 0, at);
    if (in) cand[at] = key64(T::one(row + id), id);
  }
  const uint4* vec = reinterpret_cast<const uint4*>(row + head);
  uint4 cur[NV], nxt[NV];
  auto fetch = [&](int c, uint4 (&to)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (c * NV + i) * NT + tid;
      if (at < body) to[i] = vec[at];
    }
  };
  const int chunks = (body + NV * NT - 1) / (NV * NT);
  fetch(0, cur);
  for (int c = 0; c < chunks; ++c) {
    if (c + 1 < chunks) fetch(c + 1, nxt);
    if (c == 0 && k <= NT) {
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i * NT + tid < body)
#pragma unroll
          for (int e = 0; e < T::VEC; ++e) mx = fmaxf(mx, T::get(cur[i], e));
      max_s[tid] = mx;
      __syncthreads();
      int rank = 0;   // ties by thread: ranks are 0 .. 255
      for (int j = 0; j < NT; ++j) rank += max_s[j] > mx || (max_s[j] == mx && j < tid);
      if (rank == k - 1) kth_s = (u64)order_key(mx) << 32;
      __syncthreads();
      kth = kth_s;
      kth_f = key_score((uint32_t)(kth >> 32));
    }
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (c * NV + i) * NT + tid;
      if (at < body)
#pragma unroll
        for (int e = 0; e < T::VEC; ++e) {
          const float x = T::get(cur[i], e);
          if (passes(x, head + at * T::VEC + e)) mask |= 1u << (i * T::VEC + e);
        }
    }
    int at;
    if (reserve(__popc(mask), at)) {
#pragma unroll
      for (int s = 0; s < PER; ++s)
        if (mask & (1u << s))
          cand[at++] = key64(T::get(cur[s / T::VEC], s % T::VEC), head + ((c * NV + s / T::VEC) * NT + tid) * T::VEC + s % T::VEC);
      if (have > CAP / 2) cut();
    } else {
      // a crowded chunk: one score per thread at a time, the list cut back whenever it is full
#pragma unroll 1
      for (int s = 0; s < PER; ++s) {
        float x = 0.f;
#pragma unroll
        for (int q = 0; q < PER; ++q)
          if (q == s) x = T::get(cur[q / T::VEC], q % T::VEC);
        const int id = head + ((c * NV + s / T::VEC) * NT + tid) * T::VEC + s % T::VEC;
        bool p = (mask >> s & 1) && passes(x, id);
        if (!reserve(p, at)) {
          cut();
          p = p && passes(x, id);
          reserve(p, at);        // k + 256 fit
        }
        if (p) cand[at] = key64(x, id);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) cur[i] = nxt[i];
  }
  cut();
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
  if (k <= 256)
    hipLaunchKernelGGL((topk_rows_kernel<T, 1024>), dim3(n), dim3(NT), 0, st, in, ld, vocab, k, out, index);
  else
    hipLaunchKernelGGL((topk_rows_kernel<T, 4096>), dim3(n), dim3(NT), 0, st, in, ld, vocab, k, out, index);
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
