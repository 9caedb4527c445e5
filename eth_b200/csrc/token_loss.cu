// Per-token kernels over the vocabulary: log-probabilities of given tokens with entropy and top
// alternatives, and the loss against a teacher's top logits, forward and backward.
//
// All of them are bound by reading the logits [rows, vocab] (and writing their gradient). One CTA
// owns one row; several CTAs per SM keep enough 16-byte loads in flight while others reduce.
//
//   x = z / T,  m = max z,  e_j = 2^((z_j - m) log2(e) / T),  L = sum e,  A = sum e_j log2 e_j
//   log p_j = (z_j - m) / T - ln L,        entropy = ln L - ln2 * A / L
//
// The difference z - m is formed before it is scaled: a fused multiply-add of z * s - m * s would
// overflow on masks of a type's lowest value and carry the rounding of m * s into every term.
// All sums and statistics are fp32; 16-bit types are widened on load, a gradient is rounded once.
#include "token_loss.cuh"

#include "gemm_sm100.cuh"
#include "sm100_common.cuh"

#include <math_constants.h>
#include <type_traits>

namespace ethb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

#define ETHB_DISPATCH_T(dtype, T, ...)                              \
  do {                                                              \
    if ((dtype) == kBF16) { using T = __nv_bfloat16; __VA_ARGS__; } \
    else if ((dtype) == kF16) { using T = __half; __VA_ARGS__; }    \
    else { using T = float; __VA_ARGS__; }                          \
  } while (0)

template <typename T> constexpr int kVec = 16 / static_cast<int>(sizeof(T));

template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[kVec<T>]) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    constexpr int dt = std::is_same<T, __nv_bfloat16>::value ? kBF16 : kF16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = unpack2(w[i], dt);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  } else {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
}
template <typename T>
__device__ __forceinline__ uint4 repack(const float (&f)[kVec<T>]) {
  if constexpr (sizeof(T) == 2) {
    constexpr int dt = std::is_same<T, __nv_bfloat16>::value ? kBF16 : kF16;
    return make_uint4(pack2(f[0], f[1], dt), pack2(f[2], f[3], dt), pack2(f[4], f[5], dt), pack2(f[6], f[7], dt));
  } else {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
}

// A row as `head` single elements up to a 16-byte boundary, `nvec` 16-byte vectors, and a tail. Any
// pitch and offset is taken; only the first and last few elements of a row go one by one.
template <typename T> struct Row {
  const T* p;
  int head, nvec, n;
  __device__ __forceinline__ Row(const T* row, int vocab) : p(row), n(vocab) {
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    head = min(off == 0 ? 0 : kVec<T> - off, vocab);
    nvec = (vocab - head) / kVec<T>;
  }
  __device__ __forceinline__ int tail() const { return head + nvec * kVec<T>; }
  __device__ __forceinline__ const uint4* vec() const { return reinterpret_cast<const uint4*>(p + head); }
};

// Order-preserving unsigned image of a value: larger value <=> larger key, NaN above everything,
// -0 and +0 alike (they are ties, which go to the lower token id).
// Integer steps only: float arithmetic here would flush subnormal logits.
__device__ __forceinline__ uint32_t order_key(float v) {
  uint32_t b = __float_as_uint(v);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (b == 0x80000000u) b = 0;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The kernels below issue four to five instructions per logit; the Pair arithmetic (two fp32 lanes per
// instruction) is what keeps that below the time DRAM needs.
__device__ __forceinline__ Pair exp2_pair(Pair t) {
  float x, y;
  split(t, x, y);
  return pair(exp2f(x), exp2f(y));
}

// A masked (-inf) logit has 2^t = 0 and t = -inf, whose product would be NaN. Where a sum or gradient
// needs 2^t * t, logits below kFloor are raised to it, which leaves 2^t at 0 (it is 0 in fp32 below
// t = -150) and t finite. Rows that lie so low themselves, or a temperature so high, that this does
// not hold take a clamp per element instead; so do rows so high (a token forced by the type's highest
// value), or a temperature so low, that t or its product with a gradient's factor would pass fp32's range.
constexpr float kFloor = -57344.f;   // -7 * 2^13: exact in every type
__device__ __forceinline__ bool has_floor(float mu, float s2) {
  const float depth = (mu - kFloor) * s2;   // -t of a raised logit: above 200 and finite, in one comparison
  constexpr uint32_t kLow = 0x43480000u, kInf = 0x7f800000u;   // 200, infinity
  return __float_as_uint(depth) - kLow < kInf - kLow;
}
__device__ __forceinline__ uint32_t max_nan(uint32_t x, float low) {
  uint32_t r;
  asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(__float_as_uint(low)));
  return r;
}
template <typename T>   // NaN stays
__device__ __forceinline__ uint4 at_least(uint4 u, float low) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
    const __nv_bfloat162 f = __float2bfloat162_rn(low);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], f);
  } else if constexpr (std::is_same<T, __half>::value) {
    __half2* h = reinterpret_cast<__half2*>(&u);
    const __half2 f = __float2half2_rn(low);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], f);
  } else {
    u.x = max_nan(u.x, low);
    u.y = max_nan(u.y, low);
    u.z = max_nan(u.z, low);
    u.w = max_nan(u.w, low);
  }
  return u;
}

// Running (maximum, sum of exponentials, sum of exponential * exponent). `mu` is what is subtracted:
// the maximum, or 0 while only -inf has been seen (so that -inf - mu stays -inf and not NaN).
template <bool kEntropy> struct Running {
  float mx = -INFINITY, l = 0.f, a = 0.f;
  __device__ __forceinline__ float mu() const { return mx == -INFINITY ? 0.f : mx; }
  __device__ __forceinline__ void raise(float to, float s2) {   // to > mx
    if (mx != -INFINITY) {
      const float d = (mx - to) * s2, c = exp2f(d);
      if (kEntropy) a = c == 0.f ? 0.f : c * (a + d * l);
      l *= c;
    }
    mx = to;
  }
  // the scale that brings this sum to the maximum `to`; 0 for an empty one
  __device__ __forceinline__ void rebase(float to, float s2) {
    if (l == 0.f || to == mx) return;
    const float d = (mu() - (to == -INFINITY ? 0.f : to)) * s2, c = exp2f(d);
    if (kEntropy) a = c == 0.f ? 0.f : c * (a + d * l);
    l *= c;
  }
  __device__ __forceinline__ void add(float z, float m, float s2) {
    const float t = (z - m) * s2;
    const float e = exp2f(t);
    l += e;
    if (kEntropy) a = fmaf(e, fmaxf(t, -1000.f), a);   // e is 0 far above -1000; -inf * 0 must not appear
  }
  // N vectors of one thread at once; returns their maximum.
  template <typename T, int N>
  __device__ __forceinline__ float add_group(const uint4 (&u)[N], float s2);
};

template <typename T>
__device__ __forceinline__ float max_of(const uint4& u) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return __bfloat162float(__hmax(__low2bfloat16(m), __high2bfloat16(m)));
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return __half2float(__hmax(__low2half(m), __high2half(m)));
  } else {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)),
                 fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
}

// A vector as pairs of fp32.
template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& u, Pair (&p)[kVec<T> / 2]) {
  float f[kVec<T>];
  unpack<T>(u, f);
#pragma unroll
  for (int i = 0; i < kVec<T> / 2; ++i) p[i] = pair(f[2 * i], f[2 * i + 1]);
}

template <typename T>
__device__ __noinline__ Running<true> add_clamped(Running<true> run, uint4 u, float s2) {
  float f[kVec<T>];
  unpack<T>(u, f);
  const float mu = run.mu();
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) run.add(f[j], mu, s2);
  return run;
}

template <bool kEntropy>
template <typename T, int N>
__device__ __forceinline__ float Running<kEntropy>::add_group(const uint4 (&u)[N], float s2) {
  float m = max_of<T>(u[0]);
#pragma unroll
  for (int k = 1; k < N; ++k) m = fmaxf(m, max_of<T>(u[k]));
  if (m > mx) raise(m, s2);
  const float base = mu();
  if constexpr (kEntropy) {
    if (!has_floor(base, s2)) {
#pragma unroll
      for (int k = 0; k < N; ++k) *this = add_clamped<T>(*this, u[k], s2);
      return m;
    }
  }
  const Pair neg = pair(-base, -base), scale = pair(s2, s2);
  Pair lsum = pair(0.f, 0.f), asum = lsum;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    Pair z[kVec<T> / 2];
    unpack_pairs<T>(kEntropy ? at_least<T>(u[k], kFloor) : u[k], z);
#pragma unroll
    for (int j = 0; j < kVec<T> / 2; ++j) {
      const Pair t = (z[j] + neg) * scale, e = exp2_pair(t);
      lsum = lsum + e;
      if (kEntropy) asum = fma2(e, t, asum);
    }
  }
  float x, y;
  split(lsum, x, y);
  l += x + y;
  if (kEntropy) {
    split(asum, x, y);
    a += x + y;
  }
  return m;
}

// The maxima of a thread's segments (runs of `length` groups of kGroup vectors), for select_top: at most
// kSegments, at max[segment * blockDim.x + threadIdx.x].
constexpr int kSegments = 8;
struct NoSegments {
  __device__ __forceinline__ void add(float) {}
  __device__ __forceinline__ void close() {}
};
struct Segments {
  float* max;
  int length, done = 0, segment = 0;
  float m = -INFINITY;
  __device__ __forceinline__ Segments(float* smem, int nvec, int group)
      : max(smem), length((nvec + group * kSegments * blockDim.x - 1) / (group * kSegments * blockDim.x)) {}
  __device__ __forceinline__ void add(float group_max) {
    m = fmaxf(m, group_max);
    if (++done == length) close();
  }
  __device__ __forceinline__ void close() {
    if (done == 0) return;
    max[segment++ * blockDim.x + threadIdx.x] = m;
    m = -INFINITY;
    done = 0;
  }
};

// One thread's share of a row, kGroup 16-byte loads at a time: every maximum is taken over a group
// before its exponentials, so the sums are rescaled only when the thread's maximum grows. `first` runs
// once, when the first group is through: what it loads is on its way while the rest of the row is read.
template <typename T, bool kEntropy, int kGroup, typename Seg, typename First>
__device__ __forceinline__ Running<kEntropy> scan_row(const Row<T>& r, float s2, Seg& seg, First first) {
  Running<kEntropy> run;
  auto one = [&](float z) {
    if (z > run.mx) run.raise(z, s2);
    run.add(z, run.mu(), s2);
  };
  const int tid = threadIdx.x, step = blockDim.x;
  for (int i = tid; i < r.head; i += step) one(HalfTraits<T>::to_f(r.p[i]));
  for (int i = r.tail() + tid; i < r.n; i += step) one(HalfTraits<T>::to_f(r.p[i]));
  const uint4* v = r.vec();
  int c = tid;
  for (; c + (kGroup - 1) * step < r.nvec; c += kGroup * step) {
    uint4 u[kGroup];
#pragma unroll
    for (int k = 0; k < kGroup; ++k) u[k] = v[c + k * step];
    seg.add(run.template add_group<T>(u, s2));
    if (c < step) first();
  }
  uint4 u[kGroup];   // the rest: all its loads first, too
#pragma unroll
  for (int k = 0; k < kGroup; ++k)
    if (c + k * step < r.nvec) u[k] = v[c + k * step];
  if (c < step) first();
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kGroup; ++k)
    if (c + k * step < r.nvec) {
      const uint4 single[1] = {u[k]};
      m = fmaxf(m, run.template add_group<T>(single, s2));
    }
  if (c < r.nvec) seg.add(m);   // (not an empty rest: a row of exactly kSegments full segments has no more)
  seg.close();
  return run;
}

// The block's statistics, in every thread. `red` holds 3 x 32 floats.
template <bool kEntropy>
__device__ __forceinline__ Running<kEntropy> block_merge(Running<kEntropy> run, float s2, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const float m = warp_max(run.mx);
  run.rebase(m, s2);
  run.mx = m;
  run.l = warp_sum(run.l);
  if (kEntropy) run.a = warp_sum(run.a);
  if (lane == 0) {
    red[warp] = run.mx;
    red[32 + warp] = run.l;
    if (kEntropy) red[64 + warp] = run.a;
  }
  __syncthreads();
  Running<kEntropy> all;
  for (int w = 0; w < nw; ++w) all.mx = fmaxf(all.mx, red[w]);
  for (int w = 0; w < nw; ++w) {   // the same order in every thread: the same bits
    Running<kEntropy> x;
    x.mx = red[w];
    x.l = red[32 + w];
    if (kEntropy) x.a = red[64 + w];
    x.rebase(all.mx, s2);
    all.l += x.l;
    if (kEntropy) all.a += x.a;
  }
  return all;
}

// ---------------------------------------------------------------------------------------------
// top alternatives
// ---------------------------------------------------------------------------------------------
// Exact selection without keeping the row: the k-th largest of the threads' maxima is a lower bound
// of the k-th largest element, and only segments whose own maximum reaches it can hold candidates.
// The block reads those few segments again (they are still in L2). The candidates carry
// (key, ~token id), so ties go to the lowest id and the order in which they were found does
// not matter. Where the bound is loose (a row of equal values, masked rows) and more than
// kCandidates elements reach it, the exact k-th key and then the id up to which ties are taken are
// found by bisection over their bits, with counts over the whole row.
constexpr int kCandidates = 512;

template <typename T, typename F>
__device__ __forceinline__ void for_own(const Row<T>& r, F f) {   // f(value, local id) over a thread's share
  const int tid = threadIdx.x, step = blockDim.x;
  for (int i = tid; i < r.head; i += step) f(HalfTraits<T>::to_f(r.p[i]), i);
  for (int i = r.tail() + tid; i < r.n; i += step) f(HalfTraits<T>::to_f(r.p[i]), i);
  const uint4* v = r.vec();
#pragma unroll 4
  for (int c = tid; c < r.nvec; c += step) {
    float x[kVec<T>];
    unpack<T>(v[c], x);
#pragma unroll
    for (int j = 0; j < kVec<T>; ++j) f(x[j], r.head + c * kVec<T> + j);
  }
}

// the value of a key (of NaN: some NaN)
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

template <int kThreads> struct SelectSmem {
  float segment_max[kThreads * kSegments];
  unsigned long long cand[kCandidates];
  unsigned long long best[kMaxTopAlternatives];
  unsigned short owner[kThreads * kSegments];   // segments with candidates: segment * threads + thread
  int count, owners;
  int sums[32];
};

__device__ __forceinline__ int block_count(int v, int* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if (lane == 0) sums[warp] = v;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, lane < nw ? sums[lane] : 0);
}

// s.best[0..k) = the k largest (key << 32 | ~id), in falling order. Needs k <= blockDim.x, k <= r.n.
template <typename T, int kGroup, int kThreads>
__device__ void select_top(const Row<T>& r, int k, float thread_max, bool thread_nan, const Segments& seg,
                           SelectSmem<kThreads>& s) {
  const int tid = threadIdx.x;
  uint32_t own = 0;                          // below the key of -inf: a thread without elements
  const bool any = tid < r.head || r.tail() + tid < r.n || tid < r.nvec;
  constexpr float kTiny = 1.17549435e-38f;   // below it float comparisons flush
  const bool unsure = thread_nan || fabsf(thread_max) < kTiny;
  if (unsure) {
    // NaN or +inf among this thread's elements, or a maximum so small that the float comparisons
    // behind it flushed its competitors: take the true maximum
    for_own(r, [&](float z, int) { own = max(own, order_key(z)); });
  } else if (any) {
    own = order_key(thread_max);
  }
  uint32_t bound = 0;
  // 16-bit types widen exactly: their keys differ in the upper bits only (the lower 16 are all 0 for
  // positive, all 1 for negative values), for fp16 in the upper 19
  constexpr int kLow = std::is_same<T, __nv_bfloat16>::value ? 16 : std::is_same<T, __half>::value ? 13 : 0;
  for (int bit = 31; bit >= kLow; --bit) {
    const uint32_t cand = bound | (1u << bit);
    if (__syncthreads_count(own >= cand) >= k) bound = cand;
  }
  if (tid == 0) s.count = s.owners = 0;
  __syncthreads();
  auto take = [&](float z, int id) {
    const uint32_t key = order_key(z);
    if (key >= bound) {
      const int at = atomicAdd(&s.count, 1);
      if (at < kCandidates) s.cand[at] = (static_cast<unsigned long long>(key) << 32) | (0xffffffffu - id);
    }
  };
  if (own >= bound && any) {
    const bool all = unsure || fabsf(value_of(bound)) < kTiny;
    for (int g = 0; g < seg.segment; ++g)
      if (all || order_key(seg.max[g * kThreads + tid]) >= bound)
        s.owner[atomicAdd(&s.owners, 1)] = static_cast<unsigned short>(g * kThreads + tid);
    for (int i = tid; i < r.head; i += kThreads) take(HalfTraits<T>::to_f(r.p[i]), i);
    for (int i = r.tail() + tid; i < r.n; i += kThreads) take(HalfTraits<T>::to_f(r.p[i]), i);
  }
  __syncthreads();
  // The block reads the segments' vectors together, eight lanes a segment and four loads a thread at a time.
  // What cannot be a candidate is sorted out by float comparisons (they flush below kTiny, where all pass; NaN
  // passes), the rest by its key.
  const float least = fabsf(value_of(bound)) < kTiny ? -INFINITY : value_of(bound);
  const int per = seg.length * kGroup, owners = s.owners;
  constexpr int kLanes = 8, kTeams = kThreads / kLanes;
  for (int o = tid / kLanes; o < owners; o += 4 * kTeams)
    for (int i = tid % kLanes; i < per; i += kLanes) {
      uint4 u[4];
      int at[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        at[q] = -1;
        if (o + q * kTeams < owners) {
          const int own_seg = s.owner[o + q * kTeams];
          const int c = (own_seg / kThreads * per + i) * kThreads + own_seg % kThreads;
          if (c < r.nvec) at[q] = c;
        }
        if (at[q] >= 0) u[q] = r.vec()[at[q]];
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (at[q] < 0) continue;
        float x[kVec<T>];
        unpack<T>(u[q], x);
        uint32_t in = 0;
#pragma unroll
        for (int j = 0; j < kVec<T>; ++j) in |= !(x[j] < least) ? 1u << j : 0u;
        for (; in != 0; in &= in - 1) {
          const int j = __ffs(in) - 1;
          float z = x[0];
#pragma unroll
          for (int e = 1; e < kVec<T>; ++e) z = j == e ? x[e] : z;
          take(z, r.head + at[q] * kVec<T> + j);
        }
      }
    }
  __syncthreads();
  int found = s.count;
  if (found > kCandidates || found < k) {   // (fewer than k cannot be; the exact way needs no such argument)
    uint32_t kth = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t cand = kth | (1u << bit);
      int n = 0;
      for_own(r, [&](float z, int) { n += order_key(z) >= cand; });
      if (block_count(n, s.sums) >= k) kth = cand;
    }
    int above = 0;
    for_own(r, [&](float z, int) { above += order_key(z) > kth; });
    const int ties = k - block_count(above, s.sums);     // >= 1 elements equal to the k-th are taken
    int upto = 0;                                         // the largest id with fewer than `ties` ties below it
    for (int bit = 30; bit >= 0; --bit) {
      const int cand = upto + (1 << bit);
      if (cand > r.n) continue;
      int n = 0;
      for_own(r, [&](float z, int id) { n += order_key(z) == kth && id < cand; });
      if (block_count(n, s.sums) < ties) upto = cand;
    }
    if (tid == 0) s.count = 0;
    __syncthreads();
    for_own(r, [&](float z, int id) {
      const uint32_t key = order_key(z);
      if (key > kth || (key == kth && id <= upto)) {
        const int at = atomicAdd(&s.count, 1);
        if (at < kCandidates) s.cand[at] = (static_cast<unsigned long long>(key) << 32) | (0xffffffffu - id);
      }
    });
    __syncthreads();
    found = min(s.count, kCandidates);
  }
  for (int i = tid; i < found; i += blockDim.x) {         // rank by counting: all candidates are distinct
    const unsigned long long mine = s.cand[i];
    int rank = 0;
    for (int j = 0; j < found; ++j) rank += s.cand[j] > mine;
    if (rank < k) s.best[rank] = mine;
  }
  __syncthreads();
}

// The sum of exponentials as the backward gets it: negative where the row's token lies outside the vocabulary
// (zt is NaN), so that the gradient of its log-probability, which is NaN, is NaN as well.
__device__ __forceinline__ float marked_sum(float l, bool scored, float zt) {
  return scored && zt != zt ? -l : l;
}

constexpr int kScanGroup = 8;   // loads in flight per thread of the kernels that read a row once

// ---------------------------------------------------------------------------------------------
// token log-probabilities, entropy, alternatives: forward
// ---------------------------------------------------------------------------------------------
// Bound by reading the logits. Each CTA waits at its end (merge, selection), so many small CTAs keep
// most of an SM loading, with eight loads in flight per thread so that a few of them suffice when the
// last rows run out. Without the entropy, GB/s for 128 threads x 8 per SM, 256 x 4, 512 x 2 and 1024 x 1:
// 8192 x 50304 bf16 6590, 6230, 4715, 2452; 2048 x 128000 5928, 6055, 5556, 3933; 250 x 50304 fp32
// 3816, 4203, 3920, 2938. With alternatives there are loads behind the row (select_top) that queue behind
// all that the SM's other rows have requested. 8192 x 50304 bf16 with 32 of them, back to back: eight loads a
// thread and 8 CTAs per SM 187 us, 7 and 9 CTAs 192 and 195, four loads and 10 or 12 CTAs 190 and 194. With
// 256 threads (100 of them) four loads and 6 CTAs 255, eight and 4 262.
template <typename T, bool kTop, int kThreads, int kPerSm>
__global__ void __launch_bounds__(kThreads, kPerSm)
token_scores_kernel(const T* __restrict__ z, int64_t ld, int vocab, int64_t v0, const int64_t* __restrict__ tokens,
                    int top_k, float inv_t, TokenScoresOut out, float* __restrict__ partial) {
  constexpr int kGroup = kTop && kThreads == 256 ? 4 : kScanGroup;
  __shared__ float red[96];
  __shared__ SelectSmem<kThreads> sel;
  const int64_t row = blockIdx.x;
  const Row<T> r(z + row * ld, vocab);
  const float s2 = inv_t * kLog2e;
  using Seg = std::conditional_t<kTop, Segments, NoSegments>;
  Seg seg = [&] {
    if constexpr (kTop) return Segments(sel.segment_max, r.nvec, kGroup);
    else return NoSegments{};
  }();
  bool scored = false;
  float zt = CUDART_NAN_F;
  const Running<true> own = scan_row<T, true, kGroup>(r, s2, seg, [&] {
    if (threadIdx.x != 0) return;
    const int64_t t = tokens[row], local = t - v0;
    scored = t >= 0;
    if (t >= 0 && local >= 0 && local < vocab) zt = HalfTraits<T>::to_f(r.p[local]);
  });
  const Running<true> all = block_merge<true>(own, s2, red);
  const float mu = all.mu();
  const float log_l = kLn2 * log2f(all.l);
  const int width = 4 + 2 * top_k;
  if (threadIdx.x == 0) {
    if (partial != nullptr) {
      float* q = partial + row * width;
      q[0] = all.mx; q[1] = all.l; q[2] = all.a; q[3] = zt;
    } else {
      out.logprob[row] = scored ? (zt - mu) * inv_t - log_l : 0.f;
      out.entropy[row] = log_l - kLn2 * (all.a / all.l);
      out.stats[2 * row] = mu;
      out.stats[2 * row + 1] = marked_sum(all.l, scored, zt);
    }
  }
  if constexpr (kTop) {
    select_top<T, kGroup>(r, top_k, own.mx, own.l != own.l, seg, sel);
    for (int i = threadIdx.x; i < top_k; i += blockDim.x) {
      const int id = static_cast<int>(0xffffffffu - static_cast<uint32_t>(sel.best[i]));
      const float zi = value_of(static_cast<uint32_t>(sel.best[i] >> 32));
      if (partial != nullptr) {
        partial[row * width + 4 + i] = zi;
        partial[row * width + 4 + top_k + i] = __int_as_float(static_cast<int>(id + v0));
      } else {
        out.top_logprob[row * top_k + i] = (zi - mu) * inv_t - log_l;
        out.top_index[row * top_k + i] = id + v0;
      }
    }
  }
}

// Merges the shards' parts of one row per warp. Every candidate is ranked by counting the better
// ones among all shards' candidates, as in select_top.
__global__ void token_scores_combine_kernel(const float* __restrict__ parts, int world, int64_t rows,
                                            const int64_t* __restrict__ tokens, int top_k, float inv_t,
                                            TokenScoresOut out) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int width = 4 + 2 * top_k;
  const float s2 = inv_t * kLog2e;
  float mx = -INFINITY;
  for (int w = 0; w < world; ++w) mx = fmaxf(mx, parts[(w * rows + row) * width]);
  Running<true> all;
  all.mx = mx;
  float zt = CUDART_NAN_F;
  for (int w = 0; w < world; ++w) {
    const float* q = parts + (w * rows + row) * width;
    Running<true> x;
    x.mx = q[0]; x.l = q[1]; x.a = q[2];
    x.rebase(mx, s2);
    all.l += x.l;
    all.a += x.a;
    if (q[3] == q[3]) zt = q[3];
  }
  const float mu = all.mu(), log_l = kLn2 * log2f(all.l);
  if (lane == 0) {
    out.logprob[row] = tokens[row] < 0 ? 0.f : (zt - mu) * inv_t - log_l;
    out.entropy[row] = log_l - kLn2 * (all.a / all.l);
    out.stats[2 * row] = mu;
    out.stats[2 * row + 1] = marked_sum(all.l, tokens[row] >= 0, zt);
  }
  auto key = [&](int c) {
    const float* q = parts + ((c / top_k) * rows + row) * width + 4 + c % top_k;
    return (static_cast<unsigned long long>(order_key(q[0])) << 32) |
           (0xffffffffu - static_cast<uint32_t>(__float_as_int(q[top_k])));
  };
  for (int c = lane; c < world * top_k; c += 32) {
    const unsigned long long mine = key(c);
    int rank = 0;
    for (int o = 0; o < world * top_k; ++o) rank += key(o) > mine;
    if (rank < top_k) {
      const float* q = parts + ((c / top_k) * rows + row) * width + 4 + c % top_k;
      out.top_logprob[row * top_k + rank] = (q[0] - mu) * inv_t - log_l;
      out.top_index[row * top_k + rank] = __float_as_int(q[top_k]);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// gradients: dz_j = p_j (A + B log p_j) + sum of the listed weights of j
// ---------------------------------------------------------------------------------------------
// The listed entries (a token, alternatives, a teacher's list) are few: their logits are read before
// the dense pass, which may overwrite them, and the finished values are stored after it. The same id
// may be listed several times; the first entry stores the sum of all, added in list order.
struct Listed {
  int id[kMaxTeacherEntries + 1];      // local token id, -1: not on this shard / unused
  float w[kMaxTeacherEntries + 1];
  float z[kMaxTeacherEntries + 1];
};

struct DenseTerm {
  float mu, s2;
  float a, b;       // value = 2^t (a + b t), t = (z - mu) s2; 1 / L, ln L, ln 2 and 1 / temperature are in a and b
  bool floor;       // kLog: masked logits may be raised to kFloor, see has_floor

  // p (A + B log p) with p = 2^t / l
  __device__ __forceinline__ static DenseTerm of(float mu, float l, float s2, float A, float B) {
    DenseTerm f;
    f.mu = mu;
    f.s2 = s2;
    const float inv = 1.0f / l;
    f.a = (B == 0.f ? A : A - B * (kLn2 * log2f(l))) * inv;
    f.b = B * kLn2 * inv;
    f.floor = has_floor(mu, s2) && (mu - kFloor) * s2 * fabsf(f.b) < 1e38f;
    return f;
  }
  template <bool kLog> __device__ __forceinline__ float at(float z) const {
    const float t = (z - mu) * s2, e = exp2f(t);
    return kLog ? e * fmaf(b, fmaxf(t, -1000.f), a) : e * a;
  }
  // logits that are not -inf
  template <bool kLog> __device__ __forceinline__ Pair at(Pair z) const {
    const Pair t = (z + pair(-mu, -mu)) * pair(s2, s2), e = exp2_pair(t);
    return kLog ? e * fma2(pair(b, b), t, pair(a, a)) : e * pair(a, a);
  }
  template <typename T, bool kLog> __device__ __forceinline__ uint4 at(uint4 u) const {
    if constexpr (kLog) {
      if (!floor) {
        float x[kVec<T>];
        unpack<T>(u, x);
#pragma unroll
        for (int j = 0; j < kVec<T>; ++j) x[j] = at<true>(x[j]);
        return repack<T>(x);
      }
      u = at_least<T>(u, kFloor);
    }
    Pair z[kVec<T> / 2];
    unpack_pairs<T>(u, z);
    float x[kVec<T>];
#pragma unroll
    for (int j = 0; j < kVec<T> / 2; ++j) split(at<kLog>(z[j]), x[2 * j], x[2 * j + 1]);
    return repack<T>(x);
  }
};

constexpr int kUnroll = 4;   // loads in flight per thread of the kernels that also write a row

// The whole gradient of a row. The list's logits have been staged before (li.z), behind a barrier.
// kLast: the row's logits are read for the last time.
// weight(i): what entry i adds.
template <typename T, bool kLog, bool kLast, typename Weight>
__device__ __forceinline__ void write_grad(const Row<T>& r, T* __restrict__ d, const DenseTerm& f, const Listed& li,
                                           int n, Weight weight) {
  const int tid = threadIdx.x, step = blockDim.x;
  if (((reinterpret_cast<uintptr_t>(r.p) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0) {
    for (int i = tid; i < r.head; i += step)
      d[i] = HalfTraits<T>::from_f(f.template at<kLog>(HalfTraits<T>::to_f(r.p[i])));
    for (int i = r.tail() + tid; i < r.n; i += step)
      d[i] = HalfTraits<T>::from_f(f.template at<kLog>(HalfTraits<T>::to_f(r.p[i])));
    const uint4* v = r.vec();
    uint4* o = reinterpret_cast<uint4*>(d + r.head);
    for (int c = tid; c < r.nvec; c += kUnroll * step) {
      uint4 u[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k)
        if (c + k * step < r.nvec) u[k] = kLast ? __ldcs(v + c + k * step) : v[c + k * step];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k)
        if (c + k * step < r.nvec) __stcs(o + c + k * step, f.template at<T, kLog>(u[k]));
    }
  } else {   // rows of logits and gradient at different offsets from a 16-byte boundary
    for (int i = tid; i < r.n; i += step)
      d[i] = HalfTraits<T>::from_f(f.template at<kLog>(HalfTraits<T>::to_f(r.p[i])));
  }
  __syncthreads();
  for (int i = tid; i < n; i += step) {
    const int id = li.id[i];
    if (id < 0) continue;
    bool first = true;
    for (int j = 0; j < i; ++j) first &= li.id[j] != id;
    if (!first) continue;
    float w = weight(i);
    for (int j = i + 1; j < n; ++j)
      if (li.id[j] == id) w += weight(j);
    d[id] = HalfTraits<T>::from_f(f.template at<kLog>(li.z[i]) + w);
  }
}

template <typename T>
__device__ __forceinline__ void write_zero(T* __restrict__ d, int vocab) {
  const Row<T> o(d, vocab);
  const int tid = threadIdx.x, step = blockDim.x;
  for (int i = tid; i < o.head; i += step) d[i] = HalfTraits<T>::from_f(0.f);
  for (int i = o.tail() + tid; i < vocab; i += step) d[i] = HalfTraits<T>::from_f(0.f);
  uint4* v = reinterpret_cast<uint4*>(d + o.head);
  for (int c = tid; c < o.nvec; c += step) v[c] = make_uint4(0, 0, 0, 0);
}

template <typename T, bool kLog>
__global__ void token_scores_bwd_kernel(const T* z, int64_t ld, int vocab, int64_t v0,
                                        const int64_t* __restrict__ tokens, const float* __restrict__ stats,
                                        const float* __restrict__ entropy, const int64_t* __restrict__ top_index,
                                        int top_k, float inv_t, const float* __restrict__ g,
                                        const float* __restrict__ h, const float* __restrict__ u, T* dz, int64_t ldd) {
  __shared__ Listed li;
  __shared__ float usum;
  const int64_t row = blockIdx.x;
  const Row<T> r(z + row * ld, vocab);
  const int64_t t = tokens[row];
  const float gr = g != nullptr && t >= 0 ? g[row] : 0.f;
  const float hr = kLog ? h[row] : 0.f;
  // requested before the list's barrier: the sum of exponentials (see marked_sum), the maximum, the entropy
  const float l = stats[2 * row + 1], mu = stats[2 * row], ent = kLog ? entropy[row] : 0.f;
  const int extra = u != nullptr ? top_k : 0;
  if (threadIdx.x < 32) {
    float sum = 0.f;
    for (int i = threadIdx.x; i < extra; i += 32) {
      const float w = u[row * top_k + i];
      const int64_t id = top_index[row * top_k + i] - v0;
      const bool here = id >= 0 && id < vocab && w != 0.f;
      li.id[1 + i] = here ? static_cast<int>(id) : -1;
      li.w[1 + i] = w * inv_t;
      li.z[1 + i] = here ? HalfTraits<T>::to_f(r.p[id]) : 0.f;
      sum += w;
    }
    sum = warp_sum(sum);
    if (threadIdx.x == 0) {
      const int64_t id = t - v0;
      const bool here = gr != 0.f && id >= 0 && id < vocab;
      li.id[0] = here ? static_cast<int>(id) : -1;
      li.w[0] = gr * inv_t;
      li.z[0] = here ? HalfTraits<T>::to_f(r.p[id]) : 0.f;
      usum = sum;
    }
  }
  __syncthreads();
  T* d = dz + row * ldd;
  // a row that no gradient reaches (a masked token): its logits are not looked at
  int live = gr != 0.f || hr != 0.f;
  for (int i = 0; i < extra && !live; ++i) live = u[row * top_k + i] != 0.f;
  if (!live) {
    write_zero(d, vocab);
    return;
  }
  const float A = l < 0.f && gr != 0.f ? CUDART_NAN_F : -(gr + usum + (kLog ? hr * ent : 0.f)) * inv_t;
  const DenseTerm f = DenseTerm::of(mu, fabsf(l), inv_t * kLog2e, A, kLog ? -hr * inv_t : 0.f);
  write_grad<T, kLog, false>(r, d, f, li, 1 + extra, [&](int i) { return li.w[i]; });
}

// ---------------------------------------------------------------------------------------------
// loss against a teacher's top logits
// ---------------------------------------------------------------------------------------------
// q = softmax of the listed teacher logits / T (entries at -inf have no weight; a row without any
// entry has no loss), loss = sum_k q_k (log q_k - log p_{i_k}), dz_j = g / T (p_j sum q - sum_{i_k = j} q_k).
struct TeacherRow {
  float tmax, log_sum, mass;   // mass: sum of q (1, or 0 for an empty row)
};

// The row's list in shared memory: local ids (-1: not on this shard or unused), teacher logits, student
// logits. Staged while the row is read (scan_row's `first`), so only the few warps that hold entries wait
// for the two dependent loads, the others read on; a barrier follows. `whole`: the row is the whole vocabulary,
// where a used entry that lies outside turns its teacher logit, and so the row's loss and gradient, into NaN.
template <typename T>
__device__ __forceinline__ void stage_list(const TeacherView& t, int64_t row, const Row<T>& r, int64_t v0, bool whole,
                                           Listed& li) {
  for (int i = threadIdx.x; i < t.k; i += blockDim.x) {
    const float logit = t.logit[row * t.k + i];
    const int64_t id = t.index[row * t.k + i] - v0;
    const bool used = logit != -INFINITY, here = used && id >= 0 && id < r.n;
    li.w[i] = whole && used && !here ? CUDART_NAN_F : logit;
    li.id[i] = here ? static_cast<int>(id) : -1;
    li.z[i] = here ? HalfTraits<T>::to_f(r.p[id]) : CUDART_NAN_F;
  }
}

// The teacher's side of a staged row; every warp works it out for itself.
__device__ __forceinline__ TeacherRow teacher_row(const Listed& li, int k, float inv_t) {
  const int lane = threadIdx.x & 31;
  float mx = -INFINITY, sum = 0.f;
  bool nan = false;
  for (int i = lane; i < k; i += 32) {
    mx = fmaxf(mx, li.w[i]);
    nan |= li.w[i] != li.w[i];
  }
  mx = warp_max(mx);
  nan = __any_sync(0xffffffffu, nan);
  if (mx == -INFINITY && !nan) return {mx, 0.f, 0.f};
  for (int i = lane; i < k; i += 32) sum += exp2f((li.w[i] - mx) * inv_t * kLog2e);
  sum = nan ? CUDART_NAN_F : warp_sum(sum);
  return {mx, kLn2 * log2f(sum), sum == sum ? 1.f : sum};
}
// log q of a listed teacher logit
__device__ __forceinline__ float log_weight(const TeacherRow& t, float logit, float inv_t) {
  return (logit - t.tmax) * inv_t - t.log_sum;
}

// One warp: the loss of a staged row of the whole vocabulary; 0 where there are no entries.
__device__ __forceinline__ float listed_loss(const Listed& li, int k, const TeacherRow& tr, float inv_t, float mu,
                                             float log_l) {
  float part = 0.f;
  if (tr.mass == 0.f) return 0.f;
  for (int i = threadIdx.x & 31; i < k; i += 32) {
    const float log_q = log_weight(tr, li.w[i], inv_t), q = exp2f(log_q * kLog2e);
    if (q != 0.f) part += q * (log_q - ((li.z[i] - mu) * inv_t - log_l));
  }
  return warp_sum(part);
}

// Same shape as token_scores_kernel, without the entropy (8192 x 50304 bf16: 6.6 TB/s).
template <typename T, int kThreads, int kPerSm>
__global__ void __launch_bounds__(kThreads, kPerSm)
distill_fwd_kernel(const T* __restrict__ z, int64_t ld, int vocab, int64_t v0, TeacherView t, float inv_t,
                   float* __restrict__ loss, float* __restrict__ stats, float* __restrict__ partial) {
  __shared__ float red[96];
  __shared__ Listed li;
  const int64_t row = blockIdx.x;
  const Row<T> r(z + row * ld, vocab);
  const float s2 = inv_t * kLog2e;
  NoSegments none;
  const Running<false> own = scan_row<T, false, kScanGroup>(r, s2, none, [&] {
    stage_list(t, row, r, v0, partial == nullptr, li);
  });
  const Running<false> all = block_merge<false>(own, s2, red);   // its barrier publishes the list, too
  if (threadIdx.x >= 32) return;
  const float mu = all.mu();
  const TeacherRow tr = teacher_row(li, t.k, inv_t);
  if (partial != nullptr) {
    float found = 0.f, weight = 0.f, count = 0.f;
    for (int i = threadIdx.x; i < t.k && tr.mass != 0.f; i += 32) {
      if (li.id[i] < 0) continue;
      const float q = exp2f(log_weight(tr, li.w[i], inv_t) * kLog2e);
      if (q != 0.f) found += q * ((li.z[i] - mu) * inv_t);
      weight += q;
      count += 1.f;
    }
    found = warp_sum(found);
    weight = warp_sum(weight);
    count = warp_sum(count);
    if (threadIdx.x == 0) {
      float* q = partial + row * kDistillParts;
      q[0] = all.mx; q[1] = all.l; q[2] = found; q[3] = weight; q[4] = count;
    }
    return;
  }
  const float l = listed_loss(li, t.k, tr, inv_t, mu, kLn2 * log2f(all.l));
  if (threadIdx.x == 0) {
    const bool empty = tr.mass == 0.f;   // nothing listed: no loss, whatever the logits
    loss[row] = l;
    stats[2 * row] = empty ? 0.f : mu;
    stats[2 * row + 1] = empty ? 1.f : all.l * tr.mass;   // NaN like the loss where the list is bad
  }
}

__global__ void distill_combine_kernel(const float* __restrict__ parts, int world, int64_t rows, TeacherView t,
                                       float inv_t, float* __restrict__ loss, float* __restrict__ stats) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= rows) return;
  const float s2 = inv_t * kLog2e;
  float mx = -INFINITY;
  for (int w = 0; w < world; ++w) mx = fmaxf(mx, parts[(w * rows + row) * kDistillParts]);
  Running<false> all;
  all.mx = mx;
  const float mu = all.mu();
  float found = 0.f, count = 0.f;
  for (int w = 0; w < world; ++w) {
    const float* q = parts + (w * rows + row) * kDistillParts;
    Running<false> x;
    x.mx = q[0]; x.l = q[1];
    if (q[3] != 0.f) found += q[2] + q[3] * ((x.mu() - mu) * inv_t);
    count += q[4];
    x.rebase(mx, s2);
    all.l += x.l;
  }
  const float* tl = t.logit + row * t.k;
  float tmax = -INFINITY, sum = 0.f, self = 0.f, used = 0.f;
  bool nan = false;
  for (int i = lane; i < t.k; i += 32) {
    tmax = fmaxf(tmax, tl[i]);
    nan |= tl[i] != tl[i];
    used += tl[i] != -INFINITY;
  }
  tmax = warp_max(tmax);
  used = warp_sum(used);
  nan = __any_sync(0xffffffffu, nan);
  const bool empty = tmax == -INFINITY && !nan;
  for (int i = lane; i < t.k; i += 32) sum += empty ? 0.f : exp2f((tl[i] - tmax) * inv_t * kLog2e);
  sum = nan ? CUDART_NAN_F : warp_sum(sum);
  const float log_sum = kLn2 * log2f(sum), inv = 1.0f / sum;
  for (int i = lane; i < t.k && !empty; i += 32) {
    const float x = (tl[i] - tmax) * inv_t, q = exp2f(x * kLog2e) * inv;
    if (q != 0.f) self += q * (x - log_sum);
  }
  self = warp_sum(self);
  if (lane == 0) {
    const bool whole = count == used;   // else an entry lies outside the vocabulary
    loss[row] = empty ? 0.f : whole ? self - found + kLn2 * log2f(all.l) : CUDART_NAN_F;
    stats[2 * row] = empty ? 0.f : mu;
    stats[2 * row + 1] = empty ? 1.f : whole ? all.l : CUDART_NAN_F;   // the gradient is NaN as well
  }
}

// what entry i of a list adds to its token's gradient
__device__ __forceinline__ float listed_grad(const Listed& li, const TeacherRow& tr, float inv_t, float g, int i) {
  return -g * exp2f(log_weight(tr, li.w[i], inv_t) * kLog2e);
}

template <typename T>
__global__ void distill_bwd_kernel(const T* z, int64_t ld, int vocab, int64_t v0, TeacherView t, float inv_t,
                                   const float* __restrict__ stats, const float* __restrict__ dloss, T* dz,
                                   int64_t ldd) {
  __shared__ Listed li;
  const int64_t row = blockIdx.x;
  const Row<T> r(z + row * ld, vocab);
  T* d = dz + row * ldd;
  const float g = dloss[row] * inv_t;
  stage_list(t, row, r, v0, false, li);
  __syncthreads();
  const TeacherRow tr = teacher_row(li, t.k, inv_t);
  if (tr.mass == 0.f || g == 0.f) {
    write_zero(d, vocab);
    return;
  }
  const DenseTerm f = DenseTerm::of(stats[2 * row], stats[2 * row + 1], inv_t * kLog2e, g * tr.mass, 0.f);
  write_grad<T, false, false>(r, d, f, li, t.k, [&](int i) { return listed_grad(li, tr, inv_t, g, i); });
}

// Loss and gradient of a row in one CTA: the second reading of the row comes out of L2, so DRAM sees
// the logits once and the gradient once. That needs the rows in flight to stay in L2 beside the
// gradients being written: the second reading and the stores are marked as not needed again, and long
// rows run fewer at a time (launch_step). Without the marks a burst of 8192 x 50304 bf16 takes 334 us in
// place of 268; with the row kept in shared memory instead of read again 327, as two rows per SM leave
// too little in flight.
template <typename T, int kThreads, int kPerSm>
__global__ void __launch_bounds__(kThreads, kPerSm)
distill_step_kernel(const T* z, int64_t ld, int vocab, int64_t v0, TeacherView t, float inv_t,
                    const float* __restrict__ dloss, float* __restrict__ loss, T* dz, int64_t ldd) {
  __shared__ float red[96];
  __shared__ Listed li;
  const int64_t row = blockIdx.x;
  const Row<T> r(z + row * ld, vocab);
  T* d = dz + row * ldd;
  const float s2 = inv_t * kLog2e;
  const float g = dloss[row] * inv_t;
  NoSegments none;
  const Running<false> own = scan_row<T, false, kUnroll>(r, s2, none, [&] { stage_list(t, row, r, v0, true, li); });
  const Running<false> all = block_merge<false>(own, s2, red);
  const float mu = all.mu();
  const TeacherRow tr = teacher_row(li, t.k, inv_t);
  if (tr.mass == 0.f || g == 0.f) {
    write_zero(d, vocab);
  } else {
    const DenseTerm f = DenseTerm::of(mu, all.l, s2, g * tr.mass, 0.f);
    write_grad<T, false, true>(r, d, f, li, t.k, [&](int i) { return listed_grad(li, tr, inv_t, g, i); });
  }
  if (threadIdx.x < 32) {
    const float l = listed_loss(li, t.k, tr, inv_t, mu, kLn2 * log2f(all.l));
    if (threadIdx.x == 0) loss[row] = l;
  }
}

// Below a row per SM, more threads shorten the single row.
bool few_rows(int64_t rows, int vocab) { return rows < 148 && vocab > 4096; }
int threads_for(int64_t rows, int vocab) { return few_rows(rows, vocab) ? 512 : 256; }

cudaError_t check_view(const LogitsView& a) {
  ETHB_RETURN_IF(a.rows < 0 || a.vocab <= 0, cudaErrorInvalidValue, "token loss: empty vocabulary");
  ETHB_RETURN_IF(a.rows > 0x7fffffffLL, cudaErrorInvalidValue, "token loss: too many rows for one grid");
  ETHB_RETURN_IF(a.dtype != kF32 && a.dtype != kF16 && a.dtype != kBF16, cudaErrorInvalidValue, "token loss: dtype");
  return cudaSuccess;
}

// With 128 threads the bound on the k-th alternative (the k-th largest of as many maxima) is loose for k
// near 128: about 620 elements would reach it. 256 threads leave about 180. 8192 x 50304 bf16: 235 us with
// 128 threads against 238 at k = 72, 264 against 249 at 88, 344 against 274 at 112.
template <typename T>
void launch_scores_for(const LogitsView& a, const int64_t* tokens, int top_k, const TokenScoresOut& out, float* partial,
                       cudaStream_t st) {
  const auto go = [&](auto* kernel, int threads) {
    kernel<<<static_cast<unsigned>(a.rows), threads, 0, st>>>(static_cast<const T*>(a.z), a.ld, a.vocab, a.v0, tokens,
                                                              top_k, a.inv_temperature, out, partial);
  };
  if (few_rows(a.rows, a.vocab))
    top_k > 0 ? go(token_scores_kernel<T, true, 512, 2>, 512) : go(token_scores_kernel<T, false, 512, 2>, 512);
  else if (top_k > 64)
    go(token_scores_kernel<T, true, 256, 6>, 256);
  else
    top_k > 0 ? go(token_scores_kernel<T, true, 128, 8>, 128) : go(token_scores_kernel<T, false, 128, 8>, 128);
}
cudaError_t launch_scores(const LogitsView& a, const int64_t* tokens, int top_k, const TokenScoresOut& out,
                          float* partial, cudaStream_t st) {
  ETHB_TRY(check_view(a), "token_scores");
  ETHB_RETURN_IF(top_k < 0 || top_k > kMaxTopAlternatives || top_k > a.vocab, cudaErrorInvalidValue, "top_k");
  if (a.rows == 0) return cudaSuccess;
  ETHB_DISPATCH_T(a.dtype, T, launch_scores_for<T>(a, tokens, top_k, out, partial, st));
  count_launch();
  return cudaGetLastError();
}

cudaError_t launch_distill(const LogitsView& a, const TeacherView& t, float* loss, float* stats, float* partial,
                           cudaStream_t st) {
  ETHB_TRY(check_view(a), "distill");
  ETHB_RETURN_IF(t.k < 1 || t.k > kMaxTeacherEntries, cudaErrorInvalidValue, "teacher entries");
  if (a.rows == 0) return cudaSuccess;
  ETHB_DISPATCH_T(a.dtype, T, {
    const auto go = [&](auto* kernel, int threads) {
      kernel<<<static_cast<unsigned>(a.rows), threads, 0, st>>>(static_cast<const T*>(a.z), a.ld, a.vocab, a.v0, t,
                                                                a.inv_temperature, loss, stats, partial);
    };
    few_rows(a.rows, a.vocab) ? go(distill_fwd_kernel<T, 512, 2>, 512) : go(distill_fwd_kernel<T, 128, 8>, 128);
  });
  count_launch();
  return cudaGetLastError();
}

// Rows in flight take SMs x rows per SM x row bytes of L2 (126 MB, which also passes the gradients on):
// four a SM up to 150 KB (89 MB), two beyond. Back to back at the power limit, with 4 x 320, 2 x 512, 3 x
// 512, 1 x 1024 threads: 8192 x 50304 bf16 343, 393, 388, - us; 2048 x 128000 245, 225, 243, 278 us. Between
// them, fp32: 4096 x 50304 349 us with the first, 324 with the second; 1500 x 65536 186 and 179.
template <typename T>
void launch_step(const LogitsView& a, const TeacherView& t, const float* dloss, float* loss, T* dz, int64_t ldd,
                 cudaStream_t st) {
  const auto go = [&](auto* kernel, int threads) {
    kernel<<<static_cast<unsigned>(a.rows), threads, 0, st>>>(static_cast<const T*>(a.z), a.ld, a.vocab, a.v0, t,
                                                              a.inv_temperature, dloss, loss, dz, ldd);
  };
  const int64_t row_bytes = static_cast<int64_t>(a.vocab) * sizeof(T);
  if (few_rows(a.rows, a.vocab) || row_bytes > 150 << 10) go(distill_step_kernel<T, 512, 2>, 512);
  else go(distill_step_kernel<T, 320, 4>, 320);
}

}  // namespace

cudaError_t token_scores(const LogitsView& a, const int64_t* tokens, int top_k, const TokenScoresOut& out,
                         cudaStream_t st) {
  return launch_scores(a, tokens, top_k, out, nullptr, st);
}
cudaError_t token_scores_partial(const LogitsView& a, const int64_t* tokens, int top_k, float* partial,
                                 cudaStream_t st) {
  return launch_scores(a, tokens, top_k, TokenScoresOut{}, partial, st);
}
cudaError_t token_scores_combine(const float* partials, int world, int64_t rows, const int64_t* tokens, int top_k,
                                 float inv_temperature, const TokenScoresOut& out, cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  token_scores_combine_kernel<<<static_cast<unsigned>((rows + 7) / 8), 256, 0, st>>>(partials, world, rows, tokens,
                                                                                   top_k, inv_temperature, out);
  count_launch();
  return cudaGetLastError();
}
cudaError_t token_scores_bwd(const LogitsView& a, const int64_t* tokens, const float* stats, const float* entropy,
                             const int64_t* top_index, int top_k, const float* g, const float* h, const float* u,
                             void* dz, int64_t ldd, cudaStream_t st) {
  ETHB_TRY(check_view(a), "token_scores_bwd");
  ETHB_RETURN_IF(top_k < 0 || top_k > kMaxTopAlternatives, cudaErrorInvalidValue, "top_k");
  if (a.rows == 0) return cudaSuccess;
  const int threads = threads_for(a.rows, a.vocab);
  ETHB_DISPATCH_T(a.dtype, T, {
    if (h != nullptr)
      token_scores_bwd_kernel<T, true><<<static_cast<unsigned>(a.rows), threads, 0, st>>>(
          static_cast<const T*>(a.z), a.ld, a.vocab, a.v0, tokens, stats, entropy, top_index, top_k,
          a.inv_temperature, g, h, u, static_cast<T*>(dz), ldd);
    else
      token_scores_bwd_kernel<T, false><<<static_cast<unsigned>(a.rows), threads, 0, st>>>(
          static_cast<const T*>(a.z), a.ld, a.vocab, a.v0, tokens, stats, entropy, top_index, top_k,
          a.inv_temperature, g, h, u, static_cast<T*>(dz), ldd);
  });
  count_launch();
  return cudaGetLastError();
}

cudaError_t distill_fwd(const LogitsView& a, const TeacherView& t, float* loss, float* stats, cudaStream_t st) {
  return launch_distill(a, t, loss, stats, nullptr, st);
}
cudaError_t distill_partial(const LogitsView& a, const TeacherView& t, float* partial, cudaStream_t st) {
  return launch_distill(a, t, nullptr, nullptr, partial, st);
}
cudaError_t distill_combine(const float* partials, int world, int64_t rows, const TeacherView& t,
                            float inv_temperature, float* loss, float* stats, cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  distill_combine_kernel<<<static_cast<unsigned>((rows + 7) / 8), 256, 0, st>>>(partials, world, rows, t,
                                                                              inv_temperature, loss, stats);
  count_launch();
  return cudaGetLastError();
}
cudaError_t distill_bwd(const LogitsView& a, const TeacherView& t, const float* stats, const float* dloss, void* dz,
                        int64_t ldd, cudaStream_t st) {
  ETHB_TRY(check_view(a), "distill_bwd");
  ETHB_RETURN_IF(t.k < 1 || t.k > kMaxTeacherEntries, cudaErrorInvalidValue, "teacher entries");
  if (a.rows == 0) return cudaSuccess;
  ETHB_DISPATCH_T(a.dtype, T, {
    distill_bwd_kernel<T><<<static_cast<unsigned>(a.rows), threads_for(a.rows, a.vocab), 0, st>>>(
        static_cast<const T*>(a.z), a.ld, a.vocab, a.v0, t, a.inv_temperature, stats, dloss, static_cast<T*>(dz), ldd);
  });
  count_launch();
  return cudaGetLastError();
}
cudaError_t distill_step(const LogitsView& a, const TeacherView& t, const float* dloss, float* loss, void* dz,
                         int64_t ldd, cudaStream_t st) {
  ETHB_TRY(check_view(a), "distill_step");
  ETHB_RETURN_IF(t.k < 1 || t.k > kMaxTeacherEntries, cudaErrorInvalidValue, "teacher entries");
  if (a.rows == 0) return cudaSuccess;
  ETHB_DISPATCH_T(a.dtype, T, {
    launch_step<T>(a, t, dloss, loss, static_cast<T*>(dz), ldd, st);
  });
  count_launch();
  return cudaGetLastError();
}

}  // namespace ethb
