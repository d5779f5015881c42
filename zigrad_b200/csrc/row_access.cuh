// Rows of fp32 or bf16 values read and written in 16-byte words, wherever the row starts.
//
// A row of C elements whose first one lies `lead` elements behind a 16-byte boundary is seen as C + lead positions from that
// boundary on: position p is element p - lead, a word holds kPerWord<T> positions, and only the first and the last word can
// be incomplete.  Those are touched element by element, so nothing outside the row is ever read or written.
#pragma once

#include <cfloat>
#include <cooperative_groups.h>
#include "common.cuh"

namespace zg {
namespace ra {

namespace cg = cooperative_groups;

template <typename T>
constexpr int kPerWord = 16 / (int)sizeof(T);

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The floats of a word
__device__ __forceinline__ void unpack(const uint4& w, float (&x)[4], float) {
  x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void unpack(const uint4& w, float (&x)[8], __nv_bfloat16) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack(const float (&x)[4], float) {
  return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
__device__ __forceinline__ uint4 pack(const float (&x)[8], __nv_bfloat16) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    u[i] = reinterpret_cast<const uint32_t&>(h);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
// A word of -infinity
template <typename T>
__device__ __forceinline__ uint4 nothing();
template <>
__device__ __forceinline__ uint4 nothing<float>() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
template <>
__device__ __forceinline__ uint4 nothing<__nv_bfloat16>() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }

// Elements between the 16-byte boundary in front of p and p
template <typename T>
__device__ __forceinline__ unsigned lead_of(const T* p) { return (unsigned)(reinterpret_cast<uintptr_t>(p) & 15u) / (unsigned)sizeof(T); }

template <typename T>
__device__ __noinline__ uint4 load_word_part(const T* first, unsigned lead, unsigned end, unsigned w) {
  float x[kPerWord<T>];
#pragma unroll
  for (int i = 0; i < kPerWord<T>; ++i) {
    const unsigned p = w * kPerWord<T> + i;
    x[i] = p >= lead && p < end ? as_float(first[p - lead]) : -INFINITY;
  }
  return pack(x, T());
}

template <typename T>
struct Row {
  T* first;        // element 0
  unsigned lead;
  unsigned end;    // C + lead: positions lead .. end - 1 are the row
  __device__ __forceinline__ Row(T* p, unsigned C) : first(p), lead(lead_of(p)), end(C + lead) {}
  __device__ __forceinline__ unsigned words() const { return (end + kPerWord<T> - 1) / kPerWord<T>; }
  __device__ __forceinline__ bool whole(unsigned w) const { return w * kPerWord<T> >= lead && (w + 1) * kPerWord<T> <= end; }
  __device__ __forceinline__ uint4* word(unsigned w) const { return reinterpret_cast<uint4*>(first - lead) + w; }
  // Word w, with -infinity in the positions that are not the row's
  __device__ __forceinline__ uint4 load(unsigned w) const {
    if (whole(w)) return __ldcs(word(w));
    return load_part(w);
  }
  __device__ __forceinline__ uint4 load_part(unsigned w) const { return load_word_part(first, lead, end, w); }
  __device__ __forceinline__ void store(unsigned w, const float (&x)[kPerWord<T>]) const {
    if (whole(w)) { *word(w) = pack(x, T()); return; }
#pragma unroll
    for (int i = 0; i < kPerWord<T>; ++i) {
      const unsigned p = w * kPerWord<T> + i;
      if (p >= lead && p < end) first[p - lead] = from_float<T>(x[i]);
    }
  }
};

// The most words that a row of C elements has, for rows that start ld elements apart from p on
template <typename T>
static inline size_t most_words(const void* p, size_t C, size_t ld) {
  const size_t lead = ld * sizeof(T) % 16 == 0 ? reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T) : kPerWord<T> - 1;
  return (C + lead + kPerWord<T> - 1) / kPerWord<T>;
}

constexpr float kLog2e = 1.4426950408889634f;
// 2^x: the hardware's exponential, about 2^-22 relative; results below 2^-126 are zero
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 2^((x - m) c) for m the largest of the x.  The difference comes first: of values near the type's limits a product would be
// infinite.  An infinite m (nothing but -infinity so far, or a +infinity) is left out of it: 0 and infinity instead of NaN.
__device__ __forceinline__ float shifted_exp(float x, float m, float c) { return exp2_fast((x - (fabsf(m) == INFINITY ? 0.f : m)) * c); }

// Two fp32 values in one register pair, which one instruction adds or multiplies
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair_of(float a, float b) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ void split(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair p;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair p;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}
// shifted_exp of two values: minus_m is -m (0 for an infinite m) and c twice each
__device__ __forceinline__ Pair shifted_exp(float x0, float x1, Pair minus_m, Pair c) {
  float a, b;
  split((pair_of(x0, x1) + minus_m) * c, a, b);
  return pair_of(exp2_fast(a), exp2_fast(b));
}
__device__ __forceinline__ Pair minus(float m) {
  const float v = fabsf(m) == INFINITY ? 0.f : -m;
  return pair_of(v, v);
}
// a b + c
__device__ __forceinline__ Pair fused(Pair a, Pair b, Pair c) {
  Pair p;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return p;
}

// 2^(x c) of many x over 2^(m c), m the largest of them, with m c rounded to fp32: a fused multiply-add per x whose one rounding is
// relative to the exponent itself.  Every sum of such terms is relative to 2^fl(m c), which `log2_of` and `rebased` know.  Where
// m c is not finite, or near it, (x - m) c takes its place, and an infinite m is left out.
template <bool FUSED>
struct Term {
  Pair c, shift;
  __device__ __forceinline__ Pair operator()(float x0, float x1) const {
    float a, b;
    split(FUSED ? fused(pair_of(x0, x1), c, shift) : (pair_of(x0, x1) + shift) * c, a, b);
    return pair_of(exp2_fast(a), exp2_fast(b));
  }
};
struct Scale {
  float c;
  __device__ __forceinline__ float log2_of(float m) const { return __fmul_rn(m, c); }
  __device__ __forceinline__ bool plain(float m) const { return fabsf(log2_of(m)) < 1e38f; }
  // terms relative to m1 -> terms relative to m2
  __device__ __forceinline__ float rebased(float m1, float m2) const {
    return plain(m1) && plain(m2) ? exp2_fast(__fsub_rn(log2_of(m1), log2_of(m2))) : shifted_exp(m1, m2, c);
  }
  __device__ __forceinline__ Term<true> fused_term(float m) const {  // where m is plain
    const float r = -log2_of(m);
    return Term<true>{pair_of(c, c), pair_of(r, r)};
  }
  __device__ __forceinline__ Term<false> shifted_term(float m) const {
    const float v = fabsf(m) == INFINITY ? 0.f : -m;
    return Term<false>{pair_of(c, c), pair_of(v, v)};
  }
};
// The sum of a word's terms
template <typename T, bool FUSED>
__device__ __forceinline__ Pair word_sum(const uint4& v, const Term<FUSED>& term) {
  float x[kPerWord<T>];
  unpack(v, x, T());
  Pair sum = term(x[0], x[1]);
#pragma unroll
  for (int i = 2; i < kPerWord<T>; i += 2) sum = sum + term(x[i], x[i + 1]);
  return sum;
}

// The largest of a word's values, NaNs aside
__device__ __forceinline__ float word_max(const uint4& w, float) {
  return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
}
__device__ __forceinline__ float word_max(const uint4& w, __nv_bfloat16) {
  const auto half = [](const uint32_t& u) { return reinterpret_cast<const __nv_bfloat162&>(u); };
  const __nv_bfloat162 m = __hmax2(__hmax2(half(w.x), half(w.y)), __hmax2(half(w.z), half(w.w)));
  return fmaxf(__low2float(m), __high2float(m));
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The same, and a NaN where there is one
__device__ __forceinline__ float word_max_nan(const uint4& w, float) {
  return max_nan(max_nan(__uint_as_float(w.x), __uint_as_float(w.y)), max_nan(__uint_as_float(w.z), __uint_as_float(w.w)));
}
__device__ __forceinline__ float word_max_nan(const uint4& w, __nv_bfloat16) {
  const auto half = [](const uint32_t& u) { return reinterpret_cast<const __nv_bfloat162&>(u); };
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(half(w.x), half(w.y)), __hmax2_nan(half(w.z), half(w.w)));
  return max_nan(__low2float(m), __high2float(m));
}

// of N words, relative to m
template <typename T, int N>
__device__ __forceinline__ float words_sum(const uint4 (&v)[N], const Scale& scale, float m) {
  Pair sum[N];
  if (scale.plain(m)) {
    const Term<true> term = scale.fused_term(m);
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = word_sum<T>(v[j], term);
  } else {
    const Term<false> term = scale.shifted_term(m);
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = word_sum<T>(v[j], term);
  }
#pragma unroll
  for (int n = 1; n < N; n *= 2)
#pragma unroll
    for (int j = 0; j + n < N; j += 2 * n) sum[j] = sum[j] + sum[j + n];
  float s0, s1;
  split(sum[0], s0, s1);
  return s0 + s1;
}

// A whole number that orders as the value does: NaN above all, -0 and +0 alike, 0 below -infinity
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  if (x != x) return 0xffffffffu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// Clusters of `cluster` CTAs that are on the device together, for a grid that walks its rows: the answer for the last sizes asked
// for is kept per kernel
template <typename K>
static unsigned resident_clusters(K kernel, unsigned threads, size_t smem, unsigned cluster, std::atomic<uint64_t>& last) {
  const uint64_t key = (uint64_t)smem << 36 | (uint64_t)cluster << 32, have = last.load(std::memory_order_relaxed);
  if ((have & ~(uint64_t)0xffffffffu) == key && (uint32_t)have) return (uint32_t)have;
  int n = 0;
  if (cluster == 1) {
    if (!ZG_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, (int)threads, smem))) return 0;
    n *= sm_count();
  } else {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(cluster);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    memset(&attr, 0, sizeof(attr));
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (!ZG_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg))) return 0;
  }
  if (n < 1) n = 1;
  last.store(key | (uint32_t)n, std::memory_order_relaxed);
  return (unsigned)n;
}

}  // namespace ra
}  // namespace zg
