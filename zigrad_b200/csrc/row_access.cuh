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

__device__ __forceinline__ void copy_word(void* smem_dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem_dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

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
// The sum of N words' exponentials
template <typename T, int N>
__device__ __forceinline__ float words_sum(const uint4 (&v)[N], float m, float c) {
  const Pair shift = minus(m), cc = pair_of(c, c);
  Pair sum[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float x[kPerWord<T>];
    unpack(v[j], x, T());
    sum[j] = shifted_exp(x[0], x[1], shift, cc);
#pragma unroll
    for (int i = 2; i < kPerWord<T>; i += 2) sum[j] = sum[j] + shifted_exp(x[i], x[i + 1], shift, cc);
  }
#pragma unroll
  for (int n = 1; n < N; n *= 2)
#pragma unroll
    for (int j = 0; j + n < N; j += 2 * n) sum[j] = sum[j] + sum[j + n];
  float s0, s1;
  split(sum[0], s0, s1);
  return s0 + s1;
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

// A whole number that orders as the value does: NaN above all, -0 and +0 alike, 0 below -infinity
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  if (x != x) return 0xffffffffu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

}  // namespace ra
}  // namespace zg
