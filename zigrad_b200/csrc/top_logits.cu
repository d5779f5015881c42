// The k largest logits of each row with their indices, and the row's log normaliser (include/zg_b200.h: zg_top_logits): what a
// teacher hands on (distill.cu), and the candidates that a sampler looks at.  The reference has max_along
// (src/device/host_device.zig:853-874) and no more of this kind.
//
// A row is read once.  Each thread keeps the largest value of each of its kGroups shares of the row; each warp then looks, by
// bisection over the values' order, for a bound that a few more than its part of the k group maxima reach.  Every group maximum is an
// element, so from W warps whose bounds n elements each reach, the j-th largest bound is reached by at least j n >= k
// elements: no element below it is among the k largest.  Only the groups whose maximum reaches it, about k of thousands, are
// read again (they are in L2), and what reaches the bound, k to 2k elements as a rule, is sorted.
// Where more elements than the buffer holds reach it (rows of equal values, rows with fewer finite values than k) one
// CTA finds the k-th largest value digit by digit and takes its equals by index.
#include "row_access.cuh"

namespace zg {

using namespace ra;

constexpr int kTThreads = 256;
constexpr unsigned kTMost = 1024;        // largest k
constexpr int kTGroups = 4;              // maxima per thread
constexpr unsigned kTBuffer = 4096;      // candidates of a row taken by a CTA
constexpr unsigned kTWarpBuffer = 512;   // of a row taken by a warp, all of it

struct TopArgs {
  const void* logits;
  size_t rows, ld;
  unsigned C, k;
  void* values;    // [rows, k], the logits' type
  len_t* indices;  // [rows, k]
  float* lse;      // [rows] or nullptr
  float c;         // log2(e) / temperature
  double inv_t;
};

__device__ __forceinline__ uint64_t entry_of(uint32_t key, unsigned index) { return (uint64_t)key << 32 | (0xffffffffu - index); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The largest bound with at least n of the warp's keys at or above it, or one that few more reach.  1 where fewer than n are
// no 0 (nothing), which everything reaches.
template <int K>
__device__ __forceinline__ uint32_t warp_bound(const uint32_t (&key)[K], unsigned n) {
  auto reach = [&](uint32_t b) {
    unsigned cnt = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) cnt += key[i] >= b;
    return __reduce_add_sync(0xffffffffu, cnt);
  };
  uint32_t most = key[0], least = key[0];
#pragma unroll
  for (int i = 1; i < K; ++i) { most = max(most, key[i]); least = min(least, key[i]); }
  uint32_t hi = __reduce_max_sync(0xffffffffu, most), lo = max(1u, __reduce_min_sync(0xffffffffu, least));
  if (reach(lo) < n) return 1;
  const unsigned enough = n + n / 4;
  // lo is reached by n or more, hi + 1 by none
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    const unsigned cnt = reach(mid);
    if (cnt >= n) {
      lo = mid;
      if (cnt <= enough) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// G threads sort n <= cap entries (cap a power of two; the rest is filled with zeros), largest first
template <int G, typename Sync>
__device__ __forceinline__ void sort_entries(uint64_t* buf, unsigned n, unsigned tid, Sync sync) {
  unsigned size = 32;
  while (size < n) size *= 2;
  for (unsigned i = n + tid; i < size; i += G) buf[i] = 0;
  sync();
  for (unsigned width = 2; width <= size; width *= 2)
    for (unsigned step = width / 2; step > 0; step /= 2) {
      for (unsigned i = tid; i < size / 2; i += G) {
        const unsigned lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const uint64_t a = buf[lo], b = buf[hi];
        if ((a < b) == ((lo & width) == 0)) { buf[lo] = b; buf[hi] = a; }
      }
      sync();
    }
}

template <typename T, int G, bool LSE>
__global__ void __launch_bounds__(kTThreads) top_logits_kernel(const TopArgs a) {
  constexpr int P = kPerWord<T>;
  constexpr int kWarps = G / 32;
  constexpr unsigned kCap = G == 32 ? kTWarpBuffer : kTBuffer;
  extern __shared__ __align__(16) unsigned char smem[];
  struct Part { float m, s; uint32_t bound; uint32_t pad; };
  constexpr size_t kOwn = kCap * sizeof(uint64_t) + (G == 32 ? 16 : 8 * 8 * sizeof(Part) + 1024 + 16);
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned ctas = G == 32 ? 1 : cluster.num_blocks(), rank = G == 32 ? 0 : cluster.block_rank();
  const unsigned tid = threadIdx.x % G, lane = threadIdx.x & 31, warp = tid >> 5;
  unsigned char* mine = smem + (threadIdx.x / G) * kOwn;
  uint64_t* buf = reinterpret_cast<uint64_t*>(mine);
  unsigned* count = reinterpret_cast<unsigned*>(buf + kCap);
  Part* parts = reinterpret_cast<Part*>(count + 4);
  unsigned* digits = reinterpret_cast<unsigned*>(parts + 64);  // 256
  auto sync = [] { if (G == 32) __syncwarp(); else __syncthreads(); };
  auto sync_all = [&] { if (G == 32) __syncwarp(); else if (ctas == 1) __syncthreads(); else cluster.sync(); };
  if (G > 32 && ctas > 1) cluster.barrier_arrive();
  pdl_sync();
  if (G > 32 && ctas > 1) cluster.barrier_wait();
  const size_t first = G == 32 ? (size_t)blockIdx.x * (kTThreads / 32) + threadIdx.x / 32 : blockIdx.x / ctas;
  const size_t stride = G == 32 ? (size_t)gridDim.x * (kTThreads / 32) : gridDim.x / ctas;
  for (size_t r = first; r < a.rows; r += stride) {
    const Row<T> row(const_cast<T*>(static_cast<const T*>(a.logits)) + r * a.ld, a.C);
    const unsigned words = row.words(), begin = rank * G + tid, step = ctas * G;
    if (tid == 0) *count = 0;

    // ---- one pass: largest values of the groups, sum of the exponentials
    float top[kTGroups];
#pragma unroll
    for (int g = 0; g < kTGroups; ++g) top[g] = -INFINITY;
    float m = -INFINITY, sum = 0.f;
    for (unsigned w = begin; w < words; w += kTGroups * step) {
      uint4 v[kTGroups];
#pragma unroll
      for (int g = 0; g < kTGroups; ++g) v[g] = w + g * step < words ? row.load(w + g * step) : nothing<T>();
#pragma unroll
      for (int g = 0; g < kTGroups; ++g) {
        float x[P];
        unpack(v[g], x, T());
        float t = x[0];
#pragma unroll
        for (int i = 1; i < P; ++i) t = max_nan(t, x[i]);
        top[g] = max_nan(top[g], t);
        if (LSE) {
          const float t2 = fmaxf(m, t);
          sum *= shifted_exp(m, t2, a.c);
          m = t2;
#pragma unroll
          for (int i = 0; i < P; ++i) sum += shifted_exp(x[i], m, a.c);
        }
      }
    }
    // ---- a bound that at least k elements reach
    uint32_t key[kTGroups];
#pragma unroll
    for (int g = 0; g < kTGroups; ++g) key[g] = begin + g * step < words ? key_of(top[g]) : 0u;
    const unsigned warps = ctas * kWarps;
    const unsigned need = min(a.k, (2 * a.k + warps - 1) / warps);   // of each warp
    uint32_t bound = warp_bound<kTGroups>(key, need);
    auto join = [&](float m2, float s2) {
      const float t = fmaxf(m, m2);
      sum = sum * shifted_exp(m, t, a.c) + s2 * shifted_exp(m2, t, a.c);
      m = t;
    };
    if (LSE)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) join(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, sum, o));
    if (G > 32) {
      const Part p{m, sum, bound, 0};
      if (ctas == 1) {
        if (lane == 0) parts[warp] = p;
      } else if (lane < ctas) {
        cluster.map_shared_rank(parts, lane)[rank * kWarps + warp] = p;
      }
      sync_all();
      // the j-th largest of the warps' bounds, where j `need` >= k; their sums
      const unsigned j = (a.k + need - 1) / need;
      m = -INFINITY; sum = 0.f;
      uint32_t best = 0;
      for (unsigned i = lane; i < warps; i += 32) {
        const Part q = parts[i];
        if (LSE) join(q.m, q.s);
        unsigned reach = 0;
        for (unsigned o = 0; o < warps; ++o) reach += parts[o].bound >= q.bound;
        if (reach >= j) best = max(best, q.bound);
      }
      bound = __reduce_max_sync(0xffffffffu, best);
      if (LSE)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) join(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, sum, o));
    }
    if (LSE && rank == 0 && tid == 0) a.lse[r] = (float)((double)m * a.inv_t + log((double)sum));

    // ---- what reaches the bound, into the first CTA's buffer
    uint64_t* to = rank == 0 ? buf : cluster.map_shared_rank(buf, 0);
    unsigned* tally = rank == 0 ? count : cluster.map_shared_rank(count, 0);
    auto collect = [&](unsigned w, uint32_t least) {
      const unsigned p0 = w * P;
      float x[P];
      unpack(row.load(w), x, T());
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const unsigned p = p0 + i;
        const uint32_t key = key_of(x[i]);
        if (key >= least && p >= row.lead && p < row.end) {
          const unsigned at = atomicAdd(tally, 1u);
          if (at < kCap) to[at] = entry_of(key, p - row.lead);
        }
      }
    };
    if (G == 32) sync();  // the count is cleared
#pragma unroll
    for (int g = 0; g < kTGroups; ++g)
      if (key[g] >= bound)
        for (unsigned w = begin + g * step; w < words; w += kTGroups * step) collect(w, bound);
    sync_all();
    if (rank == 0) {
      unsigned n = *count;
      if (G > 32 && n > kCap) {
        // ---- the k-th largest key digit by digit; above it everything, of its equals the first ones
        uint32_t prefix = 0;
        unsigned left = a.k;   // how many of those that agree with the prefix are wanted
        for (int shift = 24; shift >= 0; shift -= 8) {
          for (unsigned i = tid; i < 256; i += G) digits[i] = 0;
          __syncthreads();
          for (unsigned w = tid; w < words; w += G) {
            float x[P];
            unpack(row.load(w), x, T());
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const unsigned p = w * P + i;
              const uint32_t key = key_of(x[i]);
              if (p >= row.lead && p < row.end && (shift == 24 || (key ^ prefix) >> (shift + 8) == 0)) atomicAdd(digits + (key >> shift & 255), 1u);
            }
          }
          __syncthreads();
          unsigned d = 255;
          while (d > 0 && digits[d] < left) left -= digits[d--];
          prefix |= d << shift;
          __syncthreads();
        }
        if (tid == 0) *count = 0;
        __syncthreads();
        for (unsigned w = tid; w < words; w += G)
          if (prefix != 0xffffffffu) collect(w, prefix + 1);
        __syncthreads();
        n = *count;              // k - left
        unsigned have = 0;       // equals so far, in the order of their indices
        for (unsigned w0 = 0; w0 < words && have < left; w0 += G) {
          const unsigned w = w0 + tid;
          unsigned equal = 0;
          if (w < words) {
            float x[P];
            unpack(row.load(w), x, T());
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const unsigned p = w * P + i;
              if (p >= row.lead && p < row.end && key_of(x[i]) == prefix) equal |= 1u << i;
            }
          }
          const unsigned mineq = __popc(equal);
          unsigned before = mineq;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const unsigned up = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= (unsigned)o) before += up;
          }
          if (lane == 31) digits[warp] = before;
          __syncthreads();
          unsigned at = have + before - mineq, all = 0;
          for (unsigned i = 0; i < (unsigned)kWarps; ++i) {
            if (i < warp) at += digits[i];
            all += digits[i];
          }
          while (equal && at < left) {
            const unsigned i = __ffs(equal) - 1;
            equal &= equal - 1;
            buf[n + at++] = entry_of(prefix, w * P + i - row.lead);
          }
          have += all;
          __syncthreads();
        }
        n = a.k;
      }
      sort_entries<G>(buf, n, tid, sync);
      for (unsigned i = tid; i < a.k; i += G) {
        const uint64_t e = buf[i];
        static_cast<T*>(a.values)[r * a.k + i] = from_float<T>(value_of((uint32_t)(e >> 32)));
        a.indices[r * a.k + i] = 0xffffffffu - (uint32_t)e;
      }
    }
    sync_all();  // the buffers are free
  }
}

template <typename T, int G, bool LSE>
static void launch_top(cudaStream_t s, const TopArgs& a, unsigned cluster) {
  static SharedMemoryLimit limit;
  const size_t smem = G == 32 ? (kTThreads / 32) * (kTWarpBuffer * 8 + 16) : kTBuffer * 8 + 16 + 64 * 16 + 1024;
  if (smem > 48 * 1024 && !limit.raise(top_logits_kernel<T, G, LSE>, smem)) return;
  const size_t groups = G == 32 ? (a.rows + kTThreads / 32 - 1) / (kTThreads / 32) : a.rows;
  const size_t most = (size_t)1 << 20;
  launch_pdl_cluster(top_logits_kernel<T, G, LSE>, dim3((unsigned)(groups < most ? groups : most) * cluster), dim3(kTThreads), smem, s, cluster, a);
}

template <typename T>
static void launch_top_rows(cudaStream_t s, const TopArgs& a) {
  if (a.lse) launch_top<T, kTThreads, true>(s, a, 1);
  else launch_top<T, kTThreads, false>(s, a, 1);
}

}  // namespace zg

using namespace zg;

extern "C" void zg_top_logits(dtype id, StreamWrapper w, const void* logits, len_t rows, len_t C, len_t ld, len_t k, double temperature,
                              void* values_out, len_t* indices_out, void* lse_out) {
  const char* me = "zg_top_logits";
  if (id != SINGLE && id != BF16) { set_error(kUnsupported, "%s: logits are SINGLE or BF16", me); return; }
  if (ld == 0) ld = C;
  if (C == 0 || C > (len_t)0x7fffffff || ld < C) { set_error(kBadArgument, "%s: C %lu, ld %lu", me, C, ld); return; }
  if (k == 0 || k > C || k > kTMost) { set_error(kBadArgument, "%s: k %lu of %lu classes (at most %u)", me, k, C, kTMost); return; }
  if (!(temperature > 0.0) || !(temperature <= 1e30) || !(1.0 / temperature <= 1e30)) { set_error(kBadArgument, "%s: temperature %g", me, temperature); return; }
  if (rows == 0) return;
  if (!logits || !values_out || !indices_out) { set_error(kBadArgument, "%s: a required operand is NULL", me); return; }
  const size_t size = id == BF16 ? 2 : 4;
  const auto off = [](const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
  if (off(logits, size) || off(values_out, size) || off(indices_out, 8) || off(lse_out, 4)) {
    set_error(kBadArgument, "%s: an operand is not aligned to its elements", me);
    return;
  }
  TopArgs a;
  a.logits = logits; a.rows = rows; a.ld = ld; a.C = (unsigned)C; a.k = (unsigned)k; a.values = values_out; a.indices = indices_out;
  a.lse = (float*)lse_out; a.c = (float)(1.4426950408889634 / temperature); a.inv_t = 1.0 / temperature;
  if (id == SINGLE) launch_top_rows<float>(as_stream(w), a);
  else launch_top_rows<__nv_bfloat16>(as_stream(w), a);
}
