// The k largest logits of each row with their indices, and the row's log normaliser (include/zg_b200.h: zg_top_logits): what a
// teacher hands on (distill.cu), and the candidates that a sampler looks at.  The reference has max_along
// (src/device/host_device.zig:853-874) and no more of this kind.
//
// A row is read once.  Each thread keeps the largest value of each of its kTGroups shares of the row; each warp then looks, by
// bisection over the values' order, for a bound that a few more than its part of the k group maxima reach.  Every group maximum is an
// element, so from W warps whose bounds n elements each reach, the j-th largest bound is reached by at least j n >= k
// elements: no element below it is among the k largest.  Only the groups whose maximum reaches it, about k of two thousand, are
// read again (they are in L2), and what reaches the bound, k to 2k elements as a rule, is sorted.
// Where more elements than the buffer holds reach it the k-th largest value is found digit by digit and its equals are taken by
// index, which reads the row up to six more times.  So it goes with rows of equal values, with rows of fewer finite values than k, and with
// ordinary rows where k comes near the number of shares (256 of a warp, 1024 or 2048 of a CTA, fewer where a row has fewer words):
// the bound is then one of the smallest maxima, or there is none.  8192 x 4096 bf16: k 64 61 us, k 128 119, k 192 348.
//
// 4096 x 131072 bf16, 64 of them: 1.07 GB in 250 us with a cold L2, 197 with k = 1.  The pass itself runs close to the memory's rate;
// what the bound, the second look and the ranking take grows with k (1024 x 131072 fp32, 256 of them: 192 us).
#include "row_access.cuh"

namespace zg {

using namespace ra;

constexpr unsigned kTMost = 1024;        // largest k
constexpr int kTGroups = 8;              // maxima per thread
// Candidates of a row taken by a CTA: a power of two, at least kTMost.  4096 of them save long lists the digits (1000 x 131072 bf16, 1024 of
// them, 479 -> 279 us) and cost those of shorter rows, and every other call, CTAs to an SM (1000 x 16384 203 -> 272; 64 of them 24.6 -> 28.7).
constexpr unsigned kTBuffer = 2048;
constexpr unsigned kTWarpBuffer = 512;   // of a row taken by a warp
constexpr unsigned kTWarpMost = 256;     // largest k there
constexpr unsigned kTWarpWords = 512;    // longest row there

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

// The largest bound with at least n of the warp's keys at or above it, or one that a few more reach; 1 where fewer than n are
// no 0 (nothing), which everything reaches.  The low `shift` bits of a key say nothing (those that bf16 does not have).
template <int K>
__device__ __forceinline__ uint32_t warp_bound(const uint32_t (&key)[K], unsigned n, unsigned shift) {
  auto reach = [&](uint32_t b) -> unsigned {
    if (K == 1) return __popc(__ballot_sync(0xffffffffu, key[0] >= b));
    unsigned cnt = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) cnt += key[i] >= b;
    return __reduce_add_sync(0xffffffffu, cnt);
  };
  uint32_t most = key[0], least = key[0];
#pragma unroll
  for (int i = 1; i < K; ++i) { most = max(most, key[i]); least = min(least, key[i]); }
  const uint32_t unit = 1u << shift;
  uint32_t hi = __reduce_max_sync(0xffffffffu, most) >> shift, lo = max(unit, __reduce_min_sync(0xffffffffu, least)) >> shift;
  if (reach(lo << shift) < n) return 1;
  const unsigned enough = n + n / 8;
  // lo is reached by n or more, hi + 1 by none
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    const unsigned cnt = reach(mid << shift);
    if (cnt >= n) {
      lo = mid;
      if (cnt <= enough) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo << shift;
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

// What the warps of a row know of it
struct TopPart {
  float m, s;      // largest value, sum of 2^((x - m) c)
  uint32_t bound;  // `need` elements reach it
  uint32_t pad;
};
// Shared memory of G threads: candidates, their number and that of the groups, what CTAs send one another, the groups (or digits)
__host__ __device__ constexpr unsigned top_bytes(int G) {
  return G == 32 ? kTWarpBuffer * 8 + 16 + 1024 : kTBuffer * 8 + 16 + 64 * (unsigned)sizeof(TopPart) + (unsigned)G * kTGroups * 2;
}

template <typename T, int G, int THREADS, bool LSE>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) top_logits_kernel(const TopArgs a) {
  constexpr int P = kPerWord<T>;
  constexpr int kWarps = G / 32;
  constexpr unsigned kCap = G == 32 ? kTWarpBuffer : kTBuffer;
  extern __shared__ __align__(16) unsigned char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned ctas = G == 32 ? 1 : cluster.num_blocks(), rank = G == 32 ? 0 : cluster.block_rank();
  const unsigned tid = threadIdx.x % G, lane = threadIdx.x & 31, warp = tid >> 5;
  uint64_t* const buf = reinterpret_cast<uint64_t*>(smem + (threadIdx.x / G) * top_bytes(G));
  unsigned* const count = reinterpret_cast<unsigned*>(buf + kCap);       // of the candidates, of the groups
  TopPart* const parts = reinterpret_cast<TopPart*>(count + 4);          // G > 32: [ctas * kWarps], 64 at most
  uint16_t* const groups = reinterpret_cast<uint16_t*>(parts + (G == 32 ? 0 : 64));
  unsigned* const digits = reinterpret_cast<unsigned*>(groups);          // 256
  auto sync = [] { if (G == 32) __syncwarp(); else __syncthreads(); };
  auto sync_all = [&] { if (G == 32) __syncwarp(); else if (ctas == 1) __syncthreads(); else cluster.sync(); };
  if (G > 32 && ctas > 1) cluster.barrier_arrive();
  pdl_sync();
  const size_t r = G == 32 ? (size_t)blockIdx.x * (THREADS / 32) + threadIdx.x / 32 : blockIdx.x / ctas;
  if (G == 32 && r >= a.rows) return;
  const Row<T> row(const_cast<T*>(static_cast<const T*>(a.logits)) + r * a.ld, a.C);
  const unsigned words = row.words(), begin = rank * G + tid, step = ctas * G;
  const unsigned from = row.lead ? 1 : 0, inner = row.end / P > from ? row.end / P - from : 0;  // whole words, and from which on
  auto word = [&](unsigned w) { return w - from < inner ? __ldcg(row.word(w)) : row.load_part(w); };
  if (tid < 2) count[tid] = 0;

  // ---- one pass: largest values of the groups, sum of the exponentials.  Word begin + i step belongs to group i mod kTGroups.
  float top[kTGroups];
#pragma unroll
  for (int g = 0; g < kTGroups; ++g) top[g] = -INFINITY;
  float m = -INFINITY, sum = 0.f;
  auto take = [&](const uint4 (&v)[4], float* top) {
    float t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      t[j] = word_max_nan(v[j], T());
      top[j] = max_nan(top[j], t[j]);
    }
    if (LSE) {
      const float m2 = fmaxf(m, fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])));
      sum = sum * shifted_exp(m, m2, a.c) + words_sum<T>(v, m2, a.c);
      m = m2;
    }
  };
  for (unsigned w = begin; w < words; w += kTGroups * step) {
    if (w >= from && w + (kTGroups - 1) * step < from + inner) {
      uint4 v[2][4];
#pragma unroll
      for (int j = 0; j < kTGroups; ++j) v[j / 4][j % 4] = __ldcg(row.word(w + j * step));
      take(v[0], top);
      take(v[1], top + 4);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = w + (4 * h + j) * step < words ? word(w + (4 * h + j) * step) : nothing<T>();
        if (w + 4 * h * step < words) take(v, top + 4 * h);
      }
    }
  }

  // ---- a bound that at least k elements reach
  uint32_t key[kTGroups];
#pragma unroll
  for (int g = 0; g < kTGroups; ++g) key[g] = begin + g * step < words ? key_of(top[g]) : 0u;
  const unsigned warps = ctas * kWarps;
  const unsigned need = (a.k + warps - 1) / warps;   // of each warp
  constexpr unsigned kShift = sizeof(T) == 2 ? 16 : 0;
  uint32_t bound;
  if (need <= 8) {  // of a warp's 32 lanes' maxima 8 bound 9 elements as a rule; of 256 maxima, a few times the work, 8
    uint32_t most[1] = {key[0]};
#pragma unroll
    for (int g = 1; g < kTGroups; ++g) most[0] = max(most[0], key[g]);
    bound = warp_bound<1>(most, need, kShift);
  } else {
    bound = warp_bound<kTGroups>(key, need, kShift);
  }
  auto join = [&](float m2, float s2) {
    const float t = fmaxf(m, m2);
    sum = sum * shifted_exp(m, t, a.c) + s2 * shifted_exp(m2, t, a.c);
    m = t;
  };
  auto join_lanes = [&] {
    const float t = value_of(__reduce_max_sync(0xffffffffu, key_of(m)));  // no NaN: fmaxf keeps the others
    sum = warp_sum(sum * shifted_exp(m, t, a.c));
    m = t;
  };
  if (LSE) join_lanes();
  if (G > 32) {
    const TopPart p{m, sum, bound, 0};
    if (ctas == 1) {
      if (lane == 0) parts[warp] = p;
    } else {
      cluster.barrier_wait();  // every CTA of the cluster is there
      if (lane < ctas) cluster.map_shared_rank(parts, lane)[rank * kWarps + warp] = p;
    }
    sync_all();
    // the j-th largest of the warps' bounds, where j `need` >= k; their sums
    const unsigned j = (a.k + need - 1) / need;
    m = -INFINITY; sum = 0.f;
    uint32_t best = 0;
    for (unsigned i = lane; i < warps; i += 32) {
      const TopPart q = parts[i];
      if (LSE && rank == 0 && warp == 0) join(q.m, q.s);
      unsigned reach = 0;
      for (unsigned o = 0; o < warps; ++o) reach += parts[o].bound >= q.bound;
      if (reach >= j) best = max(best, q.bound);
    }
    bound = __reduce_max_sync(0xffffffffu, best);
    if (LSE && rank == 0 && warp == 0) join_lanes();
  }
  if (LSE && rank == 0 && tid == 0) a.lse[r] = (float)((double)m * a.inv_t + log((double)sum));

  // ---- the groups that reach it, and of their words what does, into the first CTA's buffer
  uint64_t* const to = rank == 0 ? buf : cluster.map_shared_rank(buf, 0);
  unsigned* const tally = rank == 0 ? count : cluster.map_shared_rank(count, 0);
  auto collect = [&](unsigned w, uint32_t least) {
    float x[P];
    unpack(word(w), x, T());
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const unsigned p = w * P + i;
      const uint32_t key = key_of(x[i]);
      if (key >= least && p >= row.lead && p < row.end) {
        const unsigned at = atomicAdd(tally, 1u);
        if (at < kCap) to[at] = entry_of(key, p - row.lead);
      }
    }
  };
  const unsigned per_group = (words + kTGroups * step - 1) / (kTGroups * step);
  if (G == 32) {  // a lane's own
    __syncwarp();
#pragma unroll
    for (int g = 0; g < kTGroups; ++g)
      if (key[g] >= bound)
        for (unsigned w = begin + g * step; w < words; w += kTGroups * step) collect(w, bound);
    __syncwarp();
  } else {
#pragma unroll
    for (int g = 0; g < kTGroups; ++g)
      if (key[g] >= bound) groups[atomicAdd(count + 1, 1u)] = (uint16_t)(tid * kTGroups + g);
    __syncthreads();
    const unsigned n = count[1] * per_group;
    for (unsigned i = tid; i < n; i += G) {
      const unsigned id = groups[i / per_group], w = rank * G + id / kTGroups + (i % per_group * kTGroups + id % kTGroups) * step;
      if (w < words) collect(w, bound);
    }
    sync_all();
  }
  if (rank != 0) return;
  unsigned n = *count;
  if (n > kCap) {
    // ---- the k-th largest key digit by digit; above it everything, of its equals the first ones
    uint32_t prefix = 0;
    unsigned left = a.k;   // how many of those that agree with the prefix are wanted
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (unsigned i = tid; i < 256; i += G) digits[i] = 0;
      sync();
      for (unsigned w = tid; w < words; w += G) {
        float x[P];
        unpack(word(w), x, T());
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const unsigned p = w * P + i;
          const uint32_t key = key_of(x[i]);
          if (p >= row.lead && p < row.end && (shift == 24 || (key ^ prefix) >> (shift + 8) == 0)) atomicAdd(digits + (key >> shift & 255), 1u);
        }
      }
      sync();
      unsigned d = 255;
      while (d > 0 && digits[d] < left) left -= digits[d--];
      prefix |= d << shift;
      sync();
    }
    if (tid == 0) *count = 0;
    sync();
    if (prefix != 0xffffffffu)
      for (unsigned w = tid; w < words; w += G) collect(w, prefix + 1);
    sync();
    n = *count;              // k - left
    unsigned have = 0;       // equals so far, in the order of their indices
    for (unsigned w0 = 0; w0 < words && have < left; w0 += G) {
      const unsigned w = w0 + tid;
      unsigned equal = 0;
      if (w < words) {
        float x[P];
        unpack(word(w), x, T());
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const unsigned p = w * P + i;
          if (p >= row.lead && p < row.end && key_of(x[i]) == prefix) equal |= 1u << i;
        }
      }
      const unsigned some = __popc(equal);
      unsigned before = some;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= (unsigned)o) before += up;
      }
      if (lane == 31) digits[warp] = before;
      sync();
      unsigned at = have + before - some, all = 0;
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
      sync();
    }
    n = a.k;
  }
  auto put = [&](unsigned i, uint64_t e) {
    static_cast<T*>(a.values)[r * a.k + i] = from_float<T>(value_of((uint32_t)(e >> 32)));
    a.indices[r * a.k + i] = 0xffffffffu - (uint32_t)e;
  };
  if (n <= 512) {  // an entry's place is the number of larger ones: no barriers, one pass over the others for each
    for (unsigned i = tid; i < n; i += G) {
      const uint64_t e = buf[i];
      unsigned larger = 0;
#pragma unroll 4
      for (unsigned o = 0; o < n; ++o) larger += buf[o] > e;
      if (larger < a.k) put(larger, e);
    }
  } else {
    sort_entries<G>(buf, n, tid, sync);
    for (unsigned i = tid; i < a.k; i += G) put(i, buf[i]);
  }
}

template <typename T, int G, int THREADS>
static void launch_top(cudaStream_t s, const TopArgs& a, unsigned cluster) {
  const size_t smem = (size_t)top_bytes(G) * (THREADS / G);  // less than 48 KB
  const unsigned grid = (unsigned)(G == 32 ? (a.rows + THREADS / 32 - 1) / (THREADS / 32) : a.rows) * cluster;
  if (a.lse) launch_pdl_cluster(top_logits_kernel<T, G, THREADS, true>, dim3(grid), dim3(THREADS), smem, s, cluster, a);
  else launch_pdl_cluster(top_logits_kernel<T, G, THREADS, false>, dim3(grid), dim3(THREADS), smem, s, cluster, a);
}

template <typename T>
static void launch_top_rows(cudaStream_t s, const TopArgs& a) {
  const size_t words = most_words<T>(a.logits, a.C, a.ld);
  // A warp a row, or 128 threads.  8192 rows: 4096 bf16 k 32 53 and 59 us, k 128 119 and 133, k 192 348 and 221, k 256 375 and 371;
  // 1000 fp32 k 10 29 and 47, k 128 90 and 135, k 256 219 and 346.  That is for rows that fill the SMs; the rule does not look at
  // their number, and of few rows 128 threads each would be faster: 512 x 4096 bf16 k 32 21 and 12 us, 8 x 1000 fp32 k 64 16 and 14, k 256 66 and 25
  if (words <= kTWarpWords && a.k <= kTWarpMost) return launch_top<T, 32, 256>(s, a, 1);
  // several CTAs to a row only while SMs would be idle: what each finds out is as much work as before
  unsigned cluster = 1;
  while (cluster < 8 && a.rows * cluster * 2 <= (size_t)sm_count() && words > 128 * cluster) cluster *= 2;
  // what 256 threads find out about a row takes twice as long as what 128 do, which pays from 64 KB on (8192 x 8192 bf16 111 and
  // 68 us, 4096 x 32768 88 and 82, 4096 x 131072 250 and 275)
  if (words <= 4096 * cluster) return launch_top<T, 128, 128>(s, a, cluster);
  launch_top<T, 256, 256>(s, a, cluster);
}

}  // namespace zg

using namespace zg;

extern "C" void zg_top_logits(dtype id, StreamWrapper w, const void* logits, len_t rows, len_t C, len_t ld, len_t k, double temperature,
                              void* values_out, len_t* indices_out, void* lse_out) {
  const char* me = "zg_top_logits";
  if (id != SINGLE && id != BF16) { set_error(kUnsupported, "%s: logits are SINGLE or BF16", me); return; }
  if (ld == 0) ld = C;
  if (C == 0 || C > (len_t)0x7fffffff || ld < C) { set_error(kBadArgument, "%s: C %lu, ld %lu", me, C, ld); return; }
  if (rows > (len_t)0x0fffffff) { set_error(kBadArgument, "%s: rows %lu", me, rows); return; }
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
