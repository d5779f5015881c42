// Distillation from a teacher's list of top logits: the divergence of the student's softmax from the teacher's and its
// gradient in one pass over the student's logits (include/zg_b200.h: zg_distill_ce).  It stands beside the softmax
// cross-entropy of loss.cu (src/nn/loss.zig:130-215), whose target is one class or a dense row.
//
// With z the student's logits over the temperature, S the list's mass and r = 1 - S the teacher's mass outside it:
//   row  = sum_i q_i (log q_i - log p_i) + r (log r - log p_r),   p_r = sum of p outside the list
//   dz_j = (S + r) p_j - q_j                 in the list
//        = (S + r) p_j - r p_j / p_r         outside it
// Where student and teacher nearly agree the row is a small difference of large logarithms, and where the list has nearly all
// mass p_r as a difference of sums would have no digits left.  So the values outside the list are summed apart from those in
// it (a bit per position says which is which), and log p_r = -log1p(listed / rest) and the coefficient (S + r) p_r - r come
// from the two sums in 64 bits.  An error e of the sum outside, made of fp32 terms, then changes the row by e (S - (1 - p_r)) only; one
// of the listed sum would change it by e (1 - p_r), so the list, k terms of C, is summed in 64 bits.
#include "row_access.cuh"

namespace zg {

using namespace ra;

constexpr int kDThreads = 256;
constexpr unsigned kDMaxList = 1024;

struct DistillArgs {
  const void* logits;     // [rows, ld]
  void* dlogits;          // [rows, ld] or nullptr; may be `logits`
  size_t rows, ld;
  unsigned C, k;
  const len_t* t_index;   // [rows, k]; an index >= C is no entry
  const void* t_logits;   // [rows, k]
  int t_bf16;
  const float* t_lse;     // [rows] or nullptr: the list's own
  const float* weight;    // [rows] or nullptr
  double inv_t;           // 1 / temperature
  float c;                // log2(e) / temperature
  double loss_div;
  float* loss;
  float* row_loss;        // [rows]
  int accumulate;
  int same_lead;          // rows of logits and dlogits start equally far behind a 16-byte boundary
  unsigned segments;      // slices of a row per CTA
  int fold;               // this grid is one CTA or cluster: it writes the loss itself
};

// What the warps of a group know of a row, put together into what all of them need.  The sums over the list are to a common
// maximum, so they only add up.
struct DistillPart {
  float m, s;       // largest value outside the list (everywhere where there is no rest), sum of 2^((x - m) c)
  double s_listed;  // sum of exp((x - m_listed) / T), each class once
  double mass;      // sum of w: q, or exp((u - u_max) / T) where the list's own sum is the normaliser
  double cross;     // sum of w (log w - (z - m_listed) / T)
};

__device__ __forceinline__ void join(float& m, float& s, float m2, float s2, float c) {
  const float top = fmaxf(m, m2);
  s = s * shifted_exp(m, top, c) + s2 * shifted_exp(m2, top, c);
  m = top;
}
__device__ __forceinline__ void join_lanes(DistillPart& p, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) join(p.m, p.s, __shfl_xor_sync(0xffffffffu, p.m, o), __shfl_xor_sync(0xffffffffu, p.s, o), c);
  p.s_listed = warp_sum(p.s_listed);
  p.mass = warp_sum(p.mass);
  p.cross = warp_sum(p.cross);
}

// G threads take a row together: a warp (short rows, eight to a CTA) or a CTA, of which a cluster shares a row.  Thread t of
// CTA r holds the words r G NV + i G + t, i < NV, in registers from the sums to the gradient, so that a row is read once;
// rows longer than that (MULTI) are walked in slices, twice.
template <typename T, int NV, int G, bool MULTI>
__global__ void __launch_bounds__(kDThreads) distill_kernel(const DistillArgs a) {
  constexpr int P = kPerWord<T>;
  constexpr unsigned kSlice = (unsigned)G * NV;              // words
  constexpr int kWarps = G / 32;
  constexpr int kOwn = (G == 32 ? 128 : kDMaxList) / G;      // list entries per thread
  extern __shared__ __align__(16) unsigned char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned ctas = G == 32 ? 1 : cluster.num_blocks(), rank = G == 32 ? 0 : cluster.block_rank();
  const unsigned tid = threadIdx.x % G, lane = threadIdx.x & 31, warp = tid >> 5;
  const size_t own_bytes = 2 * ctas * kWarps * sizeof(DistillPart) + kSlice + 12 * (size_t)((a.k + 3) & ~3u) + 16;
  unsigned char* mine = smem + (threadIdx.x / G) * own_bytes;
  DistillPart* parts = reinterpret_cast<DistillPart*>(mine);                       // [2][ctas * kWarps]
  uint32_t* bits = reinterpret_cast<uint32_t*>(parts + 2 * ctas * kWarps);         // a byte per word of the slice
  uint32_t* e_index = bits + kSlice / 4;                                           // this CTA's entries; ~0: not one of them
  float* e_q = reinterpret_cast<float*>(e_index + ((a.k + 3) & ~3u));
  float* e_z = e_q + ((a.k + 3) & ~3u);
  uint32_t* most = reinterpret_cast<uint32_t*>(e_z + ((a.k + 3) & ~3u));           // keys of the list's largest student's and teacher's logit
  auto sync = [] { if (G == 32) __syncwarp(); else __syncthreads(); };
  auto sync_any = [](bool v) -> bool { return G == 32 ? __any_sync(0xffffffffu, v) : __syncthreads_or(v); };
  const bool tail = a.t_lse != nullptr;
  const float c = a.c;
  unsigned parity = 0;
  if (G > 32 && ctas > 1) cluster.barrier_arrive();
  pdl_sync();
  if (G > 32 && ctas > 1) cluster.barrier_wait();  // every CTA of the cluster is there: its shared memory may be written
  const size_t first = G == 32 ? (size_t)blockIdx.x * (kDThreads / 32) + threadIdx.x / 32 : blockIdx.x / ctas;
  const size_t stride = G == 32 ? (size_t)gridDim.x * (kDThreads / 32) : gridDim.x / ctas;
  for (size_t r = first; r < a.rows; r += stride) {
    const Row<T> row(const_cast<T*>(static_cast<const T*>(a.logits)) + r * a.ld, a.C);
    T* const d_first = a.dlogits ? static_cast<T*>(a.dlogits) + r * a.ld : nullptr;
    const Row<T> d_row(d_first, a.C);
    const unsigned words = row.words();
    const float w = a.weight ? a.weight[r] : 1.f;
    // the gradient of one word of positions of `row`, into dlogits
    auto put = [&](unsigned word, float (&g)[P]) {
      if (a.same_lead) {
        if (a.accumulate && d_row.whole(word)) {
          float old[P];
          unpack(*d_row.word(word), old, T());
#pragma unroll
          for (int i = 0; i < P; ++i) g[i] += old[i];
        } else if (a.accumulate) {
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const unsigned p = word * P + i;
            if (p >= row.lead && p < row.end) g[i] += as_float(d_first[p - row.lead]);
          }
        }
        d_row.store(word, g);
      } else {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const unsigned p = word * P + i;
          if (p >= row.lead && p < row.end) {
            T* d = d_first + (p - row.lead);
            *d = from_float<T>(a.accumulate ? as_float(*d) + g[i] : g[i]);
          }
        }
      }
    };
    if (w == 0.f) {  // a row that counts nothing is not read: it may hold anything
      if (d_first && !a.accumulate)
        for (unsigned s = 0; s < (MULTI ? a.segments : 1u); ++s)
          for (int i = 0; i < NV; ++i) {
            const unsigned word = (s * ctas + rank) * kSlice + i * G + tid;
            float zero[P] = {};
            if (word < words) put(word, zero);
          }
      if (rank == 0 && tid == 0) a.row_loss[r] = 0.f;
      continue;
    }
    uint4 v[NV];
    auto load = [&](unsigned base) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const unsigned word = base + i * G + tid;
        v[i] = row.whole(word) ? __ldcs(row.word(word)) : nothing<T>();
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const unsigned word = base + i * G + tid;
        if (word < words && !row.whole(word)) v[i] = row.load_part(word);
      }
    };
    if (!MULTI) load(rank * kSlice);
    sync();  // the row before has been patched: lists and bits are free
    for (unsigned i = tid; i < kSlice / 4; i += G) bits[i] = 0;
    if (tid < 2) most[tid] = 0;
    sync();

    // ---- the teacher's list.  Its entries belong to the CTA whose slice they lie in.
    const len_t* index = a.t_index + r * a.k;
    auto u_of = [&](unsigned e) -> float {
      return a.t_bf16 ? as_float(static_cast<const __nv_bfloat16*>(a.t_logits)[r * a.k + e]) : static_cast<const float*>(a.t_logits)[r * a.k + e];
    };
    DistillPart part{-INFINITY, 0.f, 0.0, 0.0, 0.0};
    float old[kOwn];
    for (unsigned e = tid, j = 0; e < a.k; e += G, ++j) {
      const len_t at = index[e];
      unsigned keep = ~0u;
      if (at < a.C) {
        const float z = as_float(row.first[at]);
        atomicMax(most, key_of(z));
        if (!tail) atomicMax(most + 1, key_of(u_of(e)));
        if (((unsigned)at + row.lead) / P / kSlice % ctas == rank) {
          keep = (unsigned)at;
          e_z[e] = z;
          if (d_first && a.accumulate)
#pragma unroll
            for (int i = 0; i < kOwn; ++i)
              if (i == j) old[i] = as_float(d_first[at]);
        }
      }
      e_index[e] = keep;
    }

    // ---- largest value and sum of the rest, slice by slice
    bool twice = false;
    for (unsigned s = 0; s < (MULTI ? a.segments : 1u); ++s) {
      const unsigned base = (s * ctas + rank) * kSlice;
      if (MULTI) {
        load(base);
        if (s > 0) {
          sync();
          for (unsigned i = tid; i < kSlice / 4; i += G) bits[i] = 0;
        }
      }
      sync();
      bool seen = false;
      for (unsigned e = tid; e < a.k; e += G) {
        if (e_index[e] == ~0u) continue;
        const unsigned p = e_index[e] + row.lead, word = p / P - base;
        if (word >= kSlice) continue;  // of another slice (below this one: wraps around)
        const uint32_t bit = 1u << ((word & 3) * 8 + p % P);
        seen |= (atomicOr(bits + (word >> 2), bit) & bit) != 0;
      }
      twice |= sync_any(seen);
      if (tail) {
        const unsigned char* marks = reinterpret_cast<const unsigned char*>(bits);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const unsigned m = marks[i * G + tid];
          if (m) {
            float x[P];
            unpack(v[i], x, T());
#pragma unroll
            for (int j = 0; j < P; ++j)
              if (m >> j & 1) x[j] = -INFINITY;
            v[i] = pack(x, T());
          }
        }
      }
      float m = -INFINITY, sum = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float x[P];
        unpack(v[i], x, T());
#pragma unroll
        for (int j = 0; j < P; ++j) m = fmaxf(m, x[j]);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float x[P];
        unpack(v[i], x, T());
#pragma unroll
        for (int j = 0; j < P; ++j) sum += shifted_exp(x[j], m, c);
      }
      join(part.m, part.s, m, sum, c);
    }

    // ---- a class that is listed twice counts once among the student's values; its entries' masses add up
    auto owner = [&](unsigned e) -> bool {
      if (e_index[e] == ~0u) return false;
      if (twice)
        for (unsigned j = 0; j < e; ++j)
          if (e_index[j] == e_index[e]) return false;
      return true;
    };
    const float m_listed = value_of(most[0]);  // 0, no entry: a NaN that nothing below takes
    const double level = tail ? (double)a.t_lse[r] : 0.0, u_top = tail ? 0.0 : (double)value_of(most[1]);
    for (unsigned e = tid; e < a.k; e += G) {
      if (e_index[e] == ~0u) continue;
      const float z = e_z[e], u = u_of(e);
      const double arg = tail ? (double)u * a.inv_t - level : ((double)u - u_top) * a.inv_t, far = ((double)z - m_listed) * a.inv_t;
      const double w = u == -INFINITY ? 0.0 : exp(arg);
      e_q[e] = (float)w;
      part.mass += w;
      if (!(w <= 0.0)) part.cross += z == -INFINITY ? INFINITY : w * (arg - far);  // a class of mass that the student rules out: infinite
      if (z != -INFINITY && owner(e)) part.s_listed += exp(far);
    }

    // ---- over the lanes, the warps and the cluster's CTAs
    join_lanes(part, c);
    if (G > 32) {
      DistillPart* all = parts + parity * ctas * kWarps;
      if (ctas == 1) {
        if (lane == 0) all[warp] = part;
        __syncthreads();
      } else {
        if (lane < ctas) cluster.map_shared_rank(all, lane)[rank * kWarps + warp] = part;
        cluster.sync();  // also: nobody reads the parts of the row before any more
      }
      part = DistillPart{-INFINITY, 0.f, 0.0, 0.0, 0.0};
      for (unsigned i = lane; i < ctas * kWarps; i += 32) {
        const DistillPart p = all[i];
        join(part.m, part.s, p.m, p.s, c);
        part.s_listed += p.s_listed;
        part.mass += p.mass;
        part.cross += p.cross;
      }
      join_lanes(part, c);
      parity ^= 1;
    }

    const bool some = !(part.s_listed <= 0.0);   // a listed class that the student does not rule out
    const double norm = tail || part.mass == 0.0 ? 1.0 : 1.0 / part.mass, mass = part.mass * norm;
    const double rest = tail ? fmax(0.0, 1.0 - mass) : 0.0;
    const float top = tail && some ? fmaxf(part.m, m_listed) : part.m;
    const double s_rest = part.s * shifted_exp(part.m, top, c);   // all, where there is no rest
    const double s_listed = !tail || !some ? 0.0 : m_listed == top ? part.s_listed : part.s_listed * exp(((double)m_listed - top) * a.inv_t);
    const double total = s_rest + s_listed;
    if (rank == 0 && tid == 0) {
      double loss = tail || part.mass == 0.0 ? part.cross : part.cross * norm - log(part.mass);
      if (some) loss += mass * (((double)top - m_listed) * a.inv_t + log(total));
      // nothing outside the list but -infinity, or nothing at all: then the teacher's rest is its rounding, and left out
      if (rest > 0.0 && part.s > 0.f)
        loss += rest * (log(rest) - (s_rest >= s_listed ? -log1p(s_listed / s_rest)
                                                         : ((double)part.m - top) * a.inv_t + log((double)part.s) - log(total)));
      a.row_loss[r] = (float)(loss * w);
    }
    if (!d_first) continue;

    // ---- the gradient: outside the list a multiple of 2^((x - m) c), in the list afterwards
    const float scale = (float)((double)w * a.inv_t / a.loss_div);
    const double every = mass + rest;
    float factor = 0.f;
    if (!(part.s <= 0.f)) factor = (float)((every * (s_rest / total) - rest) / part.s) * scale;
    const float m = part.m;
    for (unsigned s = 0; s < (MULTI ? a.segments : 1u); ++s) {
      const unsigned base = (s * ctas + rank) * kSlice;
      if (MULTI) load(base);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const unsigned word = base + i * G + tid;
        float x[P];
        unpack(v[i], x, T());
#pragma unroll
        for (int j = 0; j < P; ++j) x[j] = factor * shifted_exp(x[j], m, c);
        if (word < words) put(word, x);
      }
    }
    sync();
    const float share = (float)(every / total), q_norm = (float)norm;
    for (unsigned e = tid, j = 0; e < a.k; e += G, ++j) {
      if (!owner(e)) continue;
      float q = e_q[e];
      if (twice)
        for (unsigned i = e + 1; i < a.k; ++i)
          if (e_index[i] == e_index[e]) q += e_q[i];
      float g = scale * (shifted_exp(e_z[e], top, c) * share - q * q_norm);
      if (a.accumulate)
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
          if (i == j) g += old[i];
      d_first[e_index[e]] = from_float<T>(g);
    }
  }
  if (a.fold) {
    __syncthreads();
    if (rank == 0 && threadIdx.x < 32) {
      double sum = 0.0;
      for (size_t r = threadIdx.x; r < a.rows; r += 32) sum += a.row_loss[r];
      sum = warp_sum(sum);
      if (threadIdx.x == 0) *a.loss = (float)(sum / a.loss_div);
    }
  }
}

// loss = sum of the rows' shares / loss_div, in a fixed order
__global__ void __launch_bounds__(1024) distill_loss_kernel(const float* row_loss, size_t rows, double loss_div, float* loss) {
  __shared__ double sm[32];
  pdl_sync();
  double sum = 0.0;
  for (size_t r = threadIdx.x; r < rows; r += 1024) sum += row_loss[r];
  sum = block_sum<double>(sum, sm);
  if (threadIdx.x == 0) *loss = (float)(sum / loss_div);
}

template <typename T, int NV, int G, bool MULTI>
static void launch_distill(cudaStream_t s, DistillArgs a, unsigned cluster) {
  static SharedMemoryLimit limit;
  const size_t own = 2 * cluster * (G / 32) * sizeof(DistillPart) + (size_t)G * NV + 12 * (size_t)((a.k + 3) & ~3u) + 16;
  const size_t smem = own * (kDThreads / G);
  if (smem > 48 * 1024 && !limit.raise(distill_kernel<T, NV, G, MULTI>, 100 * 1024)) return;
  const size_t groups = G == 32 ? (a.rows + kDThreads / 32 - 1) / (kDThreads / 32) : a.rows;
  const size_t most = (size_t)1 << 20;
  const unsigned grid = (unsigned)(groups < most ? groups : most) * cluster;
  a.fold = grid == cluster;
  if (!launch_pdl_cluster(distill_kernel<T, NV, G, MULTI>, dim3(grid), dim3(kDThreads), smem, s, cluster, a)) return;
  if (!a.fold) launch_pdl(distill_loss_kernel, dim3(1), dim3(1024), 0, s, (const float*)a.row_loss, a.rows, a.loss_div, a.loss);
}

template <typename T>
static void launch_distill_rows(cudaStream_t s, DistillArgs a) {
  const unsigned words = (unsigned)(((size_t)a.C + 2 * kPerWord<T> - 2) / kPerWord<T>);  // wherever a row starts
  a.segments = (words + kDThreads * 4 - 1) / (kDThreads * 4);
  launch_distill<T, 4, kDThreads, true>(s, a, 1);
}

}  // namespace zg

using namespace zg;

extern "C" void zg_distill_ce(dtype id, dtype t_id, StreamWrapper w, const void* logits, len_t rows, len_t C, len_t ld, const len_t* t_index,
                              const void* t_logits, const void* t_lse, len_t k, const void* row_weight, double temperature, double loss_div,
                              void* loss_out, void* row_loss, void* dlogits, int accumulate) {
  const char* me = "zg_distill_ce";
  if ((id != SINGLE && id != BF16) || (t_id != SINGLE && t_id != BF16)) { set_error(kUnsupported, "%s: logits are SINGLE or BF16", me); return; }
  if (ld == 0) ld = C;
  if (C == 0 || C > (len_t)0x7fffffff || ld < C) { set_error(kBadArgument, "%s: C %lu, ld %lu", me, C, ld); return; }
  if (k == 0 || k > kDMaxList) { set_error(kBadArgument, "%s: lists of 1 to %u entries, got %lu", me, kDMaxList, k); return; }
  if (!(temperature > 0.0) || !(temperature <= 1e30) || !(1.0 / temperature <= 1e30)) { set_error(kBadArgument, "%s: temperature %g", me, temperature); return; }
  if (!(loss_div > 0.0 || loss_div < 0.0)) { set_error(kBadArgument, "%s: loss_div %g", me, loss_div); return; }
  const size_t size = id == BF16 ? 2 : 4, t_size = t_id == BF16 ? 2 : 4;
  const auto off = [](const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
  if (!loss_out || off(loss_out, 4)) { set_error(kBadArgument, "%s: loss_out is missing or not aligned", me); return; }
  cudaStream_t s = as_stream(w);
  if (rows == 0) { ZG_CUDA(cudaMemsetAsync(loss_out, 0, 4, s)); return; }
  if (!logits || !t_index || !t_logits || !row_loss) { set_error(kBadArgument, "%s: a required operand is NULL", me); return; }
  if (off(logits, size) || off(t_index, 8) || off(t_logits, t_size) || off(t_lse, 4) || off(row_weight, 4) || off(row_loss, 4) || off(dlogits, size)) {
    set_error(kBadArgument, "%s: an operand is not aligned to its elements", me);
    return;
  }
  if (dlogits == logits && accumulate) { set_error(kBadArgument, "%s: a gradient in place of the logits cannot be accumulated", me); return; }
  DistillArgs a;
  a.logits = logits; a.dlogits = dlogits; a.rows = rows; a.ld = ld; a.C = (unsigned)C; a.k = (unsigned)k;
  a.t_index = t_index; a.t_logits = t_logits; a.t_bf16 = t_id == BF16; a.t_lse = (const float*)t_lse; a.weight = (const float*)row_weight;
  a.inv_t = 1.0 / temperature; a.c = (float)(1.4426950408889634 / temperature); a.loss_div = loss_div;
  a.loss = (float*)loss_out; a.row_loss = (float*)row_loss; a.accumulate = dlogits ? accumulate : 0;
  a.same_lead = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(dlogits)) % 16 == 0;
  a.segments = 1; a.fold = 0;
  if (id == SINGLE) launch_distill_rows<float>(s, a);
  else launch_distill_rows<__nv_bfloat16>(s, a);
}
