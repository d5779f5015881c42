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
  float grad_scale;       // 1 / (temperature loss_div)
  double loss_div;
  float* loss;
  float* row_loss;        // [rows]
  int accumulate;
  int same_lead;          // rows of logits and dlogits start equally far behind a 16-byte boundary
  unsigned slice;         // words of a row that a CTA (a warp) holds at a time
  unsigned segments;      // slices of a row per CTA
  int fold;               // this grid is one CTA or cluster: it writes the loss itself
};

// What the warps of a group know of a row, put together into what all of them need
struct RestPart {
  float m, s;  // largest value outside the list (everywhere where there is no rest), sum of 2^((x - m) c)
};
struct ListPart {   // to maxima that all warps know, so that these only add up
  double s_listed;  // sum of exp((x - m_listed) / T), each class once
  double mass;      // sum of w: q, or exp((u - u_max) / T) where the list's own sum is the normaliser
  double cross;     // sum of w (log w - (z - m_listed) / T)
};

// What one warp makes of them for all
struct Common {
  float m, s;      // of the rest (of all)
  float top;       // of all
  float factor;    // the gradient outside the list is factor 2^((x - m) c)
  float share;     // (mass + rest) / sum of 2^((x - top) c)
  float q_norm;    // q is q_norm times an entry's weight
};

__device__ __forceinline__ RestPart join_lanes(RestPart p, float c) {
  const float m = value_of(__reduce_max_sync(0xffffffffu, key_of(p.m)));
  return RestPart{m, warp_sum(p.s * shifted_exp(p.m, m, c))};
}
__device__ __forceinline__ ListPart join_lanes(ListPart p) { return ListPart{warp_sum(p.s_listed), warp_sum(p.mass), warp_sum(p.cross)}; }

__device__ __forceinline__ void copy_word(void* smem_dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem_dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Bytes of shared memory of a group of G threads
__host__ __device__ constexpr unsigned list_warps(unsigned k, unsigned warps) { return (k + 63) / 64 < warps ? (k + 63) / 64 : warps; }
__host__ __device__ constexpr unsigned distill_bytes(unsigned G, unsigned ctas, unsigned slice, unsigned k) {
  const unsigned parts = 2 * ctas * (G / 32 * (unsigned)sizeof(RestPart) + list_warps(k, G / 32) * (unsigned)sizeof(ListPart));
  return slice * 17 + (parts + 15) / 16 * 16 + 12 * ((k + 3) & ~3u) + 48;
}

// G threads take a row together: a warp (short rows, eight to a CTA) or a CTA, of which a cluster shares a row.  CTA r holds
// `slice` words of it (a multiple of G) in shared memory from the sums to the gradient, so that a row is read once; a thread
// copies, reads and writes words i G + t of them, its own only, which takes no barrier.  Rows longer than that (MULTI) are walked in
// several slices per CTA, twice.  The list is the work of the last warps, 64 entries or more each.
template <typename T, int G, int THREADS, bool MULTI>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) distill_kernel(const DistillArgs a) {
  constexpr int P = kPerWord<T>;
  constexpr int kGroups = THREADS / G;
  constexpr int kWarps = G / 32;
  constexpr int kOwn = G == 32 ? 4 : (int)kDMaxList / THREADS;  // list entries per thread at most
  extern __shared__ __align__(16) unsigned char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned ctas = G == 32 ? 1 : cluster.num_blocks(), rank = G == 32 ? 0 : cluster.block_rank();
  const unsigned tid = threadIdx.x % G, lane = threadIdx.x & 31, warp = tid >> 5;
  const unsigned list = list_warps(a.k, kWarps), slice = a.slice;
  const unsigned entry = tid - (kWarps - list) * 32;  // wraps around to no entry for the other warps
  unsigned char* mine = smem + (threadIdx.x / G) * distill_bytes(G, ctas, slice, a.k);
  uint4* const held = reinterpret_cast<uint4*>(mine);                                      // [slice]
  ListPart* const list_parts = reinterpret_cast<ListPart*>(held + slice);                  // [2][ctas * list]
  RestPart* const rest_parts = reinterpret_cast<RestPart*>(list_parts + 2 * ctas * list);  // [2][ctas * kWarps]
  uint32_t* const bits = reinterpret_cast<uint32_t*>(mine + distill_bytes(G, ctas, slice, a.k) - slice - 12 * ((a.k + 3) & ~3u) - 48);  // a byte per word
  uint32_t* const e_index = bits + slice / 4;                                              // this CTA's entries; ~0: not one of them
  float* const e_q = reinterpret_cast<float*>(e_index + ((a.k + 3) & ~3u));
  float* const e_z = e_q + ((a.k + 3) & ~3u);
  uint32_t* const most = reinterpret_cast<uint32_t*>(e_z + ((a.k + 3) & ~3u));             // keys of the list's largest student's and teacher's logit
  Common* const common = reinterpret_cast<Common*>(most + 2);
  auto sync = [] { if (G == 32) __syncwarp(); else __syncthreads(); };
  auto sync_any = [](bool v) -> bool {
    if (G > 32) return __syncthreads_or(v);
    v = __any_sync(0xffffffffu, v);
    __syncwarp();
    return v;
  };
  const bool tail = a.t_lse != nullptr;
  const float c = a.c;
  unsigned parity = 0;
  bool met = G == 32 || ctas == 1;  // every CTA of the cluster is there: its shared memory may be written
  if (!met) cluster.barrier_arrive();
  pdl_sync();
  const size_t first = G == 32 ? (size_t)blockIdx.x * kGroups + threadIdx.x / 32 : blockIdx.x / ctas;
  const size_t stride = G == 32 ? (size_t)gridDim.x * kGroups : gridDim.x / ctas;
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
          for (unsigned i = tid; i < slice; i += G) {
            const unsigned word = (s * ctas + rank) * slice + i;
            float zero[P] = {};
            if (word < words) put(word, zero);
          }
      if (rank == 0 && tid == 0) a.row_loss[r] = 0.f;
      continue;
    }
    // Of a slice from word `base` on, words lo .. hi - 1 are whole (the row's first and last may not be); up to `end` they are the row's
    auto limits = [&](unsigned base, unsigned& lo, unsigned& hi, unsigned& end) {
      lo = base == 0 && row.lead ? 1 : 0;
      hi = min(max(row.end / P, base + lo) - base, slice);
      end = min(max(words, base) - base, slice);
    };
    // f(i) for this thread's i of lo .. hi - 1, four at a time where there are so many
    auto each = [&](unsigned lo, unsigned hi, auto f) {
      unsigned i = tid < lo ? tid + G : tid;
      for (; i + 3 * G < hi; i += 4 * G) {
#pragma unroll
        for (unsigned j = 0; j < 4; ++j) f(i + j * G);
      }
      for (; i < hi; i += G) f(i);
    };
    auto load = [&](unsigned base) {
      unsigned lo, hi, end;
      limits(base, lo, hi, end);
      const uint4* src = row.word(base);
      each(lo, hi, [&](unsigned i) { copy_word(held + i, src + i); });
      if (tid < lo) held[0] = row.load_part(0);
      for (unsigned i = hi + (tid + G - hi % G) % G; i < slice; i += G) held[i] = i < end ? row.load_part(base + i) : nothing<T>();
    };
    if (r != first) sync();  // the row before has been patched: lists and bits are free
    const len_t* index = a.t_index + r * a.k;
    len_t at_first = ~(len_t)0;
    if (entry < a.k) at_first = index[entry];
    if (!MULTI) load(rank * slice);
    for (unsigned i = tid; i < slice / 16; i += G) reinterpret_cast<uint4*>(bits)[i] = make_uint4(0, 0, 0, 0);
    if (tid < 2) most[tid] = 0;
    sync();

    // ---- the teacher's list.  Its entries belong to the CTA whose slice they lie in.
    auto u_of = [&](unsigned e) -> float {
      return a.t_bf16 ? as_float(static_cast<const __nv_bfloat16*>(a.t_logits)[r * a.k + e]) : static_cast<const float*>(a.t_logits)[r * a.k + e];
    };
    auto mark = [&](unsigned at, unsigned base) -> bool {  // true: it was marked
      const unsigned p = at + row.lead, word = p / P - base;
      if (word >= slice) return false;  // of another slice (below this one: wraps around)
      const uint32_t bit = 1u << ((word & 3) * 8 + p % P);
      return (atomicOr(bits + (word >> 2), bit) & bit) != 0;
    };
    float old[kOwn];
    bool seen = false;
    uint32_t most_z = 0, most_u = 0;
    for (unsigned e = entry, j = 0; e < a.k; e += list * 32, ++j) {
      const len_t at = j == 0 ? at_first : index[e];
      unsigned keep = ~0u;
      if (at < a.C) {
        const float z = as_float(row.first[at]);
        const bool own = ctas == 1 || ((unsigned)at + row.lead) / P / slice % ctas == rank;
        if (own) {
          keep = (unsigned)at;
          if (!MULTI) seen |= mark(keep, rank * slice);
          e_z[e] = z;
          e_q[e] = u_of(e);
          if (d_first && a.accumulate)
#pragma unroll
            for (int i = 0; i < kOwn; ++i)
              if (i == j) old[i] = as_float(d_first[at]);
        }
        most_z = max(most_z, key_of(z));
        if (!tail) most_u = max(most_u, key_of(u_of(e)));
      }
      e_index[e] = keep;
    }
    if (entry < list * 32) {
      most_z = __reduce_max_sync(0xffffffffu, most_z);
      if (!tail) most_u = __reduce_max_sync(0xffffffffu, most_u);
      if (lane == 0) {
        atomicMax(most, most_z);
        if (!tail) atomicMax(most + 1, most_u);
      }
    }

    // ---- largest value and sum of the rest
    bool twice = false;
    RestPart rest_part{-INFINITY, 0.f};
    for (unsigned s = 0; s < (MULTI ? a.segments : 1u); ++s) {
      if (MULTI) {
        const unsigned base = (s * ctas + rank) * slice;
        load(base);
        if (s > 0) {
          sync();
          for (unsigned i = tid; i < slice / 4; i += G) bits[i] = 0;
        }
        sync();
        seen = false;
        for (unsigned e = entry; e < a.k; e += list * 32)
          if (e_index[e] != ~0u) seen |= mark(e_index[e], base);
      }
      copies_done();
      twice |= sync_any(seen);
      if (tail) {  // what is listed leaves the slice
        for (unsigned e = entry; e < a.k; e += list * 32) {
          const unsigned p = e_index[e] + row.lead - (MULTI ? s * ctas + rank : rank) * slice * P;
          if (e_index[e] != ~0u && p < slice * P) reinterpret_cast<T*>(held)[p] = from_float<T>(-INFINITY);
        }
        sync();
      }
      constexpr unsigned U = 4;  // words at a time
      const Pair cc = pair_of(c, c);
      unsigned i = tid;
      for (; i + (U - 1) * G < slice; i += U * G) {
        uint4 v[U];
#pragma unroll
        for (unsigned j = 0; j < U; ++j) v[j] = held[i + j * G];
        const float m = fmaxf(rest_part.m, fmaxf(fmaxf(word_max(v[0], T()), word_max(v[1], T())), fmaxf(word_max(v[2], T()), word_max(v[3], T()))));
        const Pair shift = minus(m);
        Pair sum[U];
#pragma unroll
        for (unsigned j = 0; j < U; ++j) {
          float x[P];
          unpack(v[j], x, T());
          sum[j] = shifted_exp(x[0], x[1], shift, cc);
#pragma unroll
          for (int l = 2; l < P; l += 2) sum[j] = sum[j] + shifted_exp(x[l], x[l + 1], shift, cc);
        }
        float s0, s1;
        split((sum[0] + sum[1]) + (sum[2] + sum[3]), s0, s1);
        rest_part = RestPart{m, rest_part.s * shifted_exp(rest_part.m, m, c) + (s0 + s1)};
      }
      for (; i < slice; i += G) {
        const uint4 v = held[i];
        const float m = fmaxf(rest_part.m, word_max(v, T()));
        const Pair shift = minus(m);
        float x[P], s0, s1;
        unpack(v, x, T());
        Pair sum = shifted_exp(x[0], x[1], shift, cc);
#pragma unroll
        for (int l = 2; l < P; l += 2) sum = sum + shifted_exp(x[l], x[l + 1], shift, cc);
        split(sum, s0, s1);
        rest_part = RestPart{m, rest_part.s * shifted_exp(rest_part.m, m, c) + (s0 + s1)};
      }
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
    ListPart list_part{0.0, 0.0, 0.0};
    if (entry < list * 32) {
      const double level = tail ? (double)a.t_lse[r] : 0.0, u_top = tail ? 0.0 : (double)value_of(most[1]);
      for (unsigned e = entry; e < a.k; e += list * 32) {
        if (e_index[e] == ~0u) continue;
        const float z = e_z[e], u = e_q[e];
        const double arg = tail ? (double)u * a.inv_t - level : ((double)u - u_top) * a.inv_t, far = ((double)z - m_listed) * a.inv_t;
        const double q = u == -INFINITY ? 0.0 : exp(arg);
        e_q[e] = (float)q;
        list_part.mass += q;
        if (!(q <= 0.0)) list_part.cross += z == -INFINITY ? INFINITY : q * (arg - far);  // a class of mass that the student rules out: infinite
        if (z != -INFINITY && owner(e)) list_part.s_listed += exp(far);
      }
      list_part = join_lanes(list_part);
    }

    // ---- over the lanes, the warps and the cluster's CTAs
    rest_part = join_lanes(rest_part, c);
    if (G > 32) {
      RestPart* const rests = rest_parts + parity * ctas * kWarps;
      ListPart* const lists = list_parts + parity * ctas * list;
      if (ctas == 1) {
        if (lane == 0) rests[warp] = rest_part;
        if (lane == 0 && entry < list * 32) lists[entry / 32] = list_part;
        __syncthreads();
      } else {
        if (!met) cluster.barrier_wait();
        met = true;
        if (lane < ctas) {
          cluster.map_shared_rank(rests, lane)[rank * kWarps + warp] = rest_part;
          if (entry < list * 32) cluster.map_shared_rank(lists, lane)[rank * list + entry / 32] = list_part;
        }
        cluster.sync();  // also: nobody reads the parts of the row before any more
      }
      if (warp == 0) {
        const unsigned n = ctas * kWarps, nl = ctas * list;
        const RestPart p = lane < n ? rests[lane] : RestPart{-INFINITY, 0.f}, q = lane + 32 < n ? rests[lane + 32] : RestPart{-INFINITY, 0.f};
        rest_part.m = fmaxf(p.m, q.m);
        rest_part.s = p.s * shifted_exp(p.m, rest_part.m, c) + q.s * shifted_exp(q.m, rest_part.m, c);
        rest_part = join_lanes(rest_part, c);
        list_part = ListPart{0.0, 0.0, 0.0};
        for (unsigned i = 0; i < nl; ++i) {
          list_part.s_listed += lists[i].s_listed;
          list_part.mass += lists[i].mass;
          list_part.cross += lists[i].cross;
        }
      }
      parity ^= 1;
    }

    // ---- by one warp, for all
    double rest = 0.0, mass = 0.0, total = 0.0;
    bool some = false;
    Common both;
    if (warp == 0) {
      some = !(list_part.s_listed <= 0.0);   // a listed class that the student does not rule out
      mass = tail || list_part.mass == 0.0 ? list_part.mass : 1.0;
      rest = tail ? fmax(0.0, 1.0 - mass) : 0.0;
      both.top = tail && some ? fmaxf(rest_part.m, m_listed) : rest_part.m;
      const double s_rest = rest_part.s * shifted_exp(rest_part.m, both.top, c);   // all, where there is no rest
      const double s_listed = !tail || !some ? 0.0 : m_listed == both.top ? list_part.s_listed : list_part.s_listed * exp(((double)m_listed - both.top) * a.inv_t);
      total = s_rest + s_listed;
      both.m = rest_part.m;
      both.s = rest_part.s;
      // ((mass + rest) p_r - rest) / s, p_r = s_rest / total
      both.factor = rest_part.s <= 0.f ? 0.f : (float)(mass * s_rest - rest * s_listed) / ((float)total * rest_part.s);
      both.share = (float)(mass + rest) / (float)total;
      both.q_norm = tail || list_part.mass == 0.0 ? 1.f : 1.f / (float)list_part.mass;
      if (G > 32 && lane == 0) *common = both;
    }
    if (G > 32) {
      __syncthreads();
      both = *common;
    }
    if (d_first) {
      // ---- the gradient: outside the list a multiple of 2^((x - m) c), in the list afterwards
      const float scale = w * a.grad_scale, factor = both.factor * scale;
      const Pair shift = minus(both.m), cc = pair_of(c, c), factors = pair_of(factor, factor);
      for (unsigned s = 0; s < (MULTI ? a.segments : 1u); ++s) {
        const unsigned base = (s * ctas + rank) * slice;
        if (MULTI) {
          load(base);
          copies_done();
        }
        unsigned lo, hi, end;
        limits(base, lo, hi, end);
        auto grad = [&](unsigned i, float (&x)[P]) {
          unpack(held[i], x, T());
#pragma unroll
          for (int j = 0; j < P; j += 2) split(shifted_exp(x[j], x[j + 1], shift, cc) * factors, x[j], x[j + 1]);
        };
        float x[P];
        if (a.same_lead && !a.accumulate) {
          uint4* dst = d_row.word(base);
          each(lo, hi, [&](unsigned i) {
            float y[P];
            grad(i, y);
            dst[i] = pack(y, T());
          });
          if (tid < lo) {
            grad(0, x);
            d_row.store(0, x);
          }
          const unsigned i = end - 1;
          if (hi < end && i % G == tid) {
            grad(i, x);
            d_row.store(base + i, x);
          }
        } else {
          for (unsigned i = tid; i < end; i += G) {
            grad(i, x);
            put(base + i, x);
          }
        }
      }
      sync();
      for (unsigned e = entry, j = 0; e < a.k; e += list * 32, ++j) {
        if (!owner(e)) continue;
        float q = e_q[e];
        if (twice)
          for (unsigned i = e + 1; i < a.k; ++i)
            if (e_index[i] == e_index[e]) q += e_q[i];
        float g = scale * (shifted_exp(e_z[e], both.top, c) * both.share - q * both.q_norm);
        if (a.accumulate)
#pragma unroll
          for (int i = 0; i < kOwn; ++i)
            if (i == j) g += old[i];
        d_first[e_index[e]] = from_float<T>(g);
      }
    }
    if (rank == 0 && tid == 0) {
      double loss = tail || list_part.mass == 0.0 ? list_part.cross : list_part.cross / list_part.mass - log(list_part.mass);
      const double log_total = log(total);
      if (some) loss += mass * (((double)both.top - m_listed) * a.inv_t + log_total);
      // nothing outside the list but -infinity, or nothing at all: then the teacher's rest is its rounding, and left out
      if (rest > 0.0 && both.s > 0.f) loss += rest * (log(rest / both.s) + ((double)both.top - both.m) * a.inv_t + log_total);
      a.row_loss[r] = (float)(loss * w);
    }
  }
  if (!met) cluster.barrier_wait();
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

template <typename T, int G, int THREADS, bool MULTI>
static void launch_distill(cudaStream_t s, DistillArgs a, unsigned cluster) {
  static SharedMemoryLimit limit;
  const size_t smem = (size_t)distill_bytes(G, cluster, a.slice, a.k) * (THREADS / G);
  if (smem > 48 * 1024 && !limit.raise(distill_kernel<T, G, THREADS, MULTI>, 227 * 1024)) return;
  const size_t groups = G == 32 ? (a.rows + THREADS / 32 - 1) / (THREADS / 32) : a.rows;
  const size_t most = (size_t)1 << 20;
  const unsigned grid = (unsigned)(groups < most ? groups : most) * cluster;
  a.fold = grid == cluster;
  if (!launch_pdl_cluster(distill_kernel<T, G, THREADS, MULTI>, dim3(grid), dim3(THREADS), smem, s, cluster, a)) return;
  if (!a.fold) launch_pdl(distill_loss_kernel, dim3(1), dim3(1024), 0, s, (const float*)a.row_loss, a.rows, a.loss_div, a.loss);
}

template <typename T>
static void launch_distill_rows(cudaStream_t s, DistillArgs a) {
  const unsigned words = (unsigned)(((size_t)a.C + 2 * kPerWord<T> - 2) / kPerWord<T>);  // wherever a row starts
  const char* env = getenv("ZG_D");
  int force_c = 0, force_g = 0, most_kb = 48, threads = 128;
  if (env) sscanf(env, "%d,%d,%d", &force_g, &force_c, &most_kb);
  if (force_g) threads = force_g;
  if (force_g == 32 || (!env && words <= 32 * 8 && a.k <= 128)) {
    a.slice = (words + 31) / 32 * 32;
    return launch_distill<T, 32, 256, false>(s, a, 1);
  }
  const unsigned most = most_kb * 64;  // words of a slice
  unsigned cluster = 1;
  while (cluster < 8 && words > most * cluster) cluster *= 2;
  while (cluster < 8 && a.rows * cluster * 2 <= (size_t)sm_count() && words > threads * cluster) cluster *= 2;
  if (force_c) cluster = force_c;
  const unsigned widest = 184 * 64;
  if (words > widest * cluster) {
    a.slice = widest / threads * threads;
    a.segments = (words + a.slice * cluster - 1) / (a.slice * cluster);
    if (threads == 128) return launch_distill<T, 128, 128, true>(s, a, cluster);
    return launch_distill<T, 256, 256, true>(s, a, cluster);
  }
  a.slice = ((words + cluster - 1) / cluster + threads - 1) / threads * threads;
  if (threads == 128) return launch_distill<T, 128, 128, false>(s, a, cluster);
  launch_distill<T, 256, 256, false>(s, a, cluster);
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
  a.inv_t = 1.0 / temperature; a.c = (float)(1.4426950408889634 / temperature); a.loss_div = loss_div; a.grad_scale = (float)(a.inv_t / loss_div);
  a.loss = (float*)loss_out; a.row_loss = (float*)row_loss; a.accumulate = dlogits ? accumulate : 0;
  a.same_lead = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(dlogits)) % 16 == 0;
  a.slice = 0; a.segments = 1; a.fold = 0;
  if (id == SINGLE) launch_distill_rows<float>(s, a);
  else launch_distill_rows<__nv_bfloat16>(s, a);
}
