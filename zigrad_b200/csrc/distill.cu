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
// it (a bit per position says which is which), and with s_r and s_l the two sums, in 64 bits from there on, p_r = s_r / (s_r + s_l) and the
// coefficient (S + r) p_r - r = (S s_r - r s_l) / (s_r + s_l).  An error e of the sum outside, made of fp32 terms, then changes the row by
// e (S - (1 - p_r)) only; one of the listed sum would change it by e (1 - p_r), so the list, k terms of C, is summed in 64 bits.
#include "row_access.cuh"

namespace zg {

using namespace ra;

constexpr unsigned kDMaxList = 1024;
constexpr unsigned kDShortList = 128;  // where a CTA has several rows (launch_distill_rows)

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
  int same_lead;          // rows of logits and dlogits start equally far behind a 16-byte boundary
  unsigned slice;         // words of a row that a CTA (a warp) holds at a time
  unsigned segments;      // slices of a row per CTA
  int fold;               // this grid is one CTA or cluster: it writes the loss itself
};

// What the workers know of a row's values outside the list (of all where there is no rest)
struct RestPart {
  float m, s;  // the largest, and the sum of 2^((x - m) c)
};
// What a CTA's manager knows of the list's entries in its slice
struct ListPart {
  double s_listed;  // sum of exp((x - m) / T), each class once
  double mass;      // sum of w: q, or exp((u - u_max) / T) where the list's own sum is the normaliser
  double cross;     // sum of w (log w - (z - m) / T)
  float m;          // the largest of the student's values there
  float pad;
};
// What comes of them
struct Common {
  float m;         // the gradient outside the list is factor 2^((x - m) c)
  float factor;
};

// over the L lanes that share a row
template <int L, typename V>
__device__ __forceinline__ V lanes_sum(V v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int L>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if constexpr (L == 32) {
    return __reduce_max_sync(0xffffffffu, v);
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
}

// Shared memory of a row: its slice, a byte per word of it, the list (index, weight, logit, gradient), what CTAs send one another, what
// the manager tells the workers
__host__ __device__ constexpr unsigned distill_row_bytes(unsigned ctas, unsigned workers, unsigned slice, unsigned k) {
  return (slice * 17 + 16 * ((k + 3) & ~3u) + ctas * ((unsigned)sizeof(ListPart) + workers * (unsigned)sizeof(RestPart)) + (unsigned)sizeof(Common) + 15) & ~15u;
}

// A CTA has ROWS rows, WORKERS warps for each and one warp, the manager, for all of them.  Workers copy a row (of a cluster's
// row their CTA's `slice` words) into shared memory, sum it and write the gradient, so that the row is read once; each
// touches its own words only.  The manager does all else, 32 / ROWS lanes to a row: the sums over the list while the
// workers sum the rest, what follows from both, the loss, and the words and entries that are not whole words.  So the arithmetic
// in 64 bits and the bookkeeping cost one warp's instructions, not every warp's: with them in all warps a row of 16384 took
// 8346 instructions.
// 4096 x 131072 bf16: 2.15 GB in 471 us with a cold L2.  What bounds it is the chain of phases: most of what warps wait for is
// a barrier, the special-function unit (two exponentials an element) is 54 % busy, an instruction issues in 42 % of the cycles.
// MULTI: rows longer than a cluster's shared memory, walked in several slices per CTA, twice.
// ADD: the gradient is added to what is there (as a parameter of its own: as a branch it cost the other calls registers, 470 -> 497 us).
template <typename T, int ROWS, int WORKERS, int CTAS, bool MULTI, bool ADD>
__global__ void __launch_bounds__((ROWS * WORKERS + 1) * 32, CTAS) distill_kernel(const DistillArgs a) {
  constexpr int P = kPerWord<T>;
  constexpr int L = 32 / ROWS;               // lanes of the manager per row
  constexpr unsigned G = WORKERS * 32;       // workers' threads per row
  extern __shared__ __align__(16) unsigned char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned ctas = ROWS > 1 ? 1 : cluster.num_blocks(), rank = ROWS > 1 ? 0 : cluster.block_rank();
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool manager = warp == ROWS * WORKERS;
  const unsigned mine = manager ? lane / L : warp / WORKERS;             // which of the CTA's rows
  const unsigned tid = manager ? lane % L : threadIdx.x % G;
  const unsigned slice = a.slice, k4 = (a.k + 3) & ~3u;
  unsigned char* const at = smem + mine * distill_row_bytes(ctas, WORKERS, slice, a.k);
  uint4* const held = reinterpret_cast<uint4*>(at);                       // [slice]
  uint32_t* const bits = reinterpret_cast<uint32_t*>(held + slice);       // a byte per word
  uint32_t* const e_index = bits + slice / 4;                             // this CTA's entries; ~0: not one of them
  float* const e_w = reinterpret_cast<float*>(e_index + k4);              // the teacher's logit, then the weight
  float* const e_z = e_w + k4;
  float* const e_old = e_z + k4;                                          // the gradient's buffer, where it is added to
  ListPart* const lists = reinterpret_cast<ListPart*>(e_old + k4);        // [ctas]
  RestPart* const rests = reinterpret_cast<RestPart*>(lists + ctas);      // [ctas * WORKERS]
  Common* const common = reinterpret_cast<Common*>(rests + ctas * WORKERS);
  const bool tail = a.t_lse != nullptr;
  const float c = a.c;
  if (ctas > 1) cluster.barrier_arrive();
  pdl_sync();
  const size_t r = ROWS > 1 ? (size_t)blockIdx.x * ROWS + mine : blockIdx.x / ctas;
  const bool there = r < a.rows;
  const Row<T> row(const_cast<T*>(static_cast<const T*>(a.logits)) + (there ? r * a.ld : 0), a.C);
  T* const d_first = a.dlogits && there ? static_cast<T*>(a.dlogits) + r * a.ld : nullptr;
  const Row<T> d_row(d_first, a.C);
  const float w = !there ? 0.f : a.weight ? a.weight[r] : 1.f;
  const bool counts = w != 0.f;  // a row that counts nothing is not read: it may hold anything
  // Of the slice from word `base` on, words lo .. hi - 1 are whole (the row's first and last may not be); up to `end` they are the row's
  unsigned base = rank * slice, lo, hi, end;
  auto set_limits = [&] {
    lo = base == 0 && row.lead ? 1 : 0;
    hi = min(max(row.end / P, base + lo) - base, slice);
    end = min(max(row.words(), base) - base, slice);
  };
  set_limits();
  // This thread's words i of from .. to - 1: four(i), for i, i + G, .. i + 3 G, where there are so many, else one(i)
  auto each = [&](unsigned from, unsigned to, auto four, auto one) {
    unsigned i = tid < from ? tid + G : tid;
    for (; i + 3 * G < to; i += 4 * G) four(i);
    for (; i < to; i += G) one(i);
  };
  auto load = [&] {
    if (!counts) return;
    if (!manager) {
      const uint4* src = row.word(base);
      auto one = [&](unsigned i) { copy_word(held + i, src + i); };
      each(lo, hi, [&](unsigned i) { one(i); one(i + G); one(i + 2 * G); one(i + 3 * G); }, one);
    } else {
      if (tid == 0 && lo) held[0] = row.load_part(0);
      for (unsigned i = hi + tid; i < slice; i += L) held[i] = i < end ? row.load_part(base + i) : nothing<T>();
    }
  };

  // ---- the row's way into shared memory; the manager reads the list.  Entries belong to the CTA whose slice they lie in.
  const unsigned k = counts ? a.k : 0;
  float u_top = 0.f;
  double level = 0.0;
  bool twice = false;
  if (!MULTI && !manager) load();
  if (manager) {
    const len_t* const index = a.t_index + (there ? r * a.k : 0);
    uint32_t most = 0;
    if (tail && counts) level = a.t_lse[r];
    // four entries at a time: what their loads take is what the manager takes
    for (unsigned e0 = tid; e0 < k; e0 += 4 * L) {
      len_t cls[4];
      float u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned e = min(e0 + j * L, k - 1);
        cls[j] = index[e];
        u[j] = a.t_bf16 ? as_float(static_cast<const __nv_bfloat16*>(a.t_logits)[r * a.k + e]) : static_cast<const float*>(a.t_logits)[r * a.k + e];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned e = e0 + j * L;
        if (e >= k) continue;
        const bool entry = cls[j] < a.C, own = entry && (ctas == 1 || ((unsigned)cls[j] + row.lead) / P / slice % ctas == rank);
        e_index[e] = own ? (unsigned)cls[j] : ~0u;
        e_w[e] = u[j];
        if (ADD && own && d_first) e_old[e] = as_float(d_first[cls[j]]);
        if (entry) most = max(most, key_of(u[j]));
      }
    }
    for (unsigned i = tid; i < slice / 16; i += L) reinterpret_cast<uint4*>(bits)[i] = make_uint4(0, 0, 0, 0);
    u_top = value_of(lanes_max<L>(most));  // 0, no entry: a NaN that nothing below takes
    if (!MULTI) load();
  }

  // ---- largest value and sum of the rest by the workers, the sums over the list by the manager
  const Pair cc = pair_of(c, c);
  RestPart part{-INFINITY, 0.f};
  ListPart list{0.0, 0.0, 0.0, -INFINITY, 0.f};
  auto owner = [&](unsigned e) -> bool {  // a class that is listed twice counts once among the student's values
    if (e_index[e] == ~0u) return false;
    if (twice)
      for (unsigned j = 0; j < e; ++j)
        if (e_index[j] == e_index[e]) return false;
    return true;
  };
  for (unsigned s = 0; s < (MULTI ? a.segments : 1u); ++s) {
    if (MULTI) {
      __syncthreads();  // the slice before has been read
      base = (s * ctas + rank) * slice;
      set_limits();
      load();
      if (manager)
        for (unsigned i = tid; i < slice / 16; i += L) reinterpret_cast<uint4*>(bits)[i] = make_uint4(0, 0, 0, 0);
    }
    copies_done();
    __syncthreads();
    if (manager) {  // the list's values; a position that is marked already is listed twice
      for (unsigned e = tid; e < k; e += L) {
        const unsigned p = e_index[e] + row.lead - base * P;
        if (e_index[e] == ~0u || p >= slice * P) continue;
        const uint32_t bit = 1u << ((p / P & 3) * 8 + p % P);
        twice |= (atomicOr(bits + (p / P >> 2), bit) & bit) != 0;
        e_z[e] = as_float(reinterpret_cast<const T*>(held)[p]);
      }
      twice = __any_sync(0xffffffffu, twice);
      __syncwarp();
      if (tail)  // what is listed leaves the slice
        for (unsigned e = tid; e < k; e += L) {
          const unsigned p = e_index[e] + row.lead - base * P;
          if (e_index[e] != ~0u && p < slice * P) reinterpret_cast<T*>(held)[p] = from_float<T>(-INFINITY);
        }
    }
    if (tail) __syncthreads();
    if (!manager && counts) {
      each(0, slice, [&](unsigned i) {
        const uint4 v[4] = {held[i], held[i + G], held[i + 2 * G], held[i + 3 * G]};
        const float m = fmaxf(part.m, fmaxf(fmaxf(word_max(v[0], T()), word_max(v[1], T())), fmaxf(word_max(v[2], T()), word_max(v[3], T()))));
        part = RestPart{m, part.s * shifted_exp(part.m, m, c) + words_sum<T>(v, m, c)};
      }, [&](unsigned i) {
        const uint4 v[1] = {held[i]};
        const float m = fmaxf(part.m, word_max(v[0], T()));
        part = RestPart{m, part.s * shifted_exp(part.m, m, c) + words_sum<T>(v, m, c)};
      });
    }
  }
  if (manager) {
    uint32_t most = 0;
    for (unsigned e = tid; e < k; e += L)
      if (e_index[e] != ~0u) most = max(most, key_of(e_z[e]));
    most = lanes_max<L>(most);
    list.m = most ? value_of(most) : -INFINITY;
    for (unsigned e = tid; e < k; e += L) {
      if (e_index[e] == ~0u) continue;
      const float z = e_z[e], u = e_w[e];
      const double arg = tail ? (double)u * a.inv_t - level : ((double)u - u_top) * a.inv_t, far = ((double)z - list.m) * a.inv_t;
      const double q = u == -INFINITY ? 0.0 : exp(arg);
      e_w[e] = (float)q;
      list.mass += q;
      if (!(q <= 0.0)) list.cross += z == -INFINITY ? INFINITY : q * (arg - far);  // a class of mass that the student rules out: infinite
      if (z != -INFINITY && owner(e)) list.s_listed += exp(far);
    }
    list = ListPart{lanes_sum<L>(list.s_listed), lanes_sum<L>(list.mass), lanes_sum<L>(list.cross), list.m, 0.f};
  } else {
    const float m = value_of(__reduce_max_sync(0xffffffffu, key_of(part.m)));
    part = RestPart{m, warp_sum(part.s * shifted_exp(part.m, m, c))};
  }

  // ---- from the warps, and the cluster's CTAs, to the manager
  if (ctas == 1) {
    if (!manager && lane == 0) rests[warp % WORKERS] = part;
    __syncthreads();
  } else {
    cluster.barrier_wait();  // every CTA of the cluster is there: its shared memory may be written
    if (lane < ctas) {
      if (manager) cluster.map_shared_rank(lists, lane)[rank] = list;
      else cluster.map_shared_rank(rests, lane)[rank * WORKERS + warp] = part;
    }
    cluster.sync();
  }
  float top = 0.f, share = 0.f, q_norm = 1.f;
  double rest = 0.0, mass = 0.0, total = 0.0, s_rest = 0.0;
  bool some = false;
  if (manager) {
    part = RestPart{-INFINITY, 0.f};
    if (ctas == 1) {  // every lane for itself
      RestPart p[WORKERS];
#pragma unroll
      for (int i = 0; i < WORKERS; ++i) {
        p[i] = rests[i];
        part.m = fmaxf(part.m, p[i].m);
      }
#pragma unroll
      for (int i = 0; i < WORKERS; ++i) part.s += p[i].s * shifted_exp(p[i].m, part.m, c);
    } else {
      for (unsigned i = tid; i < ctas * WORKERS; i += L) {  // one each, but for 8 CTAs of 8 workers
        const RestPart p = rests[i];
        const float m = fmaxf(part.m, p.m);
        part = RestPart{m, part.s * shifted_exp(part.m, m, c) + p.s * shifted_exp(p.m, m, c)};
      }
      const float m = value_of(lanes_max<L>(key_of(part.m)));
      part = RestPart{m, lanes_sum<L>(part.s * shifted_exp(part.m, m, c))};
    }
    if (ctas > 1) {  // a CTA's part per lane
      if (lane < ctas) list = lists[lane];
      else list = ListPart{0.0, 0.0, 0.0, -INFINITY, 0.f};
      const float m = value_of(lanes_max<L>(key_of(list.m)));
      const double down = list.m == m || list.m == -INFINITY ? 0.0 : ((double)list.m - m) * a.inv_t;
      if (down != 0.0) {
        list.s_listed *= exp(down);
        if (list.mass != 0.0) list.cross -= list.mass * down;
      }
      list = ListPart{lanes_sum<L>(list.s_listed), lanes_sum<L>(list.mass), lanes_sum<L>(list.cross), m, 0.f};
    }
    some = !(list.s_listed <= 0.0);   // a listed class that the student does not rule out
    mass = tail || list.mass == 0.0 ? list.mass : 1.0;
    // nothing outside the list but -infinity, or nothing at all: then no p_r is there to compare r with, and r counts as 0 in the loss
    // and in the gradient alike (of a list of all classes it is the sum's rounding)
    rest = tail && !(part.s <= 0.f) ? fmax(0.0, 1.0 - mass) : 0.0;
    top = tail && some ? fmaxf(part.m, list.m) : part.m;
    s_rest = part.s * shifted_exp(part.m, top, c);   // all, where there is no rest
    const double s_listed = !tail || !some ? 0.0 : list.m == top ? list.s_listed : list.s_listed * exp(((double)list.m - top) * a.inv_t);
    total = s_rest + s_listed;
    // ((mass + rest) p_r - rest) / s, p_r = s_rest / total: the difference, where digits cancel, in 64 bits, the division in 32, as the
    // exponentials that it is multiplied with are
    const float factor = part.s <= 0.f ? 0.f : __fdividef((float)(mass * s_rest - rest * s_listed), (float)total * part.s);
    if (tid == 0) *common = Common{part.m, factor};
  }
  __syncthreads();
  const float scale = w * a.grad_scale;

  // ---- the gradient: outside the list a multiple of 2^((x - m) c), in the list afterwards
  if (d_first) {
    const Common both = counts ? *common : Common{0.f, 0.f};
    const float factor = both.factor * scale;
    const Pair shift = minus(both.m), factors = pair_of(factor, factor);
    auto grad = [&](const uint4& v, float (&x)[P]) {
      unpack(v, x, T());
#pragma unroll
      for (int j = 0; j < P; j += 2) split(shifted_exp(x[j], x[j + 1], shift, cc) * factors, x[j], x[j + 1]);
    };
    const bool plain = a.same_lead;
    for (unsigned s = 0; s < (MULTI ? a.segments : 1u); ++s) {
      if (MULTI) {
        if (s > 0) __syncthreads();  // the slice before has been written
        base = (s * ctas + rank) * slice;
        set_limits();
        load();
        copies_done();
        __syncthreads();
      }
      if (!manager && plain) {
        uint4* const dst = d_row.word(base);
        if (counts) {
          auto word = [&](unsigned i, const uint4& old) {
            float x[P];
            grad(held[i], x);
            if constexpr (ADD) {
              float y[P];
              unpack(old, y, T());
#pragma unroll
              for (int j = 0; j < P; ++j) x[j] += y[j];
            }
            return pack(x, T());
          };
          auto before = [&](unsigned i) { return ADD ? dst[i] : uint4(); };
          each(lo, hi, [&](unsigned i) {  // all is read before anything is written: nothing tells the compiler that these differ
            const uint4 old[4] = {before(i), before(i + G), before(i + 2 * G), before(i + 3 * G)};
            const uint4 g[4] = {word(i, old[0]), word(i + G, old[1]), word(i + 2 * G, old[2]), word(i + 3 * G, old[3])};
#pragma unroll
            for (int j = 0; j < 4; ++j) dst[i + j * G] = g[j];
          }, [&](unsigned i) { dst[i] = word(i, before(i)); });
        } else if (!ADD) {
          for (unsigned i = tid < lo ? tid + G : tid; i < hi; i += G) dst[i] = make_uint4(0, 0, 0, 0);
        }
      } else if ((!manager || plain) && (counts || !ADD)) {
        // words that are not whole are the manager's; where the gradient starts elsewhere within 16 bytes, all words are the workers'
        auto by_element = [&](unsigned i) {
          float x[P] = {};
          if (counts) grad(held[i], x);
          if constexpr (ADD) {
#pragma unroll
            for (int j = 0; j < P; ++j) {
              const unsigned p = (base + i) * P + j;
              if (p >= row.lead && p < row.end) x[j] += as_float(d_first[p - row.lead]);
            }
          }
#pragma unroll
          for (int j = 0; j < P; ++j) {
            const unsigned p = (base + i) * P + j;
            if (p >= row.lead && p < row.end) d_first[p - row.lead] = from_float<T>(x[j]);
          }
        };
        if (!manager) {
          for (unsigned i = tid; i < end; i += G) by_element(i);
        } else {
          if (tid == 0 && lo) by_element(0);
          if (tid == 0 && hi < end) by_element(end - 1);
        }
      }
    }
  }
  if (manager) {
    share = total <= 0.0 ? 0.f : (float)(mass + rest) / (float)total;  // 0: a student of nothing but -infinity, p = 0
    q_norm = tail || list.mass == 0.0 ? 1.f : 1.f / (float)list.mass;
    if (there && rank == 0 && tid == 0) {
      double loss = 0.0;
      if (counts) {
        loss = tail || list.mass == 0.0 ? list.cross : list.cross / list.mass - log(list.mass);
        const double log_total = log(total);
        if (some) loss += mass * (((double)top - list.m) * a.inv_t + log_total);
        // p_r from the same s_rest as `total`: an error of one and not of the other would be all of a small divergence
        if (rest > 0.0)
          loss += rest * (s_rest > 0.0 ? log(rest / s_rest * total) : log(rest / part.s) + ((double)top - part.m) * a.inv_t + log_total);
      }
      a.row_loss[r] = (float)(loss * w);
    }
  }
  __syncthreads();
  if (!manager) return;
  if (d_first)
    for (unsigned e = tid; e < k; e += L) {
      if (!owner(e)) continue;
      float q = e_w[e];
      if (twice)
        for (unsigned i = e + 1; i < k; ++i)
          if (e_index[i] == e_index[e]) q += e_w[i];
      float g = scale * (shifted_exp(e_z[e], top, c) * share - q * q_norm);
      if (ADD) g += e_old[e];
      d_first[e_index[e]] = from_float<T>(g);
    }
  if (a.fold && rank == 0) {
    __syncwarp();
    double sum = lane < a.rows ? (double)a.row_loss[lane] : 0.0;
    sum = warp_sum(sum);
    if (lane == 0) *a.loss = (float)(sum / a.loss_div);
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

template <typename T, int ROWS, int WORKERS, int CTAS, bool MULTI, bool ADD>
static void launch_distill(cudaStream_t s, DistillArgs a, unsigned cluster) {
  static SharedMemoryLimit limit;
  const size_t smem = (size_t)distill_row_bytes(cluster, WORKERS, a.slice, a.k) * ROWS;
  const auto kernel = distill_kernel<T, ROWS, WORKERS, CTAS, MULTI, ADD>;
  if (smem > 48 * 1024 && !limit.raise(kernel, 227 * 1024)) return;
  const unsigned grid = (unsigned)((a.rows + ROWS - 1) / ROWS) * cluster;
  a.fold = grid == cluster;
  if (!launch_pdl_cluster(kernel, dim3(grid), dim3((ROWS * WORKERS + 1) * 32), smem, s, cluster, a)) return;
  if (!a.fold) launch_pdl(distill_loss_kernel, dim3(1), dim3(1024), 0, s, (const float*)a.row_loss, a.rows, a.loss_div, a.loss);
}

template <typename T, bool ADD>
static void launch_distill_rows(cudaStream_t s, DistillArgs a) {
  const unsigned words = (unsigned)most_words<T>(a.logits, a.C, a.ld);
  // A warp a row: 8192 x 4096 bf16 41 us, with 8 rows to a manager instead of 4 55, by a CTA a row 62.  A manager's eight lanes to a row
  // make long lists slow: 8192 x 1000 fp32 k 128 60 us and by a CTA a row 73, k 256 103 and 105; 8192 x 4000 bf16 k 128 73 and 79, k 256 138
  // and 113.  The rule does not look at the rows' number: of few rows with long lists a CTA each would be faster (8 x 1000 fp32 k 16 11 and
  // 13 us, k 128 22 and 15; 512 x 4000 bf16 k 16 13 and 13, k 128 26 and 15)
  if (words <= 32 * 16 && a.k <= kDShortList) {
    a.slice = (words + 31) / 32 * 32;
    return launch_distill<T, 4, 1, 6, false, ADD>(s, a, 1);
  }
  // A slice of 64 KB at most, of which an SM holds three; more CTAs to a row than that takes only while SMs would be idle
  // (777 x 50021 bf16 as two CTAs 45 us, as eight 75; 8192 x 16384 bf16 as one 102, as eight 588; 1024 x 65536 fp32 as four 125, as
  // eight 127).  Slices of 32 KB gain where they divide a row (4096 x 131072 bf16 as eight 434, as four 453) and lose elsewhere
  // (4096 x 100003 444 and 373).  Eight workers to a slice instead of four: 8192 x 16384 137 us
  constexpr unsigned kWorkers = 4, step = kWorkers * 32;
  const unsigned most = 64 * 64, widest = 184 * 64;  // words; what a CTA alone on its SM can hold
  unsigned cluster = 1;
  while (cluster < 8 && words > most * cluster) cluster *= 2;
  while (cluster < 8 && a.rows * cluster * 2 <= (size_t)sm_count() && words > step * cluster) cluster *= 2;
  if (words > widest * cluster) {
    a.slice = widest;
    a.segments = (words + a.slice * cluster - 1) / (a.slice * cluster);
    return launch_distill<T, 1, 8, 1, true, ADD>(s, a, cluster);
  }
  a.slice = ((words + cluster - 1) / cluster + step - 1) / step * step;
  // Six CTAs to an SM by their registers where shared memory allows it (8192 x 8192 bf16 73 us, with four 89; 8192 x 16384 103 and 116; longer rows
  // alike); adding, which has four more words in flight, four (4096 x 131072 bf16 766 us, with six 939; 1024 x 65536 fp32 226 and 232; above, four
  // rows to a CTA, 20000 x 200 fp32 44 with six, 56 with four)
  launch_distill<T, 1, kWorkers, ADD ? 4 : 6, false, ADD>(s, a, cluster);
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
  if (rows > (len_t)0x0fffffff) { set_error(kBadArgument, "%s: rows %lu", me, rows); return; }
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
  a.loss = (float*)loss_out; a.row_loss = (float*)row_loss;
  a.same_lead = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(dlogits)) % 16 == 0;
  a.slice = 0; a.segments = 1; a.fold = 0;
  const bool add = dlogits && accumulate;
  if (id == SINGLE) add ? launch_distill_rows<float, true>(s, a) : launch_distill_rows<float, false>(s, a);
  else add ? launch_distill_rows<__nv_bfloat16, true>(s, a) : launch_distill_rows<__nv_bfloat16, false>(s, a);
}
