// Verification of drafted tokens against the target model's probabilities, from given random numbers (include/zg_b200.h:
// zg_verify_drafts): which of a sequence's drafts stand, and the token that follows them.
//
// Draft i stands while u_i q_i(d_i) < p_i(d_i); behind the last one that does, a token is drawn from w = max(p - q, 0) (from p
// where all drafts stand): the first index whose running sum of w exceeds u sum(w).  A token's probability is then p's whatever
// q is.  Products of two fp32 values and, in 64 bits, differences and sums of them make the comparisons exact or nearly so:
// over 131072 classes (softmaxes of normal values) running sums in fp32 place one draw in ten on another class, sums of 256 that
// are then added up one in a hundred and fifty.
//
// What has to be read are two values per draft and two rows per sequence.  A cluster of CTAs shares a sequence; each warp sums
// a contiguous part, all look up in which part the random share falls, and the CTA that holds it goes on
// into eighths of it until a warp has the 256 elements in which to find the place.
//
// 256 sequences of 131072 fp32 classes, 7 drafts: 268 MB in 61 us with a cold L2.  What it waits for is memory: two loads of each
// operand in flight per thread, half the warps an SM can hold.
#include "row_access.cuh"

namespace zg {

using namespace ra;

constexpr int kVThreads = 256;
constexpr int kVWarps = kVThreads / 32;
constexpr unsigned kVMostCtas = 8;

struct VerifyArgs {
  const void* target;     // [batch, drafts + 1, ld_target]
  const void* draft;      // [batch, drafts, ld_draft] or nullptr: the drafted token has probability 1
  const len_t* tokens;    // [batch, drafts]
  const len_t* lengths;   // [batch] or nullptr
  const float* uniforms;  // [batch, drafts + 1]
  size_t batch, drafts, ld_target, ld_draft;
  unsigned C;
  len_t* out;             // [batch, drafts + 1]
  len_t* accepted;        // [batch]
};

// The weight of class e: what the target gives it beyond what the draft did.  The difference of two fp32 values is taken in 64
// bits, where it is nearly always exact; a NaN is not above anything and counts nothing.
template <typename T>
struct Weight {
  const T* p;
  const T* q;       // nullptr: none
  unsigned without; // a class that counts nothing, or ~0
  // (Two ways to say the same: 256 sequences of 131072 take 61 us by the first and 68 by the second in fp32, 51 and 45 in bf16.)
  static __device__ __forceinline__ double beyond(float p, float q) {
    const double d = (double)p - (double)q;
    return sizeof(T) == 4 ? fmax(d, 0.0) : p > q ? d : 0.0;
  }
  __device__ __forceinline__ double operator()(unsigned e) const {
    return e == without ? 0.0 : beyond(as_float(p[e]), q ? as_float(q[e]) : 0.f);
  }
  // sum over lo .. hi - 1, lo a multiple of 32, by the lanes of a warp; all have it in the end
  __device__ __forceinline__ double sum(unsigned lo, unsigned hi) const {
    constexpr int P = kPerWord<T>;
    const unsigned lane = threadIdx.x & 31;
    double s = 0.0;
    unsigned e = lo + lane;
    if (((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & 15) == 0) {  // whole words of both
      const unsigned words = (hi - lo) / P;
      const uint4 *pw = reinterpret_cast<const uint4*>(p + lo), *qw = reinterpret_cast<const uint4*>(q + lo);
      constexpr int U = 2;  // 256 x 131072 fp32 61 us, with four words in flight 76
      double sums[U] = {};  // additions that do not wait for one another
      for (unsigned w = lane; w < words; w += U * 32) {
        uint4 a[U], b[U];
#pragma unroll
        for (int j = 0; j < U; ++j) a[j] = w + j * 32 < words ? __ldcs(pw + w + j * 32) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < U; ++j) b[j] = q && w + j * 32 < words ? __ldcs(qw + w + j * 32) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < U; ++j) {
          float x[P], y[P];
          unpack(a[j], x, T());
          unpack(b[j], y, T());
          const unsigned first = lo + (w + j * 32) * P;
#pragma unroll
          for (int i = 0; i < P; ++i) sums[j] += first + i == without ? 0.0 : beyond(x[i], y[i]);
        }
      }
      s = sums[0] + sums[1];
      e = lo + words * P + lane;
    }
    for (; e + 7 * 32 < hi; e += 8 * 32) {
      T a[8], b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = __ldcs(p + e + 32 * i);
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] = q ? __ldcs(q + e + 32 * i) : from_float<T>(0.f);
      double sums[2] = {};
#pragma unroll
      for (int i = 0; i < 8; ++i) sums[i & 1] += e + 32 * i == without ? 0.0 : beyond(as_float(a[i]), as_float(b[i]));
      s += sums[0] + sums[1];
    }
    for (; e < hi; e += 32) s += (*this)(e);
    return warp_sum(s);
  }
};

// Of n <= 64 parts' sums: the first whose running sum exceeds `share`, the last positive one where none does; -1 where there is
// none.  `before` becomes the sum in front of it.  All lanes of a warp.
__device__ __forceinline__ int find_part(const double* sums, unsigned n, double share, double& before) {
  const unsigned lane = threadIdx.x & 31, i = 2 * lane;
  const double a = i < n ? sums[i] : 0.0, b = i + 1 < n ? sums[i + 1] : 0.0;
  double up = a + b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double v = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= (unsigned)o) up += v;
  }
  double down = __shfl_up_sync(0xffffffffu, up, 1);
  if (lane == 0) down = 0.0;
  const unsigned over = __ballot_sync(0xffffffffu, up > share && a + b > 0.0), some = __ballot_sync(0xffffffffu, a + b > 0.0);
  if (!some) return -1;
  const int at = over ? __ffs(over) - 1 : 31 - __clz(some);
  const double sa = __shfl_sync(0xffffffffu, a, at), sb = __shfl_sync(0xffffffffu, b, at);
  before = __shfl_sync(0xffffffffu, down, at);
  const bool second = sb > 0.0 && !(sa > 0.0 && before + sa > share);
  if (second) before += sa;
  return 2 * at + second;
}

template <typename T>
__global__ void __launch_bounds__(kVThreads, 4) verify_drafts_kernel(const VerifyArgs a) {
  __shared__ double sums[2][kVMostCtas * kVWarps];
  __shared__ double inner[2][kVWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned n_parts = ctas * kVWarps;
  if (ctas > 1) cluster.barrier_arrive();
  pdl_sync();
  if (ctas > 1) cluster.barrier_wait();
  unsigned parity = 0;
  for (size_t b = blockIdx.x / ctas; b < a.batch; b += gridDim.x / ctas) {
    const size_t n = a.drafts;
    const size_t length = a.lengths && a.lengths[b] < n ? a.lengths[b] : n;
    const T* target = static_cast<const T*>(a.target) + b * (n + 1) * a.ld_target;
    const T* draft = a.draft ? static_cast<const T*>(a.draft) + b * n * a.ld_draft : nullptr;
    const len_t* tokens = a.tokens + b * n;
    const float* u = a.uniforms + b * (n + 1);
    // ---- how many drafts stand: every warp finds out for itself
    size_t stand = 0;
    while (stand < length) {
      const size_t i = stand + lane;
      bool ok = false;
      if (i < n) {  // whether or not it is one of the sequence's: nothing waits for its length
        const len_t d = tokens[i];
        if (d < a.C) {
          const float q = draft ? as_float(draft[i * a.ld_draft + d]) : 1.f;
          ok = (double)u[i] * q < (double)as_float(target[i * a.ld_target + d]);
        }
      }
      ok &= i < length;
      const unsigned all = __ballot_sync(0xffffffffu, ok);
      stand += all == 0xffffffffu ? 32 : __ffs(~all) - 1;
      if (all != 0xffffffffu) break;
    }
    // ---- the sums of the weights
    Weight<T> w{target + stand * a.ld_target, nullptr, ~0u};
    if (stand < length) {
      if (draft) w.q = draft + stand * a.ld_draft;
      else if (tokens[stand] < a.C) w.without = (unsigned)tokens[stand];
    }
    const unsigned part = ((a.C + n_parts - 1) / n_parts + 31) / 32 * 32;
    int at;
    double share, before = 0.0;
    for (;;) {
      const unsigned g = rank * kVWarps + warp;
      const size_t lo = (size_t)g * part, hi = lo + part;
      const double s = lo < a.C ? w.sum((unsigned)lo, (unsigned)(hi < a.C ? hi : a.C)) : 0.0;
      double* all = sums[parity];
      parity ^= 1;
      if (ctas == 1) {
        if (lane == 0) all[g] = s;
        __syncthreads();
      } else {
        if (lane < ctas) cluster.map_shared_rank(all, lane)[g] = s;
        cluster.sync();
      }
      double total = 0.0;
      for (unsigned i = lane; i < n_parts; i += 32) total += all[i];
      total = warp_sum(total);
      share = (double)u[n] * total;
      at = find_part(all, n_parts, share, before);
      if (at >= 0 || (!w.q && w.without == ~0u)) break;
      w.q = nullptr;  // nothing beyond the draft's probabilities: the target's own
      w.without = ~0u;
    }
    // ---- the place, by the CTA that holds it
    const bool here = at < 0 ? rank == 0 : (unsigned)at / kVWarps == rank;
    if (here) {
      len_t token = ZG_NO_TOKEN;
      if (at >= 0) {
        size_t lo = (size_t)at * part, hi = lo + part < a.C ? lo + part : a.C;
        share -= before;
        for (unsigned k = 0; hi - lo > 256; ++k) {
          const size_t piece = ((hi - lo + kVWarps - 1) / kVWarps + 31) / 32 * 32;
          const size_t from = lo + warp * piece, to = from + piece < hi ? from + piece : hi;
          const double s = from < hi ? w.sum((unsigned)from, (unsigned)to) : 0.0;
          if (lane == 0) inner[k & 1][warp] = s;
          __syncthreads();
          const int i = find_part(inner[k & 1], kVWarps, share, before);
          share -= before;
          lo += i * piece;
          if (lo + piece < hi) hi = lo + piece;
        }
        if (warp == 0) {
          double v[8], mine = 0.0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const size_t e = lo + lane * 8 + i;
            v[i] = e < hi ? w((unsigned)e) : 0.0;
            mine += v[i];
          }
          double up = mine;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double x = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= (unsigned)o) up += x;
          }
          const unsigned over = __ballot_sync(0xffffffffu, up > share && mine > 0.0), some = __ballot_sync(0xffffffffu, mine > 0.0);
          const unsigned winner = over ? __ffs(over) - 1 : 31 - __clz(some);
          if (lane == winner) {
            double run = up - mine;
            bool done = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              run += v[i];
              if (v[i] > 0.0 && !done) {  // the last positive one, if rounding leaves none above the share
                token = lo + lane * 8 + i;
                done = run > share;
              }
            }
            a.out[b * (n + 1) + stand] = token;
          }
        }
        __syncthreads();  // `inner` is free
      } else if (threadIdx.x == 0) {
        a.out[b * (n + 1) + stand] = token;
      }
    }
    if (rank == 0) {
      if (threadIdx.x == 0) a.accepted[b] = stand;
      for (size_t i = threadIdx.x; i <= n; i += kVThreads)
        if (i != stand) a.out[b * (n + 1) + i] = i < stand ? tokens[i] : ZG_NO_TOKEN;
    }
  }
}

template <typename T>
static void launch_verify(cudaStream_t s, const VerifyArgs& a) {
  // four CTAs per SM where there are few sequences: 256 of 131072 fp32 by one CTA each 78 us, by two 61; one of
  // 32768 by one CTA 25, by eight 12
  unsigned cluster = 1;
  while (cluster < kVMostCtas && a.batch * cluster * 2 <= (size_t)sm_count() * 4 && a.C > kVThreads * 8 * cluster) cluster *= 2;
  const size_t most = (size_t)1 << 20;  // a CTA or cluster goes on to the next sequence where there are more
  launch_pdl_cluster(verify_drafts_kernel<T>, dim3((unsigned)(a.batch < most ? a.batch : most) * cluster), dim3(kVThreads), 0, s, cluster, a);
}

}  // namespace zg

using namespace zg;

extern "C" void zg_verify_drafts(dtype id, StreamWrapper w, const void* target, const void* draft, const len_t* tokens, const len_t* lengths,
                                 const void* uniforms, len_t batch, len_t drafts, len_t C, len_t ld_target, len_t ld_draft, len_t* tokens_out,
                                 len_t* accepted_out) {
  const char* me = "zg_verify_drafts";
  if (id != SINGLE && id != BF16) { set_error(kUnsupported, "%s: probabilities are SINGLE or BF16", me); return; }
  if (ld_target == 0) ld_target = C;
  if (ld_draft == 0) ld_draft = C;
  if (C == 0 || C > (len_t)0x7fffffff || ld_target < C || ld_draft < C) { set_error(kBadArgument, "%s: C %lu, ld_target %lu, ld_draft %lu", me, C, ld_target, ld_draft); return; }
  if (drafts > (len_t)0x7fffffff || batch > (len_t)0x7fffffff) { set_error(kBadArgument, "%s: batch %lu, drafts %lu", me, batch, drafts); return; }
  if (batch == 0) return;
  if (!target || !uniforms || !tokens_out || !accepted_out || (drafts && !tokens)) { set_error(kBadArgument, "%s: a required operand is NULL", me); return; }
  const size_t size = id == BF16 ? 2 : 4;
  const auto off = [](const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
  if (off(target, size) || off(draft, size) || off(tokens, 8) || off(lengths, 8) || off(uniforms, 4) || off(tokens_out, 8) || off(accepted_out, 8)) {
    set_error(kBadArgument, "%s: an operand is not aligned to its elements", me);
    return;
  }
  VerifyArgs a;
  a.target = target; a.draft = draft; a.tokens = tokens; a.lengths = lengths; a.uniforms = (const float*)uniforms; a.batch = batch; a.drafts = drafts;
  a.ld_target = ld_target; a.ld_draft = ld_draft; a.C = (unsigned)C; a.out = tokens_out; a.accepted = accepted_out;
  if (id == SINGLE) launch_verify<float>(as_stream(w), a);
  else launch_verify<__nv_bfloat16>(as_stream(w), a);
}
