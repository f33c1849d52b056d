// Operators on a language model's logits [rows][vocabulary] (f32, bf16 or f16): log probabilities of given tokens with
// entropy and top alternatives, distillation from a teacher's top logits, and their gradients.  They have no
// counterpart in the reference; they stand beside its cross entropy (engine/src/operations/loss/regression.rs:178-251).
// Every call is one or two launches, allocates nothing and keeps nothing between calls: statistics that a backward
// call needs are the caller's.  Formulas, arithmetic and conventions: vocab_rows.cuh.
// Times in the comments are of short runs of one call, at an SM clock of 1.965 GHz; under a sustained load the 1000 W cap leaves
// 1.5 to 1.7 GHz, where calls with one exponential per 2 bytes or two per element take up to 20 % longer.
#include "vocab_rows.cuh"

#include <algorithm>
#include <cmath>

namespace mtb {

// ------------------------------------------------------------------ arguments read by type
struct IndexArray {  // class or vocabulary indices, int32 or int64
  const void* p;
  int wide;
  __device__ __forceinline__ long long at(long long i) const {
    return wide ? static_cast<const long long*>(p)[i] : static_cast<long long>(static_cast<const int*>(p)[i]);
  }
};
struct RealArray {  // f32, f16 or bf16 values
  const void* p;
  int dtype;
  __device__ __forceinline__ float at(long long i) const {
    if (dtype == MTB200_F32) return static_cast<const float*>(p)[i];
    if (dtype == MTB200_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  }
};

struct ScoreArgs {
  const void* logits;
  long long ld;
  int rows, vocab, top, parts;
  IndexArray tokens;  // p == nullptr: none given
  int has_ignore;
  long long ignore;
  float inv_t, c;     // 1 / T and log2(e) / T
  float *log_probs, *entropy, *top_log_probs, *stats;
  int* top_indices;
  uint32_t* bad_label;
};

constexpr int MAX_PARTS = 8;  // blocks of a portable cluster

// A block works on one part of one row, or, where rows are short, each of its warps on a row of its own.
template <int G>
struct Block {
  static constexpr int ROWS = G == 32 ? 8 : 1;
  static constexpr int THREADS = G * ROWS;
  static __device__ __forceinline__ int slot() { return G == 32 ? threadIdx.x >> 5 : 0; }
  // row index, or -1 behind the last one (then the whole group has nothing to do)
  static __device__ __forceinline__ long long row(int rows, int parts) {
    const long long r = G == 32 ? static_cast<long long>(blockIdx.x) * ROWS + slot() : blockIdx.x / static_cast<unsigned>(parts);
    return r < rows ? r : -1;
  }
  static __device__ __forceinline__ int part(int parts) { return G == 32 ? 0 : blockIdx.x % static_cast<unsigned>(parts); }
};

// The same for kernels whose blocks do not meet: `whole` rows with a block each, then the others in `parts` parts.
template <int G>
struct Cut {
  int row;  // -1: nothing to do
  int part, parts;
  __device__ __forceinline__ Cut(int rows, int whole, int cut_parts) {
    const unsigned unit = G == 32 ? blockIdx.x * Block<G>::ROWS + Block<G>::slot() : blockIdx.x;
    if (unit < static_cast<unsigned>(whole)) {
      row = unit;
      part = 0;
      parts = 1;
    } else {
      const unsigned more = unit - whole;
      row = whole + static_cast<int>(more / static_cast<unsigned>(cut_parts));
      part = more % static_cast<unsigned>(cut_parts);
      parts = cut_parts;
      if (row >= rows) row = -1;
    }
  }
};

constexpr float LN2 = 0.693147180559945309f;
constexpr float LOG2E = 1.442695040888963407f;

// ------------------------------------------------------------------ token log probabilities
template <bool TOP, bool ENT>
__device__ __forceinline__ void put_left_out(const ScoreArgs& a, long long r, int tid, int threads) {
  if (tid == 0) {
    a.log_probs[r] = 0.0f;
    if (ENT) a.entropy[r] = 0.0f;
    a.stats[2 * r] = -INFINITY;
    a.stats[2 * r + 1] = 0.0f;
  }
  if (TOP)
    for (int i = tid; i < a.top; i += threads) {
      a.top_log_probs[r * a.top + i] = -INFINITY;
      a.top_indices[r * a.top + i] = -1;
    }
}
// A row's results from its statistics.
template <bool ENT>
struct RowOut {
  long long r;
  RowStat st;
  bool none;  // no distribution
  float ln_s;
  __device__ __forceinline__ RowOut(const ScoreArgs& a, long long row, const RowStat& stat) : r(row), st(stat) {
    none = st.m == -INFINITY && !isnan(st.s);
    ln_s = none ? 0.0f : logf(st.s);
  }
  __device__ __forceinline__ void put_scores(const ScoreArgs& a, float x_token, bool good) const {
    if (a.log_probs) a.log_probs[r] = none && good ? -INFINITY : (x_token - st.m) * a.inv_t - ln_s;
    if (ENT) a.entropy[r] = none ? 0.0f : ln_s - a.inv_t * (st.u / st.s);
    a.stats[2 * r] = st.m;
    a.stats[2 * r + 1] = ln_s;
  }
  __device__ __forceinline__ void put_top(const ScoreArgs& a, int at, unsigned long long w) const {
    a.top_log_probs[r * a.top + at] = none ? -INFINITY : (key_value(candidate_key(w)) - st.m) * a.inv_t - ln_s;
    a.top_indices[r * a.top + at] = candidate_index(w);
  }
};

// A cluster of `parts` blocks per row (one block when there are rows enough, a warp for short rows).  One pass over the
// logits: HBM-bound.  Registers decide how many blocks share an SM: 1536 threads of 40 registers without the selection; with
// it 1024, whose 64 registers keep the four loads of a round together.
template <typename T, int G, bool TOP, bool ENT>
static __global__ void __launch_bounds__(Block<G>::THREADS, (TOP ? 1024 : 1536) / Block<G>::THREADS) token_scores_kernel(ScoreArgs a) {
  using L = LogitType<T>;
  extern __shared__ __align__(16) unsigned char dynamic_smem[];
  __shared__ RowStat sm[Group<G>::WARPS + 1], parts_st[MAX_PARTS];
  TopScratch<G>& ts = reinterpret_cast<TopScratch<G>*>(dynamic_smem)[Block<G>::slot()];  // with TOP
  unsigned long long* lists = reinterpret_cast<unsigned long long*>(dynamic_smem + sizeof(TopScratch<G>));  // [parts][top]
  cg::cluster_group cluster = cg::this_cluster();
  const int part = Block<G>::part(a.parts);
  const long long r = Block<G>::row(a.rows, a.parts);
  const int tid = Group<G>::rank();
  if (r < 0) return;
  const T* row = static_cast<const T*>(a.logits) + r * a.ld;

  long long token = -1;
  bool good = true;
  if (a.tokens.p) {
    token = a.tokens.at(r);
    if (a.has_ignore && token == a.ignore) {  // the whole cluster leaves
      if (part == 0) put_left_out<TOP, ENT>(a, r, tid, G);
      return;
    }
    good = token >= 0 && token < a.vocab;
    if (!good && part == 0 && tid == 0) atomicOr(a.bad_label, 1u);
  }
  const bool split = G > 32 && a.parts > 1;
  if (split) cluster.barrier_arrive();  // waited for before the first block's memory is written to
  float x_token = 0.0f;
  if (part == 0 && tid == 0 && a.tokens.p) x_token = good ? L::up(row[token]) : NAN;

  const RowPart<T> p = row_part(row, a.vocab, part, a.parts);
  const UnitStat unit = unit_stats<T, G, ENT, TOP>(p, a.c, ts.slots);
  RowStat st = group_merge<G>(unit.sum(), a.c, sm);
  if constexpr (TOP) select_top<T, G>(p, a.top, unit.m, unit.where, ts);
  if (split) {
    cluster.barrier_wait();
    if (tid == 0) *cluster.map_shared_rank(&parts_st[part], 0) = st;
    if constexpr (TOP)
      for (int i = tid; i < a.top; i += G) cluster.map_shared_rank(lists, 0)[part * a.top + i] = ts.best[i];
    cluster.sync();
    if (part) return;
    st = parts_merge(parts_st, a.parts, a.c);
  }
  const RowOut<ENT> out(a, r, st);
  if (tid == 0) out.put_scores(a, x_token, good);
  if constexpr (TOP) {
    if (!split) {
      for (int i = tid; i < a.top; i += G) out.put_top(a, i, ts.best[i]);
    } else {
      // The parts' sorted lists together hold at least `top` entries at or above the least of their
      // ceil(top / parts)-th ones; those that reach it are counted against each other.
      const int nth = (a.top + a.parts - 1) / a.parts - 1;
      unsigned long long bound = ~0ull;
      for (int q = 0; q < a.parts; ++q) bound = min(bound, lists[q * a.top + nth]);
      if (tid == 0) ts.pool_count = 0;
      Group<G>::sync();
      for (int i = tid; i < a.parts * a.top; i += G) {  // at most 8 * 256 words
        const unsigned long long w = lists[i];
        if (w && w >= bound) ts.pool[atomicAdd(&ts.pool_count, 1)] = w;
      }
      Group<G>::sync();
      for_each_rank<G>(ts.pool, ts.pool_count, [&](int i, int above) {
        if (above < a.top) out.put_top(a, above, ts.pool[i]);
      });
    }
  }
}

struct ScoreGradArgs {
  const void* logits;
  void* dlogits;
  long long ld, ld_grad;
  int rows, vocab, top, parts, whole, same_phase;
  IndexArray tokens;
  int has_ignore;
  long long ignore;
  float inv_t, c;
  const float *stats, *entropy, *d_log_probs, *d_entropy, *d_top;
  const int* top_indices;
  uint32_t* bad_label;
};

// Blocks of a gradient kernel on an SM, which limit its registers: warps on 20000 x 1000 f32 with the entropy's gradient take 55 us
// in four blocks and 63 in the three that fit without a limit, 20000 x 2000 bf16 without it 55 and 64.  128 threads keep to the
// eight or nine blocks that they just miss or just reach without one (4096 x 8000 f32: 59.5 us either way).  In 16 bits the
// entropy's gradient needs 80 registers and more, and has them.
template <typename T, int G, bool ENT>
constexpr int grad_blocks() {
  return G == 512 ? 4 : sizeof(T) == 2 && ENT ? 1 : G == 32 ? 4 : sizeof(T) == 4 && !ENT ? 9 : 8;
}

// dx = (1/T) [ sum of weights at given indices - p (sum of all weights) - g_H p (log p + H) ], one read, one write.
template <typename T, int G, bool ENT>
static __global__ void __launch_bounds__(Block<G>::THREADS, grad_blocks<T, G, ENT>()) token_scores_grad_kernel(ScoreGradArgs a) {
  __shared__ __align__(16) int all_idx[Block<G>::ROWS][VOCAB_TOP_MAX + 4];
  __shared__ float all_weight[Block<G>::ROWS][VOCAB_TOP_MAX + 1];
  __shared__ float fold[Group<G>::WARPS];
  int* idx = all_idx[Block<G>::slot()];
  float* weight = all_weight[Block<G>::slot()];
  const Cut<G> cut(a.rows, a.whole, a.parts);
  const int part = cut.part;
  const int r = cut.row;
  const int tid = Group<G>::rank();
  if (r < 0) return;
  const T* row = static_cast<const T*>(a.logits) + static_cast<long long>(r) * a.ld;
  T* dx = static_cast<T*>(a.dlogits) + static_cast<long long>(r) * a.ld_grad;
  const RowPart<T> p = row_part(row, a.vocab, part, cut.parts);
  const long long token = a.tokens.p ? a.tokens.at(r) : -1;
  if (a.tokens.p && a.has_ignore && token == a.ignore) {
    zero_grad<T, G>(p, dx, a.same_phase);
    return;
  }
  const bool good = token >= 0 && token < a.vocab;
  if (a.tokens.p && !good && part == 0 && tid == 0) atomicOr(a.bad_label, 1u);
  const int n = a.top + 1;
  float sum = 0.0f;
  for (int e = tid; e < n; e += G) {
    int j;
    float w;
    if (e == 0) {
      j = good && a.d_log_probs ? static_cast<int>(token) : -1;
      w = j >= 0 ? a.d_log_probs[r] : 0.0f;
    } else {
      j = a.top_indices[static_cast<long long>(r) * a.top + e - 1];
      if (j < 0 || j >= a.vocab) {  // -1: no entry
        if (j >= a.vocab) atomicOr(a.bad_label, 1u);
        j = -1;
      }
      w = j >= 0 ? a.d_top[static_cast<long long>(r) * a.top + e - 1] : 0.0f;
    }
    idx[e] = j;
    weight[e] = w * a.inv_t;
    sum += w;
  }
  fill_list<G>(idx, n);
  sum = group_fold<G, false>(sum, fold);
  RowGrad g;
  const float m = a.stats[2 * r];
  g.base = m == -INFINITY ? 0.0f : m;
  g.l2 = a.stats[2 * r + 1] * LOG2E;
  const float gh = ENT ? a.d_entropy[r] : 0.0f;
  g.b = -gh * a.inv_t * LN2;
  g.a = -a.inv_t * (sum + (ENT ? gh * a.entropy[r] : 0.0f));
  dense_grad<T, G, ENT>(p, dx, a.c, g, a.same_phase);
  Group<G>::sync();
  sparse_fix<T, G, ENT>(p, dx, a.c, g, idx, weight, n);
}

// ------------------------------------------------------------------ distillation
struct DistillArgs {
  const void* logits;
  void* dlogits;           // forward: nullptr = loss only
  long long ld, ld_grad;
  int rows, vocab, top, parts, whole, same_phase;
  IndexArray index;
  RealArray value;
  float c, t;
  float scale;             // T * reduction factor * upstream: d loss / d logits = scale * weight_r * (Q p - q)
  const float* upstream_rows;
  float *row_loss, *stats;
  uint32_t *status, *bad_label;
};

constexpr int TEACHER_WARP_MAX = 128;  // entries where a warp has a row of its own: 12 KB a block
template <int G>
constexpr int TEACHER_ROOM = G == 32 ? TEACHER_WARP_MAX : VOCAB_TEACHER_MAX;

// The teacher's entries of row r into shared memory: q over the entries with an index in [0, vocab) (0 elsewhere,
// index -1), softmax of value / T, and (nullable) dv = value - largest value.  Returns whether the row has any entry;
// ln_s: log q = dv / T - ln_s (NaN if a value is NaN or +inf).
template <int G>
__device__ __forceinline__ bool load_teacher(const DistillArgs& a, long long r, bool report, int* idx, float* q, float* dv,
                                             float* fold, float* ln_s) {
  const int tid = Group<G>::rank();
  float top = -INFINITY;
  bool any = false;
  for (int e = tid; e < a.top; e += G) {
    const long long j = a.index.at(r * a.top + e);
    const bool in = j >= 0 && j < a.vocab;
    if (!in && j != -1 && report) atomicOr(a.bad_label, 1u);
    idx[e] = in ? static_cast<int>(j) : -1;
    q[e] = in ? a.value.at(r * a.top + e) : -INFINITY;
    top = fmaxf(top, q[e]);
    any = any || (in && q[e] != -INFINITY);  // NaN counts: it has to reach the result
  }
  fill_list<G>(idx, a.top);  // TEACHER_ROOM is a multiple of four
  any = G == 32 ? __any_sync(0xffffffffu, any) : Group<G>::count(any) > 0;
  if (!any) return false;
  top = group_fold<G, true>(top, fold);
  const float base = top == -INFINITY ? 0.0f : top;
  float s = 0.0f;
  for (int e = tid; e < a.top; e += G) {
    const float d = q[e] - base;
    const float w = ex2_ftz(d * a.c);
    s += w;
    q[e] = w;
    if (dv) dv[e] = d;
  }
  s = group_fold<G, false>(s, fold);
  const float inv = 1.0f / s;
  for (int e = tid; e < a.top; e += G) q[e] *= inv;
  *ln_s = logf(s);
  Group<G>::sync();
  return true;
}

// The row's gradient, for the second look at the row: the compiler is kept from computing the address before the first look,
// where its two registers are not to be had (1021 x 50257 f32 with 100 entries 102 us instead of 107, 300 x 50257 bf16 with 700
// entries 77 instead of 86).
template <typename T>
__device__ __forceinline__ T* grad_row_late(const DistillArgs& a, int r) {
  asm volatile("" : "+r"(r));
  return static_cast<T*>(a.dlogits) + static_cast<long long>(r) * a.ld_grad;
}

// Loss per row, T^2 sum_k q_k (log q_k - log p_idx_k), and with GRAD the gradient: the row's statistics, then a second
// look at the row while it is in L2.  Warps keep to five blocks on an SM (20000 x 1000 f32: 48 us, 53 in four).
template <typename T, int G, bool GRAD>
static __global__ void __launch_bounds__(Block<G>::THREADS, G == 32 && GRAD ? 5 : 0) distill_kernel(DistillArgs a) {
  using L = LogitType<T>;
  __shared__ RowStat sm[Group<G>::WARPS + 1], parts_st[MAX_PARTS];
  __shared__ __align__(16) int all_idx[Block<G>::ROWS][TEACHER_ROOM<G>];
  __shared__ float all_q[Block<G>::ROWS][TEACHER_ROOM<G>], all_dv[Block<G>::ROWS][TEACHER_ROOM<G>];
  __shared__ float fold[Group<G>::WARPS];
  int* idx = all_idx[Block<G>::slot()];
  float *q = all_q[Block<G>::slot()], *dv = all_dv[Block<G>::slot()];
  cg::cluster_group cluster = cg::this_cluster();
  const int part = Block<G>::part(a.parts);
  const int r = static_cast<int>(Block<G>::row(a.rows, a.parts));
  const int tid = Group<G>::rank();
  if (r < 0) return;
  const T* row = static_cast<const T*>(a.logits) + static_cast<long long>(r) * a.ld;
  const RowPart<T> p = row_part(row, a.vocab, part, a.parts);

  float ln_sq;
  if (!load_teacher<G>(a, r, part == 0, idx, q, dv, fold, &ln_sq)) {  // the same answer in every block of the cluster
    if (part == 0 && tid == 0) {
      a.row_loss[r] = 0.0f;
      if (a.stats) {
        a.stats[2 * r] = -INFINITY;
        a.stats[2 * r + 1] = 0.0f;
      }
    }
    if (GRAD) zero_grad<T, G>(p, grad_row_late<T>(a, r), a.same_phase);
    return;
  }
  const bool split = G > 32 && a.parts > 1;
  if (split) cluster.barrier_arrive();  // waited for before another block's memory is written to
  RowStat st = group_merge<G>(unit_stats<T, G, false, false>(p, a.c, nullptr).sum(), a.c, sm);
  if (split) {
    cluster.barrier_wait();
    if (tid < a.parts) *cluster.map_shared_rank(&parts_st[part], tid) = st;
    cluster.sync();
    st = parts_merge(parts_st, a.parts, a.c);
  }
  const bool none = st.m == -INFINITY && !isnan(st.s);
  const float ln_s = none ? 0.0f : logf(st.s);
  if (part == 0) {
    // log q - log p with the two maxima taken out first: nearly equal distributions lose nothing to the logarithms' size
    float kl = 0.0f;
    for (int e = tid; e < a.top; e += G) {
      if (idx[e] < 0 || q[e] == 0.0f) continue;
      const float dx = none ? -INFINITY : L::up(row[idx[e]]) - st.m;
      // T times the term, and T again on q: where T < 1, (dv - dx) / T or the sum without T may overflow
      kl += a.t * q[e] * (dv[e] - dx - a.t * (ln_sq - ln_s));
    }
    kl = group_fold<G, false>(kl, fold);
    if (tid == 0) {
      a.row_loss[r] = kl;
      if (a.stats) {
        a.stats[2 * r] = st.m;
        a.stats[2 * r + 1] = ln_s;
      }
    }
  }
  if constexpr (GRAD) {
    RowGrad g;
    g.base = st.m == -INFINITY ? 0.0f : st.m;
    g.l2 = ln_s * LOG2E;
    const float scale = a.upstream_rows ? a.scale * a.upstream_rows[r] : a.scale;
    g.a = isnan(ln_sq) ? NAN : scale;
    g.b = 0.0f;
    T* dx = grad_row_late<T>(a, r);
    dense_grad<T, G, false>(p, dx, a.c, g, a.same_phase);
    for (int e = tid; e < a.top; e += G) q[e] *= -scale;
    Group<G>::sync();
    sparse_fix<T, G, false>(p, dx, a.c, g, idx, q, a.top);
  }
}

// Loss and gradient of long rows: a cluster per row, so that the rows in flight stay in L2 between the two looks at them
// (2048 x 128256 f32: 398 us; with a block per row 493 us, as long as two reads and a write from HBM take).  Two
// exponentials per element and the meetings between the two looks bound it: what a row needs once is done by one warp,
// what its entries need by the warps that have entries (from the second on: thread 32 + e has entry e), and the parts
// exchange their statistics by messages instead of a cluster barrier, which would wait for all memory operations under way.
constexpr int CLUSTER_TEACHER = 480;  // entries
template <typename T>
static __global__ void __launch_bounds__(512, 3) distill_cluster_kernel(DistillArgs a) {
  using L = LogitType<T>;
  constexpr int G = 512, WARPS = Group<G>::WARPS;
  __shared__ RowStat stat_sm[WARPS], teacher_sm[WARPS];
  __shared__ float4 parts_st[MAX_PARTS], row_sm;  // row_sm: m, ln S, whether there is no distribution
  __shared__ __align__(8) unsigned long long arrived;
  __shared__ float kl_sm[WARPS], weight[CLUSTER_TEACHER];
  __shared__ int idx[CLUSTER_TEACHER], twice[CLUSTER_TEACHER];
  __shared__ uint32_t never;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, e = tid - 32;
  const bool entry = e >= 0 && e < a.top, entry_warp = warp > 0 && 32 * (warp - 1) < a.top;
  const int part = Block<G>::part(a.parts);
  const int r = static_cast<int>(Block<G>::row(a.rows, a.parts));
  const T* row = static_cast<const T*>(a.logits) + static_cast<long long>(r) * a.ld;
  const RowPart<T> p = row_part(row, a.vocab, part, a.parts);
  if (tid == 0) {
    mbar_init(smem_u32(&arrived), 1);
    fence_mbar_init();
    never = 0;
  }
  // The thread's entry.  The list is read before the logits are asked for: a row without an entry does not look at them.
  int mine = -1;
  float v = -INFINITY;
  if (entry) {
    const long long j = a.index.at(static_cast<long long>(r) * a.top + e);
    if (j >= 0 && j < a.vocab) mine = static_cast<int>(j);
    else if (j != -1 && part == 0) atomicOr(a.bad_label, 1u);
    if (mine >= 0) v = a.value.at(static_cast<long long>(r) * a.top + e);
    idx[e] = mine;
    twice[e] = 0;
  }
  const bool live = Group<G>::count(v != -INFINITY) > 0;  // NaN counts: it has to reach the result
  if (!live) {  // the same answer in every block of the cluster
    if (part == 0 && tid == 0) {
      a.row_loss[r] = 0.0f;
      if (a.stats) {
        a.stats[2 * r] = -INFINITY;
        a.stats[2 * r + 1] = 0.0f;
      }
    }
    zero_grad<T, G>(p, static_cast<T*>(a.dlogits) + static_cast<long long>(r) * a.ld_grad, a.same_phase);
    return;
  }
  if (a.parts > 1) cluster.barrier_arrive();  // waited for before another block is sent to
  const float scale = a.upstream_rows ? a.scale * a.upstream_rows[r] : a.scale;
  const bool owner = mine >= 0 && owns(p, mine);
  T x_mine = L::down(0.0f);
  if (mine >= 0 && (owner || part == 0)) x_mine = row[mine];

  const RowStat sum = warp_merge(unit_stats<T, G, false, false>(p, a.c, nullptr).sum(), a.c);
  if (lane == 0) stat_sm[warp] = sum;
  if (entry_warp) {
    const RowStat st = warp_merge(RowStat{isnan(v) ? -INFINITY : v, v == -INFINITY ? 0.0f : 1.0f + (v - v), 0.0f}, a.c);
    if (lane == 0) teacher_sm[warp] = st;
  }
  if (a.parts > 1) cluster.barrier_wait();
  __syncthreads();
  float q = 0.0f, dv = 0.0f, ln_sq = 0.0f;
  if (warp == 0) {
    RowStat st = warp_merge(lane < WARPS ? stat_sm[lane] : RowStat{-INFINITY, 0.0f, 0.0f}, a.c);
    if (a.parts > 1) {
      if (lane == 0) mbar_expect_tx(smem_u32(&arrived), uint32_t(a.parts) * 16u);
      if (lane < a.parts) send_async(&parts_st[part], &arrived, lane, make_float4(st.m, st.s, 0.0f, 0.0f));
      if (!mbar_wait(smem_u32(&arrived), 0, &never)) atomicMax(a.status, 0x1001u);
      const float4 o = parts_st[lane < a.parts ? lane : 0];
      st = warp_merge(lane < a.parts ? RowStat{o.x, o.y, 0.0f} : RowStat{-INFINITY, 0.0f, 0.0f}, a.c);
    }
    const bool none = st.m == -INFINITY && !isnan(st.s);
    if (lane == 0) row_sm = make_float4(st.m, none ? 0.0f : logf(st.s), none ? 1.0f : 0.0f, 0.0f);
  } else if (entry_warp) {
    const bool used = lane > 0 && lane < WARPS && 32 * (lane - 1) < a.top;
    const RowStat st = warp_merge(used ? teacher_sm[lane] : RowStat{-INFINITY, 0.0f, 0.0f}, a.c);
    dv = v - (st.m == -INFINITY ? 0.0f : st.m);
    q = ex2_ftz(dv * a.c) / st.s;
    ln_sq = logf(st.s);
    if (entry) weight[e] = -scale * q;
  }
  {
    // Entries whose index stands in the list more than once (1: behind, 2: before), all threads sharing the work:
    // 1 << shift threads have an entry each, and the next as many the rest of the list.
    int shift = 0;
    while ((1 << shift) < a.top) ++shift;
    const int at = tid & ((1 << shift) - 1), others = G >> shift;
    const int index = at < a.top ? idx[at] : -1;
    if (index >= 0)
      for (int k = tid >> shift; k < a.top; k += others)
        if (idx[k] == index && k != at) atomicOr(&twice[at], k < at ? 2 : 1);
  }
  __syncthreads();
  if (a.parts > 1) cluster_arrive_relaxed();  // this block has received what it waits for
  const float4 info = row_sm;
  RowGrad g;
  g.base = info.x == -INFINITY ? 0.0f : info.x;
  g.l2 = info.y * LOG2E;
  g.b = 0.0f;
  bool teacher_nan = false;  // a NaN or +inf among the teacher's values is in the sum of its warp
  for (int k = 1; k < WARPS && 32 * (k - 1) < a.top; ++k) teacher_nan = teacher_nan || isnan(teacher_sm[k].s);
  g.a = teacher_nan ? NAN : scale;
  T* dx = grad_row_late<T>(a, r);
  dense_grad<T, G, false>(p, dx, a.c, g, a.same_phase);
  if (entry_warp && part == 0) {
    // log q - log p with the two maxima taken out first: nearly equal distributions lose nothing to the logarithms' size
    float kl = 0.0f;
    // the factors T where distill_kernel has them
    if (mine >= 0 && q != 0.0f) kl = a.t * q * (dv - (info.z != 0.0f ? -INFINITY : L::up(x_mine) - info.x) - a.t * (ln_sq - info.y));
#pragma unroll
    for (int o = 16; o; o >>= 1) kl += __shfl_xor_sync(0xffffffffu, kl, o);
    if (lane == 0) kl_sm[warp] = kl;
  }
  __syncthreads();  // the dense gradient stands, with kl_sm
  if (owner && !(twice[e] & 2)) {  // as sparse_fix, with the logit at hand
    float w = weight[e];
    if (twice[e]) {
      w = 0.0f;
      for (int k = 0; k < a.top; ++k)
        if (idx[k] == mine) w += weight[k];
    }
    dx[mine] = L::down(grad_at<false>(L::up(x_mine), a.c, g) + w);
  }
  if (part == 0 && tid == 0) {
    float kl = 0.0f;
    for (int k = 1; k < WARPS && 32 * (k - 1) < a.top; ++k) kl += kl_sm[k];
    a.row_loss[r] = kl;
    if (a.stats) {
      a.stats[2 * r] = info.x;
      a.stats[2 * r + 1] = info.y;
    }
  }
  if (a.parts > 1) cluster_wait();  // no block leaves while another may still send to it
}

template <typename T, int G>
static __global__ void __launch_bounds__(Block<G>::THREADS, grad_blocks<T, G, false>()) distill_grad_kernel(DistillArgs a) {
  __shared__ __align__(16) int all_idx[Block<G>::ROWS][TEACHER_ROOM<G>];
  __shared__ float all_q[Block<G>::ROWS][TEACHER_ROOM<G>];
  __shared__ float fold[Group<G>::WARPS];
  int* idx = all_idx[Block<G>::slot()];
  float* q = all_q[Block<G>::slot()];
  const Cut<G> cut(a.rows, a.whole, a.parts);
  const int part = cut.part;
  const int r = cut.row;
  if (r < 0) return;
  const T* row = static_cast<const T*>(a.logits) + static_cast<long long>(r) * a.ld;
  T* dx = static_cast<T*>(a.dlogits) + static_cast<long long>(r) * a.ld_grad;
  const RowPart<T> p = row_part(row, a.vocab, part, cut.parts);
  float ln_sq;
  if (!load_teacher<G>(a, r, part == 0, idx, q, nullptr, fold, &ln_sq)) {
    zero_grad<T, G>(p, dx, a.same_phase);
    return;
  }
  RowGrad g;
  const float m = a.stats[2 * r];
  g.base = m == -INFINITY ? 0.0f : m;
  g.l2 = a.stats[2 * r + 1] * LOG2E;
  const float scale = a.upstream_rows ? a.scale * a.upstream_rows[r] : a.scale;
  g.a = isnan(ln_sq) ? NAN : scale;
  g.b = 0.0f;
  dense_grad<T, G, false>(p, dx, a.c, g, a.same_phase);
  for (int e = Group<G>::rank(); e < a.top; e += G) q[e] *= -scale;
  Group<G>::sync();
  sparse_fix<T, G, false>(p, dx, a.c, g, idx, q, a.top);
}

// Sum or mean of the row losses, in f64 and a fixed order.
static __global__ void __launch_bounds__(1024) distill_reduce_kernel(const float* __restrict__ row_loss, int rows,
                                                                     double factor, float* __restrict__ loss) {
  __shared__ double red[1024];
  double s = 0.0;
  for (int i = threadIdx.x; i < rows; i += 1024) s += static_cast<double>(row_loss[i]);
  red[threadIdx.x] = s;
  __syncthreads();
  for (int o = 512; o; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) *loss = static_cast<float>(red[0] * factor);
}

// ------------------------------------------------------------------ host side
static size_t logit_size(int32_t dtype) {
  return dtype == MTB200_F32 ? 4 : (dtype == MTB200_F16 || dtype == MTB200_BF16) ? 2 : 0;
}
static int32_t check_rows(const char* what, int32_t dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                          double temperature) {
  if (!logit_size(dtype)) return fail(MTB200_ERR_UNSUPPORTED, "%s: logits of dtype %d; f32, f16 and bf16 are supported", what, dtype);
  if (rows < 0 || vocab < 0) return fail(MTB200_ERR_INVALID, "%s: negative dimension", what);
  if (reinterpret_cast<uintptr_t>(logits) % logit_size(dtype)) return fail(MTB200_ERR_INVALID, "%s: misaligned logits", what);
  if (rows > INT32_MAX / 8 || vocab > INT32_MAX - 64)
    return fail(MTB200_ERR_INVALID, "%s: dimension exceeds the 32-bit limit of the device kernels", what);
  if (ld < vocab) return fail(MTB200_ERR_INVALID, "%s: row stride %lld is less than the vocabulary", what, (long long)ld);
  const float c = static_cast<float>(1.4426950408889634 / temperature);
  if (!(temperature > 0.0) || !std::isfinite(temperature) || !std::isfinite(c) || c < FLT_MIN ||
      !std::isfinite(static_cast<float>(temperature * temperature)))
    return fail(MTB200_ERR_INVALID, "%s: temperature must be positive and finite, got %g", what, temperature);
  return MTB200_OK;
}
static int32_t check_grad(const char* what, int32_t dtype, int64_t vocab, const void* logits, const void* dlogits, int64_t ld_grad) {
  if (dlogits == logits) return fail(MTB200_ERR_INVALID, "%s does not work in place", what);
  if (ld_grad < vocab)
    return fail(MTB200_ERR_INVALID, "%s: row stride %lld of the gradient is less than the vocabulary", what, (long long)ld_grad);
  if (reinterpret_cast<uintptr_t>(dlogits) % logit_size(dtype)) return fail(MTB200_ERR_INVALID, "%s: misaligned gradient", what);
  return MTB200_OK;
}
static int32_t check_index(const char* what, int32_t dtype) {
  if (dtype != MTB200_I32 && dtype != MTB200_I64)
    return fail(MTB200_ERR_UNSUPPORTED, "%s: indices must have dtype int32 or int64", what);
  return MTB200_OK;
}

// Dynamic shared memory that a kernel gets without asking.  The 48 KB of such a launch hold its static shared memory as well;
// token_scores_kernel, the only kernel here with dynamic shared memory, has 304 bytes of it at most.
constexpr size_t FREE_DYNAMIC_SMEM = 32 * 1024;

// One cluster of `parts` blocks per row, or with G = 32 a warp per row.
template <int G, typename Args>
static int32_t launch_rows(mtb200_ctx* h, void (*kernel)(Args), const Args& a, size_t smem = 0) {
  if (smem > FREE_DYNAMIC_SMEM)
    if (int32_t rc = grant_dynamic_smem(h, kernel, int(smem))) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = smem;
  cfg.gridDim = dim3(G == 32 ? unsigned((a.rows + Block<G>::ROWS - 1) / Block<G>::ROWS) : unsigned(a.rows) * unsigned(a.parts));
  cfg.blockDim = dim3(unsigned(Block<G>::THREADS));
  cfg.stream = h->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(a.parts);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.parts > 1 ? 1 : 0;
  MTB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return MTB200_OK;
}

// Threads per row and blocks per row.
struct RowPlan {
  int group, parts;
};
// A warp per row up to 8 KB where the rows are many (65536 x 1000 f32: 60 us against 460 us with a block of 512 per row; 300 x
// 4000 f16 with 20 alternatives take 16.0 us by warps and 6.4 us by 128 threads, 2000 rows 20.8 and 15.7 us, 2000 x 1000 f32
// 11.5 and 13.4 us), 128 threads up to 32 KB, or 64 KB with the selection, whose steps other rows have to hide (4096 x 16000
// f32 with 20: 63 us against 100), else blocks of 512.  The number of rows is not looked at there: rows of 32 KB are at home with
// 128 threads whether they are 1 or 2000 (16000 bf16 with 20: 7.1 us against 8.2, 24.9 against 31.1), those of 64 KB with the
// selection only from some 500 on (32000 bf16 with 20, 128 threads against blocks of 512 in parts: 1 row 9.2 and 8.2 us, 300
// rows 15.0 and 12.0, 600 rows 16.7 and 18.0, 2000 rows 36.9 and 42.6).
// Many alternatives need many units to choose from: beyond WARP_TOP the warp, beyond MID_TOP the 128 threads are the slower
// (8192 x 1000 f16 with 32: 99 us by warps and 64 us by blocks; 4096 x 4000 f32 with 100: 214 and 108 us).  Short rows with
// more than MID_TOP are slow all the same: 4096 x 1000 f16 take 258 us with 128 and 46 with 64.
// Where whole rows leave SMs without work, a row is cut into up to 8 parts of 8 KB at least, as long as the parts still find
// room side by side: 64 rows of 128256 bf16 with their best 20 take 14.2 us in 4 parts and 24.7 us in 8, which run in two waves.
constexpr int64_t WARP_BYTES = 8192, MID_BYTES = 32768, MID_BYTES_TOP = 65536, PART_BYTES = 8192;
constexpr int WARP_TOP = 20, MID_TOP = 64;
static RowPlan plan_rows(const mtb200_ctx* h, int64_t rows, int64_t row_bytes, bool warp, int64_t mid_bytes) {
  if (row_bytes <= WARP_BYTES && warp && rows > 8 * h->sm_count) return {32, 1};
  if (row_bytes <= mid_bytes) return {128, 1};
  int parts = 1;
  while (parts < MAX_PARTS && rows * parts <= h->sm_count && row_bytes / (2 * parts) >= PART_BYTES) parts *= 2;
  return {512, parts};
}

// With the selection on many rows, four blocks of 256 threads on an SM instead of two of 512: a block that selects leaves
// three that stream.  4096 x 128256 bf16 and their best 20: 206 us against 239; 4096 x 60000 f32 180 against 213.  Longer f32
// rows, bound by HBM, gain nothing (2048 x 151936 with 64: 247 us against 234); of 16-bit ones, with twice the elements to
// work on in a byte, all that were measured do (4096 x 151936 bf16 with 20: 232 us against 278, 1000 x 262144 f16: 102 against
// 109).  Fewer rows than blocks gain nothing, and from some 64 on the candidates are too many for 256 threads.
constexpr int64_t QUAD_BYTES = 256 << 10;
template <typename T, int G>
static int32_t launch_scores(mtb200_ctx* h, const ScoreArgs& a) {
  size_t smem = 0;
  if constexpr (G == 512)
    if (a.top && a.top <= MID_TOP && (sizeof(T) == 2 || a.vocab * int64_t(sizeof(T)) <= QUAD_BYTES) && a.rows > 2 * h->sm_count)
      return launch_scores<T, 256>(h, a);
  if (a.top) smem = sizeof(TopScratch<G>) * Block<G>::ROWS + (a.parts > 1 ? sizeof(unsigned long long) * a.parts * a.top : 0);
  return launch_rows<G>(h, a.top ? (a.entropy ? token_scores_kernel<T, G, true, true> : token_scores_kernel<T, G, true, false>)
                                 : (a.entropy ? token_scores_kernel<T, G, false, true> : token_scores_kernel<T, G, false, false>),
                        a, smem);
}
// The gradient kernels' blocks do not meet, so that rows can be cut unevenly: `whole` rows go to a block each, as many as
// make the same number for every SM, and the rows that are left are cut into the number of parts that spreads them best.
// 601 x 32003 f32 on 148 SMs, four rows for each and nine over in 16 parts: 31.3 us, 35.3 us with a block for each of the
// nine.  (Cutting all rows costs more than it spreads: 4096 x 128256 bf16 take 314 us whole and 366 us in parts of 64 KB.)
static void cut_rows(const mtb200_ctx* h, int rows, int64_t row_bytes, int* whole, int* parts) {
  const bool few = rows < 2 * h->sm_count;
  const int left = few ? rows : rows % h->sm_count;
  *whole = rows - left;
  *parts = 1;
  double best = 1e30;
  for (int n = few && rows <= h->sm_count ? 2 : 1; n <= 16 && (n == 1 || row_bytes / n >= PART_BYTES); ++n) {
    const double rounds = double((int64_t(left) * n + h->sm_count - 1) / h->sm_count) / n;
    if (rounds < 0.95 * best) {  // worth the further blocks
      best = rounds;
      *parts = n;
    }
  }
}
template <int G, typename Args>
static int32_t launch_cut(mtb200_ctx* h, void (*kernel)(Args), Args a, size_t row_bytes) {
  a.whole = a.rows;
  a.parts = 1;
  if (G == 512) cut_rows(h, a.rows, int64_t(row_bytes), &a.whole, &a.parts);
  const int64_t units = a.whole + int64_t(a.rows - a.whole) * a.parts;
  kernel<<<unsigned((units + Block<G>::ROWS - 1) / Block<G>::ROWS), Block<G>::THREADS, 0, h->stream>>>(a);
  MTB_CUDA(cudaGetLastError());
  return MTB200_OK;
}
template <typename T, int G>
static int32_t launch_score_grad(mtb200_ctx* h, const ScoreGradArgs& a) {
  return launch_cut<G>(h, a.d_entropy ? token_scores_grad_kernel<T, G, true> : token_scores_grad_kernel<T, G, false>, a,
                       a.vocab * sizeof(T));
}
// Parts of a row for the step that looks at it twice: the rows in flight, three blocks of 512 threads on an SM, have to
// stay in L2 beside the gradients that are written.  4096 x 128256 bf16, 114 MB of rows in flight without a cut: 435 us in 2
// parts (57 MB), 518 in 1, 538 in 4, whose blocks do too little between their meetings.  Parts are doubled: whether the rows
// then fill whole waves of clusters is not looked at (1021 x 50257 f32 run as 4.6).
constexpr int64_t L2_ROWS_BYTES = int64_t(64) << 20;
template <typename T, int G>
static int32_t launch_distill(mtb200_ctx* h, const DistillArgs& a) {
  if constexpr (G == 512)
    if (a.row_loss && a.dlogits && a.top <= CLUSTER_TEACHER) {
      DistillArgs c = a;
      const int64_t row_bytes = int64_t(a.vocab) * sizeof(T);
      while (c.parts < MAX_PARTS && 3 * h->sm_count / c.parts * row_bytes > L2_ROWS_BYTES) c.parts *= 2;
      return launch_rows<G>(h, distill_cluster_kernel<T>, c);
    }
  if (!a.row_loss) return launch_cut<G>(h, distill_grad_kernel<T, G>, a, a.vocab * sizeof(T));
  return launch_rows<G>(h, a.dlogits ? distill_kernel<T, G, true> : distill_kernel<T, G, false>, a);
}
// f(element type, group size as a compile-time number)
template <int G>
struct GroupTag {};
template <int G>
constexpr int group_of(GroupTag<G>) {
  return G;
}
template <typename F>
static int32_t by_type_and_group(int32_t dtype, int group, F f) {
  auto with = [&](auto element) {
    return group == 32 ? f(element, GroupTag<32>()) : group == 128 ? f(element, GroupTag<128>()) : f(element, GroupTag<512>());
  };
  if (dtype == MTB200_F32) return with(float());
  if (dtype == MTB200_F16) return with(__half());
  return with(__nv_bfloat16());
}
// whether each row starts at the same offset within 16 bytes in both matrices
static int same_phase(const void* x, int64_t ldx, const void* y, int64_t ldy, int32_t dtype) {
  return ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) == 0 && (ldx - ldy) * int64_t(logit_size(dtype)) % 16 == 0;
}

}  // namespace mtb

using namespace mtb;

#define MTB_CHECK_HANDLE(h)                                         \
  if (!(h)) return fail(MTB200_ERR_INVALID, "null handle");         \
  DeviceGuard guard__((h)->device);                                 \
  if (!guard__.ok) return fail(MTB200_ERR_CUDA, "cannot make device %d current", (h)->device)

extern "C" {

int32_t mtb200_token_log_probs(mtb200_handle h, int32_t dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                               const void* tokens, int32_t token_dtype, int32_t has_ignore, int64_t ignore_index,
                               double temperature, int64_t top, float* log_probs, float* entropy, float* top_log_probs,
                               int32_t* top_indices, float* stats) {
  MTB_CHECK_HANDLE(h);
  const char* what = "token_log_probs";
  if (int32_t rc = check_rows(what, dtype, rows, vocab, logits, ld, temperature)) return rc;
  if (tokens)
    if (int32_t rc = check_index(what, token_dtype)) return rc;
  if (top < 0 || top > VOCAB_TOP_MAX || top > vocab)
    return fail(MTB200_ERR_INVALID, "%s: top must be between 0 and min(%d, vocabulary), got %lld", what, VOCAB_TOP_MAX, (long long)top);
  if (rows == 0) return MTB200_OK;
  if (vocab == 0) return fail(MTB200_ERR_INVALID, "%s: empty vocabulary", what);
  if (!logits || !stats || (tokens && !log_probs) || (top && (!top_log_probs || !top_indices)))
    return fail(MTB200_ERR_INVALID, "%s: null pointer", what);
  ScoreArgs a = {};
  a.logits = logits; a.ld = ld; a.rows = int(rows); a.vocab = int(vocab); a.top = int(top);
  a.tokens = {tokens, token_dtype == MTB200_I64};
  a.has_ignore = has_ignore != 0; a.ignore = ignore_index;
  a.inv_t = float(1.0 / temperature); a.c = float(1.4426950408889634 / temperature);
  a.log_probs = tokens ? log_probs : nullptr; a.entropy = entropy; a.top_log_probs = top_log_probs;
  a.top_indices = top_indices; a.stats = stats; a.bad_label = h->status + 1;
  const RowPlan plan = plan_rows(h, rows, vocab * int64_t(logit_size(dtype)), top <= WARP_TOP,
                                 top == 0 ? MID_BYTES : top <= MID_TOP ? MID_BYTES_TOP : 0);
  a.parts = plan.parts;
  return by_type_and_group(dtype, plan.group, [&](auto element, auto tag) { return launch_scores<decltype(element), group_of(tag)>(h, a); });
}

int32_t mtb200_token_log_probs_bwd_ex(mtb200_handle h, int32_t dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                                      const void* tokens, int32_t token_dtype, int32_t has_ignore, int64_t ignore_index,
                                      double temperature, const float* stats, const float* d_log_probs, const float* entropy,
                                      const float* d_entropy, int64_t top, const int32_t* top_indices, const float* d_top,
                                      void* dlogits, int64_t ld_grad) {
  MTB_CHECK_HANDLE(h);
  const char* what = "token_log_probs_bwd";
  if (int32_t rc = check_rows(what, dtype, rows, vocab, logits, ld, temperature)) return rc;
  if (tokens)
    if (int32_t rc = check_index(what, token_dtype)) return rc;
  if (top < 0 || top > VOCAB_TOP_MAX || top > vocab)
    return fail(MTB200_ERR_INVALID, "%s: top must be between 0 and min(%d, vocabulary), got %lld", what, VOCAB_TOP_MAX, (long long)top);
  if (rows == 0 || vocab == 0) return MTB200_OK;
  if (!logits || !stats || !dlogits || (d_log_probs && !tokens) || (d_entropy && !entropy) || (top && (!top_indices || !d_top)))
    return fail(MTB200_ERR_INVALID, "%s: null pointer", what);
  if (int32_t rc = check_grad(what, dtype, vocab, logits, dlogits, ld_grad)) return rc;
  ScoreGradArgs a = {};
  a.logits = logits; a.dlogits = dlogits; a.ld = ld; a.ld_grad = ld_grad; a.rows = int(rows); a.vocab = int(vocab); a.top = int(top);
  a.tokens = {tokens, token_dtype == MTB200_I64};
  a.has_ignore = has_ignore != 0; a.ignore = ignore_index;
  a.inv_t = float(1.0 / temperature); a.c = float(1.4426950408889634 / temperature);
  a.stats = stats; a.entropy = entropy; a.d_log_probs = d_log_probs; a.d_entropy = d_entropy; a.d_top = d_top;
  a.top_indices = top_indices; a.bad_label = h->status + 1;
  a.same_phase = same_phase(logits, ld, dlogits, ld_grad, dtype);
  const RowPlan plan = plan_rows(h, rows, vocab * int64_t(logit_size(dtype)), true, MID_BYTES);
  a.parts = plan.parts;
  return by_type_and_group(dtype, plan.group, [&](auto element, auto tag) { return launch_score_grad<decltype(element), group_of(tag)>(h, a); });
}
int32_t mtb200_token_log_probs_bwd(mtb200_handle h, int32_t dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                                   const void* tokens, int32_t token_dtype, int32_t has_ignore, int64_t ignore_index,
                                   double temperature, const float* stats, const float* d_log_probs, const float* entropy,
                                   const float* d_entropy, int64_t top, const int32_t* top_indices, const float* d_top,
                                   void* dlogits) {
  return mtb200_token_log_probs_bwd_ex(h, dtype, rows, vocab, logits, ld, tokens, token_dtype, has_ignore, ignore_index, temperature,
                                       stats, d_log_probs, entropy, d_entropy, top, top_indices, d_top, dlogits, ld);
}

static int32_t distill_args(mtb200_handle h, const char* what, int32_t dtype, int64_t rows, int64_t vocab, const void* logits,
                            int64_t ld, int64_t top, const void* teacher_indices, int32_t index_dtype, const void* teacher_logits,
                            int32_t teacher_dtype, double temperature, int32_t reduction, float upstream,
                            const float* upstream_rows, void* dlogits, int64_t ld_grad, DistillArgs* a, int* group) {
  if (int32_t rc = check_rows(what, dtype, rows, vocab, logits, ld, temperature)) return rc;
  if (int32_t rc = check_index(what, index_dtype)) return rc;
  if (!logit_size(teacher_dtype))
    return fail(MTB200_ERR_UNSUPPORTED, "%s: teacher values of dtype %d; f32, f16 and bf16 are supported", what, teacher_dtype);
  if (top < 0 || top > VOCAB_TEACHER_MAX)
    return fail(MTB200_ERR_INVALID, "%s: between 0 and %d teacher entries per row, got %lld", what, VOCAB_TEACHER_MAX, (long long)top);
  if (reduction < MTB200_REDUCE_SUM || reduction > MTB200_REDUCE_NONE)
    return fail(MTB200_ERR_INVALID, "Invalid reduction mode: %d. Must be 'mean', 'sum', or 'none'", reduction);
  if (rows > 0 && vocab > 0 && (!logits || (top && (!teacher_indices || !teacher_logits))))
    return fail(MTB200_ERR_INVALID, "%s: null pointer", what);
  if (dlogits)
    if (int32_t rc = check_grad(what, dtype, vocab, logits, dlogits, ld_grad)) return rc;
  *a = {};
  a->logits = logits; a->dlogits = dlogits; a->ld = ld; a->ld_grad = ld_grad; a->rows = int(rows); a->vocab = int(vocab); a->top = int(top);
  a->index = {teacher_indices, index_dtype == MTB200_I64};
  a->value = {teacher_logits, teacher_dtype};
  a->t = float(temperature); a->c = float(1.4426950408889634 / temperature);
  a->scale = float(temperature * (reduction == MTB200_REDUCE_MEAN && rows ? 1.0 / double(rows) : 1.0) * double(upstream));
  a->upstream_rows = upstream_rows; a->status = h->status; a->bad_label = h->status + 1;
  a->same_phase = same_phase(logits, ld, dlogits, ld_grad, dtype);
  const RowPlan plan = plan_rows(h, rows, vocab * int64_t(logit_size(dtype)), top <= TEACHER_WARP_MAX, MID_BYTES);
  a->parts = plan.parts;
  *group = plan.group;
  return MTB200_OK;
}

int32_t mtb200_distill_ex(mtb200_handle h, int32_t dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, int64_t top,
                          const void* teacher_indices, int32_t index_dtype, const void* teacher_logits, int32_t teacher_dtype,
                          double temperature, int32_t reduction, float upstream, const float* upstream_rows, float* row_loss,
                          float* loss, float* stats, void* dlogits, int64_t ld_grad) {
  MTB_CHECK_HANDLE(h);
  DistillArgs a;
  int group;
  if (int32_t rc = distill_args(h, "distill", dtype, rows, vocab, logits, ld, top, teacher_indices, index_dtype, teacher_logits,
                                teacher_dtype, temperature, reduction, upstream, upstream_rows, dlogits, ld_grad, &a, &group))
    return rc;
  if ((rows > 0 && !row_loss) || (reduction != MTB200_REDUCE_NONE && !loss)) return fail(MTB200_ERR_INVALID, "null loss pointer");
  a.row_loss = row_loss;
  a.stats = stats;
  if (rows > 0) {
    if (vocab == 0) {
      if (top) return fail(MTB200_ERR_INVALID, "distill: empty vocabulary");
      MTB_CUDA(cudaMemsetAsync(row_loss, 0, sizeof(float) * size_t(rows), h->stream));
    } else {
      const int32_t rc = by_type_and_group(
          dtype, group, [&](auto element, auto tag) { return launch_distill<decltype(element), group_of(tag)>(h, a); });
      if (rc) return rc;
    }
  }
  if (reduction != MTB200_REDUCE_NONE) {
    // the mean over no rows is 0/0, as in cross entropy
    const double factor = reduction == MTB200_REDUCE_MEAN ? (rows ? 1.0 / double(rows) : double(NAN)) : 1.0;
    distill_reduce_kernel<<<1, 1024, 0, h->stream>>>(row_loss, int(rows), factor, loss);
    MTB_CUDA(cudaGetLastError());
  }
  return MTB200_OK;
}
int32_t mtb200_distill(mtb200_handle h, int32_t dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, int64_t top,
                       const void* teacher_indices, int32_t index_dtype, const void* teacher_logits, int32_t teacher_dtype,
                       double temperature, int32_t reduction, float upstream, const float* upstream_rows, float* row_loss,
                       float* loss, float* stats, void* dlogits) {
  return mtb200_distill_ex(h, dtype, rows, vocab, logits, ld, top, teacher_indices, index_dtype, teacher_logits, teacher_dtype,
                           temperature, reduction, upstream, upstream_rows, row_loss, loss, stats, dlogits, ld);
}

int32_t mtb200_distill_bwd_ex(mtb200_handle h, int32_t dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                              int64_t top, const void* teacher_indices, int32_t index_dtype, const void* teacher_logits,
                              int32_t teacher_dtype, double temperature, int32_t reduction, float upstream,
                              const float* upstream_rows, const float* stats, void* dlogits, int64_t ld_grad) {
  MTB_CHECK_HANDLE(h);
  DistillArgs a;
  int group;
  if (int32_t rc = distill_args(h, "distill_bwd", dtype, rows, vocab, logits, ld, top, teacher_indices, index_dtype,
                                teacher_logits, teacher_dtype, temperature, reduction, upstream, upstream_rows, dlogits, ld_grad, &a, &group))
    return rc;
  if (rows == 0 || vocab == 0) return MTB200_OK;
  if (!stats || !dlogits) return fail(MTB200_ERR_INVALID, "distill_bwd: null pointer");
  a.stats = const_cast<float*>(stats);
  return by_type_and_group(dtype, group,
                           [&](auto element, auto tag) { return launch_distill<decltype(element), group_of(tag)>(h, a); });
}
int32_t mtb200_distill_bwd(mtb200_handle h, int32_t dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                           int64_t top, const void* teacher_indices, int32_t index_dtype, const void* teacher_logits,
                           int32_t teacher_dtype, double temperature, int32_t reduction, float upstream,
                           const float* upstream_rows, const float* stats, void* dlogits) {
  return mtb200_distill_bwd_ex(h, dtype, rows, vocab, logits, ld, top, teacher_indices, index_dtype, teacher_logits, teacher_dtype,
                               temperature, reduction, upstream, upstream_rows, stats, dlogits, ld);
}

}  // extern "C"
