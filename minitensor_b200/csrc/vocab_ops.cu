// Operators on a language model's logits [rows][vocabulary] (f32, bf16 or f16): log probabilities of given tokens with
// entropy and top alternatives, distillation from a teacher's top logits, and their gradients.  They have no
// counterpart in the reference; they stand beside its cross entropy (engine/src/operations/loss/regression.rs:178-251).
// Every call is one or two launches, allocates nothing and keeps nothing between calls: statistics that a backward
// call needs are the caller's.  Formulas, arithmetic and conventions: vocab_rows.cuh.
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

constexpr float LN2 = 0.693147180559945309f;
constexpr float LOG2E = 1.442695040888963407f;

// ------------------------------------------------------------------ token log probabilities
// A cluster of `parts` blocks per row (one block when there are rows enough).  One pass over the logits: HBM-bound.
template <typename T, int THREADS, bool TOP, bool ENT>
static __global__ void __launch_bounds__(THREADS) token_scores_kernel(ScoreArgs a) {
  using L = LogitType<T>;
  __shared__ RowStat sm[THREADS / 32 + 1];
  __shared__ TopScratch<TOP ? THREADS : 32> ts;
  cg::cluster_group cluster = cg::this_cluster();
  const int part = blockIdx.x % a.parts;
  const long long r = blockIdx.x / a.parts;
  const int tid = threadIdx.x;
  const T* row = static_cast<const T*>(a.logits) + r * a.ld;

  long long token = -1;
  bool good = true;
  if (a.tokens.p) {
    token = a.tokens.at(r);
    if (a.has_ignore && token == a.ignore) {  // the whole cluster leaves
      if (part == 0) {
        if (tid == 0) {
          a.log_probs[r] = 0.0f;
          if (ENT) a.entropy[r] = 0.0f;
          a.stats[2 * r] = -INFINITY;
          a.stats[2 * r + 1] = 0.0f;
        }
        if (TOP)
          for (int i = tid; i < a.top; i += THREADS) {
            a.top_log_probs[r * a.top + i] = -INFINITY;
            a.top_indices[r * a.top + i] = -1;
          }
      }
      return;
    }
    good = token >= 0 && token < a.vocab;
    if (!good && part == 0 && tid == 0) atomicOr(a.bad_label, 1u);
  }
  float x_token = 0.0f;
  if (part == 0 && tid == 0 && a.tokens.p) x_token = good ? L::up(row[token]) : NAN;

  const RowPart<T> p = row_part(row, a.vocab, part, a.parts);
  int where;
  const RowStat unit = unit_stats<T, THREADS, ENT>(p, a.c, where);
  RowStat st = block_merge<THREADS>(unit, a.c, sm);
  if constexpr (TOP) select_top<T, THREADS>(p, a.top, unit.m, where, ts);
  if (a.parts > 1) {
    cluster.sync();
    if (part == 0) st = cluster_merge(cluster, &sm[THREADS / 32], a.parts, a.c);
  }
  if (part == 0) {
    const bool none = st.m == -INFINITY && !isnan(st.s);
    const float ln_s = none ? 0.0f : logf(st.s);
    if (tid == 0) {
      if (a.log_probs) a.log_probs[r] = none && good ? -INFINITY : (x_token - st.m) * a.inv_t - ln_s;
      if (ENT) a.entropy[r] = none ? 0.0f : ln_s - a.inv_t * (st.u / st.s);
      a.stats[2 * r] = st.m;
      a.stats[2 * r + 1] = ln_s;
    }
    if constexpr (TOP) {
      auto put = [&](int at, unsigned long long w) {
        a.top_log_probs[r * a.top + at] = none ? -INFINITY : (key_value(candidate_key(w)) - st.m) * a.inv_t - ln_s;
        a.top_indices[r * a.top + at] = candidate_index(w);
      };
      if (a.parts == 1) {
        for (int i = tid; i < a.top; i += THREADS) put(i, ts.best[i]);
      } else {
        // merge of the parts' sorted lists: an entry's place is its place in its own list plus the entries above it
        // in every other one
        unsigned long long* pool = ts.pool;  // parts * top <= 8 * 256 words
        const int total = a.parts * a.top;
        for (int i = tid; i < total; i += THREADS) pool[i] = cluster.map_shared_rank(ts.best, i / a.top)[i % a.top];
        __syncthreads();
        for (int i = tid; i < total; i += THREADS) {
          const unsigned long long w = pool[i];
          if (!w) continue;
          int at = i % a.top;
          for (int q = 0; q < a.parts && at < a.top; ++q)
            if (q != i / a.top) at += count_above(pool + q * a.top, a.top, w);
          if (at < a.top) put(at, w);
        }
      }
    }
  }
  if (a.parts > 1) cluster.sync();  // shared memory stays until rank 0 has read it
}

struct ScoreGradArgs {
  const void* logits;
  void* dlogits;
  long long ld;
  int rows, vocab, top, parts, same_phase;
  IndexArray tokens;
  int has_ignore;
  long long ignore;
  float inv_t, c;
  const float *stats, *entropy, *d_log_probs, *d_entropy, *d_top;
  const int* top_indices;
  uint32_t* bad_label;
};

// dx = (1/T) [ sum of weights at given indices - p (sum of all weights) - g_H p (log p + H) ], one read, one write.
template <typename T, int THREADS, bool ENT>
static __global__ void __launch_bounds__(THREADS) token_scores_grad_kernel(ScoreGradArgs a) {
  __shared__ int idx[VOCAB_TOP_MAX + 1];
  __shared__ float weight[VOCAB_TOP_MAX + 1];
  __shared__ float fold[THREADS / 32];
  const int part = blockIdx.x % a.parts;
  const long long r = blockIdx.x / a.parts;
  const int tid = threadIdx.x;
  const T* row = static_cast<const T*>(a.logits) + r * a.ld;
  T* dx = static_cast<T*>(a.dlogits) + r * a.ld;
  const RowPart<T> p = row_part(row, a.vocab, part, a.parts);
  const long long token = a.tokens.p ? a.tokens.at(r) : -1;
  if (a.tokens.p && a.has_ignore && token == a.ignore) {
    zero_grad<T, THREADS>(p, dx, a.same_phase);
    return;
  }
  const bool good = token >= 0 && token < a.vocab;
  if (a.tokens.p && !good && part == 0 && tid == 0) atomicOr(a.bad_label, 1u);
  const int n = a.top + 1;
  float sum = 0.0f;
  for (int e = tid; e < n; e += THREADS) {
    int j;
    float w;
    if (e == 0) {
      j = good && a.d_log_probs ? static_cast<int>(token) : -1;
      w = j >= 0 ? a.d_log_probs[r] : 0.0f;
    } else {
      j = a.top_indices[r * a.top + e - 1];
      if (j < 0 || j >= a.vocab) {  // -1: no entry
        if (j >= a.vocab) atomicOr(a.bad_label, 1u);
        j = -1;
      }
      w = j >= 0 ? a.d_top[r * a.top + e - 1] : 0.0f;
    }
    idx[e] = j;
    weight[e] = w * a.inv_t;
    sum += w;
  }
  sum = block_fold<THREADS, false>(sum, fold);
  RowGrad g;
  const float m = a.stats[2 * r];
  g.base = m == -INFINITY ? 0.0f : m;
  g.l2 = a.stats[2 * r + 1] * LOG2E;
  const float gh = ENT ? a.d_entropy[r] : 0.0f;
  g.b = -gh * a.inv_t * LN2;
  g.a = -a.inv_t * (sum + (ENT ? gh * a.entropy[r] : 0.0f));
  dense_grad<T, THREADS, ENT>(p, dx, a.c, g, a.same_phase);
  __syncthreads();
  sparse_fix<T, THREADS, ENT>(p, dx, a.c, g, idx, weight, n);
}

// ------------------------------------------------------------------ distillation
struct DistillArgs {
  const void* logits;
  void* dlogits;           // forward: nullptr = loss only
  long long ld;
  int rows, vocab, top, parts, same_phase;
  IndexArray index;
  RealArray value;
  float inv_t, c, t;
  float scale;             // T * reduction factor * upstream: d loss / d logits = scale * weight_r * (Q p - q)
  const float* upstream_rows;
  float *row_loss, *stats;
  uint32_t* bad_label;
};

// The teacher's entries of row r into shared memory: q over the entries with an index in [0, vocab) (0 elsewhere,
// index -1), softmax of value / T, and (nullable) dv = value - largest value.  Returns whether the row has any entry;
// ln_s: log q = dv / T - ln_s (NaN if a value is NaN or +inf).
template <int THREADS>
__device__ __forceinline__ bool load_teacher(const DistillArgs& a, long long r, bool report, int* idx, float* q, float* dv,
                                             float* fold, float* ln_s) {
  const int tid = threadIdx.x;
  float top = -INFINITY;
  bool any = false;
  for (int e = tid; e < a.top; e += THREADS) {
    const long long j = a.index.at(r * a.top + e);
    const bool in = j >= 0 && j < a.vocab;
    if (!in && j != -1 && report) atomicOr(a.bad_label, 1u);
    idx[e] = in ? static_cast<int>(j) : -1;
    q[e] = in ? a.value.at(r * a.top + e) : -INFINITY;
    top = fmaxf(top, q[e]);
    any = any || (in && q[e] != -INFINITY);  // NaN counts: it has to reach the result
  }
  any = __syncthreads_or(any);
  if (!any) return false;
  top = block_fold<THREADS, true>(top, fold);
  const float base = top == -INFINITY ? 0.0f : top;
  float s = 0.0f;
  for (int e = tid; e < a.top; e += THREADS) {
    const float d = q[e] - base;
    const float w = ex2_ftz(d * a.c);
    s += w;
    q[e] = w;
    if (dv) dv[e] = d;
  }
  s = block_fold<THREADS, false>(s, fold);
  const float inv = 1.0f / s;
  for (int e = tid; e < a.top; e += THREADS) q[e] *= inv;
  *ln_s = logf(s);
  __syncthreads();
  return true;
}

// Loss per row, T^2 sum_k q_k (log q_k - log p_idx_k), and with GRAD the gradient: the row's statistics, then a second
// look at the row while it is in L2.
template <typename T, int THREADS, bool GRAD>
static __global__ void __launch_bounds__(THREADS) distill_kernel(DistillArgs a) {
  using L = LogitType<T>;
  __shared__ RowStat sm[THREADS / 32 + 1];
  __shared__ int idx[VOCAB_TEACHER_MAX];
  __shared__ float q[VOCAB_TEACHER_MAX], dv[VOCAB_TEACHER_MAX];
  __shared__ float fold[THREADS / 32];
  cg::cluster_group cluster = cg::this_cluster();
  const int part = blockIdx.x % a.parts;
  const long long r = blockIdx.x / a.parts;
  const int tid = threadIdx.x;
  const T* row = static_cast<const T*>(a.logits) + r * a.ld;
  T* dx = GRAD ? static_cast<T*>(a.dlogits) + r * a.ld : nullptr;
  const RowPart<T> p = row_part(row, a.vocab, part, a.parts);

  float ln_sq;
  if (!load_teacher<THREADS>(a, r, part == 0, idx, q, dv, fold, &ln_sq)) {  // the same answer in every block of the cluster
    if (part == 0 && tid == 0) {
      a.row_loss[r] = 0.0f;
      if (a.stats) {
        a.stats[2 * r] = -INFINITY;
        a.stats[2 * r + 1] = 0.0f;
      }
    }
    if (GRAD) zero_grad<T, THREADS>(p, dx, a.same_phase);
    return;
  }
  int where;
  RowStat st = block_merge<THREADS>(unit_stats<T, THREADS, false>(p, a.c, where), a.c, sm);
  if (a.parts > 1) {
    cluster.sync();
    st = cluster_merge(cluster, &sm[THREADS / 32], a.parts, a.c);
  }
  const bool none = st.m == -INFINITY && !isnan(st.s);
  const float ln_s = none ? 0.0f : logf(st.s);
  if (part == 0) {
    // log q - log p with the two maxima taken out first: nearly equal distributions lose nothing to the logarithms' size
    float kl = 0.0f;
    for (int e = tid; e < a.top; e += THREADS) {
      if (idx[e] < 0 || q[e] == 0.0f) continue;
      const float dx = none ? -INFINITY : L::up(row[idx[e]]) - st.m;
      kl += q[e] * ((dv[e] - dx) * a.inv_t - (ln_sq - ln_s));
    }
    kl = block_fold<THREADS, false>(kl, fold);
    if (tid == 0) {
      a.row_loss[r] = a.t * a.t * kl;
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
    dense_grad<T, THREADS, false>(p, dx, a.c, g, a.same_phase);
    for (int e = tid; e < a.top; e += THREADS) q[e] *= -scale;
    __syncthreads();
    sparse_fix<T, THREADS, false>(p, dx, a.c, g, idx, q, a.top);
  }
  if (a.parts > 1) cluster.sync();
}

template <typename T, int THREADS>
static __global__ void __launch_bounds__(THREADS) distill_grad_kernel(DistillArgs a) {
  __shared__ int idx[VOCAB_TEACHER_MAX];
  __shared__ float q[VOCAB_TEACHER_MAX];
  __shared__ float fold[THREADS / 32];
  const int part = blockIdx.x % a.parts;
  const long long r = blockIdx.x / a.parts;
  const T* row = static_cast<const T*>(a.logits) + r * a.ld;
  T* dx = static_cast<T*>(a.dlogits) + r * a.ld;
  const RowPart<T> p = row_part(row, a.vocab, part, a.parts);
  float ln_sq;
  if (!load_teacher<THREADS>(a, r, part == 0, idx, q, nullptr, fold, &ln_sq)) {
    zero_grad<T, THREADS>(p, dx, a.same_phase);
    return;
  }
  RowGrad g;
  const float m = a.stats[2 * r];
  g.base = m == -INFINITY ? 0.0f : m;
  g.l2 = a.stats[2 * r + 1] * LOG2E;
  const float scale = a.upstream_rows ? a.scale * a.upstream_rows[r] : a.scale;
  g.a = isnan(ln_sq) ? NAN : scale;
  g.b = 0.0f;
  dense_grad<T, THREADS, false>(p, dx, a.c, g, a.same_phase);
  for (int e = threadIdx.x; e < a.top; e += THREADS) q[e] *= -scale;
  __syncthreads();
  sparse_fix<T, THREADS, false>(p, dx, a.c, g, idx, q, a.top);
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
static int32_t check_grad(const char* what, int32_t dtype, const void* logits, const void* dlogits) {
  if (dlogits == logits) return fail(MTB200_ERR_INVALID, "%s does not work in place", what);
  if (reinterpret_cast<uintptr_t>(dlogits) % logit_size(dtype)) return fail(MTB200_ERR_INVALID, "%s: misaligned gradient", what);
  return MTB200_OK;
}
static int32_t check_index(const char* what, int32_t dtype) {
  if (dtype != MTB200_I32 && dtype != MTB200_I64)
    return fail(MTB200_ERR_UNSUPPORTED, "%s: indices must have dtype int32 or int64", what);
  return MTB200_OK;
}

// Launch of one cluster of `parts` blocks per row.
template <typename... KArgs, typename... Args>
static cudaError_t launch_rows(mtb200_ctx* h, void (*kernel)(KArgs...), int64_t rows, int parts, int threads, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows * parts));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.stream = h->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(parts);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Blocks per row: one when the rows fill the machine, else up to 8 with at least `least` bytes of the row each.
static int row_parts(const mtb200_ctx* h, int64_t rows, int64_t row_bytes) {
  int parts = 1;
  while (parts < 8 && rows * parts < 2 * h->sm_count && row_bytes / (2 * parts) >= 8192) parts *= 2;
  return parts;
}

template <typename T, int THREADS>
static int32_t launch_scores(mtb200_ctx* h, const ScoreArgs& a) {
  void (*kernel)(ScoreArgs) = a.top ? (a.entropy ? token_scores_kernel<T, THREADS, true, true> : token_scores_kernel<T, THREADS, true, false>)
                                    : (a.entropy ? token_scores_kernel<T, THREADS, false, true> : token_scores_kernel<T, THREADS, false, false>);
  MTB_CUDA(launch_rows(h, kernel, a.rows, a.parts, THREADS, a));
  return MTB200_OK;
}
// The gradient kernels' blocks do not meet: a plain grid.
template <typename T>
static int32_t launch_score_grad(mtb200_ctx* h, const ScoreGradArgs& a) {
  const unsigned blocks = unsigned(a.rows) * unsigned(a.parts);
  if (a.d_entropy) token_scores_grad_kernel<T, 512, true><<<blocks, 512, 0, h->stream>>>(a);
  else token_scores_grad_kernel<T, 512, false><<<blocks, 512, 0, h->stream>>>(a);
  MTB_CUDA(cudaGetLastError());
  return MTB200_OK;
}
template <typename T>
static int32_t launch_distill(mtb200_ctx* h, const DistillArgs& a, bool forward) {
  if (forward) {
    MTB_CUDA(launch_rows(h, a.dlogits ? distill_kernel<T, 512, true> : distill_kernel<T, 512, false>, a.rows, a.parts, 512, a));
  } else {
    distill_grad_kernel<T, 512><<<unsigned(a.rows) * unsigned(a.parts), 512, 0, h->stream>>>(a);
    MTB_CUDA(cudaGetLastError());
  }
  return MTB200_OK;
}
static int same_phase(const void* x, const void* y) {
  return ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) == 0;
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
  a.parts = row_parts(h, rows, vocab * int64_t(logit_size(dtype)));
  if (dtype == MTB200_F32) return launch_scores<float, 512>(h, a);
  if (dtype == MTB200_F16) return launch_scores<__half, 512>(h, a);
  return launch_scores<__nv_bfloat16, 512>(h, a);
}

int32_t mtb200_token_log_probs_bwd(mtb200_handle h, int32_t dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                                   const void* tokens, int32_t token_dtype, int32_t has_ignore, int64_t ignore_index,
                                   double temperature, const float* stats, const float* d_log_probs, const float* entropy,
                                   const float* d_entropy, int64_t top, const int32_t* top_indices, const float* d_top,
                                   void* dlogits) {
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
  if (int32_t rc = check_grad(what, dtype, logits, dlogits)) return rc;
  ScoreGradArgs a = {};
  a.logits = logits; a.dlogits = dlogits; a.ld = ld; a.rows = int(rows); a.vocab = int(vocab); a.top = int(top);
  a.tokens = {tokens, token_dtype == MTB200_I64};
  a.has_ignore = has_ignore != 0; a.ignore = ignore_index;
  a.inv_t = float(1.0 / temperature); a.c = float(1.4426950408889634 / temperature);
  a.stats = stats; a.entropy = entropy; a.d_log_probs = d_log_probs; a.d_entropy = d_entropy; a.d_top = d_top;
  a.top_indices = top_indices; a.bad_label = h->status + 1;
  a.same_phase = same_phase(logits, dlogits);
  a.parts = row_parts(h, rows, vocab * int64_t(logit_size(dtype)));
  if (dtype == MTB200_F32) return launch_score_grad<float>(h, a);
  if (dtype == MTB200_F16) return launch_score_grad<__half>(h, a);
  return launch_score_grad<__nv_bfloat16>(h, a);
}

static int32_t distill_args(mtb200_handle h, const char* what, int32_t dtype, int64_t rows, int64_t vocab, const void* logits,
                            int64_t ld, int64_t top, const void* teacher_indices, int32_t index_dtype, const void* teacher_logits,
                            int32_t teacher_dtype, double temperature, int32_t reduction, float upstream,
                            const float* upstream_rows, void* dlogits, DistillArgs* a) {
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
    if (int32_t rc = check_grad(what, dtype, logits, dlogits)) return rc;
  *a = {};
  a->logits = logits; a->dlogits = dlogits; a->ld = ld; a->rows = int(rows); a->vocab = int(vocab); a->top = int(top);
  a->index = {teacher_indices, index_dtype == MTB200_I64};
  a->value = {teacher_logits, teacher_dtype};
  a->t = float(temperature); a->inv_t = float(1.0 / temperature); a->c = float(1.4426950408889634 / temperature);
  a->scale = float(temperature * (reduction == MTB200_REDUCE_MEAN && rows ? 1.0 / double(rows) : 1.0) * double(upstream));
  a->upstream_rows = upstream_rows; a->bad_label = h->status + 1;
  a->same_phase = same_phase(logits, dlogits);
  a->parts = row_parts(h, rows, vocab * int64_t(logit_size(dtype)));
  return MTB200_OK;
}

int32_t mtb200_distill(mtb200_handle h, int32_t dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, int64_t top,
                       const void* teacher_indices, int32_t index_dtype, const void* teacher_logits, int32_t teacher_dtype,
                       double temperature, int32_t reduction, float upstream, const float* upstream_rows, float* row_loss,
                       float* loss, float* stats, void* dlogits) {
  MTB_CHECK_HANDLE(h);
  DistillArgs a;
  if (int32_t rc = distill_args(h, "distill", dtype, rows, vocab, logits, ld, top, teacher_indices, index_dtype, teacher_logits,
                                teacher_dtype, temperature, reduction, upstream, upstream_rows, dlogits, &a))
    return rc;
  if ((rows > 0 && !row_loss) || (reduction != MTB200_REDUCE_NONE && !loss)) return fail(MTB200_ERR_INVALID, "null loss pointer");
  a.row_loss = row_loss;
  a.stats = stats;
  if (rows > 0) {
    if (vocab == 0) {
      if (top) return fail(MTB200_ERR_INVALID, "distill: empty vocabulary");
      MTB_CUDA(cudaMemsetAsync(row_loss, 0, sizeof(float) * size_t(rows), h->stream));
    } else {
      int32_t rc = dtype == MTB200_F32 ? launch_distill<float>(h, a, true)
                   : dtype == MTB200_F16 ? launch_distill<__half>(h, a, true) : launch_distill<__nv_bfloat16>(h, a, true);
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

int32_t mtb200_distill_bwd(mtb200_handle h, int32_t dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                           int64_t top, const void* teacher_indices, int32_t index_dtype, const void* teacher_logits,
                           int32_t teacher_dtype, double temperature, int32_t reduction, float upstream,
                           const float* upstream_rows, const float* stats, void* dlogits) {
  MTB_CHECK_HANDLE(h);
  DistillArgs a;
  if (int32_t rc = distill_args(h, "distill_bwd", dtype, rows, vocab, logits, ld, top, teacher_indices, index_dtype,
                                teacher_logits, teacher_dtype, temperature, reduction, upstream, upstream_rows, dlogits, &a))
    return rc;
  if (rows == 0 || vocab == 0) return MTB200_OK;
  if (!stats || !dlogits) return fail(MTB200_ERR_INVALID, "distill_bwd: null pointer");
  a.stats = const_cast<float*>(stats);
  return dtype == MTB200_F32 ? launch_distill<float>(h, a, false)
         : dtype == MTB200_F16 ? launch_distill<__half>(h, a, false) : launch_distill<__nv_bfloat16>(h, a, false);
}

}  // extern "C"
