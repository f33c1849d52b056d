// Rows of logits over a vocabulary: statistics of the softmax in one pass, the largest entries, and the gradient pass.
// Shared by the operators of vocab_ops.cu.
//
// With T the temperature, d_j = x_j - m and c = log2(e) / T, a row of logits x is reduced to
//   m = max x,   S = sum_j 2^(c d_j),   U = sum_j 2^(c d_j) d_j                            (f32, running maximum)
// from which   log p_j = d_j / T - ln S,   entropy = ln S - (U / S) / T.
// The difference d_j is taken before the multiplication: it is exact near the maximum, and a row that holds nothing
// but the type's lowest value stays a uniform distribution (m / T would overflow).  Conventions for rows without a
// distribution: every logit -inf -> p = 0, log p = -inf, entropy 0;  a NaN or +inf -> NaN throughout.
#pragma once
#include "mtb200_core.cuh"

#include <cfloat>
#include <climits>
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mtb {

namespace cg = cooperative_groups;

constexpr int VOCAB_TOP_MAX = 256;       // largest `top` of the selection
constexpr int VOCAB_TEACHER_MAX = 1024;  // largest number of teacher entries per row

__device__ __forceinline__ float ex2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------ element types
template <typename T>
struct LogitType;
template <>
struct LogitType<float> {
  static constexpr int VEC = 4;
  static constexpr int KEY_SHIFT = 0;               // bits of an f32 sort key that are the same for every value
  static constexpr uint32_t NEG_INF_WORD = 0xff800000u;
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&f)[4]) {
    f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y); f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct LogitType<__nv_bfloat16> {
  static constexpr int VEC = 8;
  static constexpr int KEY_SHIFT = 16;
  static constexpr uint32_t NEG_INF_WORD = 0xff80ff80u;
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <>
struct LogitType<__half> {
  static constexpr int VEC = 8;
  static constexpr int KEY_SHIFT = 13;
  static constexpr uint32_t NEG_INF_WORD = 0xfc00fc00u;
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};

// The part of one row that one block works on.  Only whole 16-byte vectors inside the row are read as vectors; the
// elements before the first boundary (`head`) belong to the row's first part and those after the last one (`tail`)
// to its last part, and are read one by one.  Thread t owns head element t, the vectors v0 + t, v0 + t + THREADS,
// ... and tail element t: its "unit", in ascending order of index.
template <typename T>
struct RowPart {
  const T* row;
  int head, tail;            // scalar elements owned by this part
  int v0, v1;                // vectors [v0, v1) of the row
  int vec_base;              // index of vector 0's first element
  int tail_base;             // index of the first tail element
  __device__ __forceinline__ const uint4* vecs() const { return reinterpret_cast<const uint4*>(row + vec_base); }
};
template <typename T>
__device__ __forceinline__ RowPart<T> row_part(const T* row, int n, int part, int parts) {
  constexpr int VEC = LogitType<T>::VEC;
  RowPart<T> p;
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) / int(sizeof(T));
  const int head = off ? min(n, VEC - off) : 0;
  const int nv = (n - head) / VEC;
  p.row = row;
  p.vec_base = head;
  p.v0 = static_cast<int>(static_cast<long long>(nv) * part / parts);
  p.v1 = static_cast<int>(static_cast<long long>(nv) * (part + 1) / parts);
  p.tail_base = head + nv * VEC;
  p.head = part == 0 ? head : 0;
  p.tail = part == parts - 1 ? n - p.tail_base : 0;
  return p;
}
// whether element `j` of the row lies in this part
template <typename T>
__device__ __forceinline__ bool owns(const RowPart<T>& p, int j) {
  constexpr int VEC = LogitType<T>::VEC;
  if (j < p.vec_base) return j < p.head;
  if (j >= p.tail_base) return p.tail > 0;
  const int v = (j - p.vec_base) / VEC;
  return v >= p.v0 && v < p.v1;
}

// ------------------------------------------------------------------ statistics
struct RowStat {
  float m, s, u;
};
// Both orders of a merge give the same exponents, and -inf with -inf (or +inf with +inf) must not turn 0 into NaN:
// the difference is clamped to the largest finite magnitude, whose power of two is 0; a NaN sum survives the product.
__device__ __forceinline__ RowStat merge(const RowStat& a, const RowStat& b, float c) {
  RowStat r;
  r.m = fmaxf(a.m, b.m);
  const float da = fmaxf(a.m - r.m, -FLT_MAX), db = fmaxf(b.m - r.m, -FLT_MAX);
  const float ra = ex2_ftz(da * c), rb = ex2_ftz(db * c);
  r.s = a.s * ra + b.s * rb;
  // a part that is scaled to nothing drops out (0 * -FLT_MAX is fine, an overflowed s * d is not)
  r.u = (ra == 0.0f ? a.s * 0.0f : ra * (a.u + a.s * da)) + (rb == 0.0f ? b.s * 0.0f : rb * (b.u + b.s * db));
  return r;
}

constexpr int ROW_UNROLL = 4;  // vectors a thread keeps in flight

// The thread's unit, reduced.  `where` names the place of the unit's first maximum for find_first: the base vector
// of its group of ROW_UNROLL vectors, or WHERE_HEAD / WHERE_TAIL / WHERE_START (nothing above -inf was seen).
constexpr int WHERE_START = -1, WHERE_HEAD = -2, WHERE_TAIL = -3;

template <bool ENT, int E>
__device__ __forceinline__ void accumulate(const float (&x)[E], float c, RowStat& st, int& where, int here) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i < E; ++i) top = fmaxf(top, x[i]);
  if (top > st.m) {
    const float d = fmaxf(st.m - top, -FLT_MAX);
    const float r = ex2_ftz(d * c);
    if (ENT) st.u = r == 0.0f ? st.s * 0.0f : r * (st.u + st.s * d);
    st.s *= r;
    st.m = top;
    where = here;
  }
  const float base = st.m == -INFINITY ? 0.0f : st.m;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float d = x[i] - base;
    const float e = ex2_ftz(d * c);
    st.s += e;
    if (ENT) st.u = fmaf(e, fmaxf(d, -FLT_MAX), st.u);
  }
}

template <typename T, int THREADS, bool ENT>
__device__ __forceinline__ RowStat unit_stats(const RowPart<T>& p, float c, int& where) {
  using L = LogitType<T>;
  constexpr int VEC = L::VEC;
  const int tid = threadIdx.x;
  RowStat st = {-INFINITY, 0.0f, 0.0f};
  where = WHERE_START;
  if (tid < p.head) {
    const float x[1] = {L::up(p.row[tid])};
    accumulate<ENT>(x, c, st, where, WHERE_HEAD);
  }
  const uint4* vecs = p.vecs();
  for (int v = p.v0 + tid; v < p.v1; v += THREADS * ROW_UNROLL) {
    uint4 w[ROW_UNROLL];
#pragma unroll
    for (int k = 0; k < ROW_UNROLL; ++k)
      w[k] = v + k * THREADS < p.v1 ? vecs[v + k * THREADS]
                                    : make_uint4(L::NEG_INF_WORD, L::NEG_INF_WORD, L::NEG_INF_WORD, L::NEG_INF_WORD);
    float x[ROW_UNROLL * VEC];
#pragma unroll
    for (int k = 0; k < ROW_UNROLL; ++k) {
      float f[VEC];
      L::unpack(w[k], f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[k * VEC + i] = f[i];
    }
    accumulate<ENT>(x, c, st, where, v);
  }
  if (tid < p.tail) {
    const float x[1] = {L::up(p.row[p.tail_base + tid])};
    accumulate<ENT>(x, c, st, where, WHERE_TAIL);
  }
  return st;
}

// Block-wide merge in a fixed order; every thread returns the result.  `sm` holds THREADS / 32 + 1 entries.
template <int THREADS>
__device__ __forceinline__ RowStat block_merge(RowStat st, float c, RowStat* sm) {
  constexpr int WARPS = THREADS / 32;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    RowStat other;
    other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    other.u = __shfl_xor_sync(0xffffffffu, st.u, o);
    st = merge(st, other, c);
  }
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = st;
  __syncthreads();
  if (threadIdx.x < 32) {
    st = threadIdx.x < WARPS ? sm[threadIdx.x] : RowStat{-INFINITY, 0.0f, 0.0f};
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      RowStat other;
      other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
      other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
      other.u = __shfl_xor_sync(0xffffffffu, st.u, o);
      st = merge(st, other, c);
    }
    if (threadIdx.x == 0) sm[WARPS] = st;
  }
  __syncthreads();
  return sm[WARPS];
}

// The row's statistics from those of the cluster's blocks, merged in rank order (the same bits in every block).
// `mine` is in shared memory; the caller keeps it alive until its own last cluster barrier.
__device__ __forceinline__ RowStat cluster_merge(cg::cluster_group& cluster, RowStat* mine, int parts, float c) {
  RowStat st = *cluster.map_shared_rank(mine, 0);
  for (int r = 1; r < parts; ++r) st = merge(st, *cluster.map_shared_rank(mine, r), c);
  return st;
}

// ------------------------------------------------------------------ the largest entries
// Order of the selection: larger logit first, ties to the lower index, -0 = +0, NaN ranks with -inf.  A candidate is
// one 64-bit word, the order-preserving image of the logit above the complement of the index; larger is better, no
// two are equal, and 0 is no candidate.
__device__ __forceinline__ uint32_t rank_key(float x) {
  x = isnan(x) ? -INFINITY : x + 0.0f;
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ unsigned long long candidate(uint32_t key, int index) {
  return (static_cast<unsigned long long>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ uint32_t candidate_key(unsigned long long w) { return static_cast<uint32_t>(w >> 32); }
__device__ __forceinline__ int candidate_index(unsigned long long w) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(w));
}

constexpr int TOP_CAPACITY = 2304;  // candidates the buffer holds: 256 units of one 8-element vector, head and tail
template <int THREADS>
struct TopScratch {
  unsigned long long pool[TOP_CAPACITY];
  unsigned long long best[VOCAB_TOP_MAX];  // the part's result, best first
  int hot[THREADS];
  int hot_count, pool_count;
};

// Index of the unit's first element whose key is `key`, in the group `where` that unit_stats recorded.
template <typename T, int THREADS>
__device__ __forceinline__ int find_first(const RowPart<T>& p, int where, uint32_t key) {
  using L = LogitType<T>;
  constexpr int VEC = L::VEC;
  const int tid = threadIdx.x;
  if (where == WHERE_HEAD) return tid;
  if (where == WHERE_TAIL) return p.tail_base + tid;
  if (where == WHERE_START) {  // nothing above -inf: the unit's first element
    if (tid < p.head) return tid;
    if (p.v0 + tid < p.v1) return p.vec_base + (p.v0 + tid) * VEC;
    return p.tail_base + tid;
  }
  int found = INT_MAX;
  for (int k = 0; k < ROW_UNROLL; ++k) {
    const int v = where + k * THREADS;
    if (v >= p.v1) break;
    float f[VEC];
    L::unpack(p.vecs()[v], f);
#pragma unroll
    for (int i = VEC - 1; i >= 0; --i)
      if (rank_key(f[i]) == key) found = min(found, p.vec_base + v * VEC + i);
    if (found != INT_MAX) break;
  }
  return found;
}

// The best `count` of pool[0, n) into best[0, count) in order, by counting for each candidate those above it.
template <int THREADS>
__device__ __forceinline__ void rank_pool(const unsigned long long* pool, int n, int count, unsigned long long* best) {
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const unsigned long long w = pool[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += pool[j] > w;
    if (above < count) best[above] = w;
  }
}

// The `top` best candidates of the block's part into ts.best (0 where the part has fewer).  Every unit's maximum is
// known from the statistics pass.  The top-th largest of those maxima bounds the top-th largest element from below,
// and only the `top` units whose maximum reaches the bound can hold an element that does: those units alone are read
// again (from L2), a warp per unit.  For values without order in the index some top + top^2 / (2 THREADS) elements
// pass.  Where so many pass that the pool overflows, it is cut to the best `top` between steps and the bound raised.
// Ends with a block barrier.
template <typename T, int THREADS>
__device__ void select_top(const RowPart<T>& p, int top, float unit_max, int where, TopScratch<THREADS>& ts) {
  using L = LogitType<T>;
  constexpr int VEC = L::VEC, SHIFT = L::KEY_SHIFT;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool any = tid < p.head || p.v0 + tid < p.v1 || tid < p.tail;
  const uint32_t key = any ? rank_key(unit_max) >> SHIFT : 0u;
  if (tid == 0) ts.hot_count = ts.pool_count = 0;
  for (int i = tid; i < top; i += THREADS) ts.best[i] = 0ull;
  // largest bound that `top` units reach (0: there are fewer units than that)
  uint32_t bound = 0;
  for (int b = 31 - SHIFT; b >= 0; --b) {
    const uint32_t t = bound | (1u << b);
    if (__syncthreads_count(key >= t) >= top) bound = t;
  }
  bool hot = any && key >= bound;
  int last = INT_MAX;  // among elements equal to the bound, the largest index that may count
  if (bound) {
    const int above = __syncthreads_count(key > bound), equal = __syncthreads_count(key == bound);
    if (above + equal > top) {  // ties: those units whose first such element comes first
      const int first = key == bound ? find_first<T, THREADS>(p, where, rank_key(unit_max)) : INT_MAX;
      const int want = top - above;
      last = 0;  // smallest index that `want` of the tied units do not exceed
      for (int b = 30; b >= 0; --b) {
        const int t = last | ((1 << b) - 1);  // all indices with this prefix and bit b clear
        if (__syncthreads_count(key == bound && first <= t) < want) last |= 1 << b;
      }
      hot = key > bound || (key == bound && first <= last);
    }
  }
  // the key's low SHIFT bits follow its sign bit: all ones below zero, all zeros from zero on
  const uint32_t full = SHIFT && bound < (1u << (31 - SHIFT)) ? (bound << SHIFT) | ((1u << SHIFT) - 1u) : bound << SHIFT;
  unsigned long long floor_w = bound ? candidate(full, last) : 1ull;
  if (hot) ts.hot[atomicAdd(&ts.hot_count, 1)] = tid;
  __syncthreads();
  const int units = ts.hot_count;

  auto visit = [&](int unit, int step) {  // lane's share of one step of 32 vectors of a unit
    auto offer = [&](float x, int index) {
      const unsigned long long w = candidate(rank_key(x), index);
      if (w >= floor_w) {
        const int at = atomicAdd(&ts.pool_count, 1);
        if (at < TOP_CAPACITY) ts.pool[at] = w;
      }
    };
    const int v = p.v0 + unit + (step * 32 + lane) * THREADS;
    if (v < p.v1) {
      float f[VEC];
      L::unpack(p.vecs()[v], f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) offer(f[i], p.vec_base + v * VEC + i);
    }
    if (step == 0 && lane == 0) {
      if (unit < p.head) offer(L::up(p.row[unit]), unit);
      if (unit < p.tail) offer(L::up(p.row[p.tail_base + unit]), p.tail_base + unit);
    }
  };
  const int steps = max(1, ((p.v1 - p.v0 + THREADS - 1) / THREADS + 31) / 32);
  for (int i = warp; i < units * steps; i += THREADS / 32) visit(ts.hot[i / steps], i % steps);
  __syncthreads();
  int n = ts.pool_count;
  if (n > TOP_CAPACITY) {
    // a step offers at most 32 * VEC + 2 elements: as many warps at a time as the pool surely has room for
    __syncthreads();
    if (tid == 0) ts.pool_count = 0;
    __syncthreads();
    constexpr int AT_ONCE = (TOP_CAPACITY - VOCAB_TOP_MAX) / (32 * VEC + 2) < THREADS / 32
                                ? (TOP_CAPACITY - VOCAB_TOP_MAX) / (32 * VEC + 2) : THREADS / 32;
    for (int base = 0; base < units * steps; base += AT_ONCE) {
      const int i = base + warp;
      if (warp < AT_ONCE && i < units * steps) visit(ts.hot[i / steps], i % steps);
      __syncthreads();
      n = ts.pool_count;
      __syncthreads();  // every thread has the same n before anyone offers more
      if (n > TOP_CAPACITY - AT_ONCE * (32 * VEC + 2) && base + AT_ONCE < units * steps) {
        rank_pool<THREADS>(ts.pool, n, top, ts.best);
        __syncthreads();
        for (int j = tid; j < top; j += THREADS) ts.pool[j] = ts.best[j];
        if (tid == 0) ts.pool_count = top;
        floor_w = max(floor_w, ts.best[top - 1]);
        __syncthreads();
      }
    }
    n = ts.pool_count;
  }
  rank_pool<THREADS>(ts.pool, n, top, ts.best);
  __syncthreads();
}

// How many words of list[0, n), sorted best first, lie above `w`.
__device__ __forceinline__ int count_above(const unsigned long long* list, int n, unsigned long long w) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (list[mid] > w) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// ------------------------------------------------------------------ gradient pass
// dx_j = p_j (a + b log2 p_j), plus the sparse entries that sparse_fix adds.  p_j = 2^(c (x_j - m) - l2).
struct RowGrad {
  float base;   // m, or 0 for a row without a distribution (every p_j = 2^-inf = 0)
  float l2;     // log2 S
  float a, b;
};
template <bool ENT>
__device__ __forceinline__ float grad_at(float x, float c, const RowGrad& g) {
  const float lg = fmaf(x - g.base, c, -g.l2);
  const float p = ex2_ftz(lg);
  // below 2^-1000 p is 0: the clamp keeps 0 * -inf out (a NaN comes through p)
  return ENT ? p * fmaf(g.b, fmaxf(lg, -1000.0f), g.a) : p * g.a;
}
template <typename T, int THREADS, bool ENT>
__device__ __forceinline__ void dense_grad(const RowPart<T>& p, T* dx, float c, const RowGrad& g, bool same_phase) {
  using L = LogitType<T>;
  constexpr int VEC = L::VEC;
  const int tid = threadIdx.x;
  if (tid < p.head) dx[tid] = L::down(grad_at<ENT>(L::up(p.row[tid]), c, g));
  if (tid < p.tail) dx[p.tail_base + tid] = L::down(grad_at<ENT>(L::up(p.row[p.tail_base + tid]), c, g));
  const uint4* vecs = p.vecs();
  for (int v = p.v0 + tid; v < p.v1; v += THREADS * ROW_UNROLL) {
    uint4 w[ROW_UNROLL];
#pragma unroll
    for (int k = 0; k < ROW_UNROLL; ++k)
      if (v + k * THREADS < p.v1) w[k] = vecs[v + k * THREADS];
#pragma unroll
    for (int k = 0; k < ROW_UNROLL; ++k) {
      if (v + k * THREADS >= p.v1) continue;
      float f[VEC];
      L::unpack(w[k], f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] = grad_at<ENT>(f[i], c, g);
      T* out = dx + p.vec_base + (v + k * THREADS) * VEC;
      if (same_phase) {
        *reinterpret_cast<uint4*>(out) = L::pack(f);
      } else {  // logits and gradient start at different offsets within 16 bytes
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = L::down(f[i]);
      }
    }
  }
}
template <typename T, int THREADS>
__device__ __forceinline__ void zero_grad(const RowPart<T>& p, T* dx, bool same_phase) {
  constexpr int VEC = LogitType<T>::VEC;
  const int tid = threadIdx.x;
  const T zero = LogitType<T>::down(0.0f);
  if (tid < p.head) dx[tid] = zero;
  if (tid < p.tail) dx[p.tail_base + tid] = zero;
  for (int v = p.v0 + tid; v < p.v1; v += THREADS) {
    T* out = dx + p.vec_base + v * VEC;
    if (same_phase) {
      *reinterpret_cast<uint4*>(out) = make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = zero;
    }
  }
}
// Entries (index, weight) added to the gradient: each is written once, as the rounding of dense value plus the sum of
// all weights with its index, in list order (the same index may come several times).  idx < 0 marks no entry.  Runs
// after the block barrier that follows dense_grad.
template <typename T, int THREADS, bool ENT>
__device__ __forceinline__ void sparse_fix(const RowPart<T>& p, T* dx, float c, const RowGrad& g, const int* idx,
                                           const float* weight, int n) {
  using L = LogitType<T>;
  for (int e = threadIdx.x; e < n; e += THREADS) {
    const int j = idx[e];
    if (j < 0 || !owns(p, j)) continue;
    float w = 0.0f;
    bool leader = true;
    for (int k = 0; k < n; ++k) {
      if (idx[k] != j) continue;
      leader = leader && k >= e;
      w += weight[k];
    }
    if (leader) dx[j] = L::down(grad_at<ENT>(L::up(p.row[j]), c, g) + w);
  }
}

// Row merging in small vectors: max and sum over the block, in a fixed order.  `sm`: THREADS / 32 floats.
template <int THREADS, bool MAX>
__device__ __forceinline__ float block_fold(float v, float* sm) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, w) : v + w;
  }
  __syncthreads();  // the previous use of sm is over
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
#pragma unroll
  for (int k = 1; k < THREADS / 32; ++k) v = MAX ? fmaxf(v, sm[k]) : v + sm[k];
  return v;
}

}  // namespace mtb
