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
#include "ptx_sm100.cuh"

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

// Four words into the shared memory of block `rank` of the cluster, at the place that `to` has in this block; they count on
// the barrier of that block at the place of `bar`.
__device__ __forceinline__ void send_async(const void* to, const unsigned long long* bar, int rank, float4 v) {
  asm volatile(
      "{\n\t.reg .b32 ra, rb;\n\tmapa.shared::cluster.u32 ra, %0, %2;\n\tmapa.shared::cluster.u32 rb, %1, %2;\n\t"
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [ra], {%3, %4, %5, %6}, [rb];\n\t}"
      ::"r"(smem_u32(to)), "r"(smem_u32(bar)), "r"(rank), "r"(__float_as_uint(v.x)), "r"(__float_as_uint(v.y)),
      "r"(__float_as_uint(v.z)), "r"(__float_as_uint(v.w))
      : "memory");
}

// Cluster barrier that orders no memory operations, in two halves.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }

// Two f32 operations per instruction, each rounded as its scalar form.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// ------------------------------------------------------------------ element types
template <typename T>
struct LogitType;
template <>
struct LogitType<float> {
  static constexpr int VEC = 4;
  static constexpr uint32_t NEG_INF_WORD = 0xff800000u;
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&f)[4]) {
    f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y); f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
  }
  // largest and least of N vectors; NaN counts as nothing
  template <int N>
  static __device__ __forceinline__ float most(const uint4 (&w)[N]) {
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < N; ++k)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(w[k].x), __uint_as_float(w[k].y)), fmaxf(__uint_as_float(w[k].z), __uint_as_float(w[k].w))));
    return m;
  }
  template <int N>
  static __device__ __forceinline__ float least(const uint4 (&w)[N]) {
    float m = INFINITY;
#pragma unroll
    for (int k = 0; k < N; ++k)
      m = fminf(m, fminf(fminf(__uint_as_float(w[k].x), __uint_as_float(w[k].y)), fminf(__uint_as_float(w[k].z), __uint_as_float(w[k].w))));
    return m;
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct LogitType<__nv_bfloat16> {
  static constexpr int VEC = 8;
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
  template <int N>
  static __device__ __forceinline__ float most(const uint4 (&w)[N]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
    __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
#pragma unroll
    for (int k = 1; k < N; ++k) m = __hmax2(m, __hmax2(__hmax2(h[4 * k], h[4 * k + 1]), __hmax2(h[4 * k + 2], h[4 * k + 3])));
    return fmaxf(__low2float(m), __high2float(m));
  }
  template <int N>
  static __device__ __forceinline__ float least(const uint4 (&w)[N]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
    __nv_bfloat162 m = __hmin2(__hmin2(h[0], h[1]), __hmin2(h[2], h[3]));
#pragma unroll
    for (int k = 1; k < N; ++k) m = __hmin2(m, __hmin2(__hmin2(h[4 * k], h[4 * k + 1]), __hmin2(h[4 * k + 2], h[4 * k + 3])));
    return fminf(__low2float(m), __high2float(m));
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
  template <int N>
  static __device__ __forceinline__ float most(const uint4 (&w)[N]) {
    const __half2* h = reinterpret_cast<const __half2*>(&w);
    __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
#pragma unroll
    for (int k = 1; k < N; ++k) m = __hmax2(m, __hmax2(__hmax2(h[4 * k], h[4 * k + 1]), __hmax2(h[4 * k + 2], h[4 * k + 3])));
    return fmaxf(__low2float(m), __high2float(m));
  }
  template <int N>
  static __device__ __forceinline__ float least(const uint4 (&w)[N]) {
    const __half2* h = reinterpret_cast<const __half2*>(&w);
    __half2 m = __hmin2(__hmin2(h[0], h[1]), __hmin2(h[2], h[3]));
#pragma unroll
    for (int k = 1; k < N; ++k) m = __hmin2(m, __hmin2(__hmin2(h[4 * k], h[4 * k + 1]), __hmin2(h[4 * k + 2], h[4 * k + 3])));
    return fminf(__low2float(m), __high2float(m));
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

// The threads that work on one row (or on one part of it): a warp, or the whole block.
template <int G>
struct Group {
  static constexpr int WARPS = G / 32;
  static __device__ __forceinline__ int rank() { return G == 32 ? threadIdx.x & 31 : threadIdx.x; }
  static __device__ __forceinline__ void sync() {
    if (G == 32) __syncwarp();
    else __syncthreads();
  }
  static __device__ __forceinline__ int count(bool b) {  // threads that say yes; a barrier
    return G == 32 ? __popc(__ballot_sync(0xffffffffu, b)) : __syncthreads_count(b);
  }
};

// The part of one row that one group works on.  Only whole 16-byte vectors inside the row are read as vectors; the
// elements before the first boundary (`head`) belong to the row's first part and those after the last one (`tail`)
// to its last part, and are read one by one.  Thread t of G owns head element t, the vectors v0 + t, v0 + t + G,
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
  const int share = static_cast<int>(static_cast<unsigned>(nv) / static_cast<unsigned>(parts)), more = nv - share * parts;
  p.v0 = share * part + min(part, more);  // the first `more` parts have one vector more
  p.v1 = p.v0 + share + (part < more);
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

// ------------------------------------------------------------------ order of the selection
// Larger logit first, ties to the lower index, -0 = +0, NaN ranks with -inf.  A candidate is one 64-bit word, the
// order-preserving image of the logit above the complement of the index; larger is better, no two are equal, and 0 is no
// candidate.
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

// ------------------------------------------------------------------ statistics
struct RowStat {
  float m, s, u;
};
// The same sums relative to another, not smaller maximum.  -inf from -inf (or +inf from +inf) must not turn 0 into NaN: the
// difference is clamped to the largest finite magnitude, whose power of two is 0.  Sums that are scaled to nothing drop out
// whole (0 * (s * d) could be 0 * inf); a NaN stays.
__device__ __forceinline__ void rescale(float from, float to, float c, float& s, float& u) {
  const float d = fmaxf(from - to, -FLT_MAX);
  const float r = ex2_ftz(d * c);
  u = r == 0.0f ? s * 0.0f : r * fmaf(s, d, u);
  s *= r;
}
// Merge over the lanes of a warp, in a fixed order; every lane returns it.
__device__ __forceinline__ RowStat warp_merge(RowStat st, float c) {
  const float m = key_value(__reduce_max_sync(0xffffffffu, rank_key(st.m)));
  rescale(st.m, m, c, st.s, st.u);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
    st.u += __shfl_xor_sync(0xffffffffu, st.u, o);
  }
  st.m = m;
  return st;
}

// Vectors a thread takes up together, in one round: four loads in flight.
constexpr int ROW_UNROLL = 4;

// For the selection, a part's vectors are cut into at most SLOTS spans per thread, and the upper half of the largest
// key of each span is kept.
constexpr int SLOTS = 16;
template <int G>
struct Spans {
  static constexpr int U = ROW_UNROLL;
  static_assert(U == 4, "bits()");
  int shift;  // a span is U << shift vectors of a unit
  __device__ __forceinline__ explicit Spans(int vectors) {
    const int rounds = (vectors + G * U - 1) / (G * U);
    shift = rounds <= SLOTS ? 0 : 32 - __clz((rounds - 1) / SLOTS);
  }
  __device__ __forceinline__ int size() const { return U << shift; }
  __device__ __forceinline__ int bits() const { return shift + 2; }
};

// A thread's running sums, relative to the maximum that its warp has met so far: that rises in few rounds (in the n-th
// with probability 1 / n), where some lane's own maximum rises in nearly all of them.  The pairs are two independent
// halves.  For the selection, m is the thread's own maximum and `where` the vector that holds it first, or WHERE_HEAD /
// WHERE_TAIL / WHERE_START (nothing above -inf was seen).
constexpr int WHERE_START = -1, WHERE_HEAD = -2, WHERE_TAIL = -3;
struct UnitStat {
  float base = -INFINITY, m = -INFINITY;
  float2 s = {0.0f, 0.0f}, u = {0.0f, 0.0f};
  int where = WHERE_START;
  __device__ __forceinline__ RowStat sum() const { return {base, s.x + s.y, u.x + u.y}; }
  // by all lanes of the warp
  __device__ __forceinline__ void raise(float top, float c) {
    if (!__any_sync(0xffffffffu, top > base)) return;
    const float to = key_value(__reduce_max_sync(0xffffffffu, rank_key(fmaxf(top, base))));
    rescale(base, to, c, s.x, u.x);
    rescale(base, to, c, s.y, u.y);
    base = to;
  }
  __device__ __forceinline__ void own(float x, int here) {
    if (x > m) {
      m = x;
      where = here;
    }
  }
  template <bool ENT>
  __device__ __forceinline__ void add_one(float x, float c) {  // x is not above base
    const float d = x - (base == -INFINITY ? 0.0f : base);
    const float e = ex2_ftz(d * c);
    s.x += e;
    if (ENT) u.x = fmaf(e, fmaxf(d, -FLT_MAX), u.x);
  }
};
// CLEAN: no difference is -inf (or the row is NaN anyway)
template <typename T, bool ENT, bool CLEAN>
__device__ __forceinline__ void add_vector(float2& s, float2& u, const uint4& w, float base, float c) {
  using L = LogitType<T>;
  float f[L::VEC];
  L::unpack(w, f);
  const float2 nb = make_float2(-base, -base), cc = make_float2(c, c);
#pragma unroll
  for (int i = 0; i < L::VEC; i += 2) {
    float2 d = add2(make_float2(f[i], f[i + 1]), nb);
    const float2 g = mul2(d, cc);
    const float2 e = make_float2(ex2_ftz(g.x), ex2_ftz(g.y));
    s = add2(s, e);
    if (ENT) {
      if (!CLEAN) d = make_float2(fmaxf(d.x, -FLT_MAX), fmaxf(d.y, -FLT_MAX));
      u = fma2(e, d, u);
    }
  }
}

// The thread's unit, reduced.  All threads of a warp call it together.
template <typename T, int G, bool ENT, bool TOP>
__device__ __forceinline__ UnitStat unit_stats(const RowPart<T>& p, float c, uint16_t (*slots)[G]) {
  using L = LogitType<T>;
  constexpr int U = ROW_UNROLL;
  const int tid = Group<G>::rank();
  const Spans<G> spans(p.v1 - p.v0);
  float span_top = -INFINITY;
  int round = 0;
  UnitStat st;
  auto take = [&](const uint4 (&w)[U], int v) {  // one round of the whole warp
    float top = -INFINITY;
    if (TOP) {
      float most[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const uint4 one[1] = {w[k]};
        top = fmaxf(top, most[k] = L::most(one));
      }
      if (top > st.m) {
        st.m = top;
#pragma unroll
        for (int k = U - 1; k >= 0; --k)
          if (most[k] == top) st.where = v + k * G;
      }
      span_top = fmaxf(span_top, top);
      ++round;
      if ((round & ((1 << spans.shift) - 1)) == 0 || v + G * U >= p.v1) {
        if (v < p.v1) slots[(round - 1) >> spans.shift][tid] = static_cast<uint16_t>(rank_key(span_top) >> 16);
        span_top = -INFINITY;
      }
    } else {
      top = L::most(w);
    }
    st.raise(top, c);
    const float base = st.base == -INFINITY ? 0.0f : st.base;
    // a masked element, or finite ones too far apart, make a difference of -inf
    if (!ENT || L::least(w) - base > -INFINITY) {
#pragma unroll
      for (int k = 0; k < U; ++k) add_vector<T, ENT, true>(st.s, st.u, w[k], base, c);
    } else {
#pragma unroll
      for (int k = 0; k < U; ++k) add_vector<T, ENT, false>(st.s, st.u, w[k], base, c);
    }
  };
  if (TOP && tid < p.head) st.own(L::up(p.row[tid]), WHERE_HEAD);
  const uint4* vecs = p.vecs();
  int v = p.v0;
#pragma unroll 1  // a second round's loads would cost the registers of another block
  for (; v + G * U <= p.v1; v += G * U) {
    uint4 w[U];
#pragma unroll
    for (int k = 0; k < U; ++k) w[k] = vecs[v + tid + k * G];
    take(w, v + tid);
  }
  if (v < p.v1) {
    uint4 w[U];
#pragma unroll
    for (int k = 0; k < U; ++k)
      w[k] = v + tid + k * G < p.v1 ? vecs[v + tid + k * G]
                                    : make_uint4(L::NEG_INF_WORD, L::NEG_INF_WORD, L::NEG_INF_WORD, L::NEG_INF_WORD);
    take(w, v + tid);
  }
  if (TOP && tid < p.tail) st.own(L::up(p.row[p.tail_base + tid]), WHERE_TAIL);
  if (p.head || p.tail) {
    const float x = tid < p.head ? L::up(p.row[tid]) : -INFINITY, y = tid < p.tail ? L::up(p.row[p.tail_base + tid]) : -INFINITY;
    st.raise(fmaxf(x, y), c);
    if (tid < p.head) st.add_one<ENT>(x, c);
    if (tid < p.tail) st.add_one<ENT>(y, c);
  }
  return st;
}

// Merge over the group in a fixed order; every thread returns the result.  `sm` holds Group<G>::WARPS + 1 entries and
// is not used for a warp.
template <int G>
__device__ __forceinline__ RowStat group_merge(RowStat st, float c, RowStat* sm) {
  constexpr int WARPS = Group<G>::WARPS;
  st = warp_merge(st, c);
  if (G == 32) return st;
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = st;
  Group<G>::sync();
  if (threadIdx.x < 32) {
    st = warp_merge(threadIdx.x < WARPS ? sm[threadIdx.x] : RowStat{-INFINITY, 0.0f, 0.0f}, c);
    if (threadIdx.x == 0) sm[WARPS] = st;
  }
  Group<G>::sync();
  return sm[WARPS];
}

// The row's statistics from those of its parts, merged in their order.
__device__ __forceinline__ RowStat parts_merge(const RowStat* parts, int n, float c) {
  RowStat st = {parts[0].m, 0.0f, 0.0f};
  for (int q = 1; q < n; ++q) st.m = fmaxf(st.m, parts[q].m);
  for (int q = 0; q < n; ++q) {
    float s = parts[q].s, u = parts[q].u;
    rescale(parts[q].m, st.m, c, s, u);
    st.s += s;
    st.u += u;
  }
  return st;
}

// ------------------------------------------------------------------ the largest entries
template <int G>
struct TopScratch {
  static constexpr int MOST = G < VOCAB_TOP_MAX ? G : VOCAB_TOP_MAX;  // largest `top`
  // A part with fewer units than `top` has at most one vector a unit and 14 single elements: 255 * 8 + 14 candidates for
  // a block, 31 * 8 + 14 for a warp.
  static constexpr int CAPACITY = G == 32 ? 384 : G < VOCAB_TOP_MAX ? 1152 : 2304;
  // units looked at: `top` and a few more
  static __host__ __device__ constexpr int limit(int top) { return top + top / 16 + 16; }
  static constexpr int UNITS = limit(MOST) < G ? limit(MOST) : G;
  unsigned long long pool[CAPACITY];
  unsigned long long best[MOST];  // the part's result, best first
  static constexpr int HITS = G;
  int hot[UNITS];                 // the units looked at
  int hits[HITS];                 // spans read again: unit | slot << 16
  uint16_t slots[SLOTS][G];       // upper halves of the spans' largest keys
  uint32_t nth[Group<G>::WARPS], most[Group<G>::WARPS];
  int hot_count, hit_count, pool_count;
};

// Calls f(i, above) for each entry i of list[0, n) with the number of entries above it, from one thread each.  As many
// threads as there are to spare share an entry.  Every thread of the group takes part.
template <int G, typename F>
__device__ __forceinline__ void for_each_rank(const unsigned long long* list, int n, F f) {
  const int tid = Group<G>::rank();
  const int bits = n > 1 ? max(0, min(5, __clz(n - 1) - __clz(G) - 1)) : 5;  // 1 << bits threads per entry: n << bits <= G
  const int sub = tid & ((1 << bits) - 1);
  for (int base = (tid & ~31) >> bits; base < n; base += G >> bits) {  // whole warps leave
    const int i = base + ((tid & 31) >> bits);
    const unsigned long long w = i < n ? list[i] : ~0ull;
    int above = 0;
#pragma unroll 4
    for (int j = sub; j < n; j += 1 << bits) above += list[j] > w;
    for (int o = (1 << bits) >> 1; o; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
    if (i < n && sub == 0) f(i, above);
  }
}
// The best `count` of pool[0, n) into best[0, count) in order, by counting, or by a bitonic sort where counting would take
// longer (n^2 / 128 steps of a warp).  With a candidate for each of 512 threads the sort goes by shuffles within a warp
// and through the pool across warps; with more candidates, which few units of many alternatives or ties bring about, in
// the pool (`room` words, those behind n are free).  Every thread of the group takes part.
template <int G>
__device__ __forceinline__ void rank_pool(unsigned long long* pool, int n, int room, int count, unsigned long long* best) {
  const int tid = Group<G>::rank();
  if (G == 512 && n > 160 && n <= G) {
    unsigned long long w = tid < n ? pool[tid] : 0ull;
    for (int size = 2; size <= G; size <<= 1) {
      const bool down = (tid & size) == 0 || size == G;
      for (int o = size >> 1; o; o >>= 1) {
        unsigned long long other;
        if (o >= 32) {
          Group<G>::sync();
          pool[tid] = w;
          Group<G>::sync();
          other = pool[tid ^ o];
        } else {
          other = __shfl_xor_sync(0xffffffffu, w, o);
        }
        w = ((tid & o) == 0) == down ? max(w, other) : min(w, other);
      }
    }
    if (tid < count) best[tid] = w;
    return;
  }
  const int all = n > 1 ? 1 << (32 - __clz(n - 1)) : 1;
  if (n > 512 && all <= room) {
    for (int i = n + tid; i < all; i += G) pool[i] = 0ull;
    Group<G>::sync();
    for (int size = 2; size <= all; size <<= 1)
      for (int o = size >> 1; o; o >>= 1) {
        for (int i = tid; i < all / 2; i += G) {
          const int a = 2 * i - (i & (o - 1)), b = a + o;  // i-th pair that is o apart
          const unsigned long long x = pool[a], y = pool[b];
          if ((x < y) == ((a & size) == 0)) {
            pool[a] = y;
            pool[b] = x;
          }
        }
        Group<G>::sync();
      }
    for (int i = tid; i < count; i += G) best[i] = pool[i];
    return;
  }
  for_each_rank<G>(pool, n, [&](int i, int above) {
    if (above < count) best[above] = pool[i];
  });
}

// The `top` best candidates of the group's part into ts.best (0 where the part has fewer); top <= MOST.
//  1. Every unit's maximum and its place are known from the statistics pass.  A key that at least `top` units reach bounds
//     the top-th largest element from below: the least of the warps' ceil(top / warps)-th largest maxima.  Where many more
//     units reach it, it is raised by bisection, and among units with equal keys by place, to just over `top` units.
//  2. Only the units at or above the bound can hold an element that counts, and of those only the spans whose own largest
//     key reaches it: these spans are read again.  For values without order in the index some r + r^2 / (2 G) elements of r
//     units pass.  Where so many pass that the pool overflows, the units' vectors are gone through in rounds between
//     which the pool is cut to the best `top` and the bound raised.
//  3. Counting puts the candidates in order.
// Ends with a group barrier.
template <typename T, int G>
__device__ void select_top(const RowPart<T>& p, int top, float unit_max, int where, TopScratch<G>& ts) {
  using L = LogitType<T>;
  constexpr int VEC = L::VEC, WARPS = Group<G>::WARPS, CAPACITY = TopScratch<G>::CAPACITY;
  const int tid = Group<G>::rank(), lane = tid & 31, warp = tid >> 5;
  const bool any = tid < p.head || p.v0 + tid < p.v1 || tid < p.tail;
  const uint32_t key = any ? rank_key(unit_max) : 0u;
  // the last index at which the unit's first maximum can be: a bound from below on its candidate word
  int place;
  if (where == WHERE_HEAD || (where == WHERE_START && tid < p.head)) place = tid;
  else if (where == WHERE_TAIL || (where == WHERE_START && p.v0 + tid >= p.v1)) place = p.tail_base + tid;
  else place = p.vec_base + (where == WHERE_START ? p.v0 + tid : where) * VEC + VEC - 1;
  if (tid == 0) ts.hot_count = ts.hit_count = ts.pool_count = 0;
  for (int i = tid; i < top; i += G) ts.best[i] = 0ull;

  uint32_t low, high = __reduce_max_sync(0xffffffffu, key);
  {
    bool taken = false;
    low = high;
    for (int j = (top + WARPS - 1) / WARPS;;) {
      const unsigned who = __ballot_sync(0xffffffffu, !taken && key == low);
      if (--j == 0) break;
      taken = taken || lane == __ffs(who) - 1;
      low = __reduce_max_sync(0xffffffffu, taken ? 0u : key);
    }
  }
  if (WARPS > 1) {
    if (lane == 0) {
      ts.nth[warp] = low;
      ts.most[warp] = high;
    }
    Group<G>::sync();
    low = __reduce_min_sync(0xffffffffu, lane < WARPS ? ts.nth[lane] : ~0u);
    high = __reduce_max_sync(0xffffffffu, lane < WARPS ? ts.most[lane] : 0u);
  }
  low = max(low, 1u);  // 0 is no unit
  const int limit = min(TopScratch<G>::limit(top), TopScratch<G>::UNITS);
  int reach = Group<G>::count(key >= low);
  int last = INT_MAX;  // of the units with key `low`, those up to this place
  if (reach > limit) {
    ++high;  // reached by none
    while (reach > limit && high - low > 1) {
      const uint32_t mid = low + (high - low) / 2;
      const int c = Group<G>::count(key >= mid);
      if (c >= top) {
        low = mid;
        reach = c;
      } else {
        high = mid;
      }
    }
    if (reach > limit) {  // ties
      const int want = top - Group<G>::count(key > low);
      last = 0;  // becomes the smallest place that `want` of the tied units do not exceed
      for (int b = 30; b >= 0; --b) {
        const int t = last | ((1 << b) - 1);  // all places with this prefix and bit b clear
        if (Group<G>::count(key == low && place <= t) < want) last |= 1 << b;
      }
    }
  }
  const bool hot = key > low || (key == low && place <= last);
  unsigned long long floor_w = candidate(low, last);
  {
    const unsigned who = __ballot_sync(0xffffffffu, hot);
    int at = 0;
    if (lane == 0 && who) at = atomicAdd(&ts.hot_count, __popc(who));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
    if (hot) ts.hot[at] = tid;
  }
  Group<G>::sync();
  const int units = ts.hot_count;

  auto offer = [&](float x, int index) {
    const unsigned long long w = candidate(rank_key(x), index);
    if (w >= floor_w) {
      const int at = atomicAdd(&ts.pool_count, 1);
      if (at < CAPACITY) ts.pool[at] = w;
    }
  };
  const Spans<G> spans(p.v1 - p.v0);
  auto passes = [&](int unit, int slot) { return ts.slots[slot][unit] >= static_cast<uint32_t>(floor_w >> 48); };
  auto offer_vector = [&](const uint4& w, int v) {
    float f[VEC];
    L::unpack(w, f);
#pragma unroll
    for (int i = 0; i < VEC; ++i) offer(f[i], p.vec_base + v * VEC + i);
  };
  auto offer_singles = [&]() {
    if (tid < p.head) offer(L::up(p.row[tid]), tid);
    if (tid < p.tail) offer(L::up(p.row[p.tail_base + tid]), p.tail_base + tid);
  };
  const int each = (p.v1 - p.v0 + G - 1) / G;                           // vectors of a unit, some one less
  const int span_bits = each > spans.size() ? 32 - __clz((each - 1) / spans.size()) : 0;  // spans per unit, a power of two
  for (int i = tid; i < units << span_bits; i += G) {
    const int unit = ts.hot[i >> span_bits], slot = i & ((1 << span_bits) - 1);
    if (p.v0 + unit + slot * spans.size() * G < p.v1 && passes(unit, slot)) {
      const int at = atomicAdd(&ts.hit_count, 1);
      if (at < TopScratch<G>::HITS) ts.hits[at] = unit | slot << 16;
    }
  }
  offer_singles();
  Group<G>::sync();
  const int hits = ts.hit_count;
  if (hits <= TopScratch<G>::HITS) {
    for (int i = tid; i < hits << spans.bits(); i += G) {
      const int hit = ts.hits[i >> spans.bits()];
      const int v = p.v0 + (hit & 0xffff) + ((hit >> 16) * spans.size() + (i & (spans.size() - 1))) * G;
      if (v < p.v1) offer_vector(p.vecs()[v], v);
    }
  }
  Group<G>::sync();
  int n = ts.pool_count;
  if (n > CAPACITY || hits > TopScratch<G>::HITS) {
    // as many vectors at a time as the pool surely has room for beside the best
    constexpr int ROOM = (CAPACITY - TopScratch<G>::MOST - 2 * VEC) / VEC;
    constexpr int AT_ONCE = ROOM < G ? ROOM : G;
    static_assert(AT_ONCE >= 1, "the pool must hold one vector beside the best");
    Group<G>::sync();
    if (tid == 0) ts.pool_count = 0;
    Group<G>::sync();
    offer_singles();
    const long long total = static_cast<long long>(units) * each;
    for (long long base = 0; base < total; base += AT_ONCE) {
      const long long i = base + tid;
      if (tid < AT_ONCE && i < total) {
        const int unit = ts.hot[i / each], j = static_cast<int>(i % each), v = p.v0 + unit + j * G;
        if (v < p.v1 && passes(unit, j / spans.size())) offer_vector(p.vecs()[v], v);
      }
      Group<G>::sync();
      n = ts.pool_count;
      Group<G>::sync();  // every thread has the same n before anyone offers more
      if (n > CAPACITY - AT_ONCE * VEC && base + AT_ONCE < total) {
        rank_pool<G>(ts.pool, n, CAPACITY, top, ts.best);
        Group<G>::sync();
        for (int j = tid; j < top; j += G) ts.pool[j] = ts.best[j];
        if (tid == 0) ts.pool_count = top;
        floor_w = max(floor_w, ts.best[top - 1]);
        Group<G>::sync();
      }
    }
  }
  rank_pool<G>(ts.pool, n, CAPACITY, top, ts.best);
  Group<G>::sync();
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
constexpr int GRAD_UNROLL = 4;  // vectors a thread keeps in flight
template <typename T, bool ENT>
__device__ __forceinline__ void grad_vector(T* out, const uint4& w, float c, const RowGrad& g, bool same_phase) {
  using L = LogitType<T>;
  float f[L::VEC];
  L::unpack(w, f);
  const float2 nb = make_float2(-g.base, -g.base), cc = make_float2(c, c), nl = make_float2(-g.l2, -g.l2);
  const float2 ga = make_float2(g.a, g.a), gb = make_float2(g.b, g.b);
#pragma unroll
  for (int i = 0; i < L::VEC; i += 2) {  // grad_at, two at a time
    const float2 lg = fma2(add2(make_float2(f[i], f[i + 1]), nb), cc, nl);
    const float2 p = make_float2(ex2_ftz(lg.x), ex2_ftz(lg.y));
    const float2 o = mul2(p, ENT ? fma2(gb, make_float2(fmaxf(lg.x, -1000.0f), fmaxf(lg.y, -1000.0f)), ga) : ga);
    f[i] = o.x;
    f[i + 1] = o.y;
  }
  if (same_phase) {
    *reinterpret_cast<uint4*>(out) = L::pack(f);
  } else {  // logits and gradient start at different offsets within 16 bytes
#pragma unroll
    for (int i = 0; i < L::VEC; ++i) out[i] = L::down(f[i]);
  }
}
template <typename T, int G, bool ENT>
__device__ __forceinline__ void dense_grad(const RowPart<T>& p, T* dx, float c, const RowGrad& g, bool same_phase) {
  using L = LogitType<T>;
  constexpr int VEC = L::VEC, U = GRAD_UNROLL;
  const int tid = Group<G>::rank();
  if (tid < p.head) dx[tid] = L::down(grad_at<ENT>(L::up(p.row[tid]), c, g));
  if (tid < p.tail) dx[p.tail_base + tid] = L::down(grad_at<ENT>(L::up(p.row[p.tail_base + tid]), c, g));
  const uint4* vecs = p.vecs() + tid;
  T* out = dx + p.vec_base + tid * VEC;
  int v = p.v0;
#pragma unroll 1
  for (; v + G * U <= p.v1; v += G * U) {
    uint4 w[U];
#pragma unroll
    for (int k = 0; k < U; ++k) w[k] = vecs[v + k * G];
#pragma unroll
    for (int k = 0; k < U; ++k) grad_vector<T, ENT>(out + (v + k * G) * VEC, w[k], c, g, same_phase);
  }
  for (; v + tid < p.v1; v += G) grad_vector<T, ENT>(out + v * VEC, vecs[v], c, g, same_phase);
}
template <typename T>
__device__ __forceinline__ void zero_vector(T* out, bool same_phase) {
  if (same_phase) {
    *reinterpret_cast<uint4*>(out) = make_uint4(0u, 0u, 0u, 0u);
  } else {
#pragma unroll
    for (int i = 0; i < LogitType<T>::VEC; ++i) out[i] = LogitType<T>::down(0.0f);
  }
}
template <typename T, int G>
__device__ __forceinline__ void zero_grad(const RowPart<T>& p, T* dx, bool same_phase) {
  constexpr int VEC = LogitType<T>::VEC;
  const int tid = Group<G>::rank();
  const T zero = LogitType<T>::down(0.0f);
  if (tid < p.head) dx[tid] = zero;
  if (tid < p.tail) dx[p.tail_base + tid] = zero;
  for (int v = p.v0 + tid; v < p.v1; v += G) zero_vector<T>(dx + p.vec_base + v * VEC, same_phase);
}
// Entries (index, weight) added to the gradient: each is written once, as the rounding of dense value plus the sum of
// all weights with its index, in list order (the same index may come several times).  idx < 0 marks no entry; the list is
// 16-byte aligned and read four at a time, up to three places beyond n (fill_list).  Runs after the group barrier that
// follows dense_grad.
template <int G>
__device__ __forceinline__ void fill_list(int* idx, int n) {  // before a group barrier
  if (Group<G>::rank() < (-n & 3)) idx[n + Group<G>::rank()] = -1;
}
template <typename T, int G, bool ENT>
__device__ __forceinline__ void sparse_fix(const RowPart<T>& p, T* dx, float c, const RowGrad& g, const int* idx,
                                           const float* weight, int n) {
  using L = LogitType<T>;
  const int4* list = reinterpret_cast<const int4*>(idx);
  for (int e = Group<G>::rank(); e < n; e += G) {
    const int j = idx[e];
    if (j < 0 || !owns(p, j)) continue;
    int same = 0, first = INT_MAX;
#pragma unroll 4
    for (int k = 0; k < (n + 3) / 4; ++k) {
      const int4 w = list[k];
      const int hits = (w.x == j) | (w.y == j) << 1 | (w.z == j) << 2 | (w.w == j) << 3;
      if (hits) {
        same += __popc(hits);
        first = min(first, 4 * k + __ffs(hits) - 1);
      }
    }
    if (first != e) continue;
    float w = weight[e];
    if (same > 1) {
      w = 0.0f;
      for (int k = 0; k < n; ++k)
        if (idx[k] == j) w += weight[k];
    }
    dx[j] = L::down(grad_at<ENT>(L::up(p.row[j]), c, g) + w);
  }
}

// Maximum or sum over the group, in a fixed order; every thread returns it.  `sm`: Group<G>::WARPS floats, not used for
// a warp.
template <int G, bool MAX>
__device__ __forceinline__ float group_fold(float v, float* sm) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, w) : v + w;
  }
  if (G == 32) return v;
  Group<G>::sync();  // the previous use of sm is over
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  Group<G>::sync();
  v = sm[0];
#pragma unroll
  for (int k = 1; k < Group<G>::WARPS; ++k) v = MAX ? fmaxf(v, sm[k]) : v + sm[k];
  return v;
}

}  // namespace mtb
