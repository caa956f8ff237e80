// Log-probabilities of chosen labels under rows of logits, their gradient, and the two losses built on them: paired
// log ratios (preferences) and the clipped policy ratio with a KL term.
//
// For a row x of V logits with label l:  m = max_j x_j,  s = sum_j exp(x_j - m),  log p_l = (x_l - m) - log s, and
// d(log p_l)/dx_j = [j = l] - exp(x_j - m) / s.  Statistics are fp32; the one value per row that is compared with
// other models' values (log p_l) is formed in fp64, because sequences sum thousands of them and take differences.
// A row without a label (label < 0, or owner < 0 where owners are given) is not read: log-probability 0, gradient 0.
// A label >= V gives NaN (the call cannot look at device memory without a wait).  A coefficient of zero gives a gradient
// of zero, and a weight of zero no term of a loss, whatever else the row holds: masks come that way, and behind them may
// be infinities and NaN.
#include "../../include/jtvae_hip.h"
#include "jtvae_common.h"

namespace {

using namespace jtvae;

constexpr float kLog2e = 1.44269504088896340736f;

inline int launch_status() {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}

inline unsigned grid_for(long total) { return (unsigned)((total + JTVAE_BLOCK - 1) / JTVAE_BLOCK); }

// exp(x) on the hardware's exp2.  The product with log2 e is rounded, so the result is off by up to |x| 2^-24 relative to
// itself: far from the maximum, where a softmax is small, as much as the difference x - max is rounded by anyway.  Making up
// for what the product loses brings the worst element of fp32 gradients (standard deviation 4) from 2^-18.5 to 2^-19.6 of itself
// and the log-probabilities nowhere (1e-6 at 780 columns both ways), for 13.6 -> 15.7 us of statistics at 20480 x 780.
__device__ __forceinline__ float exp_nat(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

struct Labels {
  const void* at;
  int bits;
  __device__ long operator[](long i) const {
    return bits == 64 ? (long)((const int64_t*)at)[i] : (long)((const int32_t*)at)[i];
  }
};

// Running maximum and sum of exp(x - max).  With nothing but -inf so far the sum is 0 and exponents are taken against
// 0, so that exp(-inf - -inf) never appears; a NaN or +inf logit makes the sum NaN.
struct RowStat {
  float m, s;
};

__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ RowStat join(RowStat a, RowStat b) {
  const float m = fmaxf(a.m, b.m), ref = finite_or_zero(m);
  RowStat r;
  r.m = m;
  r.s = a.s * exp_nat(a.m - ref) + b.s * exp_nat(b.m - ref);
  return r;
}

__device__ __forceinline__ RowStat wave_join(RowStat v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    RowStat o = {__shfl_xor(v.m, off, 64), __shfl_xor(v.s, off, 64)};
    v = join(v, o);
  }
  return v;
}

template <typename T>
__device__ __forceinline__ double label_log_prob(const T* row, long label, int n_cols, RowStat st) {
  if (label >= n_cols) return (double)NAN;
  return ((double)(float)row[label] - (double)st.m) - log((double)st.s);
}

// Sixteen bytes of a row.  Rows start wherever the element type may stand (odd vocabularies, sliced views): the few
// elements before the first 16-byte boundary and after the last are taken one by one (see Shape), the vectors between
// are aligned.  Reading vectors from the row's start instead, which the hardware allows, costs 12 % on 1500 x 50021
// fp16.  The gradient's rows mostly stand like the logits'; where they do not, its stores cross the boundaries.
typedef unsigned Word4 __attribute__((ext_vector_type(4)));
typedef unsigned Word4At2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned Word4At4 __attribute__((ext_vector_type(4), aligned(4)));

template <typename T>
struct Vec {
  static constexpr int E = 16 / sizeof(T);
  static __device__ __forceinline__ Word4 load(const T* p) { return *(const Word4*)p; }
  static __device__ __forceinline__ Word4 load_once(const T* p) { return __builtin_nontemporal_load((const Word4*)p); }
  static __device__ __forceinline__ void store(T* p, Word4 w) { __builtin_nontemporal_store(w, (Word4At2*)p); }
  static __device__ __forceinline__ void unpack(Word4 w, float v[E]) {
    T h[E];
    __builtin_memcpy(h, &w, 16);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = (float)h[e];
  }
  static __device__ __forceinline__ Word4 pack(const float v[E]) {
    T h[E];
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = (T)v[e];
    Word4 w;
    __builtin_memcpy(&w, h, 16);
    return w;
  }
};
template <>
struct Vec<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ Word4 load(const float* p) { return *(const Word4*)p; }
  static __device__ __forceinline__ Word4 load_once(const float* p) {
    return __builtin_nontemporal_load((const Word4*)p);
  }
  static __device__ __forceinline__ void store(float* p, Word4 w) { __builtin_nontemporal_store(w, (Word4At4*)p); }
  static __device__ __forceinline__ void unpack(Word4 w, float v[4]) { __builtin_memcpy(v, &w, 16); }
  static __device__ __forceinline__ Word4 pack(const float v[4]) {
    Word4 w;
    __builtin_memcpy(&w, v, 16);
    return w;
  }
};

// How a row is cut: `head` elements, n_vec vectors, `tail` elements.  Lane t takes the single element extra(t), if any.
template <typename T>
struct Shape {
  int head, n_vec, n_cols;
  __device__ __forceinline__ Shape(const T* row, int cols) {
    constexpr int E = Vec<T>::E;
    head = (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T);
    head = head < cols ? head : cols;
    n_vec = (cols - head) / E;
    n_cols = cols;
  }
  __device__ __forceinline__ int col(int i) const { return head + i * Vec<T>::E; }
  __device__ __forceinline__ unsigned extra(int t) const {  // >= n_cols: none (a row may have 2^31 - 1 columns)
    return t < head ? (unsigned)t : (unsigned)(n_vec * Vec<T>::E) + (unsigned)t;
  }
};

// Takes the N values of v into st: their maximum first, then one exponential each.
template <int N>
__device__ __forceinline__ void take(RowStat& st, const float* v) {
  float top = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, v[i]);
  const float m = fmaxf(st.m, top), ref = finite_or_zero(m);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) s += exp_nat(v[i] - ref);
  st.s = st.s * exp_nat(st.m - ref) + s;
  st.m = m;
}

// A policy row: r = exp(lp - old), term = w (kl_coef k3 - min(r A, clip(r) A)), k3 = exp(ref - lp) - (ref - lp) - 1
// (an unbiased, never negative estimate of the KL divergence from the sampled label alone), and
// d term / d lp = w (kl_coef (1 - exp(ref - lp)) - [r A <= clip(r) A] r A).
struct PolicyRow {
  double loss, kl, clipped;
  float coef;
};

struct PolicyIn {
  const float *old_lp, *adv, *ref, *weights;
  double lo, hi, kl_coef, scale;
};

__device__ __forceinline__ PolicyRow policy_row(const PolicyIn& in, int row, double lp) {
  PolicyRow o = {0.0, 0.0, 0.0, 0.f};
  const double w = in.scale * (in.weights ? (double)in.weights[row] : 1.0);
  if (w == 0.0) return o;
  const double a = (double)in.adv[row], r = exp(lp - (double)in.old_lp[row]);
  const double plain = r * a, cut = (r < in.lo ? in.lo : (r > in.hi ? in.hi : r)) * a;
  const bool clipped = cut < plain;
  double k3 = 0.0, dk3 = 0.0;
  if (in.ref) {
    const double gap = (double)in.ref[row] - lp, e = expm1(gap);
    k3 = gap < INFINITY ? e - gap : gap;  // an impossible label's estimate is infinite, not inf - inf
    dk3 = -e;
  }
  const bool penalty = in.kl_coef > 0.0;  // without one an infinite k3 is reported, not multiplied
  o.loss = w * ((penalty ? in.kl_coef * k3 : 0.0) - (clipped ? cut : plain));
  o.kl = w * k3;
  o.clipped = clipped ? w : 0.0;
  o.coef = (float)(w * ((penalty ? in.kl_coef * dk3 : 0.0) - (clipped ? 0.0 : plain)));
  return o;
}

template <typename T>
struct RowsIn {
  const T* x;
  long ld;
  int first, n_rows, n_cols;  // a launch takes the rows [first, n_rows)
  Labels labels;
  const int* owner;
  float2* stats;
  float* lp32;
  double* lp64;
};

// What a row's end leaves behind: statistics and the log-probability in the types asked for.
template <typename T>
__device__ __forceinline__ double finish_row(const RowsIn<T>& in, int row, long label, bool counted, RowStat st) {
  const double lp = counted ? label_log_prob(in.x + (long)row * in.ld, label, in.n_cols, st) : 0.0;
  if (in.stats) in.stats[row] = counted ? make_float2(st.m, st.s) : make_float2(0.f, 1.f);
  if (in.lp32) in.lp32[row] = (float)lp;
  if (in.lp64) in.lp64[row] = lp;
  return lp;
}

template <typename T>
__device__ __forceinline__ bool counts(const RowsIn<T>& in, int row, long label) {
  return label >= 0 && !(in.owner && in.owner[row] < 0);
}

// Statistics of one long row per block, streamed: four 16-byte loads in flight per lane; a row of any length.
template <typename T, int BLOCK>
__global__ __launch_bounds__(BLOCK) void stats_kernel(RowsIn<T> in) {
  constexpr int E = Vec<T>::E, U = 4;
  __shared__ RowStat part[BLOCK / 64];
  const int row = in.first + blockIdx.x;
  const long label = in.labels[row];
  if (!counts(in, row, label)) {
    if (threadIdx.x == 0) finish_row(in, row, label, false, RowStat{0.f, 1.f});
    return;
  }
  const T* r = in.x + (long)row * in.ld;
  const Shape<T> shape(r, in.n_cols);
  const int n_vec = shape.n_vec;
  RowStat st = {-INFINITY, 0.f};
  int i = threadIdx.x;
  for (; i + (U - 1) * BLOCK < n_vec; i += U * BLOCK) {
    Word4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = Vec<T>::load(r + shape.col(i + u * BLOCK));
    float v[U * E];
#pragma unroll
    for (int u = 0; u < U; ++u) Vec<T>::unpack(w[u], v + u * E);
    take<U * E>(st, v);
  }
  for (; i < n_vec; i += BLOCK) {
    float v[E];
    Vec<T>::unpack(Vec<T>::load(r + shape.col(i)), v);
    take<E>(st, v);
  }
  const unsigned c = shape.extra(threadIdx.x);
  if (c < (unsigned)in.n_cols) {
    const float v = (float)r[c];
    take<1>(st, &v);
  }
  st = wave_join(st);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = st;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < BLOCK / 64; ++w) st = join(st, part[w]);
    finish_row(in, row, label, true, st);
  }
}

template <typename T>
struct GradOut {
  T* dx;
  long ld, width;
};

// -ks exp(x - m), plus k at the label.
template <int E>
__device__ __forceinline__ void softmax_grad(float v[E], long col, long label, float m, float ks, float k) {
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = -ks * exp_nat(v[e] - m);
  const unsigned long at = (unsigned long)(label - col);
  if (at < (unsigned long)E) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] += e == (int)at ? k : 0.f;
  }
}

enum { kStats = 0, kPolicy = 1 };

// Whole rows in registers: RT lanes hold NV vectors of 16 bytes each, so a row is read once whatever is made of it.
// kStats: statistics and log-probabilities of short rows.  kPolicy: the row's loss terms and, the coefficient of a policy
// row depending on nothing else, its gradient in the same pass.  A block of RT * R threads owns R rows; the 64-bit
// arithmetic of a row's end is done by one lane per row, side by side.  Bound by memory: 8192 x 32000 bf16 185 us in 512
// threads x 8 vectors, 5.4 TB/s read and written (256 x 16 the same, 1024 x 4 199); 4096 x 128000 bf16, where a row
// takes the registers of a CU and loads and stores do not overlap, 428 us, 4.9 TB/s - the two passes take 538.  Eight waves
// a SIMD leave the forms of 256 and 512 lanes 12 to 20 bytes a lane short of registers; six, which spill nothing, take 181
// us at 8192 x 32000 bf16 but 43.0 instead of 39.5 at 8192 x 5000.
template <typename T, int RT, int R, int NV, int MODE>
__global__ __launch_bounds__(RT* R, NV > 8 ? 4 : RT == 64 && NV == 8 ? 6 : 8) void rows_kernel(
    RowsIn<T> in, PolicyIn policy, float* __restrict__ coef, double* __restrict__ terms, long n_terms, GradOut<T> out) {
  constexpr int E = Vec<T>::E, W = RT / 64;
  // long policy rows are read once and for all: past the caches (8192 x 32000 bf16 201 -> 191 us); short ones lose by it
  // (20480 x 780 fp32 36 -> 40 us)
  constexpr bool kOnce = MODE == kPolicy && RT > 64;
  __shared__ RowStat part[R * W];
  __shared__ float4 end[R];  // m, s, coefficient
  const int r = threadIdx.x / RT, t = threadIdx.x % RT;
  const long first = in.first + (long)blockIdx.x * R;
  const int row = (int)(first + r);
  const bool there = first + r < in.n_rows;
  const long label = there ? in.labels[row] : -1;
  const bool counted = there && counts(in, row, label);
  const T* x = in.x + (long)row * in.ld;
  const Shape<T> shape(x, in.n_cols);
  const int n_vec = shape.n_vec;
  const unsigned c_one = shape.extra(t);
  Word4 w[NV];
  float one = -INFINITY;
  RowStat st = {-INFINITY, 0.f};
  if (counted) {
#pragma unroll
    for (int u = 0; u < NV; ++u)
      if (t + u * RT < n_vec)
        w[u] = kOnce ? Vec<T>::load_once(x + shape.col(t + u * RT)) : Vec<T>::load(x + shape.col(t + u * RT));
    if (c_one < (unsigned)in.n_cols) one = (float)x[c_one];
    // the maximum of all that a lane holds first, so that every value takes one exponential
    st.m = one;
#pragma unroll
    for (int u = 0; u < NV; ++u)
      if (t + u * RT < n_vec) {
        float v[E];
        Vec<T>::unpack(w[u], v);
#pragma unroll
        for (int e = 0; e < E; ++e) st.m = fmaxf(st.m, v[e]);
      }
    const float ref = finite_or_zero(st.m);
    st.s = exp_nat(one - ref);
#pragma unroll
    for (int u = 0; u < NV; ++u)
      if (t + u * RT < n_vec) {
        float v[E];
        asm("" : "+v"(w[u]));  // unpacked again, not kept unpacked: that takes twice the registers
        Vec<T>::unpack(w[u], v);
#pragma unroll
        for (int e = 0; e < E; ++e) st.s += exp_nat(v[e] - ref);
      }
    st = wave_join(st);
    if ((t & 63) == 0) part[threadIdx.x >> 6] = st;
  }
  __syncthreads();
  if (threadIdx.x < R) {
    const int i = threadIdx.x, mine = (int)(first + i);
    if (first + i < in.n_rows) {
      const long l = in.labels[mine];
      const bool c = counts(in, mine, l);
      RowStat s = {0.f, 1.f};
      if (c) {
        s = part[i * W];
        for (int k = 1; k < W; ++k) s = join(s, part[i * W + k]);
      }
      const double lp = finish_row(in, mine, l, c, s);
      if constexpr (MODE == kPolicy) {
        PolicyRow p = {0.0, 0.0, 0.0, 0.f};
        if (c) p = policy_row(policy, mine, lp);
        coef[mine] = p.coef;
        terms[mine] = p.loss;
        terms[n_terms + mine] = p.kl;
        terms[2 * n_terms + mine] = p.clipped;
        end[i] = make_float4(s.m, s.s, p.coef, 0.f);
      }
    }
  }
  if constexpr (MODE == kPolicy) {
    if (!out.dx) return;
    __syncthreads();
    if (!there) return;
    T* d = out.dx + (long)row * out.ld;
    const float4 f = end[r];
    const float m = finite_or_zero(f.x), k = f.z, ks = k / f.y;
    const bool due = counted && k != 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int i = t + u * RT;
      if (i >= n_vec) break;
      float v[E];
      if (due) {
        Vec<T>::unpack(w[u], v);
        softmax_grad<E>(v, shape.col(i), label, m, ks, k);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = 0.f;
      }
      Vec<T>::store(d + shape.col(i), Vec<T>::pack(v));
    }
    if (c_one < (unsigned)in.n_cols) {
      float v = 0.f;
      if (due) {
        v = one;
        softmax_grad<1>(&v, c_one, label, m, ks, k);
      }
      d[c_one] = (T)v;
    }
    for (long c = (long)in.n_cols + t; c < out.width; c += RT) d[c] = (T)0.f;
  }
}

// A coefficient times the upstream factor; a factor of zero leaves out whatever the coefficient is (infinities and NaN of
// rows that do count).
__device__ __forceinline__ float times_upstream(float coef, float up) { return up == 0.f ? 0.f : coef * up; }

// dx[row, j] = c ([j = label] - exp(x_j - m) / s), c = coef[owner or row] * upstream, from saved statistics.  Rows are
// cut into tiles of RT lanes x NV vectors; a block of 256 threads owns 256 / RT tiles.  With unless_one the gradient
// for an upstream factor of one is in place already and nothing is done where the factor is one.
// Bound by memory: 4096 x 128000 bf16 341 us, 6.15 TB/s read and written.  Tiles of 8 KiB (two vectors a lane) keep the
// places the chip works on close together: 8192 x 32000 bf16 169 us, with 16 KiB 188, with 4 KiB 209.  The gradient is
// written past the caches, which leaves them to the logits: 60000 x 1500 fp32 125 us, through them 135; both passes of
// 8192 x 32000 bf16 256 us instead of 305.
template <typename T, int RT, int NV, bool ONCE>
__global__ __launch_bounds__(JTVAE_BLOCK) void grad_kernel(RowsIn<T> in, const float* __restrict__ coef,
                                                           const float* __restrict__ upstream, int unless_one,
                                                           int tiles, GradOut<T> out, float* __restrict__ scaled,
                                                           int n_scaled) {
  constexpr int E = Vec<T>::E;
  const float up = upstream ? *upstream : 1.f;
  for (long i = (long)blockIdx.x * JTVAE_BLOCK + threadIdx.x; i < n_scaled; i += (long)gridDim.x * JTVAE_BLOCK)
    scaled[i] = times_upstream(coef[i], up);
  if (unless_one && up == 1.f) return;
  // Last rows first: they are what the pass that formed the statistics has left in the caches.  Where nothing is due
  // mostly, the grid is smaller than the work and a block takes several pieces.
  const long step = (long)gridDim.x * (JTVAE_BLOCK / RT);
  long id = (long)(in.n_rows - in.first) * tiles - 1 - ((long)blockIdx.x * (JTVAE_BLOCK / RT) + threadIdx.x / RT);
  for (; id >= 0; id -= step) {
    const long r = id / tiles;
    const int row = in.first + (int)r, tile = (int)(id - r * tiles), t = threadIdx.x % RT;
    const long label = in.labels[row];
    const int own = in.owner ? in.owner[row] : row;
    const bool counted = label >= 0 && own >= 0;
    const T* x = in.x + (long)row * in.ld;
    T* d = out.dx + (long)row * out.ld;
    const Shape<T> shape(x, in.n_cols);
    const int n_vec = shape.n_vec, first = tile * RT * NV + t;
    float k = 0.f, ks = 0.f, m = 0.f;  // loads of the row are under way before its coefficient is known
    Word4 w[NV];
    if (counted) {
#pragma unroll
      for (int u = 0; u < NV; ++u)
        if (first + u * RT < n_vec)
          w[u] = ONCE ? Vec<T>::load_once(x + shape.col(first + u * RT)) : Vec<T>::load(x + shape.col(first + u * RT));
      const float2 st = in.stats[row];
      k = times_upstream(coef[own], up);
      if (label >= in.n_cols && k != 0.f) k = NAN;
      m = finite_or_zero(st.x);
      ks = k / st.y;
    }
    const bool due = counted && k != 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int i = first + u * RT;
      if (i >= n_vec) break;
      float v[E];
      if (due) {
        Vec<T>::unpack(w[u], v);
        softmax_grad<E>(v, shape.col(i), label, m, ks, k);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = 0.f;
      }
      Vec<T>::store(d + shape.col(i), Vec<T>::pack(v));
    }
    if (tile == 0) {  // single elements at the row's ends, and the padding
      const unsigned c = shape.extra(t);
      if (c < (unsigned)in.n_cols) {
        float v = 0.f;
        if (due) {
          v = (float)x[c];
          softmax_grad<1>(&v, c, label, m, ks, k);
        }
        d[c] = (T)v;
      }
      for (long p = (long)in.n_cols + t; p < out.width; p += RT) d[p] = (T)0.f;
    }
  }
}

struct Sequences {
  const int *rowptr, *rows;
  int n_seq;
  const int2* pairs;
  int n_pairs;
  const int *pair_ptr, *pair_list;
};

// Sum over the rows of a sequence by one wave, in fp64 and a fixed order; the same value in every lane.
__device__ __forceinline__ double sequence_sum(const Sequences& q, const double* lp64, const float* other, int seq,
                                               int lane) {
  double acc = 0.0;
  for (long i = (long)q.rowptr[seq] + lane; i < q.rowptr[seq + 1]; i += 64) acc += lp64[q.rows[i]];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
  return other ? acc + (double)other[seq] : acc;
}

__global__ __launch_bounds__(JTVAE_BLOCK) void sequence_sums_kernel(Sequences q, const double* __restrict__ lp64,
                                                                    const float* __restrict__ other,
                                                                    double* __restrict__ sums64,
                                                                    float* __restrict__ sums) {
  const int lane = threadIdx.x & 63;
  const long step = (long)gridDim.x * (JTVAE_BLOCK / 64);
  for (long seq = ((long)blockIdx.x * JTVAE_BLOCK + threadIdx.x) >> 6; seq < q.n_seq; seq += step) {
    const double acc = sequence_sum(q, lp64, other, (int)seq, lane);
    if (lane == 0) {
      if (sums64) sums64[seq] = acc;
      sums[seq] = (float)acc;
    }
  }
}

constexpr int kPairBlock = 1024;

struct Preference {
  const float *ref, *other;
  double beta, smoothing, scale;
};

// Pairs (a, b): D = beta ((S_a - ref_a) - (S_b - ref_b)), loss = scale sum -(1-e) log sig(D) - e log sig(-D), with
// -log sig(D) = max(-D, 0) + log1p(exp(-|D|)) and d loss / dD = scale (e sig(D) - (1-e) sig(-D)), both logistic values from
// exp(-|D|): sig(D) - 1 instead of the second would lose its digits from margins of 20 on.  Then the coefficient of every
// sequence, summed over the pairs that name it in the order of pair_list (pair * 2 + side).  One block, since the loss is
// one number; with SUMS it also forms the sequences' sums, 16 at a time.
template <bool SUMS>
__global__ __launch_bounds__(kPairBlock) void preference_kernel(Sequences q, Preference in,
                                                                const double* __restrict__ lp64, double* sums64,
                                                                float* __restrict__ sums, float* __restrict__ loss,
                                                                float* __restrict__ margins, double* dmargin,
                                                                float* __restrict__ coef) {
  __shared__ double part[kPairBlock / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if constexpr (SUMS) {
    for (int seq = wave; seq < q.n_seq; seq += kPairBlock / 64) {
      const double acc = sequence_sum(q, lp64, in.other, seq, lane);
      if (lane == 0) {
        sums64[seq] = acc;
        sums[seq] = (float)acc;
      }
    }
    __syncthreads();
  }
  double acc = 0.0;
  for (long p = threadIdx.x; p < q.n_pairs; p += kPairBlock) {
    const int2 ab = q.pairs[p];
    const double d =
        in.beta * ((sums64[ab.x] - (double)in.ref[ab.x]) - (sums64[ab.y] - (double)in.ref[ab.y]));
    const double t = exp(-fabs(d)), l = log1p(t), far = t / (1.0 + t), near = 1.0 / (1.0 + t);
    if (in.smoothing < 1.0) acc += (1.0 - in.smoothing) * (fmax(-d, 0.0) + l);  // no 0 * inf at an infinite margin
    if (in.smoothing > 0.0) acc += in.smoothing * (fmax(d, 0.0) + l);
    if (d != d) acc = d;  // fmax drops a NaN
    margins[p] = (float)d;
    dmargin[p] = in.scale * in.beta * (in.smoothing * (d < 0.0 ? far : near) - (1.0 - in.smoothing) * (d < 0.0 ? near : far));
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
  if (lane == 0) part[wave] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < kPairBlock / 64; ++w) t += part[w];
    *loss = (float)(in.scale * t);
  }
  for (long s = threadIdx.x; s < q.n_seq; s += kPairBlock) {
    double c = 0.0;
    for (int i = q.pair_ptr[s]; i < q.pair_ptr[s + 1]; ++i) {
      const int e = q.pair_list[i];
      c += (e & 1) ? -dmargin[e >> 1] : dmargin[e >> 1];
    }
    coef[s] = (float)c;
  }
}

// Loss terms and coefficients of rows whose log-probabilities are there already.
__global__ __launch_bounds__(JTVAE_BLOCK) void policy_rows_kernel(PolicyIn in, const double* __restrict__ lp64,
                                                                  Labels labels, int n_rows,
                                                                  float* __restrict__ coef,
                                                                  double* __restrict__ terms) {
  const long at = (long)blockIdx.x * JTVAE_BLOCK + threadIdx.x;
  if (at >= n_rows) return;
  const int row = (int)at;
  PolicyRow o = {0.0, 0.0, 0.0, 0.f};
  if (labels[row] >= 0) o = policy_row(in, row, lp64[row]);
  coef[row] = o.coef;
  terms[row] = o.loss;
  terms[(long)n_rows + row] = o.kl;
  terms[2L * n_rows + row] = o.clipped;
}

// Sums of the rows' three terms, [3, n_rows]: one block, fixed order.
__global__ __launch_bounds__(kPairBlock) void sum_terms_kernel(const double* __restrict__ terms, int n_rows,
                                                               float* __restrict__ loss, float* __restrict__ kl,
                                                               float* __restrict__ clipped) {
  __shared__ double part[3][kPairBlock / 64];
  double a = 0.0, b = 0.0, c = 0.0;
  const double *kls = terms + n_rows, *cut = kls + n_rows;
#pragma unroll 8
  for (long i = threadIdx.x; i < n_rows; i += kPairBlock) {
    a += terms[i];
    b += kls[i];
    c += cut[i];
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    a += __shfl_xor(a, off, 64);
    b += __shfl_xor(b, off, 64);
    c += __shfl_xor(c, off, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    part[0][threadIdx.x >> 6] = a;
    part[1][threadIdx.x >> 6] = b;
    part[2][threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x < 3) {
    double t = 0.0;
    for (int w = 0; w < kPairBlock / 64; ++w) t += part[threadIdx.x][w];
    *(threadIdx.x == 0 ? loss : threadIdx.x == 1 ? kl : clipped) = (float)t;
  }
}

int check_logits(const jtvae_logits_t* g) {
  if (!g) return JTVAE_E_NULL;
  if (g->n_rows < 0 || g->n_cols <= 0 || g->ld < g->n_cols) return JTVAE_E_SHAPE;
  if (g->dtype < JTVAE_F32 || g->dtype > JTVAE_BF16) return JTVAE_E_RANGE;
  if (g->label_bits != 32 && g->label_bits != 64) return JTVAE_E_RANGE;
  if (g->n_rows > 0 && (!g->x || !g->labels)) return JTVAE_E_NULL;
  const uintptr_t size = g->dtype == JTVAE_F32 ? 4 : 2;
  if ((uintptr_t)g->x % size || (uintptr_t)g->labels % (g->label_bits / 8)) return JTVAE_E_ALIGN;
  return 0;
}

// A wave per sequence; beyond a million of them a wave takes several.
unsigned sum_blocks(int n_seq) {
  const unsigned b = grid_for((long)n_seq * 64);
  return b < (1u << 18) ? b : 1u << 18;
}

int check_sequences(const jtvae_sequences_t* q, int n_rows, bool pairs) {
  if (!q) return JTVAE_E_NULL;
  if (q->n_seq < 0 || (pairs && q->n_pairs < 0)) return JTVAE_E_SHAPE;
  if ((n_rows && !q->row_seq) || (q->n_seq && (!q->rowptr || !q->rows))) return JTVAE_E_NULL;
  if (pairs && ((q->n_pairs && !q->pairs) || (q->n_seq && (!q->pair_ptr || !q->pair_list)))) return JTVAE_E_NULL;
  return 0;
}

Sequences sequences_of(const jtvae_sequences_t* q) {
  return Sequences{q->rowptr, q->rows, q->n_seq, (const int2*)q->pairs, q->n_pairs, q->pair_ptr, q->pair_list};
}

template <typename T>
RowsIn<T> rows_in(const jtvae_logits_t* g, const int32_t* owner, float* stats, float* lp32, double* lp64) {
  return RowsIn<T>{(const T*)g->x, (long)g->ld, 0, g->n_rows, g->n_cols, Labels{g->labels, g->label_bits}, owner,
                   (float2*)stats, lp32, lp64};
}

inline unsigned blocks_for(long items, int per) { return (unsigned)((items + per - 1) / per); }

// Calls launch(part of the rows, how many) so that no grid has more than 2^31 work-items (the limit is 2^32).
template <typename T, typename F>
int for_row_parts(RowsIn<T> in, long lanes_per_row, F launch) {
  const int n = in.n_rows;
  const long most = lanes_per_row < (1L << 31) ? (1L << 31) / lanes_per_row : 1;
  for (long r0 = 0; r0 < n; r0 += most) {
    in.first = (int)r0;
    in.n_rows = (int)(n - r0 < most ? n : r0 + most);
    launch(in, in.n_rows - in.first);
    int rc = launch_status();
    if (rc) return rc;
  }
  return 0;
}

template <typename T, int RT, int R, int NV, int MODE>
int launch_rows(const RowsIn<T>& rows, const PolicyIn& p, float* coef, double* terms, const GradOut<T>& out,
                hipStream_t s) {
  return for_row_parts(rows, RT, [&](const RowsIn<T>& in, int n) {
    hipLaunchKernelGGL((rows_kernel<T, RT, R, NV, MODE>), dim3(blocks_for(n, R)), dim3(RT * R), 0, s, in, p, coef, terms,
                       (long)rows.n_rows, out);
  });
}

template <typename T, int BLOCK>
int launch_stats(const RowsIn<T>& rows, hipStream_t s) {
  return for_row_parts(rows, BLOCK, [&](const RowsIn<T>& in, int n) {
    hipLaunchKernelGGL((stats_kernel<T, BLOCK>), dim3(n), dim3(BLOCK), 0, s, in);
  });
}

// Statistics.  Rows of up to 512 vectors (8 KiB) sit in a wave's registers, eight waves side by side; longer ones are
// streamed by a block each.  20480 fp32 rows of 129 vectors 11.5 us, streamed 24.0; of 511 30.8 and 36.9; 513, streamed, 39.9.
// Two vectors a lane do for 128 (rows of 127: 10.8 us, with eight 11.2; policy pass 26.3 and 27.5).  Up to a row per CU the
// block has 512 threads, since a CU alone is bound by its arithmetic (64 x 128000 bf16 10.7 us against 14.3, 256 rows 12.9
// against 15.6); beyond, 256, so that a CU has blocks at every stage (1024 x 30000 12.9 against 13.9, with 1024 threads
// 16.3).  Bound by memory from there on: 4096 x 128000 bf16 178 us, 5.9 TB/s read; a launch of 50 us loses 5 of them to its
// start and drain (4096 x 32000 5.3 TB/s, 16384 x 32000 6.0).
template <typename T>
int row_stats(const jtvae_logits_t* g, const int32_t* owner, float* stats, float* lp32, double* lp64, hipStream_t s) {
  const RowsIn<T> in = rows_in<T>(g, owner, stats, lp32, lp64);
  const int n_vec = g->n_cols / Vec<T>::E;
  const PolicyIn none = {};
  const GradOut<T> no_grad = {};
  if (n_vec <= 128) return launch_rows<T, 64, 8, 2, kStats>(in, none, nullptr, nullptr, no_grad, s);
  if (n_vec <= 512) return launch_rows<T, 64, 8, 8, kStats>(in, none, nullptr, nullptr, no_grad, s);
  return g->n_rows > 256 ? launch_stats<T, 256>(in, s) : launch_stats<T, 512>(in, s);
}

// The grid where the gradient mostly stands already: enough to fill the chip once.
constexpr unsigned kIdleBlocks = 2048;

template <typename T, int RT, int NV, bool ONCE>
int launch_grad(const RowsIn<T>& rows, const float* coef, const float* upstream, int unless_one, const GradOut<T>& out,
                float* scaled, int n_scaled, hipStream_t s) {
  const int n_vec = rows.n_cols / Vec<T>::E;
  const int tiles = n_vec > RT * NV ? (n_vec + RT * NV - 1) / (RT * NV) : 1;
  const auto launch = [&](const RowsIn<T>& in, int n) {
    unsigned blocks = n ? blocks_for((long)n * tiles, JTVAE_BLOCK / RT) : 1;
    if (unless_one && blocks > kIdleBlocks) blocks = kIdleBlocks;
    hipLaunchKernelGGL((grad_kernel<T, RT, NV, ONCE>), dim3(blocks), dim3(JTVAE_BLOCK), 0, s, in, coef, upstream,
                       unless_one, tiles, out, scaled, n_scaled);
    n_scaled = 0;  // once is enough
  };
  if (rows.n_rows) return for_row_parts(rows, (long)RT * tiles, launch);
  launch(rows, 0);
  return launch_status();
}

template <typename T>
int row_grad(const jtvae_logits_t* g, const int32_t* owner, const float* stats, const float* coef,
             const float* upstream, int unless_one, void* dx, int64_t ld_dx, int64_t width, float* scaled,
             int n_scaled, hipStream_t s) {
  const RowsIn<T> in = rows_in<T>(g, owner, (float*)stats, nullptr, nullptr);
  const GradOut<T> out = {(T*)dx, (long)ld_dx, (long)width};
  const int n_vec = g->n_cols / Vec<T>::E;
  // Up to 256 vectors a wave takes the row (20480 rows of 129: 14.9 us, in tiles of a block 21.1; of 255: 26.6 and 27.6).
  // Half as many vectors a lane for rows of up to 128 are no faster (96: 11.1 us both ways).
  if (n_vec <= 256) return launch_grad<T, 64, 4, false>(in, coef, upstream, unless_one, out, scaled, n_scaled, s);
  // Logits beyond what the 256 MiB cache keeps are read past it (forward and backward of 4096 x 128000 bf16: 482 us, 493
  // through it); smaller ones are found there (4000 x 3500 bf16 11.0 us, 12.7 past it).
  if ((double)g->n_rows * g->n_cols * sizeof(T) > 256e6)
    return launch_grad<T, 256, 2, true>(in, coef, upstream, unless_one, out, scaled, n_scaled, s);
  return launch_grad<T, 256, 2, false>(in, coef, upstream, unless_one, out, scaled, n_scaled, s);
}

constexpr int kTooLong = -100;  // no error code of this library or of HIP

// A policy row in one pass where its registers hold it; kTooLong when they do not.
template <typename T>
int policy_rows(const RowsIn<T>& in, const PolicyIn& p, float* coef, double* terms, const GradOut<T>& out,
                hipStream_t s) {
  const int n_vec = in.n_cols / Vec<T>::E;
  if (n_vec <= 128) return launch_rows<T, 64, 8, 2, kPolicy>(in, p, coef, terms, out, s);
  if (n_vec <= 512) return launch_rows<T, 64, 8, 8, kPolicy>(in, p, coef, terms, out, s);
  if (n_vec <= 2048) return launch_rows<T, 256, 1, 8, kPolicy>(in, p, coef, terms, out, s);
  if (n_vec <= 4096) return launch_rows<T, 512, 1, 8, kPolicy>(in, p, coef, terms, out, s);
  if (n_vec <= 8192) return launch_rows<T, 1024, 1, 8, kPolicy>(in, p, coef, terms, out, s);
  if (n_vec <= 16384) return launch_rows<T, 1024, 1, 16, kPolicy>(in, p, coef, terms, out, s);
  return kTooLong;
}

template <typename T>
int policy(const jtvae_logits_t* g, const PolicyIn& in, float* stats, float* lp, float* coef, double* lp64,
           double* terms, void* dx, int64_t ld_dx, int64_t width, hipStream_t s) {
  const GradOut<T> out = {(T*)dx, (long)ld_dx, (long)width};
  const int rc = policy_rows<T>(rows_in<T>(g, nullptr, stats, lp, nullptr), in, coef, terms, out, s);
  if (rc != kTooLong) return rc;
  int e = row_stats<T>(g, nullptr, stats, lp, lp64, s);
  if (e) return e;
  hipLaunchKernelGGL(policy_rows_kernel, dim3(grid_for(g->n_rows)), dim3(JTVAE_BLOCK), 0, s, in, lp64,
                     Labels{g->labels, g->label_bits}, g->n_rows, coef, terms);
  e = launch_status();
  return e || !dx ? e : row_grad<T>(g, nullptr, stats, coef, nullptr, 0, dx, ld_dx, width, nullptr, 0, s);
}

}  // namespace

#define JT_CHECK(expr)        \
  do {                        \
    int _rc = (expr);         \
    if (_rc) return _rc;      \
  } while (0)

extern "C" {

int jtvae_label_log_probs(const jtvae_logits_t* logits, const int32_t* owner, float* stats, float* log_probs,
                          double* log_probs64, void* stream) {
  JT_CHECK(check_logits(logits));
  if (logits->n_rows == 0) return 0;
  if (!stats) return JTVAE_E_NULL;
  hipStream_t s = (hipStream_t)stream;
  switch (logits->dtype) {
    case JTVAE_F32: return row_stats<float>(logits, owner, stats, log_probs, log_probs64, s);
    case JTVAE_F16: return row_stats<_Float16>(logits, owner, stats, log_probs, log_probs64, s);
    default: return row_stats<__bf16>(logits, owner, stats, log_probs, log_probs64, s);
  }
}

int jtvae_label_log_probs_bwd(const jtvae_logits_t* logits, const int32_t* owner, const float* stats,
                              const float* coef, const float* upstream, int32_t unless_one, void* dx, int64_t ld_dx,
                              int64_t width, float* scaled, int32_t n_scaled, void* stream) {
  JT_CHECK(check_logits(logits));
  if (width < logits->n_cols || ld_dx < width) return JTVAE_E_SHAPE;
  if (n_scaled < 0) return JTVAE_E_SHAPE;
  if (logits->n_rows == 0 && n_scaled == 0) return 0;
  if (!coef || (unless_one && !upstream) || (n_scaled && !scaled)) return JTVAE_E_NULL;
  if (logits->n_rows && (!stats || !dx)) return JTVAE_E_NULL;
  if ((uintptr_t)dx % (logits->dtype == JTVAE_F32 ? 4 : 2)) return JTVAE_E_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  switch (logits->dtype) {
    case JTVAE_F32:
      return row_grad<float>(logits, owner, stats, coef, upstream, unless_one, dx, ld_dx, width, scaled, n_scaled, s);
    case JTVAE_F16:
      return row_grad<_Float16>(logits, owner, stats, coef, upstream, unless_one, dx, ld_dx, width, scaled, n_scaled, s);
    default:
      return row_grad<__bf16>(logits, owner, stats, coef, upstream, unless_one, dx, ld_dx, width, scaled, n_scaled, s);
  }
}

size_t jtvae_sequence_log_probs_workspace_bytes(int32_t n_rows) {
  return n_rows > 0 ? (size_t)n_rows * sizeof(double) : 0;
}

int jtvae_sequence_log_probs(const jtvae_logits_t* logits, const jtvae_sequences_t* sequences, float* stats,
                             float* sums, void* workspace, size_t workspace_bytes, void* stream) {
  JT_CHECK(check_logits(logits));
  JT_CHECK(check_sequences(sequences, logits->n_rows, false));
  if (sequences->n_seq == 0) return 0;
  if (!sums || (logits->n_rows && (!stats || !workspace))) return JTVAE_E_NULL;
  if (workspace_bytes < jtvae_sequence_log_probs_workspace_bytes(logits->n_rows)) return JTVAE_E_WORKSPACE;
  double* lp64 = (double*)workspace;
  JT_CHECK(jtvae_label_log_probs(logits, sequences->row_seq, stats, nullptr, lp64, stream));
  hipLaunchKernelGGL(sequence_sums_kernel, dim3(sum_blocks(sequences->n_seq)), dim3(JTVAE_BLOCK), 0,
                     (hipStream_t)stream, sequences_of(sequences), lp64, nullptr, nullptr, sums);
  return launch_status();
}

size_t jtvae_preference_loss_workspace_bytes(int32_t n_rows, int32_t n_seq, int32_t n_pairs) {
  return n_rows < 0 || n_seq < 0 || n_pairs < 0 ? 0 : ((size_t)n_rows + n_seq + n_pairs) * sizeof(double);
}

int jtvae_preference_loss(const jtvae_logits_t* logits, const jtvae_sequences_t* sequences,
                          const jtvae_preference_t* preference, float* stats, float* sums, float* margins,
                          float* coef, float* loss, void* workspace, size_t workspace_bytes, void* stream) {
  JT_CHECK(check_logits(logits));
  JT_CHECK(check_sequences(sequences, logits->n_rows, true));
  if (!preference || !loss) return JTVAE_E_NULL;
  const int n = logits->n_rows, n_seq = sequences->n_seq, n_pairs = sequences->n_pairs;
  if ((n && !stats) || (n_seq && (!sums || !coef || !preference->ref_log_probs)) || (n_pairs && !margins))
    return JTVAE_E_NULL;
  const size_t need = jtvae_preference_loss_workspace_bytes(n, n_seq, n_pairs);
  if (need && !workspace) return JTVAE_E_NULL;
  if (workspace_bytes < need) return JTVAE_E_WORKSPACE;
  if (!(preference->label_smoothing >= 0.0 && preference->label_smoothing <= 1.0)) return JTVAE_E_RANGE;
  hipStream_t s = (hipStream_t)stream;
  double *lp64 = (double*)workspace, *sums64 = lp64 + n, *dmargin = sums64 + n_seq;
  const Sequences q = sequences_of(sequences);
  const Preference in = {preference->ref_log_probs, preference->other_log_probs, preference->beta,
                         preference->label_smoothing, preference->scale};
  JT_CHECK(jtvae_label_log_probs(logits, sequences->row_seq, stats, nullptr, lp64, stream));
  // For a few short sequences the one block of the pairs forms their sums as well, and a launch is saved (16 of 20 rows:
  // 7.3 us instead of 9.8, in a graph 7.0 and 7.9); else a wave each (64 of 130 rows: 11.6 us instead of 16.2).  At the
  // limits the two are alike: 64 sequences of 20 rows 9.9 and 10.2, of 64 rows 10.8 and 10.2; 16 of 250 9.7 and 10.4, of 1000
  // 18.7 and 18.0; 128 of 20 13.6 and 10.1.
  if (n_seq <= 64 && n <= 4096) {
    hipLaunchKernelGGL(preference_kernel<true>, dim3(1), dim3(kPairBlock), 0, s, q, in, lp64, sums64, sums, loss,
                       margins, dmargin, coef);
    return launch_status();
  }
  if (n_seq) {  // else every row is without a sequence, and a grid would be empty
    hipLaunchKernelGGL(sequence_sums_kernel, dim3(sum_blocks(n_seq)), dim3(JTVAE_BLOCK), 0, s, q, lp64,
                       in.other, sums64, sums);
    JT_CHECK(launch_status());
  }
  hipLaunchKernelGGL(preference_kernel<false>, dim3(1), dim3(kPairBlock), 0, s, q, in, lp64, sums64, sums, loss,
                     margins, dmargin, coef);
  return launch_status();
}

size_t jtvae_policy_loss_workspace_bytes(int32_t n_rows) {
  return n_rows > 0 ? (size_t)n_rows * 4 * sizeof(double) : 0;
}

int jtvae_policy_loss(const jtvae_logits_t* logits, const jtvae_policy_t* policy, float* stats, float* log_probs,
                      float* coef, float* loss, float* kl, float* clipped, void* dx, int64_t ld_dx, int64_t width,
                      void* workspace, size_t workspace_bytes, void* stream) {
  JT_CHECK(check_logits(logits));
  if (!policy || !loss || !kl || !clipped) return JTVAE_E_NULL;
  const int n = logits->n_rows;
  if (n > 0 && (!stats || !log_probs || !coef || !workspace || !policy->old_log_probs || !policy->advantages))
    return JTVAE_E_NULL;
  if (dx && (width < logits->n_cols || ld_dx < width)) return JTVAE_E_SHAPE;
  if ((uintptr_t)dx % (logits->dtype == JTVAE_F32 ? 4 : 2)) return JTVAE_E_ALIGN;
  if (workspace_bytes < jtvae_policy_loss_workspace_bytes(n)) return JTVAE_E_WORKSPACE;
  if (!(policy->clip_low >= 0.0 && policy->clip_low <= 1.0 && policy->clip_high >= 0.0)) return JTVAE_E_RANGE;
  hipStream_t s = (hipStream_t)stream;
  double* lp64 = (double*)workspace;
  double* terms = lp64 + n;
  if (n > 0) {
    const PolicyIn in = {policy->old_log_probs, policy->advantages, policy->ref_log_probs, policy->weights,
                         1.0 - policy->clip_low, 1.0 + policy->clip_high, policy->kl_coef, policy->scale};
    int rc;
    switch (logits->dtype) {
      case JTVAE_F32:
        rc = ::policy<float>(logits, in, stats, log_probs, coef, lp64, terms, dx, ld_dx, width, s);
        break;
      case JTVAE_F16:
        rc = ::policy<_Float16>(logits, in, stats, log_probs, coef, lp64, terms, dx, ld_dx, width, s);
        break;
      default: rc = ::policy<__bf16>(logits, in, stats, log_probs, coef, lp64, terms, dx, ld_dx, width, s);
    }
    if (rc) return rc;
  }
  hipLaunchKernelGGL(sum_terms_kernel, dim3(1), dim3(kPairBlock), 0, s, terms, n, loss, kl, clipped);
  return launch_status();
}

}  // extern "C"
