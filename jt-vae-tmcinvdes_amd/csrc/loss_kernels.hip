// Log-probabilities of chosen labels under rows of logits, their gradient, and the two losses built on them: paired
// log ratios (preferences) and the clipped policy ratio with a KL term.
//
// For a row x of V logits with label l:  m = max_j x_j,  s = sum_j exp(x_j - m),  log p_l = (x_l - m) - log s, and
// d(log p_l)/dx_j = [j = l] - exp(x_j - m) / s.  Statistics are fp32; the one value per row that is compared with
// other models' values (log p_l) is formed in fp64, because sequences sum thousands of them and take differences.
// A row without a label (label < 0, or owner < 0 where owners are given) is not read: log-probability 0, gradient 0.
// A label >= V gives NaN (the call cannot look at device memory without a wait).
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

// One block per row.
template <typename T>
__global__ __launch_bounds__(JTVAE_BLOCK) void row_stats_kernel(const T* __restrict__ x, long ld, int n_cols,
                                                                Labels labels, const int* __restrict__ owner,
                                                                float2* __restrict__ stats, float* __restrict__ lp32,
                                                                double* __restrict__ lp64) {
  const int row = blockIdx.x;
  const long label = labels[row];
  __shared__ RowStat part[JTVAE_BLOCK / 64];
  if (label < 0 || (owner && owner[row] < 0)) {
    if (threadIdx.x == 0) {
      stats[row] = make_float2(0.f, 1.f);
      if (lp32) lp32[row] = 0.f;
      if (lp64) lp64[row] = 0.0;
    }
    return;
  }
  const T* r = x + (long)row * ld;
  RowStat st = {-INFINITY, 0.f};
  for (int c = threadIdx.x; c < n_cols; c += JTVAE_BLOCK) {
    const float v = (float)r[c], m = fmaxf(st.m, v), ref = finite_or_zero(m);
    st.s = st.s * exp_nat(st.m - ref) + exp_nat(v - ref);
    st.m = m;
  }
  st = wave_join(st);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = st;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < JTVAE_BLOCK / 64; ++w) st = join(st, part[w]);
    stats[row] = make_float2(st.m, st.s);
    const double lp = label_log_prob(r, label, n_cols, st);
    if (lp32) lp32[row] = (float)lp;
    if (lp64) lp64[row] = lp;
  }
}

// dx[row, j] = c ([j = label] - exp(x_j - m) / s), c = coef[owner or row] * upstream.
template <typename T>
__global__ __launch_bounds__(JTVAE_BLOCK) void row_grad_kernel(const T* __restrict__ x, long ld, int n_cols,
                                                               Labels labels, const int* __restrict__ owner,
                                                               const float2* __restrict__ stats,
                                                               const float* __restrict__ coef,
                                                               const float* __restrict__ upstream,
                                                               T* __restrict__ dx, long ld_dx, long width) {
  const int row = blockIdx.x;
  const long label = labels[row];
  const int own = owner ? owner[row] : row;
  T* d = dx + (long)row * ld_dx;
  for (long c = n_cols + threadIdx.x; c < width; c += JTVAE_BLOCK) d[c] = (T)0.f;
  if (label < 0 || own < 0) {
    for (int c = threadIdx.x; c < n_cols; c += JTVAE_BLOCK) d[c] = (T)0.f;
    return;
  }
  const T* r = x + (long)row * ld;
  float k = coef[own];
  if (upstream) k *= *upstream;
  if (label >= n_cols) k = NAN;
  const float2 st = stats[row];
  const float m = finite_or_zero(st.x), ks = k / st.y;
  for (int c = threadIdx.x; c < n_cols; c += JTVAE_BLOCK) {
    const float g = -ks * exp_nat((float)r[c] - m);
    d[c] = (T)(c == label ? k + g : g);
  }
}

// Sums over the rows of every sequence (CSR), one wave per sequence, in fp64 and a fixed order.
__global__ __launch_bounds__(JTVAE_BLOCK) void sequence_sums_kernel(const double* __restrict__ lp64,
                                                                    const int* __restrict__ rowptr,
                                                                    const int* __restrict__ rows, int n_seq,
                                                                    const float* __restrict__ other,
                                                                    double* __restrict__ sums64,
                                                                    float* __restrict__ sums) {
  const int seq = (int)(((long)blockIdx.x * JTVAE_BLOCK + threadIdx.x) >> 6), lane = threadIdx.x & 63;
  if (seq >= n_seq) return;
  double acc = 0.0;
  for (int i = rowptr[seq] + lane; i < rowptr[seq + 1]; i += 64) acc += lp64[rows[i]];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
  if (lane == 0) {
    if (other) acc += (double)other[seq];
    if (sums64) sums64[seq] = acc;
    sums[seq] = (float)acc;
  }
}

constexpr int kPairBlock = 1024;

__device__ __forceinline__ double block_sum(double v, double* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n_waves = blockDim.x >> 6;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if (lane == 0) part[wave] = v;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < n_waves; ++w) t += part[w];
  return t;
}

// Pairs (a, b): D = beta ((S_a - ref_a) - (S_b - ref_b)), loss = scale sum -(1-e) log sig(D) - e log sig(-D), with
// -log sig(D) = max(-D, 0) + log1p(exp(-|D|)).  Then the coefficient of every sequence, summed over the pairs that
// name it in the order of seq_pairs (pair * 2 + side).  One block: a few thousand pairs at most in practice.
__global__ __launch_bounds__(kPairBlock) void preference_pairs_kernel(
    const double* __restrict__ sums64, const float* __restrict__ ref, const int2* __restrict__ pairs, int n_pairs,
    const int* __restrict__ seq_ptr, const int* __restrict__ seq_pairs, int n_seq, double beta, double smoothing,
    double scale, float* __restrict__ loss, float* __restrict__ margins, double* __restrict__ dmargin,
    float* __restrict__ coef) {
  __shared__ double part[kPairBlock / 64];
  double acc = 0.0;
  for (int p = threadIdx.x; p < n_pairs; p += kPairBlock) {
    const int2 ab = pairs[p];
    const double d = beta * ((sums64[ab.x] - (double)ref[ab.x]) - (sums64[ab.y] - (double)ref[ab.y]));
    const double l = log1p(exp(-fabs(d)));
    if (smoothing < 1.0) acc += (1.0 - smoothing) * (fmax(-d, 0.0) + l);  // no 0 * inf at an infinite margin
    if (smoothing > 0.0) acc += smoothing * (fmax(d, 0.0) + l);
    if (d != d) acc = d;  // fmax drops a NaN
    margins[p] = (float)d;
    dmargin[p] = scale * beta * (1.0 / (1.0 + exp(-d)) - (1.0 - smoothing));
  }
  acc = block_sum(acc, part);
  if (threadIdx.x == 0) *loss = (float)(scale * acc);
  __syncthreads();
  for (int q = threadIdx.x; q < n_seq; q += kPairBlock) {
    double c = 0.0;
    for (int i = seq_ptr[q]; i < seq_ptr[q + 1]; ++i) {
      const int e = seq_pairs[i];
      c += (e & 1) ? -dmargin[e >> 1] : dmargin[e >> 1];
    }
    coef[q] = (float)c;
  }
}

// Policy rows: r = exp(lp - old), term = w (kl_coef k3 - min(r A, clip(r) A)), k3 = exp(ref - lp) - (ref - lp) - 1
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
  PolicyRow o;
  const double w = in.scale * (in.weights ? (double)in.weights[row] : 1.0);
  const double a = (double)in.adv[row], r = exp(lp - (double)in.old_lp[row]);
  const double plain = r * a, cut = (r < in.lo ? in.lo : (r > in.hi ? in.hi : r)) * a;
  const bool clipped = cut < plain;
  double k3 = 0.0, dk3 = 0.0;
  if (in.ref) {
    const double gap = (double)in.ref[row] - lp, e = expm1(gap);
    k3 = e - gap;
    dk3 = -e;
  }
  o.loss = w * (in.kl_coef * k3 - (clipped ? cut : plain));
  o.kl = w * k3;
  o.clipped = clipped ? w : 0.0;
  o.coef = (float)(w * (in.kl_coef * dk3 - (clipped ? 0.0 : plain)));
  return o;
}

__global__ __launch_bounds__(JTVAE_BLOCK) void policy_rows_kernel(PolicyIn in, const double* __restrict__ lp64,
                                                                  Labels labels, int n_rows,
                                                                  float* __restrict__ coef,
                                                                  double* __restrict__ terms) {
  const int row = blockIdx.x * JTVAE_BLOCK + threadIdx.x;
  if (row >= n_rows) return;
  PolicyRow o = {0.0, 0.0, 0.0, 0.f};
  if (labels[row] >= 0) o = policy_row(in, row, lp64[row]);
  coef[row] = o.coef;
  terms[3L * row] = o.loss;
  terms[3L * row + 1] = o.kl;
  terms[3L * row + 2] = o.clipped;
}

// Sums of the rows' three terms: one block, fixed order.
__global__ __launch_bounds__(kPairBlock) void sum_terms_kernel(const double* __restrict__ terms, int n_rows,
                                                               float* __restrict__ loss, float* __restrict__ kl,
                                                               float* __restrict__ clipped) {
  __shared__ double part[kPairBlock / 64];
  double a = 0.0, b = 0.0, c = 0.0;
  for (long i = threadIdx.x; i < n_rows; i += kPairBlock) {
    a += terms[3 * i];
    b += terms[3 * i + 1];
    c += terms[3 * i + 2];
  }
  a = block_sum(a, part);
  b = block_sum(b, part);
  c = block_sum(c, part);
  if (threadIdx.x == 0) {
    *loss = (float)a;
    *kl = (float)b;
    *clipped = (float)c;
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

template <typename T>
int row_stats(const jtvae_logits_t* g, const int32_t* owner, float* stats, float* lp32, double* lp64, hipStream_t s) {
  hipLaunchKernelGGL(row_stats_kernel<T>, dim3(g->n_rows), dim3(JTVAE_BLOCK), 0, s, (const T*)g->x, (long)g->ld,
                     g->n_cols, Labels{g->labels, g->label_bits}, owner, (float2*)stats, lp32, lp64);
  return launch_status();
}

template <typename T>
int row_grad(const jtvae_logits_t* g, const int32_t* owner, const float* stats, const float* coef,
             const float* upstream, void* dx, int64_t ld_dx, int64_t width, hipStream_t s) {
  hipLaunchKernelGGL(row_grad_kernel<T>, dim3(g->n_rows), dim3(JTVAE_BLOCK), 0, s, (const T*)g->x, (long)g->ld,
                     g->n_cols, Labels{g->labels, g->label_bits}, owner, (const float2*)stats, coef, upstream, (T*)dx,
                     (long)ld_dx, (long)width);
  return launch_status();
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
                              const float* coef, const float* upstream, void* dx, int64_t ld_dx, int64_t width,
                              void* stream) {
  JT_CHECK(check_logits(logits));
  if (width < logits->n_cols || ld_dx < width) return JTVAE_E_SHAPE;
  if (logits->n_rows == 0) return 0;
  if (!stats || !coef || !dx) return JTVAE_E_NULL;
  if ((uintptr_t)dx % (logits->dtype == JTVAE_F32 ? 4 : 2)) return JTVAE_E_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  switch (logits->dtype) {
    case JTVAE_F32: return row_grad<float>(logits, owner, stats, coef, upstream, dx, ld_dx, width, s);
    case JTVAE_F16: return row_grad<_Float16>(logits, owner, stats, coef, upstream, dx, ld_dx, width, s);
    default: return row_grad<__bf16>(logits, owner, stats, coef, upstream, dx, ld_dx, width, s);
  }
}

int jtvae_sequence_sums(const double* log_probs64, const int32_t* rowptr, const int32_t* rows, int32_t n_seq,
                        const float* other, double* sums64, float* sums, void* stream) {
  if (n_seq < 0) return JTVAE_E_SHAPE;
  if (n_seq == 0) return 0;
  if (!log_probs64 || !rowptr || !rows || !sums) return JTVAE_E_NULL;
  hipLaunchKernelGGL(sequence_sums_kernel, dim3(grid_for((long)n_seq * 64)), dim3(JTVAE_BLOCK), 0,
                     (hipStream_t)stream, log_probs64, rowptr, rows, n_seq, other, sums64, sums);
  return launch_status();
}

int jtvae_preference_pairs(const double* sums64, const float* ref, const int32_t* pairs, int32_t n_pairs,
                           const int32_t* seq_ptr, const int32_t* seq_pairs, int32_t n_seq, double beta,
                           double smoothing, double scale, float* loss, float* margins, double* dmargin, float* coef,
                           void* stream) {
  if (n_pairs < 0 || n_seq < 0) return JTVAE_E_SHAPE;
  if (!loss || (n_seq && (!seq_ptr || !coef))) return JTVAE_E_NULL;
  if (n_pairs && (!sums64 || !ref || !pairs || !seq_pairs || !margins || !dmargin)) return JTVAE_E_NULL;
  if (!(smoothing >= 0.0 && smoothing <= 1.0)) return JTVAE_E_RANGE;
  hipLaunchKernelGGL(preference_pairs_kernel, dim3(1), dim3(kPairBlock), 0, (hipStream_t)stream, sums64, ref,
                     (const int2*)pairs, n_pairs, seq_ptr, seq_pairs, n_seq, beta, smoothing, scale, loss, margins,
                     dmargin, coef);
  return launch_status();
}

size_t jtvae_policy_loss_workspace_bytes(int32_t n_rows) {
  return n_rows > 0 ? (size_t)n_rows * 4 * sizeof(double) : 0;
}

int jtvae_policy_loss(const jtvae_logits_t* logits, const jtvae_policy_t* policy, float* stats, float* log_probs,
                      float* coef, float* loss, float* kl, float* clipped, void* workspace, size_t workspace_bytes,
                      void* stream) {
  JT_CHECK(check_logits(logits));
  if (!policy || !loss || !kl || !clipped) return JTVAE_E_NULL;
  const int n = logits->n_rows;
  if (n > 0 && (!stats || !log_probs || !coef || !workspace || !policy->old_log_probs || !policy->advantages))
    return JTVAE_E_NULL;
  if (workspace_bytes < jtvae_policy_loss_workspace_bytes(n)) return JTVAE_E_WORKSPACE;
  if (!(policy->clip_low >= 0.0 && policy->clip_low <= 1.0 && policy->clip_high >= 0.0)) return JTVAE_E_RANGE;
  hipStream_t s = (hipStream_t)stream;
  double* lp64 = (double*)workspace;
  double* terms = lp64 + n;
  if (n > 0) {
    PolicyIn in = {policy->old_log_probs, policy->advantages, policy->ref_log_probs, policy->weights,
                   1.0 - policy->clip_low, 1.0 + policy->clip_high, policy->kl_coef, policy->scale};
    JT_CHECK(jtvae_label_log_probs(logits, nullptr, stats, log_probs, lp64, stream));
    hipLaunchKernelGGL(policy_rows_kernel, dim3(grid_for(n)), dim3(JTVAE_BLOCK), 0, s, in, lp64,
                       Labels{logits->labels, logits->label_bits}, n, coef, terms);
    JT_CHECK(launch_status());
  }
  hipLaunchKernelGGL(sum_terms_kernel, dim3(1), dim3(kPairBlock), 0, s, terms, n, loss, kl, clipped);
  return launch_status();
}

}  // extern "C"
