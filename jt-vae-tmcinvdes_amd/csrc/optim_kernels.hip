// AdamW over many tensors at once: one launch for all tensors of a group, states in fp32 or in 8 bits with a scale per
// 256 elements, and the global 2-norm of the gradients that the step multiplies them down to.
//
// A workgroup owns one chunk of one tensor (the chunk list is built once), a wave whole 256-element blocks of it, so that
// a block's scale is a reduction over neighbouring lanes.  The addresses of the gradients, which change from step to
// step, travel with the launch.
#include "../../include/jtvae_hip.h"
#include "jtvae_common.h"

namespace {

constexpr int kBlock = 256;                   // threads of a workgroup
constexpr int kGroup = JTVAE_ADAMW_BLOCK;     // elements that share a scale
constexpr float kSmallest = 0x1p-100f;        // maxima up to this count as zero
constexpr float kTop = 448.f;                 // largest e4m3 value
static_assert(kGroup == 256 && JTVAE_ADAMW_CHUNK % kGroup == 0, "a wave owns whole blocks");

struct Grads {
  const void* at[JTVAE_ADAMW_MAX_TENSORS];
  int first;  // tensor of at[0]
};

inline int launch_status() {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}

// N consecutive elements from i, at the type's own alignment (the hardware takes an access of 16 bytes at any address).
// WHOLE: all of them exist, else those from n on read as zero and are not written.  ONCE: past the caches - a step
// touches every byte once, and no chip-wide cache holds a model's states until the next one.
template <int BYTES>
struct Words;
template <>
struct Words<16> {
  typedef unsigned at4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef unsigned at2 __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct Words<8> {
  typedef unsigned at2 __attribute__((ext_vector_type(2), aligned(2)));
};
template <typename T, int N, bool TWO = sizeof(T) == 2>
struct Run {
  using type = typename Words<N * sizeof(T)>::at4;
};
template <typename T, int N>
struct Run<T, N, true> {
  using type = typename Words<N * sizeof(T)>::at2;
};

template <bool WHOLE, bool ONCE, int N, typename T>
__device__ __forceinline__ void load(const T* p, long i, long n, float v[N]) {
  if constexpr (WHOLE) {
    using R = typename Run<T, N>::type;
    R r;
    if constexpr (ONCE) r = __builtin_nontemporal_load((const R*)(p + i));
    else r = *(const R*)(p + i);
    T h[N];
    __builtin_memcpy(h, &r, sizeof(h));
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = (float)h[k];
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = i + k < n ? (float)p[i + k] : 0.f;
  }
}
template <bool WHOLE, int N, typename T>
__device__ __forceinline__ void store(T* p, long i, long n, const float v[N]) {
  if constexpr (WHOLE) {
    using R = typename Run<T, N>::type;
    T h[N];
#pragma unroll
    for (int k = 0; k < N; ++k) h[k] = (T)v[k];
    R r;
    __builtin_memcpy(&r, h, sizeof(h));
    __builtin_nontemporal_store(r, (R*)(p + i));
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (i + k < n) p[i + k] = (T)v[k];
  }
}

// Sum of a lane's squares in a chunk: 32 bits over the elements of a load, 64 beyond.  Where one of those overflows, or is so
// small that squares may have vanished beside it (below 2^-126), all is formed in 64 bits, once more from the registers.
template <bool WHOLE, typename T>
__device__ __forceinline__ double chunk_squares(const T* g, long base, long n) {
  constexpr int N = 16 / sizeof(T), U = JTVAE_ADAMW_CHUNK / (kBlock * N);
  float v[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u) load<WHOLE, false, N>(g, base + (u * kBlock + threadIdx.x) * N, n, v[u]);
  double acc = 0.0;
  bool fine = true;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) s = fmaf(v[u][k], v[u][k], s);
    fine = fine && s > 0x1p-80f && s < INFINITY;
    acc += (double)s;
  }
  if (fine) return acc;
  acc = 0.0;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < N; ++k) acc = fma((double)v[u][k], (double)v[u][k], acc);
  return acc;
}

template <typename T>
__global__ __launch_bounds__(kBlock) void square_sums_kernel(const jtvae_adamw_tensor_t* __restrict__ tensors,
                                                             const int2* __restrict__ chunks, long first_chunk,
                                                             Grads grads, double* __restrict__ partials) {
  __shared__ double part[kBlock / 64];
  const long chunk = first_chunk + blockIdx.x;
  const int2 c = chunks[chunk];
  const T* g = (const T*)grads.at[c.x - grads.first];
  double acc = 0.0;
  if (g) {
    const long n = tensors[c.x].n, base = (long)c.y * JTVAE_ADAMW_CHUNK;
    acc = base + JTVAE_ADAMW_CHUNK <= n ? chunk_squares<true>(g, base, n) : chunk_squares<false>(g, base, n);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) partials[chunk] = part[0] + part[1] + part[2] + part[3];
}

constexpr int kPrepBlock = 1024;
static_assert(JTVAE_ADAMW_MAX_TENSORS <= kPrepBlock, "one thread per tensor");

struct Present {
  unsigned bits[(JTVAE_ADAMW_MAX_TENSORS + 31) / 32];
  int first, count;
};

struct Norm {
  const double* partials;
  long n;
  double max_norm;
  float* out;
};

// What the update needs before it starts.  Block 0: t = ++steps of the tensors that have a gradient and their bias
// corrections (1 / (1 - beta1^t), 1 / sqrt(1 - beta2^t)), formed in fp64.  Block 1, where the gradients are clipped: the
// norm from the chunks' sums in a fixed order, and the factor min(1, max_norm / (norm + 1e-6)).
__global__ __launch_bounds__(kPrepBlock) void prepare_kernel(int* __restrict__ steps, float2* __restrict__ bias,
                                                             Present present, double beta1, double beta2, Norm norm) {
  __shared__ double part[kPrepBlock / 64];
  const int i = threadIdx.x;
  if (blockIdx.x == 0) {
    if (i >= present.count || !(present.bits[i >> 5] >> (i & 31) & 1)) return;
    const int t = ++steps[present.first + i];
    bias[present.first + i] = make_float2((float)(1.0 / (1.0 - pow(beta1, (double)t))),
                                          (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t))));
    return;
  }
  double acc = 0.0;
#pragma unroll 8
  for (long k = i; k < norm.n; k += kPrepBlock) acc += norm.partials[k];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
  if ((i & 63) == 0) part[i >> 6] = acc;
  __syncthreads();
  if (i == 0) {
    double t = 0.0;
    for (int w = 0; w < kPrepBlock / 64; ++w) t += part[w];
    t = sqrt(t);
    const double coef = norm.max_norm / (t + 1e-6);
    norm.out[0] = (float)t;
    norm.out[1] = coef < 1.0 ? (float)coef : (coef == coef ? 1.f : (float)coef);  // a NaN norm stays visible
  }
}

struct Hyper {
  float lr, decay, beta1, one_m_beta1, beta2, one_m_beta2, eps;
  const float *lr_device, *grad_scale;
  const int* steps;  // where rounding is stochastic, else NULL
};

// The four e4m3 values of a word, and back with the format's rounding to nearest even.
__device__ __forceinline__ void unpack_e4m3(unsigned w, float v[4]) {
  auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  v[0] = lo[0];
  v[1] = lo[1];
  v[2] = hi[0];
  v[3] = hi[1];
}
__device__ __forceinline__ unsigned pack_e4m3(const float v[4]) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
  return (unsigned)w;
}

// Largest finite magnitude of a wave's 256 values: a scale is not lost to one element that overflowed.
__device__ __forceinline__ float block_top(const float v[4]) {
  float t = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float a = fabsf(v[k]);
    t = fmaxf(t, a < INFINITY ? a : 0.f);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) t = fmaxf(t, __shfl_xor(t, off, 64));
  return t;
}

// Well mixed bits of a counter (xor-shifts and odd multipliers; every output once over all counters).  The shifts and
// multipliers are the ones published by C. Wellons, "Prospecting for Hash Functions" (2018).
__device__ __forceinline__ unsigned mix(unsigned x) {
  x = (x ^ (x >> 16)) * 0x7feb352du;
  x = (x ^ (x >> 15)) * 0x846ca68bu;
  return x ^ (x >> 16);
}

// One of the two e4m3 values next to x (|x| <= 448), the nearer the likelier, so that the mean is x: the bits below the
// format's last place are added to and cut off.  Below 2^-6 the format's places are as wide as between 2^-6 and 2^-5,
// where the value is shifted for it.
__device__ __forceinline__ float round_by(float x, unsigned bits20) {
  const float a = fabsf(x), low = a < 0x1p-6f ? 0x1p-6f : 0.f;
  const unsigned w = (__float_as_uint(a + low) + bits20) & 0xfff00000u;
  return copysignf(fminf(__uint_as_float(w) - low, kTop), x);
}

// e4m3 values of v over the block's scale.  `dice`: 0 = to nearest, else 20 random bits per element (low 20 bits of each).
template <bool ROOT>
__device__ __forceinline__ unsigned quantise(const float v[4], float top, bool by_dice, const unsigned dice[4]) {
  const float inv = top > kSmallest ? 1.f / top * kTop : 0.f;
  float x[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float y = fminf(fmaxf(v[k] * inv, -kTop), kTop);
    if (by_dice) y = round_by(y, dice[k]);
    if (ROOT) y = v[k] > 0.f && inv > 0.f ? fmaxf(y, 0x1p-9f) : y;
    x[k] = fabsf(v[k]) < INFINITY ? y : NAN;
  }
  return pack_e4m3(x);
}

// sqrt on the hardware unit (1 ulp), with what it would flush brought into its range first.  Rounded correctly it takes 4 %
// of a whole step more (477 M bf16 elements, 8-bit states: 1432 us against 1377).
__device__ __forceinline__ float root(float v) {
  const bool low = v < 0x1p-96f;
  const float r = __builtin_amdgcn_sqrtf(low ? v * 0x1p96f : v);
  return low ? r * 0x1p-48f : r;
}

struct Step {
  unsigned dice;  // of the tensor and its step; 0: round to nearest
  float decay, rate, eps, beta1, one_m_beta1, beta2, one_m_beta2, grad_scale, bias2;
};

// The four elements of a tensor from `at`.  8-bit states: a wave's 256 elements are a block, which shares a scale; its
// buffers are padded to whole blocks.
template <typename T, bool MASTER, int BITS, bool WHOLE>
__device__ __forceinline__ void update(const jtvae_adamw_tensor_t& t, const T* grad, const Step& s, long at) {
  float g[4], w[4], m[4], v[4], r[4];
  load<WHOLE, true, 4>(grad, at, t.n, g);
  if constexpr (MASTER) load<WHOLE, true, 4>((const float*)t.master, at, t.n, w);
  else load<WHOLE, true, 4>((const T*)t.param, at, t.n, w);
  if constexpr (BITS == 32) {
    load<WHOLE, true, 4>((const float*)t.exp_avg, at, t.n, m);
    load<WHOLE, true, 4>((const float*)t.second, at, t.n, v);
  } else {
    const unsigned qm = __builtin_nontemporal_load((const unsigned*)((const uint8_t*)t.exp_avg + at));
    const unsigned qr = __builtin_nontemporal_load((const unsigned*)((const uint8_t*)t.second + at));
    const float sm = t.exp_avg_scale[at / kGroup], sr = t.second_scale[at / kGroup];
    unpack_e4m3(qm, m);
    unpack_e4m3(qr, r);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      m[k] *= sm;
      r[k] *= sr;
      v[k] = r[k] * r[k];
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    // the order of the elementary operations (decay, then add), which settles where an 8-bit state near a tie goes
    const float x = g[k] * s.grad_scale;
    m[k] = fmaf(s.one_m_beta1, x, s.beta1 * m[k]);
    v[k] = s.beta2 * v[k] + s.one_m_beta2 * (x * x);
    r[k] = root(v[k]);
    // decay and update are one change, rounded into w once: a factor 1 - lr * decay would hold the decay in steps of
    // 2^-24 (none at all below 2^-25).  Reciprocal on the hardware unit (1 ulp): first steps from zero, which are the
    // update itself, are off by up to 5.2 * 2^-24 of themselves (1e5 elements), 4.7 with a correctly rounded quotient, which
    // takes 0.2 % longer
    const float shrink = fabsf(w[k]) < INFINITY ? s.decay * w[k] : 0.f;  // an infinite weight stays
    w[k] -= fmaf(s.rate, m[k] * __builtin_amdgcn_rcpf(r[k] * s.bias2 + s.eps), shrink);
    // a 16-bit parameter is the 32-bit value rounded: the compiler must not round the sum to 16 bits by itself
    if constexpr (sizeof(T) == 2) asm("" : "+v"(w[k]));
  }
  if constexpr (MASTER) store<WHOLE, 4>(t.master, at, t.n, w);
  store<WHOLE, 4>((T*)t.param, at, t.n, w);
  if constexpr (BITS == 32) {
    store<WHOLE, 4>((float*)t.exp_avg, at, t.n, m);
    store<WHOLE, 4>((float*)t.second, at, t.n, v);
  } else {
    if constexpr (!WHOLE) {  // the padding after the last element stays zero
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (at + k >= t.n) m[k] = r[k] = 0.f;
    }
    const float tm = block_top(m), tr = block_top(r);
    unsigned dm[4], dr[4];
    if (s.dice) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned x = mix((unsigned)(at + k) ^ s.dice ^ (unsigned)((at + k) >> 32) * 0x9e3779b9u);
        dm[k] = x >> 12;
        dr[k] = mix(x) >> 12;
      }
    }
    __builtin_nontemporal_store(quantise<false>(m, tm, s.dice != 0, dm), (unsigned*)((uint8_t*)t.exp_avg + at));
    __builtin_nontemporal_store(quantise<true>(r, tr, s.dice != 0, dr), (unsigned*)((uint8_t*)t.second + at));
    if ((threadIdx.x & 63) == 0) {
      t.exp_avg_scale[at / kGroup] = tm > kSmallest ? tm / kTop : 0.f;
      t.second_scale[at / kGroup] = tr > kSmallest ? tr / kTop : 0.f;
    }
  }
}

// One round of a block's lanes, four elements each.  Bound by memory: 28 bytes per fp32 element with 32-bit states, 16
// per bf16 element with a copy and 8-bit states.  A copy on this card reaches 6.2-6.6 TB/s with one 16-byte access per
// lane and block and 4.2 with eight - the fewer bytes a block holds, the closer together the places the chip works on
// at a time - and so it is here: rounds of 1024 elements past the caches take 1396 us for 477 M bf16 elements with
// 8-bit states, chunks of 4096 through the caches 1642 (the norm's pass included).
constexpr int kRound = kBlock * 4, kRounds = JTVAE_ADAMW_CHUNK / kRound;
static_assert(JTVAE_ADAMW_CHUNK % kRound == 0 && kRound % kGroup == 0, "whole rounds of whole blocks");

template <typename T, bool MASTER, int BITS>
__global__ __launch_bounds__(kBlock) void adamw_kernel(const jtvae_adamw_tensor_t* __restrict__ tensors,
                                                       const int2* __restrict__ chunks, long first_chunk, Grads grads,
                                                       const float2* __restrict__ bias, Hyper h) {
  const int2 c = chunks[first_chunk + blockIdx.x / kRounds];
  const T* g = (const T*)grads.at[c.x - grads.first];
  if (!g) return;
  const jtvae_adamw_tensor_t t = tensors[c.x];
  const long base = (long)c.y * JTVAE_ADAMW_CHUNK + (blockIdx.x % kRounds) * kRound;
  const long at = base + threadIdx.x * 4;
  if (at / kGroup * kGroup >= t.n) return;  // the same for the lanes of a wave: the first element of their block
  const float2 b = bias[c.x];
  const float lr = h.lr_device ? *h.lr_device : h.lr;
  // the same rounding for the same step of the same tensor, whatever the launch
  const unsigned dice = BITS == 8 && h.steps ? mix((unsigned)h.steps[c.x] * 0x9e3779b9u + (unsigned)c.x) | 1u : 0u;
  const Step s = {dice, lr * h.decay, lr * b.x, h.eps, h.beta1, h.one_m_beta1, h.beta2, h.one_m_beta2,
                  h.grad_scale ? *h.grad_scale : 1.f, b.y};
  if (base + kRound <= t.n) update<T, MASTER, BITS, true>(t, g, s, at);
  else update<T, MASTER, BITS, false>(t, g, s, at);
}

int check_group(const jtvae_adamw_group_t* g) {
  if (!g) return JTVAE_E_NULL;
  if (g->n_tensors < 0 || g->n_chunks < 0) return JTVAE_E_SHAPE;
  if (g->dtype < JTVAE_F32 || g->dtype > JTVAE_BF16) return JTVAE_E_RANGE;
  if (g->state_bits != 32 && g->state_bits != 8) return JTVAE_E_RANGE;
  if (g->n_tensors && (!g->tensors || !g->chunk_ptr || !g->grads)) return JTVAE_E_NULL;
  if (g->n_chunks && !g->chunks) return JTVAE_E_NULL;
  if (g->n_tensors && (g->chunk_ptr[0] != 0 || g->chunk_ptr[g->n_tensors] != g->n_chunks)) return JTVAE_E_SHAPE;
  return 0;
}

// Calls launch(grads, first chunk, number of chunks) for runs of at most JTVAE_ADAMW_MAX_TENSORS tensors and of as many
// chunks as a grid may have work-items for (2^32).
template <typename F>
int for_runs(const jtvae_adamw_group_t* g, F launch) {
  constexpr int64_t kMost = (int64_t)1 << 21;
  for (int t0 = 0; t0 < g->n_tensors; t0 += JTVAE_ADAMW_MAX_TENSORS) {
    const int cnt = g->n_tensors - t0 < JTVAE_ADAMW_MAX_TENSORS ? g->n_tensors - t0 : JTVAE_ADAMW_MAX_TENSORS;
    Grads a;
    a.first = t0;
    for (int i = 0; i < cnt; ++i) a.at[i] = g->grads[t0 + i];
    const int64_t end = g->chunk_ptr[t0 + cnt];
    for (int64_t c0 = g->chunk_ptr[t0]; c0 < end; c0 += kMost) {
      launch(a, (long)c0, (unsigned)(end - c0 < kMost ? end - c0 : kMost));
      int rc = launch_status();
      if (rc) return rc;
    }
  }
  return 0;
}

template <typename T, bool MASTER>
int step(const jtvae_adamw_group_t* g, const Hyper& h, hipStream_t s) {
  return for_runs(g, [&](const Grads& a, long c0, unsigned nc) {
    if (g->state_bits == 32)
      hipLaunchKernelGGL((adamw_kernel<T, MASTER, 32>), dim3(nc * kRounds), dim3(kBlock), 0, s, g->tensors,
                         (const int2*)g->chunks, c0, a, (const float2*)g->bias, h);
    else
      hipLaunchKernelGGL((adamw_kernel<T, MASTER, 8>), dim3(nc * kRounds), dim3(kBlock), 0, s, g->tensors,
                         (const int2*)g->chunks, c0, a, (const float2*)g->bias, h);
  });
}

template <typename T>
int square_sums(const jtvae_adamw_group_t* g, double* partials, hipStream_t s) {
  return for_runs(g, [&](const Grads& a, long c0, unsigned nc) {
    hipLaunchKernelGGL(square_sums_kernel<T>, dim3(nc), dim3(kBlock), 0, s, g->tensors, (const int2*)g->chunks, c0, a,
                       partials);
  });
}

}  // namespace

#define JT_CHECK(expr)        \
  do {                        \
    int _rc = (expr);         \
    if (_rc) return _rc;      \
  } while (0)

extern "C" {

int jtvae_adamw_step(const jtvae_adamw_group_t* groups, int32_t n_groups, double max_norm, double* partials,
                     float* norm, void* stream) {
  if (n_groups < 0) return JTVAE_E_SHAPE;
  if (n_groups && !groups) return JTVAE_E_NULL;
  if (!(max_norm >= 0.0)) return JTVAE_E_RANGE;
  if (max_norm > 0.0 && (!partials || !norm)) return JTVAE_E_NULL;
  for (int i = 0; i < n_groups; ++i) {
    const jtvae_adamw_group_t& g = groups[i];
    JT_CHECK(check_group(&g));
    if (!(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0 && g.eps >= 0.0)) return JTVAE_E_RANGE;
    if (g.n_tensors && (!g.steps || !g.bias)) return JTVAE_E_NULL;
  }
  hipStream_t s = (hipStream_t)stream;
  Norm total = {partials, 0, max_norm, norm};
  if (max_norm > 0.0) {
    for (int i = 0; i < n_groups; ++i) {
      const jtvae_adamw_group_t* g = groups + i;
      double* p = partials + total.n;
      switch (g->dtype) {
        case JTVAE_F32: JT_CHECK(square_sums<float>(g, p, s)); break;
        case JTVAE_F16: JT_CHECK(square_sums<_Float16>(g, p, s)); break;
        default: JT_CHECK(square_sums<__bf16>(g, p, s));
      }
      total.n += g->n_chunks;
    }
  }
  bool norm_due = max_norm > 0.0;
  for (int i = 0; i < n_groups; ++i) {
    const jtvae_adamw_group_t& g = groups[i];
    for (int t0 = 0; t0 < g.n_tensors; t0 += JTVAE_ADAMW_MAX_TENSORS) {
      Present p = {};
      p.first = t0;
      p.count = g.n_tensors - t0 < JTVAE_ADAMW_MAX_TENSORS ? g.n_tensors - t0 : JTVAE_ADAMW_MAX_TENSORS;
      for (int k = 0; k < p.count; ++k)
        if (g.grads[t0 + k]) p.bits[k >> 5] |= 1u << (k & 31);
      hipLaunchKernelGGL(prepare_kernel, dim3(norm_due ? 2 : 1), dim3(kPrepBlock), 0, s, g.steps, (float2*)g.bias, p,
                         g.beta1, g.beta2, total);
      JT_CHECK(launch_status());
      norm_due = false;
    }
  }
  for (int i = 0; i < n_groups; ++i) {
    const jtvae_adamw_group_t& g = groups[i];
    const Hyper h = {(float)g.lr,    (float)g.weight_decay,  (float)g.beta1, (float)(1.0 - g.beta1),
                     (float)g.beta2, (float)(1.0 - g.beta2), (float)g.eps,   g.lr_device,
                     max_norm > 0.0 ? norm + 1 : nullptr,
                     g.stochastic ? g.steps : nullptr};
    const bool master = g.dtype != JTVAE_F32 && g.use_master;
    int rc;
    switch (g.dtype) {
      case JTVAE_F32: rc = step<float, false>(&g, h, s); break;
      case JTVAE_F16: rc = master ? step<_Float16, true>(&g, h, s) : step<_Float16, false>(&g, h, s); break;
      default: rc = master ? step<__bf16, true>(&g, h, s) : step<__bf16, false>(&g, h, s);
    }
    if (rc) return rc;
  }
  return 0;
}

}  // extern "C"
