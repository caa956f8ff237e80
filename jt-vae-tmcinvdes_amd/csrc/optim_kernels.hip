// AdamW over many tensors at once: one launch for all tensors of a group, states in fp32 or in 8 bits with a scale per
// 256 elements, and the global 2-norm of the gradients that the step multiplies them down to.
//
// A workgroup owns one chunk of one tensor (the chunk list is built once); a wave owns whole 256-element blocks of it,
// four elements a lane, so that a block's scale is one wave reduction.  The addresses of the gradients, which change
// from step to step, travel with the launch.
#include "../../include/jtvae_hip.h"
#include "jtvae_common.h"

namespace {

constexpr int kBlock = 256;                   // threads of a workgroup
constexpr int kGroup = JTVAE_ADAMW_BLOCK;     // elements that share a scale: 64 lanes x 4
constexpr float kSmallest = 0x1p-100f;        // maxima up to this count as zero
constexpr float kTop = 448.f;                 // largest e4m3 value
static_assert(kGroup == 256 && JTVAE_ADAMW_CHUNK % (kBlock * 4) == 0, "a wave owns whole blocks");

struct Grads {
  const void* at[JTVAE_ADAMW_MAX_TENSORS];
  int first;  // tensor of at[0]
};

inline int launch_status() {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, long i, long n, float v[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = i + k < n ? (float)p[i + k] : 0.f;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, long i, long n, const float v[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) p[i + k] = (T)v[k];
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
    for (int i = threadIdx.x * 4; i < JTVAE_ADAMW_CHUNK; i += kBlock * 4) {
      float v[4];
      load4(g, base + i, n, v);
      acc += (double)(v[0] * v[0] + v[1] * v[1] + v[2] * v[2] + v[3] * v[3]);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) partials[chunk] = part[0] + part[1] + part[2] + part[3];
}

constexpr int kNormBlock = 1024;

__global__ __launch_bounds__(kNormBlock) void grad_norm_kernel(const double* __restrict__ partials, long n,
                                                               double max_norm, float* __restrict__ norm) {
  __shared__ double part[kNormBlock / 64];
  double acc = 0.0;
  for (long i = threadIdx.x; i < n; i += kNormBlock) acc += partials[i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < kNormBlock / 64; ++w) t += part[w];
    t = sqrt(t);
    const double coef = max_norm / (t + 1e-6);
    norm[0] = (float)t;
    norm[1] = coef < 1.0 ? (float)coef : (coef == coef ? 1.f : (float)coef);  // a NaN norm stays visible
  }
}

struct Present {
  unsigned bits[(JTVAE_ADAMW_MAX_TENSORS + 31) / 32];
  int first, count;
};

// t = ++steps of the tensors that have a gradient; bias = (1 / (1 - beta1^t), 1 / sqrt(1 - beta2^t)), in fp64.
__global__ __launch_bounds__(kBlock) void steps_kernel(int* __restrict__ steps, float2* __restrict__ bias,
                                                       Present present, double beta1, double beta2) {
  const int i = blockIdx.x * kBlock + threadIdx.x;
  if (i >= present.count || !(present.bits[i >> 5] >> (i & 31) & 1)) return;
  const int t = ++steps[present.first + i];
  bias[present.first + i] =
      make_float2((float)(1.0 / (1.0 - pow(beta1, (double)t))), (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t))));
}

struct Hyper {
  float lr, decay, beta1, one_m_beta1, beta2, one_m_beta2, eps;
  const float *lr_device, *grad_scale;
};

// Four e4m3 values of one 32-bit word, and back with the format's rounding to nearest even.
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

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  return v;
}

// Largest finite magnitude of a wave's 256 values: the scale is not lost to one element that overflowed.
__device__ __forceinline__ float block_top(const float v[4]) {
  float t = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float a = fabsf(v[k]);
    if (a < INFINITY) t = fmaxf(t, a);
  }
  return wave_max(t);
}

template <bool ROOT>
__device__ __forceinline__ unsigned quantise(const float v[4], float top) {
  const float inv = top > kSmallest ? kTop / top : 0.f;
  float q[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    q[k] = v[k] * inv;
    if (ROOT && q[k] > 0.f) q[k] = fmaxf(q[k], 0x1p-9f);
    if (!(fabsf(v[k]) < INFINITY)) q[k] = NAN;
    else q[k] = fminf(fmaxf(q[k], -kTop), kTop);
  }
  return pack_e4m3(q);
}

template <typename T, bool MASTER, int BITS>
__global__ __launch_bounds__(kBlock) void adamw_kernel(const jtvae_adamw_tensor_t* __restrict__ tensors,
                                                       const int2* __restrict__ chunks, long first_chunk, Grads grads,
                                                       const float2* __restrict__ bias, Hyper h) {
  const int2 c = chunks[first_chunk + blockIdx.x];
  const T* g = (const T*)grads.at[c.x - grads.first];
  if (!g) return;
  const jtvae_adamw_tensor_t t = tensors[c.x];
  const float2 b = bias[c.x];
  const float lr = h.lr_device ? *h.lr_device : h.lr;
  const float gs = h.grad_scale ? *h.grad_scale : 1.f;
  const float keep = 1.f - lr * h.decay, rate = lr * b.x;
  const long base = (long)c.y * JTVAE_ADAMW_CHUNK;
  const int lane = threadIdx.x & 63;
  for (int i = threadIdx.x * 4; i < JTVAE_ADAMW_CHUNK; i += kBlock * 4) {
    const long at = base + i;
    if (at - lane * 4 >= t.n) break;  // the same for every lane of a wave: its first element
    float gv[4], w[4], m[4], v[4], r[4];
    load4(g, at, t.n, gv);
    if (MASTER) load4(t.master, at, t.n, w);
    else load4((const T*)t.param, at, t.n, w);
    if constexpr (BITS == 32) {
      load4((const float*)t.exp_avg, at, t.n, m);
      load4((const float*)t.second, at, t.n, v);
    } else {
      const long blk = at / kGroup;
      const float sm = t.exp_avg_scale[blk], sr = t.second_scale[blk];
      unsigned qm = 0, qr = 0;
      for (int k = 0; k < 4; ++k)
        if (at + k < t.n) {
          qm |= (unsigned)((const uint8_t*)t.exp_avg)[at + k] << (8 * k);
          qr |= (unsigned)((const uint8_t*)t.second)[at + k] << (8 * k);
        }
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
      const float x = gv[k] * gs;
      m[k] = h.beta1 * m[k] + h.one_m_beta1 * x;
      v[k] = h.beta2 * v[k] + h.one_m_beta2 * (x * x);
      r[k] = sqrtf(v[k]);
      w[k] = w[k] * keep - rate * (m[k] / (r[k] * b.y + h.eps));
    }
    if (MASTER) store4(t.master, at, t.n, w);
    store4((T*)t.param, at, t.n, w);
    if constexpr (BITS == 32) {
      store4((float*)t.exp_avg, at, t.n, m);
      store4((float*)t.second, at, t.n, v);
    } else {
      const float tm = block_top(m), tr = block_top(r);
      const unsigned qm = quantise<false>(m, tm), qr = quantise<true>(r, tr);
      for (int k = 0; k < 4; ++k)
        if (at + k < t.n) {
          ((uint8_t*)t.exp_avg)[at + k] = (uint8_t)(qm >> (8 * k));
          ((uint8_t*)t.second)[at + k] = (uint8_t)(qr >> (8 * k));
        }
      if (lane == 0) {
        t.exp_avg_scale[at / kGroup] = tm > kSmallest ? tm / kTop : 0.f;
        t.second_scale[at / kGroup] = tr > kSmallest ? tr / kTop : 0.f;
      }
    }
  }
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

// Calls launch(grads, first chunk, number of chunks) for runs of at most JTVAE_ADAMW_MAX_TENSORS tensors.
template <typename F>
int for_runs(const jtvae_adamw_group_t* g, F launch) {
  for (int t0 = 0; t0 < g->n_tensors; t0 += JTVAE_ADAMW_MAX_TENSORS) {
    const int cnt = g->n_tensors - t0 < JTVAE_ADAMW_MAX_TENSORS ? g->n_tensors - t0 : JTVAE_ADAMW_MAX_TENSORS;
    const int64_t c0 = g->chunk_ptr[t0], nc = g->chunk_ptr[t0 + cnt] - c0;
    if (nc <= 0) continue;
    Grads a;
    a.first = t0;
    for (int i = 0; i < cnt; ++i) a.at[i] = g->grads[t0 + i];
    launch(a, (long)c0, (unsigned)nc);
    int rc = launch_status();
    if (rc) return rc;
  }
  return 0;
}

template <typename T, bool MASTER>
int step(const jtvae_adamw_group_t* g, const Hyper& h, hipStream_t s) {
  return for_runs(g, [&](const Grads& a, long c0, unsigned nc) {
    if (g->state_bits == 32)
      hipLaunchKernelGGL((adamw_kernel<T, MASTER, 32>), dim3(nc), dim3(kBlock), 0, s, g->tensors,
                         (const int2*)g->chunks, c0, a, (const float2*)g->bias, h);
    else
      hipLaunchKernelGGL((adamw_kernel<T, MASTER, 8>), dim3(nc), dim3(kBlock), 0, s, g->tensors,
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

int jtvae_grad_square_sums(const jtvae_adamw_group_t* group, double* partials, void* stream) {
  JT_CHECK(check_group(group));
  if (group->n_chunks == 0) return 0;
  if (!partials) return JTVAE_E_NULL;
  hipStream_t s = (hipStream_t)stream;
  switch (group->dtype) {
    case JTVAE_F32: return square_sums<float>(group, partials, s);
    case JTVAE_F16: return square_sums<_Float16>(group, partials, s);
    default: return square_sums<__bf16>(group, partials, s);
  }
}

int jtvae_grad_norm(const double* partials, int64_t n_partials, double max_norm, float* norm, void* stream) {
  if (n_partials < 0) return JTVAE_E_SHAPE;
  if (!norm || (n_partials && !partials)) return JTVAE_E_NULL;
  if (!(max_norm > 0.0)) return JTVAE_E_RANGE;
  hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kNormBlock), 0, (hipStream_t)stream, partials, (long)n_partials,
                     max_norm, norm);
  return launch_status();
}

int jtvae_adamw_step(const jtvae_adamw_group_t* group, const float* grad_scale, void* stream) {
  JT_CHECK(check_group(group));
  const jtvae_adamw_group_t& g = *group;
  if (!(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0 && g.eps >= 0.0)) return JTVAE_E_RANGE;
  if (g.n_tensors == 0 || g.n_chunks == 0) return 0;
  if (!g.steps || !g.bias) return JTVAE_E_NULL;
  hipStream_t s = (hipStream_t)stream;
  for (int t0 = 0; t0 < g.n_tensors; t0 += JTVAE_ADAMW_MAX_TENSORS) {
    Present p = {};
    p.first = t0;
    p.count = g.n_tensors - t0 < JTVAE_ADAMW_MAX_TENSORS ? g.n_tensors - t0 : JTVAE_ADAMW_MAX_TENSORS;
    for (int i = 0; i < p.count; ++i)
      if (g.grads[t0 + i]) p.bits[i >> 5] |= 1u << (i & 31);
    hipLaunchKernelGGL(steps_kernel, dim3((p.count + kBlock - 1) / kBlock), dim3(kBlock), 0, s, g.steps,
                       (float2*)g.bias, p, g.beta1, g.beta2);
    JT_CHECK(launch_status());
  }
  const Hyper h = {(float)g.lr,    (float)g.weight_decay,  (float)g.beta1, (float)(1.0 - g.beta1),
                   (float)g.beta2, (float)(1.0 - g.beta2), (float)g.eps,   g.lr_device,
                   grad_scale};
  const bool master = g.dtype != JTVAE_F32 && g.use_master;
  switch (g.dtype) {
    case JTVAE_F32: return step<float, false>(group, h, s);
    case JTVAE_F16: return master ? step<_Float16, true>(group, h, s) : step<_Float16, false>(group, h, s);
    default: return master ? step<__bf16, true>(group, h, s) : step<__bf16, false>(group, h, s);
  }
}

}  // extern "C"
