// Softmax over a vocabulary with one given token per row: its log probability, the entropy, the most likely alternatives, and the logits'
// gradient, of the token loss or of whatever is made of the log probability and the entropy.
//
//   z = sum exp(x - m), m = max x      lse = m + ln z      logp = (x_t - m) - ln z      entropy = ln z - sum exp(x - m) (x - m) / z
//   d logp / dx_v = 1[v = t] - p_v      d entropy / dx_v = -p_v (ln p_v + entropy)
//
// All of it is f32 whatever the logits' type; x - m before the multiplication by log2 e, so that logits of any size keep their distances.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "ono_kernels.h"
#include "piece.cuh"
#include "ptx.cuh"

namespace ono {
void set_error(const char* fmt, const char* a, long long b, long long c);

constexpr int TOK_THREADS = 256;

__device__ __forceinline__ float exp_of(float d) {      // exp(d)
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.4426950408889634f));
  return r;
}

// The row's token: -1 where the row is not read.
__device__ __forceinline__ int row_target(const void* targets, int wide, long long r, int V, long long ignore_id, int* status) {
  const long long t = wide ? reinterpret_cast<const long long*>(targets)[r] : (long long)reinterpret_cast<const int*>(targets)[r];
  if (t == ignore_id) return -1;
  if (t >= 0 && t < V) return (int)t;
  if (status && threadIdx.x == 0) atomicExch(status, ONO_ERR_BAD_ARG);
  return -1;
}

// Larger for a larger logit, and among equal ones for the lower index. (-0 counts as 0.)
__device__ __forceinline__ unsigned long long top_key(float v, int j) {
  const unsigned int u = __float_as_uint(v + 0.0f);
  return ((unsigned long long)(u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u)) << 32) | (0xffffffffu - (unsigned int)j);
}
__device__ __forceinline__ float key_logit(unsigned long long key) {
  const unsigned int o = (unsigned int)(key >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}

template <class V, class F>
__device__ __forceinline__ V block_all(V v, V* s, F join) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
  for (int w = 1; w < TOK_THREADS / 32; ++w) v = join(v, s[w]);
  return v;
}

template <typename T, typename O>
__global__ void __launch_bounds__(TOK_THREADS) tokens_kernel(const OnoTokens a) {
  __shared__ unsigned long long s_red[TOK_THREADS / 32];
  float* sf = reinterpret_cast<float*>(s_red);
  const float ninf = __int_as_float(0xff800000);
  auto add = [](float p, float q) { return p + q; };
  auto largest = [](float p, float q) { return fmaxf(p, q); };
  for (long long r = blockIdx.x; r < a.R; r += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + r * a.ld;
    O* d = a.out ? reinterpret_cast<O*>(a.out) + r * a.ld_out : nullptr;
    const int t = a.targets ? row_target(a.targets, a.targets64, r, a.V, a.ignore_id, a.status) : 0;
    if (t < 0) {
      if (threadIdx.x == 0) {
        if (a.logp) a.logp[r] = 0.0f;
        if (a.lse) a.lse[r] = 0.0f;
        if (a.entropy) a.entropy[r] = 0.0f;
      }
      for (int k = threadIdx.x; k < a.top; k += TOK_THREADS) { a.top_logp[r * a.top + k] = ninf; a.top_id[r * a.top + k] = -1; }
      if (d) for (int j = threadIdx.x; j < a.V; j += TOK_THREADS) d[j] = from_f32<O>(0.0f);
      continue;
    }
    float m = ninf;
    for (int j = threadIdx.x; j < a.V; j += TOK_THREADS) m = fmaxf(m, to_f32(x[j]));
    m = block_all(m, sf, largest);
    const float base = m == ninf ? 0.0f : m;      // (a row of -inf alone sums to zero, one with NaN to NaN)
    float z = 0.0f, u = 0.0f;
    for (int j = threadIdx.x; j < a.V; j += TOK_THREADS) {
      const float dist = to_f32(x[j]) - base, e = exp_of(dist);
      z += e;
      u += e * fmaxf(dist, -1e4f);
    }
    z = block_all(z, sf, add);
    u = block_all(u, sf, add);
    const bool empty = z == 0.0f;
    const float log_z = empty ? 0.0f : logf(z);
    if (threadIdx.x == 0) {
      if (a.lse) a.lse[r] = empty ? ninf : m + log_z;
      if (a.logp) a.logp[r] = empty ? ninf : (to_f32(x[t]) - m) - log_z;
      if (a.entropy) a.entropy[r] = empty ? 0.0f : log_z - u / z;
    }
    unsigned long long prev = ~0ull;
    for (int k = 0; k < a.top; ++k) {
      unsigned long long best = 0;
      for (int j = threadIdx.x; j < a.V; j += TOK_THREADS) {
        const float v = to_f32(x[j]);
        const unsigned long long key = v > ninf ? top_key(v, j) : 0;
        if (key < prev && key > best) best = key;
      }
      best = block_all(best, s_red, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
      if (threadIdx.x == 0) {
        a.top_logp[r * a.top + k] = best ? (key_logit(best) - m) - log_z : ninf;
        a.top_id[r * a.top + k] = best ? (int)(0xffffffffu - (unsigned int)best) : -1;
      }
      prev = best;
    }
    if (d) {
      const float w = a.scale * (a.weight ? a.weight[r] : 1.0f), inv = w / z, hit = to_f32(x[t]);
      const float at_t = empty ? 0.0f : exp_of(hit - base) * inv - w;
      __syncthreads();      // out may be x: its target has been read by all
      for (int j = threadIdx.x; j < a.V; j += TOK_THREADS) {
        const float p = exp_of(to_f32(x[j]) - base) * inv;
        d[j] = from_f32<O>(empty ? 0.0f : j == t ? at_t : p);
      }
    }
  }
}

// lse comes rounded to f32: half a step of it is an error relative in p. Beyond this (2^-17 there) the row's maximum and sum are taken again;
// a row that is masked by the type's lowest value would have no sum at all beside it.
constexpr float LSE_EXACT = 128.0f;

template <typename T, typename O>
__global__ void __launch_bounds__(TOK_THREADS) tokens_grad_kernel(const OnoTokensGrad a) {
  __shared__ float s_red[TOK_THREADS / 32];
  const float ninf = __int_as_float(0xff800000);
  for (long long r = blockIdx.x; r < a.R; r += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + r * a.ld;
    O* d = reinterpret_cast<O*>(a.out) + r * a.ld_out;
    const int t = a.targets ? row_target(a.targets, a.targets64, r, a.V, a.ignore_id, a.status) : 0;
    const float lse = a.lse[r];
    if (t < 0 || lse == ninf) {
      for (int j = threadIdx.x; j < a.V; j += TOK_THREADS) d[j] = from_f32<O>(0.0f);
      continue;
    }
    const float g = a.d_logp ? a.d_logp[r] : 0.0f, h = a.d_entropy ? a.d_entropy[r] : 0.0f, H = a.d_entropy ? a.entropy[r] : 0.0f;
    float m = 0.0f, log_z = lse;
    if (fabsf(lse) > LSE_EXACT) {
      m = ninf;
      for (int j = threadIdx.x; j < a.V; j += TOK_THREADS) m = fmaxf(m, to_f32(x[j]));
      m = block_all(m, s_red, [](float p, float q) { return fmaxf(p, q); });
      float z = 0.0f;
      for (int j = threadIdx.x; j < a.V; j += TOK_THREADS) z += exp_of(to_f32(x[j]) - m);
      log_z = logf(block_all(z, s_red, [](float p, float q) { return p + q; }));
      __syncthreads();      // out may be x
    }
    for (int j = threadIdx.x; j < a.V; j += TOK_THREADS) {
      const float lp = (to_f32(x[j]) - m) - log_z, p = exp_of(lp);
      float v = -p * (g + h * (fmaxf(lp, -1e4f) + H));
      if (j == t) v += g;
      d[j] = from_f32<O>(v);
    }
  }
}
}  // namespace ono

using namespace ono;

extern "C" int ono_tokens(const OnoTokens* t, ono_stream_t stream) {
  if (!t || t->R < 0 || t->V <= 0 || t->ld < t->V || (t->R && !t->x) || t->top < 0 || t->top > ONO_TOP_MAX || t->top > t->V ||
      (t->top > 0 && t->R && (!t->top_logp || !t->top_id)) || (t->out && t->ld_out < t->V) || (!t->targets && (t->logp || t->out))) {
    set_error("bad tokens args%s", "", 0, 0);
    return -1;
  }
  if (t->out == t->x && t->out && (t->out_bf16 != t->x_bf16 || t->ld_out != t->ld)) { set_error("tokens: out over x needs the same type and rows%s", "", 0, 0); return -1; }
  if (t->R == 0) return 0;
  const unsigned grid = (unsigned)std::min<long long>(t->R, 8ll * ono_num_sms());
  cudaStream_t st = (cudaStream_t)stream;
  using B = __nv_bfloat16;
  if (t->x_bf16) {
    if (t->out_bf16) tokens_kernel<B, B><<<grid, TOK_THREADS, 0, st>>>(*t);
    else tokens_kernel<B, float><<<grid, TOK_THREADS, 0, st>>>(*t);
  } else {
    if (t->out_bf16) tokens_kernel<float, B><<<grid, TOK_THREADS, 0, st>>>(*t);
    else tokens_kernel<float, float><<<grid, TOK_THREADS, 0, st>>>(*t);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) { set_error("tokens launch: %s", cudaGetErrorString(e), 0, 0); return -7; }
  return 0;
}

extern "C" int ono_tokens_grad(const OnoTokensGrad* t, ono_stream_t stream) {
  if (!t || t->R < 0 || t->V <= 0 || t->ld < t->V || t->ld_out < t->V || (t->R && (!t->x || !t->out || !t->lse)) || (!t->d_logp && !t->d_entropy) ||
      (t->d_logp && !t->targets) || (t->entropy == nullptr) != (t->d_entropy == nullptr)) {
    set_error("bad tokens_grad args%s", "", 0, 0);
    return -1;
  }
  if (t->out == t->x && (t->out_bf16 != t->x_bf16 || t->ld_out != t->ld)) { set_error("tokens_grad: out over x needs the same type and rows%s", "", 0, 0); return -1; }
  if (t->R == 0) return 0;
  const unsigned grid = (unsigned)std::min<long long>(t->R, 8ll * ono_num_sms());
  cudaStream_t st = (cudaStream_t)stream;
  using B = __nv_bfloat16;
  if (t->x_bf16) {
    if (t->out_bf16) tokens_grad_kernel<B, B><<<grid, TOK_THREADS, 0, st>>>(*t);
    else tokens_grad_kernel<B, float><<<grid, TOK_THREADS, 0, st>>>(*t);
  } else {
    if (t->out_bf16) tokens_grad_kernel<float, B><<<grid, TOK_THREADS, 0, st>>>(*t);
    else tokens_grad_kernel<float, float><<<grid, TOK_THREADS, 0, st>>>(*t);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) { set_error("tokens_grad launch: %s", cudaGetErrorString(e), 0, 0); return -7; }
  return 0;
}
