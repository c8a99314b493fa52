// What the kernels of token_loss.cu and token_short.cu share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ono_kernels.h"
#include "piece.cuh"
#include "ptx.cuh"

namespace ono {
void set_error(const char* fmt, const char* a, long long b, long long c);

// What a launch computes: log probabilities, with entropy, with entropy and alternatives, the token loss's gradient, the gradient from
// those of log probability and entropy (of short rows, with lse_low too).
enum TokMode : int { TOK_LOGP, TOK_ENTROPY, TOK_TOP, TOK_LOSS, TOK_GRAD, TOK_GRAD_LOW };

struct TokDev {
  const void* x; const void* targets;
  long long R, ld, ld_out, ignore_id;
  int V, targets64, top, per, staged;      // per: 16-byte groups of a row that a CTA takes; staged: they are kept in shared memory
  float *logp, *lse, *lse_low, *entropy, *top_logp;
  int* top_id;
  void* out;
  const float* weight;
  float scale;
  const float *lse_in, *lse_low_in, *entropy_in, *d_logp, *d_entropy;
  int* status;
};

// lse comes rounded to f32: half a step of it is an error relative in p (2^-21 from 8 on), which lse_low takes away where it is given. Beyond this (2^-17 there)
// the gradient takes the row's maximum and sum again; a row that is masked by the type's lowest value would have no sum at all beside it.
constexpr float LSE_EXACT = 128.0f;
constexpr int TOK_CTAS = 8;      // of a cluster, at most

// 2^t
__device__ __forceinline__ float exp2_of(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
__device__ __forceinline__ float exp_of(float d) { return exp2_of(d * LOG2E); }
// Two values an instruction.
__device__ __forceinline__ float2 fma_2(float2 a, float2 b, float2 c) {
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 z, x, y, z;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(a.x), "=f"(a.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return a;
}
__device__ __forceinline__ float2 mul_2(float2 a, float2 b) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(a.x), "=f"(a.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return a;
}
__device__ __forceinline__ float2 add_2(float2 a, float2 b) {
  add_f32x2(a.x, a.y, b.x, b.y);
  return a;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// A maximum beyond this in size, times log2 e, is rounded by more than a few hundredths (and may leave f32): such a row is gone through again.
constexpr float TOK_FAR = 1e6f;
// What exponents are taken relative to, in units of log2: the maximum's, of any size, rounded; a logit is then one multiply-add, and its error
// that of the difference. Zero where there is nothing but far negative ones (all exponentials are zero then).
__device__ __forceinline__ float shift_of(float m) { return m < -TOK_FAR ? 0.0f : m * LOG2E; }

// What rounding took off `lse`, of a sum z relative to the shift `at`: to the bits of z, so in 64. With it p = 2^(x log2 e - at) / z, as if neither had been
// joined to the other; log2 e is the one that the exponents are made with. Out of line: few calls ask for it.
static __device__ __noinline__ float low_of(float at, float z, float lse) { return (float)(((double)at + log2((double)z)) / (double)LOG2E - (double)lse); }

__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// Larger for a larger float. (-0 counts as 0.)
__device__ __forceinline__ unsigned int order_of(float v) {
  const unsigned int u = __float_as_uint(v + 0.0f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_order(unsigned int o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }
// ... and among equal logits for the lower index.
__device__ __forceinline__ unsigned long long top_key(float v, int j) { return ((unsigned long long)order_of(v) << 32) | (0xffffffffu - (unsigned int)j); }

template <typename T> struct TokVec;
template <> struct TokVec<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ void get(const uint4& w, float (&v)[4]) {
    v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
  }
  static constexpr uint32_t NINF = 0xff800000u;      // a word of logits that are -inf
  static __device__ __forceinline__ float most(const uint4& w) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  static __device__ __forceinline__ float most(const uint4 (&w)[4]) {
    float m = __int_as_float(0xff800000);
#pragma unroll
    for (int k = 0; k < 4; ++k) m = fmaxf(m, most(w[k]));
    return m;
  }
};
template <> struct TokVec<__nv_bfloat16> {
  static constexpr int E = 8;
  static __device__ __forceinline__ void get(const uint4& w, float (&v)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) { v[2 * k] = __uint_as_float(u[k] << 16); v[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u); }
  }
  static constexpr uint32_t NINF = 0xff80ff80u;
  static __device__ __forceinline__ __nv_bfloat162 most2(const uint4& w) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
    return __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  }
  static __device__ __forceinline__ float most(const uint4& w) {
    const __nv_bfloat162 m = most2(w);
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ float most(const uint4 (&w)[4]) {
    const __nv_bfloat162 m = __hmax2(__hmax2(most2(w[0]), most2(w[1])), __hmax2(most2(w[2]), most2(w[3])));
    return fmaxf(__low2float(m), __high2float(m));
  }
};

// E results to a group of the output, from o on. The gradient is as large as the logits and is read after all of it is written, so the stores are marked for
// early eviction: 16384 rows of 1000 f32 logits take 20.4 us against 23.1, 4096 of 128256 bf16 519 against 533, of 50257 164.6 against 163.4.
template <typename O, int E>
__device__ __forceinline__ void store_group(O* o, const float (&w)[E]) {
  if constexpr (sizeof(O) == 4) {
#pragma unroll
    for (int k = 0; k < E; k += 4) __stcs(reinterpret_cast<float4*>(o + k), make_float4(w[k], w[k + 1], w[k + 2], w[k + 3]));
  } else {
    uint32_t u[E / 2];
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(w[2 * k], w[2 * k + 1]);
      u[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    if constexpr (E == 4) __stcs(reinterpret_cast<uint2*>(o), make_uint2(u[0], u[1]));
    else __stcs(reinterpret_cast<uint4*>(o), make_uint4(u[0], u[1], u[E / 2 - 2], u[E / 2 - 1]));
  }
}

// Rows of up to TOK_SHORT_ROW bytes, TOK_TOP of up to TOK_SHORT_TOP (token_short.cu). (Us, this against the other form: entropy of 30000 x 800 f32 16.9, 21.8, its gradient in
// bf16 21.1, 23.5; loss of 8192 x 1900 bf16 13.8, 18.1; entropy of 47107 x 123 bf16 18.4, 25.6; five alternatives of 65536 x 100 f32 55, 65, of 65536 x 300 bf16 148, 77; twenty
// of 65536 x 100 f32 135, 94, for which the rule has no case of its own.)
constexpr int TOK_SHORT_ROW = 4096, TOK_SHORT_TOP = 512;
int tok_short(const TokDev& d, int mode, int x_bf16, int out_bf16, cudaStream_t st);
// 16-byte groups that a row takes wherever it begins.
inline long long tok_groups(int V, int esz) { return ((long long)V + 2 * (16 / esz) - 2) / (16 / esz); }

}  // namespace ono
