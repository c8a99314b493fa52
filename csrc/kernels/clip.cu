// Norm of all gradients of a step and their clipping, over any number of tensors.
//
//   norm = |scale| sqrt(sum g^2)      coef = norm <= max ? 1 : max / norm      out = coef * scale * g
//
// Bound by memory: every gradient is read for the norm and, where clipped gradients are wanted, again for the product (out of L2 as far as
// they fit), or by the optimizer, which takes the coefficient along. Few values take one launch of a cluster. A launch knows its tensors from its
// parameters, CLIP_TENSORS of them, cut into chunks of 8 * CLIP_THREADS * G values; nothing is kept between calls.
//
// Squares are summed in f32 over eight values, those sums in f64, in an order that sizes and alignment give: the same bits every time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "chain.cuh"
#include "ono_kernels.h"
#include "ptx.cuh"

namespace ono {
void set_error(const char* fmt, const char* a, long long b, long long c);

constexpr int CLIP_TENSORS = 256, CLIP_THREADS = 256, CLIP_MAX_BLOCKS = 8 * 148;
// Values from which on a chunk is twice as long, of 16-bit gradients and of others.
constexpr long long CLIP_MANY_16 = 1 << 24, CLIP_MANY = 1 << 25;

// A tensor's values are counted from the 8 values' boundary in front of the first (`phase` before it), so that groups of eight
// that begin at a multiple of eight are aligned.
template <int N>
struct ClipTensors {
  const void* g[N];
  void* out[N];
  long long n[N];
  unsigned int end[N];        // chunks up to and with this tensor's
  unsigned char phase[N], type[N];      // type: that of g, and of out times four
  int count;
};
using ClipBatch = ClipTensors<CLIP_TENSORS>;
// The tensors of `c` from `next` on that fit; false where none are left.
template <int N>
static bool clip_fill(ClipTensors<N>& b, const OnoClip* c, int& next, int chunk) {
  b.count = 0;
  unsigned int end = 0;
  for (; next < c->n_tensors && b.count < N; ++next) {
    const long long n = c->n[next];
    if (n == 0) continue;
    const int k = b.count, phase = (int)(((uintptr_t)c->g[next] / (c->types[next] & 3 ? 2 : 4)) & 7);
    const long long chunks = (n + phase + chunk - 1) / chunk;
    if (end + chunks >= (1ll << 31)) break;
    b.g[k] = c->g[next]; b.out[k] = c->out ? c->out[next] : nullptr; b.n[k] = n;
    b.phase[k] = (unsigned char)phase;
    b.type[k] = c->types[next];
    b.end[k] = end += (unsigned)chunks;
    ++b.count;
  }
  return b.count > 0;
}

__device__ __forceinline__ float clip_load(const void* p, int type, long long i) {
  if (type == 0) return reinterpret_cast<const float*>(p)[i];
  if (type == 1) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void clip_store(void* p, int type, long long i, float v) {
  if (type == 0) reinterpret_cast<float*>(p)[i] = v;
  else if (type == 1) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}
// Eight values from i on: whole groups by 16-byte loads, others one by one, zeros outside [0, n).
__device__ __forceinline__ void clip_load8(const void* p, int type, long long i, long long n, float (&v)[8]) {
  if (i >= 0 && i + 8 <= n) {
    if (type == 0) {
      const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
      const float4 a = q[0], b = q[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = type == 1 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[k])) : __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
        v[2 * k] = f.x; v[2 * k + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = i + k >= 0 && i + k < n ? clip_load(p, type, i + k) : 0.0f;
  }
}
// The same in two steps, for many groups: a whole one is kept as it came until all of a thread's are under way, since a conversion under a condition waits.
// (Two groups a thread took a tenth longer by these, so the kernels have both ways.)
struct ClipGroup { uint4 w[2]; };
__device__ __forceinline__ bool clip_whole(long long i, long long n) { return i >= 0 && i + 8 <= n; }
__device__ __forceinline__ void clip_fetch8(const void* p, int type, long long i, long long n, ClipGroup& g) {
  if (!clip_whole(i, n)) return;
  if (type == 0) {
    const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + i);
    g.w[0] = q[0];
    g.w[1] = q[1];
  } else {
    g.w[0] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
  }
}
__device__ __forceinline__ void clip_values8(const void* p, int type, long long i, long long n, const ClipGroup& g, float (&v)[8]) {
  if (!clip_whole(i, n)) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = i + k >= 0 && i + k < n ? clip_load(p, type, i + k) : 0.0f;
  } else if (type == 0) {
    const uint32_t u[8] = {g.w[0].x, g.w[0].y, g.w[0].z, g.w[0].w, g.w[1].x, g.w[1].y, g.w[1].z, g.w[1].w};
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(u[k]);
  } else {
    const uint32_t u[4] = {g.w[0].x, g.w[0].y, g.w[0].z, g.w[0].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = type == 1 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[k])) : __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
      v[2 * k] = f.x; v[2 * k + 1] = f.y;
    }
  }
}
__device__ __forceinline__ void clip_store8(void* p, int type, long long i, long long n, bool aligned, const float (&v)[8]) {
  if (aligned && i >= 0 && i + 8 <= n) {
    if (type == 0) {
      float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
      q[0] = make_float4(v[0], v[1], v[2], v[3]);
      q[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (type == 1) { const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]); u[k] = *reinterpret_cast<const uint32_t*>(&h); }
        else { const __half2 h = __floats2half2_rn(v[2 * k], v[2 * k + 1]); u[k] = *reinterpret_cast<const uint32_t*>(&h); }
      }
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i) = make_uint4(u[0], u[1], u[2], u[3]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) if (i + k >= 0 && i + k < n) clip_store(p, type, i + k, v[k]);
  }
}

// The tensor that chunk c belongs to.
template <int N>
__device__ __forceinline__ int clip_find(const ClipTensors<N>& b, unsigned int c) {
  int lo = 0, hi = b.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (b.end[mid] > c) hi = mid; else lo = mid + 1;
  }
  return lo;
}

// The sum of eight squares. In f32 unless one of them is out of its range (above 2^62 in size, or below 2^-48 all of them). Zeros take the other way as well: the
// norm of 96 M f32 59.2 us, of as many zeros 60.1, of bf16 39.1 and 47.9.
__device__ __forceinline__ double squares8(const float (&v)[8]) {
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) s = fmaf(v[k], v[k], s);
  if (s > 2e37f || s < 1e-28f) {
    double t = 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += (double)v[k] * (double)v[k];
    return t;
  }
  return (double)s;
}

__device__ __forceinline__ double block_sum(double v, double* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < CLIP_THREADS / 32; ++w) v += s[w];
  return v;
}

// part[block] (+)= the squares of the block's chunks.
template <int G>
__global__ void __launch_bounds__(CLIP_THREADS) clip_norm_kernel(const __grid_constant__ ClipBatch b, double* part, int first) {
  __shared__ double s[CLIP_THREADS / 32];
  double acc = 0.0;
  for (unsigned int c = blockIdx.x; c < b.end[b.count - 1]; c += gridDim.x) {
    const int t = clip_find(b, c);
    const long long at = (long long)(c - (t ? b.end[t - 1] : 0)) * (8 * CLIP_THREADS * G) - b.phase[t];
    if constexpr (G <= 2) {
      float v[G][8];
#pragma unroll
      for (int k = 0; k < G; ++k) clip_load8(b.g[t], b.type[t] & 3, at + 8 * (k * CLIP_THREADS + (int)threadIdx.x), b.n[t], v[k]);
#pragma unroll
      for (int k = 0; k < G; ++k) acc += squares8(v[k]);
    } else {
      ClipGroup g[G];
#pragma unroll
      for (int k = 0; k < G; ++k) clip_fetch8(b.g[t], b.type[t] & 3, at + 8 * (k * CLIP_THREADS + (int)threadIdx.x), b.n[t], g[k]);
#pragma unroll
      for (int k = 0; k < G; ++k) {
        float v[8];
        clip_values8(b.g[t], b.type[t] & 3, at + 8 * (k * CLIP_THREADS + (int)threadIdx.x), b.n[t], g[k], v);
        acc += squares8(v);
      }
    }
  }
  acc = block_sum(acc, s);
  if (threadIdx.x == 0) part[blockIdx.x] = first ? acc : part[blockIdx.x] + acc;
}

// Norm and coefficient from the blocks' sums; every block that calls it gets the same ones.
__device__ __forceinline__ double clip_coef(const double* part, int parts, float scale, float max_norm, float* norm_out, float* coef_out, double* s) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += CLIP_THREADS) sum += __ldcg(part + i);
  sum = block_sum(sum, s);
  const double norm = fabs((double)scale) * sqrt(sum), coef = norm <= (double)max_norm ? 1.0 : (double)max_norm / norm;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (norm_out) *norm_out = (float)norm;
    if (coef_out) *coef_out = (float)coef;
  }
  return coef;
}

__global__ void __launch_bounds__(CLIP_THREADS) clip_finish_kernel(const double* part, int parts, float scale, float max_norm, float* norm, float* coef) {
  __shared__ double s[CLIP_THREADS / 32];
  chain_wait();
  clip_coef(part, parts, scale, max_norm, norm, coef, s);
}

template <int G>
__global__ void __launch_bounds__(CLIP_THREADS) clip_write_kernel(const __grid_constant__ ClipBatch b, const double* part, int parts, float scale, float max_norm,
                                                                  float* norm, float* coef) {
  __shared__ double s[CLIP_THREADS / 32];
  chain_wait();
  const float f = (float)(clip_coef(part, parts, scale, max_norm, norm, coef, s) * (double)scale);
  for (unsigned int c = blockIdx.x; c < b.end[b.count - 1]; c += gridDim.x) {
    const int t = clip_find(b, c), type = b.type[t] & 3, otype = b.type[t] >> 2;
    if (f == 1.0f && b.out[t] == b.g[t]) continue;
    const long long at = (long long)(c - (t ? b.end[t - 1] : 0)) * (8 * CLIP_THREADS * G) - b.phase[t];
    const bool aligned = (((uintptr_t)b.out[t] / (otype ? 2 : 4)) & 7) == b.phase[t];
    if constexpr (G <= 2) {
      float v[G][8];
#pragma unroll
      for (int k = 0; k < G; ++k) clip_load8(b.g[t], type, at + 8 * (k * CLIP_THREADS + (int)threadIdx.x), b.n[t], v[k]);
#pragma unroll
      for (int k = 0; k < G; ++k) {
        const long long i = at + 8 * (k * CLIP_THREADS + (int)threadIdx.x);
        if (i >= b.n[t]) break;
#pragma unroll
        for (int q = 0; q < 8; ++q) v[k][q] *= f;
        clip_store8(b.out[t], otype, i, b.n[t], aligned, v[k]);
      }
    } else {
      ClipGroup g[G];
#pragma unroll
      for (int k = 0; k < G; ++k) clip_fetch8(b.g[t], type, at + 8 * (k * CLIP_THREADS + (int)threadIdx.x), b.n[t], g[k]);
#pragma unroll
      for (int k = 0; k < G; ++k) {
        const long long i = at + 8 * (k * CLIP_THREADS + (int)threadIdx.x);
        if (i >= b.n[t]) break;
        float v[8];
        clip_values8(b.g[t], type, i, b.n[t], g[k], v);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] *= f;
        clip_store8(b.out[t], otype, i, b.n[t], aligned, v);
      }
    }
  }
}

// Few values of few tensors: a cluster takes them all into its registers and adds up what its blocks have found. One launch, which is what it is for: a call
// with four tensors and outputs takes the host 15 us, with two launches 20. (On the GPU, us, against the two: 101770 f32 4.9, 4.9, 17000 f32 4.1, 5.3; the norm of 1000
// values and a step by it 4.9, 5.4. Eight blocks of 1024 threads take 6.7 for the first, what a multiprocessor reads and writes.) Where a device has no room for such a
// cluster the two launches take these too.
constexpr int SMALL_CTAS = 16, SMALL_THREADS = 512, SMALL_EACH = 2, SMALL_TENSORS = 32, SMALL_CHUNKS = SMALL_CTAS * SMALL_EACH;
using ClipSmall = ClipTensors<SMALL_TENSORS>;
__global__ void __launch_bounds__(SMALL_THREADS) clip_small_kernel(const __grid_constant__ ClipSmall b, float scale, float max_norm, float* norm_out, float* coef_out, int write) {
  __shared__ double s_warp[SMALL_THREADS / 32], s_part[SMALL_CTAS];
  const unsigned int rank = cluster_ctarank(), chunks = b.end[b.count - 1];
  cluster_arrive();      // (a block's shared memory may be written to once it runs)
  ClipGroup g[SMALL_EACH];
  int of[SMALL_EACH];      // its tensor, -1 for none
  long long at[SMALL_EACH];
#pragma unroll
  for (int k = 0; k < SMALL_EACH; ++k) {
    const unsigned int c = rank + k * SMALL_CTAS;
    of[k] = -1;
    if (c >= chunks) continue;
    const int t = clip_find(b, c);
    of[k] = t;
    at[k] = (long long)(c - (t ? b.end[t - 1] : 0)) * (8 * SMALL_THREADS) - b.phase[t] + 8 * (int)threadIdx.x;
    clip_fetch8(b.g[t], b.type[t] & 3, at[k], b.n[t], g[k]);
  }
  double acc = 0.0;
#pragma unroll
  for (int k = 0; k < SMALL_EACH; ++k) {
    if (of[k] < 0) break;
    float v[8];
    clip_values8(b.g[of[k]], b.type[of[k]] & 3, at[k], b.n[of[k]], g[k], v);
    acc += squares8(v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = acc;
  __syncthreads();
  cluster_wait();
  if (threadIdx.x < 32) {
    acc = threadIdx.x < SMALL_THREADS / 32 ? s_warp[threadIdx.x] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (threadIdx.x < SMALL_CTAS)
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&s_part[rank]), threadIdx.x)), "d"(acc) : "memory");
    __syncwarp();
  }
  cluster_sync_all();
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < SMALL_CTAS; ++k) sum += s_part[k];
  const double norm = fabs((double)scale) * sqrt(sum), coef = norm <= (double)max_norm ? 1.0 : (double)max_norm / norm;
  if (rank == 0 && threadIdx.x == 0) {
    if (norm_out) *norm_out = (float)norm;
    if (coef_out) *coef_out = (float)coef;
  }
  if (!write) return;
  const float f = (float)(coef * (double)scale);
#pragma unroll
  for (int k = 0; k < SMALL_EACH; ++k) {
    const int t = of[k];
    if (t < 0) break;
    const int otype = b.type[t] >> 2;
    if ((f == 1.0f && b.out[t] == b.g[t]) || at[k] >= b.n[t]) continue;
    float v[8];
    clip_values8(b.g[t], b.type[t] & 3, at[k], b.n[t], g[k], v);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] *= f;
    clip_store8(b.out[t], otype, at[k], b.n[t], (((uintptr_t)b.out[t] / (otype ? 2 : 4)) & 7) == b.phase[t], v);
  }
}

static cudaLaunchConfig_t small_launch(cudaLaunchAttribute& attr, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(SMALL_CTAS);
  cfg.blockDim = dim3(SMALL_THREADS);
  cfg.stream = st;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = SMALL_CTAS; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cfg;
}
// Clusters of that size that the current device has room for, asked for once: 16 blocks are more than every device, or part of one, has to take.
static int clip_clusters() {
  constexpr int DEVICES = 64;
  static std::atomic<int> known[DEVICES];      // one more than there are
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= DEVICES) return 0;
  int k = known[device].load();
  if (k == 0) {
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = small_launch(attr, nullptr);
    int clusters = 0;
    if (cudaFuncSetAttribute(clip_small_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&clusters, clip_small_kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    known[device].store(k = clusters + 1);
  }
  return k - 1;
}

template <int G>
static cudaError_t clip_go(const OnoClip* c, cudaStream_t st) {
  constexpr int CLIP_CHUNK = 8 * CLIP_THREADS * G;
  double* part = reinterpret_cast<double*>(c->scratch);
  ClipBatch b;
  int next = 0;
  int parts = 0;
  while (clip_fill(b, c, next, CLIP_CHUNK)) {
    const int grid = (int)std::min<long long>(b.end[b.count - 1], std::min(CLIP_MAX_BLOCKS, 8 * ono_num_sms()));
    // later launches of a call add to the sums of the first ones; blocks that it had not start theirs
    if (grid > parts && parts) {
      const cudaError_t e = cudaMemsetAsync(part + parts, 0, (size_t)(grid - parts) * 8, st);
      if (e != cudaSuccess) return e;
    }
    clip_norm_kernel<G><<<grid, CLIP_THREADS, 0, st>>>(b, part, parts == 0);
    parts = std::max(parts, grid);
  }
  if (parts == 0) {      // no values
    clip_finish_kernel<<<1, CLIP_THREADS, 0, st>>>(part, 0, c->scale, c->max_norm, c->norm, c->coef);
  } else if (!c->out) {
    const cudaError_t e = launch_behind(clip_finish_kernel, 1u, CLIP_THREADS, st, (const double*)part, parts, c->scale, c->max_norm, c->norm, c->coef);
    if (e != cudaSuccess) return e;
  } else {
    next = 0;
    while (clip_fill(b, c, next, CLIP_CHUNK)) {
      const int grid = (int)std::min<long long>(b.end[b.count - 1], 8 * ono_num_sms());
      const cudaError_t e = launch_behind(clip_write_kernel<G>, (unsigned)grid, CLIP_THREADS, st, b, (const double*)part, parts, c->scale, c->max_norm, c->norm, c->coef);
      if (e != cudaSuccess) return e;
    }
  }
  return cudaGetLastError();
}
}  // namespace ono

using namespace ono;

extern "C" int ono_clip_one_launch(int n_tensors, long long values, int clusters) {
  return clusters > 0 && n_tensors <= SMALL_TENSORS && values <= SMALL_CHUNKS * 8ll * SMALL_THREADS;
}

extern "C" long long ono_clip_scratch(void) { return CLIP_MAX_BLOCKS * 8; }

extern "C" int ono_clip(const OnoClip* c, ono_stream_t stream) {
  if (!c || c->n_tensors < 0 || (c->n_tensors && (!c->g || !c->n || !c->types)) || !c->scratch || c->scratch_bytes < ono_clip_scratch() || ((uintptr_t)c->scratch & 7)) {
    set_error("bad clip args%s", "", 0, 0);
    return -1;
  }
  if (!(c->max_norm > 0.0f) || !isfinite(c->scale)) { set_error("clip: max_norm must be positive and scale finite%s", "", 0, 0); return -1; }
  long long values = 0;
  bool wide = false;
  for (int k = 0; k < c->n_tensors; ++k) {
    values += c->n[k];
    wide |= (c->types[k] & 3) == 0;
    const int type = c->types[k] & 3, otype = c->types[k] >> 2;
    if (c->n[k] < 0 || type > 2 || otype > 2 || (c->n[k] && (!c->g[k] || ((uintptr_t)c->g[k] & (type ? 1 : 3)) || (c->out && (!c->out[k] || ((uintptr_t)c->out[k] & (otype ? 1 : 3))))))) {
      set_error("bad clip tensor %s%lld", "", k, 0);
      return -1;
    }
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (ono_clip_one_launch(c->n_tensors, values, clip_clusters())) {
    ClipSmall b;
    int next = 0;
    if (clip_fill(b, c, next, 8 * SMALL_THREADS) && b.end[b.count - 1] <= SMALL_CHUNKS) {
      cudaLaunchAttribute attr;
      const cudaLaunchConfig_t cfg = small_launch(attr, st);
      if (cudaLaunchKernelEx(&cfg, clip_small_kernel, b, c->scale, c->max_norm, c->norm, c->coef, (int)(c->out != nullptr)) == cudaSuccess) return 0;
      cudaGetLastError();      // (fewer multiprocessors than were asked about: the form below runs on any)
    }
  }
  // Two groups a thread, or four. (Us, two, four: 200 k f32 values 4.2, 5.8; 8 M bf16 15.4, 17.6, 17 M 27.9, 25.3, 90 M 137, 119; 30 M f32 71, 69, 90 M 209, 185;
  // f32 to bf16 of 30 M 53, 55, of 90 M 154, 149.)
  const cudaError_t e = values < (wide ? CLIP_MANY : CLIP_MANY_16) ? clip_go<2>(c, st) : clip_go<4>(c, st);
  if (e != cudaSuccess) { set_error("clip launch: %s", cudaGetErrorString(e), 0, 0); return -7; }
  return 0;
}
