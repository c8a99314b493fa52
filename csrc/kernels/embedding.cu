// Rows of a table looked up by token, and the table's gradient from the rows' gradients.
//
//   out[i] = scale * table[ids[i]]            grad[v] (+)= scale * sum over i with ids[i] = v of d[i]
//
// Either is bound by memory: the rows read and written, and for the gradient the whole table where it is not added to. Sums go over the tokens
// in the order of their places, so that a gradient is the same to the bit from run to run: the places are sorted by token (stable), and
// one warp adds up a run of equal tokens, or an L-th of a long one.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "ono_kernels.h"
#include "piece.cuh"
#include "ptx.cuh"

namespace ono {
void set_error(const char* fmt, const char* a, long long b, long long c);

// The row an id stands for, -1 for none.
template <typename I>
__device__ __forceinline__ long long token_row(I id, int vocab, long long padding_id, int* status) {
  if ((long long)id == padding_id) return -1;
  if (id >= 0 && id < vocab) return (long long)id;
  if (status) atomicExch(status, ONO_ERR_BAD_ARG);
  return -1;
}

// ------------------------------------------------------------------------------------------------
// Lookup: a warp takes EMB_SEG groups of a row, a lane up to four of them, VEC values each.
// ------------------------------------------------------------------------------------------------
constexpr int EMB_SEG = 128;

template <typename TI, typename TO, int VEC, typename I>
__global__ void __launch_bounds__(256) embedding_kernel(const OnoEmbedding e, int groups, int segs) {
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long long i = item / segs;
  if (i >= e.n) return;
  const int lane = threadIdx.x & 31, g0 = (int)(item - i * segs) * EMB_SEG + lane;
  const long long row = token_row(reinterpret_cast<const I*>(e.ids)[i], e.vocab, e.padding_id, e.status);
  const TI* src = reinterpret_cast<const TI*>(e.table) + (row < 0 ? 0 : row) * e.ld_table;
  TO* dst = reinterpret_cast<TO*>(e.out) + i * e.ld_out;
  float v[4][VEC];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int g = g0 + 32 * u;
    if (g >= groups) continue;
    if (VEC > 1 && (g + 1) * VEC <= e.width) {
      constexpr int N = VEC * (int)sizeof(TI) / 16 > 0 ? VEC * (int)sizeof(TI) / 16 : 1;
      constexpr int EL = 16 / (int)sizeof(TI);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const uint4 w = row < 0 ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>(src + (long long)g * VEC) + k);
        const TI* t = reinterpret_cast<const TI*>(&w);
#pragma unroll
        for (int q = 0; q < EL && k * EL + q < VEC; ++q) v[u][k * EL + q] = to_f32(t[q]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[u][k] = row >= 0 && g * VEC + k < e.width ? to_f32(src[(long long)g * VEC + k]) : 0.0f;
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int g = g0 + 32 * u;
    if (g >= groups) continue;
    if (row >= 0) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[u][k] *= e.scale;
    }
    if (VEC > 1 && (g + 1) * VEC <= e.width) {
      constexpr int N = VEC * (int)sizeof(TO) / 16 > 0 ? VEC * (int)sizeof(TO) / 16 : 1;
      constexpr int EL = 16 / (int)sizeof(TO);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        uint4 w;
        TO* t = reinterpret_cast<TO*>(&w);
#pragma unroll
        for (int q = 0; q < EL; ++q) t[q] = from_f32<TO>(k * EL + q < VEC ? v[u][k * EL + q] : 0.0f);
        *(reinterpret_cast<uint4*>(dst + (long long)g * VEC) + k) = w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (g * VEC + k < e.width) dst[(long long)g * VEC + k] = from_f32<TO>(v[u][k]);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Gradient. First launch: cluster 0 sorts the places by token, the other CTAs fill the table with zeros.
// ------------------------------------------------------------------------------------------------
// A radix sort, `bits` (at most 9) of the token a pass, stable. The places are dealt to the cluster's warps in runs; a warp goes through its
// own 32 at a time, lanes of one digit finding each other by match. Counts per warp and digit are turned into positions by a sum over the
// warps, one over the CTAs (distributed shared memory) and one over the digits. Keys and places go through memory between passes
// (L2): the cluster barrier, release and acquire, orders them.
constexpr int SORT_CTAS = 8, SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32, SORT_BITS = 9, SORT_RADIX = 1 << SORT_BITS;
struct SortShared {
  unsigned int count[SORT_WARPS][SORT_RADIX];
  unsigned int total[SORT_RADIX];      // read by the other CTAs
  unsigned int base[SORT_RADIX];
  unsigned int warp_sum[SORT_WARPS];
};

constexpr int SORT_BATCH = 16;      // keys that a lane has in registers: their loads are in flight together

struct GradDev {
  OnoEmbeddingGrad e;
  unsigned int *key[2], *place[2];     // ping, pong
  unsigned int* runs;                  // number of long runs, then their first and last chunks
  float* part;                         // [chunks][2][pitch]
  int passes, bits, sorted;            // sorted: which of the two holds the result
  int chunk, pitch;
};

template <typename I>
__device__ void sort_places(const GradDev& p, SortShared& s) {
  const OnoEmbeddingGrad& e = p.e;
  const unsigned int n = (unsigned int)e.n;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = (int)cluster_ctarank();
  const unsigned int per = ((n + SORT_CTAS * SORT_WARPS - 1) / (SORT_CTAS * SORT_WARPS) + 31) / 32 * 32;
  const unsigned long long first64 = (unsigned long long)per * (unsigned)(rank * SORT_WARPS + warp);
  const unsigned int first = (unsigned int)min((unsigned long long)n, first64), last = (unsigned int)min((unsigned long long)n, first64 + per);
  const unsigned int below = (1u << lane) - 1u;
  if (n && rank == 0 && tid == 0) *p.runs = 0;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits, radix = 1 << p.bits;
    const unsigned int* kin = p.key[(pass + 1) & 1];
    const unsigned int* pin = p.place[(pass + 1) & 1];
    unsigned int* kout = p.key[pass & 1];
    unsigned int* pout = p.place[pass & 1];
    unsigned int key[SORT_BATCH];
    auto keys_from = [&](unsigned int j0) {
#pragma unroll
      for (int b = 0; b < SORT_BATCH; ++b) {
        const unsigned int j = j0 + 32 * b + lane;
        if (j >= last) continue;
        if (pass) {
          key[b] = __ldcg(kin + j);      // written by other SMs since this one may have read the place
        } else {
          const long long r = token_row(__ldg(reinterpret_cast<const I*>(e.ids) + j), e.vocab, e.padding_id, e.status);
          key[b] = r < 0 ? (unsigned int)e.vocab : (unsigned int)r;      // no token: behind all of them
        }
      }
    };
    for (int k = lane; k < radix; k += 32) s.count[warp][k] = 0;
    __syncwarp();
    for (unsigned int j0 = first; j0 < last; j0 += 32 * SORT_BATCH) {
      keys_from(j0);
#pragma unroll
      for (int b = 0; b < SORT_BATCH; ++b) {
        const unsigned int j = j0 + 32 * b + lane;
        if (j0 + 32 * b >= last) break;
        const unsigned int digit = j < last ? (key[b] >> shift) & (radix - 1) : 0xffffffffu;
        const unsigned int peers = __match_any_sync(0xffffffffu, digit);
        if (j < last && (peers & below) == 0) s.count[warp][digit] += __popc(peers);
        __syncwarp();
      }
    }
    __syncthreads();
    if (tid < radix) {
      unsigned int sum = 0;
#pragma unroll 8
      for (int w = 0; w < SORT_WARPS; ++w) { const unsigned int c = s.count[w][tid]; s.count[w][tid] = sum; sum += c; }
      s.total[tid] = sum;
    }
    cluster_sync_all();
    unsigned int before = 0, all = 0;
    if (tid < radix) {
#pragma unroll
      for (int q = 0; q < SORT_CTAS; ++q) {
        unsigned int v;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(&s.total[tid]), (uint32_t)q)) : "memory");
        if (q < rank) before += v;
        all += v;
      }
    }
    unsigned int run = all;                  // inclusive sum over the digits
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned int v = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run += v; }
    if (lane == 31) s.warp_sum[warp] = run;
    __syncthreads();
    if (tid < radix) {
      unsigned int lower = 0;
      for (int w = 0; w < warp; ++w) lower += s.warp_sum[w];
      s.base[tid] = lower + run - all + before;
    }
    __syncthreads();
    for (unsigned int j0 = first; j0 < last; j0 += 32 * SORT_BATCH) {
      unsigned int from[SORT_BATCH];
      if (last - first > 32 * SORT_BATCH) keys_from(j0);      // (else they are still here)
#pragma unroll
      for (int b = 0; b < SORT_BATCH; ++b) {
        const unsigned int j = j0 + 32 * b + lane;
        if (j < last) from[b] = pass ? __ldcg(pin + j) : j;
      }
#pragma unroll
      for (int b = 0; b < SORT_BATCH; ++b) {
        const unsigned int j = j0 + 32 * b + lane;
        if (j0 + 32 * b >= last) break;
        const unsigned int digit = j < last ? (key[b] >> shift) & (radix - 1) : 0xffffffffu;
        const unsigned int peers = __match_any_sync(0xffffffffu, digit);
        unsigned int at = 0;
        if (j < last) at = s.base[digit] + s.count[warp][digit] + __popc(peers & below);
        __syncwarp();
        if (j < last) {
          if ((peers & below) == 0) s.count[warp][digit] += __popc(peers);
          kout[at] = key[b];
          pout[at] = from[b];
        }
        __syncwarp();
      }
    }
    cluster_sync_all();
  }
}

template <typename I>
__global__ void __launch_bounds__(SORT_THREADS) embedding_sort_kernel(const __grid_constant__ GradDev p) {
  extern __shared__ __align__(16) unsigned char sort_smem[];
  if (blockIdx.x < SORT_CTAS) {
    sort_places<I>(p, *reinterpret_cast<SortShared*>(sort_smem));
    return;
  }
  const OnoEmbeddingGrad& e = p.e;
  const long long t = (long long)(blockIdx.x - SORT_CTAS) * SORT_THREADS + threadIdx.x, nt = (long long)(gridDim.x - SORT_CTAS) * SORT_THREADS;
  if (e.ld_grad == e.width && ((uintptr_t)e.grad & 15) == 0) {
    const long long all = (long long)e.vocab * e.width, n4 = all >> 2;
    float4* g = reinterpret_cast<float4*>(e.grad);
    for (long long i = t; i < n4; i += nt) g[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (long long i = 4 * n4 + t; i < all; i += nt) e.grad[i] = 0.0f;
  } else {
    for (long long v = t >> 5; v < e.vocab; v += nt >> 5)
      for (int k = threadIdx.x & 31; k < e.width; k += 32) e.grad[v * e.ld_grad + k] = 0.0f;
  }
}

// Second launch: a warp adds up the rows of a chunk of `chunk` sorted places, 32 * VEC columns of them. A run of equal tokens belongs to
// the chunk it starts in, whose warp follows it into the next chunk if it ends there. A longer run is summed chunk by chunk: part[c][1]
// has the sum of what starts in c, part[c][0] of what comes from before; the third launch adds them in order.
// Whether the run of token k that starts in the chunk before place b and reaches it is one of the long ones.
__device__ __forceinline__ bool long_run(const unsigned int* key, unsigned int n, unsigned int b, unsigned int chunk, unsigned int k) {
  return b + chunk <= n && key[b + chunk - 1] == k;
}

template <int VEC>
struct GradVec {      // what a lane has of an f32 row: 16-byte accesses where the row is aligned and the lane's columns are all there
  static __device__ __forceinline__ void load(float (&v)[VEC], const float* p, int left, bool aligned) {
    if (VEC > 1 && aligned && left >= VEC) {
#pragma unroll
      for (int k = 0; k < VEC; k += 4) { const float4 w = *reinterpret_cast<const float4*>(p + k); v[k] = w.x; v[(k + 1) % VEC] = w.y; v[(k + 2) % VEC] = w.z; v[(k + 3) % VEC] = w.w; }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = k < left ? p[k] : 0.0f;
    }
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[VEC], int left, bool aligned) {
    if (VEC > 1 && aligned && left >= VEC) {
#pragma unroll
      for (int k = 0; k < VEC; k += 4) *reinterpret_cast<float4*>(p + k) = make_float4(v[k], v[(k + 1) % VEC], v[(k + 2) % VEC], v[(k + 3) % VEC]);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) if (k < left) p[k] = v[k];
    }
  }
};

template <typename T, int VEC, bool ACC>
__global__ void __launch_bounds__(256) embedding_sum_kernel(const __grid_constant__ GradDev p, int tiles) {
  constexpr int U = ACC ? 4 : 8;      // rows in flight
  const OnoEmbeddingGrad& e = p.e;
  const unsigned int n = (unsigned int)e.n, L = (unsigned int)p.chunk, none = (unsigned int)e.vocab;
  const unsigned int* const key = p.key[p.sorted];
  const unsigned int* const place = p.place[p.sorted];
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const unsigned int c = (unsigned int)(item / tiles);
  const int tile = (int)(item - (long long)c * tiles), col = (tile * 32 + lane) * VEC, left = e.width - col;
  const bool aligned = (((uintptr_t)e.grad | (uintptr_t)(e.ld_grad * 4)) & 15) == 0;
  if ((unsigned long long)c * L >= n) return;
  const unsigned int s = c * L, own = min(n, s + L);
  unsigned int end = own;
  const unsigned int k0 = key[s], kl = key[own - 1], kb = s > 0 ? key[s - 1] : none, ke = own < n ? key[own] : none;
  if (k0 == none) return;
  const bool from_before = s > 0 && kb == k0, goes_on = own < n && ke == kl;
  unsigned int at = s;
  if (from_before) {
    const bool just_before = s == L || key[s - L] != k0 || key[s - L - 1] != k0;      // it starts in the chunk before
    if (just_before && !long_run(key, n, s, L, k0)) {                                 // whose warp finishes it
      if (kl == k0) return;
      for (bool found = false; !found; ) {
        const unsigned int j = at + lane;
        const unsigned int other = __ballot_sync(0xffffffffu, j < own && key[min(j, own - 1)] != k0);
        found = other != 0;
        at += found ? __ffs(other) - 1 : 32;
      }
    }
  }
  const bool head = from_before && at == s;      // a piece of a run that started earlier
  bool tail_long = false;
  if (goes_on && !(head && kl == k0) && kl != none) {
    tail_long = long_run(key, n, own, L, kl);
    if (!tail_long) {
      end = min(n, own + L);      // this warp finishes it; it stops at the next token
    } else if (tile == 0) {       // where it ends: the last place of token kl, 32 probes at a time
      unsigned int lo = own + L - 1, hi = n;      // key[lo] == kl, key[hi] != kl or hi == n
      while (hi - lo > 1) {
        const unsigned int step = (hi - lo + 31) / 32, j = lo + step * (lane + 1);
        const unsigned int same = __popc(__ballot_sync(0xffffffffu, j < hi && key[min(j, n - 1)] == kl));
        const unsigned int was = lo;
        lo = was + step * same;
        hi = min(hi, was + step * (same + 1));
      }
      if (lane == 0) {
        const unsigned int slot = atomicAdd(p.runs, 1u);
        p.runs[2 + 2 * slot] = c;
        p.runs[3 + 2 * slot] = lo / L;
      }
    }
  }
  float acc[VEC], old[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
  unsigned int cur = none;
  bool piece = head;
  auto flush = [&](bool tail) {
    if (cur == none || left <= 0) return;
    if (piece || (tail && tail_long)) {
      GradVec<VEC>::store(p.part + ((long long)c * 2 + (piece ? 0 : 1)) * p.pitch + col, acc, left, true);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = ACC ? old[k] + e.scale * acc[k] : e.scale * acc[k];
      GradVec<VEC>::store(e.grad + (long long)cur * e.ld_grad + col, acc, left, aligned);
    }
  };
  for (unsigned int j0 = at; j0 < end; j0 += 32) {
    const unsigned int j = j0 + lane;
    const unsigned int kj = j < end ? key[j] : none, pj = j < end ? place[j] : 0u;
    const int m = (int)min(32u, end - j0);
    for (int q0 = 0; q0 < m; q0 += U) {
      uint4 w[U];
      float f[U][1];
      float was[ACC ? U : 1][VEC];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int q = q0 + u;
        const unsigned int k = __shfl_sync(0xffffffffu, kj, q & 31), from = __shfl_sync(0xffffffffu, pj, q & 31);
        const unsigned int kp = __shfl_sync(0xffffffffu, kj, (q - 1) & 31);
        if (q < m && k != none && left > 0) {
          const T* row = reinterpret_cast<const T*>(e.d) + (long long)from * e.ld_d + col;
          if constexpr (VEC == 1) {
            f[u][0] = to_f32(*row);
          } else if (left >= VEC) {
            w[u] = __ldg(reinterpret_cast<const uint4*>(row));
          } else {
            T* t = reinterpret_cast<T*>(&w[u]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) t[i] = i < left ? row[i] : from_f32<T>(0.0f);
          }
          if (ACC && (q == 0 || kp != k)) GradVec<VEC>::load(was[ACC ? u : 0], e.grad + (long long)k * e.ld_grad + col, left, aligned);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int q = q0 + u;
        const unsigned int k = __shfl_sync(0xffffffffu, kj, q & 31);
        if (q >= m) break;
        if (k != cur) {
          flush(false);
          if (cur != none) piece = false;
          if (k == none || j0 + q >= own) return;              // (beyond the chunk only its last run goes on)
          cur = k;
#pragma unroll
          for (int i = 0; i < VEC; ++i) { acc[i] = 0.0f; if (ACC) old[i] = was[ACC ? u : 0][i]; }
        }
        if (left > 0) {
          if constexpr (VEC == 1) acc[0] += f[u][0];
          else add_piece<T, VEC>(acc, w[u]);
        }
      }
    }
  }
  flush(true);
}

// Third launch: a block takes a long run's sums, 32 * VEC columns of them; its warps every eighth, then one adds up theirs.
template <int VEC>
__global__ void __launch_bounds__(256) embedding_join_kernel(const __grid_constant__ GradDev p, int tiles) {
  __shared__ float s_sum[8][32 * VEC];
  const OnoEmbeddingGrad& e = p.e;
  const unsigned int L = (unsigned int)p.chunk, runs = *p.runs;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool aligned = (((uintptr_t)e.grad | (uintptr_t)(e.ld_grad * 4)) & 15) == 0;
  for (unsigned long long item = blockIdx.x; item < (unsigned long long)runs * tiles; item += gridDim.x) {
    const unsigned int run = (unsigned int)(item / tiles), c = p.runs[2 + 2 * run], c1 = p.runs[3 + 2 * run];
    const int col = ((int)(item - (unsigned long long)run * tiles) * 32 + lane) * VEC, left = e.width - col;
    float acc[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
    if (left > 0) {
#pragma unroll 4
      for (unsigned int q = c + warp; q <= c1; q += 8) {
        float v[VEC];
        GradVec<VEC>::load(v, p.part + ((long long)q * 2 + (q == c ? 1 : 0)) * p.pitch + col, left, true);
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += v[k];
      }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) s_sum[warp][lane * VEC + k] = acc[k];
    __syncthreads();
    if (warp == 0 && left > 0) {
      float* g = e.grad + (long long)p.key[p.sorted][c * L + L - 1] * e.ld_grad + col;
      float old[VEC];
      if (e.accumulate) GradVec<VEC>::load(old, g, left, aligned);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float t = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += s_sum[w][lane * VEC + k];
        acc[k] = e.accumulate ? old[k] + e.scale * t : e.scale * t;
      }
      GradVec<VEC>::store(g, acc, left, aligned);
    }
    __syncthreads();
  }
}

// Places to a chunk: as many as leave enough warps to fill the GPU (a lane has U rows in flight whatever the chunk).
static int grad_chunk(long long n, int width) {
  const long long tiles = (width + 127) / 128;
  int L = 512;
  while (L > 8 && n / L * tiles < 32ll * 148) L >>= 1;
  return L;
}

struct GradScratch { long long key, runs, part, bytes; int chunk, pitch; };
static GradScratch grad_scratch(long long n, int width) {
  GradScratch g;
  g.chunk = grad_chunk(n, width);
  g.pitch = (width + 3) / 4 * 4;
  const long long chunks = (n + g.chunk - 1) / g.chunk;
  g.key = (n * 4 + 15) / 16 * 16;
  g.runs = 4 * g.key;
  g.part = g.runs + ((2 + 2 * chunks) * 4 + 15) / 16 * 16;
  g.bytes = g.part + chunks * 2 * g.pitch * 4;
  return g;
}

template <typename TI, typename TO, typename I>
static cudaError_t embedding_go(const OnoEmbedding& e, bool vec, cudaStream_t st) {
  constexpr int VEC = sizeof(TI) == 4 && sizeof(TO) == 4 ? 4 : 8;
  const int groups = vec ? (e.width + VEC - 1) / VEC : e.width, segs = (groups + EMB_SEG - 1) / EMB_SEG;
  const long long blocks = (e.n * segs + 7) / 8;
  if (vec) embedding_kernel<TI, TO, VEC, I><<<(unsigned)blocks, 256, 0, st>>>(e, groups, segs);
  else embedding_kernel<TI, TO, 1, I><<<(unsigned)blocks, 256, 0, st>>>(e, groups, segs);
  return cudaGetLastError();
}
}  // namespace ono

using namespace ono;

extern "C" int ono_embedding(const OnoEmbedding* e, ono_stream_t stream) {
  if (!e || e->n < 0 || e->vocab <= 0 || e->width <= 0 || e->ld_table < e->width || e->ld_out < e->width || (e->n && (!e->table || !e->ids || !e->out))) {
    set_error("bad embedding args%s", "", 0, 0);
    return -1;
  }
  if (e->n * ((e->width + EMB_SEG - 1) / EMB_SEG) >= (8ll << 31)) { set_error("embedding: too many values%s", "", 0, 0); return -1; }
  if (e->n == 0) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  const int ti = e->table_bf16 ? 2 : 4, to = e->out_bf16 ? 2 : 4;
  const bool vec = (((uintptr_t)e->table | (uintptr_t)e->out) & 15) == 0 && e->ld_table * ti % 16 == 0 && e->ld_out * to % 16 == 0;
  using B = __nv_bfloat16;
  cudaError_t r;
  if (e->ids64)
    r = e->table_bf16 ? (e->out_bf16 ? embedding_go<B, B, long long>(*e, vec, st) : embedding_go<B, float, long long>(*e, vec, st))
                      : (e->out_bf16 ? embedding_go<float, B, long long>(*e, vec, st) : embedding_go<float, float, long long>(*e, vec, st));
  else
    r = e->table_bf16 ? (e->out_bf16 ? embedding_go<B, B, int>(*e, vec, st) : embedding_go<B, float, int>(*e, vec, st))
                      : (e->out_bf16 ? embedding_go<float, B, int>(*e, vec, st) : embedding_go<float, float, int>(*e, vec, st));
  if (r != cudaSuccess) { set_error("embedding launch: %s", cudaGetErrorString(r), 0, 0); return -7; }
  return 0;
}

extern "C" long long ono_embedding_grad_scratch(long long n, int vocab, int width) {
  return n < 0 || vocab <= 0 || width <= 0 ? -1 : grad_scratch(n, width).bytes;
}

extern "C" int ono_embedding_grad(const OnoEmbeddingGrad* e, ono_stream_t stream) {
  if (!e || e->n < 0 || e->n > (1ll << 31) - 65536 || e->vocab <= 0 || e->width <= 0 || e->ld_d < e->width || e->ld_grad < e->width || !e->grad ||
      (e->n && (!e->d || !e->ids || !e->scratch))) {
    set_error("bad embedding_grad args%s", "", 0, 0);
    return -1;
  }
  const GradScratch g = grad_scratch(e->n, e->width);
  if (e->n && (e->scratch_bytes < g.bytes || ((uintptr_t)e->scratch & 15))) { set_error("embedding_grad: scratch of %s%lld bytes, 16-byte aligned", "", g.bytes, 0); return -1; }
  if (e->n == 0 && e->accumulate) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  GradDev p;
  p.e = *e;
  char* at = reinterpret_cast<char*>(e->scratch);
  for (int k = 0; k < 2; ++k) {
    p.key[k] = reinterpret_cast<unsigned int*>(at + k * g.key);
    p.place[k] = reinterpret_cast<unsigned int*>(at + (2 + k) * g.key);
  }
  p.runs = reinterpret_cast<unsigned int*>(at + g.runs);
  p.part = reinterpret_cast<float*>(at + g.part);
  p.chunk = g.chunk;
  p.pitch = g.pitch;
  const int need = 32 - __builtin_clz((unsigned)e->vocab);      // tokens, and `vocab` for none
  p.passes = (need + SORT_BITS - 1) / SORT_BITS;
  p.bits = (need + p.passes - 1) / p.passes;
  p.sorted = (p.passes - 1) & 1;
  int zero = 0;
  if (!e->accumulate) {
    const long long per = 4ll * SORT_THREADS * 4;                // a few stores a thread
    zero = (int)std::min<long long>(2ll * ono_num_sms() / SORT_CTAS, ((long long)e->vocab * e->width + per * SORT_CTAS - 1) / (per * SORT_CTAS));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(SORT_CTAS * (1 + zero)));
  cfg.blockDim = dim3(SORT_THREADS);
  cfg.dynamicSmemBytes = sizeof(SortShared);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = SORT_CTAS; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto sort = [&](auto kern) -> cudaError_t {
    const cudaError_t r = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SortShared));
    return r != cudaSuccess ? r : cudaLaunchKernelEx(&cfg, kern, p);
  };
  cudaError_t r = e->ids64 ? sort(embedding_sort_kernel<long long>) : sort(embedding_sort_kernel<int>);
  if (r != cudaSuccess) { set_error("embedding_grad sort: %s", cudaGetErrorString(r), 0, 0); return -7; }
  if (e->n == 0) return 0;
  const int esz = e->d_bf16 ? 2 : 4;
  const bool vec = ((uintptr_t)e->d & 15) == 0 && e->ld_d * esz % 16 == 0;
  const int cols = 32 * (vec ? 16 / esz : 1), tiles = (e->width + cols - 1) / cols;
  const long long chunks = (e->n + g.chunk - 1) / g.chunk, blocks = (chunks * tiles + 7) / 8;
  if (blocks >= (1ll << 31)) { set_error("embedding_grad: too many values%s", "", 0, 0); return -1; }
  using B = __nv_bfloat16;
  auto sum = [&](auto kern) { kern<<<(unsigned)blocks, 256, 0, st>>>(p, tiles); };
  if (e->accumulate) {
    if (e->d_bf16) { if (vec) sum(embedding_sum_kernel<B, 8, true>); else sum(embedding_sum_kernel<B, 1, true>); }
    else { if (vec) sum(embedding_sum_kernel<float, 4, true>); else sum(embedding_sum_kernel<float, 1, true>); }
  } else {
    if (e->d_bf16) { if (vec) sum(embedding_sum_kernel<B, 8, false>); else sum(embedding_sum_kernel<B, 1, false>); }
    else { if (vec) sum(embedding_sum_kernel<float, 4, false>); else sum(embedding_sum_kernel<float, 1, false>); }
  }
  if ((r = cudaGetLastError()) != cudaSuccess) { set_error("embedding_grad sum: %s", cudaGetErrorString(r), 0, 0); return -7; }
  if (e->n > g.chunk) {      // (a long run fills a whole chunk and begins ahead of it)
    const int jt = (e->width + 127) / 128;
    const unsigned grid = (unsigned)std::min<long long>(chunks * jt, 4ll * ono_num_sms());
    embedding_join_kernel<4><<<grid, 256, 0, st>>>(p, jt);
    if ((r = cudaGetLastError()) != cudaSuccess) { set_error("embedding_grad join: %s", cudaGetErrorString(r), 0, 0); return -7; }
  }
  return 0;
}
