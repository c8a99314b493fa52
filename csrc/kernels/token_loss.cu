// Softmax over a vocabulary with one given token per row: its log probability, the entropy, the most likely alternatives, and the logits'
// gradient, of the token loss or of whatever is made of the log probability and the entropy.
//
//   z = sum exp(x - m), m = max x      lse = m + ln z      logp = (x_t - m) - ln z      entropy = ln z - sum exp(x - m) (x - m) / z
//   d logp / dx_v = 1[v = t] - p_v      d entropy / dx_v = -p_v (ln p_v + entropy)
//
// All of it is f32 whatever the logits' type; x - m before the multiplication by log2 e, so that logits of any size keep their distances.
//
// Bound by memory, so a row is read once: it lies in the shared memory of one warp, one CTA or a cluster of up to eight while it is gone through
// for its maximum, its sum, its alternatives and its gradient, and the next row is on its way meanwhile (asynchronous copies).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "ono_kernels.h"
#include "piece.cuh"
#include "ptx.cuh"

namespace ono {
void set_error(const char* fmt, const char* a, long long b, long long c);

// What a launch computes: log probabilities, with entropy, with entropy and alternatives, the token loss's gradient, the gradient from
// those of log probability and entropy.
enum TokMode : int { TOK_LOGP, TOK_ENTROPY, TOK_TOP, TOK_LOSS, TOK_GRAD };

struct TokDev {
  const void* x; const void* targets;
  long long R, ld, ld_out, ignore_id;
  int V, targets64, top, per, stages;      // per: 16-byte groups of a row that a CTA takes
  float *logp, *lse, *entropy, *top_logp;
  int* top_id;
  void* out;
  const float* weight;
  float scale;
  const float *lse_in, *entropy_in, *d_logp, *d_entropy;
  int* status;
};

// lse comes rounded to f32: half a step of it is an error relative in p. Beyond this (2^-17 there) the gradient takes the row's maximum and sum
// again; a row that is masked by the type's lowest value would have no sum at all beside it.
constexpr float LSE_EXACT = 128.0f;
constexpr int TOK_CTAS = 8;      // of a cluster, at most

__device__ __forceinline__ float exp_of(float d) {      // exp(d)
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.4426950408889634f));
  return r;
}
__device__ __forceinline__ void cp_async16(void* smem, const void* g) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(g) : "memory");
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
  static __device__ __forceinline__ float ninf() { return __int_as_float(0xff800000); }
};
template <> struct TokVec<__nv_bfloat16> {
  static constexpr int E = 8;
  static __device__ __forceinline__ void get(const uint4& w, float (&v)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) { v[2 * k] = __uint_as_float(u[k] << 16); v[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u); }
  }
  static __device__ __forceinline__ __nv_bfloat16 ninf() { return __ushort_as_bfloat16(0xff80); }
};

template <int GW>
__device__ __forceinline__ void group_sync() {
  if (GW == 1) __syncwarp(); else __syncthreads();
}

// GW warps to a row; a group of one warp has CAP places for candidates, a CTA more.
template <int GW> struct TokShared {
  static constexpr int CAP = GW == 1 ? 256 : 512;
  float top[GW];
  unsigned int cut[GW];
  float2 sum[GW];
  unsigned int count, tally[2];
};
struct TokPeers {      // what the CTAs of a cluster tell each other, for this row and the next
  float4 part[2][TOK_CTAS];
  unsigned long long key[2][TOK_CTAS][ONO_TOP_MAX];
};

// The group's sum of a whole number.
template <int GW>
__device__ __forceinline__ unsigned int group_count(unsigned int v, unsigned int* s_warp, int gt) {
  v = __reduce_add_sync(0xffffffffu, v);
  if (GW == 1) return v;
  __syncthreads();
  if ((gt & 31) == 0) s_warp[gt >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < GW; ++w) v += s_warp[w];
  return v;
}

// The candidates for the `top` largest logits of n groups of 16 bytes, group 0 being group v0 of the row, exactly: where so many logits are
// as large as the bound that there is no room for them (equal ones, mostly). The K-th largest value is found bit by bit, then come
// all that are above it, and of those equal to it the first ones.
template <typename T, int GW>
__device__ __noinline__ void exact_candidates(const uint4* buf, int n, int v0, int ph, int K, unsigned long long* cand, TokShared<GW>& s, int gt) {
  constexpr int E = TokVec<T>::E, GT = GW * 32, BITS = 8 * (int)sizeof(T);
  auto for_all = [&](auto f) {
    for (int v = gt; v < n; v += GT) {
      float x[E];
      TokVec<T>::get(buf[v], x);
#pragma unroll
      for (int k = 0; k < E; ++k) if (x[k] > __int_as_float(0xff800000)) f(order_of(x[k]) >> (32 - BITS), x[k], (v0 + v) * E + k - ph);
    }
  };
  unsigned int valid = 0;
  for_all([&](unsigned int, float, int) { ++valid; });
  valid = group_count<GW>(valid, s.cut, gt);
  const unsigned int want = min((unsigned int)K, valid);
  unsigned int value = 0;      // the largest with at least `want` logits not below it
  if (want) {
    for (int b = BITS - 1; b >= 0; --b) {
      const unsigned int t = value | 1u << b;
      unsigned int c = 0;
      for_all([&](unsigned int o, float, int) { c += o >= t; });
      if (group_count<GW>(c, s.cut, gt) >= want) value = t;
    }
  }
  unsigned int above = 0;
  for_all([&](unsigned int o, float, int) { above += o > value; });
  above = group_count<GW>(above, s.cut, gt);
  group_sync<GW>();
  if (gt == 0) s.count = 0;
  group_sync<GW>();
  if (want) for_all([&](unsigned int o, float x, int j) { if (o > value) cand[atomicAdd(&s.count, 1u)] = top_key(x, j); });
  unsigned int missing = want - above;      // of the equal ones, in the order of their places
  for (int at = 0; at < n && missing; at += GT) {
    const int v = at + gt;
    float x[E];
    unsigned int mine = 0;
    if (v < n) {
      TokVec<T>::get(buf[v], x);
#pragma unroll
      for (int k = 0; k < E; ++k) mine += x[k] > __int_as_float(0xff800000) && (order_of(x[k]) >> (32 - BITS)) == value;
    }
    unsigned int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned int w = __shfl_up_sync(0xffffffffu, before, o); if ((gt & 31) >= o) before += w; }
    unsigned int total = __shfl_sync(0xffffffffu, before, 31);
    before -= mine;
    if (GW > 1) {
      __syncthreads();
      if ((gt & 31) == 0) s.cut[gt >> 5] = total;
      __syncthreads();
      total = 0;
#pragma unroll
      for (int w = 0; w < GW; ++w) { if (w < (gt >> 5)) before += s.cut[w]; total += s.cut[w]; }
    }
    if (mine && before < missing) {
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (x[k] > __int_as_float(0xff800000) && (order_of(x[k]) >> (32 - BITS)) == value && before++ < missing)
          cand[atomicAdd(&s.count, 1u)] = top_key(x[k], (v0 + v) * E + k - ph);
    }
    missing -= min(missing, total);
  }
  group_sync<GW>();
}

template <typename T, typename O, int MODE, int GW, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) tok_kernel(const __grid_constant__ TokDev a) {
  constexpr int E = TokVec<T>::E, GT = GW * 32, NG = NT / GT, CAP = TokShared<GW>::CAP;
  constexpr bool TOP = MODE == TOK_TOP, ENT = MODE == TOK_ENTROPY || MODE == TOK_TOP, FWD = MODE <= TOK_TOP;
  const float ninf = __int_as_float(0xff800000);
  extern __shared__ __align__(16) unsigned char tok_smem[];
  __shared__ TokShared<GW> s_all[NG];
  __shared__ TokPeers s_peers;
  const int grp = threadIdx.x / GT, gt = threadIdx.x % GT, lane = threadIdx.x & 31, warp = gt >> 5;
  TokShared<GW>& s = s_all[grp];
  int C = 1, rank = 0;
  if (GW > 1) {
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
    rank = (int)cluster_ctarank();
  }
  uint4* const bufs = reinterpret_cast<uint4*>(tok_smem) + (size_t)grp * a.stages * a.per;
  unsigned long long* const cand = reinterpret_cast<unsigned long long*>(tok_smem + (size_t)NG * a.stages * a.per * 16) + (size_t)grp * (CAP + ONO_TOP_MAX);
  unsigned long long* const list = cand + CAP;
  const long long stride = (long long)(gridDim.x / C) * NG;
  const int K = TOP ? a.top : 1;

  auto raw_target = [&](long long r) -> long long {
    if (!a.targets) return 0;
    if (r >= a.R) return a.ignore_id;
    return a.targets64 ? __ldg(reinterpret_cast<const long long*>(a.targets) + r) : (long long)__ldg(reinterpret_cast<const int*>(a.targets) + r);
  };
  auto target = [&](long long t) -> int {      // -1: the row is not read
    if (a.targets && t == a.ignore_id) return -1;
    if (t >= 0 && t < a.V) return (int)t;
    if (a.status && gt == 0) atomicExch(a.status, ONO_ERR_BAD_ARG);
    return -1;
  };
  auto phase_of = [&](const T* x) { return (int)(((uintptr_t)x / sizeof(T)) & (E - 1)); };
  auto load = [&](long long r, uint4* buf) {
    const T* x = reinterpret_cast<const T*>(a.x) + r * a.ld;
    const int ph = phase_of(x), nv = (ph + a.V + E - 1) / E, v0 = rank * a.per, v1 = min(nv, v0 + a.per);
    for (int v = v0 + gt; v < v1; v += GT) {
      if (v * E >= ph && (v + 1) * E <= ph + a.V) {
        cp_async16(buf + (v - v0), x + (v * E - ph));
      } else {      // an end of the row: -inf beyond it
        T* o = reinterpret_cast<T*>(buf + (v - v0));
#pragma unroll
        for (int k = 0; k < E; ++k) { const int j = v * E + k - ph; o[k] = j >= 0 && j < a.V ? x[j] : TokVec<T>::ninf(); }
      }
    }
  };
  // f(value) of every logit of the CTA's share to the output, g(value, result) where the target is
  auto write = [&](long long r, const uint4* buf, int t, auto f, auto g) {
    const T* x = reinterpret_cast<const T*>(a.x) + r * a.ld;
    O* d = reinterpret_cast<O*>(a.out) + r * a.ld_out;
    const int ph = phase_of(x), nv = (ph + a.V + E - 1) / E, v0 = rank * a.per, v1 = min(nv, v0 + a.per);
    if ((((uintptr_t)d / sizeof(O) - ph) & (E - 1)) == 0) {
      const int vt = t < 0 ? -1 : (t + ph) / E;
      for (int v = v0 + gt; v < v1; v += GT) {
        float w[E];
        if (buf) {
          TokVec<T>::get(buf[v - v0], w);
          float q[E];
#pragma unroll
          for (int k = 0; k < E; ++k) q[k] = f(w[k]);
          if (v == vt) {
#pragma unroll
            for (int k = 0; k < E; ++k) if (v * E + k - ph == t) q[k] = g(w[k], q[k]);
          }
#pragma unroll
          for (int k = 0; k < E; ++k) w[k] = q[k];
        } else {
#pragma unroll
          for (int k = 0; k < E; ++k) w[k] = 0.0f;
        }
        O* o = d + (v * E - ph);
        if (v * E >= ph && (v + 1) * E <= ph + a.V) {
          if constexpr (sizeof(O) == 4) {
#pragma unroll
            for (int k = 0; k < E; k += 4) *reinterpret_cast<float4*>(o + k) = make_float4(w[k], w[k + 1], w[k + 2], w[k + 3]);
          } else {
            uint32_t u[E / 2];
#pragma unroll
            for (int k = 0; k < E / 2; ++k) {
              const __nv_bfloat162 h = __floats2bfloat162_rn(w[2 * k], w[2 * k + 1]);
              u[k] = *reinterpret_cast<const uint32_t*>(&h);
            }
            if constexpr (E == 4) *reinterpret_cast<uint2*>(o) = make_uint2(u[0], u[1]);
            else *reinterpret_cast<uint4*>(o) = make_uint4(u[0], u[1], u[E / 2 - 2], u[E / 2 - 1]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < E; ++k) { const int j = v * E + k - ph; if (j >= 0 && j < a.V) o[k] = from_f32<O>(w[k]); }
        }
      }
    } else {      // the output's rows are aligned another way: value by value
      const T* b = reinterpret_cast<const T*>(buf);
      for (int i = max(v0 * E, ph) + gt; i < min(v1 * E, ph + a.V); i += GT) {
        float q = 0.0f;
        if (buf) { const float w = to_f32(b[i - v0 * E]); q = f(w); if (i - ph == t) q = g(w, q); }
        d[i - ph] = from_f32<O>(q);
      }
    }
  };

  if (GW > 1 && C > 1) cluster_sync_all();      // every CTA of the cluster runs: its shared memory may be written to
  long long r = (long long)(blockIdx.x / C) * NG + grp;
  int t = target(raw_target(r)), t_next = target(raw_target(r + stride));
  int it = 0, live = 0;
  if (t >= 0 && r < a.R) load(r, bufs);
  asm volatile("cp.async.commit_group;" ::: "memory");
  float x_t = 0.0f, in0 = 0.0f, in1 = 0.0f, in2 = 0.0f, in3 = 0.0f;
  auto inputs = [&](long long q, int tq) {
    if (tq < 0 || q >= a.R) return;
    if ((FWD || MODE == TOK_LOSS) && gt == 0) x_t = to_f32(reinterpret_cast<const T*>(a.x)[q * a.ld + tq]);
    if (MODE == TOK_LOSS) in0 = a.weight ? __ldg(a.weight + q) : 1.0f;
    if (MODE == TOK_GRAD) {
      in0 = __ldg(a.lse_in + q);
      in1 = a.d_logp ? __ldg(a.d_logp + q) : 0.0f;
      if (a.d_entropy) { in2 = __ldg(a.d_entropy + q); in3 = __ldg(a.entropy_in + q); }
    }
  };
  inputs(r, t);
  for (; r < a.R; r += stride, ++it) {
    const long long raw_after = raw_target(r + 2 * stride);
    const uint4* buf = bufs + (a.stages == 2 ? (size_t)(it & 1) * a.per : 0);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    group_sync<GW>();
    const float my_xt = x_t, i0 = in0, i1 = in1, i2 = in2, i3 = in3;
    if (a.stages == 2) {
      if (t_next >= 0 && r + stride < a.R) load(r + stride, bufs + (size_t)((it + 1) & 1) * a.per);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    inputs(r + stride, t_next);
    if (t < 0) {
      if (rank == 0) {
        if (FWD || MODE == TOK_LOSS) {
          if (gt == 0) {
            if (a.logp) a.logp[r] = 0.0f;
            if (a.lse) a.lse[r] = 0.0f;
            if (ENT && a.entropy) a.entropy[r] = 0.0f;
          }
          if (TOP && gt < K) { a.top_logp[r * K + gt] = ninf; a.top_id[r * K + gt] = -1; }
        }
      }
      if (!FWD) write(r, nullptr, -1, [](float) { return 0.0f; }, [](float, float q) { return q; });
    } else {
      const T* x = reinterpret_cast<const T*>(a.x) + r * a.ld;
      const int ph = phase_of(x), v0 = rank * a.per, n = min((ph + a.V + E - 1) / E - v0, a.per);
      float m = 0.0f, z = 1.0f, u = 0.0f, log_z = 0.0f;
      const bool sums = MODE != TOK_GRAD || fabsf(i0) > LSE_EXACT;
      if (sums) {
        // the maximum; for the alternatives a bound that at least K logits reach
        float tm = ninf;
        if constexpr (E == 8) {
          __nv_bfloat162 m2 = __halves2bfloat162(TokVec<T>::ninf(), TokVec<T>::ninf());
          for (int v = gt; v < n; v += GT) {
            const uint4 w = buf[v];
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
            m2 = __hmax2(m2, __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
          }
          tm = fmaxf(__low2float(m2), __high2float(m2));
        } else {
          for (int v = gt; v < n; v += GT) {
            float w[E];
            TokVec<T>::get(buf[v], w);
#pragma unroll
            for (int k = 0; k < E; ++k) tm = fmaxf(tm, w[k]);
          }
        }
        const unsigned int mine = order_of(tm);
        unsigned int wm = __reduce_max_sync(0xffffffffu, mine), cut = wm;
        if (TOP) {
          // every warp's J-th largest of its lanes' maxima; the smallest of these: GW * J >= K logits are not below it
          unsigned int rest = mine;
          for (int q = 1; q < (K + GW - 1) / GW; ++q) {
            const unsigned int who = __ballot_sync(0xffffffffu, rest == cut);
            if (lane == __ffs(who) - 1) rest = 0;
            cut = __reduce_max_sync(0xffffffffu, rest);
          }
        }
        m = of_order(wm);
        if (GW > 1) {
          if (lane == 0) { s.top[warp] = m; s.cut[warp] = cut; }
          if (TOP && gt == 0) s.count = 0;
          if (TOP && gt < K) list[gt] = 0;
          __syncthreads();
#pragma unroll
          for (int w = 0; w < GW; ++w) { m = fmaxf(m, s.top[w]); if (TOP) cut = min(cut, s.cut[w]); }
        } else if (TOP) {
          if (gt == 0) s.count = 0;
          if (gt < K) list[gt] = 0;
          __syncwarp();
        }
        const float base = m == ninf ? 0.0f : m;      // (a row of -inf alone sums to zero, one with NaN to NaN)
        for (int careful = 0; careful < 2; ++careful) {
          z = u = 0.0f;
          for (int v = gt; v < n; v += GT) {
            float w[E];
            TokVec<T>::get(buf[v], w);
            float e[E];
#pragma unroll
            for (int k = 0; k < E; ++k) { w[k] -= base; e[k] = exp_of(w[k]); }
#pragma unroll
            for (int k = 0; k < E; ++k) z += e[k];
            if (ENT) {
#pragma unroll
              for (int k = 0; k < E; ++k) u = fmaf(e[k], careful ? fmaxf(w[k], -1e4f) : w[k], u);
            }
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) { z += __shfl_xor_sync(0xffffffffu, z, o); if (ENT) u += __shfl_xor_sync(0xffffffffu, u, o); }
          if (GW > 1) {
            if (careful) __syncthreads();
            if (lane == 0) s.sum[warp] = make_float2(z, u);
            __syncthreads();
            z = u = 0.0f;
#pragma unroll
            for (int w = 0; w < GW; ++w) { z += s.sum[w].x; u += s.sum[w].y; }
          }
          if (!ENT || u == u || z != z) break;      // zero times -inf among the terms: once more, with zero times a number
        }
        if (TOP) {
          const float bound = of_order(cut);
          if (tm >= bound && tm > ninf) {
            for (int v = gt; v < n; v += GT) {
              float w[E];
              TokVec<T>::get(buf[v], w);
#pragma unroll
              for (int k = 0; k < E; ++k)
                if (w[k] >= bound && w[k] > ninf) {
                  const unsigned int at = atomicAdd(&s.count, 1u);
                  if (at < CAP) cand[at] = top_key(w[k], (v0 + v) * E + k - ph);
                }
            }
          }
          group_sync<GW>();
          int have = (int)s.count;
          if (have > CAP) {
            group_sync<GW>();
            exact_candidates<T, GW>(buf, n, v0, ph, K, cand, s, gt);
            have = (int)s.count;
          }
          for (int i = gt; i < have; i += GT) {
            const unsigned long long key = cand[i];
            int above = 0;
            for (int q = 0; q < have; ++q) above += cand[q] > key;
            if (above < K) list[above] = key;
          }
          group_sync<GW>();
        }
        const int lead = GW > 1 ? live % C : 0;
        if (GW > 1 && C > 1) {
          const int par = live & 1;
          if (gt < C) st_cluster_v4(mapa_shared(smem_u32(&s_peers.part[par][rank]), (uint32_t)gt), make_float4(m, z, u, 0.0f));
          if (TOP && gt < K)
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&s_peers.key[par][rank][gt]), (uint32_t)lead)), "l"(list[gt]) : "memory");
          cluster_sync_all();
          m = ninf;
          for (int q = 0; q < C; ++q) m = fmaxf(m, s_peers.part[par][q].x);
          z = u = 0.0f;
          for (int q = 0; q < C; ++q) {
            const float4 w = s_peers.part[par][q];
            if (w.y == 0.0f) continue;
            const float f = exp_of(w.x - m);
            z = fmaf(w.y, f, z);
            u += f * (w.z + fmaxf(w.x - m, -1e4f) * w.y);      // (zero times a number, far below)
          }
        }
        const bool empty = z == 0.0f;
        log_z = empty ? 0.0f : logf(z);
        if ((FWD || MODE == TOK_LOSS) && gt == 0 && rank == 0) {
          if (a.lse) a.lse[r] = empty ? ninf : m + log_z;
          if (a.logp) a.logp[r] = empty ? ninf : (my_xt - m) - log_z;
          if (ENT && a.entropy) a.entropy[r] = empty ? 0.0f : log_z - u / z;
        }
        if (TOP && rank == lead) {
          float* tl = a.top_logp + r * K;
          int* ti = a.top_id + r * K;
          auto put = [&](int k, unsigned long long key) {
            tl[k] = key ? (of_order((unsigned int)(key >> 32)) - m) - log_z : ninf;
            ti[k] = key ? (int)(0xffffffffu - (unsigned int)key) : -1;
          };
          if (GW == 1 || C == 1) {
            if (gt < K) put(gt, list[gt]);
          } else {
            const unsigned long long(*keys)[ONO_TOP_MAX] = s_peers.key[live & 1];
            int there = 0;
            for (int i = gt; i < C * K; i += GT) {
              const unsigned long long key = keys[i / K][i % K];
              int above = 0;
              for (int q = 0; q < C; ++q)
                for (int k = 0; k < K; ++k) above += keys[q][k] > key;
              if (key && above < K) put(above, key);
            }
            if (gt < K) {
              for (int q = 0; q < C; ++q) for (int k = 0; k < K; ++k) there += keys[q][k] != 0;
              if (gt >= there) put(gt, 0);
            }
          }
        }
        ++live;
      }
      if (MODE == TOK_LOSS) {
        const bool empty = z == 0.0f;
        const float base = empty ? 0.0f : m, w = a.scale * i0, f = empty ? 0.0f : w / z;
        write(r, empty ? nullptr : buf, t, [&](float v) { return exp_of(v - base) * f; }, [&](float, float q) { return q - w; });
      }
      if (MODE == TOK_GRAD) {
        if (!sums) log_z = i0;
        if (!sums) m = 0.0f;
        const bool empty = i0 == ninf;
        if (a.d_entropy)
          write(r, empty ? nullptr : buf, t,
                [&](float v) { const float lp = (v - m) - log_z; return -exp_of(lp) * (i1 + i2 * (fmaxf(lp, -1e4f) + i3)); }, [&](float, float q) { return q + i1; });
        else
          write(r, empty ? nullptr : buf, t, [&](float v) { return -exp_of((v - m) - log_z) * i1; }, [&](float, float q) { return q + i1; });
      }
    }
    if (a.stages == 1) {
      group_sync<GW>();      // the row has been read by all
      if (t_next >= 0 && r + stride < a.R) load(r + stride, bufs);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    t = t_next;
    t_next = target(raw_after);
  }
}

// How a launch is laid out.
struct TokShape { int warps, ctas, per, stages; size_t smem; };

constexpr int TOK_WARP_ROW = 4096, TOK_SMALL_ROW = 16384, TOK_SLICE = 32768, TOK_SMEM = 225 * 1024;

static TokShape tok_shape(long long rows, int V, int esz, bool top) {
  const int E = 16 / esz;
  const long long groups = ((long long)V + 2 * E - 2) / E, bytes = groups * 16;      // of a row that begins anywhere
  TokShape s = {};
  auto smem = [&](int warps, int groups_in_cta) {
    const size_t cand = top ? (size_t)(8 * ((warps == 1 ? 256 : 512) + ONO_TOP_MAX)) * groups_in_cta : 0;
    return (size_t)s.per * 16 * s.stages * groups_in_cta + cand;
  };
  s.ctas = 1;
  s.stages = 2;
  if (bytes <= TOK_WARP_ROW) {
    s.warps = 1;
    s.per = (int)groups;
    s.smem = smem(1, 4);
    return s;
  }
  s.warps = bytes <= TOK_SMALL_ROW ? 4 : 8;
  while (s.ctas < TOK_CTAS && (bytes > (long long)TOK_SLICE * s.ctas || (rows * s.ctas * 2 <= ono_num_sms() && bytes > 4096ll * s.ctas))) s.ctas *= 2;
  if (s.ctas > 1) s.warps = 8;
  s.per = (int)((groups + s.ctas - 1) / s.ctas);
  if (s.per * 16 > TOK_SLICE) s.stages = 1;
  s.smem = smem(s.warps, 1);
  return s;
}

template <typename T, typename O, int MODE, int GW, int NT>
static cudaError_t tok_go(const TokDev& d, const TokShape& s, cudaStream_t st) {
  auto kern = tok_kernel<T, O, MODE, GW, NT>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)s.smem);
  if (e != cudaSuccess) return e;
  const long long units = (d.R + NT / (GW * 32) - 1) / (NT / (GW * 32));      // of a CTA, or a cluster
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)s.ctas);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = s.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)s.ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // As many clusters as are resident at once (asked for once for each size of them and of their shared memory).
  static std::atomic<unsigned long long> known[4];
  std::atomic<unsigned long long>& k = known[s.ctas == 8 ? 3 : s.ctas >> 1];
  unsigned long long v = k.load();
  if ((v >> 16) != s.smem) {
    int resident = 0;
    if ((e = cudaOccupancyMaxActiveClusters(&resident, kern, &cfg)) != cudaSuccess) return e;
    v = (unsigned long long)s.smem << 16 | (unsigned)std::max(1, std::min(resident, 65535));
    k.store(v);
  }
  cfg.gridDim = dim3((unsigned)(std::min<long long>(units, (long long)(v & 65535)) * s.ctas));
  return cudaLaunchKernelEx(&cfg, kern, d);
}

template <typename T, typename O, int MODE>
static int tok_run(TokDev& d, cudaStream_t st) {
  const TokShape s = tok_shape(d.R, d.V, sizeof(T), MODE == TOK_TOP);
  if (s.smem > (size_t)TOK_SMEM) { set_error("tokens: a row of %s%lld logits is more than a cluster's shared memory holds", "", d.V, 0); return -1; }
  d.per = s.per;
  d.stages = s.stages;
  const cudaError_t e = s.warps == 1 ? tok_go<T, O, MODE, 1, 128>(d, s, st) : s.warps == 4 ? tok_go<T, O, MODE, 4, 128>(d, s, st) : tok_go<T, O, MODE, 8, 256>(d, s, st);
  if (e != cudaSuccess) { set_error("tokens launch: %s", cudaGetErrorString(e), 0, 0); return -7; }
  return 0;
}
}  // namespace ono

using namespace ono;

extern "C" int ono_tokens(const OnoTokens* t, ono_stream_t stream) {
  if (!t || t->R < 0 || t->V <= 0 || t->ld < t->V || (t->R && !t->x) || t->top < 0 || t->top > ONO_TOP_MAX || t->top > t->V ||
      (t->top > 0 && t->R && (!t->top_logp || !t->top_id)) || (t->out && (t->ld_out < t->V || t->entropy || t->top)) || (!t->targets && (t->logp || t->out))) {
    set_error("bad tokens args%s", "", 0, 0);
    return -1;
  }
  if (t->out == t->x && t->out && (t->out_bf16 != t->x_bf16 || t->ld_out != t->ld)) { set_error("tokens: out over x needs the same type and rows%s", "", 0, 0); return -1; }
  if (t->R == 0) return 0;
  TokDev d = {};
  d.x = t->x; d.targets = t->targets; d.R = t->R; d.ld = t->ld; d.ld_out = t->ld_out; d.ignore_id = t->ignore_id;
  d.V = t->V; d.targets64 = t->targets64; d.top = t->top; d.logp = t->logp; d.lse = t->lse; d.entropy = t->entropy;
  d.top_logp = t->top_logp; d.top_id = t->top_id; d.out = t->out; d.weight = t->weight; d.scale = t->scale; d.status = t->status;
  cudaStream_t st = (cudaStream_t)stream;
  using B = __nv_bfloat16;
  if (t->out) {
    if (t->x_bf16) return t->out_bf16 ? tok_run<B, B, TOK_LOSS>(d, st) : tok_run<B, float, TOK_LOSS>(d, st);
    return t->out_bf16 ? tok_run<float, B, TOK_LOSS>(d, st) : tok_run<float, float, TOK_LOSS>(d, st);
  }
  if (t->x_bf16) return t->top ? tok_run<B, float, TOK_TOP>(d, st) : t->entropy ? tok_run<B, float, TOK_ENTROPY>(d, st) : tok_run<B, float, TOK_LOGP>(d, st);
  return t->top ? tok_run<float, float, TOK_TOP>(d, st) : t->entropy ? tok_run<float, float, TOK_ENTROPY>(d, st) : tok_run<float, float, TOK_LOGP>(d, st);
}

extern "C" int ono_tokens_grad(const OnoTokensGrad* t, ono_stream_t stream) {
  if (!t || t->R < 0 || t->V <= 0 || t->ld < t->V || t->ld_out < t->V || (t->R && (!t->x || !t->out || !t->lse)) || (!t->d_logp && !t->d_entropy) ||
      (t->d_logp && !t->targets) || (t->entropy == nullptr) != (t->d_entropy == nullptr)) {
    set_error("bad tokens_grad args%s", "", 0, 0);
    return -1;
  }
  if (t->out == t->x && (t->out_bf16 != t->x_bf16 || t->ld_out != t->ld)) { set_error("tokens_grad: out over x needs the same type and rows%s", "", 0, 0); return -1; }
  if (t->R == 0) return 0;
  TokDev d = {};
  d.x = t->x; d.targets = t->targets; d.R = t->R; d.ld = t->ld; d.ld_out = t->ld_out; d.ignore_id = t->ignore_id;
  d.V = t->V; d.targets64 = t->targets64; d.out = t->out; d.status = t->status;
  d.lse_in = t->lse; d.entropy_in = t->entropy; d.d_logp = t->d_logp; d.d_entropy = t->d_entropy;
  cudaStream_t st = (cudaStream_t)stream;
  using B = __nv_bfloat16;
  if (t->x_bf16) return t->out_bf16 ? tok_run<B, B, TOK_GRAD>(d, st) : tok_run<B, float, TOK_GRAD>(d, st);
  return t->out_bf16 ? tok_run<float, B, TOK_GRAD>(d, st) : tok_run<float, float, TOK_GRAD>(d, st);
}
