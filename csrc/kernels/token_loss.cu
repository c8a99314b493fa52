// Softmax over a vocabulary with one given token per row: its log probability, the entropy, the most likely alternatives, and the logits'
// gradient, of the token loss or of whatever is made of the log probability and the entropy.
//
//   z = sum exp(x - m), m = max x      lse = m + ln z      logp = (x_t - m) - ln z      entropy = ln z - sum exp(x - m) (x - m) / z
//   d logp / dx_v = 1[v = t] - p_v      d entropy / dx_v = -p_v (ln p_v + entropy)
//
// All of it is f32 whatever the logits' type. An exponential is one multiply-add and 2^: x log2 e less the maximum's, rounded once, so that logits keep
// their distances; those of rows far from zero, which the product would take out of f32 or round too much, are subtracted first. lse, logp and the alternatives'
// are differences from the maximum less the logarithm of the sum.
//
// Bound by memory, so a row is read once, by a warp, a CTA or a cluster of up to eight: a thread keeps a running maximum and sum of what it has seen,
// the warps hand theirs to each other, and for the loss's gradient the row waits in shared memory meanwhile. Instructions are the next
// bound (16 bits a logit leave 11 issue slots each at the memory's rate): two logits go into one instruction where there is one, nothing is
// looked at logit by logit that can be decided for a thread, and what a row costs beside its logits is spread over many of them a thread.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "token.cuh"

namespace ono {
__device__ __forceinline__ void cp_async16(void* smem, const void* g) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(g) : "memory");
}

template <int W>
__device__ __forceinline__ void group_sync() {
  if (W == 1) __syncwarp(); else __syncthreads();
}

// W warps to a row; CAP: places for candidates.
template <int W> struct TokShared {
  static constexpr int CAP = W == 1 ? 256 : 512;
  unsigned int count, threads, tally[W];
  unsigned short who[W * 32];
};
// What the warps of a row's CTAs tell each other, for this row and the next: maximum, sum, sum times exponent, bound of the alternatives.
template <bool TOP> struct TokPeers {
  float4 part[2][TOK_CTAS * 8];
  unsigned long long key[2][TOP ? TOK_CTAS : 1][ONO_TOP_MAX];
};

// The group's sum of a whole number.
template <int W>
__device__ __forceinline__ unsigned int group_count(unsigned int v, unsigned int* s_warp, int gt) {
  v = __reduce_add_sync(0xffffffffu, v);
  if (W == 1) return v;
  __syncthreads();
  if ((gt & 31) == 0) s_warp[gt >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) v += s_warp[w];
  return v;
}

// A group of 16 bytes of a row that begins `ph` logits into group 0; -inf outside of the row.
template <typename T>
__device__ __forceinline__ void tok_group(const T* x, int ph, int V, int v, float (&o)[TokVec<T>::E]) {
  constexpr int E = TokVec<T>::E;
  if (v * E >= ph && (v + 1) * E <= ph + V) {
    TokVec<T>::get(load16(x + (v * E - ph)), o);
  } else {
#pragma unroll
    for (int k = 0; k < E; ++k) { const int j = v * E + k - ph; o[k] = j >= 0 && j < V ? to_f32(x[j]) : __int_as_float(0xff800000); }
  }
}

// The candidates for the K largest logits of the groups v0 to v1 of a row, exactly: where so many logits are as large as the bound that there
// is no room for them (equal ones, mostly). The K-th largest value is found bit by bit, then come all that are above it, and of those
// equal to it the first ones.
template <typename T, int W>
__device__ __noinline__ void exact_candidates(const T* x, int ph, int V, int v0, int v1, int K, unsigned long long* cand, TokShared<W>& s, int gt) {
  constexpr int E = TokVec<T>::E, GT = W * 32, BITS = 8 * (int)sizeof(T);
  const float ninf = __int_as_float(0xff800000);
  auto for_all = [&](auto f) {
    for (int v = v0 + gt; v < v1; v += GT) {
      float q[E];
      tok_group(x, ph, V, v, q);
#pragma unroll
      for (int k = 0; k < E; ++k) if (q[k] > ninf) f(order_of(q[k]) >> (32 - BITS), q[k], v * E + k - ph);
    }
  };
  unsigned int valid = 0;
  for_all([&](unsigned int, float, int) { ++valid; });
  valid = group_count<W>(valid, s.tally, gt);
  const unsigned int want = min((unsigned int)K, valid);
  unsigned int value = 0;      // the largest with at least `want` logits not below it
  if (want) {
    for (int b = BITS - 1; b >= 0; --b) {
      const unsigned int t = value | 1u << b;
      unsigned int c = 0;
      for_all([&](unsigned int o, float, int) { c += o >= t; });
      if (group_count<W>(c, s.tally, gt) >= want) value = t;
    }
  }
  unsigned int above = 0;
  for_all([&](unsigned int o, float, int) { above += o > value; });
  above = group_count<W>(above, s.tally, gt);
  group_sync<W>();
  if (gt == 0) s.count = 0;
  group_sync<W>();
  if (want) for_all([&](unsigned int o, float q, int j) { if (o > value) cand[atomicAdd(&s.count, 1u)] = top_key(q, j); });
  unsigned int missing = want - above;      // of the equal ones, in the order of their places
  for (int at = v0; at < v1 && missing; at += GT) {
    const int v = at + gt;
    float q[E];
    unsigned int mine = 0;
    if (v < v1) {
      tok_group(x, ph, V, v, q);
#pragma unroll
      for (int k = 0; k < E; ++k) mine += q[k] > ninf && (order_of(q[k]) >> (32 - BITS)) == value;
    }
    unsigned int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned int w = __shfl_up_sync(0xffffffffu, before, o); if ((gt & 31) >= o) before += w; }
    unsigned int total = __shfl_sync(0xffffffffu, before, 31);
    before -= mine;
    if (W > 1) {
      __syncthreads();
      if ((gt & 31) == 0) s.tally[gt >> 5] = total;
      __syncthreads();
      total = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) { if (w < (gt >> 5)) before += s.tally[w]; total += s.tally[w]; }
    }
    if (mine && before < missing) {
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (q[k] > ninf && (order_of(q[k]) >> (32 - BITS)) == value && before++ < missing) cand[atomicAdd(&s.count, 1u)] = top_key(q[k], v * E + k - ph);
    }
    missing -= min(missing, total);
  }
  group_sync<W>();
}

// Maximum and sums of some logits: z = sum 2^(x log2 e - shift), u = sum 2^q q of those exponents q, shift = shift_of(m).
struct TokSums { float m, z, u; };
// The sum over the warp's lanes; every lane gets it.
template <bool ENT>
__device__ __forceinline__ TokSums tok_join(TokSums s) {
  const float m = of_order(__reduce_max_sync(0xffffffffu, order_of(s.m))), by = shift_of(s.m) - shift_of(m), f = exp2_of(by);
  if (ENT) s.u = s.z == 0.0f ? 0.0f : f * (s.u + fmaxf(by, -1e4f) * s.z);      // (zero times a number, far below)
  s.z = s.z == 0.0f ? 0.0f : f * s.z;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { s.z += __shfl_xor_sync(0xffffffffu, s.z, o); if (ENT) s.u += __shfl_xor_sync(0xffffffffu, s.u, o); }
  s.m = m;
  return s;
}

// Rows out of the ordinary, out of line.
// Sums of the groups v0 to v1 relative to the row's maximum m, differences first.
template <typename T, int W>
__device__ __noinline__ TokSums far_sums(const T* x, int ph, int V, int v0, int v1, float m, int gt) {
  constexpr int E = TokVec<T>::E;
  TokSums s = {m, 0.0f, 0.0f};
  for (int v = v0 + gt; v < v1; v += W * 32) {
    float o[E];
    tok_group(x, ph, V, v, o);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const float q = (o[k] - m) * LOG2E, e = exp2_of(q);
      s.z += e;
      s.u = fmaf(e, fmaxf(q, -1e4f), s.u);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { s.z += __shfl_xor_sync(0xffffffffu, s.z, o); s.u += __shfl_xor_sync(0xffffffffu, s.u, o); }
  return s;
}
// d = p (f + h ln p) with ln p = (x - m) - log_z, `hit` added at t.
template <typename T, typename O, int W>
__device__ __noinline__ void far_write(const T* x, O* d, int j0, int j1, float m, float log_z, float f, float h, int t, float hit, int gt) {
  for (int j = j0 + gt; j < j1; j += W * 32) {
    const float lp = (to_f32(x[j]) - m) - log_z, v = exp_of(lp) * (f + h * fmaxf(lp, -1e4f));
    d[j] = from_f32<O>(j == t ? v + hit : v);
  }
}
template <typename O, int W>
__device__ __noinline__ void zero_write(O* d, int j0, int j1, int gt) {
  constexpr int N = 16 / (int)sizeof(O);
  const int first = min(j1, j0 + (int)((N - (uintptr_t)(d + j0) / sizeof(O)) & (N - 1))), last = first + (max(j1 - first, 0) & ~(N - 1));
  if (gt < first - j0) d[j0 + gt] = from_f32<O>(0.0f);
  for (int j = first + gt * N; j < last; j += W * 32 * N) *reinterpret_cast<uint4*>(d + j) = make_uint4(0, 0, 0, 0);
  if (gt < j1 - last) d[last + gt] = from_f32<O>(0.0f);
}

// CTAs of an SM that the registers have to allow: 64 registers a thread, a few more where a row is gone through twice in one form or another (us, 1024
// threads to an SM against this: loss of 4096 x 50257 bf16 175.4 -> 165.9, gradient of 4096 x 128256 362.6 -> 357.6). A warp to a row in 64 registers spills 44 to 60
// bytes for the gradient and up to 88 for alternatives; in 80 it does not and is faster or slower by the row (us, 64 and 80: gradient of 30000 x 2500
// bf16 54, 59, of 4000 x 8000 f32 to bf16 32, 39, but of 16000 x 5000 f32 118, 111; five alternatives of 16000 x 5000 bf16 49, 52, f32 77, 71).
constexpr int tok_resident(int mode, int warps, int threads) {
  return (warps == 1 || mode <= TOK_TOP ? 1024 : mode == TOK_LOSS ? 896 : 768) / threads;
}

// Two together.
template <bool ENT>
__device__ __forceinline__ TokSums tok_two(const TokSums& a, const TokSums& b) {
  TokSums s = {fmaxf(a.m, b.m), 0.0f, 0.0f};
  const float at = shift_of(s.m), fa = shift_of(a.m) - at, fb = shift_of(b.m) - at, ea = exp2_of(fa), eb = exp2_of(fb);
  if (a.z != 0.0f) { s.z = ea * a.z; if (ENT) s.u = ea * (a.u + fmaxf(fa, -1e4f) * a.z); }
  if (b.z != 0.0f) { s.z += eb * b.z; if (ENT) s.u += eb * (b.u + fmaxf(fb, -1e4f) * b.z); }
  return s;
}

template <typename T, typename O, int MODE, int W, int NT>
__global__ void __launch_bounds__(NT, tok_resident(MODE, W, NT)) tok_kernel(const __grid_constant__ TokDev a) {
  constexpr int E = TokVec<T>::E, GT = W * 32, NG = NT / GT, CAP = TokShared<W>::CAP;
  constexpr bool TOP = MODE == TOK_TOP, ENT = MODE == TOK_ENTROPY || MODE == TOK_TOP, FWD = MODE <= TOK_TOP;
  static_assert(W == 1 || NG == 1, "a CTA takes one row, or a row a warp");
  const float ninf = __int_as_float(0xff800000);
  extern __shared__ __align__(16) unsigned char tok_smem[];
  __shared__ TokShared<W> s_all[TOP ? NG : 1];
  __shared__ TokPeers<TOP> s_peers;
  const int grp = threadIdx.x / GT, gt = threadIdx.x % GT, lane = threadIdx.x & 31, warp = gt >> 5;
  TokShared<W>& s = s_all[TOP ? grp : 0];
  int C = 1, rank = 0;
  if (W > 1) {
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(C));
    rank = (int)cluster_ctarank();
  }
  uint4* const kept = reinterpret_cast<uint4*>(tok_smem) + (size_t)grp * a.per;      // (staged)
  unsigned long long* const cand = reinterpret_cast<unsigned long long*>(tok_smem) + (size_t)grp * (CAP + ONO_TOP_MAX);      // (TOP)
  unsigned long long* const list = cand + CAP;
  const long long stride = (long long)(gridDim.x / C) * NG;
  const int K = TOP ? a.top : 1;
  auto sync_row = [&]() {      // all that share the row
    if (W == 1) __syncwarp();
    else if (C == 1) __syncthreads();
    else cluster_sync_all();
  };
  auto raw_target = [&](long long r) -> long long {
    if (!a.targets) return 0;
    if (r >= a.R) return a.ignore_id;
    return a.targets64 ? __ldg(reinterpret_cast<const long long*>(a.targets) + r) : (long long)__ldg(reinterpret_cast<const int*>(a.targets) + r);
  };
  auto target = [&](long long t) -> int {      // -1: the row counts for nothing
    if (a.targets && t == a.ignore_id) return -1;
    if (t >= 0 && t < a.V) return (int)t;
    if (a.status && gt == 0) atomicExch(a.status, ONO_ERR_BAD_ARG);
    return -1;
  };

  const bool staged = MODE == TOK_LOSS && a.staged;
  // A row that is kept: on its way into shared memory from when the one before it has left. A thread fetches what it will read itself.
  auto fetch = [&](long long r) {
    const T* const x = reinterpret_cast<const T*>(a.x) + r * a.ld;
    const int ph = (int)(((uintptr_t)x / sizeof(T)) & (E - 1)), va = max(rank * a.per, ph ? 1 : 0), vb = min(rank * a.per + a.per, (ph + a.V) / E);
    const T* src = x + ((va + gt) * E - ph);
    uint4* dst = kept + gt;
#pragma unroll 4
    for (int v = va + gt; v < vb; v += GT, src += GT * E, dst += GT) cp_async16(dst, src);
  };

  // A CTA's shared memory may be written to once it runs: said here, waited for ahead of the first word to another.
  bool met = W == 1 || C == 1;
  if (!met) cluster_arrive();
  auto meet = [&]() { if (!met) { cluster_wait(); met = true; } };
  long long r = (long long)(blockIdx.x / C) * NG + grp;
  long long raw_next = raw_target(r);
  if (staged && r < a.R && target(raw_next) >= 0) fetch(r);
  int live = 0;
  for (; r < a.R; r += stride) {
    const int t = target(raw_next);
    raw_next = raw_target(r + stride);
    const T* const x = reinterpret_cast<const T*>(a.x) + r * a.ld;
    // The row in groups of 16 bytes: whole ones from va to vb are this CTA's, and of the first and last one, if they are not whole, a logit a thread.
    const int ph = (int)(((uintptr_t)x / sizeof(T)) & (E - 1)), nv = (ph + a.V + E - 1) / E, v0 = rank * a.per, v1 = min(nv, v0 + a.per);
    const int va = max(v0, ph ? 1 : 0), vb = min(v1, (ph + a.V) / E);
    const int jh = gt - ph, jt = (nv - 1) * E + gt - ph;
    const bool has_h = gt < E && v0 == 0 && ph && jh >= 0 && jh < a.V, has_t = gt < E && nv - 1 >= v0 && nv - 1 < v1 && nv - 1 >= vb && (nv > 1 || !ph) && jt < a.V;
    O* const d = FWD ? nullptr : reinterpret_cast<O*>(a.out) + r * a.ld_out;
    const int j0 = max(v0 * E - ph, 0), j1 = min(v1 * E - ph, a.V);      // the CTA's logits
    // f(two logits) of them to the output, `hit` added where the target is
    auto write = [&](float xh, float xt, float hit, auto f) {
      auto one = [&](int j, float v) {
        float q = f(make_float2(v, v)).x;
        if (j == t) q += hit;
        d[j] = from_f32<O>(q);
      };
      if (has_h) one(jh, xh);
      if (has_t) one(jt, xt);
      if ((((uintptr_t)d / sizeof(O) - ph) & (E - 1)) == 0) {
        const int vt = t < 0 ? -1 : (t + ph) / E;
        auto put = [&](int v, const uint4& w4) {
          float w[E];
          TokVec<T>::get(w4, w);
#pragma unroll
          for (int k = 0; k < E; k += 2) { const float2 p = f(make_float2(w[k], w[k + 1])); w[k] = p.x; w[k + 1] = p.y; }
          if (v == vt) {
#pragma unroll
            for (int k = 0; k < E; ++k) if (v * E + k - ph == t) w[k] += hit;
          }
          store_group<O, E>(d + (v * E - ph), w);
        };
        int v = va + gt;
        for (; v + 3 * GT < vb; v += 4 * GT) {
          uint4 w4[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) w4[q] = staged ? kept[v + q * GT - va] : load16(x + ((v + q * GT) * E - ph));
#pragma unroll
          for (int q = 0; q < 4; ++q) put(v + q * GT, w4[q]);
        }
        if (v < vb) {
          uint4 w4[3];
#pragma unroll
          for (int q = 0; q < 3; ++q) if (v + q * GT < vb) w4[q] = staged ? kept[v + q * GT - va] : load16(x + ((v + q * GT) * E - ph));
#pragma unroll
          for (int q = 0; q < 3; ++q) if (v + q * GT < vb) put(v + q * GT, w4[q]);
        }
      } else {      // the output's rows are aligned another way: value by value
        group_sync<W>();      // (here a thread reads what others have kept)
        for (int i = va * E + gt; i < vb * E; i += GT) one(i - ph, to_f32(staged ? reinterpret_cast<const T*>(kept)[i - va * E] : x[i - ph]));
        group_sync<W>();
      }
    };
    if (t < 0) {
      if (rank == 0 && MODE != TOK_GRAD) {
        if (gt == 0) {
          if (a.logp) a.logp[r] = 0.0f;
          if (a.lse) a.lse[r] = 0.0f;
          if (FWD && a.lse_low) a.lse_low[r] = 0.0f;
          if (ENT && a.entropy) a.entropy[r] = 0.0f;
        }
        if (TOP && gt < K) { a.top_logp[r * K + gt] = ninf; a.top_id[r * K + gt] = -1; }
      }
      if (!FWD) zero_write<O, W>(d, j0, j1, gt);
      if (staged && r + stride < a.R && target(raw_next) >= 0) fetch(r + stride);
      continue;
    }
    float x_t = 0.0f, i0 = 1.0f, i1 = 0.0f, i2 = 0.0f, i3 = 0.0f, low = 0.0f;
    if (MODE != TOK_GRAD && gt == 0 && a.targets) x_t = to_f32(x[t]);
    if (MODE == TOK_LOSS && a.weight) i0 = __ldg(a.weight + r);
    if (MODE == TOK_GRAD) {
      i0 = __ldg(a.lse_in + r);
      if (a.lse_low_in) low = __ldg(a.lse_low_in + r);
      if (a.d_logp) i1 = __ldg(a.d_logp + r);
      if (a.d_entropy) { i2 = __ldg(a.d_entropy + r); i3 = __ldg(a.entropy_in + r); }
    }
    const float xh = has_h ? to_f32(x[jh]) : ninf, xt = has_t ? to_f32(x[jt]) : ninf;
    TokSums g = {0.0f, 1.0f, 0.0f};
    float log_z = 0.0f;      // ln of the row's sum relative to its maximum
    bool far = false;
    if (MODE != TOK_GRAD || fabsf(i0) > LSE_EXACT) {
      TokSums mine = {ninf, 0.0f, 0.0f};
      float2 z2[2] = {both(0.0f), both(0.0f)}, u2[2] = {both(0.0f), both(0.0f)};
      float shift = 0.0f;
      if (staged) asm volatile("cp.async.wait_all;" ::: "memory");
      auto raise = [&](float m) {
        if (m > mine.m) {
          const float to = shift_of(m), by = mine.m < -TOK_FAR ? 0.0f : shift - to;      // (what was too far below has left nothing)
          const float2 f = both(exp2_of(by));
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (ENT) u2[k] = mul_2(f, fma_2(both(fmaxf(by, -1e4f)), z2[k], u2[k]));
            z2[k] = mul_2(z2[k], f);
          }
          mine.m = m;
          shift = to;
        }
      };
      auto take = [&](int k, float2 v) {
        const float2 q = fma_2(v, both(LOG2E), both(-shift)), e = make_float2(exp2_of(q.x), exp2_of(q.y));
        z2[k] = add_2(z2[k], e);
        if (ENT) u2[k] = fma_2(e, make_float2(fmaxf(q.x, -1e4f), fmaxf(q.y, -1e4f)), u2[k]);
      };
      auto take4 = [&](const uint4& w) {
        float o[E];
        TokVec<T>::get(w, o);
#pragma unroll
        for (int k = 0; k < E; k += 2) take(k / 2 % 2, make_float2(o[k], o[k + 1]));
      };
      int v = va + gt;
      for (; v + 3 * GT < vb; v += 4 * GT) {
        uint4 w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = staged ? kept[v + q * GT - va] : load16(x + ((v + q * GT) * E - ph));
        raise(TokVec<T>::most(w));
#pragma unroll
        for (int q = 0; q < 4; ++q) take4(w[q]);
      }
      if (v < vb) {
        uint4 w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          w[q] = make_uint4(TokVec<T>::NINF, TokVec<T>::NINF, TokVec<T>::NINF, TokVec<T>::NINF);
          if (q < 3 && v + q * GT < vb) w[q] = staged ? kept[v + q * GT - va] : load16(x + ((v + q * GT) * E - ph));
        }
        raise(TokVec<T>::most(w));
#pragma unroll
        for (int q = 0; q < 3; ++q) if (v + q * GT < vb) take4(w[q]);
      }
      if (has_h || has_t) {
        raise(fmaxf(xh, xt));
        take(0, make_float2(xh, xt));
      }
      z2[0] = add_2(z2[0], z2[1]);
      mine.z = z2[0].x + z2[0].y;
      if (ENT) { u2[0] = add_2(u2[0], u2[1]); mine.u = u2[0].x + u2[0].y; }
      const float tm = mine.m;
      float cut = ninf;
      if (TOP) {
        // the warp's J-th largest of its lanes' maxima; the smallest of the warps' bounds: W * J >= K logits are not below it
        unsigned int rest = order_of(tm), best = __reduce_max_sync(0xffffffffu, rest);
        for (int q = 1; q < (K + W - 1) / W; ++q) {
          const unsigned int who = __ballot_sync(0xffffffffu, rest == best);
          if (lane == __ffs(who) - 1) rest = 0;
          best = __reduce_max_sync(0xffffffffu, rest);
        }
        cut = best ? of_order(best) : ninf;
        if (gt == 0) s.count = s.threads = 0;
        if (gt < K) list[gt] = 0;
      }
      g = tok_join<ENT>(mine);
      const int par = live & 1;
      const float4* const part = s_peers.part[par];
      if (W > 1) {
        const float4 told = make_float4(g.m, g.z, g.u, cut);
        if (C == 1) { if (lane == 0) s_peers.part[par][warp] = told; }
        else {
          meet();
          if (lane < C) st_cluster_v4(mapa_shared(smem_u32(&s_peers.part[par][rank * W + warp]), (uint32_t)lane), told);
        }
        sync_row();
        auto of = [&](int i) { return i < C * W ? TokSums{part[i].x, part[i].y, part[i].z} : TokSums{ninf, 0.0f, 0.0f}; };
        g = tok_join<ENT>(W == 8 && C > 4 ? tok_two<ENT>(of(lane), of(32 + lane)) : of(lane));
        if (TOP) {
#pragma unroll
          for (int w = 0; w < W; ++w) { const float c = part[rank * W + w].w; cut = w ? fminf(cut, c) : c; }
        }
      }
      if (TOP && W == 1) __syncwarp();
      far = fabsf(g.m) > TOK_FAR && g.m > ninf;
      if (far) {
        // logits of a size that log2 e takes out of f32: differences first. (A second exchange, by all that share the row.)
        mine = far_sums<T, W>(x, ph, a.V, v0, v1, g.m, gt);
        if (W > 1) {
          sync_row();      // the first sums have been read
          const float4 told = make_float4(0.0f, mine.z, mine.u, 0.0f);
          if (C == 1) { if (lane == 0) s_peers.part[par][warp] = told; }
          else if (lane < C) st_cluster_v4(mapa_shared(smem_u32(&s_peers.part[par][rank * W + warp]), (uint32_t)lane), told);
          sync_row();
          mine.z = mine.u = 0.0f;
          for (int i = 0; i < C * W; ++i) { mine.z += part[i].y; mine.u += part[i].z; }
        }
        g.z = mine.z;
        g.u = mine.u;
      }
      const bool empty = g.z == 0.0f;
      const float ln_z = empty ? 0.0f : logf(g.z);
      // (the sum is relative to the shift, which is the maximum times log2 e rounded)
      log_z = fabsf(g.m) <= TOK_FAR ? fmaf(-fmaf(g.m, LOG2E, -shift_of(g.m)), LN2, ln_z) : ln_z;
      // ln p of a logit: the distance from the maximum first, which is rounded once if at all
      auto lp = [&](float v) { return (v - g.m) - log_z; };
      if (MODE != TOK_GRAD && gt == 0 && rank == 0) {
        const float lse = empty ? ninf : g.m + log_z;
        if (a.lse) a.lse[r] = lse;
        if (FWD && a.lse_low) a.lse_low[r] = empty || far ? 0.0f : low_of(shift_of(g.m), g.z, lse);
        if (a.logp) a.logp[r] = empty ? ninf : lp(x_t);
        if (ENT && a.entropy) a.entropy[r] = empty ? 0.0f : fmaf(-(g.u / g.z), LN2, ln_z);
      }
      if (TOP) {
        auto offer = [&](float v, int j) {
          if (v >= cut && v > ninf) {
            const unsigned int at_c = atomicAdd(&s.count, 1u);
            if (at_c < CAP) cand[at_c] = top_key(v, j);
          }
        };
        // the threads that have seen a logit that reaches the bound; what they have seen is read again, by all
        if (tm >= cut && tm > ninf) s.who[atomicAdd(&s.threads, 1u)] = (unsigned short)gt;
        group_sync<W>();
        const unsigned int each = max(vb - va + GT - 1, 0) / GT, items = each * s.threads;
        for (unsigned int i = gt; i < items; i += 4 * GT) {
          int v[4];
          uint4 w[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const unsigned int iq = i + q * GT;
            v[q] = iq < items ? va + s.who[iq / each] + (int)(iq % each) * GT : vb;
            if (v[q] < vb) w[q] = load16(x + (v[q] * E - ph));
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (v[q] >= vb || !(TokVec<T>::most(w[q]) >= cut)) continue;
            float o[E];
            TokVec<T>::get(w[q], o);
#pragma unroll
            for (int k = 0; k < E; ++k) offer(o[k], v[q] * E + k - ph);
          }
        }
        if (has_h) offer(xh, jh);
        if (has_t) offer(xt, jt);
        group_sync<W>();
        int have = (int)s.count;
        if (have > CAP) {
          group_sync<W>();
          exact_candidates<T, W>(x, ph, a.V, v0, v1, K, cand, s, gt);
          have = (int)s.count;
        }
        for (int i = gt; i < have; i += GT) {
          const unsigned long long key = cand[i];
          int above = 0;
#pragma unroll 8
          for (int q = 0; q < have; ++q) above += cand[q] > key;
          if (above < K) list[above] = key;
        }
        group_sync<W>();
        auto put = [&](int k, unsigned long long key) {
          a.top_logp[r * K + k] = key ? lp(of_order((unsigned int)(key >> 32))) : ninf;
          a.top_id[r * K + k] = key ? (int)(0xffffffffu - (unsigned int)key) : -1;
        };
        if (W == 1 || C == 1) {
          if (gt < K) put(gt, list[gt]);
          group_sync<W>();
        } else {
          for (int i = gt; i < K * C; i += GT) {
            const uint32_t to = mapa_shared(smem_u32(&s_peers.key[par][rank][i / C]), (uint32_t)(i % C));
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(list[i / C]) : "memory");
          }
          cluster_sync_all();
          // every CTA finds its own keys' places among all, a warp a key
          unsigned long long all[TOK_CTAS * ONO_TOP_MAX / 32];
          unsigned int there = 0;
#pragma unroll
          for (int q = 0; q < TOK_CTAS * ONO_TOP_MAX / 32; ++q) {
            const int i = q * 32 + lane;
            all[q] = i < C * K ? s_peers.key[par][i / K][i % K] : 0;
            there += all[q] != 0;
          }
          for (int k = warp; k < K; k += W) {
            const unsigned long long key = list[k];
            unsigned int above = 0;
#pragma unroll
            for (int q = 0; q < TOK_CTAS * ONO_TOP_MAX / 32; ++q) above += all[q] > key;
            above = __reduce_add_sync(0xffffffffu, above);
            if (lane == 0 && key && above < (unsigned)K) put((int)above, key);
          }
          there = __reduce_add_sync(0xffffffffu, there);
          if (rank == 0 && gt < K && gt >= (int)there) put(gt, 0);
          group_sync<W>();      // (the list has been read)
        }
      }
      ++live;
      if (W == 1) __syncwarp();      // (out may be x: what was wanted of the row has been read; a CTA has met above)
    }
    const bool empty = MODE == TOK_GRAD ? i0 == ninf : g.z == 0.0f;
    if (!FWD && empty) {
      zero_write<O, W>(d, j0, j1, gt);
    } else if (MODE == TOK_LOSS) {
      const float w = a.scale * i0;
      if (far) {
        far_write<T, O, W>(x, d, j0, j1, g.m, log_z, w, 0.0f, t, -w, gt);
      } else {
        const float2 off = both(-shift_of(g.m)), fs = both(w / g.z);
        write(xh, xt, -w, [&](float2 v) { const float2 q = fma_2(v, both(LOG2E), off); return mul_2(make_float2(exp2_of(q.x), exp2_of(q.y)), fs); });
      }
    } else if (MODE == TOK_GRAD) {
      if (fabsf(i0) <= LSE_EXACT) {
        // -p (g + h (ln p + H)) with ln p = ln 2 (q - off): q = x log2 e - c, c the product lse log2 e rounded, off what that and lse's own rounding took off
        const float c = i0 * LOG2E, off = fmaf(low, LOG2E, fmaf(i0, LOG2E, -c)), f = -exp2_of(-off);
        const float2 at = both(-c), A = both(f * (i1 + i2 * (i3 - LN2 * off))), B = both(f * LN2 * i2);
        if (a.d_entropy)
          write(xh, xt, i1, [&](float2 v) {
            float2 q = fma_2(v, both(LOG2E), at);
            q = make_float2(fmaxf(q.x, -1e4f), fmaxf(q.y, -1e4f));      // (zero times a number; no NaN comes here)
            return mul_2(make_float2(exp2_of(q.x), exp2_of(q.y)), fma_2(q, B, A));
          });
        else
          write(xh, xt, i1, [&](float2 v) { const float2 q = fma_2(v, both(LOG2E), at); return mul_2(make_float2(exp2_of(q.x), exp2_of(q.y)), A); });
      } else {      // as for a NaN, which is in lse then
        far_write<T, O, W>(x, d, j0, j1, isnan(i0) ? i0 : g.m, log_z, -(i1 + i2 * i3), -i2, t, i1, gt);
      }
    }
    if (staged && r + stride < a.R && target(raw_next) >= 0) fetch(r + stride);
  }
  meet();
}

// How a launch is laid out.
struct TokShape { int warps, ctas, per, staged; size_t smem; };

// Bytes of a row that is kept, to a CTA. (Us, loss of 4096 x 50257 bf16: 16384 207, 32768 168, 65536 164; of 1000 x 128256 113, 113, 122.) Longer slices of
// the longest rows are kept up to TOK_KEPT_MAX, beyond that nothing is.
constexpr int TOK_SLICE = 32768, TOK_KEPT_MAX = 100 * 1024;

static TokShape tok_shape(long long rows, int V, int esz, int mode, int top) {
  const long long groups = tok_groups(V, esz), bytes = groups * 16;
  TokShape s = {};
  s.ctas = 1;
  // A warp to a row where there are rows for all of them: what a row costs beside its logits is then paid once (us, four warps against one:
  // entropy of 47005 x 2322 f32 123.8, 69.9, of 8000 x 15000 bf16 51.2, 45.3; loss of 16000 x 5000 bf16 79.4, 67.7, but of 8000 x 8000 57.1, 60.7;
  // entropy of 300 x 5000 4.8, 7.7).
  s.warps = rows >= 16ll * ono_num_sms() && bytes <= (mode == TOK_LOSS ? 12288 : 32768) ? 1 : 4;
  // Longer rows are shared out among CTAs where there are few. (Us, one CTA a row, CTAs by these limits, twice the CTAs allowed: entropy of 20 x 50257 bf16 6.2, 4.4, 4.3, of 150
  // 7.7, 6.6, 7.7, of 333 10.7, 9.6, 10.1, of 600 14.7, 14.7, 13.5; five alternatives of 4 x 50257 f32 11.9, 7.1, 7.1, of 333 22.2, 18.1, 22.1, of 600 33, 33, 43; half as
  // many CTAs are between. Not below 8 KB a CTA: 4 KB and 16 KB are within a tenth for 300 x 50257, 16 KB better by that for 300 x 5000.)
  if (s.warps > 1) {
    while (s.ctas < TOK_CTAS && ((mode == TOK_LOSS && bytes > (long long)TOK_SLICE * s.ctas) || (rows * s.ctas <= 4 * ono_num_sms() && bytes > 8192ll * s.ctas))) s.ctas *= 2;
  }
  // Eight warps up to two CTAs an SM. (Us, four, eight up to here, eight for four times as many: twenty alternatives of 4 x 128256 bf16 12.5, 10.3, 10.3; entropy of
  // 20 x 50257 4.1, 4.4, 4.3, of 100 5.3, 5.4, 7.9; five alternatives of 4 x 50257 f32 7.8, 7.1, 7.1, of 100 11.2, 11.2, 15.2.)
  if (s.warps > 1 && mode != TOK_LOSS && rows * s.ctas <= 2 * ono_num_sms()) s.warps = 8;
  s.per = (int)((groups + s.ctas - 1) / s.ctas);
  // A warp whose lanes have fewer logits than its share of the alternatives bounds nothing, and every logit would be a candidate (us, five of
  // 35 x 519 bf16 17.8, so 4.6; twenty of 75 x 355 f32 10.5, 6.3).
  while (mode == TOK_TOP && s.warps > 1 && s.ctas == 1 && s.per < 32 * (s.warps - 1) + (top + s.warps - 1) / s.warps) s.warps = s.warps == 8 ? 4 : 1;
  const int rows_of_cta = s.warps == 1 ? 4 : 1;
  s.staged = mode == TOK_LOSS && (long long)s.per * 16 <= TOK_KEPT_MAX;
  if (s.staged) s.smem = (size_t)s.per * 16 * rows_of_cta;
  if (mode == TOK_TOP) s.smem = (size_t)(8 * ((s.warps == 1 ? 256 : 512) + ONO_TOP_MAX)) * rows_of_cta;
  return s;
}

template <typename T, typename O, int MODE, int GW, int NT>
static cudaError_t tok_go(const TokDev& d, const TokShape& s, cudaStream_t st) {
  auto kern = tok_kernel<T, O, MODE, GW, NT>;
  // The allowance is the function's, for all threads of the host: always the most that any call takes, or one call would lower it under another's launch.
  cudaError_t e = s.smem > 32768 ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TOK_KEPT_MAX) : cudaSuccess;
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
  if (v == 0 || (v >> 16) != s.smem) {
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
  if (16 * tok_groups(d.V, sizeof(T)) <= (MODE == TOK_TOP ? TOK_SHORT_TOP : TOK_SHORT_ROW)) return tok_short(d, MODE, sizeof(T) == 2, sizeof(O) == 2, st);
  const TokShape s = tok_shape(d.R, d.V, sizeof(T), MODE, d.top);
  d.per = s.per;
  d.staged = s.staged;
  cudaError_t e;
  if constexpr (MODE == TOK_LOSS) e = s.warps == 1 ? tok_go<T, O, MODE, 1, 128>(d, s, st) : tok_go<T, O, MODE, 4, 128>(d, s, st);
  else e = s.warps == 1 ? tok_go<T, O, MODE, 1, 128>(d, s, st) : s.warps == 4 ? tok_go<T, O, MODE, 4, 128>(d, s, st) : tok_go<T, O, MODE, 8, 256>(d, s, st);
  if (e != cudaSuccess) { set_error("tokens launch: %s", cudaGetErrorString(e), 0, 0); return -7; }
  return 0;
}
}  // namespace ono

using namespace ono;

extern "C" int ono_tokens(const OnoTokens* t, ono_stream_t stream) {
  if (!t || t->R < 0 || t->V <= 0 || t->V > ONO_DIM_MAX || t->ld < t->V || (t->R && !t->x) || t->top < 0 || t->top > ONO_TOP_MAX || t->top > t->V ||
      (t->top > 0 && t->R && (!t->top_logp || !t->top_id)) || (t->out && (t->ld_out < t->V || t->entropy || t->top || t->lse_low)) || (t->lse_low && !t->lse) || (!t->targets && (t->logp || t->out))) {
    set_error("bad tokens args%s", "", 0, 0);
    return -1;
  }
  if (t->out == t->x && t->out && (t->out_bf16 != t->x_bf16 || t->ld_out != t->ld)) { set_error("tokens: out over x needs the same type and rows%s", "", 0, 0); return -1; }
  if (t->R == 0) return 0;
  TokDev d = {};
  d.x = t->x; d.targets = t->targets; d.R = t->R; d.ld = t->ld; d.ld_out = t->ld_out; d.ignore_id = t->ignore_id;
  d.V = t->V; d.targets64 = t->targets64; d.top = t->top; d.logp = t->logp; d.lse = t->lse; d.lse_low = t->lse_low; d.entropy = t->entropy;
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
  if (!t || t->R < 0 || t->V <= 0 || t->V > ONO_DIM_MAX || t->ld < t->V || t->ld_out < t->V || (t->R && (!t->x || !t->out || !t->lse)) || (!t->d_logp && !t->d_entropy) ||
      (t->d_logp && !t->targets) || (t->entropy == nullptr) != (t->d_entropy == nullptr)) {
    set_error("bad tokens_grad args%s", "", 0, 0);
    return -1;
  }
  if (t->out == t->x && (t->out_bf16 != t->x_bf16 || t->ld_out != t->ld)) { set_error("tokens_grad: out over x needs the same type and rows%s", "", 0, 0); return -1; }
  if (t->R == 0) return 0;
  TokDev d = {};
  d.x = t->x; d.targets = t->targets; d.R = t->R; d.ld = t->ld; d.ld_out = t->ld_out; d.ignore_id = t->ignore_id;
  d.V = t->V; d.targets64 = t->targets64; d.out = t->out; d.status = t->status;
  d.lse_in = t->lse; d.lse_low_in = t->lse_low; d.entropy_in = t->entropy; d.d_logp = t->d_logp; d.d_entropy = t->d_entropy;
  cudaStream_t st = (cudaStream_t)stream;
  using B = __nv_bfloat16;
  if (t->x_bf16) return t->out_bf16 ? tok_run<B, B, TOK_GRAD>(d, st) : tok_run<B, float, TOK_GRAD>(d, st);
  return t->out_bf16 ? tok_run<float, B, TOK_GRAD>(d, st) : tok_run<float, float, TOK_GRAD>(d, st);
}
