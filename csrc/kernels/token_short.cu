// The operators of token_loss.cu on short rows: a row lies in the registers of one warp, or of a few lanes of it, which load all of it at once.
// Nothing is looped over and nothing goes through shared memory; a row costs its loads, a handful of shuffles and its stores, so that
// what bounds it is memory or, of rows of a few logits, the launch and the latency of its one chain of loads. (The gradient of the longest bf16 rows spills 52 bytes in
// the 64 registers of eight CTAs; seven without take longer: 16384 x 2000 25.0 us against 22.5.)
#include <type_traits>

#include "token.cuh"

namespace ono {

// NV groups of 16 bytes to a lane. NV == 1: 2^lg lanes to a row, 32 >> lg rows to a warp. CTAs of 128 threads: of 256 they took one to three percent
// longer (16384 rows of 1000 f32 logits, loss 23.1 us against 22.4).
template <typename T, typename O, int MODE, int NV>
__global__ void __launch_bounds__(128, NV == 1 ? 12 : 8) tok_short_kernel(const __grid_constant__ TokDev a, int lg) {
  constexpr int E = TokVec<T>::E;
  constexpr bool TOP = MODE == TOK_TOP, ENT = MODE == TOK_ENTROPY || MODE == TOK_TOP, FWD = MODE <= TOK_TOP, LOW = MODE == TOK_GRAD_LOW, GRAD = MODE == TOK_GRAD || LOW;
  const float ninf = __int_as_float(0xff800000);
  const unsigned int full = 0xffffffffu;
  const int lane = threadIdx.x & 31, G = NV == 1 ? 1 << lg : 32, gl = lane & (G - 1);
  const long long job = (long long)blockIdx.x * 4 + (threadIdx.x >> 5), r = NV == 1 ? (job << (5 - lg)) + (lane >> lg) : job;
  const bool in = r < a.R;
  const long long rr = in ? r : 0;
  const T* const x = reinterpret_cast<const T*>(a.x) + rr * a.ld;
  const int ph = (int)(((uintptr_t)x / sizeof(T)) & (E - 1));
  long long raw = 0;
  if (in && a.targets) raw = a.targets64 ? __ldg(reinterpret_cast<const long long*>(a.targets) + r) : (long long)__ldg(reinterpret_cast<const int*>(a.targets) + r);
  // The ends of a row that begins anywhere: groups that are not whole. Where the row has that many lanes each takes a logit of either, else the
  // lane of the group takes them one by one.
  const bool split = G >= E;
  const int tail = (ph + a.V) / E * E - ph, jh = gl - ph, jt = tail + gl;
  const bool has_h = split && in && ph && gl < E && jh >= 0 && jh < a.V, has_t = split && in && gl < E && jt < a.V && (tail >= 0 || !ph);
  const bool ends = __any_sync(full, has_h || has_t);
  const float xh = has_h ? to_f32(x[jh]) : ninf, xt = has_t ? to_f32(x[jt]) : ninf;
  uint4 w[NV];
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int j = (gl + q * G) * E - ph;
    w[q] = make_uint4(TokVec<T>::NINF, TokVec<T>::NINF, TokVec<T>::NINF, TokVec<T>::NINF);
    if (!in || j >= a.V) continue;
    if (j >= 0 && j + E <= a.V) {
      w[q] = load16(x + j);
    } else if (!split) {
      T* o = reinterpret_cast<T*>(&w[q]);
#pragma unroll
      for (int k = 0; k < E; ++k) if (j + k >= 0 && j + k < a.V) o[k] = x[j + k];
    }
  }
  float i0 = 1.0f, i1 = 0.0f, i2 = 0.0f, i3 = 0.0f, low = 0.0f;
  if (MODE == TOK_LOSS && a.weight) i0 = __ldg(a.weight + rr);
  if (GRAD) {
    i0 = __ldg(a.lse_in + rr);
    if (LOW) low = __ldg(a.lse_low_in + rr);
    if (a.d_logp) i1 = __ldg(a.d_logp + rr);
    if (a.d_entropy) { i2 = __ldg(a.d_entropy + rr); i3 = __ldg(a.entropy_in + rr); }
  }
  int t = -1;      // the row counts for nothing
  if (in && !(a.targets && raw == a.ignore_id)) {
    if (raw >= 0 && raw < a.V) t = (int)raw;
    else if (a.status && gl == 0) atomicExch(a.status, ONO_ERR_BAD_ARG);
  }
  const bool live = t >= 0;
  float x_t = 0.0f;
  if (!GRAD && live && gl == 0) x_t = to_f32(x[t]);
  auto group = [&](float v, auto join) {      // over the row's lanes
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) if (o < G) v = join(v, __shfl_xor_sync(full, v, o));
    return v;
  };
  auto values = [&](auto f) {      // f(two logits, their places)
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      float o[E];
      TokVec<T>::get(w[q], o);
#pragma unroll
      for (int k = 0; k < E; k += 2) f(make_float2(o[k], o[k + 1]), (gl + q * G) * E - ph + k, (gl + q * G) * E - ph + k + 1);
    }
    if (ends) f(make_float2(xh, xt), jh, jt);
  };
  float m = 0.0f, z = 1.0f, u = 0.0f, log_z = 0.0f;
  bool far = false;
  if (!GRAD || __any_sync(full, live && fabsf(i0) > LSE_EXACT)) {
    m = fmaxf(xh, xt);
#pragma unroll
    for (int q = 0; q < NV; ++q) m = fmaxf(m, TokVec<T>::most(w[q]));
    m = group(m, [](float p, float q) { return fmaxf(p, q); });
    far = fabsf(m) > TOK_FAR && m > ninf;      // (differences first then, see token_loss.cu)
    const float at = shift_of(m);
    if (!__any_sync(full, far)) {
      float2 z2 = both(0.0f), u2 = both(0.0f);
      values([&](float2 v, int, int) {
        const float2 q = fma_2(v, both(LOG2E), both(-at)), e = make_float2(exp2_of(q.x), exp2_of(q.y));
        z2 = add_2(z2, e);
        if (ENT) u2 = fma_2(e, make_float2(fmaxf(q.x, -1e4f), fmaxf(q.y, -1e4f)), u2);
      });
      z = z2.x + z2.y;
      u = u2.x + u2.y;
    } else {
      z = u = 0.0f;
      values([&](float2 v, int, int) {
        const float p = far ? (v.x - m) * LOG2E : fmaf(v.x, LOG2E, -at), q = far ? (v.y - m) * LOG2E : fmaf(v.y, LOG2E, -at), e = exp2_of(p), f = exp2_of(q);
        z += e + f;
        if (ENT) u += e * fmaxf(p, -1e4f) + f * fmaxf(q, -1e4f);
      });
    }
    auto add = [](float p, float q) { return p + q; };
    z = group(z, add);
    if (ENT) u = group(u, add);
    const bool empty = z == 0.0f;
    const float ln_z = empty ? 0.0f : logf(z);
    log_z = fabsf(m) <= TOK_FAR ? fmaf(-fmaf(m, LOG2E, -at), LN2, ln_z) : ln_z;
    auto lp = [&](float v) { return (v - m) - log_z; };
    if (!GRAD && in && gl == 0) {
      const float lse = empty ? ninf : m + log_z;
      if (a.lse) a.lse[r] = !live ? 0.0f : lse;
      if (FWD && a.lse_low) a.lse_low[r] = !live || empty || far ? 0.0f : low_of(at, z, lse);
      if (a.logp) a.logp[r] = !live ? 0.0f : empty ? ninf : lp(x_t);
      if (ENT && a.entropy) a.entropy[r] = !live || empty ? 0.0f : fmaf(-(u / z), LN2, ln_z);
    }
    if constexpr (TOP) {
      // The row's lanes find the largest of their largest logits, `top` times, of equal ones the lane with the lowest place; it goes on to its next.
      // A lane's logits are in the order of their places: of the row's beginning, its group, of the row's end. 0: none left. (65536 rows of 100 f32: five take
      // 55 us, twenty 135; with the place as the lower half of 64-bit keys, and shuffles for all of it, 1.4 and 1.6 times as long.)
      static_assert(NV == 1, "one group to a lane");
      unsigned int key[E + 2], best, slot;
      auto key_of = [&](float v) { return v > ninf ? order_of(v) : 0u; };
      {
        float o[E];
        TokVec<T>::get(w[0], o);
        key[0] = key_of(xh);
#pragma unroll
        for (int k = 0; k < E; ++k) key[1 + k] = key_of(o[k]);
        key[E + 1] = key_of(xt);
      }
      auto find = [&] {
        best = slot = 0;
#pragma unroll
        for (int k = 0; k < E + 2; ++k) if (key[k] > best) { best = key[k]; slot = k; }
      };
      find();
      const int lane0 = lane - gl;
      auto most = [&](unsigned int v) {
        if (G == 32) return __reduce_max_sync(full, v);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) { const unsigned int other = __shfl_xor_sync(full, v, o & (G - 1)); v = max(v, other); }
        return v;
      };
      unsigned int out_key = 0, out_id = 0;      // the k-th at the k-th lane, G of them at a time
      auto put = [&](int k, unsigned int o, unsigned int id) {
        if (!in) return;
        a.top_logp[r * a.top + k] = live && o ? lp(of_order(o)) : ninf;
        a.top_id[r * a.top + k] = live && o ? (int)id : -1;
      };
      for (int k = 0; k < a.top; ++k) {
        const unsigned int largest = most(best);
        if (__all_sync(full, largest == 0)) {      // none left: the pending ones, and nothing behind them
          for (int i = k - (k & (G - 1)) + gl; i < a.top; i += G) put(i, i < k ? out_key : 0, out_id);
          break;
        }
        const unsigned int at = (unsigned int)(slot == 0 ? jh : slot == E + 1 ? jt : gl * E - ph + (int)slot - 1);
        const bool mine = largest != 0 && best == largest;
        unsigned int who = __ballot_sync(full, mine) >> lane0 & (full >> (32 - G));
        if (__any_sync(full, (who & (who - 1)) != 0)) {
          const unsigned int low = ~most(mine ? ~at : 0u);
          who = __ballot_sync(full, mine && at == low) >> lane0 & (full >> (32 - G));
        }
        const int taken = who ? __ffs(who) - 1 : 0;
        const unsigned int id = __shfl_sync(full, at, lane0 + taken);
        if ((k & (G - 1)) == gl) { out_key = largest; out_id = id; }
        if ((k & (G - 1)) == G - 1 || k == a.top - 1) {
          const int i = k - (k & (G - 1)) + gl;
          if (i <= k) put(i, out_key, out_id);
        }
        if (who && taken == gl) {
#pragma unroll
          for (int i = 0; i < E + 2; ++i) if (i == (int)slot) key[i] = 0;
          find();
        }
      }
    }
  }
  if (FWD) return;
  O* const d = reinterpret_cast<O*>(a.out) + rr * a.ld_out;
  // scale * 2^(x log2 e - c) * (1 or A + B * exponent), or differences first
  float c = 0.0f, A = 0.0f, B = 0.0f, hit = 0.0f;
  bool zeros = !live, slow = far;
  if (MODE == TOK_LOSS) {
    const float f = a.scale * i0;
    zeros = zeros || z == 0.0f;
    c = shift_of(m);
    A = far ? f : f / z;
    hit = -f;
  } else {
    zeros = zeros || i0 == ninf;
    hit = i1;
    slow = !(fabsf(i0) <= LSE_EXACT);
    if (isnan(i0)) m = i0;      // as for a NaN
    if (slow) {
      A = -(i1 + i2 * i3);
      B = -i2 * LN2;
    } else {      // see token_loss.cu
      c = i0 * LOG2E;
      const float off = LOW ? fmaf(low, LOG2E, fmaf(i0, LOG2E, -c)) : fmaf(i0, LOG2E, -c), f = -exp2_of(-off);
      A = f * (i1 + i2 * (i3 - LN2 * off));
      B = f * LN2 * i2;
    }
  }
  const bool aligned = (((uintptr_t)d / sizeof(O) - ph) & (E - 1)) == 0;
  const bool any_slow = __any_sync(full, live && slow);      // (and out may be x: the row is in registers, its target has been read)
  if (!in) return;
  auto write = [&](auto with_slow) {
    auto result = [&](float2 v) {
      float2 p = fma_2(v, both(LOG2E), both(-c));
      if (with_slow.value && slow) p = make_float2(((v.x - m) - log_z) * LOG2E, ((v.y - m) - log_z) * LOG2E);
      const float2 e = make_float2(exp2_of(p.x), exp2_of(p.y));
      if (MODE == TOK_LOSS) return mul_2(e, both(A));
      return mul_2(e, fma_2(make_float2(fmaxf(p.x, -1e4f), fmaxf(p.y, -1e4f)), both(B), both(A)));      // (zero times a number; a NaN is in e)
    };
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      const int j = (gl + q * G) * E - ph;
      if (j >= a.V) continue;
      float o[E];
      TokVec<T>::get(w[q], o);
#pragma unroll
      for (int k = 0; k < E; k += 2) { const float2 v = result(make_float2(o[k], o[k + 1])); o[k] = v.x; o[k + 1] = v.y; }
      if (t >= j && t < j + E) {
#pragma unroll
        for (int k = 0; k < E; ++k) if (j + k == t) o[k] += hit;
      }
      if (zeros) {
#pragma unroll
        for (int k = 0; k < E; ++k) o[k] = 0.0f;
      }
      const bool whole = j >= 0 && j + E <= a.V;
      if (whole && aligned) {
        store_group<O, E>(d + j, o);
      } else if (whole || !split) {
#pragma unroll
        for (int k = 0; k < E; ++k) if (j + k >= 0 && j + k < a.V) d[j + k] = from_f32<O>(o[k]);
      }
    }
    if (has_h || has_t) {
      const float2 v = result(make_float2(xh, xt));
      if (has_h) d[jh] = from_f32<O>(zeros ? 0.0f : v.x + (jh == t ? hit : 0.0f));
      if (has_t) d[jt] = from_f32<O>(zeros ? 0.0f : v.y + (jt == t ? hit : 0.0f));
    }
  };
  if (any_slow) write(std::true_type{});
  else write(std::false_type{});
}

template <typename T, typename O, int MODE>
static int tok_short_go(const TokDev& d, cudaStream_t st) {
  const long long groups = tok_groups(d.V, sizeof(T));
  int lg = 0;
  while (lg < 5 && groups > 1 << lg) ++lg;
  const long long rows = groups <= 32 ? 32 >> lg : 1, blocks = (d.R + 4 * rows - 1) / (4 * rows);      // rows of a warp
  if (blocks >= (1ll << 31)) { set_error("tokens: too many rows%s", "", 0, 0); return -1; }
  auto go = [&](auto kern) { kern<<<(unsigned)blocks, 128, 0, st>>>(d, lg); };
  if constexpr (MODE == TOK_TOP) {
    go(tok_short_kernel<T, O, MODE, 1>);
  } else {
    if (groups <= 32) go(tok_short_kernel<T, O, MODE, 1>);
    else if (groups <= 128) go(tok_short_kernel<T, O, MODE, 4>);
    else go(tok_short_kernel<T, O, MODE, 8>);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) { set_error("tokens launch: %s", cudaGetErrorString(e), 0, 0); return -7; }
  return 0;
}

int tok_short(const TokDev& d, int mode, int x_bf16, int out_bf16, cudaStream_t st) {
  using B = __nv_bfloat16;
  switch (mode) {
    case TOK_LOGP: return x_bf16 ? tok_short_go<B, float, TOK_LOGP>(d, st) : tok_short_go<float, float, TOK_LOGP>(d, st);
    case TOK_ENTROPY: return x_bf16 ? tok_short_go<B, float, TOK_ENTROPY>(d, st) : tok_short_go<float, float, TOK_ENTROPY>(d, st);
    case TOK_TOP: return x_bf16 ? tok_short_go<B, float, TOK_TOP>(d, st) : tok_short_go<float, float, TOK_TOP>(d, st);
    case TOK_LOSS:
      if (x_bf16) return out_bf16 ? tok_short_go<B, B, TOK_LOSS>(d, st) : tok_short_go<B, float, TOK_LOSS>(d, st);
      return out_bf16 ? tok_short_go<float, B, TOK_LOSS>(d, st) : tok_short_go<float, float, TOK_LOSS>(d, st);
    default: {      // (a form of its own with lse_low: one more value a row spills, gradient of 16384 x 1000 f32 19.6 us, so 20.6)
      auto grad = [&](auto mode) {
        constexpr int M = mode.value;
        if (x_bf16) return out_bf16 ? tok_short_go<B, B, M>(d, st) : tok_short_go<B, float, M>(d, st);
        return out_bf16 ? tok_short_go<float, B, M>(d, st) : tok_short_go<float, float, M>(d, st);
      };
      return d.lse_low_in ? grad(std::integral_constant<int, TOK_GRAD_LOW>{}) : grad(std::integral_constant<int, TOK_GRAD>{});
    }
  }
}
}  // namespace ono
