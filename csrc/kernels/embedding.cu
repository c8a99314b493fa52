// Rows of a table looked up by token, and the table's gradient from the rows' gradients.
//
//   out[i] = scale * table[ids[i]]            grad[v] (+)= scale * sum over i with ids[i] = v of d[i]
//
// Either is bound by memory: the rows read and written, and for the gradient the whole table where it is not added to. Sums go over the tokens
// in the order of their places, so that a gradient is the same to the bit from run to run: the places are sorted by token (stable), and
// one warp adds up a run of equal tokens, or a long one's part in a chunk of the sorted places. A few hundred places are not sorted: a warp looks for those
// of its token.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "chain.cuh"
#include "ono_kernels.h"
#include "piece.cuh"
#include "ptx.cuh"

namespace ono {
void set_error(const char* fmt, const char* a, long long b, long long c);

// The lanes whose digit is this one's, of `bits` bits; digits are below 2^bits, lanes without one give 2^bits.
__device__ __forceinline__ unsigned int same_digit(unsigned int digit, int bits) {
  unsigned int peers = 0xffffffffu;
#pragma unroll
  for (int b = 0; b < 10; ++b) {
    if (b > bits) break;
    const bool one = digit >> b & 1u;
    const unsigned int ones = __ballot_sync(0xffffffffu, one);
    peers &= one ? ones : ~ones;
  }
  return peers;
}

// The row an id stands for, -1 for none.
template <typename I>
__device__ __forceinline__ long long token_row(I id, int vocab, long long padding_id, int* status) {
  if ((long long)id == padding_id) return -1;
  if (id >= 0 && id < vocab) return (long long)id;
  if (status) atomicExch(status, ONO_ERR_BAD_ARG);
  return -1;
}

// ------------------------------------------------------------------------------------------------
// Lookup: a warp takes 32 * EMB_LOADS groups of VEC values of a row, or several rows where one has fewer groups than lanes.
// ------------------------------------------------------------------------------------------------
// Loads to a lane: more of them leave fewer warps, each of which waits for its row's number first. Us: eight values a load, two against four: 141, 137
// (131072 x 2048 bf16), but 2.4, 2.9 (8 x 4096); four values, two, four, eight: 251, 204, 201 (131072 x 2048 bf16 to f32), but 21.0 and 21.5 of the last
// two (30000 x 700 f32); values one by one, four, eight, sixteen: 78, 60, 50 (100000 x 517 f32 to bf16), 80, 60, 64 (bf16), 33, 22, 30 (91538 x 179). A row's loads
// are shared out evenly over its warps (517: six, six and five a lane, and not eight, eight and one; f32 to bf16 55.6).
template <typename TO> constexpr int EMB_VEC = 16 / sizeof(TO);      // values of a 16-byte store
template <int VEC> constexpr int EMB_LOADS = VEC == 1 ? 8 : VEC == 4 ? 4 : 2;
// BYTES of a row in as few accesses as there can be.
template <int BYTES> struct Words {
  using Word = std::conditional_t<BYTES == 2, unsigned short, std::conditional_t<BYTES == 4, unsigned int, std::conditional_t<BYTES == 8, uint2, uint4>>>;
  static constexpr int N = BYTES / (int)sizeof(Word);
  Word w[N];
};

template <typename TI, typename TO, int VEC, typename I>
__global__ void __launch_bounds__(256) embedding_kernel(const OnoEmbedding e, int groups, int segs, int per, int lanes) {
  constexpr int U = EMB_LOADS<VEC>;
  const long long job = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  // lanes: log2 of those that a row takes
  const long long i = lanes < 5 ? job * (32 >> lanes) + (lane >> lanes) : job / segs;
  if (i >= e.n) return;
  const int first = lanes < 5 ? 0 : (int)(job - i * segs) * 32 * per, end = min(groups, first + 32 * per);
  const int g0 = first + (lanes < 5 ? lane & ((1 << lanes) - 1) : lane);
  const long long row = token_row(reinterpret_cast<const I*>(e.ids)[i], e.vocab, e.padding_id, e.status);
  const TI* src = reinterpret_cast<const TI*>(e.table) + (row < 0 ? 0 : row) * e.ld_table;
  TO* dst = reinterpret_cast<TO*>(e.out) + i * e.ld_out;
  // Values are kept as they came until all loads are under way: converted where they are loaded, each would be waited for by itself
  // (100000 x 517 f32 to bf16 74 us, so 57; bf16 96 against 62).
  using In = Words<VEC * (int)sizeof(TI)>;
  In w[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int g = g0 + 32 * u;
    const TI* const at = src + (long long)g * VEC;
    if (row < 0 || g >= end) continue;
    if (VEC > 1 && (g + 1) * VEC > e.width) {
      TI* const t = reinterpret_cast<TI*>(&w[u]);
#pragma unroll
      for (int k = 0; k < VEC; ++k) t[k] = g * VEC + k < e.width ? at[k] : from_f32<TI>(0.0f);
    } else {
#pragma unroll
      for (int k = 0; k < In::N; ++k) w[u].w[k] = __ldg(reinterpret_cast<const typename In::Word*>(at) + k);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int g = g0 + 32 * u;
    if (g >= end) continue;
    using Out = Words<VEC * (int)sizeof(TO)>;
    Out o;
    const TI* const t = reinterpret_cast<const TI*>(&w[u]);
    TO* const q = reinterpret_cast<TO*>(&o);
#pragma unroll
    for (int k = 0; k < VEC; ++k) q[k] = from_f32<TO>(row < 0 ? 0.0f : to_f32(t[k]) * e.scale);
    TO* const to = dst + (long long)g * VEC;
    if (VEC > 1 && (g + 1) * VEC > e.width) {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (g * VEC + k < e.width) to[k] = q[k];
    } else {
#pragma unroll
      for (int k = 0; k < Out::N; ++k) reinterpret_cast<typename Out::Word*>(to)[k] = o.w[k];
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Gradient. The places are sorted by token (stable), while other CTAs of the same launches fill the table with zeros. One launch ranks them, or one counts digits and
// one to four sort by them; then embedding_sum_kernel, and embedding_join_kernel for runs of several chunks. For very few places embedding_few_kernel does all of it.
// ------------------------------------------------------------------------------------------------
struct GradDev {
  OnoEmbeddingGrad e;
  uint2* item[2];                      // token and place, ping and pong
  unsigned int* hist;                  // [3][tiles][SORT_RADIX]: of a pass, the next and the one after it, in turn
  unsigned int* runs;                  // number of long runs, then their first and last chunks
  float* part;                         // [chunks][2][pitch]
  int sorted;                          // which of `item` holds the result
  int chunk, pitch;
  int bits, tile, tiles;               // radix sort: bits a pass, places of a CTA, CTAs
  int zero;                            // values of a CTA that fills the table with zeros (a multiple of 4)
};

// Zeros for the CTAs behind the first ones of a launch: of the table's values, `zero` to a CTA, or of whole rows that many values long, value by value, where
// the table does not begin at 16 bytes (gradient of 16384 x 1024 of 50257: 68.5 us against 67.6).
constexpr int ZERO_VALUES = 1 << 16, ZERO_LEAST = 2048;
__device__ __forceinline__ void fill_zeros(const GradDev& p, long long cta) {
  const OnoEmbeddingGrad& e = p.e;
  const int threads = (int)blockDim.x;
  if (e.ld_grad == e.width && ((uintptr_t)e.grad & 15) == 0) {
    const long long all = (long long)e.vocab * e.width, end = min(all, (cta + 1) * p.zero);
    for (long long i = cta * p.zero + 4 * threadIdx.x; i < end; i += 4 * threads) {
      if (i + 4 <= all) *reinterpret_cast<float4*>(e.grad + i) = make_float4(0.f, 0.f, 0.f, 0.f);
      else for (long long k = i; k < all; ++k) e.grad[k] = 0.0f;
    }
  } else {
    const long long rows = (p.zero + e.width - 1) / e.width, end = min((long long)e.vocab, (cta + 1) * rows);
    for (long long v = cta * rows + (threadIdx.x >> 5); v < end; v += threads >> 5)
      for (int k = threadIdx.x & 31; k < e.width; k += 32) e.grad[v * e.ld_grad + k] = 0.0f;
  }
}
// A small table is shared out over four CTAs an SM, of a large one a CTA takes `most` values (gradient of 30 x 64 of 1000 rows, with 16384 a CTA 10.0 us,
// so 3.6; of 9625 x 389 of 2135 with 65536 29.8, 26.7).
static int zero_share(const OnoEmbeddingGrad& e, int most) {
  const long long even = ((long long)e.vocab * e.width / (4 * ono_num_sms()) + 3) / 4 * 4;
  return (int)std::min<long long>(most, std::max<long long>(ZERO_LEAST, even));
}
static long long zero_ctas(const OnoEmbeddingGrad& e, int share) {
  if (e.accumulate) return 0;
  if (e.ld_grad == e.width && ((uintptr_t)e.grad & 15) == 0) return ((long long)e.vocab * e.width + share - 1) / share;
  const long long rows = (share + e.width - 1) / e.width;
  return (e.vocab + rows - 1) / rows;
}

// The token of a place; `vocab`, behind all of them, where there is none.
template <typename I>
__device__ __forceinline__ unsigned int token_key(const OnoEmbeddingGrad& e, unsigned int j) {
  const long long r = token_row(__ldg(reinterpret_cast<const I*>(e.ids) + j), e.vocab, e.padding_id, e.status);
  return r < 0 ? (unsigned int)e.vocab : (unsigned int)r;
}

// Few places: each finds its rank by comparing with all of them, RANK_THREADS threads a place. One launch, no pass waits for another. (Us, the gradient by
// ranks against the radix sort: 2000 x 64 12.3, 13.8; 1500 x 256 18.0, 24.0; 3000 x 64 15.4, 14.2; 4096 x 1024 49.2, 46.3. Eight threads a place: 4096 52.2.)
constexpr int RANK_MAX = 2048, RANK_THREADS = 16, RANK_PLACES = 256 / RANK_THREADS;
template <typename I>
__global__ void __launch_bounds__(256) embedding_rank_kernel(const __grid_constant__ GradDev p, int ctas) {
  __shared__ __align__(16) unsigned int s_key[RANK_MAX];
  const OnoEmbeddingGrad& e = p.e;
  if ((int)blockIdx.x >= ctas) { fill_zeros(p, blockIdx.x - ctas); return; }
  const int n = (int)e.n, nv = (n + 3) / 4;
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.runs = 0;
#pragma unroll
  for (int q = 0; q < RANK_MAX / 256; ++q) {      // (all loads at once)
    const int j = threadIdx.x + q * 256;
    if (j < 4 * nv) s_key[j] = j < n ? token_key<I>(e, j) : 0xffffffffu;
  }
  __syncthreads();
  const int i = blockIdx.x * RANK_PLACES + threadIdx.x / RANK_THREADS, part = threadIdx.x % RANK_THREADS;
  const uint4* keys = reinterpret_cast<const uint4*>(s_key);
  unsigned int rank = 0, key = 0;
  if (i < n) {
    key = s_key[i];
    const int vi = i >> 2;
#pragma unroll 4
    for (int v = part; v < vi; v += RANK_THREADS) { const uint4 k = keys[v]; rank += (k.x <= key) + (k.y <= key) + (k.z <= key) + (k.w <= key); }
#pragma unroll 4
    for (int v = vi + 1 + part; v < nv; v += RANK_THREADS) { const uint4 k = keys[v]; rank += (k.x < key) + (k.y < key) + (k.z < key) + (k.w < key); }
    if (part < 4) {
      const unsigned int k = s_key[4 * vi + part];
      rank += k < key || (k == key && 4 * vi + part < i);
    }
  }
#pragma unroll
  for (int o = RANK_THREADS / 2; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
  if (i < n && part == 0) p.item[p.sorted][rank] = make_uint2(key, (unsigned int)i);
}

// Many: a radix sort, `bits` (at most 9) of the token a pass. A CTA has a tile of the places, its warps runs of it; a warp goes through its
// own 32 at a time, lanes of one digit finding each other by a vote on every bit (match.any takes longer the more digits there are:
// 131072 places 74 us, so 62). Positions are sums of counts: over the warps, over the tiles before (each CTA adds them up itself) and
// over the digits. The first launch counts; every pass then counts for the next one where its places go to.
constexpr int SORT_THREADS = 512, SORT_WARPS = SORT_THREADS / 32, SORT_BITS = 9, SORT_RADIX = 1 << SORT_BITS, SORT_BATCH = 2;
constexpr int SORT_TILE = SORT_THREADS * SORT_BATCH, SORT_TILES = 128;      // places of a CTA, or as many times that as leave SORT_TILES of them
// (a CTA adds up the counts of all: 131072 x 256 in 256 tiles 61.9 us, in 128 59.9, in 64 59.3, but then 600000 x 64 150 against 136)
static_assert(SORT_THREADS == SORT_RADIX, "a thread for each digit");

template <typename I>
__global__ void __launch_bounds__(SORT_THREADS) embedding_count_kernel(const __grid_constant__ GradDev p, long long zero) {
  __shared__ unsigned int s_count[SORT_RADIX];
  const OnoEmbeddingGrad& e = p.e;
  if ((int)blockIdx.x >= p.tiles) { fill_zeros(p, zero + blockIdx.x - p.tiles); return; }
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.runs = 0;
  s_count[threadIdx.x] = 0;
  unsigned int* const mine = p.hist + blockIdx.x * SORT_RADIX + threadIdx.x;
  mine[p.tiles * SORT_RADIX] = 0;
  __syncthreads();
  const long long j0 = (long long)blockIdx.x * p.tile, end = min(e.n, j0 + p.tile);
#pragma unroll 8
  for (long long j = j0 + threadIdx.x; j < end; j += SORT_THREADS) atomicAdd(&s_count[token_key<I>(e, (unsigned int)j) & ((1u << p.bits) - 1)], 1u);
  __syncthreads();
  *mine = s_count[threadIdx.x];
}

template <typename I>
__global__ void __launch_bounds__(SORT_THREADS) embedding_scatter_kernel(const __grid_constant__ GradDev p, int pass, int last, long long zero) {
  __shared__ unsigned int s_count[SORT_WARPS][SORT_RADIX], s_base[SORT_RADIX], s_sum[SORT_WARPS];
  const OnoEmbeddingGrad& e = p.e;
  if ((int)blockIdx.x >= p.tiles) { fill_zeros(p, zero + blockIdx.x - p.tiles); return; }      // (nothing ahead in the chain touches the table)
  chain_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int shift = pass * p.bits;
  const unsigned int mask = (1u << p.bits) - 1, below = (1u << lane) - 1u;
  const uint2* in = p.item[(pass + 1) & 1];
  uint2* out = p.item[pass & 1];
  const unsigned int* hist = p.hist + pass % 3 * p.tiles * SORT_RADIX;
  unsigned int* next = p.hist + (pass + 1) % 3 * p.tiles * SORT_RADIX;
  p.hist[((pass + 2) % 3 * p.tiles + blockIdx.x) * SORT_RADIX + tid] = 0;
  const long long begin = (long long)blockIdx.x * p.tile + (long long)warp * (p.tile / SORT_WARPS);
  const long long end = min(e.n, begin + p.tile / SORT_WARPS);
  uint2 it[SORT_BATCH];
  auto items_from = [&](long long j0) {
#pragma unroll
    for (int b = 0; b < SORT_BATCH; ++b) {
      const long long j = j0 + 32 * b + lane;
      if (j < end) it[b] = pass ? __ldcg(in + j) : make_uint2(token_key<I>(e, (unsigned int)j), (unsigned int)j);
    }
  };
  items_from(begin);
  for (int k = lane; k < SORT_RADIX; k += 32) s_count[warp][k] = 0;
  __syncwarp();
  for (long long j0 = begin; j0 < end; j0 += 32 * SORT_BATCH) {
    if (j0 != begin) items_from(j0);
#pragma unroll
    for (int b = 0; b < SORT_BATCH; ++b)
      if (j0 + 32 * b + lane < end) atomicAdd(&s_count[warp][it[b].x >> shift & mask], 1u);
  }
  // a digit a thread: its places in the tiles before, and in all
  unsigned int before = 0, all = 0;
#pragma unroll 16
  for (int t = 0; t < p.tiles; ++t) {
    const unsigned int h = __ldcg(hist + t * SORT_RADIX + tid);
    if (t < (int)blockIdx.x) before += h;
    all += h;
  }
  unsigned int run = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const unsigned int v = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run += v; }
  if (lane == 31) s_sum[warp] = run;
  __syncthreads();
  unsigned int lower = 0;
#pragma unroll
  for (int w = 0; w < SORT_WARPS; ++w) if (w < warp) lower += s_sum[w];
  s_base[tid] = lower + run - all + before;
  unsigned int sum = 0;
#pragma unroll
  for (int w = 0; w < SORT_WARPS; ++w) { const unsigned int c = s_count[w][tid]; s_count[w][tid] = sum; sum += c; }
  __syncthreads();
  for (long long j0 = begin; j0 < end; j0 += 32 * SORT_BATCH) {
    if (end - begin > 32 * SORT_BATCH) items_from(j0);      // (else they are still here)
#pragma unroll
    for (int b = 0; b < SORT_BATCH; ++b) {
      const long long j = j0 + 32 * b + lane;
      if (j0 + 32 * b >= end) break;
      const unsigned int digit = j < end ? it[b].x >> shift & mask : mask + 1;
      const unsigned int peers = same_digit(digit, p.bits);
      unsigned int at = 0;
      if (j < end) at = s_base[digit] + s_count[warp][digit] + __popc(peers & below);
      __syncwarp();
      if (j < end) {
        if ((peers & below) == 0) s_count[warp][digit] += __popc(peers);
        out[at] = it[b];      // (token and place in one store: scattered ones take a cycle a place)
        if (!last) atomicAdd(&next[at / (unsigned int)p.tile * SORT_RADIX + (it[b].x >> (shift + p.bits) & mask)], 1u);
      }
      __syncwarp();
    }
  }
}

// embedding_sum_kernel: a warp adds up the rows of a chunk of `chunk` sorted places, 32 * VEC columns of them. A run of equal tokens belongs to
// the chunk it starts in, whose warp follows it into the next chunk if it ends there. A longer run is summed chunk by chunk: part[c][1]
// has the sum of what starts in c, part[c][0] of what comes from before; embedding_join_kernel adds them in order.
// A lane's values of a row: VEC of them, one behind the other (STEP 1, where rows are aligned) or every 32nd (STEP 32). `left`: columns from the first
// of them on.
template <typename T, int VEC, int STEP>
struct RowPart {
  static constexpr int WORDS = STEP == 1 ? 4 : VEC;
  uint32_t w[WORDS];
  // As they lie in memory: a conversion here would wait for each row by itself (a gradient of 9916 x 3509 bf16: 102 us, so 57).
  static __device__ __forceinline__ uint32_t bits(const T* p) {
    if constexpr (sizeof(T) == 2) return __ldg(reinterpret_cast<const unsigned short*>(p)); else return __ldg(reinterpret_cast<const unsigned int*>(p));
  }
  static __device__ __forceinline__ int column(int tile, int lane) { return tile * 32 * VEC + (STEP == 1 ? lane * VEC : lane); }
  __device__ __forceinline__ void load(const T* p, int left) {
    if constexpr (STEP == 1) {
      static_assert(VEC * sizeof(T) == 16, "16 bytes");
      if (left >= VEC) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
      } else {
        T* t = reinterpret_cast<T*>(w);
#pragma unroll
        for (int k = 0; k < VEC; ++k) t[k] = k < left ? p[k] : from_f32<T>(0.0f);
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) w[k] = k * STEP < left ? bits(p + k * STEP) : 0u;
    }
  }
  __device__ __forceinline__ void add_to(float (&acc)[VEC]) const {
    if constexpr (STEP == 1) {
      add_piece<T, VEC>(acc, make_uint4(w[0], w[1], w[2], w[3]));
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += __uint_as_float(sizeof(T) == 2 ? w[k] << 16 : w[k]);
    }
  }
};
template <int VEC, int STEP>
struct GradVec {      // the same of an f32 row; 16-byte accesses where it is aligned and the lane's columns are all there
  static __device__ __forceinline__ void load(float (&v)[VEC], const float* p, int left, bool aligned) {
    if (STEP == 1 && aligned && left >= VEC) {
#pragma unroll
      for (int k = 0; k < VEC; k += 4) { const float4 w = *reinterpret_cast<const float4*>(p + k); v[k] = w.x; v[k + 1] = w.y; v[k + 2] = w.z; v[k + 3] = w.w; }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = k * STEP < left ? p[k * STEP] : 0.0f;
    }
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[VEC], int left, bool aligned) {
    if (STEP == 1 && aligned && left >= VEC) {
#pragma unroll
      for (int k = 0; k < VEC; k += 4) *reinterpret_cast<float4*>(p + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) if (k * STEP < left) p[k * STEP] = v[k];
    }
  }
};

// U rows are in flight; with ACC those of the table that they are added to as well. (Eight values a lane are many registers: fewer rows, more warps. Us,
// eight rows, four: 131072 x 512 of 200 tokens 58.0, 53.3, 16384 x 1024 58.9, 57.1, 131072 x 2048 318, 321; with ACC four, two in four blocks:
// 131072 x 2048 257.6, 251.4, 131072 x 512 73.6, 62.9, although the four blocks' 64 registers spill 64 bytes: of many tokens three blocks, without, take 262 against 253
// and 101 against 95. Four values: 60000 x 1024 f32 with ACC four, two 105.8, 112.3, without eight, four 122.0, 124.2.)
template <typename T, int VEC, int STEP, bool ACC, int U>
__global__ void __launch_bounds__(256, U == 2 ? 4 : 1) embedding_sum_kernel(const __grid_constant__ GradDev p, int tiles) {
  const OnoEmbeddingGrad& e = p.e;
  chain_wait();
  const unsigned int n = (unsigned int)e.n, L = (unsigned int)p.chunk, none = (unsigned int)e.vocab;
  const uint2* const item = p.item[p.sorted];
  const long long job = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const unsigned int c = (unsigned int)(job / tiles);
  const int tile = (int)(job - (long long)c * tiles), col = RowPart<T, VEC, STEP>::column(tile, lane), left = e.width - col;
  const bool aligned = (((uintptr_t)e.grad | (uintptr_t)(e.ld_grad * 4)) & 15) == 0;
  if ((unsigned long long)c * L >= n) return;
  const unsigned int s = c * L, own = min(n, s + L);
  unsigned int end = own;
  const unsigned int k0 = item[s].x, kl = item[own - 1].x, kb = s > 0 ? item[s - 1].x : none, ke = own < n ? item[own].x : none;
  if (k0 == none) return;
  const bool from_before = s > 0 && kb == k0, goes_on = own < n && ke == kl;
  unsigned int at = s;
  if (from_before) {
    const bool just_before = s == L || item[s - L].x != k0 || item[s - L - 1].x != k0;      // it starts in the chunk before
    const bool is_long = s + L <= n && kl == k0;                                           // and fills this one, so that all of it goes by chunks
    if (just_before && !is_long) {                                                         // that chunk's warp finishes it
      if (kl == k0) return;
      for (bool found = false; !found; ) {
        const unsigned int j = at + lane;
        const unsigned int other = __ballot_sync(0xffffffffu, j < own && item[min(j, own - 1)].x != k0);
        found = other != 0;
        at += found ? __ffs(other) - 1 : 32;
      }
    }
  }
  const bool head = from_before && at == s;      // a piece of a run that started earlier
  bool tail_long = false;
  if (goes_on && !(head && kl == k0) && kl != none) {
    tail_long = own + L <= n && item[own + L - 1].x == kl;      // the run fills the next chunk
    if (!tail_long) {
      end = min(n, own + L);      // this warp finishes it; it stops at the next token
    } else if (tile == 0) {       // where it ends: the last place of token kl, 32 probes at a time
      unsigned int lo = own + L - 1, hi = n;      // key[lo] == kl, key[hi] != kl or hi == n
      while (hi - lo > 1) {
        const unsigned int step = (hi - lo + 31) / 32, j = lo + step * (lane + 1);
        const unsigned int same = __popc(__ballot_sync(0xffffffffu, j < hi && item[min(j, n - 1)].x == kl));
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
      GradVec<VEC, STEP>::store(p.part + ((long long)c * 2 + (piece ? 0 : 1)) * p.pitch + col, acc, left, true);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = ACC ? old[k] + e.scale * acc[k] : e.scale * acc[k];
      GradVec<VEC, STEP>::store(e.grad + (long long)cur * e.ld_grad + col, acc, left, aligned);
    }
  };
  for (unsigned int j0 = at; j0 < end; j0 += 32) {
    const unsigned int j = j0 + lane;
    const uint2 ij = j < end ? item[j] : make_uint2(none, 0u);
    const unsigned int kj = ij.x, pj = ij.y;
    const int m = (int)min(32u, end - j0);
    for (int q0 = 0; q0 < m; q0 += U) {
      RowPart<T, VEC, STEP> w[U];
      float was[ACC ? U : 1][VEC];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int q = q0 + u;
        const unsigned int k = __shfl_sync(0xffffffffu, kj, q & 31), from = __shfl_sync(0xffffffffu, pj, q & 31);
        const unsigned int kp = __shfl_sync(0xffffffffu, kj, (q - 1) & 31);
        if (q < m && k != none && left > 0) {
          w[u].load(reinterpret_cast<const T*>(e.d) + (long long)from * e.ld_d + col, left);
          if (ACC && (q == 0 || kp != k)) GradVec<VEC, STEP>::load(was[ACC ? u : 0], e.grad + (long long)k * e.ld_grad + col, left, aligned);
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
        if (left > 0) w[u].add_to(acc);
      }
    }
  }
  flush(true);
}

// Very few places: no sorting. A warp takes a place and 32 * VEC columns, looks for the place's token among all, and where the place is the
// token's first adds up its rows, U in flight. The other CTAs fill the rows of the table that no token means with zeros. One launch.
constexpr int FEW_MAX = 512, FEW_VALUES = 1 << 14;      // FEW_VALUES: zeros of a CTA, at most
// Where a token has FEW_RUN places and more on average, a warp would go through too many alone: ranks. (Us, this form against ranks: 500 places of 2 tokens, 64
// columns, 38.9, 9.4; of 20 11.4, 9.9; of 100 8.7, 9.9; 100 of 5 5.9, 9.1; 300 of 50000, 256 columns, 11.9, 18.1. With FEW_MAX 1024: 1000 of 50000 15.5,
// 18.8, but of 100 15.2, 10.8.)
constexpr int FEW_RUN = 24;
static bool grad_few(long long n, int vocab) { return n > 0 && n <= FEW_MAX && n <= (long long)FEW_RUN * vocab; }
template <typename T, int VEC, int STEP, typename I>
__global__ void __launch_bounds__(256) embedding_few_kernel(const OnoEmbeddingGrad e, int tiles, int ctas, int rows) {
  constexpr int U = STEP == 1 ? 16 : 8, WORDS = FEW_MAX / 32;
  __shared__ unsigned int s_word[8 * FEW_MAX / 2];      // rows with a token, or the warps' lists of 16 bits a place
  static_assert(FEW_VALUES / 32 + 1 <= 8 * FEW_MAX / 2, "a bit for each of a CTA's rows");
  const I* ids = reinterpret_cast<const I*>(e.ids);
  const int n = (int)e.n, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool aligned = (((uintptr_t)e.grad | (uintptr_t)(e.ld_grad * 4)) & 15) == 0;
  if ((int)blockIdx.x >= ctas) {
    const long long cta = blockIdx.x - ctas;
    const long long first = cta * rows;
    const int mine = (int)min((long long)rows, e.vocab - first);
    for (int k = threadIdx.x; k <= mine / 32; k += 256) s_word[k] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += 256) {
      const long long r = token_row(ids[j], e.vocab, e.padding_id, nullptr) - first;
      if (r >= 0 && r < mine) atomicOr(&s_word[r >> 5], 1u << (r & 31));
    }
    __syncthreads();
    auto met = [&](int r) { return s_word[r >> 5] >> (r & 31) & 1u; };
    float* const g = e.grad + first * e.ld_grad;
    if (e.width >= 64) {      // a warp a row
      for (int r = warp; r < mine; r += 8) {
        if (met(r)) continue;
        float* const row = g + (long long)r * e.ld_grad;
        const int head = min(e.width, (int)((16 - ((uintptr_t)row & 15)) & 15) / 4), body = head + ((e.width - head) & ~3);
        if (lane < head) row[lane] = 0.0f;
        for (int k = head + 4 * lane; k < body; k += 128) *reinterpret_cast<float4*>(row + k) = make_float4(0.f, 0.f, 0.f, 0.f);
        if (lane < e.width - body) row[body + lane] = 0.0f;
      }
    } else {      // a thread a value
      for (int k = threadIdx.x; k < mine * e.width; k += 256) {
        const int r = k / e.width;
        if (!met(r)) g[(long long)r * e.ld_grad + k - r * e.width] = 0.0f;
      }
    }
    return;
  }
  const long long job = (long long)blockIdx.x * 8 + warp;
  const int i = (int)(job / tiles), col = RowPart<T, VEC, STEP>::column((int)(job - (long long)i * tiles), lane), left = e.width - col;
  if (i >= n) return;
  const I id = ids[i];
  unsigned int same[WORDS];
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    const int j = 32 * w + lane;
    const bool eq = j < n && ids[min(j, n - 1)] == id;
    same[w] = 32 * w < n ? __ballot_sync(0xffffffffu, eq) : 0u;
  }
  const long long row = token_row(id, e.vocab, e.padding_id, e.status);
  if (row < 0) return;
  unsigned short* const list = reinterpret_cast<unsigned short*>(s_word) + warp * FEW_MAX;
  int count = 0;
  bool first = true;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    if (32 * w < i && (32 * w + 32 <= i ? same[w] : same[w] & ((1u << (i & 31)) - 1u))) first = false;
    if (same[w] >> lane & 1u) list[count + __popc(same[w] & ((1u << lane) - 1u))] = (unsigned short)(32 * w + lane);
    count += __popc(same[w]);
  }
  if (!first) return;
  __syncwarp();
  if (left <= 0) return;
  float* const g = e.grad + row * e.ld_grad + col;
  float acc[VEC], old[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
  if (e.accumulate) GradVec<VEC, STEP>::load(old, g, left, aligned);
  for (int q0 = 0; q0 < count; q0 += U) {
    RowPart<T, VEC, STEP> w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (q0 + u < count) w[u].load(reinterpret_cast<const T*>(e.d) + (long long)list[q0 + u] * e.ld_d + col, left);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (q0 + u < count) w[u].add_to(acc);
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = e.accumulate ? old[k] + e.scale * acc[k] : e.scale * acc[k];
  GradVec<VEC, STEP>::store(g, acc, left, aligned);
}

// embedding_join_kernel: a block takes a long run's sums, 32 * VEC columns of them; its warps every JOIN_WARPS-th, then one adds up theirs.
// (Eight of them: 60000 x 256 of 1000 tokens 45.8 us against 42.6; 32: 9916 x 3509 58.0 against 56.2, but 600000 x 64 132 against 136.)
constexpr int JOIN_WARPS = 16;
template <int VEC>
__global__ void __launch_bounds__(32 * JOIN_WARPS) embedding_join_kernel(const __grid_constant__ GradDev p, int tiles) {
  __shared__ float s_sum[JOIN_WARPS][32 * VEC];
  const OnoEmbeddingGrad& e = p.e;
  chain_wait();
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
      for (unsigned int q = c + warp; q <= c1; q += JOIN_WARPS) {
        float v[VEC];
        GradVec<VEC, 1>::load(v, p.part + ((long long)q * 2 + (q == c ? 1 : 0)) * p.pitch + col, VEC, true);      // (a row of sums is whole groups)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += v[k];
      }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) s_sum[warp][lane * VEC + k] = acc[k];
    __syncthreads();
    if (warp == 0 && left > 0) {
      float* g = e.grad + (long long)p.item[p.sorted][c * L + L - 1].x * e.ld_grad + col;
      float old[VEC];
      if (e.accumulate) GradVec<VEC, 1>::load(old, g, left, aligned);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float t = 0.0f;
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; ++w) t += s_sum[w][lane * VEC + k];
        acc[k] = e.accumulate ? old[k] + e.scale * t : e.scale * t;
      }
      GradVec<VEC, 1>::store(g, acc, left, aligned);
    }
    __syncthreads();
  }
}

// Places to a chunk: as many as leave enough warps to fill the GPU (a lane has U rows in flight whatever the chunk), fewer warps for short chunks.
// Us, 64 a multiprocessor for every length: 131072 x 2048 268 against 255, 16384 x 1024 of 500 tokens 31 against 28; 128: 131072 x 256 79 against 62.
constexpr int CHUNK_MIN = 8, CHUNK_MAX = 512;
static long long chunk_least(int L, int width) {      // the fewest places that take chunks of L, or longer ones
  const long long tiles = (width + 127) / 128, warps = (L > 64 ? 128 : L > 32 ? 64 : 32) * 148;
  return L == CHUNK_MIN ? 0 : (warps + tiles - 1) / tiles * L;
}
static int grad_chunk(long long n, int width) {
  int L = CHUNK_MAX;
  while (n < chunk_least(L, width)) L >>= 1;
  return L;
}

struct GradScratch { long long items, hist, runs, part, bytes; int chunk, pitch, tile, tiles; };
static GradScratch grad_scratch(long long n, int width) {
  GradScratch g;
  g.chunk = grad_chunk(n, width);
  g.pitch = (width + 3) / 4 * 4;
  const long long chunks = (n + g.chunk - 1) / g.chunk;
  g.items = (n * 8 + 15) / 16 * 16;
  g.tile = SORT_TILE * (int)((n + (long long)SORT_TILE * SORT_TILES - 1) / ((long long)SORT_TILE * SORT_TILES));
  g.tiles = n > RANK_MAX ? (int)((n + g.tile - 1) / g.tile) : 0;
  g.hist = 2 * g.items;
  g.runs = g.hist + 3ll * g.tiles * SORT_RADIX * 4;
  g.part = g.runs + ((2 + 2 * chunks) * 4 + 15) / 16 * 16;
  g.bytes = g.part + chunks * 2 * g.pitch * 4;
  return g;
}

// Enough for n places and for any fewer: shorter chunks, and shorter tiles of the sort, of fewer places may be more of them.
static long long grad_scratch_up_to(long long n, int width) {
  const GradScratch g = grad_scratch(n, width);
  long long chunks = 0, most = n;
  for (int L = CHUNK_MAX; L >= CHUNK_MIN; L >>= 1) {
    const long long least = chunk_least(L, width);
    if (most < least || most < 0) continue;
    chunks = std::max(chunks, (most + L - 1) / L);
    most = least - 1;
  }
  const long long tiles = n > RANK_MAX ? std::min<long long>(SORT_TILES, (n + SORT_TILE - 1) / SORT_TILE) : 0;
  return 2 * g.items + 3 * tiles * SORT_RADIX * 4 + ((2 + 2 * chunks) * 4 + 15) / 16 * 16 + chunks * 2 * g.pitch * 4;
}

template <typename TI, typename TO, int VEC, typename I>
static int embedding_go(const OnoEmbedding& e, cudaStream_t st) {
  const int groups = (e.width + VEC - 1) / VEC, segs = (groups + 32 * EMB_LOADS<VEC> - 1) / (32 * EMB_LOADS<VEC>);
  const int per = ((groups + 31) / 32 + segs - 1) / segs;      // loads of a lane, the same of every warp
  int lanes = 5;
  while (lanes > 0 && groups <= 1 << (lanes - 1)) --lanes;
  const long long jobs = lanes < 5 ? (e.n + (32 >> lanes) - 1) / (32 >> lanes) : e.n * segs, blocks = (jobs + 7) / 8;
  if (blocks >= (1ll << 31)) { set_error("embedding: too many values%s", "", 0, 0); return -1; }
  embedding_kernel<TI, TO, VEC, I><<<(unsigned)blocks, 256, 0, st>>>(e, groups, segs, per, lanes);
  const cudaError_t r = cudaGetLastError();
  if (r != cudaSuccess) { set_error("embedding launch: %s", cudaGetErrorString(r), 0, 0); return -7; }
  return 0;
}
template <typename TI, typename TO>
static int embedding_go(const OnoEmbedding& e, cudaStream_t st) {
  constexpr int VEC = EMB_VEC<TO>, I = VEC * (int)sizeof(TI) < 16 ? VEC * (int)sizeof(TI) : 16;
  const bool vec = (uintptr_t)e.table % I == 0 && e.ld_table * (long long)sizeof(TI) % I == 0 && (uintptr_t)e.out % 16 == 0 && e.ld_out * (long long)sizeof(TO) % 16 == 0;
  if (e.ids64) return vec ? embedding_go<TI, TO, VEC, long long>(e, st) : embedding_go<TI, TO, 1, long long>(e, st);
  return vec ? embedding_go<TI, TO, VEC, int>(e, st) : embedding_go<TI, TO, 1, int>(e, st);
}
}  // namespace ono

using namespace ono;

extern "C" int ono_embedding(const OnoEmbedding* e, ono_stream_t stream) {
  if (!e || e->n < 0 || e->vocab <= 0 || e->vocab > ONO_DIM_MAX || e->width <= 0 || e->width > ONO_DIM_MAX || e->ld_table < e->width || e->ld_out < e->width || (e->n && (!e->table || !e->ids || !e->out))) {
    set_error("bad embedding args%s", "", 0, 0);
    return -1;
  }
  if (e->n == 0) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  using B = __nv_bfloat16;
  if (e->table_bf16) return e->out_bf16 ? embedding_go<B, B>(*e, st) : embedding_go<B, float>(*e, st);
  return e->out_bf16 ? embedding_go<float, B>(*e, st) : embedding_go<float, float>(*e, st);
}

extern "C" long long ono_embedding_grad_scratch(long long n, int vocab, int width) {
  return n < 0 || vocab <= 0 || vocab > ONO_DIM_MAX || width <= 0 || width > ONO_DIM_MAX ? -1 : n == 0 || grad_few(n, vocab) ? 0 : grad_scratch_up_to(n, width);
}

extern "C" int ono_embedding_grad(const OnoEmbeddingGrad* e, ono_stream_t stream) {
  if (!e || e->n < 0 || e->n > (1ll << 31) - 65536 || e->vocab <= 0 || e->vocab > ONO_DIM_MAX || e->width <= 0 || e->width > ONO_DIM_MAX || e->ld_d < e->width || e->ld_grad < e->width || !e->grad ||
      (e->n && (!e->d || !e->ids))) {
    set_error("bad embedding_grad args%s", "", 0, 0);
    return -1;
  }
  const GradScratch g = grad_scratch(e->n, e->width);
  const bool few_places = grad_few(e->n, e->vocab);
  if (e->n > 0 && !few_places && (!e->scratch || e->scratch_bytes < g.bytes || ((uintptr_t)e->scratch & 15))) { set_error("embedding_grad: scratch of %s%lld bytes, 16-byte aligned", "", g.bytes, 0); return -1; }
  if (e->n == 0 && e->accumulate) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  GradDev p = {};
  p.e = *e;
  char* at = reinterpret_cast<char*>(e->scratch);
  for (int k = 0; k < 2; ++k) p.item[k] = reinterpret_cast<uint2*>(at + k * g.items);
  p.hist = reinterpret_cast<unsigned int*>(at + g.hist);
  p.runs = reinterpret_cast<unsigned int*>(at + g.runs);
  p.part = reinterpret_cast<float*>(at + g.part);
  p.chunk = g.chunk;
  p.pitch = g.pitch;
  const int esz = e->d_bf16 ? 2 : 4;
  const bool vec = ((uintptr_t)e->d & 15) == 0 && e->ld_d * esz % 16 == 0;
  const int cols = 32 * (vec ? 16 / esz : 4), tiles = (e->width + cols - 1) / cols;
  const long long chunks = (e->n + g.chunk - 1) / g.chunk, blocks = (chunks * tiles + 7) / 8;
  if (blocks >= (1ll << 31)) { set_error("embedding_grad: too many values%s", "", 0, 0); return -1; }
  using B = __nv_bfloat16;
  cudaError_t r;
  if (few_places) {
    const long long ctas = (e->n * tiles + 7) / 8, rows = (zero_share(*e, FEW_VALUES) + e->width - 1) / e->width, zero = e->accumulate ? 0 : (e->vocab + rows - 1) / rows;
    auto few = [&](auto kern) { kern<<<(unsigned)(ctas + zero), 256, 0, st>>>(*e, tiles, (int)ctas, (int)rows); };
    if (ctas + zero >= (1ll << 31)) { set_error("embedding_grad: too many values%s", "", 0, 0); return -1; }
    if (e->ids64) {
      if (e->d_bf16) { if (vec) few(embedding_few_kernel<B, 8, 1, long long>); else few(embedding_few_kernel<B, 4, 32, long long>); }
      else { if (vec) few(embedding_few_kernel<float, 4, 1, long long>); else few(embedding_few_kernel<float, 4, 32, long long>); }
    } else {
      if (e->d_bf16) { if (vec) few(embedding_few_kernel<B, 8, 1, int>); else few(embedding_few_kernel<B, 4, 32, int>); }
      else { if (vec) few(embedding_few_kernel<float, 4, 1, int>); else few(embedding_few_kernel<float, 4, 32, int>); }
    }
    if ((r = cudaGetLastError()) != cudaSuccess) { set_error("embedding_grad: %s", cudaGetErrorString(r), 0, 0); return -7; }
    return 0;
  }
  p.zero = zero_share(*e, ZERO_VALUES);
  const long long zeros = zero_ctas(*e, p.zero);
  if (zeros >= (1ll << 30)) { set_error("embedding_grad: too large a table%s", "", 0, 0); return -1; }
  if (e->n <= RANK_MAX) {
    const int ctas = (int)((e->n + RANK_PLACES - 1) / RANK_PLACES);
    p.sorted = 0;
    if (e->ids64) embedding_rank_kernel<long long><<<(unsigned)(ctas + zeros), 256, 0, st>>>(p, ctas);
    else embedding_rank_kernel<int><<<(unsigned)(ctas + zeros), 256, 0, st>>>(p, ctas);
    r = cudaGetLastError();
  } else {
    const int need = 32 - __builtin_clz((unsigned)e->vocab);      // tokens, and `vocab` for none
    const int passes = (need + SORT_BITS - 1) / SORT_BITS;
    p.bits = (need + passes - 1) / passes;
    p.tile = g.tile;
    p.tiles = g.tiles;
    p.sorted = (passes - 1) & 1;
    long long done = 0;
    auto zeros_for = [&](int launch) { return zeros * (launch + 1) / (passes + 1) - done; };      // an even share of each launch
    long long now = zeros_for(0);
    if (e->ids64) embedding_count_kernel<long long><<<(unsigned)(g.tiles + now), SORT_THREADS, 0, st>>>(p, done);
    else embedding_count_kernel<int><<<(unsigned)(g.tiles + now), SORT_THREADS, 0, st>>>(p, done);
    r = cudaGetLastError();
    done += now;
    for (int pass = 0; pass < passes && r == cudaSuccess; ++pass) {
      now = zeros_for(pass + 1);
      r = launch_behind(e->ids64 ? embedding_scatter_kernel<long long> : embedding_scatter_kernel<int>, (unsigned)(g.tiles + now), SORT_THREADS, st, p, pass,
                        (int)(pass == passes - 1), done);
      done += now;
    }
  }
  if (r != cudaSuccess) { set_error("embedding_grad sort: %s", cudaGetErrorString(r), 0, 0); return -7; }
  if (e->n == 0) return 0;
  auto sum = [&](auto kern) { r = launch_behind(kern, (unsigned)blocks, 256, st, p, tiles); };
  if (e->accumulate) {
    if (e->d_bf16) { if (vec) sum(embedding_sum_kernel<B, 8, 1, true, 2>); else sum(embedding_sum_kernel<B, 4, 32, true, 4>); }
    else { if (vec) sum(embedding_sum_kernel<float, 4, 1, true, 4>); else sum(embedding_sum_kernel<float, 4, 32, true, 4>); }
  } else {
    if (e->d_bf16) { if (vec) sum(embedding_sum_kernel<B, 8, 1, false, 4>); else sum(embedding_sum_kernel<B, 4, 32, false, 8>); }
    else { if (vec) sum(embedding_sum_kernel<float, 4, 1, false, 8>); else sum(embedding_sum_kernel<float, 4, 32, false, 8>); }
  }
  if (r != cudaSuccess) { set_error("embedding_grad sum: %s", cudaGetErrorString(r), 0, 0); return -7; }
  if (e->n > g.chunk) {      // (a long run fills a whole chunk and begins ahead of it)
    const int jt = (e->width + 127) / 128;
    const unsigned grid = (unsigned)std::min<long long>(chunks * jt, 4ll * ono_num_sms());
    r = launch_behind(embedding_join_kernel<4>, grid, 32 * JOIN_WARPS, st, p, jt);
    if (r != cudaSuccess) { set_error("embedding_grad join: %s", cudaGetErrorString(r), 0, 0); return -7; }
  }
  return 0;
}
