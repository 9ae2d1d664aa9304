// The choice of a token with top-k, top-p and min-p, from given random numbers or seeded ones.
//
// Per row, with T the temperature, m the largest (penalised) logit and w_i = exp((x_i - m) / T):
//   * top-k keeps the k largest logits, of equal ones those of lowest index;
//   * top-p keeps of those what has at most p * Z of mass strictly above it, Z being the mass top-k left (equal logits
//     stay or go together, as in sampling.cu);
//   * min-p keeps what has w_i >= min_p;
//   * the draw is the first index whose running sum of kept mass, in index order, exceeds u * (kept mass).
// T <= 0 takes the first maximum.  A NaN counts as -infinity, a row without a finite entry gives index 0.
//
// A result is a whole number, so a sum that lies next to a border must fall on the same side as in 64-bit arithmetic,
// whatever the order of the additions: weights are whole multiples of 2^-43 (a rounding of 5.7e-14, relative to the
// largest weight; the exponential is taken in float64), and their sums are exact in 64-bit integers.  Weights below
// 2^-44 round to zero; only u = 0, which takes the first index that stays, can meet one, and looks at float64 itself.
//
// A row is spread over a thread-block cluster and lies in its shared memory.  The cuts are found on linear codes of
// the distance to the maximum (23 bits, monotone): histograms of 256 bins over the interval that holds the cut, with exact counts
// for top-k and masses to 2^-15 of themselves for top-p, narrow the interval until it holds at most 256 tokens, a
// single value, or the whole top-k; then the tokens of the interval are compared with one another, exactly.  Intervals
// that end otherwise (more than 256 tokens of different values within 2^-23 of the range) are cut by bisection with exact sums.
#include "common.cuh"

namespace rl {
namespace filters {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 256;
constexpr int kList = 256;
constexpr int kMaxRanks = 8;
constexpr int kMaxSlice = 48 * 1024;          // floats of one CTA's slice (192 KB)
constexpr int kCodeBits = 23;
constexpr double kUnit = 8796093022208.0;     // 2^43: a weight of one
constexpr float kNegligible = 31.0f;          // (m - x) / T beyond which a weight rounds to zero (44 ln 2 = 30.5)
using u64 = unsigned long long;

struct Args {
  const void* logits;
  long long row_stride;
  int vocab, slice;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* penalty;
  const float* uniforms;
  const u64* seeds;
  const int* counters;
  const int* seen_tokens;
  const int* seen_offsets;
  int* out;
};

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(const void* local, unsigned rank) {
  const uint32_t address = static_cast<uint32_t>(__cvta_generic_to_shared(local));
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(address), "r"(rank));
  return remote;
}
__device__ __forceinline__ unsigned peer_u32(const void* local, unsigned rank) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at_rank(local, rank)) : "memory");
  return v;
}
__device__ __forceinline__ u64 peer_u64(const void* local, unsigned rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at_rank(local, rank)) : "memory");
  return v;
}

// Floats as integers in the same order.
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ void philox_words(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(0xD2511F53u) * c[0], p1 = static_cast<uint64_t>(0xCD9E8D57u) * c[2];
    const uint32_t n0 = static_cast<uint32_t>(p1 >> 32) ^ c[1] ^ k0, n2 = static_cast<uint32_t>(p0 >> 32) ^ c[3] ^ k1;
    c[1] = static_cast<uint32_t>(p1);
    c[3] = static_cast<uint32_t>(p0);
    c[0] = n0;
    c[2] = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// w = rint(2^43 exp((x - top) / T)): 2^(t / 64) with t = (x - top) * 64 log2(e) / T as 2^(j / 64) from a table, 2^e in
// the exponent, and the rest, at most 1 / 128 of an octave, as its series to the fifth power (remainder 6e-17).
__device__ __forceinline__ u64 weight_of(float x, float top, float floor_value, double per, const double* table) {
  if (!(x >= floor_value)) return 0ull;
  const double t = (static_cast<double>(x) - static_cast<double>(top)) * per;
  const double shifted = t + 6755399441055744.0;                       // 1.5 * 2^52: the nearest whole number in the low bits
  const int m = __double2loint(shifted);
  if (m < -64 * 60) return 0ull;
  const double f = (t - (shifted - 6755399441055744.0)) * 0.010830424696249145;      // ln 2 / 64
  double p = fma(f, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  p *= table[m & 63];
  const double scaled = __hiloint2double(__double2hiint(p) + (((m >> 6) + 43) << 20), __double2loint(p));
  return static_cast<u64>(__double_as_longlong(scaled + 4503599627370496.0)) & ((1ull << 52) - 1);
}

struct Shared {
  unsigned bins[2][kBins];        // this CTA's histogram of counts, alternating
  unsigned mass[2][kBins];        // ... of masses, relative to each bin's upper edge
  double total[kBins];            // the cluster's
  unsigned counts[kBins];
  double table[64];
  u64 share[2][4];                // partial results for the peers
  u64 warp_sums[kWarps];
  unsigned warp_words[kWarps];
  float list_x[kList];            // this CTA's tokens of the interval
  int list_i[kList];
  unsigned list_n;
  float all_x[kList];             // the cluster's
  int all_i[kList];
  u64 all_w[kList];
  unsigned char all_keep[kList];
  float picked_x;
  int picked_i;
  u64 found64;
  int found_low, found_high;
  double above;
  unsigned above_n, inside_n, whole_n;
};

template <typename T>
struct Row {
  Shared& s;
  float* values;
  unsigned ranks, rank;
  int begin, count, chunk;      // this CTA's slice; tokens of a thread
  int turn = 0;                 // of the exchange buffers
  int level = 0;                // of the histogram buffers
  float top, floor_value, code_scale;
  double per;

  __device__ Row(Shared& shared, float* v) : s(shared), values(v) {}

  // ---- reductions: over the CTA, then over the cluster; every thread gets the result -------------------------
  __device__ u64 block_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp_sums[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += s.warp_sums[w];
    return total;
  }
  __device__ unsigned block_max(unsigned v) {
    v = __reduce_max_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp_words[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned best = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) best = max(best, s.warp_words[w]);
    return best;
  }
  // The peers' words of this exchange.  A buffer is written again two exchanges later, when every rank has passed the
  // barrier between and so read this one.
  template <typename Fn>
  __device__ void exchange(u64 a, u64 b, Fn&& each) {
    const int slot = turn++ & 1;
    if (threadIdx.x == 0) {
      s.share[slot][0] = a;
      s.share[slot][1] = b;
    }
    if (ranks == 1) {
      __syncthreads();
      each(0u, s.share[slot][0], s.share[slot][1]);
      return;
    }
    cluster_barrier();
    for (unsigned r = 0; r < ranks; ++r) each(r, peer_u64(&s.share[slot][0], r), peer_u64(&s.share[slot][1], r));
  }
  __device__ u64 cluster_sum(u64 v) {
    u64 total = 0;
    exchange(block_sum(v), 0, [&](unsigned, u64 a, u64) { total += a; });
    return total;
  }
  __device__ unsigned cluster_max(unsigned v) {
    unsigned best = 0;
    exchange(block_max(v), 0, [&](unsigned, u64 a, u64) { best = max(best, static_cast<unsigned>(a)); });
    return best;
  }

  template <typename Fn>
  __device__ __forceinline__ void sweep(Fn&& fn) {
    const int first = min(count, static_cast<int>(threadIdx.x) * chunk), last = min(count, first + chunk);
    for (int i = first; i < last; ++i) fn(i, values[i]);
  }
  // 23-bit code of the distance to the maximum, or more than that for what lies outside
  __device__ __forceinline__ unsigned code(float x) const {
    return __float_as_uint(fmaf(top - x, code_scale, 8388608.0f)) - 0x4B000000u;
  }
  __device__ __forceinline__ u64 weight(float x) const { return weight_of(x, top, floor_value, per, s.table); }

  struct Interval {
    unsigned low, high;         // codes, both included
    unsigned above_n, inside_n; // tokens before it and in it
    double above;               // mass before it (approximate)
  };

  // One step: histogram of the interval's codes (and masses), the bins that hold the cut become the interval.
  // kMass false: the cut is the token of rank `want` (counted from 0); true: `share_of` times the whole mass.
  template <bool kMass, typename In>
  __device__ void narrow(Interval& at, unsigned want, double share_of, double& whole, In&& in) {
    const unsigned span = at.high - at.low;
    const int shift = max(0, 24 - __clz(span));           // (span >> shift) < 256
    const int buffer = level++ & 1;
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
      s.bins[buffer][b] = 0;
      if (kMass) s.mass[buffer][b] = 0;
    }
    __syncthreads();
    const float back = 1.0f / code_scale, scale2 = static_cast<float>(per * (1.0 / 64.0));
    sweep([&](int i, float x) {
      const unsigned q = code(x);
      if (q < at.low || q > at.high || !in(i, x)) return;
      const unsigned b = (q - at.low) >> shift;
      atomicAdd(&s.bins[buffer][b], 1u);
      if (kMass) {
        // relative to the bin's upper edge: 16 bits whatever the mass
        const float edge = static_cast<float>(at.low + (b << shift)) * back;
        const float part = fminf(exp2f((edge - (top - x)) * scale2), 1.9f);
        atomicAdd(&s.mass[buffer][b], __float2uint_rn(part * 32768.0f));
      }
    });
    __syncthreads();
    if (ranks > 1) cluster_barrier();
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
      unsigned n = 0;
      double m = 0.0;
      for (unsigned r = 0; r < ranks; ++r) {
        n += ranks == 1 ? s.bins[buffer][b] : peer_u32(&s.bins[buffer][b], r);
        if (kMass) m += static_cast<double>(ranks == 1 ? s.mass[buffer][b] : peer_u32(&s.mass[buffer][b], r));
      }
      s.counts[b] = n;
      if (kMass) s.total[b] = m * exp2(-static_cast<double>(at.low + (static_cast<unsigned>(b) << shift)) * back * (per * (1.0 / 64.0)));
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      // one warp looks through the bins, eight a lane
      const int lane = threadIdx.x;
      unsigned n[8], mine = 0;
      double m[8], mass = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[i] = s.counts[lane * 8 + i];
        mine += n[i];
        m[i] = kMass ? s.total[lane * 8 + i] : 0.0;
        mass += m[i];
      }
      unsigned upto = mine;
      double upto_mass = mass;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned a = __shfl_up_sync(0xffffffffu, upto, o);
        const double b = __shfl_up_sync(0xffffffffu, upto_mass, o);
        if (lane >= o) {
          upto += a;
          upto_mass += b;
        }
      }
      unsigned before = at.above_n + upto - mine;
      double before_mass = at.above + upto_mass - mass;
      if (kMass && whole < 0.0) whole = __shfl_sync(0xffffffffu, at.above + upto_mass, 31);
      // first and last bin the cut can lie in
      int low = -1, high = -1;
      const double budget = share_of * whole, slack = 4e-5 * whole;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (n[i] > 0) {
          if (kMass) {
            // the last bin whose first token is kept: its mass above does not exceed the budget
            if (before_mass <= budget - slack) low = lane * 8 + i;
            if (before_mass <= budget + slack) high = lane * 8 + i;
          } else if (before <= want && want < before + n[i]) {
            low = high = lane * 8 + i;
          }
        }
        before += n[i];
        before_mass += m[i];
      }
      low = __reduce_max_sync(0xffffffffu, low);
      high = __reduce_max_sync(0xffffffffu, high);
      if (low < 0) low = 0;                        // (the first token is always kept)
      if (high < low) high = low;
      // what lies before bin `low`, and in the bins low .. high
      before = at.above_n;
      before_mass = at.above;
      unsigned inside = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int b = lane * 8 + i;
        if (b >= low && b <= high) inside += n[i];
      }
      inside = __reduce_add_sync(0xffffffffu, inside);
      unsigned front = 0;
      double front_mass = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (lane * 8 + i < low) {
          front += n[i];
          front_mass += m[i];
        }
      }
      front = __reduce_add_sync(0xffffffffu, front);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) front_mass += __shfl_xor_sync(0xffffffffu, front_mass, o);
      if (lane == 0) {
        s.found_low = low;
        s.found_high = high;
        s.above_n = before + front;
        s.inside_n = inside;
        s.above = before_mass + front_mass;
        s.total[0] = whole;
      }
      if (lane == 31) s.whole_n = at.above_n + upto;
    }
    __syncthreads();
    const unsigned old = at.low, old_high = at.high;
    at.low = old + (static_cast<unsigned>(s.found_low) << shift);
    at.high = min(old_high, old + (static_cast<unsigned>(s.found_high) << shift) + ((1u << shift) - 1u));
    at.above_n = s.above_n;
    at.inside_n = s.inside_n;
    at.above = s.above;
    if (kMass) whole = s.total[0];
    __syncthreads();
  }

  // Tokens of the cluster with codes low .. high (at most kList of them) into all_x, all_i, all_w of every CTA, in
  // index order of the ranks; returns how many.
  template <typename In>
  __device__ unsigned gather(unsigned low, unsigned high, In&& in) {
    if (threadIdx.x == 0) s.list_n = 0;
    __syncthreads();
    sweep([&](int i, float x) {
      const unsigned q = code(x);
      if (q < low || q > high || !in(i, x)) return;
      const unsigned place = atomicAdd(&s.list_n, 1u);
      if (place < kList) {
        s.list_x[place] = x;
        s.list_i[place] = begin + i;
      }
    });
    __syncthreads();
    if (ranks > 1) cluster_barrier();
    unsigned first = 0;
    for (unsigned r = 0; r < ranks; ++r) {
      const unsigned n = min(ranks == 1 ? s.list_n : peer_u32(&s.list_n, r), static_cast<unsigned>(kList));
      for (unsigned j = threadIdx.x; j < n && first + j < kList; j += kThreads) {
        const float x = ranks == 1 ? s.list_x[j] : __uint_as_float(peer_u32(&s.list_x[j], r));
        s.all_x[first + j] = x;
        s.all_i[first + j] = ranks == 1 ? s.list_i[j] : static_cast<int>(peer_u32(&s.list_i[j], r));
        s.all_w[first + j] = weight(x);
      }
      first += n;
    }
    if (ranks > 1) cluster_barrier();               // the lists may be written again
    __syncthreads();
    return min(first, static_cast<unsigned>(kList));
  }

  // The largest and smallest value among the tokens of an interval.
  template <typename In>
  __device__ void range_of(const Interval& at, In&& in, float& most, float& least) {
    unsigned high = 0, low = 0;
    sweep([&](int i, float x) {
      const unsigned q = code(x);
      if (q < at.low || q > at.high || !in(i, x)) return;
      high = max(high, ordered(x));
      low = max(low, ~ordered(x));
    });
    most = unordered(cluster_max(high));
    least = unordered(~cluster_max(low));
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
sample_filtered_kernel(const Args args, unsigned ranks) {
  extern __shared__ __align__(16) float slice_values[];
  __shared__ Shared s;
  pdl_trigger();
  const int row_index = blockIdx.y;
  Row<T> row(s, slice_values);
  row.ranks = ranks;
  row.rank = blockIdx.x;
  row.begin = min(args.vocab, static_cast<int>(row.rank) * args.slice);
  row.count = min(args.vocab, row.begin + args.slice) - row.begin;
  row.chunk = ((row.count + kThreads - 1) / kThreads) | 1;      // odd: a warp's lanes then read different banks
  for (int j = threadIdx.x; j < 64; j += kThreads) s.table[j] = exp2(static_cast<double>(j) / 64.0);
  pdl_wait();
  const float temp = args.temperature ? args.temperature[row_index] : 0.0f;
  const float pen = args.penalty ? args.penalty[row_index] : 1.0f;
  const int seen_begin = args.seen_offsets ? args.seen_offsets[row_index] : 0;
  const int seen_end = args.seen_offsets ? args.seen_offsets[row_index + 1] : 0;

  // ---- the slice into shared memory ------------------------------------------------------------------------
  const T* x = static_cast<const T*>(args.logits) + static_cast<size_t>(row_index) * args.row_stride + row.begin;
  const bool vector = (reinterpret_cast<uintptr_t>(x) & (sizeof(T) == 2 ? 15 : 31)) == 0;
  const int vector_count = vector ? (row.count & ~7) : 0;
  auto clean = [](float v) { return v == v ? v : -INFINITY; };
  for (int c = threadIdx.x * 8; c < vector_count; c += kThreads * 8) {
    float v[8];
    load8(x + c, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) slice_values[c + j] = clean(v[j]);
  }
  for (int i = vector_count + threadIdx.x; i < row.count; i += kThreads) slice_values[i] = clean(to_float(x[i]));
  __syncthreads();
  if (pen != 1.0f && args.seen_tokens != nullptr && seen_end > seen_begin) {
    // every generated token once: the first of equal ids in the list applies the penalty
    for (int i = seen_begin + threadIdx.x; i < seen_end; i += kThreads) {
      const int id = args.seen_tokens[i] - row.begin;
      if (id < 0 || id >= row.count) continue;
      bool first = true;
      for (int j = seen_begin; j < i && first; ++j) first = args.seen_tokens[j] != id + row.begin;
      if (first) {
        const float v = slice_values[id];
        slice_values[id] = clean(v < 0.0f ? v * pen : v / pen);
      }
    }
    __syncthreads();
  }

  // ---- the first maximum, the smallest finite value ------------------------------------------------------------
  unsigned most = 0, least = 0;
  int place = 0x7fffffff;
  row.sweep([&](int i, float v) {
    const unsigned k = ordered(v);
    if (k > most) {
      most = k;
      place = row.begin + i;
    }
    if (v > -INFINITY) least = max(least, ~k);
  });
  const unsigned mine = most;
  most = row.cluster_max(most);
  const unsigned first_at = ~row.cluster_max(mine == most && row.count > 0 ? ~static_cast<unsigned>(place) : 0u);
  float top = unordered(most);
  if (!(top > -INFINITY)) {                          // nothing to choose from
    if (row.rank == 0 && threadIdx.x == 0) args.out[row_index] = 0;
    if (ranks > 1) cluster_barrier();
    return;
  }
  if (!(temp > 0.0f)) {
    if (row.rank == 0 && threadIdx.x == 0) args.out[row_index] = static_cast<int>(first_at);
    if (ranks > 1) cluster_barrier();                // nobody leaves while its shared memory may be read
    return;
  }
  float bottom = unordered(~row.cluster_max(least));
  if (top == INFINITY) {                             // entries of +infinity share everything
    row.sweep([&](int i, float v) { slice_values[i] = v == INFINITY ? 0.0f : -INFINITY; });
    top = bottom = 0.0f;
    __syncthreads();
  }
  row.top = top;
  row.floor_value = fmaxf(top - kNegligible * temp, -3.4028235e38f);
  row.per = 92.33248261893585 / static_cast<double>(temp);       // 64 log2(e) / T
  {
    // codes: the distance times a power of two, so that the farthest that counts stays below 2^23
    const float farthest = fminf(top - bottom, kNegligible * temp * 1.01f);
    int exponent = 0;
    frexpf(fminf(fmaxf(farthest, 1e-30f), 1e38f), &exponent);    // farthest < 2^exponent
    row.code_scale = exp2f(static_cast<float>(min(kCodeBits - 1 - exponent, 120)));
  }
  constexpr unsigned kLast = (1u << kCodeBits) - 1u;

  const int want_k = args.top_k ? args.top_k[row_index] : 0;
  const float p = args.top_p ? args.top_p[row_index] : 1.0f;
  const float least_p = args.min_p ? fminf(args.min_p[row_index], 1.0f) : 0.0f;
  const double least_weight = static_cast<double>(least_p) * kUnit;
  float u;
  if (args.uniforms) {
    u = args.uniforms[row_index];
  } else {
    uint32_t c[4] = {static_cast<uint32_t>(args.counters[row_index]), 0u, 0u, 0u};
    const u64 seed = args.seeds[row_index];
    philox_words(c, static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32));
    u = static_cast<float>(c[0] >> 8) * (1.0f / 16777216.0f);
  }
  const bool by_rank = want_k > 0 && want_k < args.vocab, by_mass = p < 1.0f;
  const bool first_of_all = !(u > 0.0f);
  // whether the weight is more than zero in float64
  auto counts_at_all = [&](float v) { return exp((static_cast<double>(v) - static_cast<double>(top)) / static_cast<double>(temp)) > 0.0; };
  auto target_of = [&](u64 mass) {
    const double t = u > 0.0f ? static_cast<double>(u) * static_cast<double>(mass) : 0.0;
    return t >= static_cast<double>(mass) ? mass - 1 : min(static_cast<u64>(t), mass - 1);
  };

  // ---- top-k: the value and index of the last token that stays ------------------------------------------------------
  float cut_k = -INFINITY;
  int cut_i = 0x7fffffff;
  auto everything = [](int, float) { return true; };
  if (by_rank) {
    typename Row<T>::Interval at = {0u, kLast, 0u, 0u, 0.0};
    double unused = 0.0;
    bool fewer = false;
    for (bool first = true;; first = false) {
      row.template narrow<false>(at, static_cast<unsigned>(want_k - 1), 0.0, unused, everything);
      if (first) {
        // fewer tokens than k that can be drawn at all: the others weigh nothing, every one may stay
        fewer = s.whole_n <= static_cast<unsigned>(want_k);
      }
      if (fewer || at.above_n + at.inside_n <= kList || at.low == at.high || (at.inside_n <= kList && want_k > kList)) break;
    }
    if (fewer) {
      // nothing is cut
    } else if (at.above_n + at.inside_n <= kList) {
      // the whole of top-k and a little more fits the list: everything else happens there
      const unsigned n = row.gather(0u, at.high, everything);
      const bool have = threadIdx.x < n;
      const float my_x = have ? s.all_x[threadIdx.x] : 0.0f;
      const int my_i = have ? s.all_i[threadIdx.x] : 0;
      const u64 my_w = have ? s.all_w[threadIdx.x] : 0ull;
      unsigned rank = 0;
      if (have)
        for (unsigned j = 0; j < n; ++j) rank += s.all_x[j] > my_x || (s.all_x[j] == my_x && s.all_i[j] < my_i);
      bool keep = have && rank < static_cast<unsigned>(want_k);
      if (have) s.all_keep[threadIdx.x] = keep;
      const u64 z = row.block_sum(keep ? my_w : 0ull);
      __syncthreads();
      if (keep && by_mass) {
        u64 above = 0;
        for (unsigned j = 0; j < n; ++j) above += s.all_keep[j] && s.all_x[j] > my_x ? s.all_w[j] : 0ull;
        keep = static_cast<double>(above) <= static_cast<double>(p) * static_cast<double>(z) || my_x == top;
      }
      keep = keep && (static_cast<double>(my_w) >= least_weight) && (my_w > 0 || (first_of_all && counts_at_all(my_x)));
      __syncthreads();
      if (have) s.all_keep[threadIdx.x] = keep;
      const u64 mass = row.block_sum(keep ? my_w : 0ull);
      __syncthreads();
      if (keep && first_of_all) {
        bool first = true;
        for (unsigned j = 0; j < n; ++j) first = first && !(s.all_keep[j] && s.all_i[j] < my_i);
        if (first && row.rank == 0) args.out[row_index] = my_i;
      } else if (keep) {
        const u64 target = target_of(mass);
        u64 before = 0;
        for (unsigned j = 0; j < n; ++j) before += s.all_keep[j] && s.all_i[j] < my_i ? s.all_w[j] : 0ull;
        if (row.rank == 0 && before <= target && target < before + my_w) args.out[row_index] = my_i;
      }
      if (ranks > 1) cluster_barrier();
      return;
    } else if (at.inside_n <= kList) {
      const unsigned n = row.gather(at.low, at.high, everything);
      if (threadIdx.x < n) {
        const float my_x = s.all_x[threadIdx.x];
        const int my_i = s.all_i[threadIdx.x];
        unsigned rank = at.above_n;
        for (unsigned j = 0; j < n; ++j) rank += s.all_x[j] > my_x || (s.all_x[j] == my_x && s.all_i[j] < my_i);
        if (rank == static_cast<unsigned>(want_k - 1)) {
          s.picked_x = my_x;
          s.picked_i = my_i;
        }
      }
      __syncthreads();
      cut_k = s.picked_x;
      cut_i = s.picked_i;
      __syncthreads();
    } else {
      // more tokens than the list holds within one code: bisect their values, then their indices
      float high, low;
      row.range_of(at, everything, high, low);
      unsigned a = ordered(low), b = ordered(high);           // the k-th value lies in a .. b
      while (a < b) {
        const unsigned mid = a + (b - a) / 2;
        u64 n = 0;
        row.sweep([&](int, float v) { n += ordered(v) > mid; });
        if (row.cluster_sum(n) >= static_cast<u64>(want_k)) a = mid + 1; else b = mid;
      }
      cut_k = unordered(a);
      u64 n = 0;
      row.sweep([&](int, float v) { n += ordered(v) > a; });
      const u64 ties = static_cast<u64>(want_k) - row.cluster_sum(n);    // of the equal ones so many stay
      int from = 0, to = args.vocab - 1;
      while (from < to) {
        const int mid = from + (to - from) / 2;
        n = 0;
        row.sweep([&](int i, float v) { n += ordered(v) == a && row.begin + i <= mid; });
        if (row.cluster_sum(n) >= ties) to = mid; else from = mid + 1;
      }
      cut_i = from;
    }
  }
  auto in_k = [&](int i, float v) { return v > cut_k || (v == cut_k && row.begin + i <= cut_i); };

  // ---- top-p: the smallest value that stays ----------------------------------------------------------------------------
  float cut_p = -INFINITY;
  if (by_mass) {
    typename Row<T>::Interval at = {0u, kLast, 0u, 0u, 0.0};
    double whole = -1.0;
    for (int level = 0; level < 3; ++level) {
      row.template narrow<true>(at, 0u, fmax(static_cast<double>(p), 0.0), whole, in_k);
      if (at.inside_n <= kList || at.low == at.high) break;
    }
    float high, low;
    row.range_of(at, in_k, high, low);
    if (high == low) {
      cut_p = high;
    } else {
      // exact sums from here on: the whole mass, what lies before the interval and in it
      u64 z = 0, above = 0, inside = 0, behind = 0;
      row.sweep([&](int i, float v) {
        if (!in_k(i, v)) return;
        const u64 w = row.weight(v);
        const unsigned q = row.code(v);
        z += w;
        if (q < at.low) above += w;
        else if (q <= at.high) inside += w;
        else if (q <= kLast) behind += 1;
      });
      z = row.cluster_sum(z);
      above = row.cluster_sum(above);
      inside = row.cluster_sum(inside);
      behind = row.cluster_sum(behind);
      const double budget = fmax(static_cast<double>(p), 0.0) * static_cast<double>(z);
      if (static_cast<double>(above) > budget) {       // (not met: the approximate masses are nearer than their slack)
        at = {0u, at.low - 1u, 0u, at.above_n, 0.0};
        above = 0;
      } else if (static_cast<double>(above + inside) <= budget && behind > 0) {
        at = {at.high + 1u, kLast, at.above_n + at.inside_n, static_cast<unsigned>(behind), 0.0};
        above += inside;
      }
      // halve the interval until the list holds it: its far half if that one's first token stays
      while (at.inside_n > kList && at.low < at.high) {
        const unsigned mid = at.low + (at.high - at.low) / 2;
        u64 near_mass = 0, near_n = 0;
        row.sweep([&](int i, float v) {
          const unsigned q = row.code(v);
          if (q < at.low || q > mid || !in_k(i, v)) return;
          near_mass += row.weight(v);
          near_n += 1;
        });
        near_mass = row.cluster_sum(near_mass);
        near_n = row.cluster_sum(near_n);
        if (static_cast<double>(above + near_mass) <= budget && near_n < at.inside_n) {
          above += near_mass;
          at.low = mid + 1u;
          at.inside_n -= static_cast<unsigned>(near_n);
        } else {
          at.high = mid;
          at.inside_n = static_cast<unsigned>(near_n);
        }
      }
      if (at.inside_n <= kList) {
        const unsigned n = row.gather(at.low, at.high, in_k);
        unsigned best = 0;                             // the smallest that stays, as the largest of the complements
        if (threadIdx.x < n) {
          const float my_x = s.all_x[threadIdx.x];
          u64 mass = above;
          for (unsigned j = 0; j < n; ++j) mass += s.all_x[j] > my_x ? s.all_w[j] : 0ull;
          if (static_cast<double>(mass) <= budget) best = ~ordered(my_x);
        }
        cut_p = unordered(~row.block_max(best));
        __syncthreads();
      } else {
        // more than that within one code: by their values, the smallest v with mass(x > v) <= budget
        row.range_of(at, in_k, high, low);
        unsigned a = ordered(low), b = ordered(high);
        while (a < b) {
          const unsigned mid = a + (b - a) / 2;
          u64 mass = 0;
          row.sweep([&](int i, float v) {
            if (ordered(v) > mid && row.code(v) >= at.low && in_k(i, v)) mass += row.weight(v);
          });
          if (static_cast<double>(above + row.cluster_sum(mass)) <= budget) b = mid; else a = mid + 1;
        }
        cut_p = unordered(a);
      }
    }
  }

  // ---- the draw -----------------------------------------------------------------------------------------------------
  if (first_of_all) {
    unsigned best = 0;                               // the complement of the first index
    row.sweep([&](int i, float v) {
      if (best == 0 && v > -INFINITY && v >= cut_p && in_k(i, v) && counts_at_all(v) && static_cast<double>(row.weight(v)) >= least_weight)
        best = ~static_cast<unsigned>(row.begin + i);
    });
    best = row.cluster_max(best);
    if (row.rank == 0 && threadIdx.x == 0) args.out[row_index] = static_cast<int>(~best);
    if (ranks > 1) cluster_barrier();
    return;
  }
  const float lower = fmaxf(fmaxf(cut_p, row.floor_value), -3.4028235e38f);
  auto kept_weight = [&](int i, float v) -> u64 {
    if (v < lower || !in_k(i, v)) return 0ull;
    const u64 w = row.weight(v);
    return static_cast<double>(w) >= least_weight ? w : 0ull;
  };
  u64 local = 0;
  row.sweep([&](int i, float v) { local += kept_weight(i, v); });
  // running sums in index order: over the thread's chunk, the warp, the CTA, the ranks
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 upto = local;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += up;
  }
  __syncthreads();
  if (lane == 31) s.warp_sums[warp] = upto;
  __syncthreads();
  u64 cta = 0, base = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) base += s.warp_sums[w];
    cta += s.warp_sums[w];
  }
  u64 mass = 0, front = 0;
  row.exchange(cta, 0, [&](unsigned r, u64 theirs, u64) {
    if (r < row.rank) front += theirs;
    mass += theirs;
  });
  const u64 target = target_of(mass);
  const u64 before = front + base + upto - local;
  const bool hit = before <= target && target < before + local;
  const unsigned who = __ballot_sync(0xffffffffu, hit);
  if (who) {                                        // one thread of the cluster: its warp looks through its chunk
    const int source = __ffs(who) - 1;
    u64 running = __shfl_sync(0xffffffffu, before, source);
    const int first = (warp * 32 + source) * row.chunk, last = min(row.count, first + row.chunk);
    for (int i0 = first; i0 < last; i0 += 32) {
      const int i = i0 + lane;
      const u64 w = i < last ? kept_weight(i, slice_values[i]) : 0ull;
      u64 sum = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      const bool here = w > 0 && running + sum - w <= target && target < running + sum;
      if (here) args.out[row_index] = row.begin + i;
      if (__any_sync(0xffffffffu, here)) break;
      running += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  if (ranks > 1) cluster_barrier();
}

}  // namespace filters
}  // namespace rl

extern "C" {

// Largest vocabulary of a row.
int rl_sample_filtered_max_vocab() { return rl::filters::kMaxRanks * rl::filters::kMaxSlice; }

// logits: [rows, vocab] of `dtype`, `row_stride` elements between rows.  temperature, top_k (int32), top_p, min_p, penalty: [rows] or
// null; uniforms [rows] in [0, 1), or null with seeds and counters as in rl_sample.
int rl_sample_filtered(int dtype, const void* logits, int rows, int vocab, long long row_stride, const float* temperature,
                       const int* top_k, const float* top_p, const float* min_p, const float* penalty, const float* uniforms,
                       const unsigned long long* seeds, const int* counters, const int* seen_tokens, const int* seen_offsets,
                       int* out, int pdl, cudaStream_t stream) {
  if (rows == 0) return 0;
  if (rows < 0 || rows > 65535 || vocab <= 0 || vocab > rl_sample_filtered_max_vocab() ||
      (temperature != nullptr && uniforms == nullptr && (seeds == nullptr || counters == nullptr)))
    return static_cast<int>(cudaErrorInvalidValue);
  const int ranks = rl::filters::kMaxRanks;
  rl::filters::Args a = {};
  a.logits = logits; a.row_stride = row_stride; a.vocab = vocab;
  a.slice = ((vocab + ranks - 1) / ranks + 7) & ~7;
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.penalty = penalty; a.uniforms = uniforms;
  a.seeds = seeds; a.counters = counters; a.seen_tokens = seen_tokens; a.seen_offsets = seen_offsets; a.out = out;
  const size_t bytes = static_cast<size_t>(a.slice) * sizeof(float);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(ranks, rows);
  config.blockDim = dim3(rl::filters::kThreads);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = ranks;
  attributes[0].val.clusterDim.y = 1;
  attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attributes;
  config.numAttrs = pdl ? 2 : 1;
  RL_DISPATCH_DTYPE(dtype, {
    static std::atomic<unsigned long long> configured;
    auto kernel = rl::filters::sample_filtered_kernel<scalar_t>;
    const cudaError_t e = rl::allow_shared(kernel, rl::filters::kMaxSlice * static_cast<int>(sizeof(float)), configured);
    if (e != cudaSuccess) return static_cast<int>(e);
    return static_cast<int>(cudaLaunchKernelEx(&config, kernel, a, static_cast<unsigned>(ranks)));
  });
  return 0;
}

}  // extern "C"
