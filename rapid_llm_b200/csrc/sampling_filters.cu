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
// the distance to the maximum (23 bits, monotone): histograms of 256 bins over the interval that holds the cut, with exact
// counts for top-k and masses to 2^-15 of themselves for top-p, narrow the interval until it holds at most 256 tokens, a
// single value, or the whole top-k; then the tokens of the interval are compared with one another, exactly.  Intervals
// that end otherwise (more than 256 tokens of different values within 2^-23 of the range) are cut by bisection with exact sums.
//
// Bound by the chain of steps in a row, each a sweep of shared memory, a barrier of the cluster and a look at 256 bins (2 to
// 3 us): 15 us for one row of 151,936 with top-k 50, 51 for 32 float32 rows that only top-p cuts, whose exact sums (about
// 11 us each, float64 exponentials) come on top, 24 for 256 rows of 32,003 with top-k; the logits alone are 0.05 to 3 us.
#include "common.cuh"

namespace rl {
namespace filters {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 256;
constexpr int kList = 256;
constexpr int kMaxRanks = 8;
constexpr int kMaxSlice = 48 * 1024;          // numbers of one CTA's slice (192 KB as floats)
constexpr int kCodeBits = 23;
constexpr double kUnit = 8796093022208.0;     // 2^43: a weight of one
// What mass(before) - p * mass(all) can be off by where histograms give both, as a share of the whole.  A token's part of its bin's
// edge is off by 2^-16 at most and is 0.61 at least (64 bins or more span 31 nats), its float32 distance costs 4e-6: 2.9e-5 each.
constexpr double kSlack = 6e-5;
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

// w = rint(2^43 exp((x - top) / T)): with t = (x - top) 64 log2(e) / T, 2^(t / 64) is 2^(j / 64) from a table, 2^e in the
// exponent, and the rest, at most 1 / 128 of an octave, as its series to the fourth power (remainder 4e-14, a third of the unit).
__device__ __forceinline__ u64 weight_of(float x, double top, float floor_value, double per, const double* table) {
  if (!(x >= floor_value)) return 0ull;
  const double t = (static_cast<double>(x) - top) * per;
  const double shifted = t + 6755399441055744.0;                       // 1.5 * 2^52: the nearest whole number in the low bits
  const int m = __double2loint(shifted);
  if (m < -64 * 60) return 0ull;
  const double f = t - (shifted - 6755399441055744.0);
  constexpr double a = 0.010830424696249145;                           // ln 2 / 64
  double p = fma(f, a * a * a * a / 24.0, a * a * a / 6.0);
  p = fma(p, f, a * a / 2.0);
  p = fma(p, f, a);
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
  u64 theirs[2][kMaxRanks][4];    // the peers' results
  u64 warp_sums[4][kWarps];
  float list_x[kList];            // this CTA's tokens of the interval
  int list_i[kList];
  unsigned list_n, list_of[kMaxRanks];
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

template <typename Store>
struct Row {
  Shared& s;
  Store* values;
  unsigned ranks, rank;
  int begin, count, chunk;      // this CTA's slice; tokens of a thread
  int turn = 0;                 // of the exchange buffers
  int level = 0;                // of the histogram buffers
  float top, floor_value, code_scale;
  double per, wide_top;

  __device__ Row(Shared& shared, Store* v) : s(shared), values(v) {}

  // ---- reductions: over the CTA, then over the cluster; every thread gets the results -------------------------
  struct Sum { __device__ static u64 of(u64 a, u64 b) { return a + b; } };
  struct Most { __device__ static u64 of(u64 a, u64 b) { return a > b ? a : b; } };
  template <typename Op, int kCount>
  __device__ void block_all(u64 (&v)[kCount]) {
#pragma unroll
    for (int k = 0; k < kCount; ++k)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v[k] = Op::of(v[k], __shfl_xor_sync(0xffffffffu, v[k], o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int k = 0; k < kCount; ++k) s.warp_sums[k][threadIdx.x >> 5] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      v[k] = s.warp_sums[k][threadIdx.x & (kWarps - 1)];
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) v[k] = Op::of(v[k], __shfl_xor_sync(0xffffffffu, v[k], o));
    }
  }
  // The CTAs' words of this exchange, fetched by a few lanes for all.  A buffer is written again two exchanges later, when
  // every rank has passed the barrier between and so read this one.
  template <int kCount>
  __device__ const u64 (*exchange(const u64 (&v)[kCount]))[4] {
    const int slot = turn++ & 1;
    if (threadIdx.x == 0) {
#pragma unroll
      for (int k = 0; k < kCount; ++k) s.share[slot][k] = v[k];
    }
    if (ranks > 1) {
      cluster_barrier();
    } else {
      __syncthreads();
    }
    if (threadIdx.x < ranks * kCount) {
      const unsigned r = threadIdx.x / kCount, k = threadIdx.x % kCount;
      s.theirs[slot][r][k] = ranks > 1 ? peer_u64(&s.share[slot][k], r) : s.share[slot][k];
    }
    __syncthreads();
    return s.theirs[slot];
  }
  template <typename Op, int kCount>
  __device__ void cluster_all(u64 (&v)[kCount]) {
    block_all<Op>(v);
    const u64(*all)[4] = exchange(v);
#pragma unroll
    for (int k = 0; k < kCount; ++k) v[k] = all[0][k];
    for (unsigned r = 1; r < ranks; ++r)
#pragma unroll
      for (int k = 0; k < kCount; ++k) v[k] = Op::of(v[k], all[r][k]);
  }
  __device__ u64 block_sum(u64 v) {
    u64 one[1] = {v};
    block_all<Sum>(one);
    return one[0];
  }
  __device__ u64 cluster_sum(u64 v) {
    u64 one[1] = {v};
    cluster_all<Sum>(one);
    return one[0];
  }

  // Every token of the slice once, in any order: 16 bytes a load.
  template <typename Fn>
  __device__ __forceinline__ void sweep_any(Fn&& fn) {
    constexpr int kWide = 16 / sizeof(Store);
    const int whole = count / kWide * kWide;
    for (int i0 = threadIdx.x * kWide; i0 < whole; i0 += kThreads * kWide) {
      const uint4 raw = *reinterpret_cast<const uint4*>(values + i0);
      const Store* several = reinterpret_cast<const Store*>(&raw);
#pragma unroll
      for (int k = 0; k < kWide; ++k) fn(i0 + k, to_float(several[k]));
    }
    if (whole + threadIdx.x < count) fn(whole + threadIdx.x, to_float(values[whole + threadIdx.x]));
  }
  // A thread's tokens side by side, so that the threads' sums are in index order.
  template <typename Fn>
  __device__ __forceinline__ void sweep(Fn&& fn) {
    const int first = min(count, static_cast<int>(threadIdx.x) * chunk), last = min(count, first + chunk);
#pragma unroll 4
    for (int i = first; i < last; ++i) fn(i, to_float(values[i]));
  }
  // 23-bit code of the distance to the maximum, or more than that for what lies outside
  __device__ __forceinline__ unsigned code(float x) const {
    return __float_as_uint(fmaf(top - x, code_scale, 8388608.0f)) - 0x4B000000u;
  }
  __device__ __forceinline__ u64 weight(float x) const { return weight_of(x, wide_top, floor_value, per, s.table); }

  struct Interval {
    unsigned low, high;         // codes, both included
    unsigned above_n, inside_n; // tokens before it and in it
    double above;               // mass before it (approximate)
  };

  // One step: histogram of the interval's codes (and masses), the bins that hold the cut become the interval.
  // kMass false: the cut is the token of rank `want` (counted from 0); true: `share_of` times the whole mass.
  // kCount: counts are taken (without them a bin holds a token if it holds mass, and how many the interval holds is not known).
  template <bool kMass, bool kCount, typename In>
  __device__ void narrow(Interval& at, unsigned want, double share_of, double& whole, In&& in) {
    const unsigned span = at.high - at.low;
    const int shift = max(0, 24 - __clz(span));           // (span >> shift) < 256
    const int buffer = level++ & 1;
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
      if (kCount) s.bins[buffer][b] = 0;
      if (kMass) s.mass[buffer][b] = 0;
    }
    __syncthreads();
    const float back = 1.0f / code_scale, scale2 = static_cast<float>(per * (1.0 / 64.0));
    sweep_any([&](int i, float x) {
      const unsigned q = code(x);
      if (q < at.low || q > at.high || !in(i, x)) return;
      const unsigned b = (q - at.low) >> shift;
      if (kCount) atomicAdd(&s.bins[buffer][b], 1u);
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
        if (kCount) n += ranks == 1 ? s.bins[buffer][b] : peer_u32(&s.bins[buffer][b], r);
        if (kMass) m += static_cast<double>(ranks == 1 ? s.mass[buffer][b] : peer_u32(&s.mass[buffer][b], r));
      }
      s.counts[b] = kCount ? n : m > 0.0;
      if (kMass) {
        const double edge = static_cast<double>(at.low + (static_cast<unsigned>(b) << shift)) * back;
        s.total[b] = m * (1.0 / 32768.0) * exp2(-edge * (per * (1.0 / 64.0)));
      }
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
      const double budget = share_of * whole, slack = kSlack * whole;
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

  // Tokens of the cluster with codes low .. high (at most kList of them) into all_x, all_i, all_w of every CTA (kFirstOnly: of
  // the first, the others go on); returns how many.  A rank's list may be written again only behind a barrier of the cluster
  // (no call gathers twice without one).
  template <bool kFirstOnly, typename In>
  __device__ unsigned gather(unsigned low, unsigned high, In&& in) {
    if (threadIdx.x == 0) s.list_n = 0;
    __syncthreads();
    sweep_any([&](int i, float x) {
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
    if (kFirstOnly && rank != 0) return 0;
    if (threadIdx.x < ranks) s.list_of[threadIdx.x] = ranks == 1 ? s.list_n : peer_u32(&s.list_n, threadIdx.x);
    __syncthreads();
    unsigned all = 0;
    for (unsigned r = 0; r < ranks; ++r) all += min(s.list_of[r], static_cast<unsigned>(kList));
    all = min(all, static_cast<unsigned>(kList));
    if (threadIdx.x < all) {
      unsigned r = 0, j = threadIdx.x;
      while (j >= s.list_of[r]) j -= s.list_of[r++];
      const float x = ranks == 1 ? s.list_x[j] : __uint_as_float(peer_u32(&s.list_x[j], r));
      s.all_x[threadIdx.x] = x;
      s.all_i[threadIdx.x] = ranks == 1 ? s.list_i[j] : static_cast<int>(peer_u32(&s.list_i[j], r));
      s.all_w[threadIdx.x] = weight(x);
    }
    __syncthreads();
    return all;
  }

  // The largest and smallest value among the tokens of an interval.
  template <typename In>
  __device__ void range_of(const Interval& at, In&& in, float& most, float& least) {
    unsigned high = 0, low = 0;
    sweep_any([&](int i, float x) {
      const unsigned q = code(x);
      if (q < at.low || q > at.high || !in(i, x)) return;
      high = max(high, ordered(x));
      low = max(low, ~ordered(x));
    });
    u64 ends[2] = {high, low};
    cluster_all<Most>(ends);
    most = unordered(static_cast<unsigned>(ends[0]));
    least = unordered(~static_cast<unsigned>(ends[1]));
  }
};

constexpr int kRoomyBytes = 96 * 1024;        // of a slice of which two fit a multiprocessor

static int sm_count() {
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms <= 0)
    sms = 148;
  return sms;
}

// Store: what a slice is kept as: floats, or 16-bit logits as they are (half the shared memory, so that fewer CTAs hold a row).
template <typename T, typename Store>
__global__ void __launch_bounds__(kThreads, 2)
sample_filtered_kernel(const Args args, unsigned ranks) {
  using R = Row<Store>;
  extern __shared__ __align__(16) unsigned char slice_bytes[];
  Store* slice_values = reinterpret_cast<Store*>(slice_bytes);
  __shared__ Shared s;
  pdl_trigger();
  const int row_index = blockIdx.y;
  R row(s, slice_values);
  row.ranks = ranks;
  row.rank = blockIdx.x;
  row.begin = min(args.vocab, static_cast<int>(row.rank) * args.slice);
  row.count = min(args.vocab, row.begin + args.slice) - row.begin;
  row.chunk = ((row.count + kThreads - 1) / kThreads) | 1;      // odd: a warp's lanes then read different banks
  for (int j = threadIdx.x; j < 64; j += kThreads) s.table[j] = exp2(static_cast<double>(j) / 64.0);
  pdl_wait();
  const int want_k = args.top_k ? args.top_k[row_index] : 0;
  if (want_k < 0) return;                            // the whole cluster: this row's place in `out` stays as it is
  const float temp = args.temperature ? args.temperature[row_index] : 0.0f;
  const float pen = args.penalty ? args.penalty[row_index] : 1.0f;
  const int seen_begin = args.seen_offsets ? args.seen_offsets[row_index] : 0;
  const int seen_end = args.seen_offsets ? args.seen_offsets[row_index + 1] : 0;

  // ---- the slice into shared memory ------------------------------------------------------------------------
  const T* x = static_cast<const T*>(args.logits) + static_cast<size_t>(row_index) * args.row_stride + row.begin;
  const bool vector = (reinterpret_cast<uintptr_t>(x) & (sizeof(T) == 2 ? 15 : 31)) == 0;
  const int vector_count = vector ? (row.count & ~7) : 0;
  auto clean = [](float v) { return v == v ? v + 0.0f : -INFINITY; };      // (the sum makes a negative zero the zero it equals)
  // the largest value with the first index it has (a thread meets its own in rising order), and the smallest finite one, on the way
  float most = -INFINITY, least = INFINITY;
  int most_at = -1;
  auto seen = [&](int i, float v) {
    if (v > most) {
      most = v;
      most_at = i;
    }
    least = v > -INFINITY ? fminf(least, v) : least;
  };
  const bool penalised = pen != 1.0f && args.seen_tokens != nullptr && seen_end > seen_begin;
  constexpr int kFly = sizeof(T) == 2 ? 5 : 3;       // 8-element loads of a thread in flight, kept as they come
  struct alignas(16) Raw { uint4 word[sizeof(T) == 2 ? 1 : 2]; };
  for (int c0 = threadIdx.x * 8; c0 < vector_count; c0 += kFly * kThreads * 8) {
    Raw raw[kFly];
#pragma unroll
    for (int f = 0; f < kFly; ++f)
      if (c0 + f * kThreads * 8 < vector_count) raw[f] = *reinterpret_cast<const Raw*>(x + c0 + f * kThreads * 8);
#pragma unroll
    for (int f = 0; f < kFly; ++f) {
      const int c = c0 + f * kThreads * 8;
      if (c >= vector_count) break;
      float v[8];
      const T* values = reinterpret_cast<const T*>(&raw[f]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = clean(to_float(values[j]));
        if (!penalised) seen(c + j, v[j]);
      }
      if constexpr (sizeof(Store) == 4) {
        *reinterpret_cast<float4*>(slice_values + c) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(slice_values + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        __nv_bfloat162 two[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) two[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);      // exact: they were bfloat16
        *reinterpret_cast<uint4*>(slice_values + c) = *reinterpret_cast<const uint4*>(two);
      }
    }
  }
  for (int i = vector_count + threadIdx.x; i < row.count; i += kThreads) {
    const float v = clean(to_float(x[i]));
    slice_values[i] = from_float<Store>(v);
    if (!penalised) seen(i, v);
  }
  __syncthreads();
  if (penalised) {
    // every generated token once: the first of equal ids in the list applies the penalty.  (A walk of the list for each of the
    // slice's tokens, so this grows with the square of what was generated.)
    for (int i = seen_begin + threadIdx.x; i < seen_end; i += kThreads) {
      const int id = args.seen_tokens[i] - row.begin;
      if (id < 0 || id >= row.count) continue;
      bool first = true;
      for (int j = seen_begin; j < i && first; ++j) first = args.seen_tokens[j] != id + row.begin;
      if (first) {
        const float v = to_float(slice_values[id]);
        slice_values[id] = from_float<Store>(clean(v < 0.0f ? v * pen : v / pen));
      }
    }
    __syncthreads();
    row.sweep(seen);
  }
  u64 ends[2] = {most_at < 0 ? 0ull : static_cast<u64>(ordered(most)) << 32 | ~static_cast<unsigned>(row.begin + most_at),
                 least == INFINITY ? 0ull : static_cast<u64>(~ordered(least))};
  row.template cluster_all<typename R::Most>(ends);
  float top = ends[0] == 0ull ? -INFINITY : unordered(static_cast<unsigned>(ends[0] >> 32));
  if (!(top > -INFINITY) || !(temp > 0.0f)) {
    // nothing to choose from, or the first maximum; nobody leaves while its shared memory may be read
    if (row.rank == 0 && threadIdx.x == 0) args.out[row_index] = top > -INFINITY ? static_cast<int>(~static_cast<unsigned>(ends[0])) : 0;
    if (ranks > 1) cluster_barrier();
    return;
  }
  float bottom = ends[1] == 0ull ? top : unordered(~static_cast<unsigned>(ends[1]));
  if (top == INFINITY) {                             // entries of +infinity share everything
    row.sweep([&](int i, float v) { slice_values[i] = from_float<Store>(v == INFINITY ? 0.0f : -INFINITY); });
    top = bottom = 0.0f;
    __syncthreads();
  }
  row.top = top;
  row.floor_value = fmaxf(top - kNegligible * temp, -3.4028235e38f);
  row.per = 92.33248261893585 / static_cast<double>(temp);       // 64 log2(e) / T
  row.wide_top = static_cast<double>(top);
  {
    // codes: the distance times a power of two, so that the farthest that counts stays below 2^23
    const float farthest = fminf(top - bottom, kNegligible * temp * 1.01f);
    int exponent = 0;
    frexpf(fminf(fmaxf(farthest, 1e-30f), 1e38f), &exponent);    // farthest < 2^exponent
    row.code_scale = exp2f(static_cast<float>(min(kCodeBits - 1 - exponent, 120)));
  }
  constexpr unsigned kLast = (1u << kCodeBits) - 1u;

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
  // whether min-p leaves a weight, which may be too small for the whole multiples: in float64, and more than zero there
  auto left_at_zero = [&](float v) {
    const double w = exp((static_cast<double>(v) - static_cast<double>(top)) / static_cast<double>(temp));
    return w > 0.0 && w >= static_cast<double>(least_p);
  };
  auto target_of = [&](u64 mass) {
    const double t = u > 0.0f ? static_cast<double>(u) * static_cast<double>(mass) : 0.0;
    return t >= static_cast<double>(mass) ? mass - 1 : min(static_cast<u64>(t), mass - 1);
  };

  // ---- top-k: the value and index of the last token that stays ------------------------------------------------------
  float cut_k = -INFINITY;
  int cut_i = 0x7fffffff;
  auto everything = [](int, float) { return true; };
  if (by_rank) {
    typename R::Interval at = {0u, kLast, 0u, 0u, 0.0};
    double unused = 0.0;
    bool fewer = false;
    for (bool first = true;; first = false) {
      row.template narrow<false, true>(at, static_cast<unsigned>(want_k - 1), 0.0, unused, everything);
      if (first) {
        // fewer tokens than k that can be drawn at all: the others weigh nothing, every one may stay
        fewer = s.whole_n <= static_cast<unsigned>(want_k);
      }
      if (fewer || at.above_n + at.inside_n <= kList || at.low == at.high || (at.inside_n <= kList && want_k > kList)) break;
    }
    // The k-th value, whose place among the ordered ones is in a .. b, and the index of its last one that stays.
    auto bisect = [&](unsigned a, unsigned b) {
      while (a < b) {
        const unsigned mid = a + (b - a) / 2;
        u64 n = 0;
        row.sweep_any([&](int, float v) { n += ordered(v) > mid; });
        if (row.cluster_sum(n) >= static_cast<u64>(want_k)) a = mid + 1; else b = mid;
      }
      cut_k = unordered(a);
      u64 n = 0;
      row.sweep_any([&](int, float v) { n += ordered(v) > a; });
      const u64 ties = static_cast<u64>(want_k) - row.cluster_sum(n);    // of the equal ones so many stay
      int from = 0, to = args.vocab - 1;
      while (from < to) {
        const int mid = from + (to - from) / 2;
        n = 0;
        row.sweep_any([&](int i, float v) { n += ordered(v) == a && row.begin + i <= mid; });
        if (row.cluster_sum(n) >= ties) to = mid; else from = mid + 1;
      }
      cut_i = from;
    };
    if (fewer) {
      // Nothing is cut, as what lies beyond the codes weighs nothing.  But u = 0 may take a token out there, so the cut is
      // looked for by values, over the whole row.
      if (first_of_all) bisect(ordered(-INFINITY), ordered(top));
    } else if (at.above_n + at.inside_n <= kList) {
      // the whole of top-k and a little more fits the list: everything else happens there
      const unsigned n = row.template gather<true>(0u, at.high, everything);
      if (row.rank != 0) {
        cluster_barrier();                           // the first CTA may still read this one's list
        return;
      }
      // Each token is compared with all others by `side` neighbouring lanes.
      const unsigned padded = n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : 256, side = kThreads / padded;
      const unsigned mine = threadIdx.x / side, sub = threadIdx.x % side;
      const bool have = mine < n, lead = sub == 0;
      const float my_x = have ? s.all_x[mine] : 0.0f;
      const int my_i = have ? s.all_i[mine] : 0;
      const u64 my_w = have ? s.all_w[mine] : 0ull;
      auto over_side = [&](u64 v) {
        for (unsigned o = 1; o < side; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
      };
      u64 rank = 0;
      for (unsigned j = sub; j < n; j += side) rank += s.all_x[j] > my_x || (s.all_x[j] == my_x && s.all_i[j] < my_i);
      rank = over_side(rank);                        // (every lane takes part)
      bool keep = have && rank < static_cast<u64>(want_k);
      if (by_mass) {
        if (lead && have) s.all_keep[mine] = keep;
        const u64 z = row.block_sum(lead && keep ? my_w : 0ull);       // (its barriers publish the marks)
        u64 above = 0;
        for (unsigned j = sub; j < n; j += side) above += s.all_keep[j] && s.all_x[j] > my_x ? s.all_w[j] : 0ull;
        above = over_side(above);
        keep = keep && (static_cast<double>(above) <= static_cast<double>(p) * static_cast<double>(z) || my_x == top);
        __syncthreads();
      }
      keep = keep && (first_of_all ? left_at_zero(my_x) : my_w > 0 && static_cast<double>(my_w) >= least_weight);
      if (lead && have) s.all_keep[mine] = keep;
      const u64 mass = row.block_sum(lead && keep ? my_w : 0ull);
      u64 before = 0;
      for (unsigned j = sub; j < n; j += side)
        before += s.all_keep[j] && s.all_i[j] < my_i ? (first_of_all ? 1ull : s.all_w[j]) : 0ull;
      before = over_side(before);
      if (keep && lead) {
        const u64 target = first_of_all ? 0ull : target_of(mass);
        if (before <= target && target < before + (first_of_all ? 1ull : my_w)) args.out[row_index] = my_i;
      }
      if (ranks > 1) cluster_barrier();
      return;
    } else if (at.inside_n <= kList) {
      const unsigned n = row.template gather<false>(at.low, at.high, everything);
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
      bisect(ordered(low), ordered(high));
    }
  }
  auto in_k = [&](int i, float v) { return v > cut_k || (v == cut_k && row.begin + i <= cut_i); };

  // ---- top-p: the smallest value that stays ----------------------------------------------------------------------------
  float cut_p = -INFINITY;
  u64 weighed = 0;                                   // of this thread's chunk: the mass of codes below `weighed_to`, all of which stays
  unsigned weighed_to = 0;
  if (by_mass) {
    typename R::Interval at = {0u, kLast, 0u, 0u, 0.0};
    double whole = -1.0;
    row.template narrow<true, false>(at, 0u, fmax(static_cast<double>(p), 0.0), whole, in_k);
    for (int level = 0; level < 2; ++level) {
      row.template narrow<true, true>(at, 0u, fmax(static_cast<double>(p), 0.0), whole, in_k);
      if (at.inside_n <= kList || at.low == at.high) break;
    }
    float high, low;
    unsigned listed = 0;
    if (at.inside_n > kList) {
      row.range_of(at, in_k, high, low);
    } else {
      listed = row.template gather<false>(at.low, at.high, in_k);
      u64 ends_of[2] = {0ull, 0ull};
      if (threadIdx.x < listed) {
        ends_of[0] = ordered(s.all_x[threadIdx.x]);
        ends_of[1] = ~ordered(s.all_x[threadIdx.x]);
      }
      row.template block_all<typename R::Most>(ends_of);
      high = unordered(static_cast<unsigned>(ends_of[0]));
      low = unordered(~static_cast<unsigned>(ends_of[1]));
    }
    if (high == low) {
      cut_p = high;                                  // one value, as often as it may be there
    } else {
      // exact sums from here on: the whole mass, what lies before the interval and in it
      u64 z = 0, above = 0, inside = 0, behind = 0;
      row.sweep([&](int i, float v) {
        if (!in_k(i, v)) return;
        const u64 w = row.weight(v);
        const unsigned q = row.code(v);
        z += w;
        if (q < at.low) {
          above += w;
          behind += 1ull << 32;                        // (tokens before the interval ride in the upper half)
        } else if (q <= at.high) {
          inside += w;
        } else if (q <= kLast) {
          behind += 1;
        }
      });
      u64 sums[4] = {z, above, inside, behind};
      row.template cluster_all<typename R::Sum>(sums);
      weighed = above;
      weighed_to = at.low;
      z = sums[0];
      above = sums[1];
      inside = sums[2];
      behind = sums[3] & 0xffffffffull;
      const double budget = fmax(static_cast<double>(p), 0.0) * static_cast<double>(z);
      if (static_cast<double>(above) > budget) {       // (not met: the approximate masses are nearer than their slack)
        at = {0u, at.low - 1u, 0u, static_cast<unsigned>(sums[3] >> 32), 0.0};
        above = 0;
        weighed = 0;
        weighed_to = 0;
        listed = 0;
      } else if (static_cast<double>(above + inside) <= budget && behind > 0) {
        at = {at.high + 1u, kLast, 0u, static_cast<unsigned>(behind), 0.0};
        above += inside;
        listed = 0;
      }
      // halve the interval until the list holds it: its far half if that one's first token stays
      while (at.inside_n > kList && at.low < at.high) {
        const unsigned mid = at.low + (at.high - at.low) / 2;
        u64 near_mass = 0, near_n = 0;
        row.sweep_any([&](int i, float v) {
          const unsigned q = row.code(v);
          if (q < at.low || q > mid || !in_k(i, v)) return;
          near_mass += row.weight(v);
          near_n += 1;
        });
        u64 near_sums[2] = {near_mass, near_n};
        row.template cluster_all<typename R::Sum>(near_sums);
        near_mass = near_sums[0];
        near_n = near_sums[1];
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
        const unsigned n = listed > 0 ? listed : row.template gather<false>(at.low, at.high, in_k);
        unsigned best = 0;                             // the smallest that stays, as the largest of the complements
        if (threadIdx.x < n) {
          const float my_x = s.all_x[threadIdx.x];
          u64 mass = above;
          for (unsigned j = 0; j < n; ++j) mass += s.all_x[j] > my_x ? s.all_w[j] : 0ull;
          if (static_cast<double>(mass) <= budget) best = ~ordered(my_x);
        }
        u64 one[1] = {best};
        row.template block_all<typename R::Most>(one);
        cut_p = unordered(~static_cast<unsigned>(one[0]));
        __syncthreads();
      } else {
        // more than that within one code: by their values, the smallest v with mass(x > v) <= budget
        row.range_of(at, in_k, high, low);
        unsigned a = ordered(low), b = ordered(high);
        while (a < b) {
          const unsigned mid = a + (b - a) / 2;
          u64 mass = 0;
          row.sweep_any([&](int i, float v) {
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
      if (best == 0 && v > -INFINITY && v >= cut_p && in_k(i, v) && left_at_zero(v))
        best = ~static_cast<unsigned>(row.begin + i);
    });
    u64 one[1] = {best};
    row.template cluster_all<typename R::Most>(one);
    if (row.rank == 0 && threadIdx.x == 0) args.out[row_index] = static_cast<int>(~static_cast<unsigned>(one[0]));
    if (ranks > 1) cluster_barrier();
    return;
  }
  // (min-p's own cut, drawn a little wide, spares most weights their exponential)
  const float cut_min = least_p > 0.0f ? top + temp * (logf(least_p) * 1.001f - 0.001f) : -3.4028235e38f;
  const float lower = fmaxf(fmaxf(cut_p, row.floor_value), fmaxf(cut_min, -3.4028235e38f));
  auto kept_weight = [&](int i, float v) -> u64 {
    if (v < lower || !in_k(i, v)) return 0ull;
    const u64 w = row.weight(v);
    return static_cast<double>(w) >= least_weight ? w : 0ull;
  };
  u64 local = 0;
  if (weighed_to > 0 && least_p <= 0.0f) {
    local = weighed;
    row.sweep([&](int i, float v) {
      if (v >= lower && row.code(v) >= weighed_to) local += kept_weight(i, v);
    });
  } else {
    row.sweep([&](int i, float v) { local += kept_weight(i, v); });
  }
  // running sums in index order: over the thread's chunk, the warp, the CTA, the ranks
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 upto = local;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += up;
  }
  __syncthreads();
  if (lane == 31) s.warp_sums[0][warp] = upto;
  __syncthreads();
  u64 cta = 0, base = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) base += s.warp_sums[0][w];
    cta += s.warp_sums[0][w];
  }
  u64 mass = 0, front = 0;
  const u64 mine[1] = {cta};
  const u64(*all)[4] = row.exchange(mine);
  for (unsigned r = 0; r < ranks; ++r) {
    if (r < row.rank) front += all[r][0];
    mass += all[r][0];
  }
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
      const u64 w = i < last ? kept_weight(i, to_float(slice_values[i])) : 0ull;
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
  // A penalty makes a logit wider than 16 bits.
  const bool halves = dtype == rl::kBF16 && (penalty == nullptr || seen_tokens == nullptr);
  const int size = halves ? 2 : 4, slots = 2 * rl::filters::sm_count();
  // CTAs a row: as many as run at one time (two a multiprocessor), since a row's steps wait for one another more than they compute, as
  // long as two slices fit.  In us with 8, 4, 2 and 1 (bfloat16): 256 rows of 32,003 with top-k 50 102, 55, 36, 25, without
  // 185, 109, 82, 68; 64 rows 28, 16, 17, 19 and 53, 32, 36, 49; 64 rows of 151,936 38, 28 and 120, 103; one row 15, 19.
  // Where most rows end early, the later ones start sooner in small pieces: 64 rows of which few are long 64 with 8, 80 with 4.
  int ranks = rl::filters::kMaxRanks;
  while (ranks > 1 && rows * ranks > slots && ((vocab + ranks / 2 - 1) / (ranks / 2) + 8) * size <= rl::filters::kRoomyBytes) ranks /= 2;
  rl::filters::Args a = {};
  a.logits = logits; a.row_stride = row_stride; a.vocab = vocab;
  a.slice = ((vocab + ranks - 1) / ranks + 7) & ~7;
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.penalty = penalty; a.uniforms = uniforms;
  a.seeds = seeds; a.counters = counters; a.seen_tokens = seen_tokens; a.seen_offsets = seen_offsets; a.out = out;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(ranks, rows);
  config.blockDim = dim3(rl::filters::kThreads);
  config.dynamicSmemBytes = static_cast<size_t>(a.slice) * size;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = ranks;
  attributes[0].val.clusterDim.y = 1;
  attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = ranks > 1 ? attributes : attributes + 1;      // a row in one CTA needs no cluster
  config.numAttrs = (ranks > 1 ? 1 : 0) + (pdl ? 1 : 0);
  static std::atomic<unsigned long long> configured[3];
  auto launch = [&](auto kernel, int which) {
    const cudaError_t e = rl::allow_shared(kernel, rl::filters::kMaxSlice * size, configured[which]);
    if (e != cudaSuccess) return static_cast<int>(e);
    return static_cast<int>(cudaLaunchKernelEx(&config, kernel, a, static_cast<unsigned>(ranks)));
  };
  if (dtype == rl::kF32) return launch(rl::filters::sample_filtered_kernel<float, float>, 0);
  if (dtype != rl::kBF16) return static_cast<int>(cudaErrorInvalidValue);
  return halves ? launch(rl::filters::sample_filtered_kernel<__nv_bfloat16, __nv_bfloat16>, 1)
                : launch(rl::filters::sample_filtered_kernel<__nv_bfloat16, float>, 2);
}

}  // extern "C"
