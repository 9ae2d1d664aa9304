// Attention of a step's tokens where groups of requests share the pages of their first positions.
//
// With m a reference point per row and w_j = 2^(s_j - m), the softmax over a row's keys is a quotient of sums
// (sum_j w_j v_j) / (sum_j w_j), and both sums fall apart over any cut of the keys.  So a row's keys are cut into
// the shared ones and its own (and each of these into ranges where there are more multiprocessors than ranges): a kernel
// takes one range for all rows that see it and leaves, per row, the normalised sum and its log-sum-exp, and a last kernel
// joins the parts with weights 2^(lse - max lse).  The shared keys are then read once for a whole group, and the
// rows of a group (its members' heads of one key/value head) are the rows of ordinary matrix products.
//
// The host cuts the step into items of eight numbers (the indices below): packed rows row0 .. row0 + rows - 1 of a
// list of tokens (row p is head p % group of token members[first member + p / group]) against the keys
// first .. end - 1 of one entry's block table, of which a row sees those up to its own position.  Every (token, part) pair is
// covered by exactly one item, for all heads; a token's parts lie at part_first[token] .. part_first[token + 1] - 1.
// An item of no rows is a place without work (lists of a captured step are padded with them).
#pragma once

#include "common.cuh"

namespace rl {

constexpr int kListedInts = 8;
constexpr int kListedFirst = 1;     // first key
constexpr int kListedEnd = 2;       // end of the keys
constexpr int kListedMembers = 3;   // first member
constexpr int kListedRow0 = 4;      // first packed row
constexpr int kListedRows = 5;      // packed rows
constexpr int kListedPart = 6;      // which of its tokens' parts
constexpr int kListedFresh = 7;     // keys from here on are written by this step's earlier kernels
// (item[0]: the entry whose block table is read)

constexpr int kJoinWarps = 4;
constexpr int kJoinAtOnce = 8;      // parts whose rows a lane has in flight

// out[row] = sum_s w_s part[s] / (sum_s w_s + exp(sink)), w_s = 2^(lse_s - max): one warp a (token, head) row, parts
// in index order, float32; the only rounding to the output's type is the last.  Four columns a lane, so that a part's row is
// read as whole lines.  A chain of latencies (the statistics, then the rows, both from L2) bounds it: the first eight rows are fetched
// beside the statistics.  A part without keys counts nothing, whatever lies in its place.
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32)
attention_join_kernel(const float* part_out, const float* part_lse, const int* __restrict__ part_first, T* out,
                      int rows, int hq, int d, int out_stride, const float* __restrict__ sink, const T* gate, int gate_stride) {
  pdl_trigger();
  const int row = blockIdx.x * kJoinWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const bool mine = row < rows;
  const int token = mine ? row / hq : 0, head = mine ? row - token * hq : 0;
  const int first = part_first[token], parts = mine ? part_first[token + 1] - first : 0;
  const float sink2 = sink != nullptr ? sink[head] * 1.4426950408889634f : -INFINITY;
  const float* lse = part_lse + static_cast<size_t>(first) * hq + head;
  const float* src = part_out + (static_cast<size_t>(first) * hq + head) * d;
  T* dst = out + static_cast<size_t>(token) * out_stride + static_cast<size_t>(head) * d;
  const size_t step = static_cast<size_t>(hq) * d;
  pdl_wait();
  if (!mine) return;
  for (int c = lane * 4, turn = 0; turn * 128 < d; c += 128, ++turn) {
    const bool in = c < d;
    float4 v[kJoinAtOnce];
#pragma unroll
    for (int i = 0; i < kJoinAtOnce; ++i)
      v[i] = in && i < parts ? __ldcg(reinterpret_cast<const float4*>(src + i * step + c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // a lane keeps the statistics of parts lane, lane + 32, ...: the maximum and the sum over all of them
    const float l0 = lane < parts ? __ldcg(lse + static_cast<size_t>(lane) * hq) : -INFINITY;
    float top = fmaxf(sink2, l0);
    for (int s = lane + 32; s < parts; s += 32) top = fmaxf(top, __ldcg(lse + static_cast<size_t>(s) * hq));
    top = warp_max(top);
    const float safe = top == -INFINITY ? 0.0f : top;
    const float w0 = exp2f(l0 - safe);
    float total = w0;
    for (int s = lane + 32; s < parts; s += 32) total += exp2f(__ldcg(lse + static_cast<size_t>(s) * hq) - safe);
    total = warp_sum(total) + (sink != nullptr ? exp2f(sink2 - safe) : 0.0f);
    const float inv = (total == 0.0f ? 0.0f : 1.0f / total) * head_gate(gate, gate_stride, token, head);      // a NaN stays one
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = 0; s0 < parts; s0 += kJoinAtOnce) {
      if (s0 > 0) {
#pragma unroll
        for (int i = 0; i < kJoinAtOnce; ++i)
          v[i] = in && s0 + i < parts ? __ldcg(reinterpret_cast<const float4*>(src + (s0 + i) * step + c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int i = 0; i < kJoinAtOnce; ++i) {
        const int s = s0 + i;
        const float w = s < 32 ? __shfl_sync(0xffffffffu, w0, s & 31) : s < parts ? exp2f(__ldcg(lse + static_cast<size_t>(s) * hq) - safe) : 0.0f;
        if (w != 0.0f) {
          sum.x = fmaf(w, v[i].x, sum.x);
          sum.y = fmaf(w, v[i].y, sum.y);
          sum.z = fmaf(w, v[i].z, sum.z);
          sum.w = fmaf(w, v[i].w, sum.w);
        }
      }
    }
    if (in) {
      if constexpr (sizeof(T) == 2) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x * inv, sum.y * inv), hi = __floats2bfloat162_rn(sum.z * inv, sum.w * inv);
        uint2 both;
        both.x = *reinterpret_cast<const uint32_t*>(&lo);
        both.y = *reinterpret_cast<const uint32_t*>(&hi);
        if ((reinterpret_cast<uintptr_t>(dst) & 7) == 0) {
          *reinterpret_cast<uint2*>(dst + c) = both;
          continue;
        }
      }
      dst[c] = from_float<T>(sum.x * inv);
      dst[c + 1] = from_float<T>(sum.y * inv);
      dst[c + 2] = from_float<T>(sum.z * inv);
      dst[c + 3] = from_float<T>(sum.w * inv);
    }
  }
}

}  // namespace rl
