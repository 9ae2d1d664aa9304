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

// out[row] = sum_s w_s part[s] / (sum_s w_s + exp(sink)), w_s = 2^(lse_s - max): one warp a (token, head) row, parts
// in index order, float32; the only rounding to the output's type is the last.  Four columns a lane, so that a part's row is
// read as whole lines; kept in L2 by the kernels that wrote it.
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
  pdl_wait();
  if (!mine) return;
  const float* lse = part_lse + static_cast<size_t>(first) * hq + head;
  float top = sink2;
  for (int s = lane; s < parts; s += 32) top = fmaxf(top, __ldcg(lse + static_cast<size_t>(s) * hq));
  top = warp_max(top);
  const float safe = top == -INFINITY ? 0.0f : top;
  float total = lane == 0 && sink != nullptr ? exp2f(sink2 - safe) : 0.0f;
  for (int s = lane; s < parts; s += 32) total += exp2f(__ldcg(lse + static_cast<size_t>(s) * hq) - safe);
  total = warp_sum(total);
  const float inv = (total > 0.0f ? 1.0f / total : 0.0f) * head_gate(gate, gate_stride, token, head);
  const float* src = part_out + (static_cast<size_t>(first) * hq + head) * d;
  T* dst = out + static_cast<size_t>(token) * out_stride + static_cast<size_t>(head) * d;
  const size_t step = static_cast<size_t>(hq) * d;
  for (int c = lane * 4; c < d; c += 128) {
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = 0; s0 < parts; s0 += 4) {
      float4 v[4];
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float l = s0 + i < parts ? __ldcg(lse + static_cast<size_t>(s0 + i) * hq) : -INFINITY;
        w[i] = exp2f(l - safe);
        // a part without keys counts nothing, whatever lies in its place
        v[i] = l == -INFINITY ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : __ldcg(reinterpret_cast<const float4*>(src + (s0 + i) * step + c));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum.x = fmaf(w[i], v[i].x, sum.x);
        sum.y = fmaf(w[i], v[i].y, sum.y);
        sum.z = fmaf(w[i], v[i].z, sum.z);
        sum.w = fmaf(w[i], v[i].w, sum.w);
      }
    }
    dst[c] = from_float<T>(sum.x * inv);
    dst[c + 1] = from_float<T>(sum.y * inv);
    dst[c + 2] = from_float<T>(sum.z * inv);
    dst[c + 3] = from_float<T>(sum.w * inv);
  }
}

}  // namespace rl
