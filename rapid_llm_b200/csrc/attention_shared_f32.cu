// Attention over shared prefixes in 32 bits (attention_shared.h says what an item is): one CTA an item and key/value
// head, tiles of 32 packed rows against blocks of 64 keys, plain multiply-adds in float32.
//
// Bounded by the multiply-adds (4 d operations a row and key) wherever a group has more than a few rows: the tile of
// scores is 4 x 2 outputs a thread (six 16-byte loads from shared memory for 32 multiply-adds, of which a warp's lanes
// share most), the products with the values 4 rows x 4 columns a thread.  Keys and values of a block are brought by
// cp.async: the next keys while the softmax and the values' product run, the values while the scores are formed; page ids are
// looked up a block ahead.  Eight requests of 32 heads on 8 (128 numbers), 2,048 shared keys and 100 of their own: 28 us with the
// join, where each for itself takes 1,265 (the generic kernel).  So short a step fills a third of the multiply-adds' pipes:
// 192 CTAs of a few blocks each, whose turns (scores, softmax, values) wait for shared memory.  Scores of 8 x 4 over four
// lanes and 8 x 4 outputs of O, with half the reads, were slower (31.9 -> 33.0 us at 128 registers, 35.6 at the 151 they want).
#include "attention_shared.h"

namespace rl {

constexpr int kSfRows = 32;
constexpr int kSfKeys = 64;
constexpr int kSfThreads = 256;
constexpr int kSfPad = 4;

static size_t shared_f32_smem(int d) {
  return (static_cast<size_t>(kSfRows + 2 * kSfKeys) * (d + kSfPad) + kSfKeys * (kSfRows + kSfPad) + 3 * kSfRows) * sizeof(float);
}

struct SharedF32Args {
  const float* q;
  const float* cache;
  float* part_out;
  float* part_lse;
  const int* items;
  const int* members;
  const int* positions;
  const int* part_first;
  const int* entry_slot;
  const int* block_table;
  int hq, hkv, d, page_size, num_pages, max_pages, slots;
  float scale_log2;
  const float* slopes;
  int* fault;
};

__device__ __forceinline__ void sf_copy16(float* dst, const float* src, bool valid) {
  const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  const int bytes = valid ? 16 : 0;                 // 0: the 16 bytes become zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(src), "r"(bytes) : "memory");
}

__global__ void __launch_bounds__(kSfThreads)
attention_shared_f32_kernel(const SharedF32Args args) {
  extern __shared__ __align__(16) float sf_smem[];
  const int d = args.d, stride = d + kSfPad;
  float* q_tile = sf_smem;                               // [rows][stride]
  float* k_tile = q_tile + kSfRows * stride;             // [keys][stride]
  float* v_tile = k_tile + kSfKeys * stride;             // [keys][stride]
  float* p_tile = v_tile + kSfKeys * stride;             // [keys][rows + pad]: scores, then weights
  float* row_max = p_tile + kSfKeys * (kSfRows + kSfPad);
  float* row_sum = row_max + kSfRows;
  float* row_scale = row_sum + kSfRows;
  __shared__ long long places[2][kSfKeys];               // where a block's key rows start (-1: beyond the end), alternating
  __shared__ int row_token[kSfRows], row_pos[kSfRows];
  __shared__ float row_slope[kSfRows];
  __shared__ int first_pos;                              // the smallest of the rows' positions
  static_assert(kSfRows == 32, "a row a lane of the first warp");
  constexpr int p_stride = kSfRows + kSfPad;

  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int* item = args.items + static_cast<size_t>(blockIdx.y) * kListedInts;
  const int kv_head = blockIdx.x, group = args.hq / args.hkv;
  const int rows = min(item[kListedRows], kSfRows);
  const int slot = args.entry_slot[item[0]];
  const int first = item[kListedFirst], end = item[kListedEnd];
  const bool bad = slot < 0 || slot >= args.slots || first < 0 || end > args.max_pages * args.page_size;
  if (rows > 0 && bad && tid == 0) atomicOr(args.fault, (slot < 0 || slot >= args.slots) ? kFaultSlot : kFaultPosition);
  pdl_wait();
  if (rows <= 0) return;
  const int* table = args.block_table + static_cast<size_t>(bad ? 0 : slot) * args.max_pages;
  const int n_blocks = bad || end <= first ? 0 : (end - first + kSfKeys - 1) / kSfKeys;
  for (int r = tid; r < kSfRows; r += kSfThreads) {
    const int p = item[kListedRow0] + r, head = kv_head * group + p % group;
    const bool valid = r < rows;
    row_token[r] = valid ? args.members[item[kListedMembers] + p / group] : 0;
    row_pos[r] = valid ? args.positions[row_token[r]] : -1;
    row_slope[r] = valid && args.slopes != nullptr ? args.slopes[head] * 1.4426950408889634f : 0.0f;
    row_max[r] = -INFINITY;
    row_sum[r] = 0.0f;
    const int smallest = __reduce_min_sync(0xffffffffu, valid ? row_pos[r] : 0x7fffffff);      // (one warp, a row a lane)
    if (r == 0) first_pos = smallest;
  }
  // a block's page ids are looked up once, by a thread a key, a block ahead of its copies
  const size_t head_elements = static_cast<size_t>(args.page_size) * d;
  auto find = [&](int block) {
    if (tid >= kSfKeys) return;
    const int j = first + block * kSfKeys + tid;
    long long place = -1;
    if (j < end) {
      const int at = j / args.page_size, page = table[at];
      if (page < 0 || page >= args.num_pages)
        atomicOr(args.fault, kFaultPageId);
      else
        place = static_cast<long long>((static_cast<size_t>(page) * 2 * args.hkv + kv_head) * head_elements + static_cast<size_t>(j - at * args.page_size) * d);
    }
    places[block & 1][tid] = place;
  };
  if (n_blocks > 0) find(0);
  __syncthreads();
  const int chunks = d / 4;
  for (int i = tid; i < kSfRows * chunks; i += kSfThreads) {
    const int r = i / chunks, c = (i - r * chunks) * 4;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r < rows) {
      const int head = kv_head * group + (item[kListedRow0] + r) % group;
      v = *reinterpret_cast<const float4*>(args.q + (static_cast<size_t>(row_token[r]) * args.hq + head) * d + c);
    }
    *reinterpret_cast<float4*>(q_tile + r * stride + c) = v;
  }
  const size_t v_plane = static_cast<size_t>(args.hkv) * head_elements;
  auto load = [&](float* tile, int block, int plane) {
    const long long* place = places[block & 1];
    for (int i = tid; i < kSfKeys * chunks; i += kSfThreads) {
      const int r = i / chunks, c = (i - r * chunks) * 4;
      const long long at = place[r];
      sf_copy16(tile + r * stride + c, args.cache + (at < 0 ? 0 : at + static_cast<long long>(plane * v_plane) + c), at >= 0);
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };

  // O: units of 4 rows x 4 columns, up to two a thread (d = 256)
  const int units = (kSfRows / 4) * chunks;
  float acc[2][4][4];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[u][i][c] = 0.0f;

  if (n_blocks > 0) {
    load(k_tile, 0, 0);
    load(v_tile, 0, 1);
  }
  for (int b = 0; b < n_blocks; ++b) {
    const int kb = first + b * kSfKeys;
    if (b + 1 < n_blocks) find(b + 1);
    asm volatile("cp.async.wait_group 1;\n" ::: "memory");      // the keys are there, the values may still fly
    __syncthreads();
    {
      // scores: a warp 16 rows x 16 keys, a lane 4 rows x 2 keys
      const int r0 = (warp & 1) * 16 + (lane >> 3) * 4, k0 = (warp >> 1) * 16 + (lane & 7);
      float s[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i][0] = s[i][1] = 0.0f;
      if (r0 < rows) {
        const float* qr = q_tile + r0 * stride;
        const float* kr = k_tile + k0 * stride;
#pragma unroll 4
        for (int c = 0; c < d; c += 4) {
          const float4 k_a = *reinterpret_cast<const float4*>(kr + c), k_b = *reinterpret_cast<const float4*>(kr + 8 * stride + c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(qr + i * stride + c);
            s[i][0] = fmaf(x.x, k_a.x, fmaf(x.y, k_a.y, fmaf(x.z, k_a.z, fmaf(x.w, k_a.w, s[i][0]))));
            s[i][1] = fmaf(x.x, k_b.x, fmaf(x.y, k_b.y, fmaf(x.z, k_b.z, fmaf(x.w, k_b.w, s[i][1]))));
          }
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int k = k0 + 8 * half, j = kb + k;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int pos = row_pos[r0 + i];
          const bool keep = j < end && j <= pos;
          p_tile[k * p_stride + r0 + i] = keep ? fmaf(row_slope[r0 + i], static_cast<float>(j - pos), s[i][half] * args.scale_log2) : -INFINITY;
        }
      }
    }
    __syncthreads();
    if (b + 1 < n_blocks) {
      load(k_tile, b + 1, 0);
    } else {
      asm volatile("cp.async.commit_group;\n" ::: "memory");    // an empty group, so that the count below holds
    }
    {
      // softmax: eight lanes a row, eight keys a lane
      const int r = tid >> 3, part = tid & 7;
      float x[8], top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = p_tile[(part + 8 * i) * p_stride + r];
        top = fmaxf(top, x[i]);
      }
#pragma unroll
      for (int offset = 1; offset < 8; offset <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, offset));
      const float before = row_max[r], now = fmaxf(before, top), safe = now == -INFINITY ? 0.0f : now;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = exp2f(x[i] - safe);
        p_tile[(part + 8 * i) * p_stride + r] = e;
        sum += e;
      }
#pragma unroll
      for (int offset = 1; offset < 8; offset <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
      __syncwarp();                                  // every lane of the row has read its maximum
      if (part == 0) {
        const float alpha = exp2f(before - safe);    // 0 while nothing was seen
        row_max[r] = now;
        row_sum[r] = row_sum[r] * alpha + sum;
        row_scale[r] = alpha;
      }
    }
    asm volatile("cp.async.wait_group 1;\n" ::: "memory");      // the values are there, the next keys may still fly
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int unit = tid + u * kSfThreads;
      if (unit >= units) continue;
      const int r0 = unit / chunks * 4, c = (unit - unit / chunks * chunks) * 4;
      if (r0 >= rows) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float alpha = row_scale[r0 + i];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[u][i][e] *= alpha;
      }
      // Keys that all rows see; behind them, where tokens of one request differ, a row leaves out what it does not see:
      // zero times a value that is not finite is no zero.
      const int last = min(kSfKeys, end - kb), seen_by_all = min(last, first_pos - kb + 1);
      int k = 0;
#pragma unroll 4
      for (; k < seen_by_all; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(v_tile + k * stride + c);
        const float4 p = *reinterpret_cast<const float4*>(p_tile + k * p_stride + r0);
        const float w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[u][i][0] = fmaf(w[i], v.x, acc[u][i][0]);
          acc[u][i][1] = fmaf(w[i], v.y, acc[u][i][1]);
          acc[u][i][2] = fmaf(w[i], v.z, acc[u][i][2]);
          acc[u][i][3] = fmaf(w[i], v.w, acc[u][i][3]);
        }
      }
#pragma unroll 1
      for (; k < last; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(v_tile + k * stride + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (kb + k > row_pos[r0 + i]) continue;
          const float w = p_tile[k * p_stride + r0 + i];
          acc[u][i][0] = fmaf(w, v.x, acc[u][i][0]);
          acc[u][i][1] = fmaf(w, v.y, acc[u][i][1]);
          acc[u][i][2] = fmaf(w, v.z, acc[u][i][2]);
          acc[u][i][3] = fmaf(w, v.w, acc[u][i][3]);
        }
      }
    }
    __syncthreads();
    if (b + 1 < n_blocks) load(v_tile, b + 1, 1);
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int unit = tid + u * kSfThreads;
    if (unit >= units) continue;
    const int r0 = unit / chunks * 4, c = (unit - unit / chunks * chunks) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + i;
      if (r >= rows) continue;
      const float total = row_sum[r], inv = total > 0.0f ? 1.0f / total : 0.0f;
      const int head = kv_head * group + (item[kListedRow0] + r) % group;
      const size_t at = static_cast<size_t>(args.part_first[row_token[r]] + item[kListedPart]) * args.hq + head;
      *reinterpret_cast<float4*>(args.part_out + at * d + c) =
          make_float4(acc[u][i][0] * inv, acc[u][i][1] * inv, acc[u][i][2] * inv, acc[u][i][3] * inv);
      if (c == 0) args.part_lse[at] = total == 0.0f ? -INFINITY : row_max[r] + log2f(total);
    }
  }
}

}  // namespace rl

extern "C" {

// Packed rows of an item.
int rl_attention_shared_f32_rows() { return rl::kSfRows; }

int rl_attention_shared_f32(const float* q, const float* cache, float* out, float* part_out, float* part_lse, const int* items,
                            int n_items, const int* members, const int* positions, const int* part_first, const int* entry_slot,
                            const int* block_table, int tokens, int hq, int hkv, int d, int page_size, int num_pages,
                            int max_pages, int slots, float scale, const float* sink, const float* slopes, int out_stride,
                            const float* gate, int gate_stride, int* fault, int pdl, cudaStream_t stream) {
  if (tokens == 0) return 0;
  if (d <= 0 || d % 16 != 0 || d > 256 || hkv <= 0 || hq % hkv != 0 || page_size <= 0 || num_pages <= 0 || n_items < 0 || n_items > 65535 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(part_out)) & 15) ||
      out_stride < hq * d || (gate != nullptr && gate_stride < hq) || static_cast<long long>(tokens) * hq > 0x7fffffffll)
    return static_cast<int>(cudaErrorInvalidValue);
  int status = 0;
  if (n_items > 0) {
    rl::SharedF32Args a;
    a.q = q; a.cache = cache; a.part_out = part_out; a.part_lse = part_lse; a.items = items; a.members = members;
    a.positions = positions; a.part_first = part_first; a.entry_slot = entry_slot; a.block_table = block_table;
    a.hq = hq; a.hkv = hkv; a.d = d; a.page_size = page_size; a.num_pages = num_pages; a.max_pages = max_pages; a.slots = slots;
    a.scale_log2 = scale * 1.4426950408889634f; a.slopes = slopes; a.fault = fault;
    static std::atomic<unsigned long long> configured;
    const cudaError_t e = rl::allow_shared(rl::attention_shared_f32_kernel, static_cast<int>(rl::shared_f32_smem(256)), configured);
    if (e != cudaSuccess) return static_cast<int>(e);
    status = rl::launch_kernel(rl::attention_shared_f32_kernel, dim3(hkv, n_items), dim3(rl::kSfThreads), rl::shared_f32_smem(d),
                               stream, pdl != 0, a);
    if (status != 0) return status;
  }
  const int rows = tokens * hq;
  return rl::launch_kernel(rl::attention_join_kernel<float>, dim3((rows + rl::kJoinWarps - 1) / rl::kJoinWarps),
                           dim3(rl::kJoinWarps * 32), 0, stream, pdl != 0 || n_items > 0, part_out, part_lse, part_first, out, rows, hq, d,
                           out_stride, sink, gate, gate_stride);
}

}  // extern "C"
