// Attention of a few packed rows over a range of keys, straight from memory into the tensor cores' registers (items:
// attention_shared.h): a request's own keys behind a shared prefix, or a prefix that two or three requests share.
//
//     S^T[key, row] = K[key, :] . Q[row, :]        mma.sync  m16 (keys) x n8 (rows) x k16
//     O^T[d, row]  += V[key, d]^T . P^T[key, row]  mma.sync  m16 (d)    x n8 (rows) x k16 (keys)
//
// Such ranges are short (a few hundred keys), so what a kernel does before its first key and after its last one counts more
// than its rate: no tile in shared memory, no barrier, no ring, no tensor memory.  A warp takes sixteen keys a step, the four
// warps of a CTA every fourth step, and a lane loads 16 bytes of a row at a time in an order that IS the order of the
// instruction's operands: a sum over d may run in any order as long as Q and K agree, and which d a row of O^T stands for is
// free.  K's words are operands as they come; V's words of two neighbouring keys are interleaved by byte permutations (two
// an operand pair); P^T is S^T's fragment, transposed by movmatrix.  Sixteen 16-byte loads a lane fly per step (8 KB a
// warp, some 100 KB a multiprocessor).
//
// By themselves, with the join: 64 requests of 8 key heads and 512 keys 27.8 us for 20.5 of HBM's rate, 2,048 keys 90 for 82,
// 16 keys 6.6; heads of 64 (4 key heads) 2,048 keys 47 for 20.5: half the bytes in flight, so the loads' latency bounds them.
// An item by itself takes 1.3 us a step of its warps.  Four CTAs a multiprocessor (126 registers) instead of three took 6 %
// off 64 requests behind 8,192 shared keys; eight warps a CTA were slower, so were tiles by TMA into shared memory
// (13.5 -> 23 us for 16 requests behind 2,048) and the next step's keys ahead, for which the queries had to leave the
// registers (27.8 -> 35.9 us for the 512 keys, heads of 64 16.2 -> 16.8).
//
// Scores, maxima, sums and O are float32; P is rounded to bfloat16 before P.V, as in attention_mma.cu.  Heads of 64 and 128,
// pages of any size (a step inside one page, as with pages of 16 and its multiples, looks one page id up for the whole warp).
#pragma once

#include "attention_shared.h"

namespace rl {
namespace RL_ATTENTION_NS {

constexpr bool kRwTakes = kD == 64 || kD == 128;     // (the kernel is built for these alone)
constexpr int kRwWarps = 4;
constexpr int kRwKeys = 16;                    // keys of a step
constexpr int kRwStagedPages = 512;
constexpr int kRwRows = 16;                    // packed rows of an item, at most: two octets

struct RowsArgs {
  const bf16* q;
  const bf16* cache;
  float* part_out;
  float* part_lse;
  const int* items;
  const int* members;
  const int* positions;
  const int* part_first;
  const int* entry_slot;
  const int* block_table;
  int hq, hkv, page_size, num_pages, max_pages, slots;
  int early;                                   // as in attention_decode_tc.cuh
  float scale_log2;
  const float* slopes;
  int* fault;
};

__device__ __forceinline__ uint32_t rw_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void rw_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t rw_word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <int kOctets, bool kSloped>
__global__ void __launch_bounds__(kRwWarps * 32, kOctets == 1 ? 4 : 2)
attention_rows_kernel(const RowsArgs args) {
  constexpr int kSegs = kD / 32, kRounds = kD / 64, kTiles = kD / 16;
  __shared__ int staged_pages[kRwStagedPages];
  __shared__ __align__(16) float merge_o[kRwWarps][kOctets * 8][kD + 4];
  __shared__ float merge_max[kRwWarps][kOctets * 8], merge_sum[kRwWarps][kOctets * 8];

  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int* item = args.items + static_cast<size_t>(blockIdx.y) * kListedInts;
  const int rows = min(item[kListedRows], kOctets * 8);
  if (rows <= 0) {                             // a place of the list that holds no item
    pdl_wait();
    return;
  }
  const int row0 = item[kListedRow0], part = item[kListedPart], first = item[kListedFirst];
  const int kv_head = blockIdx.x, group = args.hq / args.hkv;
  const int slot = args.entry_slot[item[0]];
  const int* members = args.members + item[kListedMembers];
  const bool bad = slot < 0 || slot >= args.slots || first < 0 || item[kListedEnd] > args.max_pages * args.page_size;
  if (bad && tid == 0) atomicOr(args.fault, (slot < 0 || slot >= args.slots) ? kFaultSlot : kFaultPosition);
  const int end = bad ? first : item[kListedEnd];
  const int* table = args.block_table + static_cast<size_t>(bad ? 0 : slot) * args.max_pages;
  const int begin = first & ~(kRwKeys - 1);
  const int steps = end > first ? (end - begin + kRwKeys - 1) / kRwKeys : 0;
  auto checked = [&](int page) {
    if (page >= 0 && page < args.num_pages) return page;
    atomicOr(args.fault, kFaultPageId);
    return 0;                                  // the null page: readable
  };
  // With pages of 16 and its multiples a step's keys lie in one page: a lane looks up the page of the warp's step that
  // has its number, and of every 32nd behind it.  Other pages: all ids of the range are brought to shared memory.
  const bool in_page = args.page_size % kRwKeys == 0;
  auto page_of_step = [&](int step) { return step < steps ? table[(begin + step * kRwKeys) / args.page_size] : 0; };
  int my_page = in_page ? page_of_step(warp + kRwWarps * lane) : 0;

  // this lane's rows: operands of row g (of each octet), scores and sums of rows 2 c and 2 c + 1
  int limit[kOctets][2], pos[kOctets][2];
  float slope[kOctets][2];
  uint4 q[kOctets][kSegs];
  size_t q_at[kOctets];
#pragma unroll
  for (int o = 0; o < kOctets; ++o) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = o * 8 + 2 * c + i, p = row0 + r;
      pos[o][i] = r < rows ? args.positions[members[p / group]] : -1;
      limit[o][i] = min(pos[o][i], end - 1);
      slope[o][i] = kSloped && r < rows ? args.slopes[kv_head * group + p % group] * 1.4426950408889634f : 0.0f;
    }
    const int r = min(o * 8 + g, rows - 1), p = row0 + r;        // rows behind the last repeat it; nothing of theirs is kept
    q_at[o] = (static_cast<size_t>(members[p / group]) * args.hq + kv_head * group + p % group) * kD;
  }
  const int first_page = begin / args.page_size;
  const int page_count = steps > 0 ? (end - 1) / args.page_size - first_page + 1 : 0;
  const bool staged = !in_page && page_count <= kRwStagedPages;
  if (!in_page) {
    if (staged)
      for (int i = tid; i < page_count; i += kRwWarps * 32) staged_pages[i] = checked(table[first_page + i]);
    __syncthreads();
  }
  auto page_at = [&](int index) { return staged ? staged_pages[index - first_page] : checked(table[index]); };
  if (!args.early) pdl_wait();                 // queries and this step's keys come from the kernels before
#pragma unroll
  for (int o = 0; o < kOctets; ++o)
#pragma unroll
    for (int s = 0; s < kSegs; ++s) q[o][s] = __ldcg(reinterpret_cast<const uint4*>(args.q + q_at[o] + 32 * s + 8 * c));

  const size_t v_plane = static_cast<size_t>(args.hkv) * args.page_size * kD;
  const bf16* head = args.cache + static_cast<size_t>(kv_head) * args.page_size * kD;
  // where key j's row starts; keys outside the range read the nearest one inside, and weigh nothing
  auto row_of = [&](int j) {
    const int at = min(max(j, first), end - 1), index = at / args.page_size;
    return head + static_cast<size_t>(page_at(index)) * 2 * v_plane + static_cast<size_t>(at - index * args.page_size) * kD;
  };

  float run_max[kOctets][2], run_sum[kOctets][2], out[kOctets][kTiles][4];
#pragma unroll
  for (int o = 0; o < kOctets; ++o) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      run_max[o][i] = -INFINITY;
      run_sum[o][i] = 0.0f;
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) out[o][t][e] = 0.0f;
  }

  int nth = 0;
  for (int step = warp; step < steps; step += kRwWarps, ++nth) {
    const int kb = begin + step * kRwKeys;
    uint4 ka[kSegs], kc[kSegs], v[kRounds][4];
    {
      const bf16 *k_near, *k_far, *v_row[4];
      if (in_page) {
        if (nth == 32) {
          nth = 0;
          my_page = page_of_step(step + kRwWarps * lane);
        }
        const int page = checked(__shfl_sync(0xffffffffu, my_page, nth));
        const bf16* base = head + static_cast<size_t>(page) * 2 * v_plane;
        const int at = kb % args.page_size, low = max(first - kb, 0), high = min(end - kb, kRwKeys) - 1;
        auto inside = [&](int i) { return base + static_cast<size_t>(at + min(max(i, low), high)) * kD; };
        k_near = inside(g);
        k_far = inside(g + 8);
        v_row[0] = inside(2 * c);
        v_row[1] = inside(2 * c + 1);
        v_row[2] = inside(2 * c + 8);
        v_row[3] = inside(2 * c + 9);
      } else {
        k_near = row_of(kb + g);
        k_far = row_of(kb + g + 8);
        v_row[0] = row_of(kb + 2 * c);
        v_row[1] = row_of(kb + 2 * c + 1);
        v_row[2] = row_of(kb + 2 * c + 8);
        v_row[3] = row_of(kb + 2 * c + 9);
      }
#pragma unroll
      for (int s = 0; s < kSegs; ++s) {
        ka[s] = __ldcg(reinterpret_cast<const uint4*>(k_near + 32 * s + 8 * c));
        kc[s] = __ldcg(reinterpret_cast<const uint4*>(k_far + 32 * s + 8 * c));
      }
#pragma unroll
      for (int r = 0; r < kRounds; ++r)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[r][k] = __ldcg(reinterpret_cast<const uint4*>(v_row[k] + v_plane + 64 * r + 8 * g));
    }
    uint32_t p_near[kOctets], p_far[kOctets];
#pragma unroll
    for (int o = 0; o < kOctets; ++o) {
      float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kSegs; ++i) {
        rw_mma(s, ka[i].x, kc[i].x, ka[i].y, kc[i].y, q[o][i].x, q[o][i].y);
        rw_mma(s, ka[i].z, kc[i].z, ka[i].w, kc[i].w, q[o][i].z, q[o][i].w);
      }
      // s[0], s[1]: key kb + g of rows 2 c, 2 c + 1; s[2], s[3]: key kb + g + 8
      float alpha[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int j = kb + g + 8 * h;
          float x = s[2 * h + i] * args.scale_log2;
          if constexpr (kSloped) x = fmaf(slope[o][i], static_cast<float>(j - pos[o][i]), x);
          s[2 * h + i] = j >= first && j <= limit[o][i] ? x : -INFINITY;
        }
        float top = fmaxf(s[i], s[2 + i]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const float now = fmaxf(run_max[o][i], top), safe = now == -INFINITY ? 0.0f : now;
        alpha[i] = exp2f(run_max[o][i] - safe);      // 0 while nothing was seen
        run_max[o][i] = now;
        s[i] = exp2f(s[i] - safe);
        s[2 + i] = exp2f(s[2 + i] - safe);
        run_sum[o][i] = run_sum[o][i] * alpha[i] + (s[i] + s[2 + i]);
      }
      p_near[o] = rw_transpose(pack_bf16(s[0], s[1]));
      p_far[o] = rw_transpose(pack_bf16(s[2], s[3]));
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        out[o][t][0] *= alpha[0];
        out[o][t][1] *= alpha[1];
        out[o][t][2] *= alpha[0];
        out[o][t][3] *= alpha[1];
      }
    }
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        // word t of a lane's 16 bytes: d = 64 r + 8 g + 2 t and the one behind it; rows g and g + 8 of the operand
        const uint32_t x0 = rw_word(v[r][0], t), x1 = rw_word(v[r][1], t), x2 = rw_word(v[r][2], t), x3 = rw_word(v[r][3], t);
        const uint32_t a0 = __byte_perm(x0, x1, 0x5410), a1 = __byte_perm(x0, x1, 0x7632);
        const uint32_t a2 = __byte_perm(x2, x3, 0x5410), a3 = __byte_perm(x2, x3, 0x7632);
#pragma unroll
        for (int o = 0; o < kOctets; ++o) rw_mma(out[o][r * 4 + t], a0, a1, a2, a3, p_near[o], p_far[o]);
      }
    }
  }

  // the warps' states over their keys, joined through shared memory
#pragma unroll
  for (int o = 0; o < kOctets; ++o) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float total = run_sum[o][i];
      total += __shfl_xor_sync(0xffffffffu, total, 4);
      total += __shfl_xor_sync(0xffffffffu, total, 8);
      total += __shfl_xor_sync(0xffffffffu, total, 16);
      const int r = o * 8 + 2 * c + i;
      if (g == 0) {
        merge_max[warp][r] = run_max[o][i];
        merge_sum[warp][r] = total;
      }
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
        *reinterpret_cast<float2*>(&merge_o[warp][r][(t >> 2) * 64 + 8 * g + 2 * (t & 3)]) = make_float2(out[o][t][i], out[o][t][2 + i]);
    }
  }
  __syncthreads();
  for (int r = warp; r < rows; r += kRwWarps) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRwWarps; ++w) top = fmaxf(top, merge_max[w][r]);
    const float safe = top == -INFINITY ? 0.0f : top;
    float weight[kRwWarps], total = 0.0f;
#pragma unroll
    for (int w = 0; w < kRwWarps; ++w) {
      weight[w] = exp2f(merge_max[w][r] - safe);
      total += weight[w] * merge_sum[w][r];
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int p = row0 + r, token = members[p / group];
    const size_t at = static_cast<size_t>(args.part_first[token] + part) * args.hq + kv_head * group + p % group;
    if (lane * 4 < kD) {
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kRwWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(&merge_o[w][r][lane * 4]);
        sum.x = fmaf(weight[w], x.x, sum.x);
        sum.y = fmaf(weight[w], x.y, sum.y);
        sum.z = fmaf(weight[w], x.z, sum.z);
        sum.w = fmaf(weight[w], x.w, sum.w);
      }
      *reinterpret_cast<float4*>(args.part_out + at * kD + lane * 4) = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
    }
    if (lane == 0) args.part_lse[at] = total == 0.0f ? -INFINITY : top + log2f(total);
  }
  if (args.early) pdl_wait();                  // so that what follows this kernel follows the one before it too
}

}  // namespace RL_ATTENTION_NS
}  // namespace rl
