// Attention of a group's rows over its shared keys on the 5th-generation tensor cores (items: attention_shared.h).
//
//     S[row, key] = Q[row, :] . K[key, :]      tcgen05.mma  M = 128, N = 128 keys, K = D
//     O[row, d]  += P[row, key] . V[key, d]    A = P from tensor memory, B = V as it lies in the cache, M = 128, N = D
//
// A thread owns a row (a lane of S and O), so maxima and sums need no exchange; P takes the columns of S, O is rescaled
// only where a row's reference point moves by more than 2^8.  Two warpgroups of softmax threads alternate, so that the tensor core
// has work while one of them exponentiates:
//   * up to 256 rows (two tiles): a warpgroup a tile of 128 rows, both against every block of keys;
//   * up to 128 rows: both hold the SAME rows, one takes the even blocks, the other the odd ones, each with a
//     reference point, a sum and an O of its own, joined through shared memory at the end.
// A block of 128 keys and values is 64 KB, which a multiprocessor gets from HBM in some 2,800 cycles when all of them read;
// its two products of 128 rows take 1,024 (256 rows: 2,048), so the keys' stream bounds the kernel up to 256 rows a key
// head whatever part of a tile the rows fill, and warps without rows skip the softmax.  The stream is TMA, page by page, into
// rings of two (256 rows) or three blocks.  Shared keys were written by earlier steps: the copies start before the wait
// for the kernel before.
//
// Measured: 2 us until the first copies are asked for, 2.7 for the queries, then 1.83 us a block for two tiles (0.95 of
// softmax and 0.88 of products a tile, the tiles in strict turn: the tensor core, which reads Q or V from shared memory at its
// full rate, is the longer half) or 0.98 us for one (104 CTAs and more then take all of HBM's rate), and 3.7 us to the results.
// 64 requests, 32 heads on 8, 32,000 shared and 512 own keys: 58 us beside 21 of row items and 8 of the join; 8,192 keys and up to
// 512 ragged own ones: 28, 21 and 7, one over the other 43, where each request for itself takes 220; 40 heads on 8, 32,000 and up to 1,024: 69 (320
// rows: an item of 256 and one of 64 over each range, and the one of 64 takes as long a block), 31 and 7, one over the other 106.
// Tried and slower: scores of 64 keys a unit ahead (72 -> 87 us: Q is read as often for 64 keys as for 128), a share of the
// exponentials as polynomials on the multiply-add pipes (-1 % to +8 %).
#pragma once

#include "attention_prefill_tc.cuh"

namespace rl {
namespace RL_ATTENTION_NS {

constexpr int kShD = 128;
constexpr int kShKeys = 128;
constexpr int kShTileRows = 128;
constexpr int kShFirstSoftmaxWarp = 4;          // warp 0: TMA of keys, warp 1: TMA of values, warp 2: products, warp 3: idle
constexpr int kShThreads = kShFirstSoftmaxWarp * 32 + 256;
constexpr int kShFewRegisters = 80, kShManyRegisters = 208;      // as in the prompt kernel: 128 scores a thread stay in registers
static_assert(128 * kShFewRegisters + 256 * kShManyRegisters <= kShThreads * (65536 / kShThreads / 8 * 8), "register budgets of the warpgroups");
constexpr int kShHalfBytes = 128 * 128;
constexpr int kShTileBytes = 2 * kShHalfBytes;
constexpr int kShStagedPages = 256;
constexpr int kShOutStride = kShD + 4;          // floats from a row of the exchange to the next: no two lanes in one bank
constexpr int sh_stages(bool two_tiles) { return two_tiles ? 2 : 3; }
constexpr int sh_smem_bytes(bool two_tiles) { return ((two_tiles ? 2 : 1) + 2 * sh_stages(two_tiles)) * kShTileBytes + 1024; }
static_assert(2 * kShTileRows * kShOutStride * 4 <= sh_smem_bytes(true) - 1024 && kShTileRows * (kShOutStride + 2) * 4 <= sh_smem_bytes(false) - 1024,
              "the rows' results fit where the tiles were");

// Rows `first` .. 127 of a tile of 128 keys (two halves of 128-byte rows) become zeros, by one warp, for the tensor cores to see.
__device__ __forceinline__ void sh_clear_rows(uint32_t tile, int first, int lane) {
  for (int i = first * 16 + lane; i < kShKeys * 16; i += 32) {
    const uint32_t at = tile + ((i >> 3) & 1) * kShHalfBytes + (i >> 4) * 128 + (i & 7) * 16;
    asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(at), "r"(0) : "memory");
  }
  fence_async_smem();
  __syncwarp();
}

struct SharedTcArgs {
  const bf16* q;
  float* part_out;
  float* part_lse;
  const int* items;
  const int* members;
  const int* positions;
  const int* part_first;
  const int* entry_slot;
  const int* block_table;
  int hq, hkv, page_size, num_pages, max_pages, slots;
  float scale_log2;
  const float* slopes;
  int* fault;
};

template <bool kTwoTiles, bool kSloped>
__global__ void __launch_bounds__(kShThreads, 1)
attention_shared_tc_kernel(const __grid_constant__ CUtensorMap map_cache, const SharedTcArgs args) {
  constexpr int kStages = sh_stages(kTwoTiles), kQTiles = kTwoTiles ? 2 : 1;
  extern __shared__ unsigned char sh_smem_raw[];
  __shared__ __align__(8) uint64_t full_k[kStages], full_v[kStages], empty_k[kStages], empty_v[kStages];
  __shared__ __align__(8) uint64_t score_ready[2], p_ready[2], value_done[2];
  __shared__ __align__(8) uint64_t q_ready, drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int aborted_flag;
  __shared__ int staged_pages[kShStagedPages];
  __shared__ int part_rows[kQTiles * kShTileRows];       // where each row's result goes
  volatile int* aborted = &aborted_flag;

  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  const uint32_t base = (smem_addr(sh_smem_raw) + 1023u) & ~1023u;
  auto q_tile = [&](int tile) { return base + tile * kShTileBytes; };
  auto k_tile = [&](int s) { return base + (kQTiles + s) * kShTileBytes; };
  auto v_tile = [&](int s) { return base + (kQTiles + kStages + s) * kShTileBytes; };

  // ---- the item ------------------------------------------------------------------------
  const int* item = args.items + static_cast<size_t>(blockIdx.y) * kListedInts;
  const int rows = min(item[kListedRows], kQTiles * kShTileRows);
  if (rows <= 0) {                                   // a place of the list that holds no item
    pdl_wait();
    pdl_trigger();
    return;
  }
  const int row0 = item[kListedRow0], part = item[kListedPart], fresh = item[kListedFresh];
  const int kv_head = blockIdx.x;
  const int group = args.hq / args.hkv;
  const int slot = args.entry_slot[item[0]];
  const int first = item[kListedFirst];
  const bool bad = slot < 0 || slot >= args.slots || first < 0 || item[kListedEnd] > args.max_pages * args.page_size;
  if (bad && tid == 0) atomicOr(args.fault, (slot < 0 || slot >= args.slots) ? kFaultSlot : kFaultPosition);
  const int k_end = bad ? 0 : item[kListedEnd];
  const int box_rows = min(args.page_size, kShKeys);
  const int k_begin = first - first % box_rows;      // a block starts where a box of the copies does
  const int n_blocks = k_end > first && !bad ? (k_end - k_begin + kShKeys - 1) / kShKeys : 0;
  const int* members = args.members + item[kListedMembers];
  const int* table = args.block_table + static_cast<size_t>(bad ? 0 : slot) * args.max_pages;
  // streams of work for the tensor core: the tiles that have rows, or the even and the odd blocks of one tile
  const int tiles = kTwoTiles && rows > kShTileRows ? 2 : 1;
  const int steps = kTwoTiles ? n_blocks * tiles : n_blocks;
  auto block_of = [&](int step) { return kTwoTiles ? (tiles == 2 ? step >> 1 : step) : step; };
  auto stream_of = [&](int step) { return kTwoTiles ? (tiles == 2 ? step & 1 : 0) : step & 1; };
  auto index_of = [&](int step) { return kTwoTiles ? block_of(step) : step >> 1; };    // among the stream's own blocks
  auto last_use = [&](int step) { return !kTwoTiles || tiles == 1 || (step & 1); };    // of the step's block

  // ---- set-up --------------------------------------------------------------------------
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_addr(&full_k[s]), 1);
      mbar_init(smem_addr(&full_v[s]), 1);
      mbar_init(smem_addr(&empty_k[s]), 1);
      mbar_init(smem_addr(&empty_v[s]), 1);
    }
    for (int st = 0; st < 2; ++st) {
      const int rows_here = kTwoTiles ? min(kShTileRows, max(rows - st * kShTileRows, 0)) : rows;
      mbar_init(smem_addr(&score_ready[st]), 1);
      mbar_init(smem_addr(&p_ready[st]), max(1, (rows_here + 31) >> 5));     // the warps that have rows
      mbar_init(smem_addr(&value_done[st]), 1);
    }
    mbar_init(smem_addr(&q_ready), 4 * kQTiles);
    mbar_init(smem_addr(&drained), 1);
    aborted_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    tmem_alloc(smem_addr(&tmem_slot), 512);
    tmem_relinquish();
  }
  const int first_page = k_begin / args.page_size;
  const int page_count = n_blocks > 0 ? (k_end - 1) / args.page_size - first_page + 1 : 0;
  const bool staged = page_count <= kShStagedPages;
  if (staged) {
    for (int i = tid; i < page_count; i += kShThreads) {
      int page = table[first_page + i];
      if (page < 0 || page >= args.num_pages) {
        atomicOr(args.fault, kFaultPageId);
        page = 0;
      }
      staged_pages[i] = page;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = uniform(tmem_slot);
  auto tmem_score = [&](int st) { return tmem_base + st * 256; };        // 128 columns; P over its first 64
  auto tmem_out = [&](int st) { return tmem_base + st * 256 + 128; };    // 128 columns

  if (warp < kShFirstSoftmaxWarp) {
    register_budget_down<kShFewRegisters>();
    if (warp < 2) {
      // -------------------------------------------------------------------- TMA producers
      const int is_value = warp;
      uint64_t* fulls = is_value ? full_v : full_k;
      uint64_t* empties = is_value ? empty_v : empty_k;
      const int boxes = kShKeys / box_rows;
      bool waited = false, ok = true;
      int issued = 0;
      for (int b = 0; b < n_blocks && ok; ++b) {
        const int stage = b % kStages;
        const int kb = k_begin + b * kShKeys;
        if (b >= kStages) {
          int got = 1;
          if (lane == 0)
            got = mbar_wait(smem_addr(&empties[stage]), ((b / kStages) - 1) & 1, aborted, args.fault) ? 1 : 0;
          ok = __shfl_sync(0xffffffffu, got, 0) != 0;
          if (!ok) break;
        }
        if (!waited && kb + kShKeys > fresh) {
          pdl_wait();
          waited = true;
        }
        if (lane == 0) mbar_expect_tx(smem_addr(&fulls[stage]), kShTileBytes);
        __syncwarp();
        for (int i = lane; i < boxes * 2; i += 32) {
          const int x = i >> 1, half = i & 1;
          const int j = kb + x * box_rows;                   // first key of the box
          int page = 0, in_page = 0;                         // past the range: any readable page, masked and cleared later
          if (j < k_end) {
            const int page_index = j / args.page_size;
            in_page = j - page_index * args.page_size;
            if (staged) {
              page = staged_pages[page_index - first_page];
            } else {
              page = table[page_index];
              if (page < 0 || page >= args.num_pages) {
                atomicOr(args.fault, kFaultPageId);
                page = 0;
              }
            }
          }
          const int row = ((page * 2 + is_value) * args.hkv + kv_head) * args.page_size + in_page;
          const uint32_t dst = (is_value ? v_tile(stage) : k_tile(stage)) + half * kShHalfBytes + x * box_rows * 128;
          tma_load_2d(dst, &map_cache, smem_addr(&fulls[stage]), half * 64, row);
        }
        ++issued;
      }
      if (!waited) pdl_wait();
      if (lane == 0 && n_blocks > 0 && (!ok || *aborted)) {
        // copies in flight must land before the CTA may exit, whoever gave up
        volatile int go_on = 0;
        for (int s = 0; s < kStages; ++s) {
          const int fills = (issued - s + kStages - 1) / kStages;
          if (fills > 0) mbar_wait(smem_addr(&fulls[s]), (fills - 1) & 1, &go_on, args.fault);
        }
      }
    } else if (warp == 2) {
      // -------------------------------------------------------------------- tensor-core issuer
      // Step i: the values' product of its block and stream once P is written, then the scores of the stream's next
      // block, which overwrite the columns that held P (products run in the order they are issued).
      const int total = uniform(steps);
      const int kb_end = uniform(k_begin + n_blocks * kShKeys);
      const int ahead = kTwoTiles ? uniform(tiles) : 2;
      const bool issues = elect_one();
      auto wait = [&](uint64_t* bar, int phase) {
        return __all_sync(0xffffffffu, mbar_wait(smem_addr(bar), phase & 1, aborted, args.fault));
      };
      bool ok = total > 0;
      if (ok) ok = wait(&q_ready, 0);
      auto issue_scores = [&](int step) {
        const int b = block_of(step), st = stream_of(step), stage = b % kStages;
        if (!wait(&full_k[stage], b / kStages)) return false;
        tc_fence_after();
        const uint64_t q_desc = operand_desc(q_tile(kTwoTiles ? st : 0)), keys_desc = operand_desc(k_tile(stage));
        if (issues) {
#pragma unroll
          for (int k = 0; k < kShD / 16; ++k) {
            const uint32_t half = (k >> 2), within = (k & 3) * 2;
            umma_bf16(tmem_score(st), q_desc + half * (kShHalfBytes >> 4) + within, keys_desc + half * (kShHalfBytes >> 4) + within,
                      kPfIdescScore, k > 0 ? 1u : 0u);
          }
          umma_commit(smem_addr(&score_ready[st]));
          if (last_use(step)) umma_commit(smem_addr(&empty_k[stage]));
        }
        __syncwarp();
        return true;
      };
      for (int step = 0; step < min(ahead, total) && ok; ++step) ok = issue_scores(step);
      for (int step = 0; step < total && ok; ++step) {
        const int b = block_of(step), st = stream_of(step), j = index_of(step), stage = b % kStages;
        ok = wait(&p_ready[st], j) && wait(&full_v[stage], b / kStages);
        if (!ok) break;
        // what came along beyond the keys' end is cleared before its first use: zero times a NaN is no zero
        if (b == n_blocks - 1 && kb_end > k_end && (!kTwoTiles || st == 0)) sh_clear_rows(v_tile(stage), k_end - (kb_end - kShKeys), lane);
        tc_fence_after();
        const uint64_t values_desc = operand_desc_mn(v_tile(stage), kShHalfBytes);
        if (issues) {
#pragma unroll
          for (int k = 0; k < kShKeys / 16; ++k)
            umma_bf16_ts(tmem_out(st), tmem_score(st) + k * 8, values_desc + k * (2048 >> 4), kPfIdescValue, (j > 0 || k > 0) ? 1u : 0u);
          umma_commit(smem_addr(&value_done[st]));
          if (last_use(step)) umma_commit(smem_addr(&empty_v[stage]));
        }
        __syncwarp();
        if (step + ahead < total) ok = issue_scores(step + ahead);
      }
      if (issues) umma_commit(smem_addr(&drained));
      __syncwarp();
      volatile int go_on = 0;                            // products in flight end, whoever gave up
      mbar_wait(smem_addr(&drained), 0, &go_on, args.fault);
    }
  } else {
    // -------------------------------------------------------------------- softmax and output
    register_budget_up<kShManyRegisters>();
    const int st = (warp - kShFirstSoftmaxWarp) >> 2;
    const int tile = kTwoTiles ? st : 0;
    const int quarter = warp & 3;                      // tensor-memory lanes this warp may touch
    const int r = quarter * 32 + lane;                 // row of the tile = lane of S and O
    const uint32_t lane_bits = static_cast<uint32_t>(quarter * 32) << 16;
    const int rows_here = kTwoTiles ? min(kShTileRows, max(rows - st * kShTileRows, 0)) : rows;
    const bool works = quarter * 32 < rows_here;       // the warp has rows
    const bool valid = r < rows_here;
    const int p = row0 + tile * kShTileRows + r;
    const int token = valid ? members[p / group] : 0;
    const int head = kv_head * group + p % group;
    const int pos = valid ? args.positions[token] : -1;
    const int limit = min(pos, k_end - 1);             // last key the row sees here
    const int q_row = token * args.hq + head;
    const int part_row = (args.part_first[token] + part) * args.hq + head;
    if (kTwoTiles || st == 0) part_rows[tile * kShTileRows + r] = part_row;
    pdl_wait();                                        // queries come from the kernel before
    pdl_trigger();                                     // from here on nothing that follows needs to wait for that one
    if (kTwoTiles || st == 0) {
      // the warp's 32 rows of Q into the K-major operand [row][64] x 2 halves, swizzled: two rows an instruction
      uint4 fetched[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int rr = quarter * 32 + 2 * i + (lane >> 4);
        const int from = __shfl_sync(0xffffffffu, q_row, rr & 31);       // (a lane knows its own row)
        fetched[i] = make_uint4(0, 0, 0, 0);
        if (rr < rows_here) fetched[i] = __ldcg(reinterpret_cast<const uint4*>(args.q + static_cast<size_t>(from) * kShD + (lane & 15) * 8));
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int rr = quarter * 32 + 2 * i + (lane >> 4), c = lane & 15;
        const uint32_t dst = q_tile(tile) + (c >> 3) * kShHalfBytes + rr * 128 + (((c & 7) ^ (rr & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(fetched[i].x), "r"(fetched[i].y), "r"(fetched[i].z), "r"(fetched[i].w) : "memory");
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&q_ready));
    }

    const int my_blocks = !works ? 0 : kTwoTiles ? n_blocks : (n_blocks - st + 1) >> 1;
    const float post_scale = kSloped ? 1.0f : args.scale_log2;
    const float slope_log2 = kSloped && valid ? args.slopes[head] * 1.4426950408889634f : 0.0f;
    float ref_max = -INFINITY;                         // exponentials are taken against ref_max
    unsigned long long row_sum2 = pf_pack2(0.0f, 0.0f);
    bool ok = true;
    for (int j = 0; j < my_blocks && ok; ++j) {
      const int b = kTwoTiles ? j : 2 * j + st;
      const int kb = k_begin + b * kShKeys;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_addr(&score_ready[st]), j & 1, aborted, args.fault));
      if (!ok) break;
      tc_fence_after();
      uint32_t score[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_load32(tmem_score(st) + lane_bits + c * 32, score[c]);
      tmem_wait_ld();
      if constexpr (kSloped) {
        const float nearest = slope_log2 * static_cast<float>(kb - pos);
        const unsigned long long in2 = pf_pack2(args.scale_log2, args.scale_log2), slope2 = pf_pack2(slope_log2, slope_log2);
        const unsigned long long nearest2 = pf_pack2(nearest, nearest);
#pragma unroll
        for (int i = 0; i < kShKeys; i += 2) {
          const unsigned long long at2 = pf_pack2(static_cast<float>(i), static_cast<float>(i + 1));
          const unsigned long long bias2 = pf_fma2(slope2, at2, nearest2);
          float x0, x1;
          pf_unpack2(pf_fma2(pf_pack2(__uint_as_float(score[i >> 5][i & 31]), __uint_as_float(score[(i + 1) >> 5][(i + 1) & 31])), in2, bias2), x0, x1);
          score[i >> 5][i & 31] = __float_as_uint(x0);
          score[(i + 1) >> 5][(i + 1) & 31] = __float_as_uint(x1);
        }
      }
      if (__any_sync(0xffffffffu, kb + kShKeys - 1 > limit || kb < first)) {
#pragma unroll
        for (int i = 0; i < kShKeys; ++i) {
          const int key = kb + i;
          if (!(key <= limit && key >= first)) score[i >> 5][i & 31] = 0xff800000u;
        }
      }
      float lane_max[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) lane_max[i] = __uint_as_float(score[0][i]);
#pragma unroll
      for (int i = 8; i + 16 <= kShKeys; i += 16) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          lane_max[c] = pf_max3(lane_max[c], __uint_as_float(score[(i + c) >> 5][(i + c) & 31]),
                                __uint_as_float(score[(i + c + 8) >> 5][(i + c + 8) & 31]));
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) lane_max[c] = fmaxf(lane_max[c], __uint_as_float(score[3][24 + c]));
      // (a scale below zero turns the order round: then the smallest counts; see the caller, which refuses it)
      float block_max = fmaxf(fmaxf(fmaxf(lane_max[0], lane_max[1]), fmaxf(lane_max[2], lane_max[3])),
                              fmaxf(fmaxf(lane_max[4], lane_max[5]), fmaxf(lane_max[6], lane_max[7])));
      block_max *= post_scale;
      const bool moves = block_max > ref_max + kPfRescaleStep || (ref_max == -INFINITY && block_max > -INFINITY);
      float alpha = 1.0f;
      if (moves) {
        alpha = ref_max == -INFINITY ? 0.0f : fast_exp2(ref_max - block_max);
        ref_max = block_max;
        float even, odd;
        pf_unpack2(row_sum2, even, odd);
        row_sum2 = pf_pack2(even * alpha, odd * alpha);
      }
      // the stream's values product of the block before ran before these scores: O may be rescaled without a further wait
      if (j > 0 && __any_sync(0xffffffffu, moves)) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t raw[32];
          tmem_load32(tmem_out(st) + lane_bits + c * 32, raw);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) raw[i] = __float_as_uint(__uint_as_float(raw[i]) * alpha);
          tmem_store32(tmem_out(st) + lane_bits + c * 32, raw);
        }
      }
      const float shift = ref_max == -INFINITY ? 0.0f : ref_max;
      const unsigned long long scale2 = pf_pack2(post_scale, post_scale), shift2 = pf_pack2(-shift, -shift);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t packed[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x0, x1;
          pf_unpack2(pf_fma2(pf_pack2(__uint_as_float(score[c][2 * i]), __uint_as_float(score[c][2 * i + 1])), scale2, shift2), x0, x1);
          const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);
          row_sum2 = pf_add2(row_sum2, pf_pack2(e0, e1));
          const __nv_bfloat162 pair = __floats2bfloat162_rn(e0, e1);
          packed[i] = *reinterpret_cast<const uint32_t*>(&pair);
        }
        tmem_store16(tmem_score(st) + lane_bits + c * 16, packed);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&p_ready[st]));
    }
    if (ok && my_blocks > 0) ok = mbar_wait(smem_addr(&value_done[st]), (my_blocks - 1) & 1, aborted, args.fault);
    // both streams are through their products: the tiles' room is free
    ok = named_barrier_and(1, 256, ok);
    if (ok) {
      tc_fence_after();
      float* exchange = reinterpret_cast<float*>(sh_smem_raw + (base - smem_addr(sh_smem_raw)));
      float* other_max = exchange + kShTileRows * kShOutStride;        // of the odd blocks' stream
      float* other_sum = other_max + kShTileRows;
      float even, odd;
      pf_unpack2(row_sum2, even, odd);
      float row_sum = even + odd;
      float* mine = exchange + ((kTwoTiles ? st * kShTileRows : 0) + r) * kShOutStride;
      const bool has = my_blocks > 0;
      if (!kTwoTiles) {
        if (st == 1 && works) {
          if (has) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t raw[32];
              tmem_load32(tmem_out(st) + lane_bits + c * 32, raw);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<float4*>(mine + c * 32 + i) = make_float4(__uint_as_float(raw[i]), __uint_as_float(raw[i + 1]),
                                                                            __uint_as_float(raw[i + 2]), __uint_as_float(raw[i + 3]));
            }
          }
          other_max[r] = ref_max;
          other_sum[r] = row_sum;
        }
        named_barrier(1, 256);
      }
      if (works && (kTwoTiles || st == 0)) {
        float w0 = 1.0f, w1 = 0.0f, top = ref_max;
        if (!kTwoTiles) {
          const float theirs = other_max[r];
          top = fmaxf(ref_max, theirs);
          const float safe = top == -INFINITY ? 0.0f : top;
          w0 = fast_exp2(ref_max - safe);
          w1 = fast_exp2(theirs - safe);
          row_sum = row_sum * w0 + other_sum[r] * w1;
        }
        const float inv = row_sum > 0.0f ? 1.0f / row_sum : 0.0f;
        const bool both = !kTwoTiles && n_blocks > 1;
        if (has) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t raw[32];
            tmem_load32(tmem_out(st) + lane_bits + c * 32, raw);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              float4 v = make_float4(__uint_as_float(raw[i]) * w0, __uint_as_float(raw[i + 1]) * w0, __uint_as_float(raw[i + 2]) * w0,
                                     __uint_as_float(raw[i + 3]) * w0);
              if (both) {
                const float4 o = *reinterpret_cast<const float4*>(mine + c * 32 + i);
                v.x = fmaf(o.x, w1, v.x);
                v.y = fmaf(o.y, w1, v.y);
                v.z = fmaf(o.z, w1, v.z);
                v.w = fmaf(o.w, w1, v.w);
              }
              *reinterpret_cast<float4*>(mine + c * 32 + i) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
            }
          }
        }
        if (valid) args.part_lse[part_row] = row_sum == 0.0f ? -INFINITY : top + log2f(row_sum);
      }
      named_barrier(1, 256);
      // whole rows of 512 bytes, a warp a row
      if (n_blocks > 0) {
#pragma unroll 4
        for (int rr = warp - kShFirstSoftmaxWarp; rr < rows; rr += 8)
          *reinterpret_cast<float4*>(args.part_out + static_cast<size_t>(part_rows[rr]) * kShD + lane * 4) =
              *reinterpret_cast<const float4*>(exchange + rr * kShOutStride + lane * 4);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace RL_ATTENTION_NS
}  // namespace rl
