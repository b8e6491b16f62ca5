// acc[m, n] = sum_k A(m, k) B(n, k) of bf16 or fp16 matrices, on CTA pairs, with the epilogues of a head's cross entropy.
//
// A persistent kernel of clusters of two CTAs, one CTA per SM; a pair takes 256 x 256 tiles one after another:
//   warp 0, one lane : TMA producer - this CTA's 128 rows of A and its 128 of the tile's 256 rows of B, 64 of K, per stage of 32 KB
//   warp 1, one lane : MMA issuer (leader CTA) - M 256 x N 256 x K 16, cta_group::2
//   warps 4..        : epilogue - each a quarter of the CTA's 128 rows; logits: sixteen warps of 64 columns, products: eight of 128.  Their
//                      warpgroups take the registers that the first one (two of whose warps are idle) gives back
// The accumulator takes 256 of TMEM's 512 columns, so that the epilogue of a tile runs beside the products of the next.
// Operands whose M or N runs along memory's rows go in as they lie (kUmmaMnMajorA, kUmmaMnMajorB): the gradients' products
// read the logits' gradient in both directions, and no matrix is transposed.
//
// What bounds it: a pair's tile takes 64 KB of L2's bandwidth every 512 cycles of products, 64 bytes a cycle and SM, which is all that an SM gets; and
// the power cap in long runs.  8192 x 4096 x 128256 alone 1.31 PFLOP/s (torch.matmul 1.55), for seconds 1.21 to 1.24 (1.29 to 1.37).  At 4096 x 4096
// x 16032 the tensor pipe is busy for 79 (exponentials), 86 and 84 % of a launch, of 97 % that its rounds of tiles allow.  Tried and not kept:
// tiles fetched into L2 ahead of their loads (416 -> 493 us), a producer thread for each operand (566 -> 574 thousand cycles), waits of the
// producer that suspend it (541 -> 583 thousand; those of the epilogue, which are long, do).
//
// The tensor core truncates as it adds: some 2^-24 of the running sum per 16 of K.  Logits are drained from TMEM into sums in registers (round
// to nearest) every 2048 of K (`drain`; every 256 where few tokens count), gradients once: 5e-4 of one over 128256 words at most, a quarter of what its rounding to bf16 costs.
// Draining every 256 of K costs 150 of 690 thousand cycles at 4096 x 16032 x 4096: handing the accumulator over takes the tensor core about
// 700 cycles, whatever the epilogue does meanwhile.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "gemm16.h"
#include "launch_util.h"
#include "ptx.cuh"
#include "tensor_map.h"
#include "value16.cuh"

namespace soapb200 {
namespace {

constexpr int kTile = 256;                       // of the pair, both ways
constexpr int kRows = 128;                       // of a CTA, of either operand
constexpr int kBK = 64;                          // one 128-byte swizzle row of K-major operands
constexpr int kOperandBytes = kRows * kBK * 2;
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kStages = 6;
constexpr int kStagingBytes = 32 * 1024;
constexpr int kSmemBytes = kStages * kStageBytes + kStagingBytes + 1024 + 256;
constexpr int kFirstEpiWarp = 4;
// What the two kinds of epilogue have.  `kFew` and `kMany`: registers of a thread of the first warpgroup and of the others, once shared
// out; together they are what the block is launched with, 640 * 96 or (less than) 384 * 168.
template <bool LOGITS>
struct Epi {
  static constexpr int kWarps = LOGITS ? 16 : 8;
  static constexpr int kThreads = 32 * (kFirstEpiWarp + kWarps);
  static constexpr int kColumns = kTile / (kWarps / 4);      // of the tile, per thread
  static constexpr int kStaging = kStagingBytes / kWarps;    // 32 rows of 64 or 128 bytes
  static constexpr int kFew = LOGITS ? 32 : 40, kMany = LOGITS ? 112 : 224;
};
static_assert(Epi<true>::kColumns == kLogitPart, "an epilogue thread's logits are one part of its row");
static_assert(128 * 32 + 512 * 112 <= 640 * 96 && 128 * 40 + 256 * 224 <= 384 * 168, "registers to share out");
constexpr int kGroup = 8;                        // tile rows that share their tiles of B in L2 while they sweep the columns
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));      // off by 2^-22 at most
  return y;
}

struct Tiles {
  int m, n, per_group;
  __device__ __forceinline__ Tiles(int M, int N) : m((M + kTile - 1) / kTile), n((N + kTile - 1) / kTile), per_group(kGroup * n) {}
  __device__ __forceinline__ int count() const { return m * n; }
  __device__ __forceinline__ void place(int index, int& m0, int& n0) const {
    const int first = index / per_group * kGroup;
    const int rows = min(kGroup, m - first);
    const int within = index % per_group;
    m0 = (first + within % rows) * kTile;
    n0 = within / rows * kTile;
  }
};

// 32 rows of LINE bytes, one per lane, to 32 rows of a matrix: staged in shared memory (16-byte words swizzled by row, so that
// neither side has bank conflicts) and stored LINE bytes at a time.  Row i is row where[first + i] of `base`, or first + i;
// `valid` bytes of each row are inside the matrix.
template <int LINE>
__device__ __forceinline__ void store_lines(uint8_t* staging, const uint32_t (&words)[LINE / 4], uint8_t* base, int64_t pitch, const int* where,
                                            int first, int rows, int valid, int element, bool wide, int lane) {
  constexpr int kChunks = LINE / 16;                   // of a row
  const int turn = kChunks == 8 ? lane : lane >> 1;    // (eight lanes that store together hit all banks)
#pragma unroll
  for (int c = 0; c < kChunks; ++c)
    *reinterpret_cast<uint4*>(staging + lane * LINE + ((c ^ (turn & (kChunks - 1))) << 4)) =
        make_uint4(words[4 * c], words[4 * c + 1], words[4 * c + 2], words[4 * c + 3]);
  __syncwarp();
  const int chunk = lane & (kChunks - 1);
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int row = (32 / kChunks) * i + lane / kChunks;
    const int row_turn = kChunks == 8 ? row : row >> 1;
    const uint4 v = *reinterpret_cast<const uint4*>(staging + row * LINE + ((chunk ^ (row_turn & (kChunks - 1))) << 4));
    if (row < rows) {
      uint8_t* dst = base + (where ? where[first + row] : first + row) * pitch + chunk * 16;
      const int left = valid - chunk * 16;
      if (wide && left >= 16) {
        *reinterpret_cast<uint4*>(dst) = v;
      } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if (element == 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * e < left) reinterpret_cast<uint32_t*>(dst)[e] = w[e];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (2 * e < left) reinterpret_cast<uint16_t*>(dst)[e] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
        }
      }
    }
  }
  __syncwarp();
}

// 32 rows of 16-bit values, from `column` of C on.
template <int LINE>
__device__ __forceinline__ void store_values(uint8_t* staging, const uint32_t (&words)[LINE / 4], const Gemm16Problem& p, int m_warp, int column,
                                             int rows, int cols, bool wide, int lane) {
  store_lines<LINE>(staging, words, reinterpret_cast<uint8_t*>(p.C) + static_cast<int64_t>(column) * 2, p.ldc * 2, p.where, m_warp, rows,
                    min(LINE, 2 * cols), 2, wide, lane);
}

// An epilogue thread's logits of one token, as pairs of neighbouring columns.
template <int EPI, typename T>
__device__ __forceinline__ void logits_epilogue(const Gemm16Problem& p, uint64_t (&sums)[kLogitPart / 2], int M, int m_warp, int n0,
                                                uint8_t* staging, int lane) {
  const int row = m_warp + lane;
  const bool inside = row < M;
  const int cols = min(kLogitPart, p.N - n0);             // of this thread's part; may be negative
  // (the gradient's rows up to the next multiple of 64 are cleared: they are read as part of K)
  const int rows = min(32, (EPI == kLogitGradient ? min(p.M, (M + kBK - 1) / kBK * kBK) : M) - m_warp);
  const int target = inside ? p.targets[row] - n0 : -1;
  const uint64_t scale = pack_floats(kLog2e, kLog2e);
  // sums become the exponents of two that their exponentials are
  auto exponents = [&](float base) {
    const uint64_t shift = pack_floats(-base, -base);
#pragma unroll
    for (int j = 0; j < kLogitPart / 2; ++j) {
      uint64_t v = shift;
      fma_pair(v, sums[j], scale);
      sums[j] = v;
    }
  };
  auto value = [&](int j) { return pair_element(sums[j / 2], j & 1); };
  if constexpr (EPI == kLogitGradient) {
    const int wide_cols = p.second ? min(kLogitPart, (p.N + kBK - 1) / kBK * kBK - n0) : cols;
    const float factor = inside ? p.factor[row] : 0.f;
    // from the loss itself: the target's probability, less one, is small where the model knows the word
    const float of_target = inside && target >= 0 && target < cols ? expm1f(-p.loss[row]) : 0.f;
    exponents(inside ? p.lse[row] * kLog2e : 0.f);
    auto gradient = [&](int j) { return inside && j < cols ? (target == j ? of_target : exp2_fast(value(j))) * factor : 0.f; };
#pragma unroll
    for (int c = 0; c < kLogitPart; c += 32) {
      uint32_t words[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) words[j] = pack2<T>(gradient(c + 2 * j), gradient(c + 2 * j + 1));
      if (rows > 0 && c < wide_cols) {
        store_values<64>(staging, words, p, m_warp, n0 + c, rows, wide_cols - c, true, lane);
        if (p.second) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 back = unpack2<T>(words[j]);
            words[j] = pack2<T>(gradient(c + 2 * j) - back.x, gradient(c + 2 * j + 1) - back.y);
          }
          store_values<64>(staging, words, p, m_warp, n0 + c + static_cast<int>(p.second), rows, wide_cols - c, true, lane);
        }
      }
    }
  } else {
    if (cols < kLogitPart) {
#pragma unroll
      for (int j = 0; j < kLogitPart; j += 2)
        sums[j / 2] = pack_floats(j < cols ? value(j) : -INFINITY, j + 1 < cols ? value(j + 1) : -INFINITY);
    }
    float most[4] = {value(0), value(1), value(2), value(3)};
#pragma unroll
    for (int j = 4; j < kLogitPart; ++j) most[j & 3] = fmaxf(most[j & 3], value(j));
    const float largest = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    // (a row of no finite logit is taken relative to zero, so that its sum is zero, or NaN where a logit is)
    constexpr float kUp = EPI == kLogitExponential ? 15.f : 0.f;
    exponents(largest == -INFINITY ? -kUp : largest * kLog2e - kUp);
    uint64_t sum[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < kLogitPart; j += 2) {
      sums[j / 2] = pack_floats(exp2_fast(value(j)), exp2_fast(value(j + 1)));
      add_pair(sum[(j >> 1) & 1], sums[j / 2]);
    }
    add_pair(sum[0], sum[1]);
    float others = pair_element(sum[0], 0) + pair_element(sum[0], 1);
    if (inside && target >= 0 && target < cols) {      // (added up without it: where the model knows the word, nothing would be left of a difference)
      others = 0.f;
#pragma unroll
      for (int j = 0; j < kLogitPart; ++j) others += target == j ? 0.f : value(j);
    }
    if (inside && cols > 0)
      p.parts[static_cast<int64_t>(n0 / kLogitPart) * p.ld_parts + row] = make_float2(largest, EPI == kLogitExponential ? others * (1.f / 32768.f) : others);
    if constexpr (EPI == kLogitExponential) {
#pragma unroll
      for (int c = 0; c < kLogitPart; c += 32) {
        uint32_t words[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) words[j] = pack2<__half>(value(c + 2 * j), value(c + 2 * j + 1));
        if (rows > 0 && c < cols) store_values<64>(staging, words, p, m_warp, n0 + c, rows, cols - c, true, lane);
      }
    }
  }
}

// An epilogue thread's row of a product.  values(at, raw): its 32 sums from column `at` of its 128 on.
template <typename T, typename Values>
__device__ __forceinline__ void product_epilogue(const Gemm16Problem& p, int M, int m_warp, int n0, uint8_t* staging, int lane, Values values) {
  const int row = m_warp + lane;
  const bool inside = row < M;
  const int cols = min(Epi<false>::kColumns, p.N - n0);
  const int rows = min(32, M - m_warp);
  const float alpha = p.alpha ? *p.alpha : 1.f;
  const bool to16 = p.C != nullptr;
  const bool wide = (reinterpret_cast<uintptr_t>(p.C) & 15) == 0 && (p.ldc & 7) == 0;
#pragma unroll
  for (int c = 0; c < Epi<false>::kColumns; c += 64) {
    uint32_t words[32];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t raw[32];
      const int at = c + 32 * h;
      values(at, raw);
      if (p.add && inside && at < cols) {
        const float* old = p.accumulator + row * p.ld_accumulator + n0 + at;
#pragma unroll
        for (int j = 0; j < 32; j += 4) {               // (the accumulator's pitch is a multiple of 32)
          const float4 v = *reinterpret_cast<const float4*>(old + j);
          raw[j] = __float_as_uint(__uint_as_float(raw[j]) + v.x);
          raw[j + 1] = __float_as_uint(__uint_as_float(raw[j + 1]) + v.y);
          raw[j + 2] = __float_as_uint(__uint_as_float(raw[j + 2]) + v.z);
          raw[j + 3] = __float_as_uint(__uint_as_float(raw[j + 3]) + v.w);
        }
      }
      if (to16) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          words[16 * h + j] = pack2<T>(alpha * __uint_as_float(raw[2 * j]), alpha * __uint_as_float(raw[2 * j + 1]));
      } else if (rows > 0 && at < cols) {
        store_lines<128>(staging, raw, reinterpret_cast<uint8_t*>(p.accumulator + n0 + at), p.ld_accumulator * 4, nullptr, m_warp, rows, 128, 4, true, lane);
      }
    }
    if (to16 && rows > 0 && c < cols) store_values<128>(staging, words, p, m_warp, n0 + c, rows, cols - c, wide, lane);
  }
}

// What a pair does one after another: whole tiles, and where the last round has fewer tiles than there are pairs, parts of tiles' K, so
// that no pair is idle while others take a whole tile.  (A head's gradient of 4096 x 4096 hidden states is 256 tiles, 3.46 rounds of 74 pairs.)
struct Units {
  int tiles, whole, split, k_blocks;
  __device__ __forceinline__ Units(int tiles_, int k_blocks_, int pairs, bool may_split) : tiles(tiles_), whole(tiles_), split(1), k_blocks(k_blocks_) {
    const int rest = tiles % pairs;
    if (may_split && rest) {
      split = max(1, min(min(pairs, kSplitUnits) / rest, min(kMostSplit, k_blocks / kLeastBlocks)));
      if (split > 1) whole = tiles - rest;
    }
  }
  __device__ __forceinline__ int count() const { return whole + (tiles - whole) * split; }
  // tile, and first and last k-block, of a unit; its number among the parts of the split tiles, or -1
  __device__ __forceinline__ void place(int unit, int& tile, int& begin, int& end, int& part) const {
    tile = unit;
    begin = 0;
    end = k_blocks;
    part = -1;
    if (unit >= whole) {
      part = unit - whole;
      tile = whole + part / split;
      const int64_t which = part % split;
      begin = static_cast<int>(which * k_blocks / split);
      end = static_cast<int>((which + 1) * k_blocks / split);
    }
  }
  static constexpr int kLeastBlocks = 8;      // of a part: its sums go through memory once more
  static constexpr int kMostSplit = 16;
};

// K-blocks that the accumulator takes before it is drained (after `most` at the latest), `left` of them remaining.
template <bool LOGITS>
__device__ __forceinline__ int drain_blocks(int left, int most) {
  if (!LOGITS || left <= most) return left;
  const int drains = (left + most - 1) / most;      // of about the same size
  return (left + drains - 1) / drains;
}

// A producer's way through its units, k-block by k-block.
struct Cursor {
  const Units& units;
  const Tiles& tiles;
  int cta, unit, step, kb, end, m0, n0;
  __device__ __forceinline__ Cursor(const Units& units_, const Tiles& tiles_, int cta_, int first, int step_)
      : units(units_), tiles(tiles_), cta(cta_), unit(first - step_), step(step_), kb(0), end(0) { settle(); }
  __device__ __forceinline__ bool done() const { return unit >= units.count(); }
  __device__ __forceinline__ void settle() {
    while (kb >= end) {
      unit += step;
      if (done()) return;
      int tile, part;
      units.place(unit, tile, kb, end, part);
      tiles.place(tile, m0, n0);
      m0 += cta * kRows;
      n0 += cta * kRows;
    }
  }
  __device__ __forceinline__ void advance() {
    ++kb;
    settle();
  }
};

template <int EPI, bool A_K, bool B_K, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Epi<EPI != kStore16>::kThreads, 1)
gemm16_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_all,
              int all_tokens, const __grid_constant__ Gemm16Problem prob, int* status) {
  constexpr bool kLogits = EPI != kStore16;
  using E = Epi<kLogits>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + kStages * kStageBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(staging + kStagingBytes);      // used in the leader CTA only
  uint64_t* empty_bar = full_bar + kStages;         // each CTA its own: "my stage may be refilled"
  uint64_t* acc_full = empty_bar + kStages;         // [2] each CTA its own: tensor core -> epilogue
  uint64_t* acc_empty = acc_full + 2;               // [2] leader's only: epilogue warps of both CTAs -> tensor core
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int cta = static_cast<int>(cluster_cta_rank());
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * E::kWarps);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_descriptor(&map_a);
    tma_prefetch_descriptor(&map_b);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 2 * kTile);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();      // both CTAs' barriers exist before anything arrives on them remotely
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  wait_for_predecessor();
  let_successor_start();

  int M = prob.M, K = prob.K;
  int drain = prob.drain / kBK;                // in k-blocks
  const CUtensorMap *source_a = &map_a, *source_b = &map_b;
  if (prob.count) {
    const int count = *prob.count;
    int& tokens = A_K ? M : K;
    tokens = max(0, min(tokens, count - prob.first));
    if (count <= prob.few) drain = prob.drain_few / kBK;
    if (count == all_tokens) (kLogits ? source_a : source_b) = &map_all;
  }
  const Tiles tiles(M, prob.N);
  // (with two terms every block of K comes twice, the second time with A's remainder; B's tile is in L2 then)
  const int term_shift = !kLogits && prob.second ? 1 : 0;
  const int k_blocks = (K + kBK - 1) / kBK << term_shift;
  const Units units(tiles.count(), k_blocks, clusters, !kLogits && prob.split_parts);

  if (warp < kFirstEpiWarp) {
    give_registers_back<E::kFew>();
    if (warp == 0 && lane == 0) {
      // ---------------- TMA producer (each CTA its own rows; the bytes are credited to the leader) ----------------
      int s = 0;
      uint32_t parity = 1;
      bool first_round = true;
      Cursor at(units, tiles, cta, cluster, clusters);
      for (; !at.done(); at.advance()) {
        if (!first_round && !mbar_wait_bounded(&empty_bar[s], parity, abort_flag, status, kStatusSlotWaitTimeout)) break;
        uint8_t* stage = smem + s * kStageBytes;
        if (cta == 0) mbar_expect_tx(&full_bar[s], 2 * kStageBytes);
        const uint32_t bar = map_to_cta(smem_u32(&full_bar[s]), 0);
        const int k = (at.kb >> term_shift) * kBK;
        const int along = at.kb & term_shift ? static_cast<int>(prob.second) : 0;      // in A's rows
        if constexpr (A_K) {
          tma_load_2d_pair(stage, source_a, bar, k + along, at.m0);
        } else {
          tma_load_2d_pair(stage, source_a, bar, at.m0 + along, k);
          tma_load_2d_pair(stage + kOperandBytes / 2, source_a, bar, at.m0 + 64 + along, k);
        }
        if constexpr (B_K) {
          tma_load_2d_pair(stage + kOperandBytes, source_b, bar, k, at.n0);
        } else {
          tma_load_2d_pair(stage + kOperandBytes, source_b, bar, at.n0, k);
          tma_load_2d_pair(stage + kOperandBytes + kOperandBytes / 2, source_b, bar, at.n0 + 64, k);
        }
        if (++s == kStages) {
          s = 0;
          parity ^= 1;
          first_round = false;
        }
      }
      if (*abort_flag) {
        // give copies that are still in flight time to land before the CTA's shared memory is released
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
      }
    } else if (warp == 1 && lane == 0 && cta == 0) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t kIdesc = (std::is_same<T, __nv_bfloat16>::value ? umma_idesc_bf16(kTile, kTile) : umma_idesc_fp16(kTile, kTile)) |
                                  (A_K ? 0u : kUmmaMnMajorA) | (B_K ? 0u : kUmmaMnMajorB);
      constexpr uint64_t kStepA = A_K ? 32 >> 4 : 2048 >> 4, kStepB = B_K ? 32 >> 4 : 2048 >> 4;      // 16 of K
      int s = 0;
      uint32_t parity = 0;
      bool ok = true;
      int it = 0;                                // drains so far
      // Whether the next k-block's operands and the next accumulator are there is looked up while this k-block's products are still being
      // issued: a wait, however short, drains the tensor core's queue of a few products.
      bool loaded = false, drained = false;
      for (int u = cluster; u < units.count() && ok; u += clusters) {
        int tile, begin, end, part;
        units.place(u, tile, begin, end, part);
        for (int kb = begin; kb < end && ok; ++it) {
          const int buf = it & 1;
          if (it >= 2 && !drained && !mbar_wait_bounded(&acc_empty[buf], ((it >> 1) - 1) & 1, abort_flag, status, kStatusAccumWaitTimeout)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t acc = tmem_base + static_cast<uint32_t>(buf * kTile);
          const int blocks = drain_blocks<kLogits>(end - kb, drain);
          for (int i = 0; i < blocks; ++i, ++kb) {
            if (!loaded && !mbar_wait_bounded(&full_bar[s], parity, abort_flag, status, kStatusTmaWaitTimeout)) {
              ok = false;
              break;
            }
            tc_fence_after_sync();
            const uint32_t stage = smem_u32(smem + s * kStageBytes);
            const uint64_t a = A_K ? umma_desc_kmajor<128>(stage) : umma_desc_mn_major(stage);
            const uint64_t b = B_K ? umma_desc_kmajor<128>(stage + kOperandBytes) : umma_desc_mn_major(stage + kOperandBytes);
  #pragma unroll
            for (int k = 0; k < kBK / 16; ++k) {
              umma_f16_ss_pair(acc, a + k * kStepA, b + k * kStepB, kIdesc, i | k ? 1u : 0u);
              if (k == 1) {
                const int next = s + 1 == kStages ? 0 : s + 1;
                loaded = mbar_test(&full_bar[next], next ? parity : parity ^ 1);
                drained = it >= 1 && mbar_test(&acc_empty[buf ^ 1], (((it + 1) >> 1) - 1) & 1);
              }
            }
            umma_commit_pair(&empty_bar[s]);
            if (++s == kStages) {
              s = 0;
              parity ^= 1;
            }
          }
          if (ok) umma_commit_pair(&acc_full[buf]);
        }
      }
    }
  } else {
    take_registers<E::kMany>();
    // ---------------- epilogue (each CTA its own 128 rows) ----------------
    const int ew = warp - kFirstEpiWarp;
    const int quarter = warp & 3;              // TMEM lane quarter this warp may read
    const int col0 = (ew >> 2) * E::kColumns;
    uint8_t* mine = staging + ew * E::kStaging;
    const uint32_t drained = map_to_cta(smem_u32(&acc_empty[0]), 0);
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(col0);
    int it = 0;
    auto filled = [&]() {
      if (!mbar_wait_parked(&acc_full[it & 1], (it >> 1) & 1, abort_flag, status, kStatusAccumWaitTimeout)) return false;
      tc_fence_after_sync();
      return true;
    };
    auto release = [&]() {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(drained + static_cast<uint32_t>((it & 1) * sizeof(uint64_t)));
      ++it;
    };
    for (int u = cluster; u < units.count(); u += clusters) {
      int m0, n0, tile, begin, end, part;
      units.place(u, tile, begin, end, part);
      tiles.place(tile, m0, n0);
      const int m_warp = m0 + cta * kRows + quarter * 32;
      if constexpr (kLogits) {
        uint64_t sums[kLogitPart / 2];         // pairs of neighbouring columns
#pragma unroll
        for (int j = 0; j < kLogitPart / 2; ++j) sums[j] = 0;
        bool ok = true;
        for (int kb = 0; kb < k_blocks;) {
          kb += drain_blocks<true>(k_blocks - kb, drain);
          ok = filled();
          if (!ok) break;
          const uint32_t from = taddr + static_cast<uint32_t>((it & 1) * kTile);
#pragma unroll
          for (int c = 0; c < kLogitPart; c += 16) {
            uint32_t raw[16];
            tmem_ld_32x16(from + c, raw);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 8; ++j) add_pair(sums[c / 2 + j], pack_pair(raw[2 * j], raw[2 * j + 1]));
          }
          release();
        }
        if (!ok) break;
        logits_epilogue<EPI, T>(prob, sums, M, m_warp, n0 + col0, mine, lane);
      } else {
        const bool empty = k_blocks == 0;      // (nothing was added up)
        if (!empty && !filled()) break;
        const uint32_t from = taddr + static_cast<uint32_t>((it & 1) * kTile);
        auto accumulated = [&](int at, uint32_t (&raw)[32]) {
          tmem_ld_32x32(from + at, raw);
          tmem_ld_wait();
          if (empty) {
#pragma unroll
            for (int j = 0; j < 32; ++j) raw[j] = 0;
          }
        };
        if (part < 0) {
          product_epilogue<T>(prob, M, m_warp, n0 + col0, mine, lane, accumulated);
          if (!empty) release();
        } else {
          // This part's sums, 256 x 256 of them a part, as the registers hold them: a line of 32 lanes for each column of a warp's region.  The
          // warp that is the last to leave its region of the tile adds the parts up in order.
          constexpr int64_t kRegion = 32 * E::kColumns;
          const int64_t region = static_cast<int64_t>(cta * E::kWarps + ew) * kRegion + lane;
          const int first = (tile - units.whole) * units.split;
          float* mine_of = prob.split_parts + part * int64_t{kTile * kTile} + region;
#pragma unroll
          for (int at = 0; at < E::kColumns; at += 32) {
            uint32_t raw[32];
            accumulated(at, raw);
#pragma unroll
            for (int j = 0; j < 32; ++j) mine_of[(at + j) * 32] = __uint_as_float(raw[j]);
          }
          release();
          __threadfence();
          __syncwarp();
          int* counter = prob.split_counters + ((tile - units.whole) * 2 + cta) * E::kWarps + ew;
          int before = 0;
          if (lane == 0) before = atomicAdd(counter, 1);
          before = __shfl_sync(0xffffffffu, before, 0);
          if (before == units.split - 1) {
            if (lane == 0) *counter = 0;
            __threadfence();
            product_epilogue<T>(prob, M, m_warp, n0 + col0, mine, lane, [&](int at, uint32_t (&raw)[32]) {
#pragma unroll
              for (int j = 0; j < 32; ++j) raw[j] = 0;
              const float* from_part = prob.split_parts + first * int64_t{kTile * kTile} + region + at * 32;
              for (int i = 0; i < units.split; ++i, from_part += kTile * kTile) {
#pragma unroll
                for (int j = 0; j < 32; ++j) raw[j] = __float_as_uint(__uint_as_float(raw[j]) + __ldcg(from_part + j * 32));
              }
            });
          }
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();      // nobody leaves while the other CTA may still touch its shared memory or TMEM
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 2 * kTile);
  }
}

CUtensorMap map_of(bool bf16, const Matrix16& x, int64_t rows, int64_t K) {
  const CUtensorMapDataType type = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return x.k_major ? encode_k_major(type, x.data, K, rows, 2 * x.ld, kBK, kRows, CU_TENSOR_MAP_SWIZZLE_128B)
                   : encode_k_major(type, x.data, rows, K, 2 * x.ld, 64, kBK, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int EPI, bool A_K, bool B_K, typename T>
void launch(const Matrix16& a, const Matrix16& b, const Gemm16Problem& p, int* status, cudaStream_t stream, const Hidden16* hidden) {
  static PerDeviceOnce configured;
  allow_dynamic_smem(reinterpret_cast<const void*>(gemm16_kernel<EPI, A_K, B_K, T>), kSmemBytes, configured, "gemm16");
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  const int64_t more = EPI == kStore16 ? p.second : 0;
  const CUtensorMap map_a = a.k_major ? map_of(kBf16, a, p.M, p.K + more) : map_of(kBf16, a, p.M + more, p.K), map_b = map_of(kBf16, b, p.N, p.K);
  const CUtensorMap map_all = !hidden ? map_a : EPI != kStore16 ? map_of(kBf16, hidden->all, p.M, p.K) : map_of(kBf16, hidden->all, p.N, p.K);
  const int64_t tiles = static_cast<int64_t>((p.M + kTile - 1) / kTile) * ((p.N + kTile - 1) / kTile);
  if (tiles > (1 << 30)) throw std::invalid_argument("gemm16: too many tiles");
  // (where tokens are left out there may be fewer tiles in the end than here, and more parts of one)
  const int64_t parts = p.split_parts ? std::max(1, std::min(Units::kMostSplit, (p.K + kBK - 1) / kBK / Units::kLeastBlocks)) : 1;
  const int clusters = static_cast<int>(std::min<int64_t>(tiles * parts, multiprocessors() / 2));
  cudaError_t err = launch_dependent(gemm16_kernel<EPI, A_K, B_K, T>, dim3(2 * clusters), dim3(Epi<EPI != kStore16>::kThreads), kSmemBytes, stream, map_a,
                                     map_b, map_all, hidden ? hidden->tokens : -1, p, status);
  if (err != cudaSuccess) throw std::runtime_error(std::string("gemm16 launch: ") + cudaGetErrorString(err));
}

template <typename T>
void dispatch(Gemm16Epilogue epilogue, const Matrix16& a, const Matrix16& b, const Gemm16Problem& p, int* status, cudaStream_t stream,
              const Hidden16* hidden) {
  const bool logits = a.k_major && b.k_major;
  if (epilogue == kLogitStatistics && logits) launch<kLogitStatistics, true, true, T>(a, b, p, status, stream, hidden);
  else if (epilogue == kLogitGradient && logits) launch<kLogitGradient, true, true, T>(a, b, p, status, stream, hidden);
  else if (epilogue == kStore16 && a.k_major && !b.k_major && !hidden) launch<kStore16, true, false, T>(a, b, p, status, stream, hidden);
  else if (epilogue == kStore16 && !a.k_major && !b.k_major) launch<kStore16, false, false, T>(a, b, p, status, stream, hidden);
  else throw std::invalid_argument("gemm16: no kernel for these orders of the operands");
}

}  // namespace

void gemm16(Gemm16Epilogue epilogue, bool bf16, const Matrix16& a, const Matrix16& b, const Gemm16Problem& p, int* status,
            cudaStream_t stream, const Hidden16* hidden) {
  if (p.M <= 0 || p.N <= 0 || p.K <= 0) throw std::invalid_argument("gemm16: empty product");
  if (a.ld % 8 != 0 || b.ld % 8 != 0 || (hidden && hidden->all.ld % 8 != 0))
    throw std::invalid_argument("gemm16: operand pitches are multiples of 8 elements");
  if ((epilogue == kLogitGradient || epilogue == kLogitExponential) && (p.ldc % 8 != 0 || (reinterpret_cast<uintptr_t>(p.C) & 15) != 0))
    throw std::invalid_argument("gemm16: the logits' gradient needs 16-byte rows");
  auto drains = [](int every) { return every >= kBK && every % kBK == 0; };
  if (epilogue != kStore16 && (!drains(p.drain) || (p.few > 0 && !drains(p.drain_few))))
    throw std::invalid_argument("gemm16: logits are drained every multiple of 64 of K");
  if (p.second % kBK != 0 || p.second < 0 || (p.second && p.second < (epilogue == kLogitGradient ? p.N : a.k_major ? p.K : p.M)))
    throw std::invalid_argument("gemm16: the second term lies a multiple of 64 columns behind the first");
  if (epilogue == kStore16 && (p.add || !p.C) && (!p.accumulator || p.ld_accumulator % 32 != 0 || p.ld_accumulator < p.N ||
                                                  (reinterpret_cast<uintptr_t>(p.accumulator) & 15) != 0))
    throw std::invalid_argument("gemm16: the accumulator's pitch is a multiple of 32 covering the columns");
  if ((p.split_parts == nullptr) != (p.split_counters == nullptr) || (reinterpret_cast<uintptr_t>(p.split_parts) & 15) != 0)
    throw std::invalid_argument("gemm16: split tiles need aligned room for their parts and counters");
  if (epilogue == kLogitExponential) {
    if (!bf16 || !a.k_major || !b.k_major) throw std::invalid_argument("gemm16: exponentials are kept in bf16, of K-major operands");
    launch<kLogitExponential, true, true, __nv_bfloat16>(a, b, p, status, stream, hidden);
  } else if (bf16) {
    dispatch<__nv_bfloat16>(epilogue, a, b, p, status, stream, hidden);
  } else {
    dispatch<__half>(epilogue, a, b, p, status, stream, hidden);
  }
}

}  // namespace soapb200
