// Attention of sequences that share their first keys, over a paged cache in 8 bits, for sm_100a: the shared keys are read once for all of them.
//
//   A run of `each` sequences has its first S keys in common (S whole tiles of 128 keys). For the rows of all its queries, R = each * queries * heads of
//   a key head, and a part of the S keys, this kernel leaves
//     m = a reference point near max_j s_j      s_j = scale * q . k_j, in units of log2
//     l = sum_j 2^(s_j - m)                     o = sum_j 2^(s_j - m) v_j      (f32, not divided)
//   keyed.cu then takes each sequence's own keys and joins: any number of (m, l, o) of one row add up after 2^(m - max m).
//
// The products are the tensor cores' (tcgen05, f16 operands, f32 sums in tensor memory): a CTA owns one or two tiles of 128 rows and walks its part of
// the keys 128 at a time.
//
//   warps of a tile (4)   a row a thread: tcgen05.ld of its 128 scores, the keys' scales, ex2, sum; probabilities times the values' scales go
//                         back into tensor memory as f16 pairs, the A operand of the second product
//   converters (4 warps)  e4m3 codes, as TMA brought them from the pages, to f16 (exact) in the layout of the products' operands
//   producer (1 warp)     looks pages up, loads their codes (TMA) and scales
//   issuer (1 thread)     S = Q K^T and O += P V
//
// Precision: as in keyed.cu. A row of queries is brought to f16 by a power of two (only elements 2^-38 of its largest, or less, lose digits); codes are
// exact in f16; probabilities are rounded to f16 (2^-11 of each). A page's scale of the values multiplies the probabilities before that, relative to the
// largest scale of the part, so pages whose scales are 2^-kSpan of the largest or less would lose digits: they get a walk of their own with another
// reference, one for each kSpan powers of two. (Rare: a cache's scales follow its values' magnitudes.)
//
// No row is masked: a sequence with a query that does not see all the shared keys takes no part (its rows are computed and not used) and reads its keys
// itself. A page that is not there is left out, with zeros for its codes and -inf for its scores.
//
// Every wait is bounded; one that gives up sets the device status word, and the CTA leaves through the normal teardown. No load uses multicast.
#include <cuda.h>

#include <cmath>

#include "common.h"
#include "keyed.h"
#include "tcgen05.h"

namespace tq {
namespace {

constexpr int kKeys = kPrefixTile;          // a step
constexpr int kTileRows = 128;              // rows of an instruction's tile
constexpr float kSlack = 8.f;               // a row's reference point moves when a tile's maximum is more than 2^kSlack above it
constexpr int kSpan = 12;                   // powers of two of the values' scales that a walk takes
constexpr int kInfos = 8;                   // tiles whose scales are on chip
constexpr int kMostPages = kKeys / 16;      // of a tile

enum PrefixWait { kWaitReady = 0x50465831, kWaitRawEmpty, kWaitRawFull, kWaitKeysEmpty, kWaitValuesEmpty, kWaitKeysFull, kWaitValuesFull, kWaitScores,
                  kWaitProbabilities, kWaitProduct, kWaitTaken };

// D: heads of up to 64 or 128 elements. TILES: of 128 rows.
template <int D, int TILES>
struct PrefixLayout {
  static constexpr int kSub = D / 64;                                         // tiles of 64 elements (128 bytes in f16) side by side
  static constexpr uint32_t kSubBytes = 128 * 128;                            // 128 rows, keys or values of one
  static constexpr uint32_t kRawBytes = kKeys * D;
  static constexpr int kRawStages = D == 64 ? 8 : TILES == 1 ? 4 : 2;         // of keys or of values
  static constexpr uint32_t kOperandBytes = kSub * kSubBytes;
  static constexpr uint32_t kOffsetKeys = TILES * kOperandBytes;              // queries from 0 on
  static constexpr uint32_t kOffsetValues = kOffsetKeys + 2 * kOperandBytes;
  static constexpr uint32_t kOffsetRaw = kOffsetValues + 2 * kOperandBytes;
  static constexpr uint32_t kOffsetBarriers = kOffsetRaw + kRawStages * kRawBytes;
  static constexpr size_t kSmemBytes = 1024 + kOffsetBarriers + 512;
  static_assert(kSmemBytes <= 227 * 1024, "more than a CTA's shared memory");
  // Tensor memory: scores of each tile, results of each tile, and probabilities of each tile, which for two tiles of wide heads lie over the scores.
  static constexpr bool kOver = TILES == 2 && D == 128;
  static constexpr uint32_t kColumnO = TILES * kKeys, kColumnP = kOver ? 0 : kColumnO + TILES * D;
  static constexpr uint32_t kStrideP = kOver ? kKeys : kKeys / 2;
  static constexpr uint32_t kTmemColumns = kColumnO + TILES * D + (kOver ? 0 : TILES * kKeys / 2) <= 256 ? 256 : 512;
  static_assert(kColumnO + TILES * D + (kOver ? 0 : TILES * kKeys / 2) <= 512, "more than tensor memory");
  static constexpr int kThreads = TILES * 128 + 256;                          // tiles' warps, converters, producer and issuer (and two idle warps)
  // setmaxnreg: the last two groups of four warps give up what the tiles' warps take. An increase beyond that would wait for ever.
  static constexpr int kLaunchRegisters = 65536 / kThreads / 8 * 8;
  static constexpr int kTileRegisters = TILES == 1 ? 224 : 192, kConvertRegisters = TILES == 1 ? 120 : 80, kOtherRegisters = TILES == 1 ? 56 : 40;
  static_assert(TILES * kTileRegisters + kConvertRegisters + kOtherRegisters <= (TILES + 2) * kLaunchRegisters, "registers nobody releases");
};

// f32 accumulator, f16 operands, M = 128, N = n; B MN-major when `b_mn`.
__host__ __device__ constexpr uint32_t prefix_instruction(int n, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTileRows >> 4) << 24);
}

__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap* map, uint32_t bar, int column, int row) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(column), "r"(row)
      : "memory");
}
__device__ __forceinline__ void store_shared_16(uint32_t address, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint32_t half_pair(float low, float high) {
  const __half2 pair = __floats2half2_rn(low, high);
  return *reinterpret_cast<const uint32_t*>(&pair);
}
// Four e4m3 codes as two pairs of f16.
__device__ __forceinline__ uint2 decode_four(uint32_t codes) {
  uint2 pairs;
  asm("{\n\t.reg .b16 low, high;\n\tmov.b32 {low, high}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, low;\n\tcvt.rn.f16x2.e4m3x2 %1, high;\n\t}"
      : "=r"(pairs.x), "=r"(pairs.y)
      : "r"(codes));
  return pairs;
}
// A power of two near a magnitude (its own exponent, from 2^-126 on): bits of an f32.
__device__ __forceinline__ int exponent_of(float magnitude) { return max(static_cast<int>(__float_as_uint(magnitude) >> 23 & 0xff), 1) - 127; }
__device__ __forceinline__ float power_of_two(int exponent) { return __uint_as_float(static_cast<uint32_t>(exponent + 127) << 23); }      // -126 to 127

template <int D, int TILES>
__global__ void __launch_bounds__(PrefixLayout<D, TILES>::kThreads, 1)
prefix_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ KeyedParams p,
                        const bool bf16) {
  using L = PrefixLayout<D, TILES>;
  constexpr int kRaw = L::kRawStages, kSub = L::kSub;
  constexpr int kTileThreads = TILES * 128;
  extern __shared__ unsigned char raw_smem[];
  // Of a tile of keys: the page of each of its pieces is there (bits), its scale of the keys, and of the values.
  __shared__ float key_scale[kInfos][kMostPages], value_scale[kInfos][kMostPages];
  __shared__ uint32_t pages_there[kInfos];
  __shared__ int first_taker, highest, lowest;                    // the sequence whose table is read; exponents of the values' scales
  const uint32_t base = (smem_address(raw_smem) + 1023u) & ~1023u;
  const uint32_t barriers = base + L::kOffsetBarriers;
  const uint32_t ready = barriers;                                // queries, highest and lowest are there
  auto raw_full = [&](int s) { return barriers + 8u * (1 + s); };
  auto raw_empty = [&](int s) { return barriers + 8u * (1 + kRaw + s); };
  const uint32_t after_raw = barriers + 8u * (1 + 2 * kRaw);
  auto keys_full = [&](int b) { return after_raw + 8u * b; };
  auto keys_empty = [&](int b) { return after_raw + 8u * (2 + b); };
  auto values_full = [&](int b) { return after_raw + 8u * (4 + b); };
  auto values_empty = [&](int b) { return after_raw + 8u * (6 + b); };
  auto scores_full = [&](int t) { return after_raw + 8u * (8 + t); };
  auto scores_taken = [&](int t) { return after_raw + 8u * (10 + t); };      // in registers (where probabilities lie apart)
  auto probabilities = [&](int t) { return after_raw + 8u * (12 + t); };
  auto product_done = [&](int t) { return after_raw + 8u * (14 + t); };
  const uint32_t tmem_slot = after_raw + 8u * 16;
  static_assert(8 * (1 + 2 * kRaw + 16) + 4 <= 512, "barriers beyond their room");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kConvertWarp = 4 * TILES, kProducerWarp = kConvertWarp + 4, kIssuerWarp = kProducerWarp + 1;
  if (threadIdx.x == 0) {
    barrier_init(ready, 4 * TILES);
    for (int s = 0; s < kRaw; ++s) {
      barrier_init(raw_full(s), 1);
      barrier_init(raw_empty(s), 4);
    }
    for (int b = 0; b < 2; ++b) {
      barrier_init(keys_full(b), 4);
      barrier_init(keys_empty(b), 1);
      barrier_init(values_full(b), 4);
      barrier_init(values_empty(b), 1);
      barrier_init(scores_full(b), 1);
      barrier_init(scores_taken(b), 4);
      barrier_init(probabilities(b), 4);
      barrier_init(product_done(b), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    first_taker = 0x7fffffff;
    highest = -1000;
    lowest = 1000;
  }
  if (warp == kProducerWarp && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
  }
  wait_for_earlier();
  if (blockIdx.x == 0 && threadIdx.x == 0) p.status.begin();

  // Which part of which block of which key head of which run.
  const int part = static_cast<int>(blockIdx.x) % p.splits, unit = static_cast<int>(blockIdx.x) / p.splits;
  const int block = unit % p.row_blocks, head_index = unit / p.row_blocks;
  const int kv_head = head_index % p.kv_heads, run = head_index / p.kv_heads;
  const int tiles_all = shared_keys(p, run) / kKeys;
  const int tile0 = static_cast<int>(static_cast<long long>(tiles_all) * part / p.splits);
  const int tiles = static_cast<int>(static_cast<long long>(tiles_all) * (part + 1) / p.splits) - tile0;
  const int rows_each = p.group * p.q_tokens, rows = p.each * rows_each, row0 = block * p.prefix_rows;
  const long long slot0 = static_cast<long long>(blockIdx.x) * p.prefix_rows;
  __syncthreads();
  if (tiles > 0) {
    for (int i = threadIdx.x; i < p.each; i += L::kThreads) {
      const int length = min(max(p.lengths[run * p.each + i], 0), p.blocks << p.page_shift);
      if (takes_part(p, tiles_all * kKeys, length)) atomicMin(&first_taker, run * p.each + i);
    }
  }
  if (warp == kIssuerWarp && tiles > 0) tmem_alloc(tmem_slot, L::kTmemColumns);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const int taker = first_taker;
  if (tiles == 0 || taker == 0x7fffffff) {                        // nothing here, or nobody to want it: the same in the whole CTA
    for (int i = threadIdx.x; i < p.prefix_rows; i += L::kThreads) p.prefix_stats[slot0 + i] = make_float2(-INFINITY, 0.f);
    if (warp == kIssuerWarp && tiles > 0) {
      uint32_t tmem;
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
      tmem_dealloc(tmem, L::kTmemColumns);
    }
    let_later_start();
    return;
  }
  uint32_t tmem_base;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));

  const int32_t* const table = p.table + taker * p.table_stride;
  const int piece_shift = min(p.page_shift, 7), pieces = kKeys >> piece_shift;      // of a tile: what lies in one page
  // Walks over the keys, one for each kSpan powers of two of the values' scales: known once `ready` completes.
  auto walks = [&] { return highest < lowest ? 1 : (highest - lowest) / kSpan + 1; };

  if (warp >= kConvertWarp && warp < kProducerWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kConvertRegisters));
    // ---- converters: items in the order K(0), K(1), V(0), K(2), V(1), ... V(last) of all walks together ----
    if (__all_sync(0xffffffffu, barrier_wait(ready, 0, p.status, kWaitReady))) {
      const int steps = tiles * walks();
      const int thread = threadIdx.x - kConvertWarp * 32;
      constexpr int kPiecesKey = D / 16, kEach = kKeys * kPiecesKey / 128;      // 16 codes; of a key, of a thread
      for (int n = 0; n < 2 * steps; ++n) {
        const bool values = n != 0 && (n == 2 * steps - 1 || n % 2 == 0);
        const int step = n == 0 ? 0 : values ? (n == 2 * steps - 1 ? steps - 1 : n / 2 - 1) : (n + 1) / 2;
        const int stage = n % kRaw, buffer = step & 1;
        if (!__all_sync(0xffffffffu, barrier_wait(raw_full(stage), (n / kRaw) & 1, p.status, kWaitRawFull))) break;
        if (!__all_sync(0xffffffffu, barrier_wait(values ? values_empty(buffer) : keys_empty(buffer), ((step >> 1) & 1) ^ 1, p.status,
                                                  values ? kWaitValuesEmpty : kWaitKeysEmpty)))
          break;
        const uint32_t from = base + L::kOffsetRaw + stage * L::kRawBytes;
        const uint32_t to = base + (values ? L::kOffsetValues : L::kOffsetKeys) + buffer * L::kOperandBytes;
        const uint32_t there = pages_there[step % kInfos];
        const bool whole = there == (1u << pieces) - 1;
        constexpr int kAtOnce = 4;
#pragma unroll
        for (int k = 0; k < kEach; k += kAtOnce) {
          uint4 codes[kAtOnce];
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) {
            const int i = thread + (k + u) * 128;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(codes[u].x), "=r"(codes[u].y), "=r"(codes[u].z), "=r"(codes[u].w)
                         : "r"(from + i * 16));
          }
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) {
            const int i = thread + (k + u) * 128, key = i / kPiecesKey, piece = i % kPiecesKey;
            if (!whole && !(there >> (key >> piece_shift) & 1)) codes[u] = make_uint4(0, 0, 0, 0);
            const uint2 a = decode_four(codes[u].x), b = decode_four(codes[u].y), c = decode_four(codes[u].z), d = decode_four(codes[u].w);
            // units of 16 bytes, exchanged within 128 by the key's place in 8; pieces of the second 64 elements write their odd unit first, so that
            // eight neighbouring threads write to eight different ones
            const uint32_t line = to + (piece / 4) * L::kSubBytes + key * 128;
            const int even = piece % 4 * 2, turn = key & 7;
            const bool odd_first = piece >= 4;
            store_shared_16(line + (((even + (odd_first ? 1 : 0)) ^ turn) << 4), odd_first ? c.x : a.x, odd_first ? c.y : a.y, odd_first ? d.x : b.x,
                            odd_first ? d.y : b.y);
            store_shared_16(line + (((even + (odd_first ? 0 : 1)) ^ turn) << 4), odd_first ? a.x : c.x, odd_first ? a.y : c.y, odd_first ? b.x : d.x,
                            odd_first ? b.y : d.y);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          barrier_arrive(values ? values_full(buffer) : keys_full(buffer));
          barrier_arrive(raw_empty(stage));
        }
      }
    }
  } else if (warp >= kProducerWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kOtherRegisters));
    if (warp == kProducerWarp) {
      // ---- producer: the whole warp, a lane for each piece of a tile ----
      bool known = false;
      int steps = tiles, issued = 0;
      for (int n = 0; n < 2 * steps; ++n) {
        // (the first items leave before the number of walks is known, which says what follows the last keys of the first)
        if (!known && n == min(kRaw, 2 * tiles - 1)) {
          if (!__all_sync(0xffffffffu, barrier_wait(ready, 0, p.status, kWaitReady))) break;
          known = true;
          steps = tiles * walks();
        }
        const bool values = n != 0 && (n == 2 * steps - 1 || n % 2 == 0);
        const int step = n == 0 ? 0 : values ? (n == 2 * steps - 1 ? steps - 1 : n / 2 - 1) : (n + 1) / 2;
        const int stage = n % kRaw;
        if (!__all_sync(0xffffffffu, barrier_wait(raw_empty(stage), ((n / kRaw) & 1) ^ 1, p.status, kWaitRawEmpty))) break;
        const int key0 = (tile0 + step % tiles) * kKeys + (lane << piece_shift);
        int page = -1;
        if (lane < pieces) {
          const int at_block = key0 >> p.page_shift;
          page = table[at_block];
          if (page < 0 || page >= p.pages) {
            if (!values) report(p.status, kKeyedPage, taker, at_block);
            page = -1;
          }
        }
        const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
        const uint32_t piece_bytes = static_cast<uint32_t>(D) << piece_shift;
        if (!values) {
          // (last used by step - kInfos, whose scores were taken long ago: the operands' buffers are two deep)
          if (lane < pieces) {
            const long long at = static_cast<long long>(page) * p.kv_heads + kv_head;
            key_scale[step % kInfos][lane] = page >= 0 ? p.k_scales[at] : 0.f;
            value_scale[step % kInfos][lane] = page >= 0 ? p.v_scales[at] : 0.f;
          }
          if (lane == 0) pages_there[step % kInfos] = there;
        }
        __syncwarp();
        if (lane == 0) barrier_expect_tx(raw_full(stage), piece_bytes * __popc(there));
        __syncwarp();
        if (page >= 0) {
          const int row = ((page * p.kv_heads + kv_head) << p.page_shift) + (key0 & ((1 << p.page_shift) - 1));      // (below 2^31: prefix_maps)
          tma_load_rows(base + L::kOffsetRaw + stage * L::kRawBytes + lane * piece_bytes, values ? &map_v : &map_k, raw_full(stage), 0, row);
        }
        issued = n + 1;
      }
      // where a wait gave up: copies that are under way land before the CTA leaves
      for (int n = max(0, issued - kRaw); n < issued; ++n) {
        for (uint32_t spin = 0; spin < kSpinLimit && !barrier_try_wait(raw_full(n % kRaw), (n / kRaw) & 1); ++spin) {
        }
      }
    } else if (warp == kIssuerWarp) {
      if (elect_one()) {
        constexpr uint32_t kHigh = kDescriptorHigh;
        constexpr uint32_t scores_instruction = prefix_instruction(kKeys, false), values_instruction = prefix_instruction(D, true);
        const uint32_t low_q = descriptor_low(base, 0), low_k = descriptor_low(base + L::kOffsetKeys, 0);
        const uint32_t low_v = descriptor_low(base + L::kOffsetValues, L::kSubBytes);
        // both operands K-major: 16 elements are 32 bytes in the swizzled line
        auto scores = [&](int t, int step) {
          const uint32_t q = low_q + t * (L::kOperandBytes >> 4), k = low_k + (step & 1) * (L::kOperandBytes >> 4);
#pragma unroll
          for (int h = 0; h < kSub; ++h) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f16_split(tmem_base + t * kKeys, q + h * (L::kSubBytes >> 4) + kk * 2, kHigh, k + h * (L::kSubBytes >> 4) + kk * 2, kHigh, scores_instruction,
                            (h != 0 || kk != 0) ? 1u : 0u);
          }
          mma_commit(scores_full(t));
        };
        // P from tensor memory (16 keys are 8 columns), V MN-major (16 keys are 2048 bytes)
        auto product = [&](int t, int step) {
          const uint32_t v = low_v + (step & 1) * (L::kOperandBytes >> 4);
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            mma_f16_tmem_a(tmem_base + L::kColumnO + t * D, tmem_base + L::kColumnP + t * L::kStrideP + kk * 8, v + kk * (2048 >> 4), kHigh, values_instruction,
                           (step % tiles != 0 || kk != 0) ? 1u : 0u);
          mma_commit(product_done(t));
        };
        if (barrier_wait(ready, 0, p.status, kWaitReady) && barrier_wait(keys_full(0), 0, p.status, kWaitKeysFull)) {
          const int steps = tiles * walks();
          tcgen05_fence_after();
          for (int t = 0; t < TILES; ++t) scores(t, 0);
          mma_commit(keys_empty(0));
          bool alive = true;
          for (int j = 0; alive && j < steps; ++j) {
            const bool more = j + 1 < steps;
            if (more && !barrier_wait(keys_full((j + 1) & 1), ((j + 1) >> 1) & 1, p.status, kWaitKeysFull)) break;
            if constexpr (!L::kOver) {
              // the next scores, as soon as this step's are in registers
              if (more) {
                for (int t = 0; alive && t < TILES; ++t) {
                  alive = barrier_wait(scores_taken(t), j & 1, p.status, kWaitTaken);
                  if (!alive) break;
                  tcgen05_fence_after();
                  scores(t, j + 1);
                }
                if (!alive) break;
                mma_commit(keys_empty((j + 1) & 1));
              }
            }
            if (!barrier_wait(values_full(j & 1), (j >> 1) & 1, p.status, kWaitValuesFull)) break;
            for (int t = 0; alive && t < TILES; ++t) {
              alive = barrier_wait(probabilities(t), j & 1, p.status, kWaitProbabilities);
              if (!alive) break;
              tcgen05_fence_after();
              product(t, j);
              // (over the columns of the probabilities, which the product before has read by then: one thread's products run in order)
              if (L::kOver && more) scores(t, j + 1);
            }
            if (!alive) break;
            mma_commit(values_empty(j & 1));
            if (L::kOver && more) mma_commit(keys_empty((j + 1) & 1));
          }
        }
      }
    }
  } else {
    // ---- a row a thread ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kTileRegisters));
    const int tile = warp / 4, row_in_block = static_cast<int>(threadIdx.x), row = row0 + row_in_block;
    // The values' scales of the part: how far apart they are.
    {
      int high = -1000, low = 1000;
      const int block0 = (tile0 * kKeys) >> p.page_shift, block1 = ((tile0 + tiles) * kKeys - 1) >> p.page_shift;
      for (int n = block0 + static_cast<int>(threadIdx.x); n <= block1; n += kTileThreads) {
        const int page = table[n];
        if (page < 0 || page >= p.pages) continue;
        const float scale = fabsf(p.v_scales[static_cast<long long>(page) * p.kv_heads + kv_head]);
        if (scale > 0.f && scale < INFINITY) {
          const int exponent = exponent_of(scale);
          high = max(high, exponent);
          low = min(low, exponent);
        }
      }
      high = __reduce_max_sync(0xffffffffu, high);
      low = __reduce_min_sync(0xffffffffu, low);
      if (lane == 0) {
        atomicMax(&highest, high);
        atomicMin(&lowest, low);
      }
    }
    // The row of queries, as f16 times a power of two.
    float row_scale = p.scale_log2;
    {
      const bool there = row < rows;
      const int sequence = run * p.each + row / rows_each, inside = row % rows_each;
      const int token = inside / p.group, head = kv_head * p.group + inside % p.group;
      const char* const from = static_cast<const char*>(p.q) + 2 * (sequence * p.q_strides[0] + head * p.q_strides[1] + token * p.q_strides[2]);
      auto widen = [&](uint32_t pair) {
        if (bf16) return make_float2(__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u));
        return __half22float2(*reinterpret_cast<const __half2*>(&pair));
      };
      uint4 word[D / 8];
      float largest = 0.f;
#pragma unroll
      for (int u = 0; u < D / 8; ++u) {
        word[u] = make_uint4(0, 0, 0, 0);
        if (there && u * 8 < p.head_dim) word[u] = *reinterpret_cast<const uint4*>(from + u * 16);
      }
#pragma unroll
      for (int u = 0; u < D / 8; ++u) {
        const uint32_t pairs[4] = {word[u].x, word[u].y, word[u].z, word[u].w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float2 pair = widen(pairs[c]);
          largest = fmaxf(largest, fmaxf(fabsf(pair.x), fabsf(pair.y)));
        }
      }
      // to [2^14, 2^15), by 2^126 at most; none for infinities (as in keyed.cu)
      int exponent = max(static_cast<int>(__float_as_uint(largest) >> 23) - 127, -112);
      if (exponent > 127) exponent = 14;
      const float up = power_of_two(14 - exponent);
      row_scale *= power_of_two(exponent - 14);
      const uint32_t line = base + tile * L::kOperandBytes + (row_in_block % kTileRows) * 128;
#pragma unroll
      for (int u = 0; u < D / 8; ++u) {
        const float2 a = widen(word[u].x), b = widen(word[u].y), c = widen(word[u].z), d = widen(word[u].w);
        store_shared_16(line + (u / 8) * L::kSubBytes + (((u % 8) ^ (row_in_block & 7)) << 4), half_pair(a.x * up, a.y * up), half_pair(b.x * up, b.y * up),
                        half_pair(c.x * up, c.y * up), half_pair(d.x * up, d.y * up));
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) barrier_arrive(ready);
    bool alive = __all_sync(0xffffffffu, barrier_wait(ready, 0, p.status, kWaitReady));
    const int steps = alive ? tiles * walks() : 0, top_exponent = highest;

    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const uint32_t tmem_s = tmem_base + tile * kKeys + lanes, tmem_p = tmem_base + L::kColumnP + tile * L::kStrideP + lanes;
    const uint32_t tmem_o = tmem_base + L::kColumnO + tile * D + lanes;
    float reference = -INFINITY, row_sum = 0.f, sum_kept = 0.f;
    for (int j = 0; j < steps; ++j) {
      const int walk = j / tiles, in_walk = j % tiles;
      // of the walk: powers of two [2^(top - kSpan), 2^top], brought to 1 at most; what is no number, or zero, is everybody's
      const int top = max(top_exponent - walk * kSpan, -126);
      const float down = highest < lowest ? 1.f : power_of_two(min(max(-top - 1, -126), 126));
      auto weight_of = [&](float scale) {
        const float magnitude = fabsf(scale);
        const int exponent = exponent_of(magnitude);
        const bool mine = !(magnitude > 0.f && magnitude < INFINITY) || (exponent <= top && exponent > top - kSpan) || (walk + 1 == steps / tiles && exponent <= top);
        return mine ? scale * down : 0.f;
      };
      if (!__all_sync(0xffffffffu, barrier_wait(scores_full(tile), j & 1, p.status, kWaitScores))) { alive = false; break; }
      tcgen05_fence_after();
      uint32_t r[kKeys];
#pragma unroll
      for (int i = 0; i < kKeys; i += 32) tmem_load_32(tmem_s + i, *reinterpret_cast<uint32_t(*)[32]>(&r[i]));
      tmem_load_wait();
      if constexpr (!L::kOver) {
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) barrier_arrive(scores_taken(tile));
      }
      const int info = j % kInfos;
      const uint32_t there = pages_there[info];
      float most = -INFINITY;
#pragma unroll
      for (int s = 0; s < kMostPages; ++s) {
        const int piece = (s * 16) >> piece_shift;
        const float by = row_scale * key_scale[info][piece];
        const float2 by2 = make_float2(by, by);
        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
        for (int i = s * 16; i < s * 16 + 16; i += 2) {
          const float2 scaled = __fmul2_rn(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), by2);
          r[i] = __float_as_uint(scaled.x);
          r[i + 1] = __float_as_uint(scaled.y);
        }
        if (!(there >> piece & 1)) {
#pragma unroll
          for (int i = s * 16; i < s * 16 + 16; ++i) r[i] = 0xff800000u;
        }
#pragma unroll
        for (int i = s * 16; i < s * 16 + 16; i += 4) {
          m0 = fmaxf(m0, fmaxf(__uint_as_float(r[i]), __uint_as_float(r[i + 1])));
          m1 = fmaxf(m1, fmaxf(__uint_as_float(r[i + 2]), __uint_as_float(r[i + 3])));
        }
        most = fmaxf(most, fmaxf(m0, m1));
      }
      if (in_walk == 0) {
        reference = -INFINITY;
        row_sum = 0.f;
      }
      float factor = 1.f;
      const bool moves = in_walk == 0 || most > reference + kSlack;      // (-inf + kSlack is -inf; false for NaN)
      if (moves) {
        if (in_walk != 0) factor = reference == most ? 1.f : exp2_ftz(reference - most);
        reference = most;
      }
      const bool rescales = in_walk != 0 && __any_sync(0xffffffffu, moves);
      const float shift = reference == -INFINITY ? 0.f : kHalfLift - reference;
      const float2 shift2 = make_float2(shift, shift);
      if constexpr (!L::kOver) {
        // the product before still reads the probabilities and adds to the result
        if (j > 0 && !__all_sync(0xffffffffu, barrier_wait(product_done(tile), (j - 1) & 1, p.status, kWaitProduct))) { alive = false; break; }
        tcgen05_fence_after();
      }
      if (rescales) {      // rare: some row of the warp has moved (over the scores, the product before is done: its results came first)
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          tmem_load_16(tmem_o + c * 16, o);
          tmem_load_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
          tmem_store_16(tmem_o + c * 16, o);
        }
      }
      float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
#pragma unroll
      for (int c = 0; c < kKeys / 32; ++c) {
        uint32_t packed[16];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const float weight = weight_of(value_scale[info][(c * 32 + s * 16) >> piece_shift]);
          const float2 weight2 = make_float2(weight, weight);
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const int at = c * 32 + s * 16 + i;
            const float2 t0 = __fadd2_rn(make_float2(__uint_as_float(r[at]), __uint_as_float(r[at + 1])), shift2);
            const float2 t1 = __fadd2_rn(make_float2(__uint_as_float(r[at + 2]), __uint_as_float(r[at + 3])), shift2);
            const float2 e0 = make_float2(exp2_ftz(t0.x), exp2_ftz(t0.y)), e1 = make_float2(exp2_ftz(t1.x), exp2_ftz(t1.y));
            sum0 = __fadd2_rn(sum0, e0);
            sum1 = __fadd2_rn(sum1, e1);
            const float2 w0 = __fmul2_rn(e0, weight2), w1 = __fmul2_rn(e1, weight2);
            packed[(s * 16 + i) / 2] = half_pair(w0.x, w0.y);
            packed[(s * 16 + i) / 2 + 1] = half_pair(w1.x, w1.y);
          }
        }
        tmem_store_16(tmem_p + c * 16, packed);
      }
      const float2 sum01 = __fadd2_rn(sum0, sum1);
      row_sum = row_sum * factor + (sum01.x + sum01.y);
      tmem_store_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) barrier_arrive(probabilities(tile));

      if (in_walk == tiles - 1) {
        // ---- the end of a walk: the part leaves ----
        if (!__all_sync(0xffffffffu, barrier_wait(product_done(tile), j & 1, p.status, kWaitProduct))) { alive = false; break; }
        tcgen05_fence_after();
        if (walk == 0) sum_kept = row_sum;
        const float up = 1.f / down;
        float* const to = p.prefix_parts + (slot0 + row_in_block) * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          if (c * 32 >= p.head_dim) break;
          uint32_t o[32];
          tmem_load_32(tmem_o + c * 32, o);
          tmem_load_wait();
          if (row < rows) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              float4 four = make_float4(__uint_as_float(o[i]) * up, __uint_as_float(o[i + 1]) * up, __uint_as_float(o[i + 2]) * up, __uint_as_float(o[i + 3]) * up);
              float4* const at = reinterpret_cast<float4*>(to + c * 32 + i);
              if (walk > 0) {
                const float4 before = *at;
                four = make_float4(before.x + four.x, before.y + four.y, before.z + four.z, before.w + four.w);
              }
              *at = four;
            }
          }
          __syncwarp();
        }
        tcgen05_fence_before();
      }
    }
    p.prefix_stats[slot0 + row_in_block] = make_float2(alive ? reference : -INFINITY, sum_kept);
  }

  tcgen05_fence_before();
  __syncthreads();
  let_later_start();
  if (warp == kIssuerWarp) {
    tcgen05_fence_after();
    tmem_dealloc(tmem_base, L::kTmemColumns);
  }
}

// Rows of a page and head, `D` columns wide (what a head has less arrives as zeros), as many as a tile takes of a page.
tq_status prefix_maps(CUtensorMap* maps, const KeyedParams& p, int width) {
  EncodeTiled encode = encode_tiled();
  TQ_REQUIRE(encode != nullptr, TQ_EXTERNAL, "the CUDA driver does not provide cuTensorMapEncodeTiled");
  if (p.pages == 0) return TQ_OK;
  const void* operands[2] = {p.k, p.v};
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.head_dim), (static_cast<cuuint64_t>(p.pages) * p.kv_heads) << p.page_shift};
  TQ_REQUIRE(dims[1] < (1ull << 31), TQ_UNSUPPORTED, "a pool of more than 2^31 tokens and heads");
  const cuuint64_t byte_strides[1] = {static_cast<cuuint64_t>(p.head_dim)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(width), static_cast<cuuint32_t>(p.page_shift < 7 ? 1 << p.page_shift : kKeys)};
  const cuuint32_t element_strides[2] = {1, 1};
  for (int i = 0; i < 2; ++i) {
    const CUresult result = encode(&maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(operands[i]), dims, byte_strides, box, element_strides,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    TQ_REQUIRE(result == CUDA_SUCCESS, TQ_UNSUPPORTED, "this cache cannot be described to TMA (driver code %d)", static_cast<int>(result));
  }
  return TQ_OK;
}

template <int D, int TILES>
tq_status launch_prefix(const KeyedParams& p, bool bf16, long long ctas, cudaStream_t stream) {
  using L = PrefixLayout<D, TILES>;
  CUtensorMap maps[2] = {};
  if (tq_status s = prefix_maps(maps, p, D)) return s;
  TQ_CUDA(cudaFuncSetAttribute(prefix_attention_kernel<D, TILES>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(L::kSmemBytes)));
  TQ_CUDA(launch_overlapped(prefix_attention_kernel<D, TILES>, dim3(static_cast<unsigned>(ctas)), L::kThreads, L::kSmemBytes, stream, maps[0], maps[1], p, bf16));
  return check_launch("prefix_attention_kernel");
}

// Parts of each unit (run, key head, block of rows): enough CTAs for the SMs. The tiles of keys are known up to the table's width only.
struct PrefixPlan {
  int rows, row_blocks, splits;
  long long units;
  size_t stats_bytes, parts_bytes;
  size_t bytes() const { return stats_bytes + parts_bytes; }
};

PrefixPlan plan_prefix(const KeyedParams& p, int runs, long long keys, int32_t device) {
  PrefixPlan plan = {};
  const long long rows = static_cast<long long>(p.each) * p.group * p.q_tokens;
  plan.rows = rows <= kTileRows ? kTileRows : 2 * kTileRows;
  plan.row_blocks = static_cast<int>((rows + plan.rows - 1) / plan.rows);
  plan.units = static_cast<long long>(runs) * p.kv_heads * plan.row_blocks;
  const long long tiles = keys / kKeys;
  const long long sms = sm_count(device);
  long long splits = plan.units >= sms ? 1 : sms / plan.units;
  if (splits > tiles / 2) splits = tiles / 2;
  plan.splits = static_cast<int>(splits < 1 ? 1 : splits);
  const long long slots = plan.units * plan.splits * plan.rows;
  plan.stats_bytes = static_cast<size_t>(slots) * sizeof(float2);
  plan.parts_bytes = static_cast<size_t>(slots) * (p.head_dim <= 64 ? 64 : 128) * sizeof(float);
  return plan;
}

}  // namespace
}  // namespace tq

namespace {

// A block of scratch for both kernels: this one's statistics and parts, then keyed.cu's.
bool prefix_takes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_tokens, int64_t head_dim, int64_t page_tokens, int64_t blocks, int64_t runs) {
  const int page_shift = tq::page_shift_of(page_tokens);
  return batch > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && q_tokens > 0 && blocks > 0 && page_shift >= 0 && blocks < (1LL << 30) >> page_shift &&
         batch < (1LL << 24) && kv_heads < 65536 && q_tokens < (1LL << 24) && heads / kv_heads * q_tokens < (1LL << 24) && head_dim > 0 && head_dim <= 128 && runs > 0 && batch % runs == 0 &&
         batch / runs * (heads / kv_heads * q_tokens) < (1LL << 30);
}

}  // namespace

extern "C" tq_status tq_prefix_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_tokens, int64_t head_dim,
                                                         int64_t page_tokens, int64_t blocks, int64_t runs, int32_t device, size_t* bytes) {
  TQ_REQUIRE(bytes != nullptr, TQ_INVALID_ARGUMENT, "null out-pointer");
  *bytes = 0;
  if (!prefix_takes(batch, heads, kv_heads, q_tokens, head_dim, page_tokens, blocks, runs)) return TQ_OK;
  tq::KeyedParams p = {};
  tq::keyed_extents(p, batch, heads, kv_heads, q_tokens, head_dim, 1.0, 0, 0);
  p.each = static_cast<int>(batch / runs);
  *bytes = tq::plan_prefix(p, static_cast<int>(runs), blocks * page_tokens, device).bytes() + tq::keyed_workspace(true, p, blocks * page_tokens, device);
  return TQ_OK;
}

extern "C" tq_status tq_prefix_attention_launch(tq_dtype dtype, const void* q, const void* k_pages, const void* v_pages, const float* k_scales,
                                                const float* v_scales, const int32_t* table, const int32_t* lengths, const int32_t* shared, void* out,
                                                int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_tokens, int64_t head_dim, int64_t pages,
                                                int64_t page_tokens, int64_t blocks, int64_t table_stride, int64_t runs, const int64_t* q_strides,
                                                const int64_t* out_strides, double scale, void* workspace, size_t workspace_bytes, int32_t device,
                                                void* stream) {
  TQ_REQUIRE(q_strides != nullptr && out_strides != nullptr, TQ_INVALID_ARGUMENT, "null strides");
  if (tq::recording()) {
    struct Kept { int64_t q[3], out[3]; } kept;
    for (int i = 0; i < 3; ++i) {
      kept.q[i] = q_strides[i];
      kept.out[i] = out_strides[i];
    }
    return tq::record([=](int32_t d, void* s) {
      return tq_prefix_attention_launch(dtype, q, k_pages, v_pages, k_scales, v_scales, table, lengths, shared, out, batch, heads, kv_heads, q_tokens, head_dim,
                                        pages, page_tokens, blocks, table_stride, runs, kept.q, kept.out, scale, workspace, workspace_bytes, d, s);
    });
  }
  if (tq_status s = tq::cache_checks(dtype, batch, kv_heads, head_dim, pages, page_tokens, blocks)) return s;
  TQ_REQUIRE(heads >= 0 && q_tokens >= 0 && runs >= 0, TQ_INVALID_ARGUMENT, "negative heads=%lld, q_tokens=%lld or runs=%lld", (long long)heads,
             (long long)q_tokens, (long long)runs);
  if (batch == 0 || heads == 0 || q_tokens == 0) return TQ_OK;
  TQ_REQUIRE(kv_heads > 0 && heads % kv_heads == 0, TQ_INVALID_ARGUMENT, "%lld heads do not share %lld key heads evenly", (long long)heads, (long long)kv_heads);
  TQ_REQUIRE(runs > 0 && batch % runs == 0, TQ_INVALID_ARGUMENT, "%lld sequences are not %lld equal runs", (long long)batch, (long long)runs);
  TQ_REQUIRE(scale > 0.0 && scale <= tq::kKeyedMostScale, TQ_UNSUPPORTED, "the score scale must be positive and finite in f32, not %g", scale);
  TQ_REQUIRE(q != nullptr && out != nullptr && lengths != nullptr && shared != nullptr, TQ_INVALID_ARGUMENT, "null operand or result");
  TQ_REQUIRE(blocks == 0 || table != nullptr, TQ_INVALID_ARGUMENT, "null table");
  TQ_REQUIRE(pages == 0 || (k_pages != nullptr && v_pages != nullptr && k_scales != nullptr && v_scales != nullptr), TQ_INVALID_ARGUMENT, "null cache");
  TQ_REQUIRE(tq::keyed_query_fits(q, q_strides, out, out_strides, batch, heads, q_tokens), TQ_UNSUPPORTED,
             "queries must be 16-byte aligned with strides that are multiples of 8 elements, results aligned to their type, with no negative strides");
  TQ_REQUIRE(tq::aligned_to(k_pages, 16) && tq::aligned_to(v_pages, 16) && tq::aligned_to(k_scales, 4) && tq::aligned_to(v_scales, 4) &&
                 tq::aligned_to(table, 4) && tq::aligned_to(lengths, 4) && tq::aligned_to(shared, 4),
             TQ_UNSUPPORTED, "the cache's codes must be 16-byte aligned, its other tensors 4-byte aligned");
  TQ_REQUIRE(blocks == 0 || prefix_takes(batch, heads, kv_heads, q_tokens, head_dim, page_tokens, blocks, runs), TQ_UNSUPPORTED,
             "extents beyond the kernel's index range");
  tq::DeviceScope device_scope(device);
  if (tq_status s = device_scope.status()) return s;
  tq::KeyedParams p = {};
  p.status = tq::wait_status_for(device);
  TQ_REQUIRE(p.status.abort != nullptr, TQ_RESOURCE_EXHAUSTED, "no device memory for the status word");
  p.q = q;
  p.k = k_pages;
  p.v = v_pages;
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.table = table;
  p.lengths = lengths;
  p.table_stride = table_stride;
  p.blocks = static_cast<int>(blocks);
  p.page_shift = tq::page_shift_of(page_tokens);
  p.pages = static_cast<int>(pages);
  p.out = out;
  for (int i = 0; i < 3; ++i) {
    p.q_strides[i] = q_strides[i];
    p.out_strides[i] = out_strides[i];
  }
  tq::keyed_extents(p, batch, heads, kv_heads, q_tokens, head_dim, scale, 0, 0);
  const cudaStream_t cuda_stream = static_cast<cudaStream_t>(stream);
  const long long keys = blocks * page_tokens;
  if (keys < tq::kPrefixTile || pages == 0) return tq::keyed_attention(dtype, true, p, keys, workspace, workspace_bytes, device, cuda_stream);      // nothing to share
  p.each = static_cast<int>(batch / runs);
  const tq::PrefixPlan plan = tq::plan_prefix(p, static_cast<int>(runs), keys, device);
  TQ_REQUIRE(workspace != nullptr && workspace_bytes >= plan.bytes() && tq::aligned_to(workspace, 16), TQ_INVALID_ARGUMENT,
             "this attention needs %zu bytes of workspace and more, 16-byte aligned, and was given %zu", plan.bytes(), workspace_bytes);
  TQ_REQUIRE(plan.units * plan.splits < (1LL << 31), TQ_UNSUPPORTED, "too many heads and rows for one launch");
  p.shared = shared;
  p.prefix_rows = plan.rows;
  p.row_blocks = plan.row_blocks;
  p.splits = plan.splits;
  p.prefix_parts = static_cast<float*>(workspace);
  p.prefix_stats = reinterpret_cast<float2*>(static_cast<char*>(workspace) + plan.parts_bytes);
  char* const rest = static_cast<char*>(workspace) + plan.bytes();
  const long long ctas = plan.units * plan.splits;
  const bool bf16 = dtype == TQ_BF16, wide = head_dim > 64, two = plan.rows > tq::kTileRows;
  const auto held = tq::hold_scratch(workspace);      // all kernels, one after the other
  const tq_status s = wide ? (two ? tq::launch_prefix<128, 2>(p, bf16, ctas, cuda_stream) : tq::launch_prefix<128, 1>(p, bf16, ctas, cuda_stream))
                           : (two ? tq::launch_prefix<64, 2>(p, bf16, ctas, cuda_stream) : tq::launch_prefix<64, 1>(p, bf16, ctas, cuda_stream));
  if (s != TQ_OK) return s;
  return tq::keyed_attention(dtype, true, p, keys, rest, workspace_bytes - plan.bytes(), device, cuda_stream);
}
