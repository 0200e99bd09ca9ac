// Attention of sequences that share their first keys, over a paged cache in 8 bits, for sm_100a: the shared keys are read once for all of them.
//
//   A run of `each` sequences has its first S keys in common (S whole tiles of 128 keys). For the rows of all its queries, R = each * queries * heads of
//   a key head, and a part of the S keys, this kernel leaves
//     m = a reference point near max_j s_j      s_j = scale * q . k_j, in units of log2
//     l = sum_j 2^(s_j - m)                     o = sum_j 2^(s_j - m) v_j      (f32, not divided)
//   keyed.cu then takes each sequence's own keys and joins: any number of (m, l, o) of one row add up after 2^(m - max m).
//
// The products are the tensor cores' (tcgen05, f16 operands, f32 sums in tensor memory): a CTA owns one or two tiles of 128 rows and walks its part of
// the keys 128 at a time, in steps of 64: of each tile two steps' scores lie in tensor memory, so that one is in its softmax while the products of the
// other run (128 keys at once over single scores: 256 x 64/8 heads of 128 behind 30000 tokens 479 us, so 343).
//
// Bound: no unit is above 40 % (tensor pipe 32, issue slots 38, special functions 33, shared memory 25 % with two tiles): 128 keys take 2.5 us for two
// tiles and 1.75 for one (heads of 128; of 64 2.3 and 1.55). Without the exponentials they would take 2.2, without the conversion, or 7 in 8 of the first
// products, 2.35: what is left is the chain of a step (scores, maximum, exponentials, probabilities, product), of which a CTA holds two or four.
//
//   warps of a tile (4)   a row a thread: tcgen05.ld of a step's 64 scores, the keys' scales, ex2, sum; probabilities times the values' scales go
//                         back into tensor memory as f16 pairs, the A operand of the second product
//   converters (4 warps)  e4m3 codes, as TMA brought them from the pages, to f16 (exact) in the layout of the products' operands
//   producer (1 warp)     looks pages up, loads their codes (TMA) and scales
//   issuer (1 thread)     S = Q K^T and O += P V
//
// Precision: as in keyed.cu. A row of queries is brought to f16 by a power of two (only elements 2^-38 of its largest, or less, lose digits); codes are
// exact in f16; probabilities are rounded to f16 (2^-11 of each). A page's scale of the values multiplies the probabilities before that, relative to the
// largest scale of the part: pages whose scales are kSpan or more powers of two below would lose digits in f16, so they get a walk of their own with
// another reference, one for each kSpan powers of two. (Rare: a cache's scales follow its values' magnitudes.)
//
// No row is masked: a sequence with a query that does not see all the shared keys takes no part (its rows are computed and not used) and reads its keys
// itself. A page that is not there is left out, with zeros for its codes and -inf for its scores.
//
// Every wait is bounded; one that gives up sets the device status word, and the CTA leaves through the normal teardown. No load uses multicast.
#include <cuda.h>

#include <cmath>
#include <type_traits>

#include "common.h"
#include "keyed.h"
#include "tcgen05.h"

namespace tq {
namespace {

constexpr int kKeys = kPrefixTile;          // of a tile, which is loaded and converted at a time
constexpr int kStep = kKeys / 2;            // a step
constexpr int kTileRows = 128;              // rows of an instruction's tile
constexpr float kSlack = 8.f;               // a row's reference point moves when a step's maximum is more than kSlack (in units of log2) above it
constexpr int kSpan = 12;                   // powers of two of the values' scales that a walk takes
constexpr int kInfos = 8;                   // tiles whose scales are on chip
constexpr int kSixteens = kKeys / 16;       // of a tile: the smallest page

enum PrefixWait { kWaitReady = 0x50465831, kWaitRawEmpty, kWaitRawFull, kWaitSpent, kWaitKeysFull, kWaitValuesFull,
                  kWaitScores, kWaitProbabilities, kWaitProduct };

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
  // Tensor memory: the scores of each tile for two steps, with their probabilities over them, and the results.
  static constexpr uint32_t kColumnO = TILES * 2 * kStep;
  static constexpr uint32_t kTmemColumns = kColumnO + TILES * D <= 256 ? 256 : 512;
  static_assert(kColumnO + TILES * D <= 512, "more than tensor memory");
  static constexpr int kThreads = TILES * 128 + 256;                          // tiles' warps, converters, producer and issuer (and two idle warps)
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
__device__ __forceinline__ uint4 load_shared_16(uint32_t address) {
  uint4 word;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(word.x), "=r"(word.y), "=r"(word.z), "=r"(word.w) : "r"(address));
  return word;
}
__device__ __forceinline__ void store_shared_16(uint32_t address, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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
__device__ __forceinline__ float power_of_two(int exponent) { return __uint_as_float(static_cast<uint32_t>(exponent + 127) << 23); }      // -126 to 127
// The exponent of a scale of values, from 2^-126 on (what is smaller is as good as that); zero, infinities and NaN have none.
__device__ __forceinline__ bool is_plain(float scale) { return fabsf(scale) > 0.f && fabsf(scale) < INFINITY; }
__device__ __forceinline__ int exponent_of(float scale) { return max(static_cast<int>(__float_as_uint(scale) >> 23 & 0xff), 1) - 127; }
// A scale relative to 2^(top + 1), in [2^-kSpan, 1) if it is the walk's; 0 for a page that is another walk's.
__device__ __forceinline__ float weight_of(float scale, int top) {
  if (!is_plain(scale)) return scale;
  const int below = top - exponent_of(scale);
  if (below < 0 || below >= kSpan) return 0.f;
  return top == 127 ? scale * power_of_two(-126) * 0.25f : top == 126 ? scale * power_of_two(-126) * 0.5f : scale * power_of_two(-top - 1);
}

template <int D, int TILES>
__global__ void __launch_bounds__(PrefixLayout<D, TILES>::kThreads, 1)
prefix_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ KeyedParams p,
                        const bool bf16) {
  using L = PrefixLayout<D, TILES>;
  constexpr int kRaw = L::kRawStages, kSub = L::kSub;
  extern __shared__ unsigned char raw_smem[];
  // Of a tile of keys, by sixteens: the scale of the keys, without its sign (-1: no page), and of the values, then relative to the walk's largest; by
  // pieces (what lies in one page): bits of those whose page is there, and of those whose keys' scale is negative.
  __shared__ __align__(16) float key_scale[kInfos][kSixteens], value_scale[kInfos][kSixteens], value_weight[kInfos][kSixteens];
  __shared__ uint32_t pages_there[kInfos], turned_keys[kInfos];
  __shared__ int highest, lowest;                                 // exponents of the values' scales
  const uint32_t base = (smem_address(raw_smem) + 1023u) & ~1023u;
  const uint32_t barriers = base + L::kOffsetBarriers;
  const uint32_t ready = barriers;                                // queries, highest and lowest are there
  auto raw_full = [&](int s) { return barriers + 8u * (1 + s); };
  auto raw_empty = [&](int s) { return barriers + 8u * (1 + kRaw + s); };
  const uint32_t after_raw = barriers + 8u * (1 + 2 * kRaw);
  auto keys_full = [&](int b) { return after_raw + 8u * b; };
  auto values_full = [&](int b) { return after_raw + 8u * (2 + b); };
  auto spent = [&](int b) { return after_raw + 8u * (4 + b); };   // the values of a tile j with j % 2 == b, and the keys of the next, have been read
  auto scores_full = [&](int t, int b) { return after_raw + 8u * (8 + 2 * t + b); };
  auto probabilities = [&](int t, int b) { return after_raw + 8u * (12 + 2 * t + b); };
  auto product_done = [&](int t) { return after_raw + 8u * (6 + t); };        // the last of a walk
  auto product_before = [&](int t) { return after_raw + 8u * (16 + t); };     // the one before it
  const uint32_t tmem_slot = after_raw + 8u * 18;
  static_assert(8 * (1 + 2 * kRaw + 18) + 4 <= 512, "barriers beyond their room");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kConvertWarp = 4 * TILES, kProducerWarp = kConvertWarp + 4, kIssuerWarp = kProducerWarp + 1;
  if (threadIdx.x == 0) {
    barrier_init(ready, 4 * TILES + 1);
    for (int s = 0; s < kRaw; ++s) {
      barrier_init(raw_full(s), 1);
      barrier_init(raw_empty(s), 4);
    }
    for (int b = 0; b < 2; ++b) {
      barrier_init(keys_full(b), 4);
      barrier_init(values_full(b), 4);
      barrier_init(spent(b), TILES);
      barrier_init(product_done(b), 1);
      barrier_init(product_before(b), 1);
      for (int t = 0; t < 2; ++t) {
        barrier_init(scores_full(t, b), 1);
        barrier_init(probabilities(t, b), 4);
      }
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kProducerWarp && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
  }
  if (warp == kIssuerWarp) tmem_alloc(tmem_slot, L::kTmemColumns);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  uint32_t tmem_base;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
  wait_for_earlier();
  let_later_start();                                              // (what each sequence has of its own: keyed.cu, which waits for this at its end)
  if (blockIdx.x == 0 && threadIdx.x == 0) p.status.begin();

  // Which part of which block of which key head of which run.
  const int splits = p.part_count - 1;
  const int part = static_cast<int>(blockIdx.x) % splits, unit = static_cast<int>(blockIdx.x) / splits;
  constexpr int kBlockRows = TILES * kTileRows;
  const int blocks = p.part_rows / kBlockRows;
  const int block = unit % blocks, head_index = unit / blocks;
  const int kv_head = head_index % p.kv_heads, run = head_index / p.kv_heads;
  const int rows_each = p.group * p.q_tokens, rows = p.each * rows_each, row0 = block * kBlockRows;
  const long long slot0 = part_slot(p, run, kv_head, part, row0);

  // A tile's warp has 32 rows of queries, kLanes neighbouring lanes 16 bytes each of kRowsAtOnce rows at a time; lane l works out where row l lies.
  constexpr int kLanes = D / 8, kRowsAtOnce = 32 / kLanes, kLoads = 32 / kRowsAtOnce;
  uint4 word[kLoads];
  if (warp < kConvertWarp && row0 + warp * 32 < rows) {
    const int mine = min(row0 + warp * 32 + lane, rows - 1);
    const int of = mine / rows_each, inside = mine - of * rows_each, token = inside / p.group, head = kv_head * p.group + (inside - token * p.group);
    const long long offset = (run * static_cast<long long>(p.each) + of) * p.q_strides[0] + head * p.q_strides[1] + token * p.q_strides[2];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int from = i * kRowsAtOnce + lane / kLanes, column = lane % kLanes * 8;
      const long long there = __shfl_sync(0xffffffffu, offset, from);
      word[i] = make_uint4(0, 0, 0, 0);
      if (row0 + warp * 32 + from < rows && column < p.head_dim) word[i] = *reinterpret_cast<const uint4*>(static_cast<const char*>(p.q) + 2 * (there + column));
    }
  } else {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) word[i] = make_uint4(0, 0, 0, 0);
  }
  // Every warp finds for itself what the part has, and the first sequence that takes part.
  const int tiles_all = shared_keys(p, run) / kKeys;
  const int tile0 = static_cast<int>(static_cast<long long>(tiles_all) * part / splits);
  const int tiles = static_cast<int>(static_cast<long long>(tiles_all) * (part + 1) / splits) - tile0;
  int taker = -1;
  for (int i0 = 0; tiles > 0 && taker < 0 && i0 < p.each; i0 += 32) {
    const int length = i0 + lane < p.each ? min(max(p.lengths[run * p.each + i0 + lane], 0), p.blocks << p.page_shift) : 0;
    const uint32_t takers = __ballot_sync(0xffffffffu, i0 + lane < p.each && takes_part(p, tiles_all * kKeys, length));
    if (takers != 0) taker = run * p.each + i0 + __ffs(takers) - 1;
  }
  if (taker < 0) {                                                // nothing here, or nobody to want it: the same in the whole CTA
    for (int i = threadIdx.x; i < kBlockRows; i += L::kThreads) p.row_stats[slot0 + i] = make_float2(-INFINITY, 0.f);
    if (warp == kIssuerWarp) tmem_dealloc(tmem_base, L::kTmemColumns);
    return;
  }

  const int32_t* const table = p.table + static_cast<long long>(taker) * p.table_stride;
  const int piece_shift = min(p.page_shift, 7), pieces = kKeys >> piece_shift;      // of a tile: what lies in one page
  // Walks over the keys, one for each kSpan powers of two of the values' scales: known once `ready` completes.
  auto walks = [&] { return highest < lowest ? 1 : (highest - lowest) / kSpan + 1; };

  if (warp >= kConvertWarp && warp < kProducerWarp) {
    // ---- converters: items in the order K(0), K(1), V(0), K(2), V(1), ... V(last) of all walks together ----
    if (__all_sync(0xffffffffu, barrier_wait(ready, 0, p.status, kWaitReady))) {
      const int steps = tiles * walks();
      const int thread = threadIdx.x - kConvertWarp * 32;
      constexpr unsigned kPiecesKey = D / 16, kEach = kKeys * kPiecesKey / 128;      // 16 codes; of a key, of a thread
      for (int n = 0; n < 2 * steps; ++n) {
        const bool values = n != 0 && (n == 2 * steps - 1 || n % 2 == 0);
        const int step = n == 0 ? 0 : values ? (n == 2 * steps - 1 ? steps - 1 : n / 2 - 1) : (n + 1) / 2;
        const int stage = n % kRaw, buffer = step & 1;
        if (!__all_sync(0xffffffffu, barrier_wait(raw_full(stage), (n / kRaw) & 1, p.status, kWaitRawFull))) break;
        // V(j) and K(j + 1) lie where V(j - 2) and K(j - 1) were
        const int j = values ? step : step - 1;
        if (j >= 1 && !__all_sync(0xffffffffu, barrier_wait(spent(j & 1), ((j - 1) >> 1) & 1, p.status, kWaitSpent))) break;
        const uint32_t from = base + L::kOffsetRaw + stage * L::kRawBytes;
        const uint32_t to = base + (values ? L::kOffsetValues : L::kOffsetKeys) + buffer * L::kOperandBytes;
        const int info = step % kInfos;
        const uint32_t there = pages_there[info], turned = values ? 0u : turned_keys[info];
        if (!values && thread < kSixteens) value_weight[info][thread] = weight_of(value_scale[info][thread], highest - step / tiles * kSpan);
        // A thread has the same 16 elements of every kStride-th key. Units of 16 bytes are exchanged within 128 by the key's place in 8. Eight neighbouring
        // threads have four pieces of an even key and four of the next; of wide heads, one's first half and the other's second: they read from
        // eight different places in 128 bytes, and write to eight.
        constexpr unsigned kStride = 128 / kPiecesKey, kAtOnce = 4;
        const unsigned eight = static_cast<unsigned>(thread) / 8, in_eight = static_cast<unsigned>(thread) % 8;
        const unsigned key0 = D == 64 ? static_cast<unsigned>(thread) / 4 : eight / 2 * 2 + in_eight / 4;
        const unsigned piece = D == 64 ? in_eight % 4 : in_eight % 4 + 4 * (in_eight / 4 ^ (eight & 1)), turn = key0 & 7;
        const uint32_t from0 = from + key0 * D + piece * 16;
        const uint32_t line = to + piece / 4 * L::kSubBytes + key0 * 128, unit = piece % 4 * 2;
        const uint32_t to0 = line + ((unit ^ turn) << 4), to1 = line + (((unit + 1) ^ turn) << 4);
        auto convert = [&](auto is_plain_tile) {
#pragma unroll
          for (unsigned k = 0; k < kEach; k += kAtOnce) {
            uint4 codes[kAtOnce];
#pragma unroll
            for (unsigned u = 0; u < kAtOnce; ++u) codes[u] = load_shared_16(from0 + (k + u) * kStride * D);
#pragma unroll
            for (unsigned u = 0; u < kAtOnce; ++u) {
              if (!is_plain_tile) {
                const unsigned at_page = (key0 + (k + u) * kStride) >> piece_shift;
                const uint32_t keeps = there >> at_page & 1 ? 0xffffffffu : 0u, turns = turned >> at_page & 1 ? 0x80808080u : 0u;
                codes[u] = make_uint4((codes[u].x & keeps) ^ turns, (codes[u].y & keeps) ^ turns, (codes[u].z & keeps) ^ turns, (codes[u].w & keeps) ^ turns);
              }
              const uint2 a = decode_four(codes[u].x), b = decode_four(codes[u].y), c = decode_four(codes[u].z), d = decode_four(codes[u].w);
              store_shared_16(to0 + (k + u) * kStride * 128, a.x, a.y, b.x, b.y);
              store_shared_16(to1 + (k + u) * kStride * 128, c.x, c.y, d.x, d.y);
            }
          }
        };
        if (there == (1u << pieces) - 1 && turned == 0) convert(std::true_type{});
        else convert(std::false_type{});
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          barrier_arrive(values ? values_full(buffer) : keys_full(buffer));
          barrier_arrive(raw_empty(stage));
        }
      }
    }
  } else if (warp >= kProducerWarp) {
    if (warp == kProducerWarp) {
      // ---- producer: the whole warp, a lane for each piece of a tile ----
      bool known = false;
      int steps = tiles, issued = 0;
      // A lane's piece of a tile: its page (-1: none), looked up two steps before its keys are asked for, and that page's scales, one step before.
      auto key_of = [&](int step) { return (tile0 + step % tiles) * kKeys + (lane << piece_shift); };
      auto look_up = [&](int step) {
        if (lane >= pieces) return -1;
        const int at_block = key_of(step) >> p.page_shift, page = table[at_block];
        if (page >= 0 && page < p.pages) return page;
        report(p.status, kKeyedPage, taker, at_block);
        return -1;
      };
      float scale_k = 1.f, scale_v = 1.f;
      auto ask_scales = [&](int page) {
        const long long at = static_cast<long long>(page) * p.kv_heads + kv_head;
        scale_k = page >= 0 ? p.k_scales[at] : 1.f;
        scale_v = page >= 0 ? p.v_scales[at] : 1.f;
      };
      int page_here = look_up(0), page_next = look_up(1);      // of the keys that are asked for next, and of those behind
      int page_before = -1, page_values = -1;                  // of the keys asked for last, and of those before them
      ask_scales(page_here);
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
        // (keys are a step ahead of values, but for the last)
        const int page = values ? (n == 2 * steps - 1 ? page_before : page_values) : page_here;
        const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
        const uint32_t piece_bytes = static_cast<uint32_t>(D) << piece_shift;
        if (!values) {
          // (last used by step - kInfos, whose scores were taken long ago: the operands' buffers are two deep)
          const float magnitude = __shfl_sync(0xffffffffu, page >= 0 ? fabsf(scale_k) : -1.f, (lane * 16) >> piece_shift & 7);
          const float of_values = __shfl_sync(0xffffffffu, scale_v, (lane * 16) >> piece_shift & 7);
          if (lane < kSixteens) {
            key_scale[step % kInfos][lane] = magnitude;
            value_scale[step % kInfos][lane] = of_values;
          }
          const uint32_t turned = __ballot_sync(0xffffffffu, scale_k < 0.f);
          if (lane == 0) {
            pages_there[step % kInfos] = there;
            turned_keys[step % kInfos] = turned;
          }
        }
        __syncwarp();
        if (lane == 0) barrier_expect_tx(raw_full(stage), piece_bytes * __popc(there));
        __syncwarp();
        if (page >= 0) {
          const int row = ((page * p.kv_heads + kv_head) << p.page_shift) + (key_of(step) & ((1 << p.page_shift) - 1));      // (below 2^31: prefix_maps)
          tma_load_rows(base + L::kOffsetRaw + stage * L::kRawBytes + lane * piece_bytes, values ? &map_v : &map_k, raw_full(stage), 0, row);
        }
        if (!values) {
          page_values = page_before;
          page_before = page_here;
          page_here = page_next;
          ask_scales(page_here);
          page_next = look_up(step + 2);
        }
        issued = n + 1;
      }
      // where a wait gave up: copies that are under way land before the CTA leaves
      for (int n = max(0, issued - kRaw); n < issued; ++n) {
        for (uint32_t spin = 0; spin < kSpinLimit && !barrier_try_wait(raw_full(n % kRaw), (n / kRaw) & 1); ++spin) {
        }
      }
    } else if (warp == kIssuerWarp + 1) {
      // ---- the values' scales of the part: how far apart they are ----
      int high = -1000, low = 1000;
      const int block0 = (tile0 * kKeys) >> p.page_shift, block1 = ((tile0 + tiles) * kKeys - 1) >> p.page_shift;
#pragma unroll 4
      for (int n = block0 + lane; n <= block1; n += 32) {
        const int page = table[n];
        if (page < 0 || page >= p.pages) continue;
        const float scale = p.v_scales[static_cast<long long>(page) * p.kv_heads + kv_head];
        if (is_plain(scale)) {
          const int exponent = exponent_of(scale);
          high = max(high, exponent);
          low = min(low, exponent);
        }
      }
      high = __reduce_max_sync(0xffffffffu, high);
      low = __reduce_min_sync(0xffffffffu, low);
      if (lane == 0) {
        highest = high;
        lowest = low;
        barrier_arrive(ready);
      }
    } else if (warp == kIssuerWarp) {
      // ---- issuer ----
      if (elect_one()) {
        constexpr uint32_t kHigh = kDescriptorHigh;
        constexpr uint32_t scores_instruction = prefix_instruction(kStep, false), values_instruction = prefix_instruction(D, true);
        const uint32_t low_q = descriptor_low(base, 0), low_k = descriptor_low(base + L::kOffsetKeys, 0);
        const uint32_t low_v = descriptor_low(base + L::kOffsetValues, L::kSubBytes);
        // both operands K-major: 16 elements are 32 bytes in the swizzled line
        // (step H of four: a thread issues these one after another, and what it works out in between is time the tensor cores wait)
        auto scores = [&](int t, auto which) {
          constexpr int H = decltype(which)::value;
          const uint32_t q = low_q + t * (L::kOperandBytes >> 4), k = low_k + (H / 2) * (L::kOperandBytes >> 4) + (H % 2) * (kStep * 128 >> 4);
#pragma unroll
          for (int s = 0; s < kSub; ++s) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f16_split(tmem_base + (2 * t + H % 2) * kStep, q + s * (L::kSubBytes >> 4) + kk * 2, kHigh, k + s * (L::kSubBytes >> 4) + kk * 2, kHigh,
                            scores_instruction, (s != 0 || kk != 0) ? 1u : 0u);
          }
          mma_commit(scores_full(t, H % 2));
        };
        // P from tensor memory (16 keys are 8 columns), V MN-major (16 keys are 2048 bytes)
        auto product = [&](int t, auto which, uint32_t goes_on) {
          constexpr int H = decltype(which)::value;
          const uint32_t v = low_v + (H / 2) * (L::kOperandBytes >> 4) + (H % 2) * (kStep / 16) * (2048 >> 4), from = tmem_base + (2 * t + H % 2) * kStep;
#pragma unroll
          for (int kk = 0; kk < kStep / 16; ++kk)
            mma_f16_tmem_a(tmem_base + L::kColumnO + t * D, from + kk * 8, v + kk * (2048 >> 4), kHigh, values_instruction, kk != 0 ? 1u : goes_on);
        };
        if (barrier_wait(ready, 0, p.status, kWaitReady) && barrier_wait(keys_full(0), 0, p.status, kWaitKeysFull)) {
          const int steps = 2 * tiles * walks();
          tcgen05_fence_after();
#pragma unroll
          for (int t = 0; t < TILES; ++t) {
            scores(t, std::integral_constant<int, 0>{});
            scores(t, std::integral_constant<int, 1>{});
            mma_commit(spent(1));                                 // (the keys of the first tile)
          }
          int h = 0, left = 2 * tiles;                            // left: steps of the walk
          uint32_t goes_on = 0, phase = 0;                        // phase: of the operands' buffers, which come round every four steps
          auto step = [&](auto which) {
            constexpr int H = decltype(which)::value, kNext = (H + 2) % 4;
            if (H % 2 == 0 && !barrier_wait(values_full(H / 2), phase, p.status, kWaitValuesFull)) return false;
            const bool more = h + 2 < steps;
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
              if (!barrier_wait(probabilities(t, H % 2), H / 2, p.status, kWaitProbabilities)) return false;
              tcgen05_fence_after();
              product(t, which, goes_on);
              if (left <= 2) mma_commit(left == 1 ? product_done(t) : product_before(t));
              // the scores of the step after next, over the probabilities that this product reads before: what one thread issues runs in order
              if (more) {
                if (H % 2 == 0 && t == 0) {
                  if (!barrier_wait(keys_full(kNext / 2), H < 2 ? phase : phase ^ 1, p.status, kWaitKeysFull)) return false;
                  tcgen05_fence_after();
                }
                scores(t, std::integral_constant<int, kNext>{});
              }
              if (H % 2 == 1) mma_commit(spent(H / 2));
            }
            goes_on = 1;
            if (--left == 0) {
              left = 2 * tiles;
              goes_on = 0;
            }
            return ++h < steps;
          };
          while (step(std::integral_constant<int, 0>{}) && step(std::integral_constant<int, 1>{}) && step(std::integral_constant<int, 2>{}) &&
                 step(std::integral_constant<int, 3>{}))
            phase ^= 1;
        }
      }
    }
  } else {
    // ---- a row a thread ----
    const int tile = warp / 4, row_in_block = static_cast<int>(threadIdx.x), row = row0 + row_in_block;
    // The rows of queries, as f16 times a power of two.
    float row_scale = 0.f;
    auto store_queries = [&](auto widen) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const float2 pairs[4] = {widen(word[i].x), widen(word[i].y), widen(word[i].z), widen(word[i].w)};
        float largest = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) largest = fmaxf(largest, fmaxf(fabsf(pairs[c].x), fabsf(pairs[c].y)));
#pragma unroll
        for (int offset = 1; offset < kLanes; offset *= 2) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, offset));
        // to [2^14, 2^15), by 2^126 at most; none for infinities (as in keyed.cu)
        int exponent = max(static_cast<int>(__float_as_uint(largest) >> 23) - 127, -112);
        if (exponent > 127) exponent = 14;
        const float up = power_of_two(14 - exponent), back = __shfl_sync(0xffffffffu, p.scale_log2 * power_of_two(exponent - 14), lane % kRowsAtOnce * kLanes);
        if (lane / kRowsAtOnce == i) row_scale = back;
        const int in_tile = warp % 4 * 32 + i * kRowsAtOnce + lane / kLanes, unit = lane % kLanes;
        store_shared_16(base + tile * L::kOperandBytes + unit / 8 * L::kSubBytes + in_tile * 128 + ((unit % 8 ^ (in_tile & 7)) << 4),
                        half_pair(pairs[0].x * up, pairs[0].y * up), half_pair(pairs[1].x * up, pairs[1].y * up), half_pair(pairs[2].x * up, pairs[2].y * up),
                        half_pair(pairs[3].x * up, pairs[3].y * up));
      }
    };
    if (bf16) store_queries([](uint32_t pair) { return make_float2(__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u)); });
    else store_queries([](uint32_t pair) { return __half22float2(*reinterpret_cast<const __half2*>(&pair)); });
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) barrier_arrive(ready);
    bool alive = __all_sync(0xffffffffu, barrier_wait(ready, 0, p.status, kWaitReady));
    const int steps = alive ? 2 * tiles * walks() : 0, top_exponent = highest;

    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const uint32_t tmem_s = tmem_base + tile * 2 * kStep + lanes, tmem_o = tmem_base + L::kColumnO + tile * D + lanes;
    float reference = -INFINITY, row_sum = 0.f, sum_kept = 0.f;
    if (row0 + warp * 32 >= rows) {
      // A warp without rows takes part in the hand-overs only: its scores and its result mean nothing.
      for (int h = 0; h < steps; ++h) {
        if (!__all_sync(0xffffffffu, barrier_wait(scores_full(tile, h & 1), (h >> 1) & 1, p.status, kWaitScores))) break;
        if (lane == 0) barrier_arrive(probabilities(tile, h & 1));
        __syncwarp();
      }
      alive = false;
    }
    for (int h = 0, walk = 0, in_walk = 0; alive && h < steps; ++h) {
      if (!__all_sync(0xffffffffu, barrier_wait(scores_full(tile, h & 1), (h >> 1) & 1, p.status, kWaitScores))) { alive = false; break; }
      tcgen05_fence_after();
      uint32_t r[kStep];
      const uint32_t tmem_step = tmem_s + (h & 1) * kStep;
#pragma unroll
      for (int i = 0; i < kStep; i += 32) tmem_load_32(tmem_step + i, *reinterpret_cast<uint32_t(*)[32]>(&r[i]));
      const int info = (h >> 1) % kInfos, first = (h & 1) * (kSixteens / 2);
      float scale[kSixteens / 2], weight[kSixteens / 2], most_of[kSixteens / 2];
      *reinterpret_cast<float4*>(scale) = *reinterpret_cast<const float4*>(&key_scale[info][first]);
      *reinterpret_cast<float4*>(weight) = *reinterpret_cast<const float4*>(&value_weight[info][first]);
      tmem_load_wait();
#pragma unroll
      for (int s = 0; s < kSixteens / 2; ++s) {
        auto at = [&](int i) { return __uint_as_float(r[s * 16 + i]); };
        const float m0 = max3(max3(at(0), at(1), at(2)), at(3), at(4)), m1 = max3(max3(at(5), at(6), at(7)), at(8), at(9));
        const float m2 = max3(max3(at(10), at(11), at(12)), at(13), at(14));
        most_of[s] = scale[s] < 0.f ? -INFINITY : fmaxf(max3(m0, m1, m2), at(15)) * (row_scale * scale[s]);
      }
      const float most = fmaxf(max3(most_of[0], most_of[1], most_of[2]), most_of[3]);
      if (in_walk == 0) row_sum = 0.f;
      float factor = 1.f;
      const bool moves = in_walk == 0 || most > reference + kSlack;      // (-inf + kSlack is -inf; false for NaN)
      if (moves) {
        if (in_walk != 0) factor = reference == most ? 1.f : exp2_ftz(reference - most);
        reference = most;
      }
      const float shift = reference == -INFINITY ? 0.f : kHalfLift - reference;
      if (in_walk != 0 && __any_sync(0xffffffffu, moves)) {      // rare: some row of the warp has moved
        // the product of the step before is done: the next scores come after it, or it is told
        const bool last = in_walk + 1 == 2 * tiles;
        if (!__all_sync(0xffffffffu, last ? barrier_wait(product_before(tile), walk & 1, p.status, kWaitProduct)
                                          : barrier_wait(scores_full(tile, (h + 1) & 1), ((h + 1) >> 1) & 1, p.status, kWaitScores))) {
          alive = false;
          break;
        }
        tcgen05_fence_after();
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
      for (int i = 0; i < kStep; i += 2) {
        const float by = row_scale * scale[i / 16], to = scale[i / 16] < 0.f ? -INFINITY : shift;      // (scores of codes of 0 are 0)
        const float2 t = __ffma2_rn(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), make_float2(by, by), make_float2(to, to));
        const float2 e = make_float2(exp2_ftz(t.x), exp2_ftz(t.y));
        if (i % 4 == 0) sum0 = __fadd2_rn(sum0, e);
        else sum1 = __fadd2_rn(sum1, e);
        const float2 weighted = __fmul2_rn(e, make_float2(weight[i / 16], weight[i / 16]));
        r[i / 2] = half_pair(weighted.x, weighted.y);
      }
      tmem_store_32(tmem_step, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
      tmem_store_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) barrier_arrive(probabilities(tile, h & 1));
      const float2 sum01 = __fadd2_rn(sum0, sum1);
      row_sum = row_sum * factor + (sum01.x + sum01.y);

      if (++in_walk == 2 * tiles) {
        // ---- the end of a walk: the part leaves ----
        if (!__all_sync(0xffffffffu, barrier_wait(product_done(tile), walk & 1, p.status, kWaitProduct))) { alive = false; break; }
        tcgen05_fence_after();
        if (walk == 0) sum_kept = row_sum;
        const int top = highest < lowest ? -1 : top_exponent - walk * kSpan;
        const float up = power_of_two(min(top + 1, 127)), twice = top == 127 ? 2.f : 1.f;
        // 32 columns at a time. A thread has a row, and a store to each of 32 rows is as many lines; through the tile's queries' place, which nobody
        // reads any more behind the last walk, eight lanes write 128 bytes of a row (256 rows of 128: 8600 cycles without).
        const uint32_t stage = base + tile * L::kOperandBytes + warp % 4 * (L::kOperandBytes / 4);
        const bool staged = steps == 2 * tiles;
        float* const to = p.row_parts + (slot0 + warp * 32) * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          if (c * 32 >= p.head_dim) break;
          uint32_t o[32];
          tmem_load_32(tmem_o + c * 32, o);
          tmem_load_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * up * twice);
          if (staged) {
#pragma unroll
            for (int u = 0; u < 8; ++u) store_shared_16(stage + lane * 128 + ((u ^ (lane & 7)) << 4), o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
            __syncwarp();
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              const int of = n * 4 + lane / 8, unit = lane % 8;
              const uint4 four = load_shared_16(stage + of * 128 + ((unit ^ (of & 7)) << 4));
              if (row0 + warp * 32 + of < rows) *reinterpret_cast<uint4*>(to + of * D + c * 32 + unit * 4) = four;
            }
          } else if (row < rows) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              float4 four = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
              float4* const at = reinterpret_cast<float4*>(to + lane * D + c * 32 + i);
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
        ++walk;
        in_walk = 0;
      }
    }
    if (row < rows) p.row_stats[slot0 + row_in_block] = make_float2(alive ? reference : -INFINITY, sum_kept);
  }

  tcgen05_fence_before();
  __syncthreads();
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

// Joins the parts of each row: the last one is the sequence's own keys', the others the shared keys', which count for sequences that take part. GROUP
// neighbouring lanes have eight elements of a row, and every GROUP-th of its parts each.
constexpr int kJoinThreads = 256;
template <typename T, int W, int GROUP>
__global__ void __launch_bounds__(kJoinThreads) prefix_join_kernel(const __grid_constant__ KeyedParams p, const long long items) {
  wait_for_earlier();
  const long long item = (static_cast<long long>(blockIdx.x) * kJoinThreads + threadIdx.x) / GROUP;
  const int member = threadIdx.x % GROUP;
  const bool there = item < items;
  const int eights = p.head_dim / 8;
  const int column = static_cast<int>(item % eights) * 8;
  long long rest = item / eights;
  const int head = static_cast<int>(rest % p.heads);
  rest /= p.heads;
  const int token = static_cast<int>(rest % p.q_tokens), sequence = there ? static_cast<int>(rest / p.q_tokens) : 0;
  const int run = sequence / p.each, kv_head = head / p.group;
  const int row = ((sequence - run * p.each) * p.q_tokens + token) * p.group + head % p.group;
  const int length = min(max(p.lengths[sequence], 0), p.blocks << p.page_shift), shared = shared_keys(p, run);
  const int first = shared > 0 && takes_part(p, shared, length) ? 0 : p.part_count - 1;
  float most = -INFINITY, total = 0.f, value[8] = {};
  auto rescale = [](float from, float to) { return from == to ? 1.f : exp2_ftz(from - to); };
  if (there) {
    constexpr int kAtOnce = 4;
    for (int part0 = first + member; part0 < p.part_count; part0 += kAtOnce * GROUP) {
      float2 stats[kAtOnce];
      float4 near[kAtOnce], far[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int part = part0 + u * GROUP;
        stats[u] = make_float2(-INFINITY, 0.f);
        if (part < p.part_count) {
          const long long slot = part_slot(p, run, kv_head, part, row);
          stats[u] = p.row_stats[slot];
          const float4* from = reinterpret_cast<const float4*>(p.row_parts + slot * W + column);
          near[u] = from[0];
          far[u] = from[1];
        }
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        // no keys: what lies there is nothing then (of keys of which some are none, and others' scores NaN, the sum is)
        if (stats[u].x == -INFINITY && stats[u].y == stats[u].y) continue;
        const float both = fmaxf(most, stats[u].x), mine = rescale(most, both), theirs = rescale(stats[u].x, both);
        const float x[8] = {near[u].x, near[u].y, near[u].z, near[u].w, far[u].x, far[u].y, far[u].z, far[u].w};
        most = both;
        total = total * mine + stats[u].y * theirs;
#pragma unroll
        for (int c = 0; c < 8; ++c) value[c] = value[c] * mine + x[c] * theirs;
      }
    }
  }
#pragma unroll
  for (int offset = 1; offset < GROUP; offset *= 2) {
    const float other = __shfl_xor_sync(0xffffffffu, most, offset), both = fmaxf(most, other);
    const float mine = rescale(most, both), theirs = rescale(other, both);
    most = both;
    total = total * mine + __shfl_xor_sync(0xffffffffu, total, offset) * theirs;
#pragma unroll
    for (int c = 0; c < 8; ++c) value[c] = value[c] * mine + __shfl_xor_sync(0xffffffffu, value[c], offset) * theirs;
  }
  if (!there || member != 0) return;
  const bool sees_some = length - p.q_tokens + token >= 0;      // (a query before the first key: zeros)
  const float inverse = 1.f / total;
  T* const to = static_cast<T*>(p.out) + sequence * p.out_strides[0] + head * p.out_strides[1] + token * p.out_strides[2] + column;
  Vec<T, 8> out;
#pragma unroll
  for (int c = 0; c < 8; ++c) out.v[c] = from_compute<T, float>(sees_some ? value[c] * inverse : 0.f);
  if ((reinterpret_cast<uintptr_t>(to) & 15) == 0) {
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(&out);
  } else {
#pragma unroll
    for (int c = 0; c < 8; ++c) to[c] = out.v[c];
  }
}

template <typename T, int W>
tq_status launch_join(const KeyedParams& p, cudaStream_t stream) {
  const long long items = static_cast<long long>(p.batch) * p.heads * p.q_tokens * (p.head_dim / 8);
  const int group = p.part_count > 16 ? 8 : p.part_count > 4 ? 4 : 1;
  const long long ctas = (items * group + kJoinThreads - 1) / kJoinThreads;
  TQ_REQUIRE(ctas < (1LL << 31), TQ_UNSUPPORTED, "too many rows for one launch");
  const dim3 grid(static_cast<unsigned>(ctas));
  TQ_CUDA(group == 8   ? launch_overlapped(prefix_join_kernel<T, W, 8>, grid, kJoinThreads, 0, stream, p, items)
          : group == 4 ? launch_overlapped(prefix_join_kernel<T, W, 4>, grid, kJoinThreads, 0, stream, p, items)
                       : launch_overlapped(prefix_join_kernel<T, W, 1>, grid, kJoinThreads, 0, stream, p, items));
  return check_launch("prefix_join_kernel");
}

// What becomes of a call, by expected time (us, B200): each sequence reads all its keys (kApart), or the shared ones are taken for all rows of a run
// together, streamed through warps of 8 or 16 rows as a sequence's are (kStreamed), or on the tensor cores' tiles (kTiles). How many keys are shared is
// known on the device only: the table's width stands for it. Measured (us, from a graph, cold caches), apart, streamed, on tiles: 16 x 4 sequences of 12
// heads of 64 behind 1024 tokens 24.6, 30.7, 53.2; 12 x 4 of them behind 2048 30.7, 28.7, 49.2; 64 x 4 of 32/8 heads of 128 behind 2000 172, 96, 186; 16 x 16 of 12
// heads of 64 behind 4000 189, 62, 125; 16 of 32/8 heads of 128 behind 4000 30.5, -, 34.8; 64 behind 8001 143, -, 57; 32 of 12 heads of 64 behind 4000 38.9, -, 26.7.
// Tiles of 256 rows halve what is converted, and double what parts cost: 64 x 32/8 behind 8001 57 with 128 rows, 65 with 256; 256 x 64/8 behind 30000 494, 350.
enum PrefixForm { kApart, kStreamed, kTiles };
struct PrefixPlan {
  PrefixForm form;
  int tiles;                       // of 128 rows, of a CTA
  int part_rows, part_count, typical;
  long long ctas;
  size_t parts_bytes, stats_bytes, keyed_bytes;
  size_t apart_bytes;              // (over a pool of no pages each sequence is its own)
  size_t bytes() const {
    const size_t together = parts_bytes + stats_bytes + keyed_bytes;
    return together > apart_bytes ? together : apart_bytes;
  }
};
constexpr double kStartTime = 10.0;                    // a CTA's, to its first scores and behind its last ones
constexpr double kTileTimes[2][2] = {{1.55, 2.3}, {1.75, 2.5}};     // 128 keys: heads up to 64, 128; one tile of rows, two
constexpr double kPartBytesPerMicrosecond = 2.2e6;
constexpr double kOwnTime = 9.0, kJoinTime = 3.0;      // what each sequence has behind the shared keys; the join
constexpr double kStreamedTime = 6.0;                  // the join, and runs that end later than sequences
constexpr int kMostStreamed = 16;                      // rows of a run: a warp's
constexpr long long kOwnKeys = 128;                    // what a sequence is taken to have behind the shared keys, beside streamed ones
// And behind those on tiles, which says how many warps its CTA has. (24 of 20/4 heads of 128 behind 9000 tokens, with up to 3000 of their own: 63 us by
// kOwnKeys, so 53; with up to 60 39 both.)
constexpr long long kTailKeys = 512;

PrefixPlan plan_prefix(KeyedParams p, int runs, long long keys, int32_t device) {
  PrefixPlan plan = {};
  const long long rows = static_cast<long long>(p.each) * p.group * p.q_tokens, tiles = keys / kKeys, sms = sm_count(device);
  const int wide = p.head_dim > 64;
  const double apart = keyed_time(true, p, keys, device);
  plan.apart_bytes = keyed_workspace(true, p, keys, device);
  plan.form = kApart;
  if (p.each == 1 || tiles < 2) return plan;
  // (streamed, runs and sequences are one launch's units, of one tile of rows each)
  KeyedParams both = p;
  both.runs = runs;
  both.batch = runs + p.batch;
  both.typical = static_cast<int>((runs * keys + p.batch * (keys < kOwnKeys ? keys : kOwnKeys)) / (runs + p.batch));
  const double streamed = rows <= kMostStreamed ? kStreamedTime + keyed_time(true, both, keys, device) : INFINITY;
  double on_tiles = INFINITY;
  long long blocks = 0, units = 0, splits = 0;
  for (int t = 1; t <= (rows <= kTileRows ? 1 : 2); ++t) {
    const long long t_blocks = (rows + t * kTileRows - 1) / (t * kTileRows), t_units = static_cast<long long>(runs) * p.kv_heads * t_blocks;
    for (long long waves = 1; waves <= 4; ++waves) {
      const long long most = waves * sms / t_units;
      const long long t_splits = most < 1 ? 1 : most < tiles ? most : tiles;
      const double part_bytes = 2.0 * t_units * t_splits * t * kTileRows * (wide ? 512 : 256);      // written and read
      const double all_waves = std::ceil(static_cast<double>(t_units * t_splits) / sms);
      const double time = kOwnTime + kJoinTime + all_waves * (kStartTime + std::ceil(static_cast<double>(tiles) / t_splits) * kTileTimes[wide][t - 1]) +
                          part_bytes / kPartBytesPerMicrosecond;
      if (time >= on_tiles) continue;
      on_tiles = time;
      plan.tiles = t;
      blocks = t_blocks;
      units = t_units;
      splits = t_splits;
    }
  }
  if (apart <= streamed && apart <= on_tiles) return plan;
  plan.form = streamed <= on_tiles ? kStreamed : kTiles;
  plan.part_rows = static_cast<int>(plan.form == kStreamed ? rows : blocks * plan.tiles * kTileRows);
  plan.part_count = plan.form == kStreamed ? 2 : static_cast<int>(splits) + 1;
  plan.ctas = units * splits;
  const size_t slots = static_cast<size_t>(runs) * p.kv_heads * plan.part_count * plan.part_rows;
  plan.parts_bytes = slots * (wide ? 128 : 64) * sizeof(float);
  plan.stats_bytes = (slots * sizeof(float2) + 15) / 16 * 16;
  plan.typical = both.typical;
  if (plan.form == kTiles) {
    both = p;
    both.typical = plan.typical = static_cast<int>(keys < kTailKeys ? keys : kTailKeys);
  }
  plan.keyed_bytes = keyed_workspace(true, both, keys, device);
  return plan;
}

bool prefix_takes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_tokens, int64_t head_dim, int64_t page_tokens, int64_t blocks, int64_t runs) {
  const int page_shift = page_shift_of(page_tokens);
  return batch > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && q_tokens > 0 && blocks > 0 && page_shift >= 0 && blocks < (1LL << 30) >> page_shift &&
         batch < (1LL << 24) && kv_heads < 65536 && q_tokens < (1LL << 24) && heads / kv_heads * q_tokens < (1LL << 24) && head_dim > 0 && head_dim <= 128 &&
         runs > 0 && batch % runs == 0 && batch / runs * (heads / kv_heads * q_tokens) < (1LL << 24);
}

// The extents of a call as both kinds of kernels take them, and what becomes of it.
PrefixPlan plan_call(KeyedParams& p, int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_tokens, int64_t head_dim, int64_t page_tokens, int64_t blocks,
                     int64_t runs, double scale, int32_t device) {
  keyed_extents(p, batch, heads, kv_heads, q_tokens, head_dim, scale, 0, 0);
  p.each = static_cast<int>(batch / runs);
  return plan_prefix(p, static_cast<int>(runs), blocks * page_tokens, device);
}

}  // namespace
}  // namespace tq

extern "C" tq_status tq_prefix_attention_form(int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_tokens, int64_t head_dim, int64_t page_tokens,
                                              int64_t blocks, int64_t runs, int32_t device, int32_t* form, int32_t* parts, int32_t* block_rows) {
  TQ_REQUIRE(form != nullptr && parts != nullptr && block_rows != nullptr, TQ_INVALID_ARGUMENT, "null out-pointer");
  TQ_REQUIRE(tq::prefix_takes(batch, heads, kv_heads, q_tokens, head_dim, page_tokens, blocks, runs), TQ_INVALID_ARGUMENT, "no attention of these extents");
  tq::KeyedParams p = {};
  const tq::PrefixPlan plan = tq::plan_call(p, batch, heads, kv_heads, q_tokens, head_dim, page_tokens, blocks, runs, 1.0, device);
  *form = plan.form == tq::kApart ? TQ_ATTENTION_APART : plan.form == tq::kStreamed ? TQ_ATTENTION_STREAMED : TQ_ATTENTION_TILES;
  *parts = plan.form == tq::kApart ? 0 : plan.part_count - 1;
  *block_rows = plan.form == tq::kApart ? 0 : plan.form == tq::kStreamed ? plan.part_rows : plan.tiles * tq::kTileRows;
  return TQ_OK;
}

extern "C" tq_status tq_prefix_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_tokens, int64_t head_dim,
                                                         int64_t page_tokens, int64_t blocks, int64_t runs, int32_t device, size_t* bytes) {
  TQ_REQUIRE(bytes != nullptr, TQ_INVALID_ARGUMENT, "null out-pointer");
  *bytes = 0;
  if (!tq::prefix_takes(batch, heads, kv_heads, q_tokens, head_dim, page_tokens, blocks, runs)) return TQ_OK;
  tq::KeyedParams p = {};
  *bytes = tq::plan_call(p, batch, heads, kv_heads, q_tokens, head_dim, page_tokens, blocks, runs, 1.0, device).bytes();
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
  TQ_REQUIRE(blocks == 0 || tq::prefix_takes(batch, heads, kv_heads, q_tokens, head_dim, page_tokens, blocks, runs), TQ_UNSUPPORTED,
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
  const cudaStream_t cuda_stream = static_cast<cudaStream_t>(stream);
  const long long keys = blocks * page_tokens;
  const tq::PrefixPlan plan = tq::plan_call(p, batch, heads, kv_heads, q_tokens, head_dim, page_tokens, blocks, runs, scale, device);
  TQ_REQUIRE(plan.bytes() == 0 || (workspace != nullptr && workspace_bytes >= plan.bytes() && tq::aligned_to(workspace, 16)), TQ_INVALID_ARGUMENT,
             "this attention needs %zu bytes of workspace, 16-byte aligned, and was given %zu", plan.bytes(), workspace_bytes);
  if (plan.form == tq::kApart || pages == 0) return tq::keyed_attention(dtype, true, p, keys, workspace, workspace_bytes, device, cuda_stream);
  TQ_REQUIRE(plan.ctas < (1LL << 31), TQ_UNSUPPORTED, "too many heads and rows for one launch");
  char* const scratch = static_cast<char*>(workspace);
  p.shared = shared;
  p.part_rows = plan.part_rows;
  p.part_count = plan.part_count;
  p.row_parts = reinterpret_cast<float*>(scratch);
  p.row_stats = reinterpret_cast<float2*>(scratch + plan.parts_bytes);
  const bool bf16 = dtype == TQ_BF16, wide = head_dim > 64;
  const auto held = tq::hold_scratch(workspace);      // all kernels, one after the other
  tq::KeyedParams keyed = p;
  keyed.typical = plan.typical;
  if (plan.form == tq::kStreamed) {
    keyed.runs = static_cast<int>(runs);
    keyed.batch = static_cast<int>(runs + batch);
  } else {
    const tq_status s = wide ? (plan.tiles == 2 ? tq::launch_prefix<128, 2>(p, bf16, plan.ctas, cuda_stream) : tq::launch_prefix<128, 1>(p, bf16, plan.ctas, cuda_stream))
                             : (plan.tiles == 2 ? tq::launch_prefix<64, 2>(p, bf16, plan.ctas, cuda_stream) : tq::launch_prefix<64, 1>(p, bf16, plan.ctas, cuda_stream));
    if (s != TQ_OK) return s;
    keyed.late = true;
    keyed.status = tq::wait_status_for(device);               // (the kernel before may still run, with its own word)
  }
  if (tq_status s = tq::keyed_attention(dtype, true, keyed, keys, scratch + plan.parts_bytes + plan.stats_bytes, plan.keyed_bytes, device, cuda_stream)) return s;
  if (bf16) return wide ? tq::launch_join<__nv_bfloat16, 128>(p, cuda_stream) : tq::launch_join<__nv_bfloat16, 64>(p, cuda_stream);
  return wide ? tq::launch_join<__half, 128>(p, cuda_stream) : tq::launch_join<__half, 64>(p, cuda_stream);
}
