// Attention of a few query rows a head against many keys, with a window, sinks and shared key heads, for sm_100a: over a
// paged cache in 8 bits, or over dense keys and values in 16.
//
//   position of query i of a sequence of L keys and Q queries: p = L - Q + i (aligned at the ends)
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j    over j <= p with (j > p - window or j < sinks); zeros where p < 0
//   8 bits: k_j = code_j * k_scale[page, head], v_j likewise (e4m3 codes, an f32 scale a page and head)
//
// Heads that share a key head are rows of one tile, so a key is read once for all of them. Bound: HBM (the visible keys' and
// values' bytes). The multiply-adds of up to 16 rows would not fit the CUDA cores beside it, so both products are warp-level
// matrix instructions, transposed: S^T = K Q^T and O^T = V^T P^T, keys (then head elements) the instruction's 16 rows and query rows its 8
// columns, so that a head of its own wastes 7 columns of 8 and not 15 rows of 16. The order of the summed-over axis of
// a product is free, so a lane's 16 contiguous bytes of a key are whatever elements of the head the instruction takes
// from it, and the query is laid out to match; a value's bytes are paired with the next key's by one byte permute.
//
// Memory: a warp has a ring of two stages of 8 KB (16 to 64 keys and their values) that TMA fills from a page or through the dense
// strides; no warp waits for another. Keys straight into registers left too little under way (616 us for 16 x 8 key heads of 128 of 20001 to
// 40000 keys with a CTA a head, 232 with the split below; rings 178).
//
// Split: the chunks of all (sequence, key head, 8 or 16 rows), each unit counted a little longer than it is, are one range in equal shares, a
// warp each; whole units are written at once, and what a border between shares cuts is left in scratch as (maximum, sum, unscaled result) and
// joined by a second kernel whose start passes under the first one's end. With a CTA for each share, units of a chunk or two (short sequences of
// a ragged batch) queued up behind one another's latency: 64 x 12 heads of 64 of 1 to 2000 keys 94 us, with a warp 24 (without the host). Few
// units have a CTA's warps join theirs before (one head of 128000 keys 121 -> 23 us). Units of few chunks have a CTA of 2, 4 or 8 warps each
// and no second kernel (plan_shape). Tried beside the second kernel: the last CTA to arrive at a ticket joins (48 us for 33 + 6: fences, and code that nobody
// has run yet, at the very end).
//
// Measured (kernels and join; us, and of HBM's 6456 GB/s): 16 x 64/8 heads of 128, 20001 to 40000 keys in 8 bits 163 (0.93); 32 x 32/8 heads,
// 2052 keys in 16 bits 50 (0.83); 64 x 12 heads of 64, 1 to 2000 keys 27 (0.57), all 1000 21 (0.74); four queries of 48 x 32/8, 1028 keys 34.5
// (0.44); 12 heads of 64, 1500 keys 7. How chunks are split goes by the table's width, not by lengths, which are on the device. A fixed 12 us (launch, lengths, first pages and keys, join) is what dealt-out short ones pay, 5 us what
// units do, and 16 rows twice the products; the special functions, tensor pipe and issue slots are below 50 %.
//
// Precision: scores, maxima, sums and results in f32. e4m3 to f16 is exact, and so is the query in f16: a row is scaled by a power of two to
// a maximum of 2^14 (by 2^126 at most, which brings every bf16 into f16's range), so only elements 2^-38 of it or less lose digits. Probabilities
// against f16 values (cache codes too) are rounded to f16: half a step is 2^-11, under the result's 2^-8 in bf16, and below 2^-21 of the row's largest
// 2^-32 of that (kLift). Against bf16 values they take two bf16 operands, the rounded value and what rounding took off (2^-16).
//
// A masked key must not reach a result through 0 * NaN: its score is replaced, and a value that no row of the tile sees becomes zeros in the
// stage. Where rows see different keys (several queries, at an end of the window) and a value they do see is no number, or its page's scale, the
// chunk's product is taken once a query with that query's keys alone, and each row keeps its own.
#include <cuda.h>

#include <cmath>
#include <mutex>
#include <type_traits>

#include "common.h"
#include "keyed.h"
#include "tcgen05.h"

namespace tq {
namespace {

constexpr int kKeyedWarps = 4;
constexpr int kKeyedThreads = 32 * kKeyedWarps;

// Chunks of a warp in flight or in use. Measured, 16 x 8 key heads of 128 of 20001 to 40000 keys: two stages and two CTAs an SM 165 us, three
// stages 164, two stages and three CTAs 181 (registers spill); four queries under a window 45.2, 49.2, 44.8.
constexpr int kKeyedStages = 2;
constexpr uint32_t kStageBytes = 8192;
constexpr uint32_t kWarpRing = kKeyedStages * kStageBytes;
constexpr int kWaitKeyed = 0x4b455931;      // "KEY1"
constexpr float kSlack = 8.f;
template <typename M>
constexpr float kLift = std::is_same_v<M, __half> ? kHalfLift : 0.f;

// BITS of a key element, W: the head's elements, rounded up to 64 or 128.
template <int BITS, int W>
struct KeyedShape {
  static constexpr int kKeys = static_cast<int>(kStageBytes) * 4 / (W * BITS);      // a chunk: what a warp takes at a time, keys and then values in a stage
  static constexpr int kTiles = kKeys / 16;
  static constexpr int kPieces = W * BITS / 512;                      // 16-byte pieces of a key a lane takes (four lanes a key)
  static constexpr int kPieceWidth = 128 / BITS;                      // head elements in one
  static constexpr int kValueWords = W * BITS / 256;                  // 32-bit words of a value a lane takes (eight lanes a value)
  static constexpr int kSlices = W / 16;                              // 16 head elements of the result
  static constexpr int kLine = W * BITS / 8 < 128 ? W * BITS / 8 : 128;      // bytes of a key in a box: 64 or 128, swizzled as many
  static constexpr int kLines = W * BITS / 8 / kLine;                 // boxes side by side (two for 16-bit heads over 64)
  static constexpr uint32_t kBoxBytes = kKeys * kLine;                // a chunk's keys (or values), one of the boxes side by side
  // Where byte `column` of key `key` of a chunk lies: TMA exchanges 16-byte units within a line by the line's place in 8.
  static __device__ __forceinline__ uint32_t at(int key, int column) {
    const uint32_t box = kLines == 1 ? 0u : static_cast<uint32_t>(column / kLine) * kBoxBytes;
    const int unit = (column % kLine) / 16;
    const int turned = kLine == 128 ? unit ^ (key & 7) : unit ^ ((key >> 1) & 3);
    return box + key * kLine + turned * 16 + column % 16;
  }
};
// The rings and, where a CTA's warps join their parts of a unit first, room for each warp's first part (its last one goes where its ring was).
constexpr size_t keyed_smem(bool gather, int w, int nt, int warps = kKeyedWarps) { return 1024 + warps * (kWarpRing + (gather ? 8 * nt * w * sizeof(float) : 0)); }

__device__ __forceinline__ uint4 load_shared_16(uint32_t address) {
  uint4 word;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(word.x), "=r"(word.y), "=r"(word.z), "=r"(word.w) : "r"(address));
  return word;
}
__device__ __forceinline__ uint2 load_shared_8(uint32_t address) {
  uint2 word;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(word.x), "=r"(word.y) : "r"(address));
  return word;
}
__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap* map, uint32_t bar, int column, int row) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(column), "r"(row)
      : "memory");
}
__device__ __forceinline__ void tma_load_tokens(uint32_t dst, const CUtensorMap* map, uint32_t bar, int column, int token, int head, int batch) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(column), "r"(token), "r"(head), "r"(batch)
      : "memory");
}

// Two e4m3 codes (the low or the high half of a word) as f16.
__device__ __forceinline__ uint32_t decode_low(uint32_t codes) {
  uint32_t pair;
  asm("{\n\t.reg .b16 low, high;\n\tmov.b32 {low, high}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, low;\n\t}" : "=r"(pair) : "r"(codes));
  return pair;
}
__device__ __forceinline__ uint32_t decode_high(uint32_t codes) {
  uint32_t pair;
  asm("{\n\t.reg .b16 low, high;\n\tmov.b32 {low, high}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, high;\n\t}" : "=r"(pair) : "r"(codes));
  return pair;
}

// D = A B + C, 16 x 8 x 16. (C apart from D: the first product of a sum has zeros there, which cost no register.)
template <typename M>
__device__ __forceinline__ void multiply(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
  if constexpr (std::is_same_v<M, __half>) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  }
}
template <typename M>
__device__ __forceinline__ void multiply(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
  if (first) multiply<M>(d, a, b0, b1, 0.f, 0.f, 0.f, 0.f);
  else multiply<M>(d, a, b0, b1, d[0], d[1], d[2], d[3]);
}

// An 8 x 8 tile of 16-bit elements, transposed across the warp.
__device__ __forceinline__ uint32_t transpose_tile(uint32_t pair) {
  uint32_t out;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(out) : "r"(pair));
  return out;
}

template <typename M>
__device__ __forceinline__ uint32_t round_pair(float low, float high) {
  if constexpr (std::is_same_v<M, __nv_bfloat16>) {
    const __nv_bfloat162 pair = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&pair);
  } else {
    const __half2 pair = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&pair);
  }
}

template <typename T>
__device__ __forceinline__ float2 widen_pair(uint32_t pair) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    return make_float2(__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&pair));
  }
}

// The factor that brings what was gathered against one reference point to another; 1 where nothing finite was seen on either side.
__device__ __forceinline__ float rescale(float from, float to) { return from == to ? 1.f : exp2_ftz(from - to); }

// The keys that some query from position `low` to position `high` sees, in chunks: [0, sinks) and [start, stop), counted through.
struct ChunkList {
  int sinks, start, stop;
  __device__ int count() const { return sinks + stop - start; }
  __device__ int at(int i) const { return i < sinks ? i : i - sinks + start; }
};
__device__ __forceinline__ ChunkList chunks_of(int low, int high, int window, int sinks, int chunk) {
  ChunkList list;
  list.stop = (high + chunk) / chunk;                                            // high + 1 keys, rounded up (high >= -1)
  const int from = low - window + 1;
  list.start = min(max(from, 0) / chunk, list.stop);
  list.sinks = min((min(sinks, high + 1) + chunk - 1) / chunk, list.start);
  return list;
}

// Eight elements of a result row: the gathered values over their sum, zeros for a query before the first key.
template <typename T>
__device__ __forceinline__ void write_values(const KeyedParams& p, int batch, int kv_head, int row, int column, int length, float total, const float (&value)[8]) {
  const int token = row / p.group, head = kv_head * p.group + row % p.group;
  const bool sees_some = length - p.q_tokens + token >= 0;
  T* to = static_cast<T*>(p.out) + batch * p.out_strides[0] + head * p.out_strides[1] + token * p.out_strides[2] + column;
  const float inverse = sees_some ? 1.f / total : 0.f;
  uint32_t word[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) word[c] = sees_some ? round_pair<T>(value[2 * c] * inverse, value[2 * c + 1] * inverse) : 0u;
  if ((reinterpret_cast<uintptr_t>(to) & 15) == 0) {
    *reinterpret_cast<uint4*>(to) = make_uint4(word[0], word[1], word[2], word[3]);
  } else {
#pragma unroll
    for (int c = 0; c < 8; ++c) to[c] = reinterpret_cast<const T*>(word)[c];
  }
}

// PARTS: left as a part of the row's result.
template <typename T, int W, bool PARTS>
__device__ __forceinline__ void write_result(const KeyedParams& p, int batch, int kv_head, int row, int column, int length, float most, float total,
                                             const float (&value)[8]) {
  if constexpr (!PARTS) {
    write_values<T>(p, batch, kv_head, row, column, length, total, value);
  } else {
    const int own = batch - p.runs, run = own < 0 ? batch : own / p.each;
    const long long slot = part_slot(p, run, kv_head, own < 0 ? 0 : p.part_count - 1, own < 0 ? row : (own - run * p.each) * p.group * p.q_tokens + row);
    float4* const to = reinterpret_cast<float4*>(p.row_parts + slot * W + column);
    to[0] = make_float4(value[0], value[1], value[2], value[3]);
    to[1] = make_float4(value[4], value[5], value[6], value[7]);
    if (column == 0) p.row_stats[slot] = make_float2(most, total);
  }
}

// A sequence's chunks, by every query of it.
template <int BITS, int CHUNK, bool PARTS>
__device__ __forceinline__ int length_of(const KeyedParams& p, int sequence) {
  if constexpr (BITS == 16) return p.k_tokens;
  if constexpr (PARTS) {
    if (sequence < p.runs) return shared_keys(p, sequence);
    sequence -= p.runs;
  }
  return min(max(p.lengths[sequence], 0), p.blocks << p.page_shift);
}
// PARTS: a list without the keys that the sequence shares with its run.
template <int CHUNK, bool PARTS>
__device__ __forceinline__ ChunkList behind_prefix(const KeyedParams& p, int sequence, int length, ChunkList list) {
  if constexpr (PARTS) {
    static_assert(kPrefixTile % CHUNK == 0, "the keys behind the shared ones begin with a chunk");
    if (sequence < p.runs) return list;
    const int shared = shared_keys(p, (sequence - p.runs) / p.each);
    if (takes_part(p, shared, length)) list.start = min(max(list.start, shared / CHUNK), list.stop);
  }
  return list;
}
template <int BITS, int CHUNK, bool PARTS>
__device__ __forceinline__ ChunkList sequence_chunks(const KeyedParams& p, int sequence, int length) {
  // (rows of a run see all the shared keys; there is no window then)
  return behind_prefix<CHUNK, PARTS>(p, sequence, length, chunks_of(length - p.q_tokens, max(length - 1, -1), p.window, p.sinks, CHUNK));
}

// Where the chunks of all units (sequence, key head, tile of rows) are dealt out as one range of equal shares, a CTA each: a place in that range.
struct Place {
  int sequence;
  int before;      // places of the sequences before it
};

// The chunks that a head of sequence `sequence` counts for: one at least, so that each has somebody to write its result.
template <int BITS, int CHUNK, bool PARTS>
__device__ __forceinline__ int counted(const KeyedParams& p, int sequence) {
  return max(sequence_chunks<BITS, CHUNK, PARTS>(p, sequence, length_of<BITS, CHUNK, PARTS>(p, sequence)).count(), 1);
}

// What a unit costs beside its chunks, in chunks: to find it, its pages and its first keys, one after another, and its masked ends. Measured with
// 2, 4 and 6 of them, us: heads of 128, 48 x 8 of four queries under a window 41.2, 39.3, 40.4, 30 x 4 of 96 55.7, 51.4, 52.8; heads of 64
// (chunks of twice the keys) 100 x 12 34.3, 36.9, 39.0.
constexpr int unit_cost(int chunk) { return chunk > 32 ? 2 : 4; }
constexpr int kLeastShare = 4;       // of the same

// The range has less than 2^31 places (plan_shape sees to it). The first `longer` shares have one place more than the others.
struct Dealt {
  int total, shares, each, longer;
  __device__ int start(int share) const { return share * each + min(share, longer); }
  // the share that has place `at` of the range
  __device__ int holder(int at) const {
    const int border = longer * (each + 1);
    return at < border ? at / (each + 1) : longer + (at - border) / each;
  }
};

// All threads: the range, and where in it the share of each warp, first_share + warp, starts. Each thread adds up a run of sequences.
template <int BITS, int CHUNK, bool PARTS>
__device__ __forceinline__ Dealt deal(const KeyedParams& p, int first_share, Place& place) {
  __shared__ int warp_sum_of[kKeyedWarps];
  __shared__ Place found[kKeyedWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int units = p.kv_heads * p.row_tiles;
  if constexpr (BITS == 16) {      // all sequences are alike
    const int each = (unit_cost(CHUNK) + counted<BITS, CHUNK, PARTS>(p, 0)) * units;
    Dealt dealt;
    dealt.total = each * p.batch;
    dealt.shares = min(p.shares, (dealt.total + kLeastShare - 1) / kLeastShare);
    dealt.each = dealt.total / dealt.shares;
    dealt.longer = dealt.total % dealt.shares;
    const int sequence = dealt.start(min(first_share + warp, dealt.shares - 1)) / each;
    place = {sequence, sequence * each};
    return dealt;
  }
  const int run = (p.batch + kKeyedThreads - 1) / kKeyedThreads;
  const int first = min(static_cast<int>(threadIdx.x) * run, p.batch), last = min(first + run, p.batch);
  int mine = 0;
  for (int b = first; b < last; ++b) mine += unit_cost(CHUNK) + counted<BITS, CHUNK, PARTS>(p, b);
  mine *= units;
  int upto = mine;
#pragma unroll
  for (int offset = 1; offset < 32; offset *= 2) {
    const int other = __shfl_up_sync(0xffffffffu, upto, offset);
    if (lane >= offset) upto += other;
  }
  if (lane == 31) warp_sum_of[warp] = upto;
  __syncthreads();
  Dealt dealt;
  dealt.total = 0;
#pragma unroll
  for (int w = 0; w < kKeyedWarps; ++w) {
    if (w < warp) upto += warp_sum_of[w];
    dealt.total += warp_sum_of[w];
  }
  dealt.shares = min(p.shares, (dealt.total + kLeastShare - 1) / kLeastShare);
  dealt.each = dealt.total / dealt.shares;
  dealt.longer = dealt.total % dealt.shares;
#pragma unroll
  for (int w = 0; w < kKeyedWarps; ++w) {
    if (first_share + w >= dealt.shares) break;
    const int at = dealt.start(first_share + w);
    int before = upto - mine;
    if (before <= at && at < upto) {
      int b = first;
      for (; b < last; ++b) {
        const int here = (unit_cost(CHUNK) + counted<BITS, CHUNK, PARTS>(p, b)) * units;
        if (at < before + here) break;
        before += here;
      }
      found[w] = {b, before};
    }
  }
  __syncthreads();
  place = found[warp];
  return dealt;
}

// T: the type of q and out. BITS, W as above. NT: eights of rows of a tile. JOINS > 0 (SHARED): the chunks of all units are dealt out in equal
// shares, one a warp (then keyed_join_kernel follows), or each unit has a CTA, whose warps take every WARPS-th chunk each and meet in shared
// memory. ONE: a chunk lies in one page (or in none: dense keys).
template <typename T, int BITS, int W, int NT, int JOINS, bool ONE, int WARPS = kKeyedWarps, bool PARTS = false>
__global__ void __launch_bounds__(32 * WARPS, 8 / WARPS)
keyed_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ KeyedParams p) {
  using S = KeyedShape<BITS, W>;
  using M = std::conditional_t<BITS == 8, __half, T>;      // what the matrix instructions take
  constexpr bool SHARED = JOINS > 0;
  static_assert(!SHARED || WARPS == kKeyedWarps, "shares are dealt out to CTAs of four warps");
  constexpr int kUnitCost = unit_cost(S::kKeys);
  constexpr bool kTwoOperands = std::is_same_v<M, __nv_bfloat16>;
  constexpr int kRows = 8 * NT, kTiles = S::kTiles, kSlices = S::kSlices;
  static_assert(kRows * W * sizeof(float) <= kWarpRing, "a warp leaves its part where its stages were");
  extern __shared__ unsigned char raw_smem[];
  __shared__ float part_top[SHARED ? 1 : WARPS][kRows], part_sum[SHARED ? 1 : WARPS][kRows];
  __shared__ __align__(8) uint64_t full[WARPS][kKeyedStages];
  __shared__ int staged_page[WARPS][kKeyedStages][4];      // of each box of a stage; -1: not there

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring_all = (smem_address(raw_smem) + 1023u) & ~1023u, ring = ring_all + warp * kWarpRing;
  unsigned char* const parts_at = raw_smem + (ring_all - smem_address(raw_smem));      // [warp][row][column] f32, a ring apart
  const uint32_t barrier0 = smem_address(&full[warp][0]);
  if (lane == 0) {
    for (int st = 0; st < kKeyedStages; ++st) barrier_init(barrier0 + 8 * st, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if ((BITS == 8 ? p.pages : p.k_tokens) > 0) {      // (else there is no map)
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    }
  }
  if (!PARTS || !p.late) wait_for_earlier();
  if constexpr (SHARED || PARTS) let_later_start();      // (the joining kernel, or the next part's; see launch_overlapped)
  if (blockIdx.x == 0 && threadIdx.x == 0) p.status.begin();
  __syncwarp();
  // JOINS > 1: what a warp has of units that others have parts of too: of one that began before its share (0), of one that goes on behind it (1)
  struct Piece {
    int sequence, unit, first, last;                   // shares with parts of the unit
    bool there, begins, ends;
  };
  __shared__ Piece pieces[JOINS > 1 ? kKeyedWarps : 1][2];
  __shared__ float2 piece_stats[JOINS > 1 ? kKeyedWarps : 1][2][JOINS > 1 ? kRows : 1];
  unsigned char* const heads_at = parts_at + kKeyedWarps * kWarpRing;      // [warp][row][column] f32
  auto piece_at = [&](int of, int which) { return reinterpret_cast<float*>(which ? parts_at + of * kWarpRing : heads_at + of * (kRows * W * 4)); };
  if (JOINS > 1 && lane == 0) pieces[JOINS > 1 ? warp : 0][0].there = pieces[JOINS > 1 ? warp : 0][1].there = false;      // (by the lane that fills them in)
  uint32_t turn = 0;                                   // chunks this warp has waited for: the stage and the phase of the next
  const int quad = lane >> 2, corner = lane & 3;       // the instruction's row (or column) of eight, and the lane's place in it
  const int rows_each = p.group * p.q_tokens;          // of a sequence and key head: row = token * group + head in the group

  // SHARED: this warp's share of the range, [at, until)
  constexpr int kStep = SHARED ? 1 : WARPS;            // a warp takes every chunk of its share, or every WARPS-th of the unit
  const int share = static_cast<int>(blockIdx.x) * kKeyedWarps + warp;
  Place place = {0, 0};
  int at = 0, until = 1;
  Dealt dealt = {};
  if constexpr (SHARED) {
    dealt = deal<BITS, S::kKeys, PARTS>(p, blockIdx.x * kKeyedWarps, place);
    if (lane == 0) p.borders[share] = make_int4(0, 0, 0, 0);               // (the border behind this share; see below)
    if (share < dealt.shares) {
      at = dealt.start(share);
      until = dealt.start(share + 1);
    } else {
      until = 0;
    }
  }
  while (at < until) {
    // ---- one unit, or what of it is in the share: chunks [first_chunk, last_chunk) ----
    int batch, kv_head, tile, first_chunk = 0, last_chunk;
    bool whole = true, begins = true;
    int counted_length;
    ChunkList list;
    if constexpr (SHARED) {
      batch = place.sequence;
      counted_length = length_of<BITS, S::kKeys, PARTS>(p, batch);
      list = sequence_chunks<BITS, S::kKeys, PARTS>(p, batch, counted_length);
      const int cost = kUnitCost + max(list.count(), 1), units = p.kv_heads * p.row_tiles;
      const int inside = at - place.before;
      const int unit = inside / cost;
      tile = unit % p.row_tiles;
      kv_head = unit / p.row_tiles;
      const int from = inside - unit * cost, to = min(cost, from + (until - at));
      first_chunk = max(from - kUnitCost, 0);
      last_chunk = max(to - kUnitCost, 0);
      begins = first_chunk == 0;
      whole = begins && to == cost;
      const int unit_start = at - from;
      at += to - from;
      if (last_chunk > 0 && !whole && lane == 0) {         // which shares have parts of the unit
        const int first = dealt.holder(unit_start + kUnitCost), last = dealt.holder(unit_start + cost - 1);
        if constexpr (JOINS > 1) pieces[warp][begins ? 1 : 0] = {batch, unit, first, last, true, begins, to == cost};
        else if (to < cost) p.borders[share] = make_int4(batch, unit, first, last);      // the border behind this share cuts it
      }
      if (at - place.before >= units * cost) place = {batch + 1, place.before + units * cost};
      if (last_chunk == 0) continue;                     // a border just before its first chunk: it is the next share's
      last_chunk = min(last_chunk, list.count());
    } else {
      const long long unit = blockIdx.x;
      tile = static_cast<int>(unit % p.row_tiles);
      const long long head_index = unit / p.row_tiles;
      kv_head = static_cast<int>(head_index % p.kv_heads);
      batch = static_cast<int>(head_index / p.kv_heads);
      counted_length = length_of<BITS, S::kKeys, PARTS>(p, batch);
      at = until;
    }
    const int length = counted_length;
    const bool all_see = PARTS && batch < p.runs;        // a run, whose every row sees every key
    const int own = PARTS ? batch - p.runs : batch, rows = all_see ? p.each * rows_each : rows_each;
    const int row0 = tile * kRows;
    if constexpr (BITS == 8) {
      if ((SHARED ? lane : threadIdx.x) == 0 && !all_see && p.lengths[own] > length) report(p.status, kKeyedLength, own, p.lengths[own]);      // the table does not go that far
    }
    const int first_token = row0 / p.group, last_token = (min(row0 + kRows, rows) - 1) / p.group;
    const int low = all_see ? length - 1 : length - p.q_tokens + first_token, high = all_see ? length - 1 : length - p.q_tokens + last_token;
    if constexpr (!SHARED) {
      list = behind_prefix<S::kKeys, PARTS>(p, batch, length, chunks_of(low, max(high, -1), p.window, p.sinks, S::kKeys));
      last_chunk = list.count();
    }

    // ---- the warp's chunks ----
    if constexpr (!SHARED) first_chunk = warp;
    int mine = max(last_chunk - first_chunk + kStep - 1, 0) / kStep;
    long long table_row = own;
    if constexpr (PARTS) {
      if (all_see) {                                     // through the table row of the first sequence that is long enough; none is: nobody wants it
        int taker = 0x7fffffff;
        for (int i = lane; i < p.each; i += 32) {
          const int theirs = min(max(p.lengths[batch * p.each + i], 0), p.blocks << p.page_shift);
          if (takes_part(p, length, theirs)) {
            taker = i;
            break;
          }
        }
        taker = __reduce_min_sync(0xffffffffu, taker);
        if (taker == 0x7fffffff) mine = 0;
        else table_row = static_cast<long long>(batch) * p.each + taker;
      }
    }
    auto chunk_at = [&](int n) { return list.at(first_chunk + n * kStep); };
    // Lane l looks up the page of box l % boxes of chunk n + l / boxes, so one look-up serves the next 32 / boxes chunks. Pages that no row sees are
    // not looked at: a window may have left them behind, and the table may name anything there.
    const int boxes = ONE ? 1 : p.boxes, box_shift = ONE ? 31 : p.box_shift;
    const int ahead = ONE ? 32 : 32 / boxes, box_keys = ONE ? S::kKeys : 1 << box_shift;
    auto look_up = [&](int n) {
      if constexpr (BITS == 8) {
        n += ONE ? lane : lane / boxes;
        if (n >= mine) return -1;
        const int key = chunk_at(n) * S::kKeys + (ONE ? 0 : (lane % boxes) << box_shift);
        if (key > high || (key + box_keys - 1 <= low - p.window && key >= p.sinks)) return -1;
        const int at_block = key >> p.page_shift;
        const int page = p.table[table_row * p.table_stride + at_block];
        if (page >= 0 && page < p.pages) return page;
        report(p.status, kKeyedPage, static_cast<int>(table_row), at_block);
      }
      return -1;
    };
    int page_now = look_up(0), page_next = look_up(ahead);
    // The query: row `quad` of each eight, the elements that the lane's pieces of a key hold.
    constexpr int kWords = S::kPieceWidth / 2;                     // of a piece's query elements: 8 or 4
    uint32_t word[NT][S::kPieces][kWords];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = row0 + n * 8 + quad;
      const int inside = all_see ? row % rows_each : row, token = inside / p.group, head = kv_head * p.group + inside % p.group;
      const long long sequence = all_see ? static_cast<long long>(batch) * p.each + row / rows_each : own;
      const T* from = static_cast<const T*>(p.q) + sequence * p.q_strides[0] + head * p.q_strides[1] + token * p.q_strides[2];
#pragma unroll
      for (int j = 0; j < S::kPieces; ++j) {
        const int column = (4 * j + corner) * S::kPieceWidth;
#pragma unroll
        for (int w = 0; w < kWords; w += 4) {
          uint4 four = make_uint4(0, 0, 0, 0);
          if (row < rows && column + 2 * w < p.head_dim) four = *reinterpret_cast<const uint4*>(from + column + 2 * w);
          word[n][j][w] = four.x;
          word[n][j][w + 1] = four.y;
          word[n][j][w + 2] = four.z;
          word[n][j][w + 3] = four.w;
        }
      }
    }
    auto fill = [&](int n, int stage) {                  // chunk n of the warp into a stage that nobody reads any more
      const int key0 = chunk_at(n) * S::kKeys;
      const uint32_t to = ring + stage * kStageBytes, bar = barrier0 + 8 * stage;
      if constexpr (BITS == 8) {
        if (n > 0 && n % ahead == 0) {
          page_now = page_next;
          page_next = look_up(n + ahead);
        }
        const int inside = key0 & ((1 << p.page_shift) - 1);
        if constexpr (ONE) {
          const int page = __shfl_sync(0xffffffffu, page_now, n & 31);
          if (lane == 0) {
            staged_page[warp][stage][0] = page;
            barrier_expect_tx(bar, page >= 0 ? kStageBytes : 0);
            if (page >= 0) {
              const int row = ((page * p.kv_heads + kv_head) << p.page_shift) + inside;      // (below 2^31: keyed_maps)
              tma_load_rows(to, &map_k, bar, 0, row);
              tma_load_rows(to + kStageBytes / 2, &map_v, bar, 0, row);
            }
          }
          __syncwarp();                                  // every lane reads staged_page for the chunk's scales
        } else {
          const int page = __shfl_sync(0xffffffffu, page_now, (n % ahead) * boxes + lane % boxes);
          const bool loads = lane < boxes && page >= 0;
          const uint32_t box_bytes = static_cast<uint32_t>(S::kLine) << box_shift;
          const uint32_t bytes = 2u * box_bytes * __popc(__ballot_sync(0xffffffffu, loads));
          if (lane < boxes) staged_page[warp][stage][lane] = page;
          if (lane == 0) barrier_expect_tx(bar, bytes);
          __syncwarp();
          if (loads) {
            const int row = ((page * p.kv_heads + kv_head) << p.page_shift) + ((key0 + (lane << box_shift)) & ((1 << p.page_shift) - 1));
            tma_load_rows(to + lane * box_bytes, &map_k, bar, 0, row);
            tma_load_rows(to + kStageBytes / 2 + lane * box_bytes, &map_v, bar, 0, row);
          }
        }
      } else {
        if (lane == 0) {
          barrier_expect_tx(bar, kStageBytes);
#pragma unroll
          for (int l = 0; l < S::kLines; ++l) {
            tma_load_tokens(to + l * S::kBoxBytes, &map_k, bar, l * 64, key0, kv_head, batch);
            tma_load_tokens(to + kStageBytes / 2 + l * S::kBoxBytes, &map_v, bar, l * 64, key0, kv_head, batch);
          }
        }
      }
    };
    // The scales of the next chunk's pages (of its tile t in lane t, unless they are one page's) are asked for a step before they are used; 0: no
    // page.
    float k_scale_next = 0.f, v_scale_next = 0.f;
    auto ask_scales = [&](int stage) {
      if constexpr (BITS == 8) {
        if (ONE || lane < kTiles) {
          const int page = staged_page[warp][stage][ONE ? 0 : (lane * 16) >> box_shift];
          k_scale_next = v_scale_next = 0.f;
          if (page >= 0) {
            const int block = page * p.kv_heads + kv_head;
            k_scale_next = p.k_scales[block];
            v_scale_next = p.v_scales[block];
          }
        }
      }
    };
    for (int first = 0; first < min(mine, kKeyedStages); ++first) fill(first, (turn + first) % kKeyedStages);
    __syncwarp();
    if (mine > 0) ask_scales(turn % kKeyedStages);

    // ... as the matrix instructions take it: [piece][step of 16 elements][operand word]
    uint32_t query[NT][S::kPieces][32 / BITS][2];
    float row_scale[NT][2];                                        // of the lane's two columns: rows 2 corner and 2 corner + 1
    int position[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float back = p.scale_log2;
      if constexpr (BITS == 8) {
        float largest = 0.f;
#pragma unroll
        for (int j = 0; j < S::kPieces; ++j) {
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            const float2 pair = widen_pair<T>(word[n][j][w]);
            largest = fmaxf(largest, fmaxf(fabsf(pair.x), fabsf(pair.y)));
          }
        }
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        // a power of two that brings the row's largest element to [2^14, 2^15), 2^126 at most (from 2^-126 to 1); none for infinities
        int exponent = max(static_cast<int>(__float_as_uint(largest) >> 23) - 127, -112);
        if (exponent > 127) exponent = 14;
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - exponent) << 23);
        back *= __uint_as_float(static_cast<uint32_t>(127 - 14 + exponent) << 23);
#pragma unroll
        for (int j = 0; j < S::kPieces; ++j) {
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            const float2 pair = widen_pair<T>(word[n][j][w]);
            word[n][j][w] = round_pair<__half>(pair.x * up, pair.y * up);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < S::kPieces; ++j) {
#pragma unroll
        for (int w = 0; w < kWords; ++w) query[n][j][w / 2][w % 2] = word[n][j][w];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        row_scale[n][e] = __shfl_sync(0xffffffffu, back, (2 * corner + e) * 4);
        const int here = row0 + n * 8 + 2 * corner + e;
        position[n][e] = here < rows && !all_see ? length - p.q_tokens + here / p.group : high;
      }
    }

    float top[NT][2], sum[NT][2], result[NT][kSlices][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[n][e] = -INFINITY;
        sum[n][e] = 0.f;
      }
#pragma unroll
      for (int s = 0; s < kSlices; ++s) {
#pragma unroll
        for (int e = 0; e < 4; ++e) result[n][s][e] = 0.f;
      }
    }

    for (int step = 0; step < mine; ++step, ++turn) {
      const int key0 = chunk_at(step) * S::kKeys;
      const int stage = turn % kKeyedStages;
      // (by a vote: lanes that gave up leave the loop, and its shuffles, with all the others)
      if (!__all_sync(0xffffffffu, barrier_wait(barrier0 + 8 * stage, (turn / kKeyedStages) & 1, p.status, kWaitKeyed))) {
        // the result is lost (the status says so); the copies that are under way still have to land before the stages are used otherwise
        for (int m = step; m < min(step + kKeyedStages, mine); ++m, ++turn) {
          for (uint32_t spin = 0; spin < kSpinLimit && !barrier_try_wait(barrier0 + 8 * (turn % kKeyedStages), (turn / kKeyedStages) & 1); ++spin) {
          }
        }
        break;
      }
      const uint32_t k_at = ring + stage * kStageBytes, v_at = k_at + kStageBytes / 2;
      // Whether a key's page is there: of a chunk in one page all keys or none (from `stop` on), else by bits, bit t of the 16 keys from 16 t on. (Bits for
      // both: drafts 35.1 us, so 34.2.)
      constexpr uint32_t kAllTiles = (1u << kTiles) - 1;
      int stop = length;
      uint32_t tiles = kAllTiles;
      auto there = [&](int t, int key) { return ONE ? key < stop : (tiles >> t & 1) != 0; };
      constexpr int kScales = BITS == 8 && !ONE ? kTiles : 1;
      float k_scale[kScales], v_scale[kScales], v_scale_now = 0.f;
      k_scale[0] = k_scale_next;
      v_scale[0] = v_scale_next;
      if constexpr (BITS == 8) {
        if constexpr (ONE) {
          if (staged_page[warp][stage][0] < 0) stop = key0;
        } else {
#pragma unroll
          for (int t = kTiles - 1; t >= 0; --t) {
            k_scale[t] = __shfl_sync(0xffffffffu, k_scale_next, t);
            v_scale[t] = __shfl_sync(0xffffffffu, v_scale_next, t);
            if (staged_page[warp][stage][(t * 16) >> box_shift] < 0) tiles &= ~(1u << t);
          }
        }
        v_scale_now = v_scale_next;
        if (step + 1 < mine) ask_scales((turn + 1) % kKeyedStages);
      }

      // S^T: keys quad and quad + 8 of each tile by rows 2 corner and 2 corner + 1
      float score[kTiles][NT][4];
#pragma unroll
      for (int j = 0; j < S::kPieces; ++j) {
        uint4 near[kTiles], far[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          near[t] = load_shared_16(k_at + S::at(t * 16 + quad, (4 * j + corner) * 16));
          far[t] = load_shared_16(k_at + S::at(t * 16 + quad + 8, (4 * j + corner) * 16));
        }
#pragma unroll
        for (int w = 0; w < 32 / BITS; ++w) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const uint32_t x[4] = {near[t].x, near[t].y, near[t].z, near[t].w}, y[4] = {far[t].x, far[t].y, far[t].z, far[t].w};
            uint32_t a[4];
            if constexpr (BITS == 8) {
              a[0] = decode_low(x[w]);
              a[1] = decode_low(y[w]);
              a[2] = decode_high(x[w]);
              a[3] = decode_high(y[w]);
            } else {
              a[0] = x[2 * w];
              a[1] = y[2 * w];
              a[2] = x[2 * w + 1];
              a[3] = y[2 * w + 1];
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) multiply<M>(score[t][n], a, query[n][j][w][0], query[n][j][w][1], j == 0 && w == 0);
          }
        }
      }

      // A chunk whose keys every row sees needs no mask.
      const int last = key0 + S::kKeys - 1;
      const bool open = last <= low && (ONE ? last < stop : tiles == kAllTiles) && (key0 > high - p.window || last < p.sinks);
      auto sees = [&](int at, int t, int key) { return key <= at && there(t, key) && (key > at - p.window || key < p.sinks); };
      // Any reference point gives the same softmax: a row's moves only when a score lies more than 2^kSlack above it, which one vote tells.
      float most[NT][2];
      bool rises = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        most[n][0] = most[n][1] = -INFINITY;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          float2 by = make_float2(row_scale[n][0], row_scale[n][1]);
          if constexpr (BITS == 8) by = __fmul2_rn(by, make_float2(k_scale[t % kScales], k_scale[t % kScales]));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 scaled = __fmul2_rn(make_float2(score[t][n][2 * h], score[t][n][2 * h + 1]), by);
            score[t][n][2 * h] = scaled.x;
            score[t][n][2 * h + 1] = scaled.y;
            if (!open) {
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (!sees(position[n][e], t, key0 + t * 16 + quad + 8 * h)) score[t][n][2 * h + e] = -INFINITY;
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) most[n][e] = fmaxf(most[n][e], fmaxf(score[t][n][e], score[t][n][2 + e]));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) rises |= most[n][e] > top[n][e] + kSlack;      // (-inf + kSlack is -inf)
      }
      if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float now = most[n][e];
            now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 4));
            now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 8));
            now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 16));
            now = fmaxf(now, top[n][e]);
            const float factor = rescale(top[n][e], now);
            top[n][e] = now;
            sum[n][e] *= factor;
#pragma unroll
            for (int s = 0; s < kSlices; ++s) {
              result[n][s][e] *= factor;
              result[n][s][2 + e] *= factor;
            }
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 shift = make_float2(top[n][0] == -INFINITY ? 0.f : kLift<M> - top[n][0], top[n][1] == -INFINITY ? 0.f : kLift<M> - top[n][1]);
        float2 gained = make_float2(sum[n][0], sum[n][1]);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 moved = __fadd2_rn(make_float2(score[t][n][2 * h], score[t][n][2 * h + 1]), shift);
            score[t][n][2 * h] = exp2_ftz(moved.x);
            score[t][n][2 * h + 1] = exp2_ftz(moved.y);
            gained = __fadd2_rn(gained, make_float2(score[t][n][2 * h], score[t][n][2 * h + 1]));
          }
        }
        sum[n][0] = gained.x;
        sum[n][1] = gained.y;
      }

      // P^T in the layout of the second product: keys 2 corner ... of row quad
      uint32_t weight[kTiles][NT][2], rest[kTiles][kTwoOperands ? NT : 1][2];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float x = score[t][n][2 * h], y = score[t][n][2 * h + 1];
            const uint32_t rounded = round_pair<M>(x, y);
            weight[t][n][h] = transpose_tile(rounded);
            if constexpr (kTwoOperands) {
              const float2 wide = widen_pair<M>(rounded);
              rest[t][n][h] = transpose_tile(round_pair<M>(x - wide.x, y - wide.y));
            }
          }
        }
      }

      bool apart = false;                                // the rows' products have to be taken one query at a time
      if (!open) {
        // Values of keys that no row sees become zeros; where several queries see different keys, a probability of zero is mask enough if
        // all the values are numbers, and their scales.
        if constexpr (BITS == 8) apart = low != high && (kScales == 1 || lane < kTiles) && !(fabsf(v_scale_now) < INFINITY);
        constexpr int kUnits = W * BITS / 128;           // 16-byte units of a value
#pragma unroll 1
        for (int i = lane; i < S::kKeys * kUnits; i += 32) {
          const int inside = i / kUnits, key = key0 + inside;
          const uint32_t unit_at = v_at + S::at(inside, i % kUnits * 16);
          if (!(key <= high && there(inside / 16, key) && (key > low - p.window || key < p.sinks))) {
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(unit_at), "r"(0) : "memory");
          } else if (low != high) {
            const uint4 unit = load_shared_16(unit_at);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t four = c == 0 ? unit.x : c == 1 ? unit.y : c == 2 ? unit.z : unit.w;
              if constexpr (BITS == 8) {
                apart |= (((four & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
              } else {
                constexpr uint32_t kExponent = std::is_same_v<M, __nv_bfloat16> ? 0x7f80u : 0x7c00u;
                apart |= (four & kExponent) == kExponent || (four >> 16 & kExponent) == kExponent;
              }
            }
          }
        }
        apart = __any_sync(0xffffffffu, apart);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // TMA fills the stage again
        __syncwarp();
      }

      // One slice of V^T (16 head elements) for one tile of keys, as the instruction takes it, from the words of the lane's four keys.
      auto operand = [&](const uint32_t (&v)[4], int half, uint32_t (&a)[4]) {
        if constexpr (BITS == 8) {
          const uint32_t near = __byte_perm(v[0], v[1], half ? 0x7362 : 0x5140), far = __byte_perm(v[2], v[3], half ? 0x7362 : 0x5140);
          a[0] = decode_low(near);
          a[1] = decode_high(near);
          a[2] = decode_low(far);
          a[3] = decode_high(far);
        } else {
          a[0] = __byte_perm(v[0], v[1], 0x5410);
          a[1] = __byte_perm(v[0], v[1], 0x7632);
          a[2] = __byte_perm(v[2], v[3], 0x5410);
          a[3] = __byte_perm(v[2], v[3], 0x7632);
        }
      };
      auto key_of = [&](int t, int r) { return t * 16 + 2 * corner + (r & 1) + 8 * (r >> 1); };
      constexpr int kHalves = BITS == 8 ? 2 : 1;
      if (!apart) {
        // O^T += V^T P^T
        uint32_t value[kTiles][4][S::kValueWords];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (S::kValueWords == 2) {
              const uint2 two = load_shared_8(v_at + S::at(key_of(t, r), quad * 8));
              value[t][r][0] = two.x;
              value[t][r][1] = two.y;
            } else {
#pragma unroll
              for (int w = 0; w < S::kValueWords; w += 4) {
                const uint4 four = load_shared_16(v_at + S::at(key_of(t, r), ((w / 4) * 8 + quad) * 16));
                value[t][r][w] = four.x;
                value[t][r][w + 1] = four.y;
                value[t][r][w + 2] = four.z;
                value[t][r][w + 3] = four.w;
              }
            }
          }
        }
#pragma unroll
        for (int w = 0; w < S::kValueWords; ++w) {
#pragma unroll
          for (int half = 0; half < kHalves; ++half) {
            const int slice = kHalves * w + half;
            float d[NT][4];
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
              uint32_t a[4];
              const uint32_t v[4] = {value[t][0][w], value[t][1][w], value[t][2][w], value[t][3][w]};
              operand(v, half, a);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if constexpr (BITS == 16) {
                  multiply<M>(result[n][slice], a, weight[t][n][0], weight[t][n][1], false);
                  if constexpr (kTwoOperands) multiply<M>(result[n][slice], a, rest[t][n][0], rest[t][n][1], false);
                } else {
                  multiply<M>(d[n], a, weight[t][n][0], weight[t][n][1], kScales > 1 || t == 0);
                }
                if constexpr (kScales > 1) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) result[n][slice][e] = fmaf(d[n][e], v_scale[t], result[n][slice][e]);
                }
              }
            }
            if constexpr (BITS == 8 && kScales == 1) {
#pragma unroll
              for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                  const float2 sum2 = __ffma2_rn(make_float2(d[n][e], d[n][e + 1]), make_float2(v_scale[0], v_scale[0]), make_float2(result[n][slice][e], result[n][slice][e + 1]));
                  result[n][slice][e] = sum2.x;
                  result[n][slice][e + 1] = sum2.y;
                }
              }
            }
          }
        }
      } else {
        // (Rare, and written to be small.) The probabilities go where the chunk's keys were, and each query has a pass of its own over the tiles,
        // with the values it does not see as zeros; each row keeps what its own query's pass gives.
        uint32_t* const kept = reinterpret_cast<uint32_t*>(parts_at + warp * kWarpRing + stage * kStageBytes);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              kept[((t * NT + n) * 4 + h) * 32 + lane] = weight[t][n][h];
              if constexpr (kTwoOperands) kept[((t * NT + n) * 4 + 2 + h) * 32 + lane] = rest[t][n][h];
            }
          }
        }
#pragma unroll 1
        for (int at = low; at <= high; ++at) {
#pragma unroll 1
          for (int t = 0; t < kTiles; ++t) {
            float scale = v_scale[0];
            if constexpr (kScales > 1) scale = __shfl_sync(0xffffffffu, v_scale_now, t);
            const int tile0 = key0 + t * 16;
            if (tile0 > at || (tile0 + 15 <= at - p.window && tile0 >= p.sinks)) continue;      // nothing of the tile, its scale neither
#pragma unroll
            for (int w = 0; w < S::kValueWords; ++w) {
              uint32_t v[4];
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int column = S::kValueWords == 2 ? quad * 8 + w * 4 : ((w / 4) * 8 + quad) * 16 + w % 4 * 4;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[r]) : "r"(v_at + S::at(key_of(t, r), column)));
                if (!sees(at, t, key0 + key_of(t, r))) v[r] = 0;
              }
#pragma unroll
              for (int half = 0; half < kHalves; ++half) {
                uint32_t a[4];
                operand(v, half, a);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  const uint32_t* b = kept + (t * NT + n) * 4 * 32 + lane;
                  float d[4];
                  multiply<M>(d, a, b[0], b[32], true);
                  if constexpr (kTwoOperands) multiply<M>(d, a, b[64], b[96], false);
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    if (position[n][e & 1] == at) {
                      float& into = result[n][kHalves * w + half][e];
                      into = BITS == 8 ? fmaf(d[e], scale, into) : into + d[e];
                    }
                  }
                }
              }
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();                                      // the stage has been read
      if (step + kKeyedStages < mine) fill(step + kKeyedStages, stage);
    }

#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int offset = 4; offset < 32; offset *= 2) sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], offset);
      }
    }
    // A lane has, of its rows, runs of eight neighbouring elements.
    constexpr int kRuns = kSlices / 4;
    auto column_of = [&](int run) { return BITS == 8 ? quad * (W / 8) + 8 * run : run * 64 + quad * 8; };
    auto run_of = [&](int n, int e, int run, float (&value)[8]) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        value[2 * c] = result[n][4 * run + c][e];
        value[2 * c + 1] = result[n][4 * run + c][2 + e];
      }
    };
    if constexpr (SHARED) {
      const long long slot0 = (2LL * share + (begins ? 1 : 0)) * kRows;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = n * 8 + 2 * corner + e;
          if (row0 + row >= rows) continue;
          if (!whole && quad == 0) *(JOINS > 1 ? &piece_stats[JOINS > 1 ? warp : 0][begins ? 1 : 0][JOINS > 1 ? row : 0] : p.part_stats + slot0 + row) = make_float2(top[n][e], sum[n][e]);
#pragma unroll
          for (int run = 0; run < kRuns; ++run) {
            float value[8];
            run_of(n, e, run, value);
            const int column = column_of(run);
            if (column >= p.head_dim) continue;
            if (whole) {
              write_result<T, W, PARTS>(p, batch, kv_head, row0 + row, column, length, top[n][e], sum[n][e], value);
            } else {
              float4* to = reinterpret_cast<float4*>((JOINS > 1 ? piece_at(warp, begins ? 1 : 0) + row * W : p.parts + (slot0 + row) * W) + column);
              to[0] = make_float4(value[0], value[1], value[2], value[3]);
              to[1] = make_float4(value[4], value[5], value[6], value[7]);
            }
          }
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = n * 8 + 2 * corner + e;
          if (quad == 0) {
            part_top[warp][row] = top[n][e];
            part_sum[warp][row] = sum[n][e];
          }
#pragma unroll
          for (int run = 0; run < kRuns; ++run) {
            float value[8];
            run_of(n, e, run, value);
            float4* to = reinterpret_cast<float4*>(parts_at + warp * kWarpRing + (row * W + column_of(run)) * 4);
            to[0] = make_float4(value[0], value[1], value[2], value[3]);
            to[1] = make_float4(value[4], value[5], value[6], value[7]);
          }
        }
      }
      __syncthreads();
      for (int item = threadIdx.x; item < kRows * (W / 8); item += 32 * WARPS) {
        const int row = item / (W / 8), column = item % (W / 8) * 8;
        if (row0 + row >= rows || column >= p.head_dim) continue;
        float most = part_top[0][row];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) most = fmaxf(most, part_top[w][row]);
        float total = 0.f, value[8] = {};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float by = rescale(part_top[w][row], most);
          total += part_sum[w][row] * by;
#pragma unroll
          for (int c = 0; c < 8; ++c) value[c] += reinterpret_cast<const float*>(parts_at + w * kWarpRing)[row * W + column + c] * by;
        }
        write_result<T, W, PARTS>(p, batch, kv_head, row0 + row, column, length, most, total, value);
      }
    }
  }
  if constexpr (!SHARED && !PARTS) let_later_start();
  if constexpr (JOINS > 1) {
    // The pieces of a unit meet, in the order of the warps; what other CTAs have parts of too goes to memory, as the part of the first of its
    // warps.
    __syncthreads();
    for (int i = 0; i < 2 * kKeyedWarps;) {
      if (!pieces[i / 2][i % 2].there) {
        ++i;
        continue;
      }
      const Piece head = pieces[i / 2][i % 2];
      const int share0 = static_cast<int>(blockIdx.x) * kKeyedWarps + i / 2;
      int last = i;
      bool ends = head.ends;
      for (int next = i + 1; next < 2 * kKeyedWarps && !ends; ++next) {
        if (!pieces[next / 2][next % 2].there) continue;
        last = next;
        ends = pieces[next / 2][next % 2].ends;
      }
      if (!ends && threadIdx.x == 0)
        p.borders[blockIdx.x * kKeyedWarps + kKeyedWarps - 1] = make_int4(head.sequence, head.unit, head.first, head.last);
      const int tile = head.unit % p.row_tiles, kv_head = head.unit / p.row_tiles;
      const bool whole = head.begins && ends;
      const long long slot0 = (2LL * share0 + (head.begins ? 1 : 0)) * kRows;
#pragma unroll 1
      for (int item = threadIdx.x; item < kRows * (W / 8); item += kKeyedThreads) {
        const int row = item / (W / 8), column = item % (W / 8) * 8;
        if (tile * kRows + row >= (PARTS && head.sequence < p.runs ? p.each : 1) * rows_each || column >= p.head_dim) continue;
        float most = -INFINITY, total = 0.f, value[8] = {};
#pragma unroll 1
        for (int j = i; j <= last; ++j) {
          if (!pieces[j / 2][j % 2].there) continue;
          const float2 stats = piece_stats[j / 2][j % 2][row];
          const float4* from = reinterpret_cast<const float4*>(piece_at(j / 2, j % 2) + row * W + column);
          const float4 near = from[0], far = from[1];
          const float both = fmaxf(most, stats.x), mine = rescale(most, both), theirs = rescale(stats.x, both);
          const float x[8] = {near.x, near.y, near.z, near.w, far.x, far.y, far.z, far.w};
          most = both;
          total = total * mine + stats.y * theirs;
#pragma unroll
          for (int c = 0; c < 8; ++c) value[c] = value[c] * mine + x[c] * theirs;
        }
        if (whole) {
          write_result<T, W, PARTS>(p, head.sequence, kv_head, tile * kRows + row, column, length_of<BITS, S::kKeys, PARTS>(p, head.sequence), most, total, value);
        } else {
          float4* to = reinterpret_cast<float4*>(p.parts + (slot0 + row) * W + column);
          to[0] = make_float4(value[0], value[1], value[2], value[3]);
          to[1] = make_float4(value[4], value[5], value[6], value[7]);
          if (column == 0) p.part_stats[slot0 + row] = make_float2(most, total);
        }
      }
      i = last + 1;
    }
  }
  if (PARTS && p.late) wait_for_earlier();      // (what comes after this kernel comes after the one before it)
}

// SHARED: joins the parts of the units that a border between two shares (or two CTAs' shares: JOINS of them) cut. A CTA for each border; the CTAs
// of a unit's borders split its result, 64 elements of a row at a time: eight lanes of eight elements, by as many groups as there are parts, four
// groups in a warp or, of many parts, sixteen in the CTA.
template <typename T, int W, int NT, int JOINS, bool PARTS = false>
__global__ void __launch_bounds__(kKeyedThreads) keyed_join_kernel(const __grid_constant__ KeyedParams p) {
  constexpr int kRows = 8 * NT;
  __shared__ float2 warp_stats[kKeyedWarps][8];
  __shared__ float4 warp_value[kKeyedWarps][8][2];
  wait_for_earlier();
  const int share = static_cast<int>(blockIdx.x) * JOINS + JOINS - 1;         // the border lies behind it
  const int4 border = p.borders[share];
  const int batch = border.x, unit = border.y, first = border.z, last = border.w;
  const int borders = last / JOINS - first / JOINS, nth = share / JOINS - first / JOINS, parts = borders + 1;
  if (first == last || borders == 0) return;              // it lies between two units
  const int tile = unit % p.row_tiles, kv_head = unit / p.row_tiles;
  const int rows = min(kRows, (PARTS && batch < p.runs ? p.each : 1) * p.group * p.q_tokens - tile * kRows);
  const int length = PARTS ? 0 : p.lengths == nullptr ? p.k_tokens : min(max(p.lengths[batch], 0), p.blocks << p.page_shift);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool many = JOINS > 1 && parts > 16;              // (uniform in the CTA)
  constexpr int kAtOnce = NT == 1 ? 2 : 4;                // rows whose loads are under way together
  const int groups = many ? 16 : 4, group = many ? threadIdx.x >> 3 : lane >> 3;
  const int items = rows * (W / 64), mine0 = many ? nth : nth * kKeyedWarps + warp, stride = many ? borders : borders * kKeyedWarps;
  for (int item0 = mine0; item0 < items; item0 += kAtOnce * stride) {
    float most[kAtOnce], total[kAtOnce], value[kAtOnce][8];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      most[i] = -INFINITY;
      total[i] = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) value[i][c] = 0.f;
    }
#pragma unroll 2
    for (int of = group; of < parts; of += groups) {
      const int from = of == 0 ? first : (first / JOINS + of) * JOINS;
      float2 stats[kAtOnce];
      float4 part[kAtOnce][2];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int item = item0 + i * stride, column = item % (W / 64) * 64 + lane % 8 * 8;
        stats[i] = make_float2(-INFINITY, 0.f);
        part[i][0] = part[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (item < items) {
          const long long slot = (2LL * from + (of == 0 ? 1 : 0)) * kRows + item / (W / 64);
          stats[i] = p.part_stats[slot];
          if (column < p.head_dim) {
            const float4* at = reinterpret_cast<const float4*>(p.parts + slot * W + column);
            part[i][0] = at[0];
            part[i][1] = at[1];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const float both = fmaxf(most[i], stats[i].x);
        const float mine = rescale(most[i], both), theirs = rescale(stats[i].x, both);
        const float x[8] = {part[i][0].x, part[i][0].y, part[i][0].z, part[i][0].w, part[i][1].x, part[i][1].y, part[i][1].z, part[i][1].w};
        most[i] = both;
        total[i] = total[i] * mine + stats[i].y * theirs;
#pragma unroll
        for (int c = 0; c < 8; ++c) value[i][c] = value[i][c] * mine + x[c] * theirs;
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int item = item0 + i * stride, column = item % (W / 64) * 64 + lane % 8 * 8;
#pragma unroll
      for (int offset = 8; offset < 32; offset *= 2) {
        const float other = __shfl_xor_sync(0xffffffffu, most[i], offset), both = fmaxf(most[i], other);
        const float mine = rescale(most[i], both), theirs = rescale(other, both);
        most[i] = both;
        total[i] = total[i] * mine + __shfl_xor_sync(0xffffffffu, total[i], offset) * theirs;
#pragma unroll
        for (int c = 0; c < 8; ++c) value[i][c] = value[i][c] * mine + __shfl_xor_sync(0xffffffffu, value[i][c], offset) * theirs;
      }
      if (many) {
        __syncthreads();
        if (lane < 8) {
          warp_stats[warp][lane] = make_float2(most[i], total[i]);
          warp_value[warp][lane][0] = make_float4(value[i][0], value[i][1], value[i][2], value[i][3]);
          warp_value[warp][lane][1] = make_float4(value[i][4], value[i][5], value[i][6], value[i][7]);
        }
        __syncthreads();
        if (warp == 0 && lane < 8) {
#pragma unroll
          for (int w = 1; w < kKeyedWarps; ++w) {
            const float2 stats = warp_stats[w][lane];
            const float4 near = warp_value[w][lane][0], far = warp_value[w][lane][1];
            const float both = fmaxf(most[i], stats.x), mine = rescale(most[i], both), theirs = rescale(stats.x, both);
            const float x[8] = {near.x, near.y, near.z, near.w, far.x, far.y, far.z, far.w};
            most[i] = both;
            total[i] = total[i] * mine + stats.y * theirs;
#pragma unroll
            for (int c = 0; c < 8; ++c) value[i][c] = value[i][c] * mine + x[c] * theirs;
          }
        }
      }
      if (item < items && lane < 8 && (!many || warp == 0) && column < p.head_dim)
        write_result<T, W, PARTS>(p, batch, kv_head, tile * kRows + item / (W / 64), column, length, most[i], total[i], value[i]);
    }
  }
}

// Warps for which an SM of a B200 has registers: of the kernels below, those of 168 a thread or fewer as compiled leave room for three in each quarter of it, of
// up to 255 for two.
constexpr int register_warps(int bits, int w, int nt, int joins) { return w == 64 && (nt == 1 || (bits == 16 && joins == 0)) ? 12 : 8; }

// How many CTAs of a kernel run at once on `device`, asked once for each; without a GPU, on a B200, whose SMs have shared memory of 228 KB and registers for
// SM_WARPS of its warps.
template <auto kKernel, int WARPS, int SM_WARPS>
int resident(int32_t device, size_t smem) {
  static std::mutex mutex;
  static int known[64] = {};
  const int by_registers = SM_WARPS / WARPS, by_memory = static_cast<int>(228 * 1024 / (smem + 1024)), assumed = by_registers < by_memory ? by_registers : by_memory;
  if (device < 0 || device >= 64) return assumed * 148;
  std::lock_guard<std::mutex> lock(mutex);
  if (known[device] == 0) {
    int per_sm = 0;
    DeviceScope device_scope(device);
    if (device_scope.status() != TQ_OK) return assumed * 148;      // (a plan without a GPU)
    if (cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kKernel, 32 * WARPS, smem) != cudaSuccess || per_sm <= 0) {
      cudaGetLastError();
      per_sm = assumed;
    }
    known[device] = per_sm * sm_count(device);
  }
  return known[device];
}

// The most chunks that some of `tokens` neighbouring queries can see: all keys, or what a window and the sinks leave.
long long most_chunks(const KeyedParams& p, long long tokens, long long keys, int chunk) {
  const long long all = (keys + chunk - 1) / chunk;
  const long long seen = (p.sinks + chunk - 1LL) / chunk + (p.window + tokens + chunk - 2LL) / chunk + 1;
  return all < seen ? all : seen;
}

// Whether a unit is a CTA's, of 2, 4 or 8 warps, or the chunks of all units are dealt out, is decided by expected time (us, B200). Dealing out costs
// the finding of places at the start and the join at the end, a CTA a unit the wait for the longest, and for the next wave. A step (a chunk a
// warp) takes kStepTime at least, and at most what memory makes of the chunks under way. Always four warps or dealt out, and by this rule: 12 heads
// of 64, 1500 keys 14.5, 8.5; 64 x 12 heads, 1000 keys 29.0, 22.9; 48 x 32/8 heads of 128, 300 keys 16.5, 12.4, 1000 keys 28.8, 25.1, 1500 keys
// 36.8, 36.8; four queries of the same under a window of 1024 39.4, 36.0. (Since launches overlap, each is 1 to 2 us less.)
constexpr double kStepTime[2] = {0.9, 1.3};              // of 8 rows, of 16
constexpr double kBytesPerMicrosecond[2] = {6.2e6, 4.4e6};
constexpr double kWholeTime = 5.5, kWaveTime = 4.0, kDealtTime = 13.0;
constexpr int kMostSteps = 20;                           // beyond, equal shares are worth more than what they cost

// From as many parts a unit on, the warps of a CTA join theirs before they go to memory.
constexpr int kManyParts = 8;

struct KeyedPlan {
  int nt, row_tiles, shares, joins, warps;      // shares 0: a CTA of `warps` a unit
  size_t bytes;
  double time;                                  // expected, us
};

template <int BITS, int W>
KeyedPlan plan_shape(const KeyedParams& p, long long keys, int32_t device) {
  KeyedPlan plan = {};
  const int rows = (p.runs > 0 ? p.each : 1) * p.group * p.q_tokens;
  plan.nt = rows <= 8 ? 1 : 2;
  plan.row_tiles = (rows + 8 * plan.nt - 1) / (8 * plan.nt);
  // a tile's own, and of all the sequence's queries together, which is what every tile walks where chunks are dealt out
  const long long tokens = (8 * plan.nt + p.group - 2) / p.group + 1;
  long long own = most_chunks(p, tokens < p.q_tokens ? tokens : p.q_tokens, keys, KeyedShape<BITS, W>::kKeys);
  const long long chunks = most_chunks(p, p.q_tokens, keys, KeyedShape<BITS, W>::kKeys);
  const long long units = static_cast<long long>(p.batch) * p.kv_heads * plan.row_tiles;
  const long long average = p.typical > 0 && p.typical < keys ? most_chunks(p, p.q_tokens, p.typical, KeyedShape<BITS, W>::kKeys) : chunks;
  if (p.runs == 0 && average < own) own = average;      // sequences without the keys of their runs: none of them is taken to be long
  const int sixteen = plan.nt - 1;
  auto most_of = [&](auto joins, auto warps) {
    constexpr int kJoins = decltype(joins)::value, kWarps = decltype(warps)::value;
    return plan.nt == 1 ? resident<keyed_attention_kernel<__nv_bfloat16, BITS, W, 1, kJoins, true, kWarps>, kWarps, register_warps(BITS, W, 1, kJoins)>(
                              device, keyed_smem(false, W, 1, kWarps))
                        : resident<keyed_attention_kernel<__nv_bfloat16, BITS, W, 2, kJoins, true, kWarps>, kWarps, register_warps(BITS, W, 2, kJoins)>(
                              device, keyed_smem(false, W, 2, kWarps));
  };
  auto whole_time = [&](auto warps) {
    constexpr int kWarps = decltype(warps)::value;
    const double most = most_of(std::integral_constant<int, 0>{}, warps), waves = units <= most ? 1.0 : std::ceil(units / most);
    const double memory = (units < most ? units : most) * kWarps * kStageBytes / kBytesPerMicrosecond[sixteen];
    const double steps = static_cast<double>((own + kWarps - 1) / kWarps), step = memory > kStepTime[sixteen] ? memory : kStepTime[sixteen];
    if (average < own) return kWholeTime + steps * step + (waves - 1) * (std::ceil(static_cast<double>(average) / kWarps) * step + kWaveTime);
    return kWholeTime + waves * steps * step + (waves - 1) * kWaveTime;
  };
  const double times[3] = {whole_time(std::integral_constant<int, 2>{}), whole_time(std::integral_constant<int, 4>{}), whole_time(std::integral_constant<int, 8>{})};
  int best = 0;
  for (int i = 1; i < 3; ++i)
    if (times[i] < times[best]) best = i;
  plan.warps = 2 << best;
  const double dealt = kDealtTime + static_cast<double>(average) * units * kStageBytes / kBytesPerMicrosecond[sixteen];
  plan.time = times[best] < dealt ? times[best] : dealt;
  const bool whole = (own + plan.warps - 1) / plan.warps <= kMostSteps && times[best] <= dealt;
  if (!whole && chunks <= 2 * own && (chunks + unit_cost(KeyedShape<BITS, W>::kKeys)) * units < (1LL << 31)) {
    const int most = most_of(std::integral_constant<int, 1>{}, std::integral_constant<int, kKeyedWarps>{});
    plan.shares = kKeyedWarps * static_cast<int>(chunks * units / kKeyedWarps < most ? (chunks * units + kKeyedWarps - 1) / kKeyedWarps : most);
    plan.joins = plan.shares >= kManyParts * units ? kKeyedWarps : 1;
    plan.bytes = plan.shares * (sizeof(int4) + 2ull * 8 * plan.nt * (W + 2) * sizeof(float));
  }
  return plan;
}

KeyedPlan plan_keyed(bool paged, const KeyedParams& p, long long keys, int32_t device) {
  if (paged) return p.head_dim <= 64 ? plan_shape<8, 64>(p, keys, device) : plan_shape<8, 128>(p, keys, device);
  return p.head_dim <= 64 ? plan_shape<16, 64>(p, keys, device) : plan_shape<16, 128>(p, keys, device);
}

tq_status keyed_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* pointer, const cuuint64_t* dims, const cuuint64_t* byte_strides,
                    const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  EncodeTiled encode = encode_tiled();
  TQ_REQUIRE(encode != nullptr, TQ_EXTERNAL, "the CUDA driver does not provide cuTensorMapEncodeTiled");
  const cuuint32_t element_strides[4] = {1, 1, 1, 1};
  const CUresult result = encode(map, type, rank, const_cast<void*>(pointer), dims, byte_strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TQ_REQUIRE(result == CUDA_SUCCESS, TQ_UNSUPPORTED, "this operand layout cannot be described to TMA (driver code %d)", static_cast<int>(result));
  return TQ_OK;
}

// Maps of the keys and of the values: rows of a page and head, or [batch, head, token] through the caller's strides. What a row has less than W
// elements, and rows behind the last token, arrive as zeros.
template <typename T, int BITS, int W>
tq_status keyed_maps(CUtensorMap* maps, KeyedParams& p) {
  using S = KeyedShape<BITS, W>;
  const CUtensorMapSwizzle swizzle = S::kLine == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  const void* operands[2] = {p.k, p.v};
  for (int i = 0; i < 2; ++i) {
    if constexpr (BITS == 8) {
      const int box_rows = 1 << p.page_shift < S::kKeys ? 1 << p.page_shift : S::kKeys;
      p.boxes = S::kKeys / box_rows;
      p.box_shift = 31 - __builtin_clz(static_cast<unsigned>(box_rows));
      if (p.pages == 0) continue;
      const cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.head_dim), (static_cast<cuuint64_t>(p.pages) * p.kv_heads) << p.page_shift};
      const cuuint64_t byte_strides[1] = {static_cast<cuuint64_t>(p.head_dim)};
      const cuuint32_t box[2] = {static_cast<cuuint32_t>(W), static_cast<cuuint32_t>(box_rows)};
      TQ_REQUIRE(dims[1] < (1ull << 31), TQ_UNSUPPORTED, "a pool of more than 2^31 tokens and heads");
      if (tq_status s = keyed_map(&maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, operands[i], dims, byte_strides, box, swizzle)) return s;
    } else {
      if (p.k_tokens == 0) continue;
      const long long* strides = i == 0 ? p.k_strides : p.v_strides;
      const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p.head_dim), static_cast<cuuint64_t>(p.k_tokens), static_cast<cuuint64_t>(p.kv_heads),
                                  static_cast<cuuint64_t>(p.batch)};
      // an axis of extent 1 never moves, so its stride only has to be legal
      const cuuint64_t byte_strides[3] = {static_cast<cuuint64_t>(p.k_tokens > 1 ? strides[2] : p.head_dim) * 2,
                                          static_cast<cuuint64_t>(p.kv_heads > 1 ? strides[1] : p.head_dim) * 2,
                                          static_cast<cuuint64_t>(p.batch > 1 ? strides[0] : p.head_dim) * 2};
      const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(S::kKeys), 1, 1};
      const CUtensorMapDataType type = std::is_same_v<T, __nv_bfloat16> ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
      if (tq_status s = keyed_map(&maps[i], type, 4, operands[i], dims, byte_strides, box, swizzle)) return s;
    }
  }
  return TQ_OK;
}

template <typename T, int BITS, int W, int NT, bool PARTS>
tq_status launch_keyed(KeyedParams& p, int warps, cudaStream_t stream) {
  CUtensorMap maps[2] = {};
  if (tq_status s = keyed_maps<T, BITS, W>(maps, p)) return s;
  auto start = [&](auto kernel, int each, long long ctas) -> tq_status {
    const size_t smem = keyed_smem(p.joins > 1, W, NT, each);
    TQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    TQ_CUDA(launch_overlapped(kernel, dim3(static_cast<unsigned>(ctas)), 32 * each, smem, stream, maps[0], maps[1], p));
    return check_launch("keyed_attention_kernel");
  };
  auto start_boxes = [&](auto joins, auto each, long long ctas) {
    constexpr int kJoins = decltype(joins)::value, kWarps = decltype(each)::value;
    if constexpr (BITS == 8) {
      if (p.boxes > 1) return start(keyed_attention_kernel<T, BITS, W, NT, kJoins, false, kWarps, PARTS>, kWarps, ctas);
    }
    return start(keyed_attention_kernel<T, BITS, W, NT, kJoins, true, kWarps, PARTS>, kWarps, ctas);
  };
  constexpr std::integral_constant<int, 0> kWhole{};
  constexpr std::integral_constant<int, kKeyedWarps> kFour{};
  if (p.shares == 0) {
    const long long units = static_cast<long long>(p.batch) * p.kv_heads * p.row_tiles;
    TQ_REQUIRE(units < (1LL << 31), TQ_UNSUPPORTED, "too many heads and rows for one launch");
    return warps == 2 ? start_boxes(kWhole, std::integral_constant<int, 2>{}, units) : warps == 4 ? start_boxes(kWhole, kFour, units)
                                                                                              : start_boxes(kWhole, std::integral_constant<int, 8>{}, units);
  }
  const bool gathers = p.joins > 1;
  // both launches, one after the other: recorded ones may share their scratch on a stream (of parts, prefix.cu holds it)
  const auto held = hold_scratch(PARTS ? nullptr : p.borders);
  if (tq_status s = gathers ? start_boxes(kFour, kFour, p.shares / kKeyedWarps) : start_boxes(std::integral_constant<int, 1>{}, kFour, p.shares / kKeyedWarps)) return s;
  const dim3 borders(static_cast<unsigned>((p.shares - 1) / p.joins + (p.joins == 1 ? 0 : 1)));
  TQ_CUDA(gathers ? launch_overlapped(keyed_join_kernel<T, W, NT, kKeyedWarps, PARTS>, borders, kKeyedThreads, 0, stream, p)
                  : launch_overlapped(keyed_join_kernel<T, W, NT, 1, PARTS>, borders, kKeyedThreads, 0, stream, p));
  return check_launch("keyed_join_kernel");
}

template <typename T, int BITS, bool PARTS = false>
tq_status launch_keyed_width(KeyedParams& p, const KeyedPlan& plan, cudaStream_t stream) {
  if (p.head_dim <= 64)
    return plan.nt == 1 ? launch_keyed<T, BITS, 64, 1, PARTS>(p, plan.warps, stream) : launch_keyed<T, BITS, 64, 2, PARTS>(p, plan.warps, stream);
  return plan.nt == 1 ? launch_keyed<T, BITS, 128, 1, PARTS>(p, plan.warps, stream) : launch_keyed<T, BITS, 128, 2, PARTS>(p, plan.warps, stream);
}

}  // namespace

size_t keyed_workspace(bool paged, const KeyedParams& p, long long keys, int32_t device) { return plan_keyed(paged, p, keys, device).bytes; }

double keyed_time(bool paged, const KeyedParams& p, long long keys, int32_t device) { return plan_keyed(paged, p, keys, device).time; }

tq_status keyed_attention(tq_dtype dtype, bool paged, KeyedParams& p, long long keys, void* workspace, size_t workspace_bytes, int32_t device,
                          cudaStream_t stream) {
  const KeyedPlan plan = plan_keyed(paged, p, keys, device);
  TQ_REQUIRE(plan.bytes == 0 || (workspace != nullptr && workspace_bytes >= plan.bytes && aligned_to(workspace, 16)), TQ_INVALID_ARGUMENT,
             "this attention needs %zu bytes of workspace, 16-byte aligned, and was given %zu", plan.bytes, workspace_bytes);
  p.row_tiles = plan.row_tiles;
  p.shares = plan.shares;
  p.joins = plan.joins;
  const size_t slots = 2ull * plan.shares * 8 * plan.nt;
  p.borders = static_cast<int4*>(workspace);
  p.part_stats = reinterpret_cast<float2*>(p.borders + plan.shares);
  p.parts = reinterpret_cast<float*>(p.part_stats + slots);
  if (p.shared != nullptr) return dtype == TQ_BF16 ? launch_keyed_width<__nv_bfloat16, 8, true>(p, plan, stream) : launch_keyed_width<__half, 8, true>(p, plan, stream);
  if (dtype == TQ_BF16) return paged ? launch_keyed_width<__nv_bfloat16, 8>(p, plan, stream) : launch_keyed_width<__nv_bfloat16, 16>(p, plan, stream);
  return paged ? launch_keyed_width<__half, 8>(p, plan, stream) : launch_keyed_width<__half, 16>(p, plan, stream);
}

}  // namespace tq
