// The paged cache in 8 bits, for sm_100a: what writes new tokens into it and what copies its pages. (keyed.cu reads it.)
//
// Writing. A team of threads takes what one page and head gets of a sequence's new tokens:
//   s = the smallest power of two >= max |x| / 448, at least 2^-126 and at least what the page's earlier tokens need
//   code = e4m3(x / s), to nearest even
// e4m3 is a floating format, so a power of two costs it no precision, x / s is exact, and an earlier code brought to a larger scale only steps
// down in exponent: exact again, except for what falls under its smallest normal. The tokens are read once, kept in registers between the maximum
// and the encoding. Bound: HBM (2 bytes read and 1 written an element: 402 MB in 64.5 us, 6.2 TB/s); for one new token a sequence, the host (4 us;
// from a graph the latency of start, table entry, scale and token, one after another: 2.4). Divisions by the vectors of a token in the addresses had it at
// 94 us and bound by instructions; the next head's tokens loaded ahead took the registers of half the CTAs and gained nothing.
//
// Copying. Source and target pages are given by the host, which is where a cache's pages are handed out; they travel to the kernel as its
// argument, so nothing is uploaded before it. Bound: HBM (each byte read and written once: 551 MB in 85 us, 6.5 TB/s). Small pages of several
// layers are one CTA's: scales with a CTA for each layer, and two launches of 384 pairs, made that 96.
//
// Advancing. A step of beam search as the books see it, without the host: rows of the table go on from other rows, pages count how many rows have them,
// last pages that several rows would write into are copied, new pages are the lowest free ones. One CTA, or a cluster of sixteen (eight where there is no
// room for it), makes the new table and counts (what its CTAs tell each other goes through memory between cluster barriers); a second kernel copies the
// pages that it names. Bound: the latency of those barriers and of dependent reads, and the copied pages' bytes.
#include <cmath>
#include <mutex>
#include <new>
#include <type_traits>
#include <vector>

#include "common.h"
#include "keyed.h"

namespace tq {
namespace {

constexpr int kStoreThreads = 128;

struct StoreParams {
  const void* x[2];                // keys, values
  uint8_t* codes[2];
  float* scales[2];
  long long strides[2][3];         // batch, head, token, in elements
  const int32_t *table, *starts, *counts;
  long long table_stride;
  int blocks, page_shift, pages;
  int batch, kv_heads, tokens, head_dim;
  int touched;                     // pages that `tokens` tokens touch at most
  int each, runs;                  // of the 2 * kv_heads a page has, how many a team takes, and how many teams that makes
  WaitStatus status;
};

template <typename T>
__device__ __forceinline__ float2 pair_of(uint32_t word) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    return make_float2(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&word));
  }
}

// The larger of two magnitudes, of those that are finite, as bits (16-bit floats order like integers).
template <typename T>
__device__ __forceinline__ uint32_t larger(uint32_t most, uint32_t word) {
  constexpr uint32_t kInfinity = std::is_same_v<T, __nv_bfloat16> ? 0x7f80u : 0x7c00u;
  const uint32_t low = word & 0x7fffu, high = (word >> 16) & 0x7fffu;
  if (low < kInfinity) most = max(most, low);
  if (high < kInfinity) most = max(most, high);
  return most;
}

// Four floats as e4m3, the first in the low byte. Beyond 448 (which the scale rules out) it saturates; NaN stays NaN.
__device__ __forceinline__ uint32_t encode(float a, float b, float c, float d) {
  uint32_t word;
  asm("{\n\t.reg .b16 low, high;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 low, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 high, %4, %3;\n\t"
      "mov.b32 %0, {low, high};\n\t}"
      : "=r"(word)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return word;
}

// The larger magnitudes of two pairs; a NaN is passed over.
template <typename T>
__device__ __forceinline__ uint32_t larger_pair(uint32_t most, uint32_t word) {
  word &= 0x7fff7fffu;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) asm("max.bf16x2 %0, %0, %1;" : "+r"(most) : "r"(word));
  else asm("max.f16x2 %0, %0, %1;" : "+r"(most) : "r"(word));
  return most;
}

// x / s for a power of two s, NaN where x is not finite.
__device__ __forceinline__ float scaled(float x, float inverse) { return fmaf(x, inverse, x - x); }

// Eight elements over s. FINITE: there is no infinity among them.
template <typename T, bool FINITE>
__device__ __forceinline__ uint2 encode_vector(uint4 word, float inverse) {
  const float2 a = pair_of<T>(word.x), b = pair_of<T>(word.y), c = pair_of<T>(word.z), d = pair_of<T>(word.w);
  if constexpr (FINITE) {
    const float2 by = make_float2(inverse, inverse);
    const float2 e = __fmul2_rn(a, by), f = __fmul2_rn(b, by), g = __fmul2_rn(c, by), h = __fmul2_rn(d, by);
    return make_uint2(encode(e.x, e.y, f.x, f.y), encode(g.x, g.y, h.x, h.y));
  }
  return make_uint2(encode(scaled(a.x, inverse), scaled(a.y, inverse), scaled(b.x, inverse), scaled(b.y, inverse)),
                    encode(scaled(c.x, inverse), scaled(c.y, inverse), scaled(d.x, inverse), scaled(d.y, inverse)));
}

__device__ __forceinline__ uint32_t encode_again(uint32_t codes, float ratio) {
  float2 pair[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t wide;
    asm("{\n\t.reg .b16 pair;\n\tcvt.u16.u32 pair, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, pair;\n\t}" : "=r"(wide) : "r"(codes >> (16 * h)));
    pair[h] = __half22float2(*reinterpret_cast<const __half2*>(&wide));
  }
  return encode(scaled(pair[0].x, ratio), scaled(pair[0].y, ratio), scaled(pair[1].x, ratio), scaled(pair[1].y, ratio));
}

// TEAM threads (half a warp, a warp, or all) take some heads of the keys and values of one page, one after another.
template <typename T, int TEAM, int HELD>
__global__ void __launch_bounds__(kStoreThreads, TEAM == kStoreThreads ? (HELD == 8 ? 8 : 12) : HELD == 8 ? 7 : 10)
cache_store_kernel(const __grid_constant__ StoreParams p) {
  constexpr int kHeld = HELD;              // vectors of 8 elements a thread keeps: 8 are a page of 64 tokens of 128 for 128 threads
  __shared__ uint32_t warp_most[3][kStoreThreads / 32];
  wait_for_earlier();
  let_later_start();
  const int thread = threadIdx.x % TEAM;
  const uint32_t team = TEAM == 16 ? 0xffffu << (threadIdx.x & 16) : 0xffffffffu;      // of this warp
  long long item = static_cast<long long>(blockIdx.x) * (kStoreThreads / TEAM) + threadIdx.x / TEAM;
  if (item >= static_cast<long long>(p.batch) * p.touched * p.runs) return;      // whole teams
  const int run = static_cast<int>(item % p.runs);
  item /= p.runs;
  const int nth = static_cast<int>(item % p.touched), sequence = static_cast<int>(item / p.touched);

  const int start = p.starts[sequence];
  const int count = p.counts == nullptr ? p.tokens : min(max(p.counts[sequence], 0), p.tokens);
  if (start < 0) return;
  const long long block = (start >> p.page_shift) + nth;
  const long long first_position = max(block << p.page_shift, static_cast<long long>(start));       // of the tokens that go here
  const long long last_position = min((block + 1) << p.page_shift, static_cast<long long>(start) + count);
  if (first_position >= last_position) return;
  if (block >= p.blocks) {
    if (thread == 0) report(p.status, kKeyedLength, sequence, start);
    return;
  }
  const int page = p.table[sequence * p.table_stride + block];
  const int held_tokens = static_cast<int>(first_position - (block << p.page_shift));      // earlier ones, in this page
  const int vectors = p.head_dim / 8;
  const int work = static_cast<int>(last_position - first_position) * vectors;
  const int first = run * p.each, last = min(first + p.each, 2 * p.kv_heads);       // the keys' heads, then the values'

  auto source_of = [&](int n) {
    const int which = n >= p.kv_heads ? 1 : 0, head = n - which * p.kv_heads;
    return static_cast<const T*>(p.x[which]) + sequence * p.strides[which][0] + head * p.strides[which][1] + (first_position - start) * p.strides[which][2];
  };
  // A thread's vectors are every TEAM-th of the page's: from the place of one to the next without a division.
  const int token0 = thread / vectors, column0 = thread % vectors, token_step = TEAM / vectors, column_step = TEAM % vectors;
  auto each_vector = [&](const T* from, long long token_stride, auto visit) {      // visit(number, whether it is there, where)
    const T* at = from + token0 * token_stride + column0 * 8;
    int column = column0, i = thread;
    const long long step = token_step * token_stride + column_step * 8, wrap = token_stride - vectors * 8;
    auto go_on = [&] {
      column += column_step;
      at += step;
      if (column >= vectors) {
        column -= vectors;
        at += wrap;
      }
      i += TEAM;
    };
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      visit(h, i, at);
      go_on();
    }
#pragma unroll 1
    for (; i < work; go_on()) visit(kHeld, i, at);
  };
  if (page < 0 || page >= p.pages) {
    if (thread == 0) report(p.status, kKeyedPage, sequence, static_cast<int>(block));
    return;
  }
  for (int n = first; n < last; ++n) {
    const int which = n >= p.kv_heads ? 1 : 0;
    const long long slot = static_cast<long long>(page) * p.kv_heads + (n - which * p.kv_heads);
    uint8_t* const page_at = p.codes[which] + (slot << p.page_shift) * p.head_dim;
    uint2* const to = reinterpret_cast<uint2*>(page_at + held_tokens * p.head_dim);
    float* const scale_at = p.scales[which] + slot;
    float old = 0.f;
    if (held_tokens > 0) old = *scale_at;  // (every thread reads it before the team meets, and one writes it after)
    const T* const from = source_of(n);
    const long long token_stride = p.strides[which][2];
    uint4 kept[kHeld];
    // The team's maximum by `step`, which takes a pair of elements into a pair of maxima; `loads`: the first vectors are not in registers yet.
    auto team_most = [&](auto step, int turn, auto loads) {
      uint32_t pair = 0;
      auto take = [&](uint4 word) { pair = step(step(step(step(pair, word.x), word.y), word.z), word.w); };
      each_vector(from, token_stride, [&](int h, int i, const T* at) {
        if (h == kHeld) take(*reinterpret_cast<const uint4*>(at));
        else if (decltype(loads)::value) kept[h] = i < work ? *reinterpret_cast<const uint4*>(at) : make_uint4(0, 0, 0, 0);
      });
#pragma unroll
      for (int h = 0; h < kHeld; ++h) take(kept[h]);
      uint32_t most = __reduce_max_sync(team, max(pair & 0xffffu, pair >> 16));      // (magnitudes order like integers)
      if constexpr (TEAM > 32) {           // (places in turn: the next maxima do not overtake these)
        if (threadIdx.x % 32 == 0) warp_most[turn][threadIdx.x / 32] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < TEAM / 32; ++w) most = max(most, warp_most[turn][w]);
      }
      return most;
    };
    constexpr uint32_t kInfinity = std::is_same_v<T, __nv_bfloat16> ? 0x7f80u : 0x7c00u;
    uint32_t most = team_most([](uint32_t m, uint32_t w) { return larger_pair<T>(m, w); }, n & 1, std::true_type{});
    const bool finite = most < kInfinity;  // (the same for the team)
    if (!finite) most = team_most([](uint32_t m, uint32_t w) { return larger<T>(m, w); }, 2, std::false_type{});
    // the power of two: amax = m 2^e needs 2^(e - 8) where m <= 1.75 = 448 / 2^8, else twice that
    const float largest = pair_of<T>(most).x;
    const uint32_t bits = __float_as_uint(largest);
    int exponent = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    const uint32_t old_bits = __float_as_uint(old) & 0x7fffffffu;
    const bool old_finite = old_bits < 0x7f800000u;
    if (old_finite) exponent = max(exponent, min(static_cast<int>(old_bits >> 23) + ((old_bits & 0x7fffffu) != 0 ? 1 : 0), 254));
    exponent = max(exponent, 1);
    const float scale = __uint_as_float(static_cast<uint32_t>(exponent) << 23);
    const float inverse = __uint_as_float(exponent == 254 ? 0x400000u : static_cast<uint32_t>(254 - exponent) << 23);      // (2^-127 is subnormal)
    if (held_tokens > 0 && scale != old) {
      const float ratio = old_finite ? old * inverse : NAN;
      uint2* const earlier = reinterpret_cast<uint2*>(page_at);
      for (int i = thread; i < held_tokens * vectors; i += TEAM) {
        const uint2 word = earlier[i];
        earlier[i] = make_uint2(encode_again(word.x, ratio), encode_again(word.y, ratio));
      }
    }
    __syncwarp(team);
    if (thread == 0) *scale_at = scale;
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      const int i = thread + h * TEAM;
      if (i < work) to[i] = finite ? encode_vector<T, true>(kept[h], inverse) : encode_vector<T, false>(kept[h], inverse);
    }
    if (work > kHeld * TEAM) {
      each_vector(from, token_stride, [&](int h, int i, const T* at) {
        if (h == kHeld) to[i] = encode_vector<T, false>(*reinterpret_cast<const uint4*>(at), inverse);
      });
    }
  }
}

// ---------------------------------------------------------------------------------------------

constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = 16 * 1024;      // a CTA's piece: of one layer's page, or of several layers' small ones
constexpr int kCopyTensors = 16, kCopyPairs = 1024;

struct CopyTensor {
  char* base;
  long long layer_stride, page_stride;
  long long page_bytes;
  int layers, width;                       // bytes a load moves: 16, 4 or 1
  int layer_pieces, piece_layers;          // pieces of a layer's page (1 where a piece has several layers), layers of a piece
};
struct CopyParams {
  CopyTensor tensors[kCopyTensors];
  int sources[kCopyPairs], targets[kCopyPairs];
  int count, pairs;
};

// `layers` runs of `bytes` bytes, `stride` apart.
template <typename V>
__device__ __forceinline__ void copy_piece(char* to, const char* from, int bytes, int layers, long long stride) {
  const int each = bytes / static_cast<int>(sizeof(V)), n = each * layers;
  constexpr int kUnroll = 4;
  auto place = [&](int i) { return layers == 1 ? static_cast<long long>(i) * sizeof(V) : i / each * stride + static_cast<long long>(i % each) * sizeof(V); };
  for (int i = threadIdx.x; i < n; i += kUnroll * kCopyThreads) {
    V kept[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i + u * kCopyThreads < n) kept[u] = *reinterpret_cast<const V*>(from + place(i + u * kCopyThreads));
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i + u * kCopyThreads < n) *reinterpret_cast<V*>(to + place(i + u * kCopyThreads)) = kept[u];
  }
}

// grid: (pieces of all tensors, pairs)
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyParams p) {
  wait_for_earlier();
  let_later_start();
  int piece = static_cast<int>(blockIdx.x), t = 0;
  auto pieces_of = [&](const CopyTensor& tensor) { return (tensor.layers + tensor.piece_layers - 1) / tensor.piece_layers * tensor.layer_pieces; };
  while (t + 1 < p.count && piece >= pieces_of(p.tensors[t])) piece -= pieces_of(p.tensors[t++]);
  const CopyTensor& tensor = p.tensors[t];
  const int layer = piece / tensor.layer_pieces * tensor.piece_layers;
  const long long first = static_cast<long long>(piece % tensor.layer_pieces) * kCopyBytes;
  const int bytes = static_cast<int>(min(tensor.page_bytes - first, static_cast<long long>(kCopyBytes)));
  const int layers = min(tensor.piece_layers, tensor.layers - layer);
  char* const base = tensor.base + layer * tensor.layer_stride + first;
  const char* from = base + p.sources[blockIdx.y] * tensor.page_stride;
  char* to = base + p.targets[blockIdx.y] * tensor.page_stride;
  if (tensor.width == 16) copy_piece<uint4>(to, from, bytes, layers, tensor.layer_stride);
  else if (tensor.width == 4) copy_piece<uint32_t>(to, from, bytes, layers, tensor.layer_stride);
  else copy_piece<uint8_t>(to, from, bytes, layers, tensor.layer_stride);
}

CopyTensor copy_tensor(const tq_paged_tensor& from) {
  const bool sixteen = aligned_to(from.base, 16) && from.layer_stride % 16 == 0 && from.page_stride % 16 == 0 && from.page_bytes % 16 == 0;
  const bool four = aligned_to(from.base, 4) && from.layer_stride % 4 == 0 && from.page_stride % 4 == 0 && from.page_bytes % 4 == 0;
  return {static_cast<char*>(from.base), from.layer_stride, from.page_stride, from.page_bytes, static_cast<int>(from.layers), sixteen ? 16 : four ? 4 : 1,
          static_cast<int>((from.page_bytes + kCopyBytes - 1) / kCopyBytes), static_cast<int>(from.page_bytes < kCopyBytes ? kCopyBytes / from.page_bytes : 1)};
}

tq_status copy_pages(const std::vector<tq_paged_tensor>& tensors, const std::vector<int64_t>& sources, const std::vector<int64_t>& targets, int32_t device,
                     cudaStream_t stream) {
  DeviceScope device_scope(device);
  if (tq_status s = device_scope.status()) return s;
  for (size_t t0 = 0; t0 < tensors.size();) {
    CopyParams p = {};
    long long pieces = 0;
    for (; t0 < tensors.size() && p.count < kCopyTensors; ++t0) {
      const tq_paged_tensor& from = tensors[t0];
      CopyTensor& to = p.tensors[p.count];
      to = copy_tensor(from);
      const long long more = (from.layers + to.piece_layers - 1) / to.piece_layers * to.layer_pieces;
      if (p.count > 0 && pieces + more >= (1LL << 31)) break;
      pieces += more;
      ++p.count;
    }
    for (size_t i = 0; i < sources.size(); i += kCopyPairs) {
      p.pairs = static_cast<int>(sources.size() - i < kCopyPairs ? sources.size() - i : kCopyPairs);
      for (int n = 0; n < p.pairs; ++n) {
        p.sources[n] = static_cast<int>(sources[i + n]);
        p.targets[n] = static_cast<int>(targets[i + n]);
      }
      const dim3 grid(static_cast<unsigned>(pieces), static_cast<unsigned>(p.pairs));
      TQ_CUDA(launch_overlapped(copy_pages_kernel, grid, kCopyThreads, 0, stream, p));
      if (tq_status s = check_launch("copy_pages_kernel")) return s;
    }
  }
  return TQ_OK;
}

// ---------------------------------------------------------------------------------------------

constexpr int kAdvanceThreads = 1024, kAdvanceWarps = kAdvanceThreads / 32, kAdvanceCtas = 16;
constexpr int kAdvanceSmall = 1 << 14;     // entries and pages that one CTA takes by itself
constexpr int kAdvanceRows = 4096;         // of a cluster, whose books each CTA has in shared memory

// Codes of the status word for a step that could not be made: nothing has changed then, and each row starts at -1.
enum AdvanceFault { kAdvanceFull = 0x46554c4c, kAdvanceParent = 0x50415245 };      // "FULL", "PARE"

struct AdvanceParams {
  const int32_t *table, *lengths, *references, *counts, *parents;      // parents null: each row goes on
  long long table_stride, new_stride;
  int32_t *new_table, *new_lengths, *new_references, *starts;          // results; may be the operands
  bool same_table, same_lengths, same_references, counts_apart;        // counts_apart: not counted in new_references
  int batch, blocks, pages, page_shift;
  // scratch
  int32_t* rows;                       // same_table: the new rows, packed
  int32_t* counted;                    // counts_apart; what follows is in shared memory where one CTA does it all: rows that have a page,
  int32_t* writer;                     // [pages], of last pages alone: the last row that writes into it
  int32_t *row_parent, *row_start, *row_last;      // [batch]: parent, its tokens, the page they end inside (-1: they do not, or nothing is written there)
  int32_t *needs_before, *copies_before;           // [batch]: pages needed, and copies made, by the rows before
  int32_t* free_pages;                 // the lowest free ones
  int32_t *sources, *targets;          // of the copies
  int32_t* totals;                     // {needed, copies, faults} and from 8 on the free pages of each CTA's stretch
};
constexpr int kTotals = 8 + kAdvanceCtas;

__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Exclusive sums over the CTA of two numbers a thread; `total` of all.
__device__ __forceinline__ int2 sums_before(int2 mine, int2* warp_totals, int2& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int2 upto = mine;
#pragma unroll 1
  for (int offset = 1; offset < 32; offset *= 2) {
    const int x = __shfl_up_sync(0xffffffffu, upto.x, offset), y = __shfl_up_sync(0xffffffffu, upto.y, offset);
    if (lane >= offset) {
      upto.x += x;
      upto.y += y;
    }
  }
  if (lane == 31) warp_totals[warp] = upto;
  __syncthreads();
  int2 before = make_int2(0, 0);
  total = before;
#pragma unroll 4
  for (int w = 0; w < kAdvanceWarps; ++w) {
    const int2 one = warp_totals[w];
    total.x += one.x;
    total.y += one.y;
    if (w < warp) {
      before.x += one.x;
      before.y += one.y;
    }
  }
  return make_int2(upto.x - mine.x + before.x, upto.y - mine.y + before.y);
}

// SMALL: one CTA with all books in shared memory; else a cluster with them in scratch (of sixteen: 1024 rows of 138 in a pool of 92000 pages 32 us, of
// eight 42). Each step is few instructions and few loads after one another: a kernel of a few microseconds waits for both (a warp a row, page counts in
// memory and their writers counted apart: 4 rows 17 us, so 10; 256 rows 35).
template <bool SMALL>
__global__ void __launch_bounds__(kAdvanceThreads) cache_advance_kernel(const __grid_constant__ AdvanceParams p, const WaitStatus status) {
  extern __shared__ __align__(16) int32_t books[];      // (read four at a time)
  __shared__ int2 warp_totals[kAdvanceWarps];
  __shared__ int stretch_free[kAdvanceWarps], totals_here[kTotals];
  const int ctas = SMALL ? 1 : static_cast<int>(gridDim.x), cta = SMALL ? 0 : static_cast<int>(blockIdx.x);
  const int thread = cta * kAdvanceThreads + static_cast<int>(threadIdx.x), threads = ctas * kAdvanceThreads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = ctas * kAdvanceWarps, nth_warp = cta * kAdvanceWarps + warp;
  const int page_tokens = 1 << p.page_shift;
  int32_t* const counted = SMALL ? books : p.counts_apart ? p.counted : p.new_references;
  int32_t* const writer = SMALL ? counted + p.pages : p.writer;
  int32_t* const row_parent = SMALL ? writer + p.pages : p.row_parent;
  int32_t* const row_start = SMALL ? row_parent + p.batch : p.row_start;
  int32_t* const row_last = SMALL ? row_start + p.batch : p.row_last;
  int32_t* const needs_before = SMALL ? row_last + p.batch : p.needs_before;
  int32_t* const copies_before = SMALL ? needs_before + p.batch : p.copies_before;
  int32_t* const free_pages = SMALL ? copies_before + p.batch : p.free_pages;
  int32_t* const totals = SMALL ? totals_here : p.totals;
  int32_t* const rows = p.same_table ? p.rows : p.new_table;
  const long long row_stride = p.same_table ? p.blocks : p.new_stride;
  const long long capacity = static_cast<long long>(p.blocks) << p.page_shift;
  auto meet = [&] {
    if constexpr (SMALL) __syncthreads();
    else cluster_meet();
  };
  auto peek = [&](const int32_t* at) {      // what another thread has written
    if constexpr (SMALL) return *at;
    else return __ldcg(at);
  };
  auto fault = [&](int code, int row, int what) {
    atomicCAS(totals + 2, 0, code);
    report(status, code, row, what);
  };
  auto blocks_of = [&](long long tokens) { return static_cast<int>((tokens + page_tokens - 1) >> p.page_shift); };
  auto in_table = [&](int tokens) { return static_cast<int>(min(static_cast<long long>(max(tokens, 0)), capacity)); };
  wait_for_earlier();
  let_later_start();                   // (the copying kernel)

  // Rows, and what there is of each page.
  if (thread < kTotals) totals[thread] = 0;
#pragma unroll 4
  for (int i = thread; i < p.pages; i += threads) {
    counted[i] = p.references[i];
    writer[i] = -1;
  }
  meet();
#pragma unroll 1
  for (int row = thread; row < p.batch; row += threads) {
    const int parent = p.parents == nullptr ? row : p.parents[row], own = p.lengths[row], count = p.counts[row];
    const int tokens = parent < 0 || parent >= p.batch ? 0 : p.lengths[parent];
    row_parent[row] = parent < 0 || parent >= p.batch ? -1 : parent;
    row_start[row] = in_table(tokens);
    row_last[row] = -1;
    if (parent >= p.batch) fault(kAdvanceParent, row, parent);
    else if (own > capacity || tokens > capacity || static_cast<long long>(max(tokens, 0)) + max(count, 0) > capacity) fault(kKeyedLength, row, max(tokens, own));
  }
  meet();

  // Entries: the parents' pages, and how many rows have each; a row that will write into its last page gives that up, for now.
  const bool near = !SMALL && p.batch <= kAdvanceRows;      // each CTA has all rows' books at hand
  if (near) {
#pragma unroll 1
    for (int row = threadIdx.x; row < p.batch; row += kAdvanceThreads) {
      books[row] = peek(row_parent + row);
      books[kAdvanceRows + row] = peek(row_start + row);
      books[2 * kAdvanceRows + row] = p.lengths[row];
    }
    __syncthreads();
  }
  // A thread has several entries at a time, so that their loads are under way together: of one row by a warp, or, of up to 32 entries, of several rows by
  // as many lanes as hold a row. (Of 1024 rows of 138 this takes 7.5 us of 28; entries
  // of all rows one after another, a division each, 2 us more.)
  constexpr int kAtOnce = 4;
  auto take = [&](const int (&row)[kAtOnce], const int (&i)[kAtOnce]) {
    int before[kAtOnce], now[kAtOnce], start[kAtOnce], had[kAtOnce];
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      if (row[n] >= p.batch || i[n] >= p.blocks) continue;
      const int parent = near ? books[row[n]] : peek(row_parent + row[n]);
      start[n] = near ? books[kAdvanceRows + row[n]] : peek(row_start + row[n]);
      had[n] = blocks_of(in_table(near ? books[2 * kAdvanceRows + row[n]] : p.lengths[row[n]]));
      before[n] = p.table[row[n] * p.table_stride + i[n]];
      now[n] = i[n] < blocks_of(start[n]) ? p.table[parent * p.table_stride + i[n]] : before[n];
    }
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      if (row[n] >= p.batch || i[n] >= p.blocks) continue;
      rows[row[n] * row_stride + i[n]] = now[n];
      const bool drops = i[n] < had[n], takes = i[n] < blocks_of(start[n]);
      if ((drops && (before[n] < 0 || before[n] >= p.pages)) || (takes && (now[n] < 0 || now[n] >= p.pages))) {
        fault(kKeyedPage, row[n], i[n]);
        continue;
      }
      const bool writes = takes && i[n] == start[n] >> p.page_shift && p.counts[row[n]] > 0;      // (the tokens end inside this page)
      if (drops != takes || before[n] != now[n]) {
        if (drops) atomicAdd(counted + before[n], -1);
        if (takes && !writes) atomicAdd(counted + now[n], 1);
      } else if (writes) {
        atomicAdd(counted + now[n], -1);
      }
      if (writes) {
        atomicMax(writer + now[n], row[n]);
        row_last[row[n]] = now[n];
      }
    }
  };
  if (p.blocks > 32) {
#pragma unroll 1
    for (int row = nth_warp; row < p.batch; row += warps) {
#pragma unroll 1
      for (int i = lane; i < p.blocks; i += 32 * kAtOnce) {
        int of[kAtOnce], at[kAtOnce];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
          of[n] = row;
          at[n] = i + 32 * n;
        }
        take(of, at);
      }
    }
  } else {
    const int shift = p.blocks <= 1 ? 0 : 32 - __clz(p.blocks - 1), step = threads >> shift;      // lanes of a row: 2^shift
#pragma unroll 1
    for (int row = thread >> shift; row < p.batch; row += kAtOnce * step) {
      int of[kAtOnce], at[kAtOnce];
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        of[n] = row + n * step;
        at[n] = thread & ((1 << shift) - 1);
      }
      take(of, at);
    }
  }
  meet();

  // The last of the rows that write into a page keeps it where nobody else has it (-2 - page from here on); the others copy it. What each row needs (the first CTA).
  if (cta == 0) {
    const int run = (p.batch + kAdvanceThreads - 1) / kAdvanceThreads;
    const int first = min(static_cast<int>(threadIdx.x) * run, p.batch), last = min(first + run, p.batch);
    int2 mine = make_int2(0, 0);
#pragma unroll 1
    for (int row = first; row < last; ++row) {
      const int start = peek(row_start + row), count = max(p.counts[row], 0), page = peek(row_last + row);
      const int copies = page >= 0 && (peek(counted + page) > 0 || peek(writer + page) != row) ? 1 : 0;
      if (page >= 0 && copies == 0) row_last[row] = -2 - page;
      needs_before[row] = mine.x;      // (within the run so far)
      copies_before[row] = mine.y;
      mine.x += copies + blocks_of(static_cast<long long>(start) + count) - blocks_of(start);
      mine.y += copies;
    }
    int2 total;
    const int2 before = sums_before(mine, warp_totals, total);      // (the CTA meets in there, after which pages that are kept count again)
#pragma unroll 1
    for (int row = first; row < last; ++row) {
      const int page = row_last[row];
      needs_before[row] += before.x;
      copies_before[row] += before.y;
      if (page <= -2) atomicExch(counted + (-2 - page), 1);
    }
    if (threadIdx.x == 0) {
      totals[0] = total.x;
      totals[1] = total.y;
    }
  }
  meet();

  // Where the free pages are; a warp has a stretch of pages, a lane four neighbouring ones at a time (`counted` is 16-byte aligned).
  const int stretch = ((p.pages + warps - 1) / warps + 127) / 128 * 128;
  const int page0 = static_cast<int>(min(static_cast<long long>(nth_warp) * stretch, static_cast<long long>(p.pages)));
  const int page1 = static_cast<int>(min(static_cast<long long>(page0) + stretch, static_cast<long long>(p.pages)));
  auto free_of_four = [&](int page) {      // bits
    page += 4 * lane;
    if (page + 3 < page1) {
      const int4 four = SMALL ? *reinterpret_cast<const int4*>(counted + page) : __ldcg(reinterpret_cast<const int4*>(counted + page));
      return (four.x == 0 ? 1 : 0) | (four.y == 0 ? 2 : 0) | (four.z == 0 ? 4 : 0) | (four.w == 0 ? 8 : 0);
    }
    int bits = 0;
    for (int n = 0; n < 4; ++n)
      if (page + n < page1 && peek(counted + page + n) == 0) bits |= 1 << n;
    return bits;
  };
  int free_here = 0;
#pragma unroll 4
  for (int page = page0; page < page1; page += 128) free_here += __popc(free_of_four(page));
  free_here = __reduce_add_sync(0xffffffffu, free_here);
  if (lane == 0) stretch_free[warp] = free_here;
  __syncthreads();
  int free_before = 0, free_all = 0;
#pragma unroll 4
  for (int w = 0; w < kAdvanceWarps; ++w) {
    const int there = stretch_free[w];
    if (w < warp) free_before += there;
    free_all += there;
  }
  if constexpr (!SMALL) {
    if (threadIdx.x == 0) totals[8 + cta] = free_all;
    meet();
    const int there = lane < ctas ? peek(totals + 8 + lane) : 0;
    free_before += __reduce_add_sync(0xffffffffu, lane < cta ? there : 0);
    free_all = __reduce_add_sync(0xffffffffu, there);
  }
  const int needed = peek(totals), copies = peek(totals + 1), fault_before = peek(totals + 2);
  const bool good = fault_before == 0 && needed <= free_all;
  if (good) {
#pragma unroll 1
    for (int page = page0; page < page1 && free_before < needed; page += 128) {
      const int bits = free_of_four(page), mine = __popc(bits);
      int upto = mine;
#pragma unroll
      for (int offset = 1; offset < 32; offset *= 2) {
        const int other = __shfl_up_sync(0xffffffffu, upto, offset);
        if (lane >= offset) upto += other;
      }
      int place = free_before + upto - mine;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        if ((bits >> n & 1) == 0) continue;
        if (place < needed) free_pages[place] = page + 4 * lane + n;
        ++place;
      }
      free_before += __shfl_sync(0xffffffffu, upto, 31);
    }
  } else if (thread == 0 && fault_before == 0) {
    report(status, kAdvanceFull, needed, free_all);
  }
  meet();

  // The rows take their pages, which then have one row each.
#pragma unroll 1
  for (int row = thread; good && row < p.batch; row += threads) {
    const int start = peek(row_start + row), has = blocks_of(start), will = blocks_of(static_cast<long long>(start) + max(p.counts[row], 0));
    int at = peek(needs_before + row);
    const int last = peek(row_last + row);
    if (last >= 0) {
      const int pair = peek(copies_before + row), page = peek(free_pages + at++);
      p.sources[pair] = last;
      p.targets[pair] = page;
      rows[row * row_stride + has - 1] = page;
    }
#pragma unroll 1
    for (int i = has; i < will; ++i) rows[row * row_stride + i] = peek(free_pages + at++);
  }
#pragma unroll 1
  for (int i = thread; good && i < needed; i += threads) atomicExch(counted + peek(free_pages + i), 1);
  if (thread == 0) *p.totals = good ? copies : 0;      // how many the next kernel copies
  // (lengths and counts are read until here, results that may be these written from here on)
#pragma unroll 1
  for (int row = thread; row < p.batch; row += threads) p.starts[row] = good ? peek(row_start + row) : -1;
  if (p.same_lengths || p.same_table || p.same_references || !SMALL) meet();
  else __syncthreads();
#pragma unroll 1
  for (int row = thread; row < p.batch; row += threads) {
    if (good) p.new_lengths[row] = peek(row_start + row) + max(p.counts[row], 0);
    else if (!p.same_lengths) p.new_lengths[row] = p.lengths[row];
  }
  if (good ? SMALL || p.counts_apart : !p.same_references) {
#pragma unroll 4
    for (int i = thread; i < p.pages; i += threads) p.new_references[i] = good ? peek(counted + i) : p.references[i];
  }
  if (good ? p.same_table : !p.same_table) {
#pragma unroll 1
    for (int row = nth_warp; row < p.batch; row += warps) {
#pragma unroll 4
      for (int i = lane; i < p.blocks; i += 32)
        p.new_table[row * p.new_stride + i] = good ? __ldcg(rows + row * row_stride + i) : p.table[row * p.table_stride + i];
    }
  }
}

struct NamedCopies {
  CopyTensor tensors[4];
  int count;
  const int32_t *sources, *targets, *pairs;      // device memory
};

// grid: (pieces of all tensors, pairs at once)
__global__ void __launch_bounds__(kCopyThreads) copy_named_pages_kernel(const __grid_constant__ NamedCopies p) {
  wait_for_earlier();
  let_later_start();
  const int pairs = *p.pairs;
  if (static_cast<int>(blockIdx.y) >= pairs) return;
  int piece = static_cast<int>(blockIdx.x), t = 0;
  auto pieces_of = [&](const CopyTensor& tensor) { return (tensor.layers + tensor.piece_layers - 1) / tensor.piece_layers * tensor.layer_pieces; };
  while (t + 1 < p.count && piece >= pieces_of(p.tensors[t])) piece -= pieces_of(p.tensors[t++]);
  const CopyTensor& tensor = p.tensors[t];
  const int layer = piece / tensor.layer_pieces * tensor.piece_layers;
  const long long first = static_cast<long long>(piece % tensor.layer_pieces) * kCopyBytes;
  const int bytes = static_cast<int>(min(tensor.page_bytes - first, static_cast<long long>(kCopyBytes)));
  const int layers = min(tensor.piece_layers, tensor.layers - layer);
  char* const base = tensor.base + layer * tensor.layer_stride + first;
  for (int pair = blockIdx.y; pair < pairs; pair += gridDim.y) {
    const char* from = base + p.sources[pair] * tensor.page_stride;
    char* to = base + p.targets[pair] * tensor.page_stride;
    if (tensor.width == 16) copy_piece<uint4>(to, from, bytes, layers, tensor.layer_stride);
    else if (tensor.width == 4) copy_piece<uint32_t>(to, from, bytes, layers, tensor.layer_stride);
    else copy_piece<uint8_t>(to, from, bytes, layers, tensor.layer_stride);
  }
}

// Scratch of an advance: where each array begins, in int32. `small`: what one CTA keeps in shared memory, and how much of that there is.
constexpr size_t kAdvanceShared = 200 * 1024;
struct AdvanceScratch {
  bool small;
  size_t shared_bytes;
  int64_t rows, counted, writer, parent, start, last, needs, copies, free_pages, sources, targets, totals, all;
};
AdvanceScratch advance_scratch(int64_t batch, int64_t blocks, int64_t pages) {
  AdvanceScratch at = {};
  at.shared_bytes = static_cast<size_t>(3 * pages + 5 * batch) * sizeof(int32_t);
  at.small = batch * blocks + pages <= kAdvanceSmall && at.shared_bytes <= kAdvanceShared;
  int64_t end = 0;
  auto take = [&](int64_t count) {
    const int64_t begin = end;
    end += (count + 3) / 4 * 4;
    return begin;
  };
  at.rows = take(batch * blocks);
  at.sources = take(batch);
  at.targets = take(batch);
  at.totals = take(kTotals);
  if (!at.small) {
    at.counted = take(pages);
    at.writer = take(pages);
    at.parent = take(batch);
    at.start = take(batch);
    at.last = take(batch);
    at.needs = take(batch);
    at.copies = take(batch);
    at.free_pages = take(pages);
  }
  at.all = end;
  return at;
}

cudaLaunchConfig_t advance_cluster(int ctas, cudaLaunchAttribute* attribute) {
  attribute->id = cudaLaunchAttributeClusterDimension;
  attribute->val.clusterDim.x = static_cast<unsigned>(ctas);
  attribute->val.clusterDim.y = attribute->val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(ctas));
  config.blockDim = dim3(kAdvanceThreads);
  config.dynamicSmemBytes = 3 * kAdvanceRows * sizeof(int32_t);
  config.attrs = attribute;
  config.numAttrs = 1;
  return config;
}

// CTAs of the cluster: sixteen where `device` has room for them in one (not every part of a GPU has), or the eight that always have. Asked once for each.
tq_status advance_ctas(int32_t device, int* ctas) {
  static std::mutex mutex;
  static int known[64] = {};
  std::lock_guard<std::mutex> lock(mutex);
  int asked = 0;
  int& of = device >= 0 && device < 64 ? known[device] : asked;
  if (of == 0) {
    cudaLaunchAttribute attribute;
    const cudaLaunchConfig_t config = advance_cluster(kAdvanceCtas, &attribute);
    TQ_CUDA(cudaFuncSetAttribute(cache_advance_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(config.dynamicSmemBytes)));
    int clusters = 0;
    const bool fits = cudaFuncSetAttribute(cache_advance_kernel<false>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                      cudaOccupancyMaxActiveClusters(&clusters, cache_advance_kernel<false>, &config) == cudaSuccess && clusters > 0;
    if (!fits) cudaGetLastError();
    of = fits ? kAdvanceCtas : 8;
  }
  *ctas = of;
  return TQ_OK;
}

bool advance_takes(int64_t batch, int64_t blocks, int64_t pages, int64_t page_tokens) {
  const int page_shift = page_shift_of(page_tokens);
  return batch > 0 && blocks >= 0 && pages >= 0 && page_shift >= 0 && pages < (1LL << 30) && batch < (1LL << 20) && blocks < (1LL << 30) >> page_shift &&
         batch * blocks < (1LL << 30);
}

}  // namespace
}  // namespace tq

extern "C" tq_status tq_cache_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_tokens, int64_t head_dim,
                                                        int64_t page_tokens, int64_t blocks, int64_t window, int64_t sinks, int32_t device,
                                                        size_t* bytes) {
  TQ_REQUIRE(bytes != nullptr, TQ_INVALID_ARGUMENT, "null out-pointer");
  *bytes = 0;
  // (of what the launch has nothing to do for, or refuses: nothing)
  const int page_shift = tq::page_shift_of(page_tokens);
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || q_tokens <= 0 || blocks <= 0 || page_shift < 0 || blocks >= (1LL << 30) >> page_shift ||
      batch >= (1LL << 24) || kv_heads >= 65536 || heads / kv_heads * q_tokens >= (1LL << 24) || window < 0 || sinks < 0 || head_dim <= 0 || head_dim > 128)
    return TQ_OK;
  tq::KeyedParams p = {};
  tq::keyed_extents(p, batch, heads, kv_heads, q_tokens, head_dim, 1.0, window, sinks);
  *bytes = tq::keyed_workspace(true, p, blocks * page_tokens, device);
  return TQ_OK;
}

extern "C" tq_status tq_cache_attention_launch(tq_dtype dtype, const void* q, const void* k_pages, const void* v_pages, const float* k_scales,
                                               const float* v_scales, const int32_t* table, const int32_t* lengths, void* out, int64_t batch,
                                               int64_t heads, int64_t kv_heads, int64_t q_tokens, int64_t head_dim, int64_t pages, int64_t page_tokens,
                                               int64_t blocks, int64_t table_stride, const int64_t* q_strides, const int64_t* out_strides, double scale,
                                               int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes, int32_t device, void* stream) {
  TQ_REQUIRE(q_strides != nullptr && out_strides != nullptr, TQ_INVALID_ARGUMENT, "null strides");
  if (tq::recording()) {
    struct Kept { int64_t q[3], out[3]; } kept;
    for (int i = 0; i < 3; ++i) {
      kept.q[i] = q_strides[i];
      kept.out[i] = out_strides[i];
    }
    return tq::record([=](int32_t d, void* s) {
      return tq_cache_attention_launch(dtype, q, k_pages, v_pages, k_scales, v_scales, table, lengths, out, batch, heads, kv_heads, q_tokens, head_dim, pages,
                                       page_tokens, blocks, table_stride, kept.q, kept.out, scale, window, sinks, workspace, workspace_bytes, d, s);
    });
  }
  if (tq_status s = tq::cache_checks(dtype, batch, kv_heads, head_dim, pages, page_tokens, blocks)) return s;
  const int page_shift = tq::page_shift_of(page_tokens);
  TQ_REQUIRE(heads >= 0 && q_tokens >= 0 && window >= 0 && sinks >= 0, TQ_INVALID_ARGUMENT, "negative heads=%lld, q_tokens=%lld, window=%lld or sinks=%lld",
             (long long)heads, (long long)q_tokens, (long long)window, (long long)sinks);
  if (batch == 0 || heads == 0 || q_tokens == 0) return TQ_OK;
  TQ_REQUIRE(kv_heads > 0 && heads % kv_heads == 0, TQ_INVALID_ARGUMENT, "%lld heads do not share %lld key heads evenly", (long long)heads, (long long)kv_heads);
  TQ_REQUIRE(scale > 0.0 && scale <= tq::kKeyedMostScale, TQ_UNSUPPORTED, "the score scale must be positive and finite in f32, not %g", scale);
  TQ_REQUIRE(q != nullptr && out != nullptr && lengths != nullptr, TQ_INVALID_ARGUMENT, "null operand or result");
  TQ_REQUIRE(blocks == 0 || table != nullptr, TQ_INVALID_ARGUMENT, "null table");
  TQ_REQUIRE(pages == 0 || (k_pages != nullptr && v_pages != nullptr && k_scales != nullptr && v_scales != nullptr), TQ_INVALID_ARGUMENT, "null cache");
  TQ_REQUIRE(tq::keyed_query_fits(q, q_strides, out, out_strides, batch, heads, q_tokens), TQ_UNSUPPORTED,
             "queries must be 16-byte aligned with strides that are multiples of 8 elements, results aligned to their type, with no negative strides");
  TQ_REQUIRE(tq::aligned_to(k_pages, 16) && tq::aligned_to(v_pages, 16) && tq::aligned_to(k_scales, 4) && tq::aligned_to(v_scales, 4) &&
                 tq::aligned_to(table, 4) && tq::aligned_to(lengths, 4),
             TQ_UNSUPPORTED, "the cache's codes must be 16-byte aligned, its other tensors 4-byte aligned");
  TQ_REQUIRE(heads / kv_heads * q_tokens < (1LL << 24), TQ_UNSUPPORTED, "extents beyond the kernel's index range");
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
  p.page_shift = page_shift;
  p.pages = static_cast<int>(pages);
  p.out = out;
  for (int i = 0; i < 3; ++i) {
    p.q_strides[i] = q_strides[i];
    p.out_strides[i] = out_strides[i];
  }
  tq::keyed_extents(p, batch, heads, kv_heads, q_tokens, head_dim, scale, window, sinks);
  return tq::keyed_attention(dtype, true, p, blocks * page_tokens, workspace, workspace_bytes, device, static_cast<cudaStream_t>(stream));
}

extern "C" tq_status tq_cache_store_launch(tq_dtype dtype, const void* k, const void* v, void* k_pages, void* v_pages, float* k_scales, float* v_scales,
                                           const int32_t* table, const int32_t* starts, const int32_t* counts, int64_t batch, int64_t kv_heads,
                                           int64_t tokens, int64_t head_dim, int64_t pages, int64_t page_tokens, int64_t blocks, int64_t table_stride,
                                           const int64_t* k_strides, const int64_t* v_strides, int32_t device, void* stream) {
  TQ_REQUIRE(k_strides != nullptr && v_strides != nullptr, TQ_INVALID_ARGUMENT, "null strides");
  if (tq::recording()) {
    struct Kept { int64_t k[3], v[3]; } kept;
    for (int i = 0; i < 3; ++i) {
      kept.k[i] = k_strides[i];
      kept.v[i] = v_strides[i];
    }
    return tq::record([=](int32_t d, void* s) {
      return tq_cache_store_launch(dtype, k, v, k_pages, v_pages, k_scales, v_scales, table, starts, counts, batch, kv_heads, tokens, head_dim, pages,
                                   page_tokens, blocks, table_stride, kept.k, kept.v, d, s);
    });
  }
  if (tq_status s = tq::cache_checks(dtype, batch, kv_heads, head_dim, pages, page_tokens, blocks)) return s;
  const int page_shift = tq::page_shift_of(page_tokens);
  TQ_REQUIRE(tokens >= 0, TQ_INVALID_ARGUMENT, "negative extent in tokens=%lld", (long long)tokens);
  TQ_REQUIRE(tokens < (1LL << 30), TQ_UNSUPPORTED, "extents beyond the kernel's index range");
  if (batch == 0 || kv_heads == 0 || tokens == 0) return TQ_OK;
  TQ_REQUIRE(k != nullptr && v != nullptr && starts != nullptr, TQ_INVALID_ARGUMENT, "null operand");
  TQ_REQUIRE(blocks == 0 || table != nullptr, TQ_INVALID_ARGUMENT, "null table");
  TQ_REQUIRE(pages == 0 || (k_pages != nullptr && v_pages != nullptr && k_scales != nullptr && v_scales != nullptr), TQ_INVALID_ARGUMENT, "null cache");
  for (const int64_t* strides : {k_strides, v_strides}) {
    const bool whole = (batch == 1 || strides[0] % 8 == 0) && (kv_heads == 1 || strides[1] % 8 == 0) && (tokens == 1 || strides[2] % 8 == 0);
    TQ_REQUIRE(whole, TQ_UNSUPPORTED, "the strides of new keys and values must be multiples of 8 elements");
  }
  TQ_REQUIRE(tq::aligned_to(k, 16) && tq::aligned_to(v, 16) && tq::aligned_to(k_pages, 16) && tq::aligned_to(v_pages, 16) && tq::aligned_to(k_scales, 4) &&
                 tq::aligned_to(v_scales, 4) && tq::aligned_to(table, 4) && tq::aligned_to(starts, 4) && tq::aligned_to(counts, 4),
             TQ_UNSUPPORTED, "new keys and values and the cache's codes must be 16-byte aligned, the other tensors 4-byte aligned");
  tq::DeviceScope device_scope(device);
  if (tq_status s = device_scope.status()) return s;
  tq::StoreParams p = {};
  p.status = tq::wait_status_for(device);
  TQ_REQUIRE(p.status.abort != nullptr, TQ_RESOURCE_EXHAUSTED, "no device memory for the status word");
  p.x[0] = k;
  p.x[1] = v;
  p.codes[0] = static_cast<uint8_t*>(k_pages);
  p.codes[1] = static_cast<uint8_t*>(v_pages);
  p.scales[0] = k_scales;
  p.scales[1] = v_scales;
  for (int i = 0; i < 3; ++i) {
    p.strides[0][i] = k_strides[i];
    p.strides[1][i] = v_strides[i];
  }
  p.table = table;
  p.starts = starts;
  p.counts = counts;
  p.table_stride = table_stride;
  p.blocks = static_cast<int>(blocks);
  p.page_shift = page_shift;
  p.pages = static_cast<int>(pages);
  p.batch = static_cast<int>(batch);
  p.kv_heads = static_cast<int>(kv_heads);
  p.tokens = static_cast<int>(tokens);
  p.head_dim = static_cast<int>(head_dim);
  p.touched = static_cast<int>((tokens + page_tokens - 2) / page_tokens + 1);
  // Half a warp where it keeps a page's new tokens in registers (eight vectors a thread), else a warp, else a CTA: a team waits for its loads a head
  // at a time, and more and smaller teams have more of them under way (32 x 12 heads of 64, 2047 tokens in pages of 16 with a warp 73.2 us, with
  // half a one 52.6; one token of 128 x 8 heads of 128 4.2 and 3.8). Registers for eight vectors where four or one do cost CTAs an SM and empty
  // instructions (the same in pages of 64, a CTA each: 64.4 and 54.4). A team takes several heads where there would be more than four times as
  // many teams as run at once; with as many as run at once, four times as many and one for every head: 32 x 8 heads of 2047 tokens of 128, pages
  // of 64 68.4, 65.8, 65.7, pages of 16 (then a warp each) 77.7, 71.5, 71.6; 32 x 12 of 64, pages of 16 82.4, 74.8, 85.9.
  const long long vectors = (tokens < page_tokens ? tokens : page_tokens) * head_dim / 8;
  const int team = vectors <= 8 * 16 ? 16 : vectors <= 8 * 32 ? 32 : tq::kStoreThreads;
  const long long pairs = static_cast<long long>(p.batch) * p.touched;
  const long long teams_at_once = static_cast<long long>(tq::sm_count(device)) * (32 * tq::kStoreThreads / team);
  const long long runs = teams_at_once / pairs < 1 ? 1 : teams_at_once / pairs < 2 * kv_heads ? teams_at_once / pairs : 2 * kv_heads;
  p.each = static_cast<int>((2 * kv_heads + runs - 1) / runs);
  p.runs = (2 * p.kv_heads + p.each - 1) / p.each;
  const long long items = pairs * p.runs, ctas = (items * team + tq::kStoreThreads - 1) / tq::kStoreThreads;
  TQ_REQUIRE(ctas < (1LL << 31), TQ_UNSUPPORTED, "too many pages and heads for one launch");
  cudaStream_t cuda_stream = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel) -> tq_status {
    TQ_CUDA(tq::launch_overlapped(kernel, dim3(static_cast<unsigned>(ctas)), tq::kStoreThreads, 0, cuda_stream, p));
    return tq::check_launch("cache_store_kernel");
  };
  auto with_held = [&](auto type) -> tq_status {
    using T = decltype(type);
    if (team == 16) return vectors <= 16 ? go(tq::cache_store_kernel<T, 16, 1>) : go(tq::cache_store_kernel<T, 16, 8>);
    if (team == 32) return go(tq::cache_store_kernel<T, 32, 8>);
    return vectors <= 512 ? go(tq::cache_store_kernel<T, tq::kStoreThreads, 4>) : go(tq::cache_store_kernel<T, tq::kStoreThreads, 8>);
  };
  return dtype == TQ_BF16 ? with_held(__nv_bfloat16{}) : with_held(__half{});
}

extern "C" tq_status tq_copy_pages_launch(const tq_paged_tensor* tensors, int32_t count, int64_t pages, const int64_t* sources, const int64_t* targets,
                                          int64_t pairs, int32_t device, void* stream) {
  TQ_REQUIRE(count >= 0 && pages >= 0 && pairs >= 0, TQ_INVALID_ARGUMENT, "negative count=%d, pages=%lld or pairs=%lld", count, (long long)pages,
             (long long)pairs);
  if (count == 0 || pairs == 0) return TQ_OK;
  TQ_REQUIRE(tensors != nullptr && sources != nullptr && targets != nullptr, TQ_INVALID_ARGUMENT, "null argument");
  TQ_REQUIRE(pages < (1LL << 31), TQ_UNSUPPORTED, "extents beyond the kernel's index range");
  try {
    std::vector<tq_paged_tensor> some;
    for (int32_t i = 0; i < count; ++i) {
      const tq_paged_tensor& t = tensors[i];
      TQ_REQUIRE(t.layers >= 0 && t.page_bytes >= 0 && t.layer_stride >= 0 && t.page_stride >= 0, TQ_INVALID_ARGUMENT, "negative extent of tensor %d", i);
      if (t.layers == 0 || t.page_bytes == 0) continue;
      TQ_REQUIRE(t.base != nullptr, TQ_INVALID_ARGUMENT, "tensor %d is null", i);
      TQ_REQUIRE(t.page_stride >= t.page_bytes, TQ_INVALID_ARGUMENT, "the pages of tensor %d overlap", i);
      TQ_REQUIRE(t.layers <= 65535 && t.page_bytes < (1LL << 34) && t.layers * ((t.page_bytes + tq::kCopyBytes - 1) / tq::kCopyBytes) < (1LL << 31),
                 TQ_UNSUPPORTED, "extents beyond the kernel's index range");
      some.push_back(t);
    }
    // what is a source, what a target: a bit each
    std::vector<uint8_t> marks(static_cast<size_t>(pages), 0);
    for (int64_t i = 0; i < pairs; ++i) {
      TQ_REQUIRE(sources[i] >= 0 && sources[i] < pages && targets[i] >= 0 && targets[i] < pages, TQ_INVALID_ARGUMENT,
                 "pair %lld names page %lld or %lld of %lld pages", (long long)i, (long long)sources[i], (long long)targets[i], (long long)pages);
      marks[sources[i]] |= 1;
      TQ_REQUIRE((marks[targets[i]] & 2) == 0, TQ_INVALID_ARGUMENT, "page %lld is a target twice", (long long)targets[i]);
      marks[targets[i]] |= 2;
    }
    for (int64_t i = 0; i < pairs; ++i)
      TQ_REQUIRE(marks[targets[i]] == 2, TQ_INVALID_ARGUMENT, "page %lld is a source and a target", (long long)targets[i]);
    std::vector<int64_t> from(sources, sources + pairs), to(targets, targets + pairs);
    if (tq::recording()) {
      return tq::record([some, from, to](int32_t d, void* s) { return tq::copy_pages(some, from, to, d, static_cast<cudaStream_t>(s)); });
    }
    return tq::copy_pages(some, from, to, device, static_cast<cudaStream_t>(stream));
  } catch (const std::bad_alloc&) {
    return tq::fail(TQ_RESOURCE_EXHAUSTED, "no host memory for %lld pages and %lld pairs", (long long)pages, (long long)pairs);
  }
}

extern "C" tq_status tq_cache_advance_workspace_bytes(int64_t batch, int64_t blocks, int64_t pages, int64_t page_tokens, size_t* bytes) {
  TQ_REQUIRE(bytes != nullptr, TQ_INVALID_ARGUMENT, "null out-pointer");
  *bytes = tq::advance_takes(batch, blocks, pages, page_tokens) ? static_cast<size_t>(tq::advance_scratch(batch, blocks, pages).all) * sizeof(int32_t) : 0;
  return TQ_OK;
}

extern "C" tq_status tq_cache_advance_launch(const tq_paged_tensor* tensors, int32_t count, const int32_t* table, const int32_t* lengths,
                                             const int32_t* references, const int32_t* counts, const int32_t* parents, int32_t* new_table,
                                             int32_t* new_lengths, int32_t* new_references, int32_t* starts, int64_t batch, int64_t blocks, int64_t pages,
                                             int64_t page_tokens, int64_t table_stride, int64_t new_stride, void* workspace, size_t workspace_bytes,
                                             int32_t device, void* stream) {
  TQ_REQUIRE(count >= 0 && count <= 4 && (count == 0 || tensors != nullptr), TQ_INVALID_ARGUMENT, "%d tensors of pages, not up to 4", count);
  if (tq::recording()) {
    struct Kept { tq_paged_tensor tensors[4]; } kept = {};
    for (int i = 0; i < count; ++i) kept.tensors[i] = tensors[i];
    return tq::record([=](int32_t d, void* s) {
      return tq_cache_advance_launch(kept.tensors, count, table, lengths, references, counts, parents, new_table, new_lengths, new_references, starts, batch,
                                     blocks, pages, page_tokens, table_stride, new_stride, workspace, workspace_bytes, d, s);
    });
  }
  TQ_REQUIRE(batch >= 0 && blocks >= 0 && pages >= 0, TQ_INVALID_ARGUMENT, "negative extent in batch=%lld blocks=%lld pages=%lld", (long long)batch,
             (long long)blocks, (long long)pages);
  TQ_REQUIRE(tq::page_shift_of(page_tokens) >= 0, TQ_UNSUPPORTED, "a page holds 16, 32, 64, ... 1024 tokens, not %lld", (long long)page_tokens);
  if (batch == 0) {
    TQ_REQUIRE(pages == 0 || references == new_references, TQ_UNSUPPORTED, "a table of no rows advances in place alone");
    return TQ_OK;
  }
  TQ_REQUIRE(tq::advance_takes(batch, blocks, pages, page_tokens), TQ_UNSUPPORTED, "extents beyond the kernel's index range");
  TQ_REQUIRE(lengths != nullptr && counts != nullptr && new_lengths != nullptr && starts != nullptr && (blocks == 0 || (table != nullptr && new_table != nullptr)) &&
                 (pages == 0 || (references != nullptr && new_references != nullptr)),
             TQ_INVALID_ARGUMENT, "null operand or result");
  TQ_REQUIRE(table_stride >= blocks || batch == 1, TQ_INVALID_ARGUMENT, "the table's rows overlap");
  TQ_REQUIRE(new_stride >= blocks || batch == 1, TQ_INVALID_ARGUMENT, "the new table's rows overlap");
  TQ_REQUIRE(new_table != table || new_stride == table_stride || batch == 1 || blocks == 0, TQ_INVALID_ARGUMENT, "a table in place has one stride");
  for (const void* each : {static_cast<const void*>(table), static_cast<const void*>(lengths), static_cast<const void*>(references),
                           static_cast<const void*>(counts), static_cast<const void*>(parents), static_cast<const void*>(new_table),
                           static_cast<const void*>(new_lengths), static_cast<const void*>(new_references), static_cast<const void*>(starts)})
    TQ_REQUIRE(tq::aligned_to(each, 4), TQ_UNSUPPORTED, "the books' tensors must be 4-byte aligned");
  const tq::AdvanceScratch at = tq::advance_scratch(batch, blocks, pages);
  TQ_REQUIRE(workspace != nullptr && workspace_bytes >= static_cast<size_t>(at.all) * sizeof(int32_t) && tq::aligned_to(workspace, 16), TQ_INVALID_ARGUMENT,
             "this advance needs %zu bytes of workspace, 16-byte aligned, and was given %zu", static_cast<size_t>(at.all) * sizeof(int32_t), workspace_bytes);
  tq::NamedCopies copies = {};
  long long pieces = 0;
  for (int32_t i = 0; i < count; ++i) {
    const tq_paged_tensor& t = tensors[i];
    TQ_REQUIRE(t.layers >= 0 && t.page_bytes >= 0 && t.layer_stride >= 0 && t.page_stride >= 0, TQ_INVALID_ARGUMENT, "negative extent of tensor %d", i);
    if (t.layers == 0 || t.page_bytes == 0) continue;
    TQ_REQUIRE(t.base != nullptr, TQ_INVALID_ARGUMENT, "tensor %d is null", i);
    TQ_REQUIRE(t.page_stride >= t.page_bytes, TQ_INVALID_ARGUMENT, "the pages of tensor %d overlap", i);
    TQ_REQUIRE(t.layers <= 65535 && t.page_bytes < (1LL << 34) && t.layers * ((t.page_bytes + tq::kCopyBytes - 1) / tq::kCopyBytes) < (1LL << 29),
               TQ_UNSUPPORTED, "extents beyond the kernel's index range");
    tq::CopyTensor& to = copies.tensors[copies.count++];
    to = tq::copy_tensor(t);
    pieces += (to.layers + to.piece_layers - 1) / to.piece_layers * static_cast<long long>(to.layer_pieces);
  }
  tq::DeviceScope device_scope(device);
  if (tq_status s = device_scope.status()) return s;
  const tq::WaitStatus status = tq::wait_status_for(device);
  TQ_REQUIRE(status.abort != nullptr, TQ_RESOURCE_EXHAUSTED, "no device memory for the status word");
  int32_t* const scratch = static_cast<int32_t*>(workspace);
  tq::AdvanceParams p = {};
  p.table = table;
  p.lengths = lengths;
  p.references = references;
  p.counts = counts;
  p.parents = parents;
  p.table_stride = table_stride;
  p.new_stride = new_stride;
  p.new_table = new_table;
  p.new_lengths = new_lengths;
  p.new_references = new_references;
  p.starts = starts;
  p.same_table = new_table == table;
  p.same_lengths = new_lengths == lengths;
  p.same_references = new_references == references;
  p.counts_apart = p.same_references || !tq::aligned_to(new_references, 16);
  p.batch = static_cast<int>(batch);
  p.blocks = static_cast<int>(blocks);
  p.pages = static_cast<int>(pages);
  p.page_shift = tq::page_shift_of(page_tokens);
  p.rows = scratch + at.rows;
  p.counted = scratch + at.counted;
  p.writer = scratch + at.writer;
  p.row_parent = scratch + at.parent;
  p.row_start = scratch + at.start;
  p.row_last = scratch + at.last;
  p.needs_before = scratch + at.needs;
  p.copies_before = scratch + at.copies;
  p.free_pages = scratch + at.free_pages;
  p.sources = scratch + at.sources;
  p.targets = scratch + at.targets;
  p.totals = scratch + at.totals;
  cudaStream_t cuda_stream = static_cast<cudaStream_t>(stream);
  const auto held = tq::hold_scratch(workspace);
  if (at.small) {
    TQ_CUDA(cudaFuncSetAttribute(tq::cache_advance_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(tq::kAdvanceShared)));
    TQ_CUDA(tq::launch_overlapped(tq::cache_advance_kernel<true>, dim3(1), tq::kAdvanceThreads, at.shared_bytes, cuda_stream, p, status));
  } else {
    int ctas = 0;
    if (tq_status s = tq::advance_ctas(device, &ctas)) return s;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = tq::advance_cluster(ctas, attributes + 1);
    config.stream = cuda_stream;
    config.attrs = attributes;
    config.numAttrs = 2;
    TQ_CUDA(cudaLaunchKernelEx(&config, tq::cache_advance_kernel<false>, p, status));
  }
  if (tq_status s = tq::check_launch("cache_advance_kernel")) return s;
  if (copies.count == 0) return TQ_OK;
  copies.sources = p.sources;
  copies.targets = p.targets;
  copies.pairs = p.totals;
  const long long at_once = tq::sm_count(device) * 8LL / pieces;
  const dim3 grid(static_cast<unsigned>(pieces), static_cast<unsigned>(at_once < 1 ? 1 : at_once < batch ? at_once : batch));
  TQ_CUDA(tq::launch_overlapped(tq::copy_named_pages_kernel, grid, tq::kCopyThreads, 0, cuda_stream, copies));
  return tq::check_launch("copy_named_pages_kernel");
}
