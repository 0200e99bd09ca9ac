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
#include <cmath>
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

tq_status copy_pages(const std::vector<tq_paged_tensor>& tensors, const std::vector<int64_t>& sources, const std::vector<int64_t>& targets, int32_t device,
                     cudaStream_t stream) {
  DeviceScope device_scope(device);
  if (tq_status s = device_scope.status()) return s;
  for (size_t t0 = 0; t0 < tensors.size();) {
    CopyParams p = {};
    long long pieces = 0;
    for (; t0 < tensors.size() && p.count < kCopyTensors; ++t0) {
      const tq_paged_tensor& from = tensors[t0];
      const bool sixteen = aligned_to(from.base, 16) && from.layer_stride % 16 == 0 && from.page_stride % 16 == 0 && from.page_bytes % 16 == 0;
      const bool four = aligned_to(from.base, 4) && from.layer_stride % 4 == 0 && from.page_stride % 4 == 0 && from.page_bytes % 4 == 0;
      CopyTensor& to = p.tensors[p.count];
      to = {static_cast<char*>(from.base), from.layer_stride, from.page_stride, from.page_bytes, static_cast<int>(from.layers), sixteen ? 16 : four ? 4 : 1,
            static_cast<int>((from.page_bytes + kCopyBytes - 1) / kCopyBytes), static_cast<int>(from.page_bytes < kCopyBytes ? kCopyBytes / from.page_bytes : 1)};
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

// log2 of a page's tokens, or -1.
int page_shift_of(int64_t page_tokens) {
  for (int shift = 4; shift <= 10; ++shift)
    if (page_tokens == (1LL << shift)) return shift;
  return -1;
}

}  // namespace
}  // namespace tq

#define TQ_CACHE_CHECKS()                                                                                                                          \
  TQ_REQUIRE(dtype == TQ_BF16 || dtype == TQ_F16, TQ_UNSUPPORTED, "the cache takes and gives bf16 or f16, not %s", tq::dtype_name(dtype));         \
  TQ_REQUIRE(head_dim >= 16 && head_dim <= 128 && head_dim % 16 == 0, TQ_UNSUPPORTED, "the cache holds heads of 16, 32, ... 128 elements, not %lld", \
             (long long)head_dim);                                                                                                                 \
  const int page_shift = tq::page_shift_of(page_tokens);                                                                                           \
  TQ_REQUIRE(page_shift >= 0, TQ_UNSUPPORTED, "a page holds 16, 32, 64, ... 1024 tokens, not %lld", (long long)page_tokens);                       \
  TQ_REQUIRE(pages >= 0 && blocks >= 0 && kv_heads >= 0 && batch >= 0, TQ_INVALID_ARGUMENT,                                                        \
             "negative extent in batch=%lld kv_heads=%lld pages=%lld blocks=%lld", (long long)batch, (long long)kv_heads, (long long)pages, (long long)blocks); \
  TQ_REQUIRE(pages < (1LL << 31) && kv_heads < 65536 && batch < (1LL << 24) && blocks < (1LL << 30) >> page_shift, TQ_UNSUPPORTED,                    \
             "extents beyond the kernel's index range")

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
  TQ_CACHE_CHECKS();
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
  TQ_CACHE_CHECKS();
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
