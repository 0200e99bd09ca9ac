// What the entry points of window and cache attention (cache.cu, attention.cu) hand to the kernels of keyed.cu.
#pragma once

#include "common.h"

namespace tq {

// Codes of the status word for a cache whose table or lengths a kernel could not follow: it leaves out the keys that are not there.
enum KeyedFault { kKeyedPage = 0x50414745, kKeyedLength = 0x4c454e47 };      // "PAGE", "LENG"

struct KeyedParams {
  const void *q, *k, *v;
  void* out;
  long long q_strides[3], k_strides[3], v_strides[3], out_strides[3];      // batch, head, token, in elements; k and v: dense keys only
  const float *k_scales, *v_scales;                                        // paged keys: [pages, kv_heads]
  const int32_t *table, *lengths;
  long long table_stride;
  int blocks, page_shift, pages;
  int boxes, box_shift;                                                    // of a chunk: its pieces of a page, and log2 of their tokens
  int batch, heads, kv_heads, group, q_tokens, k_tokens, head_dim;
  int window, sinks;
  int row_tiles, shares, joins;                                            // joins: shares whose parts of a unit are joined before they go to memory
  float* parts;                                                            // of units that a border between two shares cuts
  int4* borders;                                                           // the border behind each share: {sequence, unit, first and last share
                                                                           // with parts of it}, none where these are equal
  float2* part_stats;                                                      // ... their maximum and sum
  float scale_log2;
  WaitStatus status;
  // Sequences in runs of `each` that share their first keys (null: none do). Parts of a row's result are left, not the result: prefix.cu joins them.
  const int32_t* shared;                                                   // of each run: how many first keys its sequences have in common
  int each;
  int runs;                                                                // so many of the first "sequences" are runs: the shared keys, for the rows of
                                                                           // a run together; the others are sequences, and what each has behind them
  bool late;                                                               // the kernel before in the stream leaves other parts and need not have ended
  int typical;                                                             // for the plan: the keys a unit has on average, where that is known to be less
                                                                           // than the most; else 0
  int part_rows, part_count;                                               // rows of a run and key head, rounded up; parts of each, the sequences' own last
  float* row_parts;                                                        // [run][key head][part][row][64 or 128]
  float2* row_stats;                                                       // ... their maximum and sum
};

// The keys of a run's beginning are taken together in tiles of so many; what is left of it each sequence reads itself.
constexpr int kPrefixTile = 128;

constexpr double kKeyedMostScale = 2e38;      // times log2(e) it still is an f32

// log2 of a page's tokens, or -1.
inline int page_shift_of(int64_t page_tokens) {
  for (int shift = 4; shift <= 10; ++shift)
    if (page_tokens == (1LL << shift)) return shift;
  return -1;
}

// What every call over the cache checks of it first.
inline tq_status cache_checks(tq_dtype dtype, int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t pages, int64_t page_tokens, int64_t blocks) {
  TQ_REQUIRE(dtype == TQ_BF16 || dtype == TQ_F16, TQ_UNSUPPORTED, "the cache takes and gives bf16 or f16, not %s", dtype_name(dtype));
  TQ_REQUIRE(head_dim >= 16 && head_dim <= 128 && head_dim % 16 == 0, TQ_UNSUPPORTED, "the cache holds heads of 16, 32, ... 128 elements, not %lld",
             (long long)head_dim);
  const int page_shift = page_shift_of(page_tokens);
  TQ_REQUIRE(page_shift >= 0, TQ_UNSUPPORTED, "a page holds 16, 32, 64, ... 1024 tokens, not %lld", (long long)page_tokens);
  TQ_REQUIRE(pages >= 0 && blocks >= 0 && kv_heads >= 0 && batch >= 0, TQ_INVALID_ARGUMENT,
             "negative extent in batch=%lld kv_heads=%lld pages=%lld blocks=%lld", (long long)batch, (long long)kv_heads, (long long)pages, (long long)blocks);
  TQ_REQUIRE(pages < (1LL << 31) && kv_heads < 65536 && batch < (1LL << 24) && blocks < (1LL << 30) >> page_shift, TQ_UNSUPPORTED,
             "extents beyond the kernel's index range");
  return TQ_OK;
}

// What queries and results have to be: read 16 bytes at a time, written through any strides.
inline bool keyed_query_fits(const void* q, const int64_t* q_strides, const void* out, const int64_t* out_strides, int64_t batch, int64_t heads,
                             int64_t q_tokens) {
  const bool whole = (batch == 1 || q_strides[0] % 8 == 0) && (heads == 1 || q_strides[1] % 8 == 0) && (q_tokens == 1 || q_strides[2] % 8 == 0);
  return whole && aligned_to(q, 16) && aligned_to(out, 2) && out_strides[0] >= 0 && out_strides[1] >= 0 && out_strides[2] >= 0;
}

// `window` 0: none. Positions stay below 2^30, so this one reaches them all and position - window does not wrap.
constexpr int64_t kKeyedEverything = 1LL << 30;
inline void keyed_extents(KeyedParams& p, int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_tokens, int64_t head_dim, double scale,
                          int64_t window, int64_t sinks) {
  p.batch = static_cast<int>(batch);
  p.heads = static_cast<int>(heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.group = static_cast<int>(heads / kv_heads);
  p.q_tokens = static_cast<int>(q_tokens);
  p.head_dim = static_cast<int>(head_dim);
  p.window = static_cast<int>(window == 0 || window > kKeyedEverything ? kKeyedEverything : window);
  p.sinks = static_cast<int>(sinks > kKeyedEverything ? kKeyedEverything : sinks);
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
}

// Probabilities that are rounded to f16 are taken 2^kHalfLift times as large, which cancels in the quotient: 2^(kSlack + kHalfLift) is the largest then,
// inside f16's 2^16, and those that fall under its normal range, 2^-14, are under 2^-21 of the row's largest.
constexpr float kHalfLift = 7.f;

// Few rows a key head against many keys: `p` is complete but for what follows from the plan; no sequence has more than `keys` keys. With `p.shared`
// (paged keys, no window): parts of the rows' results.
size_t keyed_workspace(bool paged, const KeyedParams& p, long long keys, int32_t device);
// The time it is expected to take, us.
double keyed_time(bool paged, const KeyedParams& p, long long keys, int32_t device);
tq_status keyed_attention(tq_dtype dtype, bool paged, KeyedParams& p, long long keys, void* workspace, size_t workspace_bytes, int32_t device,
                          cudaStream_t stream);

#ifdef __CUDACC__
// Launches `kernel` so that its start (CTAs placed, barriers set up) passes under the end of the kernel before it in the stream. Each of its
// threads calls wait_for_earlier() before it touches memory. Every CTA waits, also one with nothing to do: what comes after this kernel then
// comes after the one before it too. (One new token of 64 x 12 heads stored: 5.7 us without, 4.3 with; a kernel of the libraries before it ends
// first, as ever.) A kernel whose CTAs have much to do calls let_later_start() at their end: earlier, the next kernel's first CTAs would gather
// where places become free first, and unevenly (2 x 32/8 heads of 64, 2501 tokens under a window of 513 one after another 52.4 us, and 46.4; a
// step of 64 x 12 heads over 1000 keys 21.9 and 20.7).
template <typename... Parameters, typename... Arguments>
cudaError_t launch_overlapped(void (*kernel)(Parameters...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, const Arguments&... arguments) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, arguments...);
}
__device__ __forceinline__ void wait_for_earlier() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_later_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// How many of a sequence's first keys are taken together with those of its run: whole tiles, and only if all of its queries see them all.
__device__ __forceinline__ int shared_keys(const KeyedParams& p, int run) {
  return min(max(p.shared[run], 0), p.blocks << p.page_shift) / kPrefixTile * kPrefixTile;
}
__device__ __forceinline__ bool takes_part(const KeyedParams& p, int shared, int length) { return length - p.q_tokens + 1 >= shared; }
// Where part `part` of a row (of the run's rows of a key head) lies.
__device__ __forceinline__ long long part_slot(const KeyedParams& p, int run, int kv_head, int part, int row) {
  return ((static_cast<long long>(run) * p.kv_heads + kv_head) * p.part_count + part) * p.part_rows + row;
}

// The first fault since the last poll is kept, with where it was.
__device__ __forceinline__ void report(const WaitStatus& status, int code, int sequence, int what) {
  int* words = status.sticky();
  if (atomicCAS(words, 0, code) == 0) {
    words[1] = static_cast<int>(blockIdx.x);
    words[2] = static_cast<int>(threadIdx.x);
    words[3] = sequence;
    words[4] = what;
  }
}
#endif

}  // namespace tq
