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
};

constexpr double kKeyedMostScale = 2e38;      // times log2(e) it still is an f32

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

// Few rows a key head against many keys: `p` is complete but for what follows from the plan; no sequence has more than `keys` keys.
size_t keyed_workspace(bool paged, const KeyedParams& p, long long keys, int32_t device);
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
