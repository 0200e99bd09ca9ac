// Beam search's selection, for sm_100a: of all beams and tokens of a request the best `keep`, by
//
//   value(b, t) = score_b + x[b, t] - log sum_u exp(x[b, u])       x: logits; in falling order, ties to the lower beam, then the lower token
//
// Within a beam the order is that of the logits, so a beam's candidates are its `keep` largest logits, and the logarithm of its sum is needed to compare
// beams alone. Bound: HBM by the bytes (each logit is read once), the instructions of the first kernel by what they are (12 a logit of bf16: half of
// them to widen, scale, add and compare, an exponential, the rest what chunks, lists and their pruning cost).
//
// First kernel: a CTA takes a part of a beam's logits, 16 KB chunks one after another through a ring of two in shared memory (cp.async; four CTAs an SM.
// Smaller chunks in deeper rings, and three, five or six CTAs an SM, were no faster; in registers, the next one's loads under way, a third slower): their
// sum of exponentials, and their `keep` largest. In the first chunk every warp's r-th largest thread maximum, r = keep / warps, is a bound below
// which nothing is needed (warps * r threads have something at or above it); what is at or above the lowest of these goes to a list, a few times
// `keep` long. Its `keep`-th best is the bound for the chunks behind, of which 32 / n of the n-th reach it. Places in a list are counted by comparing
// its members with each other. A list that overflows (very many equal logits, a mask of -inf) is answered by `keep` rounds of the CTA's maximum, a chunk
// after the other for as long as the bound lets that many logits through: a mask that leaves few tokens is dear, see below.
// Second kernel: a CTA a request joins the parts: sums, values in f64, a bound by the digits of their order, and places by comparison.
//
// Measured (B200, from a graph, cold caches): 32 x 16 beams of 128000 bf16 logits, 32 kept, 61 us (131 MB; the first kernel 48: issue slots 58 % taken, the
// special-function unit 46 %, warps that wait for the list's pruning), 64 x 4 beams of 50257 in f32 31 us (51 MB), one request of 4 beams 16 us, nearly all of
// it launches and waits for what came before (the parts 6.4, the join 8). 32 x 16 x 128000 of which all but 16 tokens are hidden: 8 kept 0.47 ms, 32 kept
// 2.6 ms. A second look (8 of 100 such calls without masks) 40 us for each of its beams; 64 x 4 x 50257 where a request's beams are alike 103 us.
//
// Precision: a thread adds up to 16 exponentials of a chunk in f32 at a time (8 roundings after one another), and these sums in f64. An exponent's rounding
// grows with the logit's distance from what the sum stands at, so that is a logit, and not far from the largest: the first chunk's, until a later chunk
// has one that is kStand above it; the sum is brought to that one then, and the chunk's taken again. A lone token's logarithm is exact. Values of
// neighbours are as close as 1e-7 now and then, so candidates of two beams that their sums cannot tell apart (near_values: 4e-6) have these taken again,
// in f64 throughout.
#include <cmath>
#include <type_traits>

#include "common.h"
#include "keyed.h"
#include "tcgen05.h"

namespace tq {
namespace {

constexpr int kSelectThreads = 256, kSelectWarps = kSelectThreads / 32;
constexpr int kVecs = 4;                                    // a thread's vectors of 16 bytes of a chunk
constexpr int kChunkBytes = kSelectThreads * kVecs * 16;
constexpr int kStages = 2;                                  // chunks on chip
constexpr int kListed = 1024;                               // candidates on chip
constexpr int kJoinThreads = 512, kJoinWarps = kJoinThreads / 32;
constexpr int kUppers = 6144;                               // candidates of which the joining kernel keeps half the order
constexpr int kMostBeams = 128, kMostKept = 128;
constexpr int kSelectCtas = 592;                            // at once on a B200, four an SM
// How far above what a sum stands at a logit may lie: no farther than most of a vocabulary lies below it. (Each move takes a chunk's sum again: 32 x 16 x
// 128000 bf16 with tokens that stand out 56.7 us, by 4 57.9, without any moves 56.3.)
constexpr float kStand = 8.f;
constexpr float kLog2E = 1.4426950408889634f;

struct SelectParams {
  const void* logits;
  long long request_stride, beam_stride;                    // elements
  const float* scores;                                      // [requests, beams]
  const uint8_t* finished;                                  // the same, or null
  int beams, vocab, keep, parts, chunk, end;
  double near;                                              // near_values
  double2* sums;                                            // [rows, parts]: the logit the sum stands at, and the sum of exponentials over it
  unsigned long long* keys;                                 // [rows, parts, keep]: candidates of a part, the best first; 0: none
  float* out_scores;                                        // [requests, keep]
  int32_t *out_parents, *out_tokens;
};

// Order of floats as unsigned integers, -inf at 0x007fffff; 0 is less than any.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t bits = __float_as_uint(x + 0.f);           // (-0 is 0)
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ unsigned long long ordered(double x) {
  const unsigned long long bits = static_cast<unsigned long long>(__double_as_longlong(x + 0.0));
  return bits >> 63 ? ~bits : bits | 1ull << 63;
}

// The r-th largest of a warp's 32 numbers, counted with repetition; 0 where there are fewer above 0.
__device__ __forceinline__ uint32_t warp_nth(uint32_t mine, int r) {
  uint32_t most = 0;
  for (int n = 0; n < r; ++n) {
    most = __reduce_max_sync(0xffffffffu, mine);
    const uint32_t holders = __ballot_sync(0xffffffffu, mine == most);
    if ((threadIdx.x & 31) == __ffs(holders) - 1) mine = 0;
  }
  return most;
}

template <typename T>
__device__ __forceinline__ void widen(const uint4& word, float* to) {
  const uint32_t w[4] = {word.x, word.y, word.z, word.w};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if constexpr (std::is_same_v<T, float>) {
      to[c] = __uint_as_float(w[c]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      to[2 * c] = __uint_as_float(w[c] << 16);
      to[2 * c + 1] = __uint_as_float(w[c] & 0xffff0000u);
    } else {
      const float2 pair = __half22float2(*reinterpret_cast<const __half2*>(&w[c]));
      to[2 * c] = pair.x;
      to[2 * c + 1] = pair.y;
    }
  }
}

// How many of a list on chip come before an item (the same list for all threads: its reads are under way together).
template <typename Item, typename Before>
__device__ __forceinline__ int place_in(const Item* list, int found, Before&& before_it) {
  int place = 0;
#pragma unroll 8
  for (int j = 0; j < found; ++j) place += before_it(list[j]) ? 1 : 0;
  return place;
}

__device__ __forceinline__ void copy_async_16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_address(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kSelectThreads, 4) beam_parts_kernel(const __grid_constant__ SelectParams p) {
  constexpr int kVec = 16 / sizeof(T), kChunk = kChunkBytes / sizeof(T);
  __shared__ uint4 ring[kStages][kVecs][kSelectThreads];    // a thread reads what it has copied itself
  __shared__ uint32_t warp_most[kSelectWarps], warp_bound[kSelectWarps];
  __shared__ double warp_sum[kSelectWarps];
  __shared__ unsigned long long lists[kListed + kMostKept], warp_key[kSelectWarps];      // the list, and room for the best of it
  __shared__ int listed;
  const int part = static_cast<int>(blockIdx.x), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.y;
  const int request = static_cast<int>(row / p.beams), beam = static_cast<int>(row % p.beams);
  unsigned long long* const list = lists;
  unsigned long long* const kept = lists + kListed;
  if (threadIdx.x == 0) listed = 0;
  wait_for_earlier();
  if (p.finished != nullptr && p.finished[row]) return;     // (its one candidate is made in the joining kernel)
  const int first = part * p.chunk, count = min(p.chunk, p.vocab - first);
  const T* const from = static_cast<const T*>(p.logits) + request * p.request_stride + beam * p.beam_stride + first;
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(from) & 15) / sizeof(T));
  const int chunks = (count + skew + kChunk - 1) / kChunk;

  // A thread's vectors of a chunk, whole vectors of 16 bytes from the one that the part begins in; what lies before or behind the part is -inf.
  auto place_of = [&](int chunk, int i) { return ((chunk * kVecs + i) * kSelectThreads + static_cast<int>(threadIdx.x)) * kVec - skew; };      // in the part
  auto ask = [&](int chunk) {
    if (chunk < chunks) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int at = place_of(chunk, i);
        uint4* const to = &ring[chunk % kStages][i][threadIdx.x];
        if (at >= 0 && at + kVec <= count) {
          copy_async_16(to, from + at);
        } else {
          for (int c = 0; c < kVec; ++c) reinterpret_cast<T*>(to)[c] = at + c >= 0 && at + c < count ? from[at + c] : from_compute<T, float>(-INFINITY);
        }
      }
    }
    copy_async_commit();
  };
  auto words = [&](int chunk, int i, float (&x)[kVec]) { widen<T>(ring[chunk % kStages][i][threadIdx.x], x); };
  auto key_of = [&](float x, int at) { return static_cast<unsigned long long>(ordered(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(first + at)); };
  float threshold = -INFINITY, shift = 0.f, bar = -INFINITY;      // the sum stands at `shift` (at no logit yet: bar is -inf); logits above `bar` move it
  double sum = 0.0, here = 0.0;                                   // here: of the chunk
  // Sums a chunk up, and adds what reaches the bound to the list: whether that has become long, or a logit is above the bar, for the CTA.
  auto take = [&](int chunk) {
    float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
    float chunk_most = -INFINITY;
    uint32_t reaching = 0;                                    // vectors; few do
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      float x[kVec];
      words(chunk, i, x);
      float most = -INFINITY;
#pragma unroll
      for (int c = 0; c < kVec; c += 2) {
        const float2 t = __fmul2_rn(__fadd2_rn(make_float2(x[c], x[c + 1]), make_float2(-shift, -shift)), make_float2(kLog2E, kLog2E));
        const float2 e = make_float2(exp2_ftz(t.x), exp2_ftz(t.y));
        if (c % 4 == 0) sum0 = __fadd2_rn(sum0, e);
        else sum1 = __fadd2_rn(sum1, e);
        most = fmaxf(most, fmaxf(x[c], x[c + 1]));
      }
      reaching |= most >= threshold ? 1u << i : 0u;
      chunk_most = fmaxf(chunk_most, most);                   // (above the bar it is above all before, and so among the best)
    }
    const float2 both = __fadd2_rn(sum0, sum1);
    here = static_cast<double>(both.x) + static_cast<double>(both.y);
    int last = 0;
    if (reaching != 0) {                                      // (behind the loop, so that a warp's threads go through this together)
      static_assert(kVecs * kVec <= 32, "a bit for each of a thread's logits of a chunk");
      uint32_t taken = 0;
#pragma unroll 1
      for (uint32_t left = reaching; left != 0; left &= left - 1) {
        const int i = __ffs(left) - 1, at = place_of(chunk, i);
        float x[kVec];
        words(chunk, i, x);
        uint32_t some = 0;
#pragma unroll
        for (int c = 0; c < kVec; ++c) some |= x[c] >= threshold && at + c >= 0 && at + c < count ? 1u << c : 0u;
        taken |= some << (i * kVec);
      }
      last = atomicAdd(&listed, __popc(taken));
#pragma unroll 1
      for (; taken != 0; taken &= taken - 1, ++last) {
        const int bit = __ffs(taken) - 1, i = bit / kVec, c = bit % kVec;
        if (last < kListed) list[last] = key_of(to_compute(reinterpret_cast<const T*>(&ring[chunk % kStages][i][threadIdx.x])[c]), place_of(chunk, i) + c);
      }
    }
    return __syncthreads_or(chunk_most > bar || last >= max(2 * p.keep, 32)) != 0;
  };
  // Brings the sum to a logit above the bar, the best of the list now, and takes the chunk's again.
  auto stand = [&](int chunk) {
    const float top = from_ordered(static_cast<uint32_t>(list[0] >> 32));
    if (!(top > bar)) return;
    sum *= exp(static_cast<double>(bar == -INFINITY ? bar : shift) - top);      // (no logits before: 0, or NaN)
    shift = top;
    bar = top + kStand;
    here = 0.0;
#pragma unroll 1
    for (int i = 0; i < kVecs; ++i) {
      float x[kVec];
      words(chunk, i, x);
#pragma unroll
      for (int c = 0; c < kVec; ++c) here += static_cast<double>(exp2_ftz((x[c] - shift) * kLog2E));
    }
  };
  // The list's best `keep` in their order, as the list; all threads.
  auto prune = [&] {
    const int found = listed;
    for (int i = threadIdx.x; i < p.keep; i += kSelectThreads) kept[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < found; i += kSelectThreads) {
      const unsigned long long key = list[i];
      const int place = place_in(list, found, [&](unsigned long long other) { return other > key; });
      if (place < p.keep) kept[place] = key;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.keep; i += kSelectThreads) list[i] = kept[i];
    if (threadIdx.x == 0) listed = min(found, p.keep);
    __syncthreads();                                          // (nobody adds before that)
    if (found >= p.keep) threshold = from_ordered(static_cast<uint32_t>(list[p.keep - 1] >> 32));
  };
  // The same where the list has overflown (very many equal logits, a mask of -inf), by as many rounds: over what the list has, and the chunk.
  auto prune_chunk = [&](int chunk) {
    unsigned long long last = ~0ull;
    for (int n = 0; n < p.keep; ++n) {
      unsigned long long best = 0;
      for (int i = threadIdx.x; i < kListed; i += kSelectThreads)
        if (list[i] < last && list[i] > best) best = list[i];
#pragma unroll 1
      for (int i = 0; i < kVecs; ++i) {
        float x[kVec];
        words(chunk, i, x);
        const int at = place_of(chunk, i);
#pragma unroll
        for (int c = 0; c < kVec; ++c) {
          const unsigned long long key = at + c >= 0 && at + c < count ? key_of(x[c], at + c) : 0;
          if (key < last && key > best) best = key;
        }
      }
#pragma unroll
      for (int offset = 16; offset > 0; offset /= 2) best = max(best, __shfl_xor_sync(0xffffffffu, best, offset));
      if (lane == 0) warp_key[warp] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kSelectWarps; ++w) best = max(best, warp_key[w]);
      if (threadIdx.x == 0) kept[n] = best;
      last = best;
      __syncthreads();
    }
    for (int i = threadIdx.x; i < p.keep; i += kSelectThreads) list[i] = kept[i];
    if (threadIdx.x == 0) listed = p.keep;                    // (some may be 0, none)
    __syncthreads();
    if (list[p.keep - 1] != 0) threshold = from_ordered(static_cast<uint32_t>(list[p.keep - 1] >> 32));
  };

  for (int chunk = 0; chunk < kStages; ++chunk) ask(chunk);
  copy_async_wait<kStages - 1>();
  // The first chunk says what the sum stands at, its maximum (+inf and NaN make the sum NaN), and a bound.
  {
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      float x[kVec];
      words(0, i, x);
#pragma unroll
      for (int c = 0; c < kVec; ++c) most = fmaxf(most, x[c]);
    }
    // Warps of which every thread has logits: of 2048 or more all.
    const int vectors = (count + skew + kVec - 1) / kVec, full = min(vectors / 32, kSelectWarps);
    const int nth = full == 0 ? 33 : (p.keep + full - 1) / full;
    const uint32_t mine = ordered(most);
    const uint32_t in_warp = __reduce_max_sync(0xffffffffu, mine);
    const uint32_t bound = nth > 32 ? 0 : nth == 1 ? in_warp : warp_nth(mine, nth);
    if (lane == 0) {
      warp_most[warp] = in_warp;
      warp_bound[warp] = bound;
    }
    __syncthreads();
    uint32_t top = 0, least = 0xffffffffu;
#pragma unroll
    for (int w = 0; w < kSelectWarps; ++w) {
      top = max(top, warp_most[w]);
      if (w < full) least = min(least, warp_bound[w]);
    }
    if (nth > 32) least = 0;
    threshold = least <= 0x007fffffu ? -INFINITY : from_ordered(least);
    most = from_ordered(top);
    if (most > -INFINITY) {
      shift = most;
      bar = most + kStand;
    }
  }
  for (int chunk = 0; chunk < chunks; ++chunk) {
    copy_async_wait<kStages - 1>();
    if (take(chunk)) {
      if (listed > kListed) prune_chunk(chunk);
      else prune();
      stand(chunk);
    } else if (chunk == 0 && chunks > 1) {
      prune();                                                // (a tighter bound for the others)
    }
    sum += here;
    ask(chunk + kStages);
  }
  copy_async_wait<0>();
  let_later_start();
#pragma unroll
  for (int offset = 16; offset > 0; offset /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
  if (lane == 0) warp_sum[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kSelectWarps; ++w) all += warp_sum[w];
    p.sums[row * p.parts + part] = make_double2(shift, all);
  }
  unsigned long long* const to = p.keys + (row * p.parts + part) * p.keep;
  const int found = listed;
  for (int i = threadIdx.x; i < found; i += kSelectThreads) {
    const unsigned long long key = list[i];
    const int place = place_in(list, found, [&](unsigned long long other) { return other > key; });
    if (place < p.keep) to[place] = key;
  }
  for (int i = found + threadIdx.x; i < p.keep; i += kSelectThreads) to[i] = 0;
}

enum BeamState { kGoesOn = 0, kFinished, kNothing, kNoNumber };      // kNothing: every logit, or the score, is -inf; kNoNumber: NaN, or +inf

struct Candidate {
  unsigned long long order;      // of the value; 0: none
  uint32_t beam, token;
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
  return a.order != b.order ? a.order > b.order : a.beam != b.beam ? a.beam < b.beam : a.token < b.token;
}

// A sum that stands at `from`, at `to` >= `from` (-inf: no sum; what is +inf is NaN by now).
__device__ __forceinline__ double brought(double sum, float from, float to) { return from == to || from == -INFINITY ? sum : sum * exp(static_cast<double>(from) - to); }

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) beam_join_kernel(const __grid_constant__ SelectParams p) {
  __shared__ double logarithm[kMostBeams], score_of[kMostBeams];
  __shared__ uint8_t state[kMostBeams], again[kMostBeams];
  __shared__ Candidate list[kListed], warp_best[kJoinWarps];
  __shared__ int bins[6][16];
  __shared__ uint32_t uppers[kUppers];
  __shared__ double warp_sum[kJoinWarps];
  __shared__ int listed, near;
  const int request = static_cast<int>(blockIdx.x), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  wait_for_earlier();
  const int slots = p.parts * p.keep + 1, all = p.beams * slots;      // of a beam, and of the request
  const long long keys0 = static_cast<long long>(request) * p.beams * (slots - 1);
  if (threadIdx.x == 0) near = 0;
  __syncthreads();
  for (int beam = warp; beam < p.beams; beam += kJoinWarps) {
    const long long row = static_cast<long long>(request) * p.beams + beam;
    const float score = p.scores[row];
    const bool finished = p.finished != nullptr && p.finished[row];
    float at = -INFINITY;
    double sum = 0.0;
    if (!finished) {
      for (int part = lane; part < p.parts; part += 32) {
        const double2 one = p.sums[row * p.parts + part];
        // (a part of -inf alone has the sum 0 at 0; of a NaN its sum is one)
        if (one.y == 0.0) continue;
        const float there = static_cast<float>(one.x), both = fmaxf(at, there);
        sum = brought(sum, at, both) + brought(one.y, there, both);
        at = both;
      }
      const float lane_at = at;
#pragma unroll
      for (int offset = 16; offset > 0; offset /= 2) at = fmaxf(at, __shfl_xor_sync(0xffffffffu, at, offset));
      sum = brought(sum, lane_at, at);
#pragma unroll
      for (int offset = 16; offset > 0; offset /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
    }
    if (lane == 0) {
      score_of[beam] = score;
      again[beam] = 0;
      int now = kGoesOn;
      if (!(score < INFINITY)) now = kNoNumber;
      else if (finished) now = kFinished;
      else if (!(sum >= 0.0) || !(sum < INFINITY) || at == INFINITY) now = kNoNumber;
      else if (sum == 0.0 || score == -INFINITY) now = kNothing;
      state[beam] = static_cast<uint8_t>(now);
      logarithm[beam] = now == kGoesOn ? at + log(sum) : 0.0;
    }
  }
  __syncthreads();
  const int most_tokens = min(p.keep, p.vocab);
  auto candidate = [&](int i) {
    const int beam = i / slots, c = i - beam * slots;
    Candidate one = {0, static_cast<uint32_t>(beam), static_cast<uint32_t>(c)};
    if (state[beam] == kGoesOn) {
      const unsigned long long key = c == slots - 1 ? 0ull : p.keys[keys0 + i - beam];
      if (key == 0) return one;
      one.token = 0xffffffffu - static_cast<uint32_t>(key);
      one.order = ordered(score_of[beam] + (static_cast<double>(from_ordered(static_cast<uint32_t>(key >> 32))) - logarithm[beam]));
    } else if (state[beam] == kFinished) {
      const bool ends = c == slots - 1 ? p.end >= most_tokens : c == p.end;      // (among the first tokens, or in the last place)
      if (!ends && c >= most_tokens) return one;
      if (ends) one.token = static_cast<uint32_t>(p.end);
      one.order = ordered(ends ? score_of[beam] : -INFINITY);
    } else if (c < most_tokens) {
      one.order = state[beam] == kNothing ? ordered(-static_cast<double>(INFINITY)) : ~0ull;
    }
    return one;
  };
  auto value_of = [](unsigned long long order) {
    return order == ~0ull ? static_cast<double>(NAN) : __longlong_as_double(static_cast<long long>(order >> 63 ? order & ~(1ull << 63) : ~order));
  };
  for (int round = 0;; ++round) {
    // The upper halves of the candidates' orders stay on chip (beyond kUppers they are made again and again). Loops as they are: what runs once waits for
    // its instructions, and unrolled this took twice as long.
    auto upper = [&](int i) { return i < kUppers ? uppers[i] : static_cast<uint32_t>(candidate(i).order >> 32); };
#pragma unroll 1
    for (int i = threadIdx.x; i < min(all, kUppers); i += kJoinThreads) uppers[i] = static_cast<uint32_t>(candidate(i).order >> 32);
    // The largest bound that `keep` candidates reach, four of the order's upper 24 bits (12 of f64's fraction) at a time; lowered by what is close.
    uint32_t least = 0;
    for (int i = threadIdx.x; i < 6 * 16; i += kJoinThreads) bins[i / 16][i % 16] = 0;
    __syncthreads();
    int above = 0;                                            // candidates above the bits found so far
#pragma unroll 1
    for (int n = 0; n < 6; ++n) {
      const int low = 28 - 4 * n;
#pragma unroll 1
      for (int i = threadIdx.x; i < all; i += kJoinThreads) {
        const uint32_t order = upper(i);
        if (order != 0 && (n == 0 || order >> (low + 4) == least >> (low + 4))) atomicAdd(&bins[n][order >> low & 15], 1);
      }
      __syncthreads();
      // Lane d has how many reach digit d: the last lane that `keep` reach, or 0.
      const int mine = lane < 16 ? bins[n][lane] : 0;
      int reach = mine;
#pragma unroll
      for (int offset = 1; offset < 16; offset *= 2) {
        const int more = __shfl_down_sync(0xffffffffu, reach, offset);
        if (lane + offset < 16) reach += more;
      }
      const uint32_t enough = __ballot_sync(0xffffffffu, lane < 16 && above + reach >= p.keep);
      const int digit = enough == 0 ? 0 : 31 - __clz(enough);
      above += __shfl_sync(0xffffffffu, reach - mine, digit);
      least |= static_cast<uint32_t>(digit) << low;
    }
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    unsigned long long threshold = static_cast<unsigned long long>(least) << 32;
    if (round == 0 && least != 0 && least != 0xffffff00u) {
      const double lower = value_of(threshold) - p.near;
      if (lower == lower) threshold = ordered(lower);      // (of -inf: -inf)
    }
    if (threshold == 0) threshold = 1;
#pragma unroll 1
    for (int i = threadIdx.x; i < all; i += kJoinThreads) {
      if (upper(i) < static_cast<uint32_t>(threshold >> 32)) continue;
      const Candidate one = candidate(i);
      if (one.order < threshold) continue;
      const int place = atomicAdd(&listed, 1);
      if (place < kListed) list[place] = one;
    }
    __syncthreads();
    const int found = listed;
    auto write = [&](int place, const Candidate& one) {
      const long long to = static_cast<long long>(request) * p.keep + place;
      p.out_scores[to] = static_cast<float>(value_of(one.order));
      p.out_parents[to] = request * p.beams + static_cast<int>(one.beam);
      p.out_tokens[to] = static_cast<int>(one.token);
    };
    if (found <= kListed) {
      for (int i = threadIdx.x; i < found; i += kJoinThreads) {
        const Candidate one = list[i];
        int place = 0;
#pragma unroll 4
        for (int j = 0; j < found; ++j) place += before(list[j], one) ? 1 : 0;
        if (place >= p.keep) continue;
        write(place, one);
        if (round > 0) continue;
        // (-inf and NaN are close to nothing. Beams whose sums are equal may yet differ: roundings make one number of several.)
        const double value = value_of(one.order);
#pragma unroll 1
        for (int j = 0; j < found; ++j) {
          const Candidate other = list[j];
          if (other.beam != one.beam && fabs(value_of(other.order) - value) < p.near && (state[one.beam] == kGoesOn || state[other.beam] == kGoesOn))
            near = again[one.beam] = again[other.beam] = 1;
        }
      }
    } else {
      // Very many values that are equal or close. Where they are several beams', these beams' sums are taken again first.
      if (round == 0) {
#pragma unroll 1
        for (int i = threadIdx.x; i < all; i += kJoinThreads) {
          const Candidate one = candidate(i);
          if (one.order >= threshold && fabs(value_of(one.order)) < static_cast<double>(INFINITY)) again[one.beam] = 1;
        }
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < p.beams && again[threadIdx.x] && state[threadIdx.x] == kGoesOn) {
          for (int beam = 0; beam < p.beams; ++beam)
            if (again[beam] && beam != static_cast<int>(threadIdx.x)) near = 1;
        }
        __syncthreads();
      }
      Candidate last = {~0ull, 0, 0};
#pragma unroll 1
      for (int n = 0; n < p.keep && (round > 0 || near == 0); ++n) {
        Candidate best = {0, 0, 0};
#pragma unroll 1
        for (int i = threadIdx.x; i < all; i += kJoinThreads) {
          const Candidate one = candidate(i);
          if (one.order != 0 && (n == 0 || before(last, one)) && (best.order == 0 || before(one, best))) best = one;
        }
#pragma unroll
        for (int offset = 16; offset > 0; offset /= 2) {
          const Candidate other = {__shfl_xor_sync(0xffffffffu, best.order, offset), __shfl_xor_sync(0xffffffffu, best.beam, offset),
                                   __shfl_xor_sync(0xffffffffu, best.token, offset)};
          if (other.order != 0 && (best.order == 0 || before(other, best))) best = other;
        }
        if (lane == 0) warp_best[warp] = best;
        __syncthreads();
#pragma unroll 1
        for (int w = 0; w < kJoinWarps; ++w) {
          const Candidate other = warp_best[w];
          if (other.order != 0 && (best.order == 0 || before(other, best))) best = other;
        }
        if (threadIdx.x == 0) write(n, best);
        last = best;
        __syncthreads();
      }
    }
    __syncthreads();
    if (round > 0 || near == 0) break;
    // Sums of the beams that are close, in f64, over the largest logit (alike beams have the same sum then), which the parts know.
    for (int beam = 0; beam < p.beams; ++beam) {
      if (!again[beam] || state[beam] != kGoesOn) continue;
      const T* const from = static_cast<const T*>(p.logits) + request * p.request_stride + beam * p.beam_stride;
      const unsigned long long* const best = p.keys + keys0 + static_cast<long long>(beam) * (slots - 1);
      uint32_t top = 0;
#pragma unroll 1
      for (int part = lane; part < p.parts; part += 32) top = max(top, static_cast<uint32_t>(best[part * p.keep] >> 32));
      const double shift = from_ordered(__reduce_max_sync(0xffffffffu, top));
      double sum = 0.0;
      constexpr int kLoads = 16;                                // of a thread, under way together
#pragma unroll 1
      for (int t0 = threadIdx.x; t0 < p.vocab; t0 += kLoads * kJoinThreads) {
        float x[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) x[u] = t0 + u * kJoinThreads < p.vocab ? to_compute(from[t0 + u * kJoinThreads]) : -INFINITY;
#pragma unroll
        for (int u = 0; u < kLoads; ++u) sum += exp(static_cast<double>(x[u]) - shift);
      }
#pragma unroll
      for (int offset = 16; offset > 0; offset /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
      if (lane == 0) warp_sum[warp] = sum;
      __syncthreads();
      if (threadIdx.x == 0) {
        double whole = 0.0;
#pragma unroll 1
        for (int w = 0; w < kJoinWarps; ++w) whole += warp_sum[w];
        logarithm[beam] = shift + log(whole);
      }
      __syncthreads();
    }
  }
}

struct SelectPlan {
  int parts, chunk;
  size_t sums_bytes, keys_bytes;
};
// Candidates of two beams whose values are closer than this may be in either order: both beams' logarithms are off by half of it at most. A logit at a
// distance d from what the sum stands at has its exponent off by 1.33e-7 d (subtraction and product by 2^-24 each, log2 e by 2^-26), its exponential by 2^-22 and
// the sums in f32 by 8 * 2^-24, 7.2e-7 together. With their exponentials as weights, distances average at ln N - 1 at most: N logits at d below the largest
// weigh N e^-d / (1 + N e^-d), which times d is W(N / e) <= ln(N / e) at its largest (W: Lambert's function). Above, none is farther than kStand.
double near_values(int64_t vocab) { return 2.0 * (1.33e-7 * std::fmax(std::log(static_cast<double>(vocab)) - 1.0, kStand + 0.5) + 7.2e-7); }

// As many parts of a row as there are CTAs at once for it, and one at least. (512 rows of 128000 in one part 49 us, in two 80.)
SelectPlan plan_select(int64_t rows, int64_t vocab, int64_t keep, int64_t bytes) {
  SelectPlan plan = {};
  const int64_t chunk = kChunkBytes / bytes - 8, chunks = (vocab + chunk - 1) / chunk;      // (a row may begin inside a vector)
  const int64_t parts = kSelectCtas / rows < 1 ? 1 : kSelectCtas / rows < chunks ? kSelectCtas / rows : chunks;
  plan.chunk = static_cast<int>(((vocab + parts - 1) / parts + 7) / 8 * 8);
  plan.parts = static_cast<int>((vocab + plan.chunk - 1) / plan.chunk);
  plan.keys_bytes = static_cast<size_t>(rows) * plan.parts * keep * sizeof(unsigned long long);
  plan.sums_bytes = static_cast<size_t>(rows) * plan.parts * sizeof(double2);
  return plan;
}

bool select_takes(int64_t requests, int64_t beams, int64_t vocab, int64_t keep) {
  return requests > 0 && beams > 0 && vocab > 0 && keep > 0 && beams <= kMostBeams && keep <= kMostKept && vocab < (1LL << 24) && requests * beams < 65536;
}

}  // namespace
}  // namespace tq

extern "C" tq_status tq_beam_select_workspace_bytes(tq_dtype dtype, int64_t requests, int64_t beams, int64_t vocab, int64_t keep, size_t* bytes) {
  TQ_REQUIRE(bytes != nullptr, TQ_INVALID_ARGUMENT, "null out-pointer");
  *bytes = 0;
  if (tq::dtype_size(dtype) == 0 || requests > (1LL << 31) || !tq::select_takes(requests, beams, vocab, keep)) return TQ_OK;
  const tq::SelectPlan plan = tq::plan_select(requests * beams, vocab, keep, tq::dtype_size(dtype));
  *bytes = plan.sums_bytes + plan.keys_bytes;
  return TQ_OK;
}

extern "C" tq_status tq_beam_select_launch(tq_dtype dtype, const void* logits, const float* scores, const uint8_t* finished, float* out_scores,
                                           int32_t* out_parents, int32_t* out_tokens, int64_t requests, int64_t beams, int64_t vocab, int64_t keep,
                                           int64_t end, int64_t request_stride, int64_t beam_stride, void* workspace, size_t workspace_bytes, int32_t device,
                                           void* stream) {
  if (tq::recording()) {
    return tq::record([=](int32_t d, void* s) {
      return tq_beam_select_launch(dtype, logits, scores, finished, out_scores, out_parents, out_tokens, requests, beams, vocab, keep, end, request_stride,
                                   beam_stride, workspace, workspace_bytes, d, s);
    });
  }
  TQ_REQUIRE(dtype == TQ_F32 || dtype == TQ_F16 || dtype == TQ_BF16, TQ_UNSUPPORTED, "beams are selected by f32, f16 or bf16 logits, not %s", tq::dtype_name(dtype));
  TQ_REQUIRE(requests >= 0 && beams >= 0 && vocab >= 0 && keep >= 0, TQ_INVALID_ARGUMENT, "negative extent in requests=%lld beams=%lld vocab=%lld keep=%lld",
             (long long)requests, (long long)beams, (long long)vocab, (long long)keep);
  if (requests == 0 || keep == 0) return TQ_OK;
  TQ_REQUIRE(vocab < (1LL << 24) && beams <= tq::kMostBeams && keep <= tq::kMostKept && requests < 65536 && requests * beams < 65536, TQ_UNSUPPORTED,
             "there is no selection of %lld from %lld x %lld beams by %lld tokens: 128 of 128 beams a request, 65535 beams in all and 2^24 - 1 tokens at most",
             (long long)keep, (long long)requests, (long long)beams, (long long)vocab);
  TQ_REQUIRE(keep <= beams * vocab, TQ_INVALID_ARGUMENT, "%lld of %lld beams by %lld tokens cannot be kept", (long long)keep, (long long)beams, (long long)vocab);
  TQ_REQUIRE(logits != nullptr && scores != nullptr && out_scores != nullptr && out_parents != nullptr && out_tokens != nullptr, TQ_INVALID_ARGUMENT,
             "null operand or result");
  TQ_REQUIRE(finished == nullptr || (end >= 0 && end < vocab), TQ_INVALID_ARGUMENT, "there is no token %lld among %lld to end with", (long long)end, (long long)vocab);
  TQ_REQUIRE(request_stride >= 0 && beam_stride >= 0 && tq::aligned_to(logits, tq::dtype_size(dtype)) && tq::aligned_to(scores, 4), TQ_UNSUPPORTED,
             "logits have no negative strides and are aligned to their type");
  const tq::SelectPlan plan = tq::plan_select(requests * beams, vocab, keep, tq::dtype_size(dtype));
  TQ_REQUIRE(workspace != nullptr && workspace_bytes >= plan.sums_bytes + plan.keys_bytes && tq::aligned_to(workspace, 16), TQ_INVALID_ARGUMENT,
             "this selection needs %zu bytes of workspace, 16-byte aligned, and was given %zu", plan.sums_bytes + plan.keys_bytes, workspace_bytes);
  tq::DeviceScope device_scope(device);
  if (tq_status s = device_scope.status()) return s;
  tq::SelectParams p = {};
  p.logits = logits;
  p.request_stride = request_stride;
  p.beam_stride = beam_stride;
  p.scores = scores;
  p.finished = finished;
  p.beams = static_cast<int>(beams);
  p.vocab = static_cast<int>(vocab);
  p.keep = static_cast<int>(keep);
  p.parts = plan.parts;
  p.chunk = plan.chunk;
  p.end = static_cast<int>(end);
  p.near = tq::near_values(vocab);
  p.sums = static_cast<double2*>(workspace);
  p.keys = reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + plan.sums_bytes);
  p.out_scores = out_scores;
  p.out_parents = out_parents;
  p.out_tokens = out_tokens;
  const cudaStream_t cuda_stream = static_cast<cudaStream_t>(stream);
  const auto held = tq::hold_scratch(workspace);
  auto go = [&](auto type) -> tq_status {
    using T = decltype(type);
    const dim3 grid(static_cast<unsigned>(plan.parts), static_cast<unsigned>(requests * beams));
    TQ_CUDA(tq::launch_overlapped(tq::beam_parts_kernel<T>, grid, tq::kSelectThreads, 0, cuda_stream, p));
    if (tq_status s = tq::check_launch("beam_parts_kernel")) return s;
    TQ_CUDA(tq::launch_overlapped(tq::beam_join_kernel<T>, dim3(static_cast<unsigned>(requests)), tq::kJoinThreads, 0, cuda_stream, p));
    return tq::check_launch("beam_join_kernel");
  };
  return dtype == TQ_F32 ? go(0.f) : dtype == TQ_F16 ? go(__half{}) : go(__nv_bfloat16{});
}
