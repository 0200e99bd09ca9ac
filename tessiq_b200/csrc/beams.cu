// Beam search's selection, for sm_100a: of all beams and tokens of a request the best `keep`, by
//
//   value(b, t) = score_b + x[b, t] - log sum_u exp(x[b, u])       x: logits; in falling order, ties to the lower beam, then the lower token
//
// Within a beam the order is that of the logits, so a beam's candidates are its `keep` largest logits, and the logarithm of its sum is needed to compare
// beams alone. Bound: HBM (each logit is read once).
//
// First kernel: a CTA takes up to 8184 logits of a beam, into registers: their maximum and sum of exponentials, and their `keep` largest. Every warp's
// r-th largest thread maximum, r = keep / warps, is a bound below which nothing is needed (warps * r threads have something at or above it); what is
// at or above the lowest of these bounds goes to a list, a few times `keep` long, and its members' places are counted against each other. A list that
// overflows (very many equal logits, a mask of -inf) is answered by `keep` rounds of the CTA's maximum over what is still in registers.
// Second kernel: a CTA a request joins the parts: sums, values in f64, and the same two steps over all its candidates.
//
// Precision: sums of exponentials in f32 a thread (32 of them), then f64: a logarithm is off by 1e-7 or so. Values of neighbours are as close as that
// now and then, so candidates of two beams within kNear of each other have their beams' sums taken again, in f64 throughout. Ties are then ties.
#include <cmath>
#include <type_traits>

#include "common.h"
#include "keyed.h"
#include "tcgen05.h"

namespace tq {
namespace {

constexpr int kSelectThreads = 256, kSelectWarps = kSelectThreads / 32;
constexpr int kEach = 32;                                   // logits of a thread
constexpr int kChunk = kSelectThreads * kEach - 8;          // of a CTA: a row may begin inside a vector of 16 bytes
constexpr int kListed = 1024;                               // candidates on chip
constexpr int kJoinThreads = 512, kJoinWarps = kJoinThreads / 32;
constexpr int kMostBeams = 128, kMostKept = 128;
constexpr float kLog2E = 1.4426950408889634f;

struct SelectParams {
  const void* logits;
  long long request_stride, beam_stride;                    // elements
  const float* scores;                                      // [requests, beams]
  const uint8_t* finished;                                  // the same, or null
  int beams, vocab, keep, parts, chunk, end;
  float2* sums;                                             // [rows, parts]: the exponent the sum stands at, in log2, and the sum
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

template <typename T>
__global__ void __launch_bounds__(kSelectThreads, 4) beam_parts_kernel(const __grid_constant__ SelectParams p) {
  constexpr int kVec = 16 / sizeof(T), kVecs = kEach / kVec;
  __shared__ uint32_t warp_most[kSelectWarps], warp_bound[kSelectWarps];
  __shared__ double warp_sum[kSelectWarps];
  __shared__ unsigned long long list[kListed], warp_key[kSelectWarps];
  __shared__ int listed;
  const int part = static_cast<int>(blockIdx.x), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.y;
  const int request = static_cast<int>(row / p.beams), beam = static_cast<int>(row % p.beams);
  if (threadIdx.x == 0) listed = 0;
  wait_for_earlier();
  if (p.finished != nullptr && p.finished[row]) return;     // (its one candidate is made below)
  const int first = part * p.chunk, count = min(p.chunk, p.vocab - first);
  const T* const from = static_cast<const T*>(p.logits) + request * p.request_stride + beam * p.beam_stride + first;
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(from) & 15) / sizeof(T));
  const T* const whole = from - skew;

  // A thread's vectors; what lies before or behind the part is -inf.
  uint4 word[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int at = (i * kSelectThreads + static_cast<int>(threadIdx.x)) * kVec - skew;      // of its first element, in the part
    if (at >= 0 && at + kVec <= count) {
      const Vec<T, kVec> vector = load_stream<T, kVec>(whole + at + skew);
      word[i] = *reinterpret_cast<const uint4*>(&vector);
    } else {
      Vec<T, kVec> vector;
#pragma unroll
      for (int c = 0; c < kVec; ++c) vector.v[c] = at + c >= 0 && at + c < count ? from[at + c] : from_compute<T, float>(-INFINITY);
      word[i] = *reinterpret_cast<const uint4*>(&vector);
    }
  }
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    float x[kVec];
    widen<T>(word[i], x);
#pragma unroll
    for (int c = 0; c < kVec; ++c) most = fmaxf(most, x[c]);
  }
  // Warps of which every thread has logits: of a part of 2048 or more all.
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
  const float threshold = least <= 0x007fffffu ? -INFINITY : from_ordered(least);
  most = from_ordered(top);
  const float shift = most == -INFINITY ? 0.f : most * kLog2E;      // (rounded, and the sum stands at what it was rounded to)
  float sum0 = 0.f, sum1 = 0.f;
  auto key_of = [&](float x, int at) { return static_cast<unsigned long long>(ordered(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(first + at)); };
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    float x[kVec];
    widen<T>(word[i], x);
    const int at = (i * kSelectThreads + static_cast<int>(threadIdx.x)) * kVec - skew;
    bool any = false;
#pragma unroll
    for (int c = 0; c < kVec; c += 2) {
      sum0 += exp2_ftz(fmaf(x[c], kLog2E, -shift));
      sum1 += exp2_ftz(fmaf(x[c + 1], kLog2E, -shift));
      any |= x[c] >= threshold || x[c + 1] >= threshold;
    }
    if (any) {
#pragma unroll
      for (int c = 0; c < kVec; ++c) {
        if (x[c] >= threshold && at + c >= 0 && at + c < count) {
          const int place = atomicAdd(&listed, 1);
          if (place < kListed) list[place] = key_of(x[c], at + c);
        }
      }
    }
  }
  double sum = static_cast<double>(sum0) + static_cast<double>(sum1);
#pragma unroll
  for (int offset = 16; offset > 0; offset /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
  if (lane == 0) warp_sum[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kSelectWarps; ++w) all += warp_sum[w];
    p.sums[row * p.parts + part] = make_float2(shift, static_cast<float>(all));
  }
  unsigned long long* const to = p.keys + (row * p.parts + part) * p.keep;
  const int found = listed;
  if (found <= kListed) {
    for (int i = threadIdx.x; i < found; i += kSelectThreads) {
      const unsigned long long key = list[i];
      int place = 0;
      for (int j = 0; j < found; ++j) place += list[j] > key ? 1 : 0;
      if (place < p.keep) to[place] = key;
    }
    for (int i = found + threadIdx.x; i < p.keep; i += kSelectThreads) to[i] = 0;
  } else {
    unsigned long long before = ~0ull;
    for (int n = 0; n < p.keep; ++n) {
      unsigned long long best = 0;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        float x[kVec];
        widen<T>(word[i], x);
        const int at = (i * kSelectThreads + static_cast<int>(threadIdx.x)) * kVec - skew;
#pragma unroll
        for (int c = 0; c < kVec; ++c) {
          const unsigned long long key = at + c >= 0 && at + c < count ? key_of(x[c], at + c) : 0;
          if (key < before && key > best) best = key;
        }
      }
#pragma unroll
      for (int offset = 16; offset > 0; offset /= 2) best = max(best, __shfl_xor_sync(0xffffffffu, best, offset));
      if (lane == 0) warp_key[warp] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kSelectWarps; ++w) best = max(best, warp_key[w]);
      if (threadIdx.x == 0) to[n] = best;
      before = best;
      __syncthreads();
    }
  }
}

enum BeamState { kGoesOn = 0, kFinished, kNothing, kNoNumber };      // kNothing: every logit, or the score, is -inf; kNoNumber: NaN, or +inf

// Candidates whose values lie closer than this, times 1 + the larger magnitude of a logit's log2 / 16: sums of two beams may be off by as much.
constexpr double kNear = 1e-6;

struct Candidate {
  unsigned long long order;      // of the value; 0: none
  uint32_t beam, token;
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
  return a.order != b.order ? a.order > b.order : a.beam != b.beam ? a.beam < b.beam : a.token < b.token;
}

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) beam_join_kernel(const __grid_constant__ SelectParams p) {
  __shared__ double logarithm[kMostBeams], score_of[kMostBeams];
  __shared__ uint8_t state[kMostBeams], again[kMostBeams];
  __shared__ Candidate list[kListed], warp_best[kJoinWarps];
  __shared__ uint32_t warp_bound[kJoinWarps];
  __shared__ double warp_sum[kJoinWarps];
  __shared__ float largest_shift;
  __shared__ int listed, near;
  const int request = static_cast<int>(blockIdx.x), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  wait_for_earlier();
  if (threadIdx.x == 0) {
    largest_shift = 0.f;
    near = 0;
  }
  __syncthreads();
  for (int beam = warp; beam < p.beams; beam += kJoinWarps) {
    const long long row = static_cast<long long>(request) * p.beams + beam;
    const float score = p.scores[row];
    const bool finished = p.finished != nullptr && p.finished[row];
    float at = -INFINITY;
    double sum = 0.0;
    if (!finished) {
      for (int part = lane; part < p.parts; part += 32) {
        const float2 one = p.sums[row * p.parts + part];
        // (a part of -inf alone has the sum 0 at 0; of a NaN its sum is one)
        if (one.y == 0.f) continue;
        const float both = fmaxf(at, one.x);
        sum = sum * (at == both ? 1.0 : exp2(static_cast<double>(at) - both)) + one.y * (one.x == both ? 1.0 : exp2(static_cast<double>(one.x) - both));
        at = both;
      }
#pragma unroll
      for (int offset = 16; offset > 0; offset /= 2) {
        const float other = __shfl_xor_sync(0xffffffffu, at, offset), both = fmaxf(at, other);
        const double theirs = __shfl_xor_sync(0xffffffffu, sum, offset);
        sum = sum * (at == both ? 1.0 : exp2(static_cast<double>(at) - both)) + theirs * (other == both ? 1.0 : exp2(static_cast<double>(other) - both));
        at = both;
      }
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
      logarithm[beam] = now == kGoesOn ? (static_cast<double>(at) + log2(sum)) * 0.6931471805599453 : 0.0;
      if (now == kGoesOn) atomicMax(reinterpret_cast<int*>(&largest_shift), __float_as_int(fabsf(at)));
    }
  }
  __syncthreads();
  const int most_tokens = min(p.keep, p.vocab);
  const int slots = p.parts * p.keep + 1, all = p.beams * slots;      // of a beam, and of the request
  const double close = kNear * (1.0 + static_cast<double>(largest_shift) / 16.0);
  auto candidate = [&](int i) {
    const int beam = i / slots, c = i % slots;
    Candidate one = {0, static_cast<uint32_t>(beam), static_cast<uint32_t>(c)};
    if (state[beam] == kGoesOn) {
      if (c == slots - 1) return one;
      const unsigned long long key = p.keys[(static_cast<long long>(request) * p.beams + beam) * p.parts * p.keep + c];
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
    // A bound that `keep` candidates reach, from the order's upper half; lowered by what is close.
    uint32_t mine = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < all; i += kJoinThreads) mine = max(mine, static_cast<uint32_t>(candidate(i).order >> 32));
    const int full = min(all / 32, kJoinWarps), nth = full == 0 ? 33 : (p.keep + full - 1) / full;
    const uint32_t bound = nth > 32 ? 0 : warp_nth(mine, nth);
    if (lane == 0) warp_bound[warp] = bound;
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    uint32_t least = 0xffffffffu;
    for (int w = 0; w < full; ++w) least = min(least, warp_bound[w]);
    if (nth > 32) least = 0;
    unsigned long long threshold = static_cast<unsigned long long>(least) << 32;
    if (round == 0 && least != 0 && least != 0xffffffffu) {
      const double lower = value_of(threshold) - 2.0 * close;
      if (lower == lower) threshold = ordered(lower);      // (of -inf: -inf)
    }
    if (threshold == 0) threshold = 1;
#pragma unroll 4
    for (int i = threadIdx.x; i < all; i += kJoinThreads) {
      const Candidate one = candidate(i);
      if (one.order >= threshold) {
        const int place = atomicAdd(&listed, 1);
        if (place < kListed) list[place] = one;
      }
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
        const double value = value_of(one.order);
        int place = 0;
        for (int j = 0; j < found; ++j) place += before(list[j], one) ? 1 : 0;
        if (place >= p.keep) continue;
        write(place, one);
        if (round > 0) continue;
        for (int j = 0; j < found; ++j) {      // (-inf and NaN are close to nothing; beams of one sum and one score compare as their logits do)
          const Candidate other = list[j];
          if (other.beam != one.beam && fabs(value_of(other.order) - value) < close &&
              !(logarithm[one.beam] == logarithm[other.beam] && score_of[one.beam] == score_of[other.beam]))
            near = again[one.beam] = again[other.beam] = 1;
        }
      }
    } else {
      // (very many equal values, of which only the order of beams and tokens tells)
      Candidate last = {~0ull, 0, 0};
      for (int n = 0; n < p.keep; ++n) {
        Candidate best = {0, 0, 0};
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
    // Sums of the beams that are close, in f64.
    for (int beam = 0; beam < p.beams; ++beam) {
      if (!again[beam] || state[beam] != kGoesOn) continue;
      const T* const from = static_cast<const T*>(p.logits) + request * p.request_stride + beam * p.beam_stride;
      double sum = 0.0;
      const double shift = logarithm[beam];
      for (int t = threadIdx.x; t < p.vocab; t += kJoinThreads) sum += exp(static_cast<double>(to_compute(from[t])) - shift);
#pragma unroll
      for (int offset = 16; offset > 0; offset /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
      if (lane == 0) warp_sum[warp] = sum;
      __syncthreads();
      if (threadIdx.x == 0) {
        double whole = 0.0;
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
SelectPlan plan_select(int64_t rows, int64_t vocab, int64_t keep) {
  SelectPlan plan = {};
  const int64_t parts = (vocab + kChunk - 1) / kChunk;
  plan.chunk = static_cast<int>(((vocab + parts - 1) / parts + 7) / 8 * 8);
  plan.parts = static_cast<int>((vocab + plan.chunk - 1) / plan.chunk);
  plan.keys_bytes = static_cast<size_t>(rows) * plan.parts * keep * sizeof(unsigned long long);
  plan.sums_bytes = static_cast<size_t>(rows) * plan.parts * sizeof(float2);
  return plan;
}

bool select_takes(int64_t requests, int64_t beams, int64_t vocab, int64_t keep) {
  return requests > 0 && beams > 0 && vocab > 0 && keep > 0 && beams <= kMostBeams && keep <= kMostKept && vocab < (1LL << 24) && requests * beams < 65536;
}

}  // namespace
}  // namespace tq

extern "C" tq_status tq_beam_select_workspace_bytes(int64_t requests, int64_t beams, int64_t vocab, int64_t keep, size_t* bytes) {
  TQ_REQUIRE(bytes != nullptr, TQ_INVALID_ARGUMENT, "null out-pointer");
  *bytes = 0;
  if (requests > (1LL << 31) || !tq::select_takes(requests, beams, vocab, keep)) return TQ_OK;
  const tq::SelectPlan plan = tq::plan_select(requests * beams, vocab, keep);
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
  const tq::SelectPlan plan = tq::plan_select(requests * beams, vocab, keep);
  TQ_REQUIRE(workspace != nullptr && workspace_bytes >= plan.sums_bytes + plan.keys_bytes && tq::aligned_to(workspace, 8), TQ_INVALID_ARGUMENT,
             "this selection needs %zu bytes of workspace, 8-byte aligned, and was given %zu", plan.sums_bytes + plan.keys_bytes, workspace_bytes);
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
  p.keys = static_cast<unsigned long long*>(workspace);
  p.sums = reinterpret_cast<float2*>(static_cast<char*>(workspace) + plan.keys_bytes);
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
