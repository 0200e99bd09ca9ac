// Fused attention on the 5th-generation tensor cores (tcgen05), for sm_100a.
//
//   out[b,h,i,:] = sum_j softmax_j(scale * q[b,h,i,:] . k[b,h,j,:]) v[b,h,j,:]     (j <= i when causal)
//
// bf16 or f16 operands, heads of up to 128 elements, f32 scores and sums, one rounding of the result. The
// score matrix never leaves the SM: one CTA owns 128 query rows of one head and walks the keys 64 or 128 at a
// time (choose_attention_form) with a row reference point and row sum (the online form of softmax).
//
//   warps 0..3          softmax, one thread per query row: tcgen05.ld of the row's f32 scores of a step (held in
//                       registers for both the maximum and the exponentials), ex2, row sum; the
//                       probabilities go back into tensor memory with tcgen05.st as packed bf16/f16 pairs —
//                       the A operand of the second product. The result accumulates in tensor memory
//                       across the steps and is read once, at the end.
//   warp 4, one lane    producer: TMA loads (128-byte swizzle) of the query tile once, then one key tile and
//                       one value tile per step into two rings; the first filling leaves before the CTA's
//                       set-up barrier.
//   warp 5, one lane    issuer: S = Q K^T (128 x keys x head, both operands K-major in shared memory) and
//                       O = P V (128 x head x keys, P from tensor memory, V consumed MN-major exactly as it
//                       lies in memory). The scores of step j + 1 are computed while the softmax warps work
//                       on step j, which hand the columns back as soon as they have them in registers.
//
// softmax is exp(s - m) / sum exp(s - m) for ANY m, so a row keeps the maximum of its first 128 keys
// as its reference point and moves it only when a later tile rises more than 2^8 above it — then,
// and only then, the row's sum and its accumulators in tensor memory are rescaled (a warp-wide
// slow path, rare on real data). Without that, nothing is read back per step: the second product
// accumulates O += P V in place. Probabilities are at most 2^8, well inside bf16 and f16. (With 64 keys a step the second
// tile's scores are computed ahead for it, into the result's columns: from the first 64 keys alone a row's largest
// probability was exactly 1 less often, and the error against 64 bits 1 to 3 % larger.)
//
// A few queries (FEW) leave three of the four softmax warps without a row and the tensor cores idle, so their probabilities
// are taken as two 16-bit operands, the rounded value and what rounding took off: the result is as exact as the
// streaming kernel's, whose probabilities are never rounded (error against 64 bits 1.65e-3 in bf16, all of it the result's
// rounding; 2.3e-3 with one operand).
//
// What bounds it: a step of 64 keys of one CTA is a chain (scores seen, tcgen05.ld, maximum, ex2, tcgen05.st, signal) of about
// 1 500 cycles of which the special-function unit works 512, so an SM needs several chains. Three CTAs of one
// softmax warp per scheduler each (two for heads above 64) keep the unit busy 65 % of the time, and one CTA's
// start and end run under the others' steps; two CTAs with 128 keys a step pay a step's hand-overs half as often and reach
// as much. One CTA an SM with two groups of 128 rows and 128-key steps, as it
// was once, spent 5 000 cycles on every start: 64 x 12 heads, 1024 tokens of 64 causal 256 us, now 229, no mask 377, now 323,
// 4 x 12 x 4096 no mask 332, now 296; 64 x 6 heads of 128, whose second group had idled, 235, now 175.
// Measured beside it (before the reference point took 128 keys, when the first two of those were 225 and 320): two CTAs with two groups each and the probabilities over the scores (four chains, each
// with both products inside it) 216 / 307 / 312 / 205; one exponential in four, or in sixteen, as a polynomial of
// degree 5 on the FMA pipes 328 and 322 instead of 312; scalar instead of two-element FMA and add 311 - 318; the
// row sum after the signal 333; skipping the rows past the diagonal of a whole warp: no change.
//
// The softmax warps run with 120 registers per thread where three CTAs share an SM, 200 where two do, the other four with 40 and 56
// (setmaxnreg). Q, K, V and the result are addressed through (batch, head, token) strides, so the three slices
// of a fused QKV projection are read in place and the result is written directly in [batch, token, head, head_dim]
// order: none of the four packing copies around `bmm -> where -> softmax -> bmm` remains.
//
// Every wait is bounded; a wait that gives up sets the device status word (tq_status_poll) and the
// CTA leaves through the normal teardown, freeing its tensor memory. No load uses multicast.
//
// The reference has no attention kernel: its compiler emits bmm (csrc/tessiq/codegen/gemm.cpp:100-175),
// a host-side mask, the softmax custom op (csrc/custom_ops/softmax/softmax.cu:19-61) and a second bmm
// for the pattern in tests/python/test_models.py:64-67, with the [batch, heads, T, T] scores in memory.
#include <cuda.h>

#include <cmath>
#include <mutex>
#include <type_traits>

#include "common.h"
#include "keyed.h"
#include "tcgen05.h"

namespace tq {
namespace {

constexpr int kHeadDim = 64;
constexpr int kRows = 128;            // query rows per CTA
constexpr int kAttnThreads = 256;     // four softmax warps; producer and issuer in a second group of four
constexpr uint32_t kQueryBytes = kRows * kHeadDim * 2;       // 16 KiB: 128 rows of 64 elements, one TMA box, one swizzled operand tile
// D: heads of up to 64 elements, or of up to 128 (two 64-wide sub-tiles side by side in every tile). KEYS: keys per step. FEW:
// the form for a few queries, whose probabilities take two operands (below). Shared memory: the query tile, the key
// ring, the value ring, the barriers. Tensor memory, f32 columns: scores (KEYS), packed probabilities (KEYS / 2, twice with FEW),
// result (D). An allocation is a power of two, so heads of 64 with 64 keys a step take two (scores and result,
// probabilities: 160 columns, and three CTAs have 480 of the 512) and the other forms a single one.
template <int D, int KEYS, bool FEW>
struct AttnLayout {
  static constexpr int kSubTiles = D / kHeadDim;
  static constexpr bool kTwoAllocations = D == kHeadDim && KEYS == 64 && !FEW;
  static constexpr int kCtasPerSm = kTwoAllocations ? 3 : KEYS == 64 || (D == kHeadDim && !FEW) ? 2 : 1;
  static constexpr int kRing = D == kHeadDim && KEYS == 64 ? 3 : 2;          // stages of the key ring and of the value ring
  static constexpr uint32_t kSubTileBytes = KEYS * kHeadDim * 2;            // 8 or 16 KiB: 64 elements of a tile's keys or values
  static constexpr uint32_t kTileBytes = kSubTiles * kSubTileBytes;
  static constexpr uint32_t kOffsetK = kSubTiles * kQueryBytes;
  static constexpr uint32_t kOffsetV = kOffsetK + kRing * kTileBytes;
  static constexpr uint32_t kOffsetBarriers = kOffsetV + kRing * kTileBytes;
  static constexpr size_t kSmemBytes = 1024 + kOffsetBarriers + 256;
  static constexpr uint32_t kColumnP = KEYS, kColumnO = kTwoAllocations ? 64 : D == kHeadDim && !FEW ? KEYS + KEYS / 2 : 2 * KEYS;
  static constexpr uint32_t kTmemColumns = kTwoAllocations ? 128 : kColumnO + D <= 256 ? 256 : 512;      // scores from column 0 on
  static_assert(kTwoAllocations || (kColumnP + (FEW ? KEYS : KEYS / 2) <= kColumnO && kColumnO + D <= kTmemColumns), "the columns overlap");
  static_assert(kTwoAllocations ? kCtasPerSm * 160 <= 512 : kCtasPerSm * kTmemColumns <= 512, "more CTAs an SM than it has tensor memory for");
  static_assert(kCtasPerSm * (kSmemBytes + 1024) <= 228 * 1024, "the staging has to fit as often as there are CTAs an SM");
  // setmaxnreg moves registers inside the CTA's own allocation: what the second group of four warps gives up is
  // at least what the softmax warps take. An increase beyond what was released would wait for ever. (A CTA that has
  // its SM to itself has registers enough from the start.)
  static constexpr int kLaunchRegisters = (65536 / kCtasPerSm / kAttnThreads) / 8 * 8;
  static constexpr int kSoftmaxRegisters = kCtasPerSm == 3 ? 120 : 200, kOtherRegisters = kCtasPerSm == 3 ? 40 : 56;
  static constexpr bool kMovesRegisters = kCtasPerSm > 1;
  static_assert(!kMovesRegisters || 128 * (kSoftmaxRegisters - kLaunchRegisters) <= 128 * (kLaunchRegisters - kOtherRegisters),
                "the softmax warps would wait for registers nobody releases");
};
constexpr uint32_t kTmemColumnsP = 32;       // of the second allocation
constexpr float kSlack = 8.f;                // a row's reference point moves when a tile's maximum is more than 2^kSlack above it

enum AttnWait { kWaitQ = 201, kWaitKeyEmpty = 202, kWaitValueEmpty = 203, kWaitKeyFull = 204, kWaitValueFull = 205,
                kWaitScores = 206, kWaitProbabilities = 207, kWaitPartial = 208, kWaitBufferFree = 209 };

struct AttnParams {
  int batch, heads, q_tokens, k_tokens;
  int head_dim;                    // 8, 16, ... 128: narrower heads ride in tiles of 64 or 128 whose other columns TMA fills with zeros
  int q_blocks;                    // CTAs per head
  int causal;
  float scale_log2;                // scale * log2(e)
  void* out;
  long long out_batch, out_head, out_token;   // element strides
  WaitStatus status;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// f32 accumulator, A and B of type T, M = 128, N = `n`; B MN-major when `b_mn`.
template <typename T>
__host__ __device__ constexpr uint32_t attn_instruction_descriptor(int n, bool b_mn) {
  constexpr uint32_t format = std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;
  return (1u << 4) | (format << 7) | (format << 10) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kRows >> 4) << 24);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float low, float high) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const __nv_bfloat162 pair = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&pair);
  } else {
    const __half2 pair = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&pair);
  }
}

// What rounding took off a pair of probabilities, rounded itself.
template <typename T>
__device__ __forceinline__ uint32_t pack_rest(uint32_t rounded, float2 exact) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    return pack_pair<T>(exact.x - __uint_as_float(rounded << 16), exact.y - __uint_as_float(rounded & 0xffff0000u));
  } else {
    const float2 wide = __half22float2(*reinterpret_cast<const __half2*>(&rounded));
    return pack_pair<T>(exact.x - wide.x, exact.y - wide.y);
  }
}

template <typename T, int D, int KEYS, bool FEW>
__global__ void __launch_bounds__(kAttnThreads, AttnLayout<D, KEYS, FEW>::kCtasPerSm)
attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const AttnParams p) {
  using L = AttnLayout<D, KEYS, FEW>;
  constexpr int kKeys = KEYS;
  constexpr bool kAhead = KEYS < 128;      // the reference point takes the second tile's scores too
  constexpr uint32_t kSubTileBytes = L::kSubTileBytes;
  constexpr int kRing = L::kRing;
  constexpr uint32_t kTileBytes = L::kTileBytes, kOffsetK = L::kOffsetK, kOffsetV = L::kOffsetV;
  constexpr uint32_t kOffsetBarriers = L::kOffsetBarriers, kColumnO = L::kColumnO;
  constexpr int kSubTiles = L::kSubTiles;
  extern __shared__ unsigned char raw_smem[];
  const uint32_t base = (smem_address(raw_smem) + 1023u) & ~1023u;
  unsigned char* aligned = raw_smem + (base - smem_address(raw_smem));
  const uint32_t barriers = base + kOffsetBarriers;
  // barrier slots, 8 bytes each
  const uint32_t q_full = barriers;
  auto k_full = [&](int s) { return barriers + 8u * (1 + s); };
  auto k_empty = [&](int s) { return barriers + 8u * (1 + kRing + s); };
  auto v_full = [&](int s) { return barriers + 8u * (1 + 2 * kRing + s); };
  auto v_empty = [&](int s) { return barriers + 8u * (1 + 3 * kRing + s); };
  const uint32_t s_full = barriers + 8u * (1 + 4 * kRing);      // the scores of a step are in tensor memory
  const uint32_t s_free = s_full + 8;                           // ... and in the softmax warps' registers
  const uint32_t p_full = s_full + 16;                          // the probabilities of a step are in tensor memory
  const uint32_t pv_done = s_full + 24;                         // ... and the second product has consumed them
  constexpr int kBarrierCount = 1 + 4 * kRing + 4;
  const uint32_t tmem_slot = barriers + 8u * kBarrierCount;
  volatile uint32_t* tmem_slot_pointer = reinterpret_cast<volatile uint32_t*>(aligned + kOffsetBarriers + 8 * kBarrierCount);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // Which rows of which head: heads in launch order, the long (late) query blocks of a head first.
  const int q_block = p.q_blocks - 1 - static_cast<int>(blockIdx.x % p.q_blocks);
  const int head_index = static_cast<int>(blockIdx.x / p.q_blocks);
  const int head = head_index % p.heads, batch = head_index / p.heads;
  const int q0 = q_block * kRows;
  const int key_tiles = (p.k_tokens + kKeys - 1) / kKeys;
  // under a causal mask only the key tiles that hold a key <= the CTA's last row; at least one step
  const int steps = p.causal ? min(key_tiles, (min(q0 + kRows, p.q_tokens) - 1) / kKeys + 1) : key_tiles;

  auto load_tile = [&](const CUtensorMap* map, uint32_t ring, uint32_t full, int j) {
    barrier_expect_tx(full, kTileBytes);
    for (int h = 0; h < kSubTiles; ++h)
      tma_load_4d(base + ring + (j % kRing) * kTileBytes + h * kSubTileBytes, map, full, h * kHeadDim, j * kKeys, head, batch);
  };

  // The producer lane sets the barriers up and fills the rings for the first time before the CTA meets: the
  // loads' latency runs under the tensor-memory allocation and the barrier.
  const int early = min(steps, kRing);
  if (warp == 4 && elect_one()) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    if (blockIdx.x == 0) p.status.begin();   // this launch's abort word starts clear
    barrier_init(q_full, 1);
    for (int s = 0; s < kRing; ++s) {
      barrier_init(k_full(s), 1);
      barrier_init(k_empty(s), 1);
      barrier_init(v_full(s), 1);
      barrier_init(v_empty(s), 1);
    }
    barrier_init(s_full, 1);
    barrier_init(pv_done, 1);
    barrier_init(p_full, kRows / 32);          // one arrival per softmax warp
    barrier_init(s_free, kRows / 32);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    barrier_expect_tx(q_full, kSubTiles * kQueryBytes);
    for (int h = 0; h < kSubTiles; ++h) tma_load_4d(base + h * kQueryBytes, &map_q, q_full, h * kHeadDim, q0, head, batch);
    for (int j = 0; j < early; ++j) load_tile(&map_k, kOffsetK, k_full(j), j);
    for (int j = 0; j < early; ++j) load_tile(&map_v, kOffsetV, v_full(j), j);
  }
  if (warp == 5) {
    if constexpr (L::kTwoAllocations) {
      tmem_alloc_more(tmem_slot, L::kTmemColumns);
      tmem_alloc(tmem_slot + 4, kTmemColumnsP);
    } else {
      tmem_alloc(tmem_slot, L::kTmemColumns);
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = tmem_slot_pointer[0];
  const uint32_t tmem_p = L::kTwoAllocations ? tmem_slot_pointer[1] : tmem_base + L::kColumnP;

  if (L::kMovesRegisters && warp >= 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kOtherRegisters));
  if (warp == 4) {
    // ---- producer: what did not fit the first filling --------------------------------------------
    if (elect_one()) {
      for (int j = early; j < steps; ++j) {
        const int s = j % kRing;
        const uint32_t phase = (j / kRing) & 1;
        if (!barrier_wait(k_empty(s), phase ^ 1, p.status, kWaitKeyEmpty)) break;
        load_tile(&map_k, kOffsetK, k_full(s), j);
        if (!barrier_wait(v_empty(s), phase ^ 1, p.status, kWaitValueEmpty)) break;
        load_tile(&map_v, kOffsetV, v_full(s), j);
      }
    }
  } else if (warp == 5) {
    // ---- issuer ----------------------------------------------------------------------------------
    if (elect_one()) {
      constexpr uint32_t idesc_s = attn_instruction_descriptor<T>(kKeys, false);
      constexpr uint32_t idesc_o = attn_instruction_descriptor<T>(kHeadDim, true);
      // Descriptors as (low, high) words: one constant high word, low words stepped by adds.
      constexpr uint32_t kHighWord = kDescriptorHigh;
      const uint32_t low_q = descriptor_low(base, 0), low_k = descriptor_low(base + kOffsetK, 0);
      const uint32_t low_v = descriptor_low(base + kOffsetV, kSubTileBytes);
      // S(i) = Q K_i^T: both operands K-major, 16 elements of K = 32 B in the swizzle row
      auto scores = [&](int i, uint32_t into) {
        const uint32_t k = low_k + (i % kRing) * (kTileBytes >> 4);
        // (a 128-wide head is two 64-wide sub-tiles side by side: the same steps in the second one)
#pragma unroll
        for (int h = 0; h < kSubTiles; ++h) {
#pragma unroll
          for (int kk = 0; kk < kHeadDim / 16; ++kk)
            mma_f16_split(into, low_q + h * (kQueryBytes >> 4) + kk * 2, kHighWord, k + h * (kSubTileBytes >> 4) + kk * 2, kHighWord, idesc_s,
                          (h != 0 || kk != 0) ? 1u : 0u);
        }
      };
      // O += P_i V_i (O = for the first step): P from tensor memory (16 keys = 8 columns), V MN-major
      // from shared memory (16 keys = 2048 B)
      auto partial = [&](int i) {
        const uint32_t v = low_v + (i % kRing) * (kTileBytes >> 4);
        // (a 128-wide head: the second sub-tile of V gives result columns 64..127)
#pragma unroll
        for (int h = 0; h < kSubTiles; ++h) {
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            mma_f16_tmem_a(tmem_base + kColumnO + h * kHeadDim, tmem_p + kk * 8, v + h * (kSubTileBytes >> 4) + kk * (2048 >> 4), kHighWord, idesc_o,
                           (i != 0 || kk != 0) ? 1u : 0u);
          if constexpr (FEW) {      // ... and what rounding took off the probabilities
#pragma unroll
            for (int kk = 0; kk < kKeys / 16; ++kk)
              mma_f16_tmem_a(tmem_base + kColumnO + h * kHeadDim, tmem_p + kKeys / 2 + kk * 8, v + h * (kSubTileBytes >> 4) + kk * (2048 >> 4), kHighWord,
                             idesc_o, 1u);
          }
        }
        mma_commit(pv_done);
      };
      if (barrier_wait(q_full, 0, p.status, kWaitQ) && barrier_wait(k_full(0), 0, p.status, kWaitKeyFull) &&
          (!kAhead || steps == 1 || barrier_wait(k_full(1), 0, p.status, kWaitKeyFull))) {
        tcgen05_fence_after();
        // (the second tile's scores too, for the reference point: into result columns, which nothing uses before the first
        // product of probabilities and values)
        scores(0, tmem_base);
        if (kAhead && steps > 1) scores(1, tmem_base + kColumnO);
        mma_commit(s_full);
        for (int i = 0; i < steps; ++i) {
          // the scores of step i + 1, once the softmax warps hold those of step i in registers
          if (i + 1 < steps) {
            if (!barrier_wait(k_full((i + 1) % kRing), ((i + 1) / kRing) & 1, p.status, kWaitKeyFull)) break;
            if (!barrier_wait(s_free, i & 1, p.status, kWaitBufferFree)) break;
            tcgen05_fence_after();
            scores(i + 1, tmem_base);
            mma_commit(s_full);
          }
          // the second product of step i, once its probabilities are in tensor memory
          if (!barrier_wait(v_full(i % kRing), (i / kRing) & 1, p.status, kWaitValueFull)) break;
          if (!barrier_wait(p_full, i & 1, p.status, kWaitProbabilities)) break;
          tcgen05_fence_after();
          partial(i);
        }
      }
    }
  } else if (warp < 4) {
    // ---- softmax: warp w owns tensor-memory lanes 32 w .. +31, one thread per query row ------------
    if constexpr (L::kMovesRegisters) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kSoftmaxRegisters));
    const int query = q0 + static_cast<int>(threadIdx.x);
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t tmem_s = tmem_base + lanes, tmem_o = tmem_base + kColumnO + lanes, tmem_mine = tmem_p + lanes;
    float reference = -INFINITY, row_sum = 0.f;     // -inf: the row has seen no finite score yet
    bool alive = true;
    const int last_allowed = p.causal ? min(query, p.k_tokens - 1) : p.k_tokens - 1;   // the last key this row may see
    const int open_until = p.causal ? min(q0, p.k_tokens - 1) : p.k_tokens - 1;         // ... and the last that every row of the CTA may

    if (FEW && q0 + warp * 32 >= p.q_tokens) {
      // A warp without a query takes part in the hand-overs only: its rows of scores and of the result mean nothing.
      for (int j = 0; alive && j < steps; ++j) {
        alive = barrier_wait(s_full, j & 1, p.status, kWaitScores);
        if (alive && lane == 0) barrier_arrive(s_free);
        if (alive && j > 0) alive = barrier_wait(pv_done, (j - 1) & 1, p.status, kWaitPartial);
        if (alive && lane == 0) barrier_arrive(p_full);
        __syncwarp();
      }
      alive = false;
    }

    // the second product of step j has finished: its probabilities and its value tile are spent
    auto wait_product = [&](int j) {
      if (!barrier_wait(pv_done, j & 1, p.status, kWaitPartial)) return false;
      tcgen05_fence_after();
      if (threadIdx.x == 0) barrier_arrive(v_empty(j % kRing));
      return true;
    };

    // One tile's scores: a row per thread, held in registers for both the maximum and the exponentials.
    using Scores = uint32_t[kKeys];
    auto load_scores = [&](Scores& r, uint32_t from) {
#pragma unroll
      for (int i = 0; i < kKeys; i += 32) tmem_load_32(from + i, *reinterpret_cast<uint32_t(*)[32]>(&r[i]));
      tmem_load_wait();
    };
    auto mask = [&](Scores& r, int key0) {
      if (key0 + kKeys - 1 > open_until) {            // uniform in the CTA
        const int limit = last_allowed - key0;        // columns > limit are masked for this row
#pragma unroll
        for (int i = 0; i < kKeys; ++i) {
          if (i > limit) r[i] = 0xff800000u;   // -inf
        }
      }
    };
    // (three-input maximum, and below two-element FMA and add: every element costs half an instruction for
    // the maximum, half for the scaling, one ex2, half for the sum and half for the rounding)
    auto maximum = [&](const Scores& r) {
      float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
      for (int i = 0; i < kKeys; i += 8) {
        m0 = max3(m0, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
        m1 = max3(m1, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
        m2 = max3(m2, __uint_as_float(r[i + 4]), __uint_as_float(r[i + 5]));
        m3 = max3(m3, __uint_as_float(r[i + 6]), __uint_as_float(r[i + 7]));
      }
      return fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
    };

    // The second tile's maximum, for the row's reference point.
    float second_max = -INFINITY;
    if (kAhead && alive && steps > 1) {
      alive = barrier_wait(s_full, 0, p.status, kWaitScores);
      if (alive) {
        Scores r;
        tcgen05_fence_after();
        load_scores(r, tmem_o);
        mask(r, kKeys);
        second_max = maximum(r);
      }
    }
    for (int j = 0; alive && j < steps; ++j) {
      if (!barrier_wait(s_full, j & 1, p.status, kWaitScores)) { alive = false; break; }
      tcgen05_fence_after();
      if (threadIdx.x == 0) barrier_arrive(k_empty(j % kRing));      // the first product has read key tile j
      Scores r;
      load_scores(r, tmem_s);         // the columns go back to the issuer at once
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) barrier_arrive(s_free);
      mask(r, j * kKeys);
      const float tile_max = maximum(r);
      // The reference point: the first two tiles' maximum, moved only when a tile rises more than
      // 2^kSlack above it (from -inf, any finite maximum does). `factor` rescales what the row has
      // gathered so far; it is 1 for a row that stays.
      float factor = 1.f;
      const bool moves = j == 0 || (tile_max - reference) * p.scale_log2 > kSlack;       // false for NaN
      if (moves) {
        if (j != 0) factor = exp2_ftz((reference - tile_max) * p.scale_log2);             // from -inf: 0, and nothing was gathered
        reference = j == 0 ? fmaxf(tile_max, second_max) : tile_max;
      }
      const bool rescale = j != 0 && __any_sync(0xffffffffu, moves);
      const float shift = reference == -INFINITY ? 0.f : -reference * p.scale_log2;       // all scores -inf so far: every probability is 0

      // probabilities and their sum; the probabilities go into tensor memory as the A operand of the second
      // product (16-bit pairs)
      float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
      uint32_t packed[kKeys / 2], rest[FEW ? kKeys / 2 : 1];
      const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), shift2 = make_float2(shift, shift);
#pragma unroll
      for (int chunk = 0; chunk < kKeys / 4; ++chunk) {
        const float2 t0 = __ffma2_rn(make_float2(__uint_as_float(r[chunk * 4 + 0]), __uint_as_float(r[chunk * 4 + 1])), scale2, shift2);
        const float2 t1 = __ffma2_rn(make_float2(__uint_as_float(r[chunk * 4 + 2]), __uint_as_float(r[chunk * 4 + 3])), scale2, shift2);
        const float2 e0 = make_float2(exp2_ftz(t0.x), exp2_ftz(t0.y));
        const float2 e1 = make_float2(exp2_ftz(t1.x), exp2_ftz(t1.y));
        sum0 = __fadd2_rn(sum0, e0);
        sum1 = __fadd2_rn(sum1, e1);
        packed[chunk * 2 + 0] = pack_pair<T>(e0.x, e0.y);
        packed[chunk * 2 + 1] = pack_pair<T>(e1.x, e1.y);
        if constexpr (FEW) {
          rest[chunk * 2 + 0] = pack_rest<T>(packed[chunk * 2 + 0], e0);
          rest[chunk * 2 + 1] = pack_rest<T>(packed[chunk * 2 + 1], e1);
        }
      }
      const float2 sum01 = __fadd2_rn(sum0, sum1);
      row_sum = row_sum * factor + (sum01.x + sum01.y);

      // The previous step's product still reads the probability columns and adds into the result: wait for it
      // (it had this step's loads and exponentials to finish), then write.
      if (j > 0) {
        if (!wait_product(j - 1)) { alive = false; break; }
        if (rescale) {       // rare: some row of this warp moved its reference point
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {      // sixteen result columns at a time: the probabilities are still in registers
            uint32_t o[16];
            tmem_load_16(tmem_o + c * 16, o);
            tmem_load_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
            tmem_store_16(tmem_o + c * 16, o);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kKeys / 2; i += 32) {
        tmem_store_32(tmem_mine + i, *reinterpret_cast<uint32_t(*)[32]>(&packed[i]));
        if constexpr (FEW) tmem_store_32(tmem_mine + kKeys / 2 + i, *reinterpret_cast<uint32_t(*)[32]>(&rest[i]));
      }
      tmem_store_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) barrier_arrive(p_full);
    }

    if (alive && wait_product(steps - 1)) {
      // the result row leaves tensor memory 32 columns at a time (the loads are warp-wide: every lane takes
      // part, rows beyond the queries only skip the stores)
      const bool stores = query < p.q_tokens;
      const float inverse = 1.0f / row_sum;
      T* out_row = static_cast<T*>(p.out) + batch * p.out_batch + head * p.out_head + static_cast<long long>(query) * p.out_token;
      const bool vector_ok = (reinterpret_cast<uintptr_t>(out_row) & 15) == 0;
      const int width = p.head_dim;       // a multiple of 8: whole 16-byte vectors
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        if (c * 32 >= width) break;
        uint32_t o[32];
        tmem_load_32(tmem_o + c * 32, o);
        tmem_load_wait();
        if (stores && vector_ok) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            if (c * 32 + v * 8 < width) {
              uint4 word;
              word.x = pack_pair<T>(__uint_as_float(o[v * 8 + 0]) * inverse, __uint_as_float(o[v * 8 + 1]) * inverse);
              word.y = pack_pair<T>(__uint_as_float(o[v * 8 + 2]) * inverse, __uint_as_float(o[v * 8 + 3]) * inverse);
              word.z = pack_pair<T>(__uint_as_float(o[v * 8 + 4]) * inverse, __uint_as_float(o[v * 8 + 5]) * inverse);
              word.w = pack_pair<T>(__uint_as_float(o[v * 8 + 6]) * inverse, __uint_as_float(o[v * 8 + 7]) * inverse);
              *reinterpret_cast<uint4*>(out_row + c * 32 + v * 8) = word;
            }
          }
        } else if (stores) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (c * 32 + i < width) out_row[c * 32 + i] = from_compute<T, float>(__uint_as_float(o[i]) * inverse);
          }
        }
        __syncwarp();
      }
    }
  }

  // ---- teardown: every thread arrives here, also after a wait that gave up -------------------
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 5) {
    tcgen05_fence_after();
    if constexpr (L::kTwoAllocations) tmem_dealloc(tmem_p, kTmemColumnsP);
    tmem_dealloc(tmem_base, L::kTmemColumns);
  }
}

// ---- With a window, sinks and shared key heads ------------------------------------------------------
//
// The same products, softmax and hand-overs as above, for rows that see the keys j <= p with j > p - window or j < sinks (p = row + k_tokens -
// q_tokens): a block of rows walks the tiles of the sinks and then those from its first row's window to its last row. Under a short window such a
// walk is a few steps, and a CTA's start (barriers, tensor memory, first loads: about 8 us of latency beside 0.9 a step) would be most of it; so
// CTAs stay, as many as fit, and take blocks one after another. Counted through all blocks, step g of a CTA has ring stage g % kRing and the
// phases that g gives, and the first loads and scores of the next block run under the last step and the result of the one before: its query tile
// is loaded once the last scores of that block are out (q_empty), and its first product writes the result columns only after p_full, which the
// softmax warps signal when they have read the result before it.
//
// Blocks are dealt out by length, the longest of all heads first, so that CTAs get sums of about the same length.
// With a window: what a query sees (keyed.h), which key head it shares, and, for rows whose result has to be taken again, where the operands lie.
struct WindowAttnParams : AttnParams {
  int group, offset;               // heads a key head serves; k_tokens - q_tokens
  int window, sinks;
  const void *q, *k, *v;
  long long q_strides[3], k_strides[3], v_strides[3];
  bool out_vectors;                // every eight elements of the result lie on 16 bytes
};

// Heads above 64: a softmax warp's results on their way out, 32 rows of 32 elements. A thread has a row, and a store of 16 bytes to each of 32 rows
// is as many halves of sectors; eight rows of 64 bytes are whole ones (4 x 37 heads of 128, 2048 tokens under a window of 257 91 us, without
// 103; 2 x 32 x 2501 under 333 58.9 and 60.5). Heads of 64 have half the bytes a row and a third CTA's stores beside: 1 to 4 % slower with it.
template <int D, int KEYS>
struct WindowLayout : AttnLayout<D, KEYS, false> {
  using Base = AttnLayout<D, KEYS, false>;
  static constexpr bool kStaged = D > kHeadDim;
  static constexpr uint32_t kStageBytes = 32 * 32 * 2, kOffsetStages = Base::kOffsetBarriers + 256;
  static constexpr size_t kSmemBytes = Base::kSmemBytes + (kStaged ? kRows / 32 * kStageBytes : 0);
  static_assert(Base::kCtasPerSm * (kSmemBytes + 1024) <= 228 * 1024, "as many CTAs an SM");
};

// The first n of 32 bits; none for n <= 0, all for n >= 32.
__device__ __forceinline__ uint32_t first_bits(int n) {
  uint32_t bits;
  asm("shl.b32 %0, 1, %1;" : "=r"(bits) : "r"(min(max(n, 0), 32)));      // (shifted by 32: 0)
  return bits - 1;
}

struct WindowBlock {
  int q0, head, batch, key_head;
  int sink_tiles, gap, steps;        // tiles of the sinks; tiles left out behind them; at least one step
};
template <int KEYS>
__device__ __forceinline__ WindowBlock window_block(const WindowAttnParams& p, int item) {
  WindowBlock b;
  const int heads = p.batch * p.heads, head_index = item % heads;
  b.q0 = (p.q_blocks - 1 - item / heads) * kRows;
  b.head = head_index % p.heads;
  b.batch = head_index / p.heads;
  b.key_head = b.head / p.group;
  const int low = b.q0 + p.offset, high = min(b.q0 + kRows, p.q_tokens) - 1 + p.offset;       // positions
  const int stop = (max(high, -1) + KEYS) / KEYS, start = min(max(low - p.window + 1, 0) / KEYS, stop);
  b.sink_tiles = min((min(p.sinks, max(high, -1) + 1) + KEYS - 1) / KEYS, start);
  b.gap = start - b.sink_tiles;
  b.steps = max(stop - b.gap, 1);
  return b;
}

// Which columns of the values are a NaN (bit 0), an infinity (1), minus infinity (2) in some key that all rows from position `first` to `last` see, by a
// warp: column 64 h + 2 lane + e in bits 3 (2 h + e) and up. Ends where every column is a NaN.
template <typename T, int D>
__device__ __forceinline__ uint32_t not_finite_for_all(const WindowAttnParams& p, int batch, int key_head, int first, int last) {
  constexpr uint32_t kInfinity = std::is_same_v<T, __nv_bfloat16> ? 0x7f80u : 0x7c00u;
  constexpr int kPairs = D / 64, kAtOnce = 8;
  const int lane = threadIdx.x & 31;
  const T* v = static_cast<const T*>(p.v) + batch * p.v_strides[0] + key_head * p.v_strides[1] + 2 * lane;
  const int start = max(last - p.window + 1, 0), sinks = max(min(min(p.sinks, first + 1), start), 0), count = sinks + max(first + 1 - start, 0);
  uint32_t found = 0, all = 0;
#pragma unroll
  for (int h = 0; h < kPairs; ++h) all |= 64 * h + 2 * lane < p.head_dim ? 9u << 6 * h : 0u;
#pragma unroll 1
  for (int nth0 = 0; nth0 < count && !__all_sync(0xffffffffu, (found & all) == all); nth0 += kAtOnce) {
    uint32_t pair[kAtOnce][kPairs];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int nth = nth0 + i, key = nth < sinks ? nth : nth - sinks + start;
#pragma unroll
      for (int h = 0; h < kPairs; ++h) {
        pair[i][h] = 0;
        if (nth < count && 64 * h + 2 * lane < p.head_dim) pair[i][h] = *reinterpret_cast<const uint32_t*>(v + key * p.v_strides[2] + 64 * h);
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
#pragma unroll
      for (int n = 0; n < 2 * kPairs; ++n) {
        const uint32_t x = n % 2 ? pair[i][n / 2] >> 16 : pair[i][n / 2] & 0xffffu, size = x & 0x7fffu;
        found |= (size > kInfinity ? 1u : size < kInfinity ? 0u : x >> 15 ? 4u : 2u) << 3 * n;
      }
    }
  }
  return found;
}

// Whether what is no finite number in a result row is what the row's own keys make it, by what not_finite_for_all has found: a NaN where a value is one or
// values are infinities of both signs, an infinity (which a NaN of any other key would not have left) where a value is that.
template <typename T, int D>
__device__ __forceinline__ bool row_stands(const WindowAttnParams& p, int batch, int head, int row, uint32_t found) {
  constexpr uint32_t kInfinity = std::is_same_v<T, __nv_bfloat16> ? 0x7f80u : 0x7c00u;
  const T* out = static_cast<const T*>(p.out) + batch * p.out_batch + head * p.out_head + row * p.out_token;
  bool stands = true;
#pragma unroll
  for (int n = 0; n < D / 32; ++n) {
    const int column = 64 * (n / 2) + 2 * (threadIdx.x & 31) + n % 2;
    if (column < p.head_dim) {
      const uint32_t x = reinterpret_cast<const unsigned short*>(out)[column], size = x & 0x7fffu, here = found >> 3 * n & 7u;
      if (size > kInfinity) stands &= (here & 1u) != 0 || here == 6u;
      else if (size == kInfinity) stands &= (here & (x >> 15 ? 4u : 2u)) != 0;
    }
  }
  return __all_sync(0xffffffffu, stands);
}

// One result row from the keys it sees and nothing else, by a warp: 32 keys at a time, a key a lane for its score, D / 32 elements of the head a
// lane for the result.
template <typename T, int D>
__device__ __forceinline__ void take_row_again(const WindowAttnParams& p, int batch, int head, int key_head, int row) {
  const int lane = threadIdx.x & 31, position = row + p.offset;
  const T* q = static_cast<const T*>(p.q) + batch * p.q_strides[0] + head * p.q_strides[1] + row * p.q_strides[2];
  const T* k = static_cast<const T*>(p.k) + batch * p.k_strides[0] + key_head * p.k_strides[1];
  const T* v = static_cast<const T*>(p.v) + batch * p.v_strides[0] + key_head * p.v_strides[1];
  constexpr int kMine = D / 32;
  float most = -INFINITY, total = 0.f, result[kMine];
#pragma unroll
  for (int c = 0; c < kMine; ++c) result[c] = 0.f;
  const int start = max(position - p.window + 1, 0), sinks = min(min(p.sinks, position + 1), start);
  const int count = sinks + position + 1 - start;
#pragma unroll 1
  for (int first = 0; first < count; first += 32) {
    const int nth = first + lane, key = nth < sinks ? nth : nth - sinks + start;
    float score = -INFINITY;
    if (nth < count) {
      const T* from = k + key * p.k_strides[2];
      score = 0.f;
#pragma unroll 2
      for (int c = 0; c < p.head_dim; c += 8) {      // (rows of q and k are 16-byte aligned: TMA reads them too)
        const uint4 a = *reinterpret_cast<const uint4*>(q + c), b = *reinterpret_cast<const uint4*>(from + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) score = fmaf(to_compute(reinterpret_cast<const T*>(&a)[e]), to_compute(reinterpret_cast<const T*>(&b)[e]), score);
      }
      score *= p.scale_log2;
    }
    float top = score;
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, offset));
    top = fmaxf(top, most);
    const float factor = most == top ? 1.f : exp2_ftz(most - top);
    most = top;
    const float weight = nth < count ? exp2_ftz(score - (top == -INFINITY ? 0.f : top)) : 0.f;
    total = total * factor + warp_sum(weight);
#pragma unroll
    for (int c = 0; c < kMine; ++c) result[c] *= factor;
#pragma unroll 4
    for (int i = 0; i < min(32, count - first); ++i) {
      const float w = __shfl_sync(0xffffffffu, weight, i);
      const T* from = v + __shfl_sync(0xffffffffu, key, i) * p.v_strides[2];
#pragma unroll
      for (int c = 0; c < kMine; ++c) {
        const int column = c * 32 + lane;
        if (column < p.head_dim) result[c] = fmaf(w, to_compute(from[column]), result[c]);
      }
    }
  }
  T* out = static_cast<T*>(p.out) + batch * p.out_batch + head * p.out_head + row * p.out_token;
#pragma unroll
  for (int c = 0; c < kMine; ++c) {
    const int column = c * 32 + lane;
    if (column < p.head_dim) out[column] = from_compute<T, float>(result[c] / total);
  }
  __syncwarp();
}

template <typename T, int D, int KEYS>
__global__ void __launch_bounds__(kAttnThreads, AttnLayout<D, KEYS, false>::kCtasPerSm)
window_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const WindowAttnParams p) {
  using L = WindowLayout<D, KEYS>;
  constexpr int kKeys = KEYS, kRing = L::kRing, kSubTiles = L::kSubTiles;
  constexpr uint32_t kSubTileBytes = L::kSubTileBytes, kTileBytes = L::kTileBytes, kOffsetK = L::kOffsetK, kOffsetV = L::kOffsetV;
  constexpr uint32_t kOffsetBarriers = L::kOffsetBarriers, kColumnO = L::kColumnO;
  extern __shared__ unsigned char raw_smem[];
  const uint32_t base = (smem_address(raw_smem) + 1023u) & ~1023u;
  unsigned char* aligned = raw_smem + (base - smem_address(raw_smem));
  const uint32_t barriers = base + kOffsetBarriers;
  const uint32_t q_full = barriers;
  auto k_full = [&](uint32_t s) { return barriers + 8u * (1 + s); };
  auto k_empty = [&](uint32_t s) { return barriers + 8u * (1 + kRing + s); };
  auto v_full = [&](uint32_t s) { return barriers + 8u * (1 + 2 * kRing + s); };
  auto v_empty = [&](uint32_t s) { return barriers + 8u * (1 + 3 * kRing + s); };
  const uint32_t s_full = barriers + 8u * (1 + 4 * kRing), s_free = s_full + 8, p_full = s_full + 16, pv_done = s_full + 24;
  const uint32_t q_empty = s_full + 32;                         // all scores of a block are out: its queries are spent
  constexpr int kBarrierCount = 1 + 4 * kRing + 5;
  const uint32_t tmem_slot = barriers + 8u * kBarrierCount;
  volatile uint32_t* tmem_slot_pointer = reinterpret_cast<volatile uint32_t*>(aligned + kOffsetBarriers + 8 * kBarrierCount);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* const stage = aligned + L::kOffsetStages + (warp & 3) * L::kStageBytes;      // kStaged: of a softmax warp's results
  const int items = p.q_blocks * p.batch * p.heads;

  auto load_queries = [&](const WindowBlock& b) {
    barrier_expect_tx(q_full, kSubTiles * kQueryBytes);
    for (int h = 0; h < kSubTiles; ++h) tma_load_4d(base + h * kQueryBytes, &map_q, q_full, h * kHeadDim, b.q0, b.head, b.batch);
  };
  // step j of a block, the CTA's step g
  auto load_tile = [&](const CUtensorMap* map, uint32_t ring, uint32_t full, const WindowBlock& b, int j, uint32_t g) {
    barrier_expect_tx(full, kTileBytes);
    const int key = (j < b.sink_tiles ? j : j + b.gap) * kKeys;
    for (int h = 0; h < kSubTiles; ++h)
      tma_load_4d(base + ring + (g % kRing) * kTileBytes + h * kSubTileBytes, map, full, h * kHeadDim, key, b.key_head, b.batch);
  };

  const int early = min(window_block<KEYS>(p, blockIdx.x).steps, kRing);      // steps of the first block whose tiles are loaded before the CTA meets
  if (warp == 4 && elect_one()) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    barrier_init(q_full, 1);
    for (int s = 0; s < kRing; ++s) {
      barrier_init(k_full(s), 1);
      barrier_init(k_empty(s), 1);
      barrier_init(v_full(s), 1);
      barrier_init(v_empty(s), 1);
    }
    barrier_init(s_full, 1);
    barrier_init(pv_done, 1);
    barrier_init(p_full, kRows / 32);
    barrier_init(s_free, kRows / 32);
    barrier_init(q_empty, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    const WindowBlock b = window_block<KEYS>(p, blockIdx.x);
    wait_for_earlier();
    if (blockIdx.x == 0) p.status.begin();
    load_queries(b);
    for (int j = 0; j < early; ++j) load_tile(&map_k, kOffsetK, k_full(j), b, j, j);
    for (int j = 0; j < early; ++j) load_tile(&map_v, kOffsetV, v_full(j), b, j, j);
  }
  if (warp == 5) {
    if constexpr (L::kTwoAllocations) {
      tmem_alloc_more(tmem_slot, L::kTmemColumns);
      tmem_alloc(tmem_slot + 4, kTmemColumnsP);
    } else {
      tmem_alloc(tmem_slot, L::kTmemColumns);
    }
  }
  wait_for_earlier();
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = tmem_slot_pointer[0];
  const uint32_t tmem_p = L::kTwoAllocations ? tmem_slot_pointer[1] : tmem_base + L::kColumnP;

  if (L::kMovesRegisters && warp >= 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kOtherRegisters));
  if (warp == 4) {
    // ---- producer --------------------------------------------------------------------------------
    if (elect_one()) {
      uint32_t g = 0, block = 0, keys_loaded = early, values_loaded = early, queries_of = 0;      // steps and blocks before this one, what was asked for
      bool alive = true;
      for (int item = blockIdx.x; alive && item < items; item += gridDim.x, ++block) {
        const WindowBlock b = window_block<KEYS>(p, item);
        for (int j = block == 0 ? early : 0; alive && j < b.steps; ++j) {
          const uint32_t n = g + j, phase = (n / kRing) & 1;
          alive = barrier_wait(k_empty(n % kRing), phase ^ 1, p.status, kWaitKeyEmpty);
          if (!alive) break;
          load_tile(&map_k, kOffsetK, k_full(n % kRing), b, j, n);
          keys_loaded = n + 1;
          if (j == 0) {      // (of a later block)
            alive = barrier_wait(q_empty, (block - 1) & 1, p.status, kWaitQ);
            if (!alive) break;
            load_queries(b);
            queries_of = block;
          }
          alive = barrier_wait(v_empty(n % kRing), phase ^ 1, p.status, kWaitValueEmpty);
          if (!alive) break;
          load_tile(&map_v, kOffsetV, v_full(n % kRing), b, j, n);
          values_loaded = n + 1;
        }
        g += b.steps;
      }
      let_later_start();
      if (!alive) {      // what is under way has to land before the CTA leaves
        auto landed = [&](uint32_t bar, uint32_t parity) {
          for (uint32_t spin = 0; spin < kSpinLimit && !barrier_try_wait(bar, parity); ++spin) {
          }
        };
        landed(q_full, queries_of & 1);
        for (uint32_t n = keys_loaded > kRing ? keys_loaded - kRing : 0; n < keys_loaded; ++n) landed(k_full(n % kRing), (n / kRing) & 1);
        for (uint32_t n = values_loaded > kRing ? values_loaded - kRing : 0; n < values_loaded; ++n) landed(v_full(n % kRing), (n / kRing) & 1);
      }
    }
  } else if (warp == 5) {
    // ---- issuer ----------------------------------------------------------------------------------
    if (elect_one()) {
      constexpr uint32_t idesc_s = attn_instruction_descriptor<T>(kKeys, false);
      constexpr uint32_t idesc_o = attn_instruction_descriptor<T>(kHeadDim, true);
      constexpr uint32_t kHighWord = kDescriptorHigh;
      const uint32_t low_q = descriptor_low(base, 0), low_k = descriptor_low(base + kOffsetK, 0);
      const uint32_t low_v = descriptor_low(base + kOffsetV, kSubTileBytes);
      // the scores of step g, once its keys (and a block's queries) are there and the softmax warps hold the scores before in registers
      auto scores = [&](uint32_t g, bool ends) {
        if (!barrier_wait(k_full(g % kRing), (g / kRing) & 1, p.status, kWaitKeyFull)) return false;
        if (g > 0 && !barrier_wait(s_free, (g - 1) & 1, p.status, kWaitBufferFree)) return false;
        tcgen05_fence_after();
        const uint32_t k = low_k + (g % kRing) * (kTileBytes >> 4);
#pragma unroll
        for (int h = 0; h < kSubTiles; ++h) {
#pragma unroll
          for (int kk = 0; kk < kHeadDim / 16; ++kk)
            mma_f16_split(tmem_base, low_q + h * (kQueryBytes >> 4) + kk * 2, kHighWord, k + h * (kSubTileBytes >> 4) + kk * 2, kHighWord, idesc_s,
                          (h != 0 || kk != 0) ? 1u : 0u);
        }
        mma_commit(s_full);
        if (ends) mma_commit(q_empty);
        return true;
      };
      auto partial = [&](uint32_t g, bool first) {
        if (!barrier_wait(v_full(g % kRing), (g / kRing) & 1, p.status, kWaitValueFull)) return false;
        if (!barrier_wait(p_full, g & 1, p.status, kWaitProbabilities)) return false;
        tcgen05_fence_after();
        const uint32_t v = low_v + (g % kRing) * (kTileBytes >> 4);
#pragma unroll
        for (int h = 0; h < kSubTiles; ++h) {
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            mma_f16_tmem_a(tmem_base + kColumnO + h * kHeadDim, tmem_p + kk * 8, v + h * (kSubTileBytes >> 4) + kk * (2048 >> 4), kHighWord, idesc_o,
                           (!first || kk != 0) ? 1u : 0u);
        }
        mma_commit(pv_done);
        return true;
      };
      uint32_t g = 0, block = 0;
      int item = blockIdx.x, left = window_block<KEYS>(p, item).steps;      // of the block of step g, g among them
      bool first = true;                                                     // step g is the first of its block
      bool alive = barrier_wait(q_full, 0, p.status, kWaitQ) && scores(0, left == 1);
      while (alive) {
        if (left > 1) {      // the scores of the block's next step, then the product of this one
          alive = scores(g + 1, left == 2) && partial(g, first);
          first = false;
          --left;
        } else {             // the block's last product first: its result is what the softmax warps wait for
          alive = partial(g, first);
          item += gridDim.x;
          if (!alive || item >= items) break;
          left = window_block<KEYS>(p, item).steps;
          first = true;
          alive = barrier_wait(q_full, ++block & 1, p.status, kWaitQ) && scores(g + 1, left == 1);
        }
        ++g;
      }
    }
  } else if (warp < 4) {
    // ---- softmax ---------------------------------------------------------------------------------
    if constexpr (L::kMovesRegisters) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kSoftmaxRegisters));
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t tmem_s = tmem_base + lanes, tmem_o = tmem_base + kColumnO + lanes, tmem_mine = tmem_p + lanes;
    uint32_t g = 0;
    bool alive = true;
    auto wait_product = [&](uint32_t n) {
      if (!barrier_wait(pv_done, n & 1, p.status, kWaitPartial)) return false;
      tcgen05_fence_after();
      if (threadIdx.x == 0) barrier_arrive(v_empty(n % kRing));
      return true;
    };
    for (int item = blockIdx.x; alive && item < items; item += gridDim.x) {
      const WindowBlock b = window_block<KEYS>(p, item);
      const int query = b.q0 + static_cast<int>(threadIdx.x), position = query + p.offset, low = b.q0 + p.offset;
      float reference = -INFINITY, row_sum = 0.f;
      for (int j = 0; j < b.steps; ++j, ++g) {
        alive = barrier_wait(s_full, g & 1, p.status, kWaitScores);
        if (!alive) break;
        tcgen05_fence_after();
        if (threadIdx.x == 0) barrier_arrive(k_empty(g % kRing));
        uint32_t r[kKeys];
#pragma unroll
        for (int i = 0; i < kKeys; i += 32) tmem_load_32(tmem_s + i, *reinterpret_cast<uint32_t(*)[32]>(&r[i]));
        tmem_load_wait();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) barrier_arrive(s_free);
        // Masks, where the tile has a key that some row does not see (uniform in the CTA): what the row sees as bits, 32 keys a word, which the
        // compiler turns into predicates eight at a time; two comparisons and selections for each key were half of all instructions under a
        // window of 64.
        const int key0 = (j < b.sink_tiles ? j : j + b.gap) * kKeys;
        if (key0 + kKeys - 1 > low || (key0 <= low + kRows - 1 - p.window && key0 + kKeys > p.sinks)) {
#pragma unroll
          for (int i0 = 0; i0 < kKeys; i0 += 32) {
            const int at = key0 + i0;
            const uint32_t sees = first_bits(position + 1 - at) & (~first_bits(position - p.window + 1 - at) | first_bits(p.sinks - at));
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (!(sees >> i & 1)) r[i0 + i] = 0xff800000u;
            }
          }
        }
        float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
        for (int i = 0; i < kKeys; i += 8) {
          m0 = max3(m0, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
          m1 = max3(m1, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
          m2 = max3(m2, __uint_as_float(r[i + 4]), __uint_as_float(r[i + 5]));
          m3 = max3(m3, __uint_as_float(r[i + 6]), __uint_as_float(r[i + 7]));
        }
        const float tile_max = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
        float factor = 1.f;
        const bool moves = j == 0 || (tile_max - reference) * p.scale_log2 > kSlack;       // false for NaN
        if (moves) {
          if (j != 0) factor = exp2_ftz((reference - tile_max) * p.scale_log2);             // from -inf: 0, and nothing was gathered
          reference = tile_max;
        }
        const bool rescale = j != 0 && __any_sync(0xffffffffu, moves);
        // (f16: probabilities 2^7 times as large, up to 2^(8 + 7), so that those under 2^-21 of the largest and not of 2^-14 on lose digits)
        constexpr float kLift = std::is_same_v<T, __half> ? 7.f : 0.f;
        const float shift = reference == -INFINITY ? 0.f : fmaf(-reference, p.scale_log2, kLift);
        float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
        uint32_t packed[kKeys / 2];
        const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), shift2 = make_float2(shift, shift);
#pragma unroll
        for (int chunk = 0; chunk < kKeys / 4; ++chunk) {
          const float2 t0 = __ffma2_rn(make_float2(__uint_as_float(r[chunk * 4 + 0]), __uint_as_float(r[chunk * 4 + 1])), scale2, shift2);
          const float2 t1 = __ffma2_rn(make_float2(__uint_as_float(r[chunk * 4 + 2]), __uint_as_float(r[chunk * 4 + 3])), scale2, shift2);
          const float2 e0 = make_float2(exp2_ftz(t0.x), exp2_ftz(t0.y));
          const float2 e1 = make_float2(exp2_ftz(t1.x), exp2_ftz(t1.y));
          sum0 = __fadd2_rn(sum0, e0);
          sum1 = __fadd2_rn(sum1, e1);
          packed[chunk * 2 + 0] = pack_pair<T>(e0.x, e0.y);
          packed[chunk * 2 + 1] = pack_pair<T>(e1.x, e1.y);
        }
        const float2 sum01 = __fadd2_rn(sum0, sum1);
        row_sum = row_sum * factor + (sum01.x + sum01.y);
        if (j > 0) {
          alive = wait_product(g - 1);
          if (!alive) break;
          if (rescale) {
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
        }
#pragma unroll
        for (int i = 0; i < kKeys / 2; i += 32) tmem_store_32(tmem_mine + i, *reinterpret_cast<uint32_t(*)[32]>(&packed[i]));
        tmem_store_wait();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) barrier_arrive(p_full);
      }
      if (!alive || !wait_product(g - 1)) {
        alive = false;
        break;
      }
      // the result row leaves tensor memory 32 columns at a time (every lane takes part; rows beyond the queries only skip the stores)
      const bool stores = query < p.q_tokens, sees_some = position >= 0;      // a query before the first key: zeros
      const float inverse = sees_some ? 1.0f / row_sum : 0.f;
      T* const out = static_cast<T*>(p.out) + b.batch * p.out_batch + b.head * p.out_head;
      T* const out_row = out + static_cast<long long>(query) * p.out_token;
      bool odd = false;                                  // something in the row is no finite number
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        if (c * 32 >= p.head_dim) break;
        uint32_t o[32];
        tmem_load_32(tmem_o + c * 32, o);
        tmem_load_wait();
        float value[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          value[i] = sees_some ? __uint_as_float(o[i]) * inverse : 0.f;
          odd |= !(fabsf(value[i]) < INFINITY);
        }
        if (L::kStaged && p.out_vectors) {
#pragma unroll
          for (int v = 0; v < 4; ++v)
            *reinterpret_cast<uint4*>(stage + lane * 64 + (v ^ (lane >> 1 & 3)) * 16) =
                make_uint4(pack_pair<T>(value[v * 8], value[v * 8 + 1]), pack_pair<T>(value[v * 8 + 2], value[v * 8 + 3]),
                           pack_pair<T>(value[v * 8 + 4], value[v * 8 + 5]), pack_pair<T>(value[v * 8 + 6], value[v * 8 + 7]));
          __syncwarp();
          const int column = c * 32 + lane % 4 * 8;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + lane / 4;
            const uint4 part = *reinterpret_cast<const uint4*>(stage + row * 64 + ((lane ^ (row >> 1)) & 3) * 16);
            const int at = b.q0 + warp * 32 + row;
            if (at < p.q_tokens && column < p.head_dim) *reinterpret_cast<uint4*>(out + static_cast<long long>(at) * p.out_token + column) = part;
          }
        } else if (stores && p.out_vectors) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            if (c * 32 + v * 8 < p.head_dim) {
              *reinterpret_cast<uint4*>(out_row + c * 32 + v * 8) =
                  make_uint4(pack_pair<T>(value[v * 8], value[v * 8 + 1]), pack_pair<T>(value[v * 8 + 2], value[v * 8 + 3]),
                             pack_pair<T>(value[v * 8 + 4], value[v * 8 + 5]), pack_pair<T>(value[v * 8 + 6], value[v * 8 + 7]));
            }
          }
        } else if (stores) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (c * 32 + i < p.head_dim) out_row[c * 32 + i] = from_compute<T, float>(value[i]);
          }
        }
        __syncwarp();
      }
      tcgen05_fence_before();
      // The products take every key of a tile, at a probability of zero where a row does not see it, and zero times an infinity or a NaN is a
      // NaN. So a row that came out with one is taken again from its own keys alone, by the warp, in plain f32, unless it must be one: its sum, which
      // no other key is in, is no positive number (a NaN in the queries or in a key it sees), or values that all rows of the warp see make it one. Without
      // these two a NaN that everybody sees was a thousand times the launch (2 x 12 x 4096 under a window of 1024 54 us, all NaN 43.5 ms).
      uint32_t again = __ballot_sync(0xffffffffu, odd && stores && row_sum > 0.f);
      if (again != 0) {
        const int first = b.q0 + warp * 32 + p.offset, last = min(first + 31, p.q_tokens - 1 + p.offset);
        const uint32_t found = not_finite_for_all<T, D>(p, b.batch, b.key_head, first, last);
        do {
          const int row = b.q0 + warp * 32 + __ffs(again) - 1;
          again &= again - 1;
          if (!row_stands<T, D>(p, b.batch, b.head, row, found)) take_row_again<T, D>(p, b.batch, b.head, b.key_head, row);
        } while (again != 0);
      }
    }
  }

  // ---- teardown: every thread arrives here, also after a wait that gave up -------------------
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 5) {
    tcgen05_fence_after();
    if constexpr (L::kTwoAllocations) tmem_dealloc(tmem_p, kTmemColumnsP);
    tmem_dealloc(tmem_base, L::kTmemColumns);
  }
}

// A four-axis map over one of Q, K, V: `head_dim` contiguous elements, then tokens, heads, batch with
// the caller's element strides; box = 64 x `rows` x 1 x 1 (128 queries, or a step's keys), 128-byte swizzle. Rows beyond the tokens read
// 0, and so do the columns beyond a head narrower than its tiles: zeros add nothing to q . k and give
// result columns nobody stores, so a narrow head runs through the same 64-wide tiles.
tq_status attention_map(CUtensorMap* map, tq_dtype dtype, const void* pointer, long long head_dim, long long tokens, long long heads,
                        long long batch, const int64_t* strides, int rows) {
  EncodeTiled encode = encode_tiled();
  TQ_REQUIRE(encode != nullptr, TQ_EXTERNAL, "the CUDA driver does not provide cuTensorMapEncodeTiled");
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(tokens), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(batch)};
  // an axis of extent 1 never moves, so its stride only has to be legal
  const long long token_stride = tokens > 1 ? strides[2] : head_dim;
  const long long head_stride = heads > 1 ? strides[1] : head_dim;
  const long long batch_stride = batch > 1 ? strides[0] : head_dim;
  const cuuint64_t byte_strides[3] = {static_cast<cuuint64_t>(token_stride) * 2, static_cast<cuuint64_t>(head_stride) * 2,
                                      static_cast<cuuint64_t>(batch_stride) * 2};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(kHeadDim), static_cast<cuuint32_t>(rows), 1, 1};
  const cuuint32_t element_strides[4] = {1, 1, 1, 1};
  const CUresult result = encode(map, dtype == TQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                                 const_cast<void*>(pointer), dims, byte_strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TQ_REQUIRE(result == CUDA_SUCCESS, TQ_UNSUPPORTED, "this operand layout cannot be described to TMA (driver code %d)", static_cast<int>(result));
  return TQ_OK;
}

bool legal_strides(const void* pointer, const int64_t* strides, long long head_dim, long long tokens, long long heads, long long batch) {
  if (!aligned_to(pointer, 16)) return false;
  if (tokens > 1 && (strides[2] < head_dim || strides[2] % 8 != 0)) return false;
  if (heads > 1 && (strides[1] <= 0 || strides[1] % 8 != 0)) return false;
  if (batch > 1 && (strides[0] <= 0 || strides[0] % 8 != 0)) return false;
  return true;
}

}  // namespace

// decode.cu
tq_status attention_decode(tq_dtype dtype, const void* q, const void* k, const void* v, void* out, long long batch, long long heads,
                           long long q_tokens, long long k_tokens, long long head_dim, const int64_t* q_strides, const int64_t* k_strides,
                           const int64_t* v_strides, const int64_t* out_strides, float scale_log2, bool causal, int32_t device, cudaStream_t stream);
constexpr int kDecodeQueries = 4;

struct AttentionForm {
  bool decode;      // decode.cu
  int keys;         // keys a step of the tensor-core kernel
  bool few;         // its form for a few queries
};

// Kernel times (graphs of launches over rotating operands, B200, bf16, us) behind the rules. `heads` is batch times heads.
//
// One to four queries: streaming the keys (decode.cu) costs multiply-adds per query, the tensor cores' few-query form does not, but
// it walks a head's keys in one CTA. Four queries of 64 x 12 heads over 1000 keys: heads of 64 streamed 73, few 53; heads of 128
// 143 and 74; two queries of heads of 128 85 and 74, one 75 and 74; but over 100 keys, heads of 64, 14.0 and 17. Where heads do
// not fill the SMs a head's keys are shared when streamed: four queries of 8 heads of 128 over 4000 keys 36 and 47, of 96 heads
// 80 and 50. From there to one head an SM clusters of four no longer fit: one query, 144 heads of 96, 4000 keys 57 and 53.
//
// More queries: 128 keys a step halve the hand-overs of a chain, but only two CTAs share an SM (one for heads above 64)
// where 64 keys let three (two). 1 x 8 x 4096 causal 68.9 with 64, 54.4 with 128; 64 x 12 x 1024 causal 228.7 and 228.7; 5 ... 9 waves
// of 200 to 256 tokens 0 - 4 % better with 64; 64 x 6 x 1024 of 128 174.7 and 225. Without a mask, CTAs that fit
// three an SM but not two are one wave with 64 (384 CTAs over 4096 keys 90.6 and 92.9). Half of a 128-key step may be empty: of the only
// one (64 x 12 x 64 11.4 and 15.5) or of the last (without a mask 64 x 12 x 700 185.4 and 204).
AttentionForm choose_attention_form(long long heads, long long q_tokens, long long k_tokens, long long head_dim, bool causal, long long sms) {
  const bool wide = head_dim > kHeadDim;
  if (q_tokens <= kDecodeQueries) {
    const long long keys = causal && q_tokens < k_tokens ? q_tokens : k_tokens;       // that any query sees
    const bool no_fours = heads * 25 > sms * 24;                                    // clusters of four: 142 of them on 148 SMs
    if (heads > sms) {
      const long long enough = q_tokens >= 3 ? (wide ? heads / 4 : heads / 2) : heads;
      if ((wide ? q_tokens >= 2 : q_tokens >= 3) && keys >= enough && keys >= 64) return {false, 64, true};
    } else if (keys > kHeadDim) {
      const bool half = heads * 2 > sms;
      const bool many = q_tokens >= 3 && (wide ? half || keys <= 512 : keys <= 128 || (half && keys <= 300) || no_fours);
      if (many || (wide && no_fours && keys >= 256)) return {false, 128, true};
    }
    return {true, 0, false};
  }
  const long long ctas = heads * ((q_tokens + kRows - 1) / kRows);
  if (k_tokens <= 64) return {false, 64, false};
  if (wide) return {false, ctas <= sms ? 128 : 64, false};
  const bool thirds = !causal && ctas > 2 * sms && ctas <= 3 * sms;
  const bool half_step = !causal && k_tokens < 1280 && (k_tokens + 63) / 64 % 2 == 1;
  return {false, ctas <= 2 * sms || (k_tokens >= 512 && !thirds && !half_step) ? 128 : 64, false};
}

// Keys a step of the tensor-core tiles for window attention, or 0: the keys are streamed (keyed.cu), which shares a head's keys among all SMs but
// takes 16 rows of a key head at a time where a tile has 128 and walks its keys in one CTA. The smaller of two expected times, each coarser than
// what runs: the streamed one counts CTAs of four warps (keyed.cu has two, four or eight, by an estimate of its own), the tiles' 128 keys a step. Both
// sides measured (us, bf16; tiles / streamed): 12 heads of 64, 8000 keys, 8 queries 79 / 14.6, 128 queries 80 / 36, 300 queries 80 / 70; 8 x 12
// heads 40 queries 82 / 79 (the rule takes the tiles), 100 queries 83 / 183; 2000 keys, 17 queries 24.2 / 21.5 (tiles: the farthest from the
// better one of 20 shapes); 8 key heads of 128 for 32, 100 queries, 300 keys 8.7 / 10.2, 2000 keys 23.4 / 39, 8000 keys 80 / 105, 5 queries 79 /
// 20.5. Tiles: 128 keys a step where few CTAs leave the steps' latency bare (up to two an SM, one of heads above 64), and for heads up to 64
// where there are many steps: 8 x 12 x 4096 tokens under a window of 64 83.0 with 128 and 63.4 with 64, of 1024 179.5 and 177.8, of 4096 311.9 and
// 326.4; 2 x 32/8 x 2501 of 128 under 333 78.7 and 60.9.
int window_tile_keys(const KeyedParams& p, long long sms) {
  const bool wide = p.head_dim > kHeadDim;
  const long long rows = static_cast<long long>(p.group) * p.q_tokens;
  if (p.k_tokens == 0 || rows <= 16) return 0;      // (of one tile of rows streaming was the quicker in every case)
  const long long keys = p.window < p.k_tokens ? p.window : p.k_tokens;
  auto steps_of = [&](long long queries, long long step) {      // that some row of a block sees
    const long long all = (p.k_tokens + step - 1) / step, seen = (p.sinks + step - 1) / step + (keys + queries + step - 2) / step + 1;
    return all < seen ? all : seen;
  };
  const long long blocks = (p.q_tokens + kRows - 1) / kRows, ctas = blocks * p.heads * p.batch, at_once = wide ? sms : 2 * sms;
  const double tiles = 5.5 + 1.2 * steps_of(p.q_tokens < kRows ? p.q_tokens : kRows, 128) * (ctas > at_once ? static_cast<double>(ctas) / at_once : 1.0);
  const long long tile_rows = rows <= 8 ? 8 : 16, units = (rows + tile_rows - 1) / tile_rows * p.kv_heads * p.batch;
  const long long chunks = steps_of((tile_rows + p.group - 1) / p.group, wide ? 16 : 32);
  const bool whole = chunks <= 8 || (chunks <= 32 && units <= 4 * sms);      // a CTA a unit
  const double steps = static_cast<double>((chunks + 3) / 4), waves = units > 2 * sms ? units / (2.0 * sms) : 1.0;
  const double streamed = whole ? 1.0 + waves * (5.0 + steps) : 13.0 + units * chunks * 1.2 / (8.0 * sms);
  if (streamed <= tiles) return 0;
  return ctas <= at_once || (!wide && keys >= 2048) ? 128 : 64;
}

tq_status window_tiles(tq_dtype dtype, const KeyedParams& from, int keys, int sms, cudaStream_t stream) {
  CUtensorMap map_q, map_k, map_v;
  const int64_t q_strides[3] = {from.q_strides[0], from.q_strides[1], from.q_strides[2]}, k_strides[3] = {from.k_strides[0], from.k_strides[1], from.k_strides[2]},
                v_strides[3] = {from.v_strides[0], from.v_strides[1], from.v_strides[2]};
  if (tq_status s = attention_map(&map_q, dtype, from.q, from.head_dim, from.q_tokens, from.heads, from.batch, q_strides, kRows)) return s;
  if (tq_status s = attention_map(&map_k, dtype, from.k, from.head_dim, from.k_tokens, from.kv_heads, from.batch, k_strides, keys)) return s;
  if (tq_status s = attention_map(&map_v, dtype, from.v, from.head_dim, from.k_tokens, from.kv_heads, from.batch, v_strides, keys)) return s;
  WindowAttnParams p = {};
  p.batch = from.batch;
  p.heads = from.heads;
  p.q_tokens = from.q_tokens;
  p.k_tokens = from.k_tokens;
  p.head_dim = from.head_dim;
  p.q_blocks = (from.q_tokens + kRows - 1) / kRows;
  p.causal = 1;
  p.scale_log2 = from.scale_log2;
  p.out = from.out;
  p.out_batch = from.out_strides[0];
  p.out_head = from.out_strides[1];
  p.out_token = from.out_strides[2];
  p.out_vectors = from.head_dim % 8 == 0 && aligned_to(from.out, 16) &&
                  (((p.batch > 1 ? p.out_batch : 0) | (p.heads > 1 ? p.out_head : 0) | (p.q_tokens > 1 ? p.out_token : 0)) & 7) == 0;
  p.status = from.status;
  p.group = from.group;
  p.offset = from.k_tokens - from.q_tokens;
  p.window = from.window;
  p.sinks = from.sinks;
  p.q = from.q;
  p.k = from.k;
  p.v = from.v;
  for (int i = 0; i < 3; ++i) {
    p.q_strides[i] = from.q_strides[i];
    p.k_strides[i] = from.k_strides[i];
    p.v_strides[i] = from.v_strides[i];
  }
  const long long blocks = static_cast<long long>(p.q_blocks) * p.heads * p.batch;
  TQ_REQUIRE(blocks < (1LL << 30), TQ_UNSUPPORTED, "too many query blocks for one launch");
  auto go = [&](auto width, auto step) -> tq_status {
    constexpr int kWidth = decltype(width)::value, kKeys = decltype(step)::value;
    constexpr size_t smem = WindowLayout<kWidth, kKeys>::kSmemBytes;
    auto start = [&](auto kernel) -> tq_status {
      TQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
      const long long fit = static_cast<long long>(sms) * AttnLayout<kWidth, kKeys, false>::kCtasPerSm;
      TQ_CUDA(launch_overlapped(kernel, dim3(static_cast<unsigned>(blocks < fit ? blocks : fit)), kAttnThreads, smem, stream, map_q, map_k, map_v, p));
      return check_launch("window_attention_kernel");
    };
    if (dtype == TQ_BF16) return start(window_attention_kernel<__nv_bfloat16, kWidth, kKeys>);
    return start(window_attention_kernel<__half, kWidth, kKeys>);
  };
  auto with_keys = [&](auto width) {
    return keys == 128 ? go(width, std::integral_constant<int, 128>{}) : go(width, std::integral_constant<int, 64>{});
  };
  return from.head_dim > kHeadDim ? with_keys(std::integral_constant<int, 2 * kHeadDim>{}) : with_keys(std::integral_constant<int, kHeadDim>{});
}

}  // namespace tq

extern "C" tq_status tq_attention_form(int64_t heads, int64_t q_tokens, int64_t k_tokens, int64_t head_dim, int32_t causal, int32_t device, int32_t* form,
                                       int32_t* keys) {
  TQ_REQUIRE(form != nullptr && keys != nullptr, TQ_INVALID_ARGUMENT, "null out-pointer");
  TQ_REQUIRE(heads > 0 && q_tokens > 0 && k_tokens > 0, TQ_INVALID_ARGUMENT, "extents must be positive, not heads=%lld q_tokens=%lld k_tokens=%lld",
             (long long)heads, (long long)q_tokens, (long long)k_tokens);
  TQ_REQUIRE(head_dim >= 8 && head_dim <= 2 * tq::kHeadDim && head_dim % 8 == 0, TQ_UNSUPPORTED,
             "fused attention has a kernel for heads of 8, 16, ... %d elements, not %lld", 2 * tq::kHeadDim, (long long)head_dim);
  const tq::AttentionForm chosen = tq::choose_attention_form(heads, q_tokens, k_tokens, head_dim, causal != 0, device < 0 ? 148 : tq::sm_count(device));
  *form = chosen.decode ? TQ_ATTENTION_STREAMED : chosen.few ? TQ_ATTENTION_TILES_FEW : TQ_ATTENTION_TILES;
  *keys = chosen.keys;
  return TQ_OK;
}

extern "C" tq_status tq_attention_launch(tq_dtype dtype, const void* q, const void* k, const void* v, void* out, int64_t batch,
                                         int64_t heads, int64_t q_tokens, int64_t k_tokens, int64_t head_dim,
                                         const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                         const int64_t* out_strides, double scale, int32_t causal, int32_t device, void* stream) {
  TQ_REQUIRE(q_strides != nullptr && k_strides != nullptr && v_strides != nullptr && out_strides != nullptr, TQ_INVALID_ARGUMENT,
             "null strides");
  if (tq::recording()) {
    struct Kept { int64_t q[3], k[3], v[3], out[3]; } kept;
    for (int i = 0; i < 3; ++i) {
      kept.q[i] = q_strides[i];
      kept.k[i] = k_strides[i];
      kept.v[i] = v_strides[i];
      kept.out[i] = out_strides[i];
    }
    return tq::record([=](int32_t d, void* s) {
      return tq_attention_launch(dtype, q, k, v, out, batch, heads, q_tokens, k_tokens, head_dim, kept.q, kept.k, kept.v, kept.out,
                                 scale, causal, d, s);
    });
  }
  TQ_REQUIRE(dtype == TQ_BF16 || dtype == TQ_F16, TQ_UNSUPPORTED, "fused attention takes bf16 or f16 operands, not %s",
             tq::dtype_name(dtype));
  TQ_REQUIRE(batch >= 0 && heads >= 0 && q_tokens >= 0 && k_tokens >= 0, TQ_INVALID_ARGUMENT,
             "negative extent in batch=%lld heads=%lld q_tokens=%lld k_tokens=%lld", (long long)batch, (long long)heads,
             (long long)q_tokens, (long long)k_tokens);
  TQ_REQUIRE(head_dim >= 8 && head_dim <= 2 * tq::kHeadDim && head_dim % 8 == 0, TQ_UNSUPPORTED,
             "fused attention has a kernel for heads of 8, 16, ... %d elements, not %lld", 2 * tq::kHeadDim, (long long)head_dim);
  if (batch == 0 || heads == 0 || q_tokens == 0) return TQ_OK;
  TQ_REQUIRE(k_tokens > 0, TQ_UNSUPPORTED, "a softmax over no keys has no kernel");
  TQ_REQUIRE(std::isfinite(scale) && scale > 0.0, TQ_UNSUPPORTED, "the score scale must be positive and finite, not %g", scale);
  TQ_REQUIRE(q != nullptr && k != nullptr && v != nullptr && out != nullptr, TQ_INVALID_ARGUMENT, "null operand or result");
  TQ_REQUIRE(q_tokens < (1LL << 30) && k_tokens < (1LL << 30) && heads < 65536 && batch * heads < (1LL << 24), TQ_UNSUPPORTED,
             "extents beyond the kernel's index range");
  TQ_REQUIRE(tq::legal_strides(q, q_strides, head_dim, q_tokens, heads, batch) && tq::legal_strides(k, k_strides, head_dim, k_tokens, heads, batch) &&
                 tq::legal_strides(v, v_strides, head_dim, k_tokens, heads, batch),
             TQ_UNSUPPORTED, "Q, K and V must be 16-byte aligned with positive strides that are multiples of 8 elements (TMA's rules)");
  TQ_REQUIRE(tq::aligned_to(out, 2) && out_strides[0] >= 0 && out_strides[1] >= 0 && out_strides[2] >= 0, TQ_INVALID_ARGUMENT,
             "misaligned result or negative result stride");
  tq::DeviceScope device_scope(device);
  if (tq_status s = device_scope.status()) return s;
  const bool wide = head_dim > tq::kHeadDim;             // two sub-tiles side by side
  const tq::AttentionForm form = tq::choose_attention_form(batch * heads, q_tokens, k_tokens, head_dim, causal != 0, tq::sm_count(device));
  // (The decoding form's batch * heads * split CTAs stay below 2^28.)
  if (form.decode) {
    return tq::attention_decode(dtype, q, k, v, out, batch, heads, q_tokens, k_tokens, head_dim, q_strides, k_strides, v_strides, out_strides,
                                static_cast<float>(scale * 1.4426950408889634), causal != 0, device, static_cast<cudaStream_t>(stream));
  }
  const tq::WaitStatus status = tq::wait_status_for(device);
  TQ_REQUIRE(status.abort != nullptr, TQ_RESOURCE_EXHAUSTED, "no device memory for the status word");

  CUtensorMap map_q, map_k, map_v;
  if (tq_status s = tq::attention_map(&map_q, dtype, q, head_dim, q_tokens, heads, batch, q_strides, tq::kRows)) return s;
  if (tq_status s = tq::attention_map(&map_k, dtype, k, head_dim, k_tokens, heads, batch, k_strides, form.keys)) return s;
  if (tq_status s = tq::attention_map(&map_v, dtype, v, head_dim, k_tokens, heads, batch, v_strides, form.keys)) return s;

  tq::AttnParams p = {};
  p.batch = static_cast<int>(batch);
  p.heads = static_cast<int>(heads);
  p.q_tokens = static_cast<int>(q_tokens);
  p.k_tokens = static_cast<int>(k_tokens);
  p.head_dim = static_cast<int>(head_dim);
  p.q_blocks = static_cast<int>((q_tokens + tq::kRows - 1) / tq::kRows);
  p.causal = causal != 0;
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  p.out = out;
  p.out_batch = out_strides[0];
  p.out_head = out_strides[1];
  p.out_token = out_strides[2];
  p.status = status;
  const long long ctas = static_cast<long long>(p.q_blocks) * heads * batch;
  TQ_REQUIRE(ctas < (1LL << 31), TQ_UNSUPPORTED, "too many query blocks for one launch");
  cudaStream_t cuda_stream = static_cast<cudaStream_t>(stream);
  auto go = [&](auto width, auto keys, auto few) -> tq_status {
    constexpr int kWidth = decltype(width)::value, kKeys = decltype(keys)::value;
    constexpr bool kFew = decltype(few)::value;
    constexpr size_t smem = tq::AttnLayout<kWidth, kKeys, kFew>::kSmemBytes;
    auto start = [&](auto kernel) -> tq_status {
      TQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
      kernel<<<static_cast<unsigned>(ctas), tq::kAttnThreads, smem, cuda_stream>>>(map_q, map_k, map_v, p);
      return tq::check_launch("attention_kernel");
    };
    if (dtype == TQ_BF16) return start(tq::attention_kernel<__nv_bfloat16, kWidth, kKeys, kFew>);
    return start(tq::attention_kernel<__half, kWidth, kKeys, kFew>);
  };
  auto with_width = [&](auto keys, auto few) {
    return wide ? go(std::integral_constant<int, 2 * tq::kHeadDim>{}, keys, few) : go(std::integral_constant<int, tq::kHeadDim>{}, keys, few);
  };
  auto with_keys = [&](auto few) {
    return form.keys == 128 ? with_width(std::integral_constant<int, 128>{}, few) : with_width(std::integral_constant<int, 64>{}, few);
  };
  return form.few ? with_keys(std::true_type{}) : with_keys(std::false_type{});
}

extern "C" tq_status tq_window_attention_form(int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_tokens, int64_t k_tokens, int64_t head_dim, int64_t window,
                                              int64_t sinks, int32_t device, int32_t* form, int32_t* keys) {
  TQ_REQUIRE(form != nullptr && keys != nullptr, TQ_INVALID_ARGUMENT, "null out-pointer");
  TQ_REQUIRE(batch > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && q_tokens > 0 && k_tokens > 0 && window >= 0 && sinks >= 0 && k_tokens < (1LL << 30) &&
                 q_tokens < (1LL << 24) && batch * heads < (1LL << 24),
             TQ_INVALID_ARGUMENT, "no such launch");
  tq::KeyedParams p = {};
  tq::keyed_extents(p, batch, heads, kv_heads, q_tokens, head_dim, 1.0, window, sinks);
  p.k_tokens = static_cast<int>(k_tokens);
  *keys = tq::window_tile_keys(p, device < 0 ? 148 : tq::sm_count(device));
  *form = *keys == 0 ? TQ_ATTENTION_STREAMED : TQ_ATTENTION_TILES;
  return TQ_OK;
}

extern "C" tq_status tq_window_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t q_tokens, int64_t k_tokens,
                                                         int64_t head_dim, int64_t window, int64_t sinks, int32_t device, size_t* bytes) {
  TQ_REQUIRE(bytes != nullptr, TQ_INVALID_ARGUMENT, "null out-pointer");
  *bytes = 0;
  // (of what the launch has nothing to do for, or refuses: nothing)
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || q_tokens <= 0 || k_tokens <= 0 || k_tokens >= (1LL << 30) || q_tokens >= (1LL << 24) ||
      batch * heads >= (1LL << 24) || window < 0 || sinks < 0 || head_dim <= 0 || head_dim > 2 * tq::kHeadDim)
    return TQ_OK;
  tq::KeyedParams p = {};
  tq::keyed_extents(p, batch, heads, kv_heads, q_tokens, head_dim, 1.0, window, sinks);
  p.k_tokens = static_cast<int>(k_tokens);
  if (tq::window_tile_keys(p, tq::sm_count(device)) == 0) *bytes = tq::keyed_workspace(false, p, k_tokens, device);
  return TQ_OK;
}

extern "C" tq_status tq_window_attention_launch(tq_dtype dtype, const void* q, const void* k, const void* v, void* out, int64_t batch, int64_t heads,
                                                int64_t kv_heads, int64_t q_tokens, int64_t k_tokens, int64_t head_dim, const int64_t* q_strides,
                                                const int64_t* k_strides, const int64_t* v_strides, const int64_t* out_strides, double scale,
                                                int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes, int32_t device, void* stream) {
  TQ_REQUIRE(q_strides != nullptr && k_strides != nullptr && v_strides != nullptr && out_strides != nullptr, TQ_INVALID_ARGUMENT,
             "null strides");
  if (tq::recording()) {
    struct Kept { int64_t q[3], k[3], v[3], out[3]; } kept;
    for (int i = 0; i < 3; ++i) {
      kept.q[i] = q_strides[i];
      kept.k[i] = k_strides[i];
      kept.v[i] = v_strides[i];
      kept.out[i] = out_strides[i];
    }
    return tq::record([=](int32_t d, void* s) {
      return tq_window_attention_launch(dtype, q, k, v, out, batch, heads, kv_heads, q_tokens, k_tokens, head_dim, kept.q, kept.k, kept.v, kept.out, scale,
                                        window, sinks, workspace, workspace_bytes, d, s);
    });
  }
  TQ_REQUIRE(dtype == TQ_BF16 || dtype == TQ_F16, TQ_UNSUPPORTED, "window attention takes bf16 or f16 operands, not %s", tq::dtype_name(dtype));
  TQ_REQUIRE(batch >= 0 && heads >= 0 && kv_heads >= 0 && q_tokens >= 0 && k_tokens >= 0 && window >= 0 && sinks >= 0, TQ_INVALID_ARGUMENT,
             "negative extent in batch=%lld heads=%lld kv_heads=%lld q_tokens=%lld k_tokens=%lld window=%lld sinks=%lld", (long long)batch,
             (long long)heads, (long long)kv_heads, (long long)q_tokens, (long long)k_tokens, (long long)window, (long long)sinks);
  TQ_REQUIRE(head_dim >= 8 && head_dim <= 2 * tq::kHeadDim && head_dim % 8 == 0, TQ_UNSUPPORTED,
             "window attention has a kernel for heads of 8, 16, ... %d elements, not %lld", 2 * tq::kHeadDim, (long long)head_dim);
  if (batch == 0 || heads == 0 || q_tokens == 0) return TQ_OK;
  TQ_REQUIRE(kv_heads > 0 && heads % kv_heads == 0, TQ_INVALID_ARGUMENT, "%lld heads do not share %lld key heads evenly", (long long)heads, (long long)kv_heads);
  TQ_REQUIRE(scale > 0.0 && scale <= tq::kKeyedMostScale, TQ_UNSUPPORTED, "the score scale must be positive and finite in f32, not %g", scale);
  TQ_REQUIRE(q != nullptr && out != nullptr && (k_tokens == 0 || (k != nullptr && v != nullptr)), TQ_INVALID_ARGUMENT, "null operand or result");
  TQ_REQUIRE(q_tokens < (1LL << 24) && k_tokens < (1LL << 30) && heads < 65536 && batch * heads < (1LL << 24) && heads / kv_heads * q_tokens < (1LL << 24),
             TQ_UNSUPPORTED, "extents beyond the kernel's index range");
  TQ_REQUIRE(tq::legal_strides(q, q_strides, head_dim, q_tokens, heads, batch) && tq::legal_strides(k, k_strides, head_dim, k_tokens, kv_heads, batch) &&
                 tq::legal_strides(v, v_strides, head_dim, k_tokens, kv_heads, batch),
             TQ_UNSUPPORTED, "Q, K and V must be 16-byte aligned with positive strides that are multiples of 8 elements (TMA's rules)");
  TQ_REQUIRE(tq::keyed_query_fits(q, q_strides, out, out_strides, batch, heads, q_tokens), TQ_INVALID_ARGUMENT,
             "misaligned result or negative result stride");
  tq::DeviceScope device_scope(device);
  if (tq_status s = device_scope.status()) return s;
  tq::KeyedParams p = {};
  p.status = tq::wait_status_for(device);
  TQ_REQUIRE(p.status.abort != nullptr, TQ_RESOURCE_EXHAUSTED, "no device memory for the status word");
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  for (int i = 0; i < 3; ++i) {
    p.q_strides[i] = q_strides[i];
    p.k_strides[i] = k_strides[i];
    p.v_strides[i] = v_strides[i];
    p.out_strides[i] = out_strides[i];
  }
  p.k_tokens = static_cast<int>(k_tokens);
  tq::keyed_extents(p, batch, heads, kv_heads, q_tokens, head_dim, scale, window, sinks);
  const int tile_keys = tq::window_tile_keys(p, tq::sm_count(device));
  if (tile_keys != 0) return tq::window_tiles(dtype, p, tile_keys, tq::sm_count(device), static_cast<cudaStream_t>(stream));
  return tq::keyed_attention(dtype, false, p, k_tokens, workspace, workspace_bytes, device, static_cast<cudaStream_t>(stream));
}
