// Attention of a few query rows a head against many keys, with a window, sinks and shared key heads, for sm_100a: over a
// paged cache in 8 bits, or over dense keys and values in 16.
//
//   position of query i of a sequence of L keys and Q queries: p = L - Q + i (aligned at the ends)
//   out_i = sum_j softmax_j(scale * q_i . k_j) v_j    over j <= p with (j > p - window or j < sinks); zeros where p < 0
//   8 bits: k_j = code_j * k_scale[page, head], v_j likewise (e4m3 codes, an f32 scale a page and head)
//
// Heads that share a key head are rows of one tile, so a key is read once for all of them. Bound: HBM (the visible keys' and
// values' bytes); the multiply-adds of up to 16 rows would not fit the CUDA cores beside it, so both products are warp-level
// matrix instructions over keys and values that go from memory to registers in the instructions' own layout, without
// shared memory: the order of the summed-over axis of a product is free, so a lane's 16 contiguous bytes of a key are
// whatever elements of the head the instruction takes from it, and the query is laid out to match. Transposed, S^T = K Q^T
// and O^T = V^T P^T: keys (then head elements) are the instruction's 16 rows and query rows its 8 columns, so that a
// head of its own wastes 7 columns of 8 and not 15 rows of 16.
//
// Precision: scores, maxima, sums and results in f32. e4m3 to f16 is exact, and so is the query in f16: a row is scaled by a power of two to
// a maximum of 2^14, so only elements 2^-38 of it or less lose digits. Probabilities against f16 values (cache codes too) are rounded to
// f16 (half a step is 2^-12, under the result's 2^-9 in bf16); against bf16 values they take two bf16 operands, the
// rounded value and what rounding took off (2^-17).
//
// A masked key must not reach a result through 0 * NaN: its score is replaced, and where the rows of a tile see a chunk's keys
// alike its value is replaced by zeros. Where they do not (several queries, at an end of the window) the chunk's product is
// taken once a query with that query's keys alone, and each row keeps its own.
#include <cmath>
#include <type_traits>

#include "common.h"
#include "keyed.h"
#include "tcgen05.h"

namespace tq {
namespace {

constexpr int kKeyedWarps = 4;
constexpr int kKeyedThreads = 32 * kKeyedWarps;

// BITS of a key element, W: the head's elements, rounded up to 64 or 128.
template <int BITS, int W>
struct KeyedShape {
  static constexpr int kKeys = BITS == 16 && W == 128 ? 16 : 32;      // a chunk: what a warp takes at a time
  static constexpr int kTiles = kKeys / 16;
  static constexpr int kPieces = W * BITS / 512;                      // 16-byte pieces of a key a lane holds (four lanes a key)
  static constexpr int kPieceWidth = 128 / BITS;                      // head elements in one
  static constexpr int kValueWords = W * BITS / 256;                  // 32-bit words of a value a lane holds (eight lanes a value)
  static constexpr int kSlices = W / 16;                              // 16 head elements of the result
};

__device__ __forceinline__ uint4 load_piece(const void* pointer) {
  uint4 word;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(word.x), "=r"(word.y), "=r"(word.z), "=r"(word.w) : "l"(pointer));
  return word;
}
__device__ __forceinline__ uint2 load_half_piece(const void* pointer) {
  uint2 word;
  asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(word.x), "=r"(word.y) : "l"(pointer));
  return word;
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

template <typename M>
__device__ __forceinline__ void multiply(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<M, __half>) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
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

// T: the type of q and out. BITS, W as above. NT: eights of rows of a tile.
template <typename T, int BITS, int W, int NT>
__global__ void __launch_bounds__(kKeyedThreads) keyed_attention_kernel(const __grid_constant__ KeyedParams p) {
  using S = KeyedShape<BITS, W>;
  using M = std::conditional_t<BITS == 8, __half, T>;      // what the matrix instructions take
  constexpr bool kTwoOperands = std::is_same_v<M, __nv_bfloat16>;
  constexpr int kRows = 8 * NT, kTiles = S::kTiles, kSlices = S::kSlices;
  __shared__ float part_top[kKeyedWarps][kRows], part_sum[kKeyedWarps][kRows];
  __shared__ __align__(16) float part_out[kKeyedWarps][kRows][W];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = lane >> 2, corner = lane & 3;       // the instruction's row (or column) of eight, and the lane's place in it

  const long long unit = blockIdx.x;
  const int tile = static_cast<int>(unit % p.row_tiles);
  const long long head_index = unit / p.row_tiles;
  const int kv_head = static_cast<int>(head_index % p.kv_heads), batch = static_cast<int>(head_index / p.kv_heads);
  const int rows = p.group * p.q_tokens;               // of a key head: row = token * group + head in the group
  const int row0 = tile * kRows;

  int length = p.k_tokens;
  if constexpr (BITS == 8) {
    length = max(p.lengths[batch], 0);
    if (length > p.blocks << p.page_shift) {           // the table does not go that far
      length = p.blocks << p.page_shift;
      if (threadIdx.x == 0) report(p.status, kKeyedLength, batch, p.lengths[batch]);
    }
  }
  const int first_token = row0 / p.group, last_token = min(row0 + kRows, rows) - 1 < 0 ? 0 : (min(row0 + kRows, rows) - 1) / p.group;
  const int low = length - p.q_tokens + first_token, high = length - p.q_tokens + last_token;
  const ChunkList list = chunks_of(low, max(high, -1), p.window, p.sinks, S::kKeys);

  // The query: row `quad` of each eight, the elements that the lane's pieces of a key hold.
  uint32_t query[NT][S::kPieces][32 / BITS][2];      // [piece][step of 16 elements][operand word]
  float row_scale[NT][2];                                        // of the lane's two columns: rows 2 corner and 2 corner + 1
  int position[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = row0 + n * 8 + quad;
    const int token = row / p.group, head = kv_head * p.group + row % p.group;
    const T* from = static_cast<const T*>(p.q) + batch * p.q_strides[0] + head * p.q_strides[1] + token * p.q_strides[2];
    constexpr int kWords = S::kPieceWidth / 2;                   // of a piece's query elements: 8 or 4
    uint32_t word[S::kPieces][kWords];
    float largest = 0.f;
#pragma unroll
    for (int j = 0; j < S::kPieces; ++j) {
      const int column = (4 * j + corner) * S::kPieceWidth;
#pragma unroll
      for (int w = 0; w < kWords; w += 4) {
        uint4 four = make_uint4(0, 0, 0, 0);
        if (row < rows && column + 2 * w < p.head_dim) four = *reinterpret_cast<const uint4*>(from + column + 2 * w);
        word[j][w] = four.x;
        word[j][w + 1] = four.y;
        word[j][w + 2] = four.z;
        word[j][w + 3] = four.w;
      }
      if constexpr (BITS == 8) {
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          const float2 pair = widen_pair<T>(word[j][w]);
          largest = fmaxf(largest, fmaxf(fabsf(pair.x), fabsf(pair.y)));
        }
      }
    }
    float back = p.scale_log2;
    if constexpr (BITS == 8) {
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
      // a power of two that brings the row's largest element to [2^14, 2^15); none for zeros and infinities
      int exponent = static_cast<int>(__float_as_uint(largest) >> 23) - 127;
      if (exponent < -100 || exponent > 127) exponent = 14;
      const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - exponent) << 23);
      back *= __uint_as_float(static_cast<uint32_t>(127 - 14 + exponent) << 23);
#pragma unroll
      for (int j = 0; j < S::kPieces; ++j) {
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          const float2 pair = widen_pair<T>(word[j][w]);
          word[j][w] = round_pair<__half>(pair.x * up, pair.y * up);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < S::kPieces; ++j) {
#pragma unroll
      for (int w = 0; w < kWords; ++w) query[n][j][w / 2][w % 2] = word[j][w];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      row_scale[n][e] = __shfl_sync(0xffffffffu, back, (2 * corner + e) * 4);
      const int mine = row0 + n * 8 + 2 * corner + e;
      position[n][e] = mine < rows ? length - p.q_tokens + mine / p.group : high;
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

  const int chunks = list.count();
  for (int i = warp; i < chunks; i += kKeyedWarps) {
    const int key0 = list.at(i) * S::kKeys;
    // where the chunk's tiles of 16 keys lie
    const char *k_base[kTiles], *v_base[kTiles];
    float k_scale[kTiles], v_scale[kTiles];
    long long k_step, v_step;                          // bytes from a key to the next
    int stop = length;                                 // keys from here on are not there
    if constexpr (BITS == 8) {
      k_step = v_step = p.head_dim;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const int key = key0 + t * 16;
        k_base[t] = v_base[t] = nullptr;
        k_scale[t] = v_scale[t] = 0.f;
        if (key < stop) {
          const int page = p.table[batch * p.table_stride + (key >> p.page_shift)];
          if (page < 0 || page >= p.pages) {
            if (lane == 0) report(p.status, kKeyedPage, batch, key >> p.page_shift);
            stop = key;
          } else {
            const long long block = static_cast<long long>(page) * p.kv_heads + kv_head;
            const long long offset = ((block << p.page_shift) + (key & ((1 << p.page_shift) - 1))) * p.head_dim;
            k_base[t] = static_cast<const char*>(p.k) + offset;
            v_base[t] = static_cast<const char*>(p.v) + offset;
            k_scale[t] = p.k_scales[block];
            v_scale[t] = p.v_scales[block];
          }
        }
      }
    } else {
      k_step = p.k_strides[2] * 2;
      v_step = p.v_strides[2] * 2;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const long long key = key0 + t * 16;
        k_base[t] = static_cast<const char*>(p.k) + (batch * p.k_strides[0] + kv_head * p.k_strides[1] + key * p.k_strides[2]) * 2;
        v_base[t] = static_cast<const char*>(p.v) + (batch * p.v_strides[0] + kv_head * p.v_strides[1] + key * p.v_strides[2]) * 2;
      }
    }
    uint4 key_piece[kTiles][2][S::kPieces];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int inside = quad + 8 * h;
#pragma unroll
        for (int j = 0; j < S::kPieces; ++j) {
          const int column = (4 * j + corner) * S::kPieceWidth;
          key_piece[t][h][j] = make_uint4(0, 0, 0, 0);
          if (column < p.head_dim && key0 + t * 16 + inside < stop) key_piece[t][h][j] = load_piece(k_base[t] + inside * k_step + column * BITS / 8);
        }
      }
    }
    uint32_t value[kTiles][4][S::kValueWords];         // keys 2 corner, 2 corner + 1, and those 8 further on
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int inside = 2 * corner + (r & 1) + 8 * (r >> 1);
        const bool there = key0 + t * 16 + inside < stop;
        const char* from = v_base[t] + inside * v_step;
        if constexpr (S::kValueWords == 2) {
          uint2 word = make_uint2(0, 0);
          if (there && quad * 8 < p.head_dim) word = load_half_piece(from + quad * 8);
          value[t][r][0] = word.x;
          value[t][r][1] = word.y;
        } else {
#pragma unroll
          for (int w = 0; w < S::kValueWords; w += 4) {
            const int column = (w / 4) * 64 + quad * S::kPieceWidth;
            uint4 word = make_uint4(0, 0, 0, 0);
            if (there && column < p.head_dim) word = load_piece(from + column * BITS / 8);
            value[t][r][w] = word.x;
            value[t][r][w + 1] = word.y;
            value[t][r][w + 2] = word.z;
            value[t][r][w + 3] = word.w;
          }
        }
      }
    }

    // S^T: keys quad and quad + 8 of each tile by rows 2 corner and 2 corner + 1
    float score[kTiles][NT][4];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
#pragma unroll
      for (int n = 0; n < NT; ++n) score[t][n][0] = score[t][n][1] = score[t][n][2] = score[t][n][3] = 0.f;
#pragma unroll
      for (int j = 0; j < S::kPieces; ++j) {
        const uint32_t a[4] = {key_piece[t][0][j].x, key_piece[t][0][j].y, key_piece[t][0][j].z, key_piece[t][0][j].w};
        const uint32_t b[4] = {key_piece[t][1][j].x, key_piece[t][1][j].y, key_piece[t][1][j].z, key_piece[t][1][j].w};
        if constexpr (BITS == 8) {
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const uint32_t a0 = decode_low(a[s]), a1 = decode_low(b[s]), a2 = decode_high(a[s]), a3 = decode_high(b[s]);
#pragma unroll
            for (int n = 0; n < NT; ++n) multiply<M>(score[t][n], a0, a1, a2, a3, query[n][j][s][0], query[n][j][s][1]);
          }
        } else {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
              multiply<M>(score[t][n], a[2 * s], b[2 * s], a[2 * s + 1], b[2 * s + 1], query[n][j][s][0], query[n][j][s][1]);
          }
        }
      }
    }

    // A chunk whose keys every row sees needs no mask.
    const int last = key0 + S::kKeys - 1;
    const bool open = last <= low && last < stop && (key0 > high - p.window || last < p.sinks);
    auto sees = [&](int at, int key) { return key <= at && key < stop && (key > at - p.window || key < p.sinks); };
    float factor[NT][2];
    bool moved = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float most = -INFINITY;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const float by = BITS == 8 ? row_scale[n][e] * k_scale[t] : row_scale[n][e];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& s = score[t][n][2 * h + e];
            s *= by;
            if (!open && !sees(position[n][e], key0 + t * 16 + quad + 8 * h)) s = -INFINITY;
            most = fmaxf(most, s);
          }
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
        most = fmaxf(most, top[n][e]);
        factor[n][e] = rescale(top[n][e], most);
        moved |= factor[n][e] != 1.f;
        top[n][e] = most;
        const float reference = most == -INFINITY ? 0.f : most;
        float gained = 0.f;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& s = score[t][n][2 * h + e];
            s = exp2_ftz(s - reference);
            gained += s;
          }
        }
        sum[n][e] = sum[n][e] * factor[n][e] + gained;
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int s = 0; s < kSlices; ++s) {
#pragma unroll
          for (int e = 0; e < 4; ++e) result[n][s][e] *= factor[n][e & 1];
        }
      }
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

    // O^T += V^T P^T of one tile of keys, for the rows of token `only` (all rows: -1) and the keys that `kept` has (a bit for each of the lane's four)
    auto add_product = [&](int t, uint32_t kept, int only) {
#pragma unroll
      for (int w = 0; w < S::kValueWords; ++w) {
        uint32_t v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = value[t][r][w] & (kept >> r & 1 ? 0xffffffffu : 0u);
#pragma unroll
        for (int half = 0; half < (BITS == 8 ? 2 : 1); ++half) {
          uint32_t a0, a1, a2, a3;
          if constexpr (BITS == 8) {
            const uint32_t near = __byte_perm(v[0], v[1], half ? 0x7362 : 0x5140), far = __byte_perm(v[2], v[3], half ? 0x7362 : 0x5140);
            a0 = decode_low(near);
            a1 = decode_high(near);
            a2 = decode_low(far);
            a3 = decode_high(far);
          } else {
            a0 = __byte_perm(v[0], v[1], 0x5410);
            a1 = __byte_perm(v[0], v[1], 0x7632);
            a2 = __byte_perm(v[2], v[3], 0x5410);
            a3 = __byte_perm(v[2], v[3], 0x7632);
          }
          const int slice = BITS == 8 ? 2 * w + half : w;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (BITS == 16 && only < 0) {
              multiply<M>(result[n][slice], a0, a1, a2, a3, weight[t][n][0], weight[t][n][1]);
              if constexpr (kTwoOperands) multiply<M>(result[n][slice], a0, a1, a2, a3, rest[t][n][0], rest[t][n][1]);
            } else {
              float d[4] = {0.f, 0.f, 0.f, 0.f};
              multiply<M>(d, a0, a1, a2, a3, weight[t][n][0], weight[t][n][1]);
              if constexpr (kTwoOperands) multiply<M>(d, a0, a1, a2, a3, rest[t][n][0], rest[t][n][1]);
              const float by = BITS == 8 ? v_scale[t] : 1.f;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (only < 0 || position[n][e & 1] == only) result[n][slice][e] = fmaf(d[e], by, result[n][slice][e]);
              }
            }
          }
        }
      }
    };
    if (open) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) add_product(t, 15u, -1);
    } else {
#pragma unroll 1
      for (int at = low; at <= high; ++at) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          uint32_t kept = 0;
#pragma unroll
          for (int r = 0; r < 4; ++r) kept |= (sees(at, key0 + t * 16 + 2 * corner + (r & 1) + 8 * (r >> 1)) ? 1u : 0u) << r;
          if (__any_sync(0xffffffffu, kept != 0)) add_product(t, kept, at);
        }
      }
    }
  }

  // The warps meet in shared memory.
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int offset = 4; offset < 32; offset *= 2) sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], offset);
      const int row = n * 8 + 2 * corner + e;
      if (quad == 0) {
        part_top[warp][row] = top[n][e];
        part_sum[warp][row] = sum[n][e];
      }
#pragma unroll
      for (int s = 0; s < kSlices; ++s) {
        const int column = BITS == 8 ? quad * (W / 8) + 2 * s : (s / 4) * 64 + quad * 8 + 2 * (s % 4);
        *reinterpret_cast<float2*>(&part_out[warp][row][column]) = make_float2(result[n][s][e], result[n][s][2 + e]);
      }
    }
  }
  __syncthreads();
  for (int item = threadIdx.x; item < kRows * (W / 8); item += kKeyedThreads) {
    const int row = item / (W / 8), column = item % (W / 8) * 8;
    const int mine = row0 + row;
    if (mine >= rows || column >= p.head_dim) continue;
    float most = part_top[0][row];
#pragma unroll
    for (int w = 1; w < kKeyedWarps; ++w) most = fmaxf(most, part_top[w][row]);
    float total = 0.f, value[8] = {};
#pragma unroll
    for (int w = 0; w < kKeyedWarps; ++w) {
      const float by = rescale(part_top[w][row], most);
      total += part_sum[w][row] * by;
#pragma unroll
      for (int c = 0; c < 8; ++c) value[c] += part_out[w][row][column + c] * by;
    }
    const int token = mine / p.group, head = kv_head * p.group + mine % p.group;
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
}

template <typename T, int BITS, int W, int NT>
tq_status launch_keyed(const KeyedParams& p, cudaStream_t stream) {
  const long long units = static_cast<long long>(p.batch) * p.kv_heads * p.row_tiles;
  TQ_REQUIRE(units < (1LL << 31), TQ_UNSUPPORTED, "too many heads and rows for one launch");
  keyed_attention_kernel<T, BITS, W, NT><<<static_cast<unsigned>(units), kKeyedThreads, 0, stream>>>(p);
  return check_launch("keyed_attention_kernel");
}

template <typename T, int BITS>
tq_status launch_keyed_width(KeyedParams& p, cudaStream_t stream) {
  const int rows = p.group * p.q_tokens;
  const int nt = rows <= 8 ? 1 : 2;
  p.row_tiles = (rows + 8 * nt - 1) / (8 * nt);
  if (p.head_dim <= 64) return nt == 1 ? launch_keyed<T, BITS, 64, 1>(p, stream) : launch_keyed<T, BITS, 64, 2>(p, stream);
  return nt == 1 ? launch_keyed<T, BITS, 128, 1>(p, stream) : launch_keyed<T, BITS, 128, 2>(p, stream);
}

}  // namespace

tq_status keyed_attention(tq_dtype dtype, bool paged, KeyedParams& p, cudaStream_t stream) {
  if (dtype == TQ_BF16) return paged ? launch_keyed_width<__nv_bfloat16, 8>(p, stream) : launch_keyed_width<__nv_bfloat16, 16>(p, stream);
  return paged ? launch_keyed_width<__half, 8>(p, stream) : launch_keyed_width<__half, 16>(p, stream);
}

}  // namespace tq
