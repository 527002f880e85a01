// Attention over the paged 4-bit cache (include/dimmerkv.h states the cache): softmax(scaling * q k^T) v for the newest
// tokens of many requests, causal, optionally within a sliding window, query heads sharing KV heads.
//
// One pass over the pages with the running maximum and sum of a softmax.  The rows of a workgroup are query heads that
// share a KV head, times consecutive tokens; its four waves take chunks of tokens in turn and join at the end, so nothing
// is shared between them on the way: no barrier, no staging.  Codes become matrix operands in registers, one conversion
// for two values:
//   scores^T = K q^T: operand A is 16 tokens x 32 dimensions, a lane's part of a row being 16 consecutive bytes (D = 128)
//     of one block, so one load and one exponent; the dimensions' order in the products is the queries' own.
//   out^T = V^T p^T: the scores leave the first product with a lane holding tokens 4g..4g+3 of its query row, which is
//     what operand B of the second wants if V's lanes take the same tokens: the weights never change lanes, and the
//     pages keep values in fours of tokens so that a lane's share is one load.
// K is exact in bfloat16 and float16 alike, V in float16 (the exponents are clamped for that).  Queries go in as they are
// (float32 as three bfloat16 pieces that add up to it).  The weights are rounded to float16, 2^-11 relative, and are held
// times 2^8 so that weights down to 2^-22 of the row's reference keep that (smaller ones are off by 2^-33 of it): an eighth
// of a bfloat16 result's own rounding, but as much as a float16 one's.  So float16 results take a second piece of the
// weights, and so do float32 results, held times 2^15.  Sums, maxima and accumulators are float32.
// Measured: one token over 2K-32K tokens of 32 requests (8 KV heads of 128 dimensions, 617 MB of pages) 134 us a call, 4.6
// TB/s against a copy's 5.1: the memory bounds it.  2,048 query tokens of 24 heads over 16K tokens (387 GFLOP) 414 us a call
// with its join, 0.93 PFLOP/s; a large library product makes 1.17.  There the issue of vector instructions bounds it
// (conversions, exponentials and the matrix instructions' own slots: 63 % of the SIMDs' cycles, the matrix cores 41 %), at
// two waves a SIMD.
#include <math.h>

#include "dkv_device.h"
#include "dkv_fp4.h"
#include "dkv_host.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

constexpr int kMaxSplits = 256, kFewSplits = 4;

struct AttendArgs {
  dkv_fp4_cache_t c;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* cu;
  const void* query;
  void* out;
  float* part;      // [rows * q_heads][splits][D] sums when the tokens are split over workgroups
  float2* part_ml;  // [rows * q_heads][splits] maximum and sum
  uint32_t* arrivals;  // [requests][blocks][kv_heads] when the launch joins its splits itself
  int64_t query_token, query_head;
  int requests, width, shift, rows, groups, window, splits, share, fill;
  float scale;  // |scaling| * log2 e
  int negate;   // scaling < 0: the queries change sign
};

DKV_DEVICE void set_result(float& y, float x) { y = x; }
DKV_DEVICE void set_result(half_t& y, float x) { y = (half_t)x; }
DKV_DEVICE void set_result(dkv_bf16& y, float x) { y.bits = float_to_bf16_bits(x); }

template <typename T>
struct Operand;  // what a query type's products are made of
template <>
struct Operand<half_t> {
  typedef half8 frag;
  static constexpr int kPieces = 1;
  static DKV_DEVICE half2_t pair(uint32_t word, float scale, int sel) {
    switch (sel) {
      case 0: return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 0);
      case 1: return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 1);
      case 2: return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 2);
      default: return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 3);
    }
  }
  static DKV_DEVICE floatx4 mfma(frag a, frag b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Operand<dkv_bf16> {
  typedef bf16x8 frag;
  static constexpr int kPieces = 1;
  static DKV_DEVICE bf16x2 pair(uint32_t word, float scale, int sel) {
    switch (sel) {
      case 0: return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0);
      case 1: return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1);
      case 2: return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2);
      default: return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3);
    }
  }
  static DKV_DEVICE floatx4 mfma(frag a, frag b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Operand<float> : Operand<dkv_bf16> {
  static constexpr int kPieces = 3;
};

// A row with an infinite query value has no finite score (that value's products are infinite, or NaN with a key of 0), so no
// finite result where it sees a token.  Infinities become NaN, and the row's scores with them: those of -infinity alone
// would pass for tokens that the row does not see.
DKV_DEVICE void quiet(half8 (&q)[1]) { q[0] = __builtin_elementwise_fma(q[0], (half8)(half_t)0.0f, q[0]); }  // x + 0 * x
DKV_DEVICE void quiet(bf16x8 (&q)[1]) {  // the bit below an exponent of all ones set
  uint32_t w[4];
  __builtin_memcpy(w, &q[0], 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] |= (((w[i] & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 9;
  __builtin_memcpy(&q[0], w, 16);
}
DKV_DEVICE void quiet(bf16x8 (&)[3]) {}  // (where they are cut into pieces)

// 8 query values into kPieces operands.
DKV_DEVICE uint4 signed_words(const void* p, uint32_t sign) {
  const uint4 w = *(const uint4*)p;
  return make_uint4(w.x ^ sign, w.y ^ sign, w.z ^ sign, w.w ^ sign);
}
DKV_DEVICE void query_pieces(const half_t* p, bool negate, half8 (&out)[1]) {
  const uint4 w = signed_words(p, negate ? 0x80008000u : 0u);
  __builtin_memcpy(&out[0], &w, 16);
}
DKV_DEVICE void query_pieces(const dkv_bf16* p, bool negate, bf16x8 (&out)[1]) {
  const uint4 w = signed_words(p, negate ? 0x80008000u : 0u);
  __builtin_memcpy(&out[0], &w, 16);
}
DKV_DEVICE void query_pieces(const float* p, bool negate, bf16x8 (&out)[3]) {
  const uint32_t sign = negate ? 0x80000000u : 0u;
  const uint4 first = signed_words(p, sign), second = signed_words(p + 4, sign);
  const uint32_t value[8] = {first.x, first.y, first.z, first.w, second.x, second.y, second.z, second.w};
  // upper halves of the value, of what they leave, and the rest: 8 bits each of the 24
  uint32_t words[3][4] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = __uint_as_float(value[i]);
    const uint32_t a = __float_as_uint(x) & 0xffff0000u;
    const float left = x - __uint_as_float(a);
    const uint32_t b = __float_as_uint(left) & 0xffff0000u;
    const uint32_t c = __float_as_uint(left - __uint_as_float(b));
    const bool finite = (a & 0x7f800000u) != 0x7f800000u;  // an infinity or NaN is one piece, a NaN
    words[0][i >> 1] |= (a >> 16 | (finite ? 0u : 0x40u)) << (16 * (i & 1));
    words[1][i >> 1] |= (finite ? b >> 16 : 0u) << (16 * (i & 1));
    words[2][i >> 1] |= (finite ? c >> 16 : 0u) << (16 * (i & 1));
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) __builtin_memcpy(&out[k], words[k], 16);
}

// The larger of two floats (a NaN loses), without the quieting that the compiler puts before fmaxf.
DKV_DEVICE float larger(float a, float b) {
  float c;
  asm("v_max_f32 %0, %1, %2" : "=v"(c) : "v"(a), "v"(b));
  return c;
}

DKV_DEVICE float larger(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}

DKV_DEVICE float exponent(uint32_t byte) { return __uint_as_float(byte << 23); }

// The tables are read through the scalar cache: an index the same in every lane costs no vector load, and no wait for the
// page loads on their way.
typedef const __attribute__((address_space(4))) int32_t* scalar_ints;
DKV_DEVICE scalar_ints as_scalar(const int32_t* p) { return (scalar_ints)(uintptr_t)p; }

// One chunk in this lane, CH tiles of 16 tokens: codes and exponents, and which tiles hold something (the same in every
// lane).
template <int D, int CH>
struct Codes {
  uint32_t words[CH][D / 32], scales[CH];
};
template <int CH>
struct Tiles {
  uint64_t first[CH];  // token of the arrays where the tile begins
  bool valid[CH];
  bool whole;
};

// Loads through a buffer descriptor: a base in scalar registers and the lane's offset, and nothing read past `bytes`.
typedef __amdgpu_buffer_rsrc_t buffer;
DKV_DEVICE buffer buffer_of(const uint8_t* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, 0x00020000);
}
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
template <int N>
DKV_DEVICE void load_words(buffer from, uint32_t at, uint32_t (&w)[N]) {
  if constexpr (N == 2) {
    const uint2_t x = __builtin_amdgcn_raw_buffer_load_b64(from, at, 0, 0);
    w[0] = x[0]; w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4_t x = __builtin_amdgcn_raw_buffer_load_b128(from, at + i * 4, 0, 0);
      w[i] = x[0]; w[i + 1] = x[1]; w[i + 2] = x[2]; w[i + 3] = x[3];
    }
  }
}

// A lane's bytes inside a tile, behind the tile's first byte of codes (16 tokens of D / 2) and of exponents.
template <int D>
struct LaneOffsets {
  uint32_t key, key_scale, value, value_scale;
  DKV_DEVICE LaneOffsets() {
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    key = i * (D / 2) + g * (D / 8);
    key_scale = i * (D / 32) + (D == 64 ? g >> 1 : D == 128 ? g : 2 * g);
    value = g * (2 * D) + i * (D / 8);
    value_scale = g * (D / 8) + (i * (D / 16) / 32) * 4;
  }
};

// The table entries of a chunk's tiles, one a lane (lane t, and every 16th from it, tile t).  They are loaded a chunk
// ahead of the pages, so that no page load waits for its address.
template <int CH>
DKV_DEVICE int load_entries(const AttendArgs& a, const int32_t* row, int len, int chunk) {
  const uint32_t token = (uint32_t)(chunk * CH + (int)(threadIdx.x & 15) % CH) * 16;
  return row[token < (uint32_t)len ? token >> a.shift : 0];  // (checked where it is used, so that nothing waits for it here)
}

template <int CH>
DKV_DEVICE void find_tiles(const AttendArgs& a, int entries, int len, int h, int chunk, Tiles<CH>& tiles) {
  const uint32_t page = a.c.page;
  tiles.whole = true;
#pragma unroll
  for (int t = 0; t < CH; ++t) {
    const uint32_t id = (uint32_t)__builtin_amdgcn_readlane(entries, t), token = (uint32_t)(chunk * CH + t) * 16;
    tiles.valid[t] = token < (uint32_t)len && id < (uint32_t)a.c.pages;
    tiles.whole = tiles.whole && tiles.valid[t];
    tiles.first[t] = tiles.valid[t] ? ((uint64_t)id * a.c.kv_heads + h) * page + (token & (page - 1)) : 0;
  }
}

// Loads are made for every tile, so that the ones on their way are the same count on every path; of a tile that holds
// nothing (behind the request, or an entry that is no page) no byte is read, and its codes and exponents are 0.
template <int D, int CH>
DKV_DEVICE void load_keys(const AttendArgs& a, const Tiles<CH>& tiles, const LaneOffsets<D>& at, Codes<D, CH>& c) {
#pragma unroll
  for (int t = 0; t < CH; ++t) {
    load_words(buffer_of(a.c.key_codes + tiles.first[t] * (D / 2), tiles.valid[t] ? 8 * D : 0), at.key, c.words[t]);
    const buffer scales = buffer_of(a.c.key_scales + tiles.first[t] * (D / 32), tiles.valid[t] ? D / 2 : 0);
    if constexpr (D == 256) c.scales[t] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(scales, at.key_scale, 0, 0);
    else c.scales[t] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(scales, at.key_scale, 0, 0);
  }
}
template <int D, int CH>
DKV_DEVICE void load_values(const AttendArgs& a, const Tiles<CH>& tiles, const LaneOffsets<D>& at, Codes<D, CH>& c) {
#pragma unroll
  for (int t = 0; t < CH; ++t) {
    load_words(buffer_of(a.c.value_codes + tiles.first[t] * (D / 2), tiles.valid[t] ? 8 * D : 0), at.value, c.words[t]);
    c.scales[t] = __builtin_amdgcn_raw_buffer_load_b32(
        buffer_of(a.c.value_scales + tiles.first[t] * (D / 32), tiles.valid[t] ? D / 2 : 0), at.value_scale, 0, 0);
  }
}

template <int D, typename T, int NT, int CH, int kWaves>
__global__ __launch_bounds__(kWaves * 64, NT == 2 && D > 64 ? 1 : 2) void fp4_attend_kernel(AttendArgs a) {
  using Op = Operand<T>;
  using frag = typename Op::frag;
  constexpr int kRows = 16 * NT, kSteps = D / 32, kLane = D / 16, kPieces = Op::kPieces;
  // float16 pieces of a weight: a second one for float32 and float16 results.  One piece for float16 costs 464 us instead
  // of 615 at 2,048 query tokens of 24 heads over 16K tokens of 128 dimensions, and rounds as much as the result does.
  constexpr int kWeights = kPieces > 1 || __is_same(T, half_t) ? 2 : 1;
  // Weights are held times 2^kShift, against a reference that scores may pass by kSlack: 2^15 at the most, below the
  // largest float16.
  constexpr float kSlack = kPieces == 1 ? 7.0f : 0.0f, kShift = 15.0f - kSlack;
  constexpr int kStride = D + 4;                  // a row of sums in LDS
  constexpr bool kJoins = NT <= 2 && kWaves == 4;  // may join its splits itself (sums hold 6 floats a thread)
  // With 64 rows the accumulators leave no registers for the queries and a second chunk, and two waves a SIMD matter more
  // (one fills the other's waits): queries lie in LDS, and a chunk's loads follow the last use of the one before.
  constexpr bool kLean = NT == 4;
  __shared__ frag held[kLean ? NT * kSteps * 64 : 1];
  __shared__ float sums[4 * 16 * kStride];
  __shared__ float stat[2][kWaves][kRows];

  const int h = blockIdx.x, b = blockIdx.z, split = blockIdx.y % a.splits, blocks = gridDim.y / a.splits;
  __shared__ int last;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
  const int q_heads = a.c.kv_heads * a.groups;
  const scalar_ints cu = as_scalar(a.cu) + b;
  const int32_t* table = a.table + (long)b * a.width;
  const int q0 = min(max(cu[0], 0), a.rows), q1 = min(max(cu[1], q0), a.rows);
  const int n_rows = (q1 - q0) * a.groups;
  const int len = min(max(as_scalar(a.lengths)[b], 0), a.width << a.shift);
  const LaneOffsets<D> at;
  const int first_position = len - (q1 - q0);  // of the request's first query token; below 0 it sees nothing

  if (a.fill && b == 0 && blockIdx.y == 0) {  // rows behind the last request
    T* out = (T*)a.out;
    const int end = min(max(a.cu[a.requests], 0), a.rows);
    const long n = (long)(a.rows - end) * a.groups * D;
    for (long x = threadIdx.x; x < n; x += kWaves * 64)
      __builtin_memset(out + ((end + x / (a.groups * D)) * q_heads + h * a.groups) * D + x % (a.groups * D), 0, sizeof(T));
  }

  // (the last rows first: they see the most tokens, and the card is left with short work at the end)
  const long row_blocks = ((long)n_rows + kRows - 1) / kRows;
  // (more rows than the launch was shaped for: a workgroup takes several row blocks, and splits could not tell whose
  // arrivals they count; one of them then takes all tokens)
  const bool alone = a.arrivals && row_blocks > blocks;
  if (alone && split) return;
  const int splits = alone ? 1 : a.splits;
  for (long turn = blockIdx.y / a.splits; turn < row_blocks; turn += blocks) {
    const int block = (int)(row_blocks - 1 - turn);
    const int row0 = block * kRows, row1 = min(row0 + kRows, n_rows);
    // queries: operand B, lane i a row, 8 dimensions of g * D/4 + 8 * step
    frag q[kLean ? 1 : NT][kSteps][kPieces];
    // the last token a row sees, and the one before the first (made where a chunk has a mask, and not held)
    auto last_seen = [&](int nt) { return first_position + min(row0 + nt * 16 + i, n_rows - 1) / a.groups; };
    auto before_first = [&](int last) { return (int)max((long)last - a.window, -1L); };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = min(row0 + nt * 16 + i, n_rows - 1);  // (rows past the last one repeat it, and go nowhere)
      const int token = r / a.groups;
      const T* p = (const T*)a.query + (q0 + token) * a.query_token + (h * a.groups + r - token * a.groups) * a.query_head;
      if constexpr (kLean) {
        if (nt == wave) {
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            query_pieces(p + g * (D / 4) + s * 8, a.negate, q[0][0]);
            quiet(q[0][0]);
            held[(nt * kSteps + s) * 64 + lane] = q[0][0][0];
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) query_pieces(p + g * (D / 4) + s * 8, a.negate, q[nt][s]);
      }
    }
    if constexpr (kLean) __syncthreads();
    const int low_position = first_position + row0 / a.groups, high_position = first_position + (row1 - 1) / a.groups;
    const int begin = (int)max((long)low_position - a.window + 1, 0L), end = high_position + 1;  // tokens some row sees
    const int all_from = (int)max((long)high_position - a.window + 1, 0L);                       // and all rows, from here
    const int chunk_begin = begin / (16 * CH), chunk_end = max((end + 16 * CH - 1) / (16 * CH), chunk_begin);
    const long chunks = end > begin ? chunk_end - chunk_begin : 0;
    // as many chunks a split as the plan gives (so that a short request takes few), or what covers them all
    const long share = max((long)a.share / CH, (chunks + splits - 1) / splits);
    const int c0 = chunk_begin + (int)min(split * share, chunks), c1 = chunk_begin + (int)min((split + 1) * share, chunks);

    floatx4 o[NT][kLane];
    float m[NT], l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt] = -INFINITY;
      l[nt] = 0.0f;
#pragma unroll
      for (int j = 0; j < kLane; ++j) o[nt][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    Codes<D, CH> keys, values, next_keys, next_values;
    Tiles<CH> tiles, next_tiles;
    int chunk = __builtin_amdgcn_readfirstlane(c0 + wave);
    int entries = load_entries<CH>(a, table, chunk < c1 ? len : 0, chunk);
    find_tiles<CH>(a, entries, chunk < c1 ? len : 0, h, chunk, tiles);
    load_keys<D, CH>(a, tiles, at, keys);
    load_values<D, CH>(a, tiles, at, values);
    entries = load_entries<CH>(a, table, chunk + kWaves < c1 ? len : 0, chunk + kWaves);
    if constexpr (!kLean) {  // (here, so that the first chunk's loads do not wait for the queries')
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) quiet(q[nt][s]);
    }
    for (; chunk < c1; chunk += kWaves) {
      const int later = load_entries<CH>(a, table, chunk + 2 * kWaves < c1 ? len : 0, chunk + 2 * kWaves);
      find_tiles<CH>(a, entries, chunk + kWaves < c1 ? len : 0, h, chunk + kWaves, next_tiles);
      entries = later;
      if constexpr (!kLean) {
        load_keys<D, CH>(a, next_tiles, at, next_keys);
        load_values<D, CH>(a, next_tiles, at, next_values);
      }

      // scores^T: lane i a row, tokens 4g..4g+3 of each tile
      floatx4 s[NT][CH];
#pragma unroll
      for (int t = 0; t < CH; ++t)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
      frag key[CH];
      auto convert_keys = [&](int st, frag (&out)[CH]) {
#pragma unroll
        for (int t = 0; t < CH; ++t) {
          const float e = exponent(D == 256 ? (st < 4 ? keys.scales[t] & 255 : keys.scales[t] >> 8) : keys.scales[t]);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const auto two = Op::pair(keys.words[t][st], e, x);
            out[t][2 * x] = two[0];
            out[t][2 * x + 1] = two[1];
          }
        }
      };
      frag lean[2][kLean ? NT : 1];
      if constexpr (kLean)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) lean[0][nt] = held[(nt * kSteps) * 64 + lane];
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        if constexpr (kLean) __builtin_amdgcn_sched_barrier(0);
        convert_keys(st, key);
        if (st + 1 < kSteps) {  // (an LDS read takes as long as a step's products)
          if constexpr (kLean)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) lean[(st + 1) & 1][nt] = held[(nt * kSteps + st + 1) * 64 + lane];
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int p = kPieces - 1; p >= 0; --p)
#pragma unroll
            for (int t = 0; t < CH; ++t)
              s[nt][t] = Op::mfma(key[t], kLean ? lean[st & 1][kLean ? nt : 0] : q[kLean ? 0 : nt][kLean ? 0 : st][p], s[nt][t]);
      }
      if constexpr (kLean) {
        load_keys<D, CH>(a, next_tiles, at, keys);
        __builtin_amdgcn_sched_barrier(0);
      }

      const int base = chunk * CH * 16;
      const bool masked = !tiles.whole || base + CH * 16 > low_position + 1 || base < all_from;
      if (masked) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int last = last_seen(nt), before = before_first(last);
#pragma unroll
          for (int t = 0; t < CH; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int token = base + t * 16 + g * 4 + r;
              if (!tiles.valid[t] || token > last || token <= before) s[nt][t][r] = -INFINITY;
            }
        }
        // what lies behind the request is stale: its values become zeros
#pragma unroll
        for (int t = 0; t < CH; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!tiles.valid[t] || base + t * 16 + g * 4 + r >= len) values.scales[t] &= ~(255u << (8 * r));
      }

      half8 w[NT][CH / 2][kWeights];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // The reference m of a row follows its maximum only when a score passes it by kSlack: most chunks then need no
        // exchange between the four lanes of a row, and no rescaling.
        float top = s[nt][0][0];
#pragma unroll
        for (int t = 0; t < CH; ++t) top = larger(larger(top, s[nt][t][0], s[nt][t][1]), s[nt][t][2], s[nt][t][3]);
        if (__any(top * a.scale > m[nt] + kSlack)) {
          const float higher = larger(m[nt], max_xor32(max_xor16(top)) * a.scale);
          const float factor = __builtin_amdgcn_exp2f(m[nt] - (higher == -INFINITY ? 0.0f : higher));
          l[nt] *= factor;
#pragma unroll
          for (int j = 0; j < kLane; ++j) o[nt][j] *= factor;
          m[nt] = higher;
        }
        const float shift = kShift - (m[nt] == -INFINITY ? 0.0f : m[nt]);
#pragma unroll
        for (int t = 0; t < CH; ++t) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[nt][t][r], a.scale, shift));
            l[nt] += p;
            w[nt][t / 2][0][(t & 1) * 4 + r] = (half_t)p;
            if constexpr (kWeights == 2) w[nt][t / 2][1][(t & 1) * 4 + r] = (half_t)(p - (float)(half_t)p);
          }
        }
      }

      if (masked) {
        // A block of NaN belongs to the rows that see its token, and a product would give it (0 * NaN) to all: where a
        // chunk has rows that do not see all of it, such blocks become zeros and the rows that see them NaN by hand.
#pragma unroll
        for (int u = 0; u < CH / 2; ++u) {
          uint32_t bad[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t& vs = values.scales[2 * u + x];
            bad[x] = ((vs & 0x7f7f7f7fu) + 0x01010101u) & vs & 0x80808080u;  // the bytes that are 255
            vs &= ~((bad[x] >> 7) * 255u);
          }
          if (__any((bad[0] | bad[1]) != 0)) {
            half8 is_bad;
#pragma unroll
            for (int x = 0; x < 8; ++x) is_bad[x] = (bad[x >> 2] >> (8 * (x & 3) + 7)) & 1 ? (half_t)1.0f : (half_t)0.0f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const int last = last_seen(nt), before = before_first(last);
              half8 sees;
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const int token = base + (2 * u + (x >> 2)) * 16 + g * 4 + (x & 3);
                sees[x] = token <= last && token > before ? (half_t)1.0f : (half_t)0.0f;
              }
              const floatx4 hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(is_bad, sees, floatx4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
              for (int j = 0; j < kLane; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (hit[r] > 0.0f) o[nt][j][r] = __builtin_nanf("");
            }
          }
        }
      }

      // out^T: operand A is 16 lanes' dimensions i * kLane + j over the 32 tokens of two tiles
      constexpr int kPairs = kLane / 2, kTurns = CH / 2 * kPairs;
      auto convert_values = [&](int turn, half8& even, half8& odd) {
        const int u = turn / kPairs, pair = turn % kPairs;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float e = exponent((values.scales[2 * u + (x >> 2)] >> (8 * (x & 3))) & 255);
          const int byte = (x & 3) * (D / 32) + pair;
          const half2_t two = Operand<half_t>::pair(values.words[2 * u + (x >> 2)][byte / 4], e, byte % 4);
          even[x] = two[0];
          odd[x] = two[1];
        }
      };
#pragma unroll
      for (int turn = 0; turn < kTurns; ++turn) {
        if constexpr (kLean) __builtin_amdgcn_sched_barrier(0);
        const int u = turn / kPairs, j = turn % kPairs * 2;
        half8 even, odd;
        convert_values(turn, even, odd);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int p = kWeights - 1; p >= 0; --p) {
            o[nt][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, w[nt][u][p], o[nt][j], 0, 0, 0);
            o[nt][j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, w[nt][u][p], o[nt][j + 1], 0, 0, 0);
          }
      }
      tiles = next_tiles;
      if constexpr (kLean) {
        load_values<D, CH>(a, tiles, at, values);
      } else {
        keys = next_keys;
        values = next_values;
      }
    }

    // the waves' sums, 16 rows at a time and four waves at a time
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float total = sum_xor32(sum_xor16(l[nt]));
      // a row whose scores are all NaN has no maximum, but is not one that sees nothing
      if (m[nt] == -INFINITY && total != 0.0f) m[nt] = 0.0f;
      if (g == 0) {
        stat[0][wave][nt * 16 + i] = m[nt];
        stat[1][wave][nt * 16 + i] = total;
      }
    }
    __syncthreads();
    constexpr int kParts = kWaves * 4, kPart = D / kParts;
    const int row = threadIdx.x / kParts, part = threadIdx.x % kParts;  // in the join: a row, and kPart of its dimensions
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top = -INFINITY;
#pragma unroll
      for (int x = 0; x < kWaves; ++x) top = fmaxf(top, stat[0][x][nt * 16 + i]);
      const float factor = m[nt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[nt] - top);
      float* mine = sums + ((wave & 3) * 16 + i) * kStride + g * (D / 4);
#pragma unroll
      for (int j = 0; j < kLane; ++j) o[nt][j] *= factor;
      if constexpr (kWaves == 8) {
        if (wave >= 4) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < kLane; ++j) mine[r * kLane + j] = o[nt][j][r];
        }
        __syncthreads();
        if (wave < 4) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < kLane; ++j) mine[r * kLane + j] += o[nt][j][r];
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < kLane; ++j) mine[r * kLane + j] = o[nt][j][r];
      }
      __syncthreads();
      const int r = row0 + nt * 16 + row;
      if (r < n_rows) {
        float highest = -INFINITY, total = 0.0f, acc[kPart] = {};
#pragma unroll
        for (int x = 0; x < kWaves; ++x) highest = fmaxf(highest, stat[0][x][nt * 16 + row]);
#pragma unroll
        for (int x = 0; x < kWaves; ++x) {
          const float mx = stat[0][x][nt * 16 + row];
          total += mx == -INFINITY ? 0.0f : stat[1][x][nt * 16 + row] * __builtin_amdgcn_exp2f(mx - highest);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int j = 0; j < kPart; ++j) acc[j] += sums[(x * 16 + row) * kStride + part * kPart + j];
        const int token = r / a.groups;
        const long out_row = (long)(q0 + token) * q_heads + h * a.groups + (r - token * a.groups);
        if (splits == 1) {
          T* out = (T*)a.out + out_row * D + part * kPart;
          const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
          for (int j = 0; j < kPart; ++j) set_result(out[j], total == 0.0f ? 0.0f : acc[j] * inverse);
        } else {
          const long at = out_row * splits + split;
          float* out = a.part + at * D + part * kPart;
          if (a.arrivals) {
            if (highest != -INFINITY)
#pragma unroll
              for (int j = 0; j < kPart; j += 2) leave2(out + j, acc[j], acc[j + 1]);
            if (part == 0) leave2((float*)(a.part_ml + at), highest, total);
          } else {
            if (highest != -INFINITY)
#pragma unroll
              for (int j = 0; j < kPart; ++j) out[j] = acc[j];
            if (part == 0) a.part_ml[at] = make_float2(highest, total);
          }
        }
      }
      __syncthreads();
    }
    if constexpr (kJoins) {
      if (splits > 1 && a.arrivals) {
        left_behind();
        __syncthreads();
        if (threadIdx.x == 0) last = last_of(a.arrivals + ((long)b * blocks + turn) * a.c.kv_heads + h, splits);
        __syncthreads();
        // the last workgroup of the row block joins its splits: D / 4 threads for a row's dimensions in fours, the sets of
        // them dealt out to the rows and their splits
        constexpr int kSet = D / 4, kSets = kWaves * 64 / kSet;
        const int rows = row1 - row0;
        int per_row = kSets;
        while (per_row > 1 && per_row * rows > kSets) per_row >>= 1;
        const int set = threadIdx.x / kSet, dim = threadIdx.x % kSet * 4, share = set % per_row;
        for (int first = 0; last && first < rows; first += kSets / per_row) {
          const int r = row0 + first + set / per_row;
          const bool mine = first + set / per_row < rows;
          const int token = r / a.groups;
          const long out_row = (long)(q0 + token) * q_heads + h * a.groups + (r - token * a.groups);
          float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          float top = -INFINITY, total = 0.0f;
          if (mine) {
            const float* ml = (const float*)(a.part_ml + out_row * splits);
            const float* part_of = a.part + out_row * splits * D + dim;
            constexpr int kBatch = 8;
            for (int s0 = share; s0 < splits; s0 += kBatch * per_row) {
              float2 x[kBatch], v[kBatch][2];
#pragma unroll
              for (int k = 0; k < kBatch; ++k) {
                const int s = min(s0 + k * per_row, splits - 1);
                x[k] = pick_up2(ml + 2 * s);
                v[k][0] = pick_up2(part_of + (long)s * D);
                v[k][1] = pick_up2(part_of + (long)s * D + 2);
                if (s0 + k * per_row >= splits) x[k].x = -INFINITY;
              }
              float higher = top;
#pragma unroll
              for (int k = 0; k < kBatch; ++k) higher = fmaxf(higher, x[k].x);
              const float before = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - higher);
              acc.x *= before; acc.y *= before; acc.z *= before; acc.w *= before;
              total *= before;
              top = higher;
#pragma unroll
              for (int k = 0; k < kBatch; ++k) {
                if (x[k].x == -INFINITY) continue;  // nothing seen there, and nothing left
                const float f = __builtin_amdgcn_exp2f(x[k].x - top);
                total += x[k].y * f;
                acc.x = fmaf(v[k][0].x, f, acc.x); acc.y = fmaf(v[k][0].y, f, acc.y);
                acc.z = fmaf(v[k][1].x, f, acc.z); acc.w = fmaf(v[k][1].y, f, acc.w);
              }
            }
          }
          float* slot = sums + threadIdx.x * 6;
          slot[0] = acc.x; slot[1] = acc.y; slot[2] = acc.z; slot[3] = acc.w; slot[4] = top; slot[5] = total;
          __syncthreads();
          if (mine && share == 0) {
            float highest = -INFINITY;
            for (int k = 0; k < per_row; ++k) highest = fmaxf(highest, slot[k * kSet * 6 + 4]);
            float v[4] = {}, whole = 0.0f;
            for (int k = 0; k < per_row; ++k) {
              const float* other = slot + k * kSet * 6;
              const float f = other[4] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(other[4] - highest);
              whole += other[5] * f;
#pragma unroll
              for (int j = 0; j < 4; ++j) v[j] = fmaf(other[j], f, v[j]);
            }
            T* out = (T*)a.out + out_row * D + dim;
#pragma unroll
            for (int j = 0; j < 4; ++j) set_result(out[j], whole == 0.0f ? 0.0f : v[j] / whole);
          }
          __syncthreads();
        }
      }
    }
  }
}

// The splits of a row joined: a workgroup per row, D / 4 threads for its dimensions in fours, the splits dealt out to the
// 256 / (D / 4) sets of them and their sums added in LDS.
template <int D, typename T>
__global__ __launch_bounds__(256) void fp4_join_kernel(AttendArgs a, int q_heads) {
  constexpr int kSet = D / 4, kSets = 256 / kSet;
  __shared__ float weight[kMaxSplits];
  __shared__ float4 sums[kSets][kSet];
  __shared__ float whole;
  const long row = blockIdx.x;
  if (row >= (long)min(max(a.cu[a.requests], 0), a.rows) * q_heads) return;
  const float2* ml = a.part_ml + row * a.splits;
  if (threadIdx.x < 64) {
    float top = -INFINITY, total = 0.0f;
    float2 x[kMaxSplits / 64];
#pragma unroll
    for (int k = 0; k < kMaxSplits / 64; ++k) {
      const int s = k * 64 + (int)threadIdx.x;
      x[k] = s < a.splits ? ml[s] : make_float2(-INFINITY, 0.0f);
      top = fmaxf(top, x[k].x);
    }
    top = wave_max(top);
#pragma unroll
    for (int k = 0; k < kMaxSplits / 64; ++k) {
      // (a split that saw nothing wrote nothing; one whose weight is 0 did, and may hold a NaN)
      const float factor = x[k].x == -INFINITY ? -1.0f : __builtin_amdgcn_exp2f(x[k].x - top);
      weight[k * 64 + threadIdx.x] = factor;
      total += factor < 0.0f ? 0.0f : x[k].y * factor;
    }
    total = wave_sum(total);
    if (threadIdx.x == 0) whole = total;
  }
  __syncthreads();
  const int at = threadIdx.x % kSet, set = threadIdx.x / kSet;
  const float4* part = (const float4*)(a.part + row * a.splits * D) + at;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int s = set; s < a.splits; s += kSets) {
    const float w = weight[s];
    if (w < 0.0f) continue;
    const float4 v = part[s * kSet];
    acc.x = fmaf(v.x, w, acc.x); acc.y = fmaf(v.y, w, acc.y); acc.z = fmaf(v.z, w, acc.z); acc.w = fmaf(v.w, w, acc.w);
  }
  sums[set][at] = acc;
  __syncthreads();
  if (set) return;
#pragma unroll
  for (int x = 1; x < kSets; ++x) {
    const float4 v = sums[x][at];
    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
  }
  T* out = (T*)a.out + row * D + at * 4;
  const float v[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) set_result(out[j], whole == 0.0f ? 0.0f : v[j] / whole);
}

// The same for few splits: a set of D / 4 threads per row.  49,152 rows of two splits: 13 us, 40 with a workgroup for
// each row.
template <int D, typename T>
__global__ __launch_bounds__(256) void fp4_join_few_kernel(AttendArgs a, int q_heads) {
  constexpr int kSet = D / 4, kSets = 256 / kSet;
  const int at = threadIdx.x % kSet;
  const long row = (long)blockIdx.x * kSets + threadIdx.x / kSet;
  if (row >= (long)min(max(a.cu[a.requests], 0), a.rows) * q_heads) return;
  const float2* ml = a.part_ml + row * a.splits;
  const float4* part = (const float4*)(a.part + row * a.splits * D) + at;
  float top = -INFINITY, whole = 0.0f;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[s].x);
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s = 0; s < a.splits; ++s) {
    const float2 x = ml[s];
    if (x.x == -INFINITY) continue;  // nothing seen there, and nothing written
    const float w = __builtin_amdgcn_exp2f(x.x - top);
    const float4 v = part[s * kSet];
    whole += x.y * w;
    acc.x = fmaf(v.x, w, acc.x); acc.y = fmaf(v.y, w, acc.y); acc.z = fmaf(v.z, w, acc.z); acc.w = fmaf(v.w, w, acc.w);
  }
  T* out = (T*)a.out + row * D + at * 4;
  const float v[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) set_result(out[j], whole == 0.0f ? 0.0f : v[j] / whole);
}

struct Plan {
  int tiles;   // 16-row tiles a workgroup takes
  int waves;   // of a workgroup
  int blocks;  // row blocks a request is given
  int splits;
  int share;   // 16-token tiles a split takes at the least
  bool joins;  // the launch joins its splits itself
};

constexpr long kWorkgroups = 512;  // of four waves: what the card holds at two waves a SIMD

Plan plan_of(const dkv_fp4_attend_args_t& p) {
  Plan plan;
  const long groups = p.q_heads / p.cache.kv_heads, rows = (long)(p.most < 1 ? 1 : p.most) * groups;
  const bool narrow = p.query_dtype == DKV_F32 || p.cache.head_dim == 256;
  plan.tiles = rows <= 16 || (p.query_dtype == DKV_F32 && p.cache.head_dim == 256) ? 1 : rows <= 32 || narrow ? 2 : 4;
  const long blocks = (rows + plan.tiles * 16 - 1) / (plan.tiles * 16);
  plan.blocks = (int)(blocks < 4096 ? blocks : 4096);
  const long each = (long)p.requests * p.cache.kv_heads * plan.blocks;
  long longest = p.longest < 1 ? 1 : p.longest;  // the tokens a row block may see
  if (p.window) longest = min(longest, (long)p.window + plan.tiles * 16 / groups + 16);
  // Workgroups enough for the card, of 256 tokens at the least; of 1,024 where that makes more than the card holds at
  // once, so that requests of different lengths even out.
  const long fill = (kWorkgroups + each - 1) / each, even = p.requests > 1 ? (8 * kWorkgroups + each - 1) / each : 1;
  const long wanted = max(min(fill, (longest + 255) / 256), min(even, (longest + 1023) / 1024));
  // Short requests of few rows are not split: eight waves take them in two turns, four where requests alone fill the card.
  // In a captured graph, 8 KV heads of 128 bfloat16 dimensions: 700 tokens of 32 requests 9.1 us against 13.5 split and
  // joined, 2,000 of them 16.5 against 18.8; one request of 500 tokens 8.2 against 9.0, of 1,000 10.3 against 9.7, of 2,000
  // 14.1 against 9.0.  Called from Python the second launch costs 3 us more.
  const long brief = p.cache.head_dim < 256 ? 1024 : p.query_dtype == DKV_F32 ? 256 : 512;
  plan.waves = plan.tiles == 1 && longest <= (each >= 256 ? 2 * brief : brief) ? 8 : 4;
  plan.splits = plan.waves == 8 ? 1 : (int)min(max(wanted, 1L), (long)kMaxSplits);
  // Blocks of 64 rows that fill the card once and a half leave half of it idle at the end: two or three splits where that
  // makes fuller rounds, by more than the join costs.
  if (plan.splits == 1 && plan.tiles == 4 && longest >= 4096) {
    const auto rounds = [&](long x) { return (double)((each * x + kWorkgroups - 1) / kWorkgroups) / x; };
    for (int x = 2; x <= 3; ++x)
      if (rounds(x) < 0.85 * rounds(plan.splits)) plan.splits = x;
  }
  // A row block whose rows times splits are few is joined by the last of its workgroups to arrive, others by a launch of
  // their own, which costs the caller 3 us.  Fewer splits are made for that where a wave then takes one more chunk at most.
  // 8 KV heads of 128 bfloat16 dimensions, 3 query heads each: 3,000 tokens 9.3 us in a graph and 11.2 a call against 9.5
  // and 13.8 by two launches, 6,000 tokens 11.5 and 11.3 against 9.8 and 13.9; 16K tokens stay with 64 splits (13.0 and
  // 13.9; 14.5 and 14.4 with the 21 that one workgroup would join).  A launch that fills the card is not joined in itself
  // (4 requests of 12,000 tokens, 64 dimensions, 16 splits: 13.5 and 14.0 against 14.6 and 14.4), and at 256 dimensions
  // fewer rows are (8 rows, 12 splits of 3,000 tokens, 2 KV heads: 10.7 and 13.8 against 14.7 and 14.7).
  const long row_block = min(rows, plan.tiles * 16L), joined = p.cache.head_dim < 256 ? 64 : 32;
  plan.joins = false;
  if (p.arrivals && plan.tiles <= 2 && plan.splits > 1 && each <= p.arrivals_count && row_block <= joined / 2) {
    const long fewer = min((long)plan.splits, joined / row_block), chunk = plan.tiles == 1 && p.cache.head_dim < 256 ? 256 : 128;
    const auto turns = [&](long splits) { return (longest + chunk * splits - 1) / (chunk * splits); };
    plan.joins = each * fewer < kWorkgroups && turns(fewer) - turns(plan.splits) <= (p.cache.head_dim < 256 ? 1 : 0);
    if (plan.joins) plan.splits = (int)fewer;
  }
  while ((long)plan.blocks * plan.splits > 65535) plan.blocks /= 2;
  const long tiles = (longest + 15) / 16;
  plan.share = (int)(((tiles + plan.splits - 1) / plan.splits + 15) / 16 * 16);
  return plan;
}

int check_attend(const dkv_fp4_attend_args_t* p, const char* what) {
  DKV_REQUIRE(p, DKV_EINVAL, "%s: null arguments", what);
  const int rc = dkv::check_fp4_cache(&p->cache, what);
  if (rc) return rc;
  DKV_REQUIRE(p->query_dtype == DKV_F32 || p->query_dtype == DKV_F16 || p->query_dtype == DKV_BF16, DKV_EINVAL,
              "%s: query dtype %d not supported", what, p->query_dtype);
  DKV_REQUIRE(p->requests > 0 && p->requests <= 8192 && p->width > 0 && (int64_t)p->width * p->cache.page < dkv::kMostTokens && p->rows >= 0,
              DKV_ESHAPE, "%s: bad shape (requests=%d width=%d rows=%d)", what, p->requests, p->width, p->rows);
  DKV_REQUIRE(p->q_heads > 0 && p->q_heads % p->cache.kv_heads == 0, DKV_ESHAPE,
              "%s: %d query heads over %d KV heads", what, p->q_heads, p->cache.kv_heads);
  DKV_REQUIRE((int64_t)p->rows * p->q_heads < (1L << 31) - 65536, DKV_ESHAPE, "%s: %d rows of %d heads pass 2^31", what, p->rows, p->q_heads);
  DKV_REQUIRE((uintptr_t)p->arrivals % 4 == 0 && p->arrivals_count >= 0, DKV_EINVAL, "%s: misaligned arrivals, or %d of them", what,
              p->arrivals_count);
  DKV_REQUIRE(p->window >= 0, DKV_ESHAPE, "%s: window %d", what, p->window);
  return DKV_OK;
}

size_t part_bytes(const dkv_fp4_attend_args_t& p, const Plan& plan) {
  if (plan.splits == 1) return 0;
  return (size_t)p.rows * p.q_heads * plan.splits * (p.cache.head_dim * sizeof(float) + sizeof(float2));
}

template <int D, typename T>
void launch(const AttendArgs& a, const Plan& plan, int q_heads, hipStream_t st) {
  const dim3 grid(a.c.kv_heads, plan.blocks * plan.splits, a.requests), block(plan.waves * 64);
  constexpr bool wide = D < 256 && sizeof(T) == 2;
  if (plan.tiles == 1) {
    if (plan.waves == 8) hipLaunchKernelGGL((fp4_attend_kernel<D, T, 1, D == 256 ? 2 : 4, 8>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((fp4_attend_kernel<D, T, 1, D == 256 ? 2 : 4, 4>), grid, block, 0, st, a);
  } else if (plan.tiles == 2) {
    if constexpr (D < 256 || sizeof(T) == 2) hipLaunchKernelGGL((fp4_attend_kernel<D, T, 2, 2, 4>), grid, block, 0, st, a);
  } else {
    if constexpr (wide) hipLaunchKernelGGL((fp4_attend_kernel<D, T, 4, 2, 4>), grid, block, 0, st, a);
  }
  const long rows = (long)a.rows * q_heads;
  if (plan.splits == 1 || a.arrivals) return;
  if (plan.splits > kFewSplits) {
    hipLaunchKernelGGL((fp4_join_kernel<D, T>), dim3((unsigned)rows), dim3(256), 0, st, a, q_heads);
  } else {
    constexpr int kSets = 1024 / D;
    hipLaunchKernelGGL((fp4_join_few_kernel<D, T>), dim3((unsigned)((rows + kSets - 1) / kSets)), dim3(256), 0, st, a, q_heads);
  }
}

template <int D>
void launch_type(const AttendArgs& a, const Plan& plan, int q_heads, int dtype, hipStream_t st) {
  if (dtype == DKV_F32) launch<D, float>(a, plan, q_heads, st);
  else if (dtype == DKV_F16) launch<D, half_t>(a, plan, q_heads, st);
  else launch<D, dkv_bf16>(a, plan, q_heads, st);
}

}  // namespace

extern "C" size_t dkv_fp4_attend_workspace_bytes(const dkv_fp4_attend_args_t* p) {
  if (check_attend(p, "dkv_fp4_attend_workspace_bytes")) return 0;
  return part_bytes(*p, plan_of(*p)) + 16;
}

extern "C" int dkv_fp4_attend(const dkv_fp4_attend_args_t* p, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_attend(p, "dkv_fp4_attend");
  if (rc) return rc;
  if (p->rows == 0) return DKV_OK;
  DKV_REQUIRE(p->table && p->lengths && p->cu && p->query && p->out, DKV_EINVAL, "dkv_fp4_attend: null pointer");
  const int unit = p->query_dtype == DKV_F32 ? 4 : 8;
  DKV_REQUIRE((((uintptr_t)p->query | (uintptr_t)p->out) & 15) == 0 && p->query_token % unit == 0 && p->query_head % unit == 0,
              DKV_EINVAL, "dkv_fp4_attend: query rows and out must be 16-byte aligned");
  const Plan plan = plan_of(*p);
  const size_t need = part_bytes(*p, plan);
  DKV_REQUIRE(need == 0 || workspace, DKV_EINVAL, "dkv_fp4_attend: null workspace");
  DKV_REQUIRE(need <= workspace_bytes, DKV_EWORKSPACE, "dkv_fp4_attend: workspace %zu < %zu bytes", workspace_bytes, need);
  DKV_REQUIRE(((uintptr_t)workspace & 15) == 0, DKV_EINVAL, "dkv_fp4_attend: workspace must be 16-byte aligned");
  AttendArgs a{};
  a.c = p->cache;
  a.table = p->table; a.lengths = p->lengths; a.cu = p->cu; a.query = p->query; a.out = p->out;
  a.part = (float*)workspace;
  a.part_ml = (float2*)(a.part + (size_t)p->rows * p->q_heads * plan.splits * p->cache.head_dim);
  if (plan.joins) a.arrivals = p->arrivals;
  a.query_token = p->query_token; a.query_head = p->query_head;
  a.requests = p->requests; a.width = p->width; a.shift = dkv::page_shift(p->cache.page); a.rows = p->rows;
  a.groups = p->q_heads / p->cache.kv_heads;
  a.window = p->window ? p->window : INT32_MAX;
  a.splits = plan.splits; a.share = plan.share; a.fill = p->fill;
  // a positive factor keeps the order of the scores; one of 0 weighs every token the same, as the smallest does
  a.scale = fmaxf(fabsf(p->scaling) * 1.44269504088896340736f, 1.1754944e-38f);
  if (p->scaling != p->scaling) a.scale = p->scaling;
  a.negate = p->scaling < 0.0f;
  hipStream_t st = dkv::as_stream(stream);
  if (a.c.head_dim == 64) launch_type<64>(a, plan, p->q_heads, p->query_dtype, st);
  else if (a.c.head_dim == 128) launch_type<128>(a, plan, p->q_heads, p->query_dtype, st);
  else launch_type<256>(a, plan, p->q_heads, p->query_dtype, st);
  return dkv::check_launch("dkv_fp4_attend");
}
