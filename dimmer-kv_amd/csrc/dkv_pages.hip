// A paged KV cache in 4 bits: block tables and slot maps from request lengths, rows quantized into pages and read back.
// The form of the values, of a page and of the tables is stated in include/dimmerkv.h.
#include "dkv_device.h"
#include "dkv_fp4.h"
#include "dkv_host.h"

namespace {

// ---------------------------------------------------------------------------
// Pages for new tokens, and pages given back.  Both are a running sum over the requests (rows and pages of those before
// it) followed by independent work on rows and pages, which find their request by bisection in the sums.  Every workgroup
// makes the sums for itself in LDS, so one launch serves; what the sums are made of (lengths, free count) is rewritten by
// the workgroup that ends last, when all others have read it.  Latency is what it costs: one token each of 256 requests
// 4.4 us, 217K rows of 48 prompts 7.3 us (68 us with a device-wide fence before each arrival, which writes a die's cache
// back).
// ---------------------------------------------------------------------------
constexpr int kPageThreads = 1024;
constexpr int kMaxRequests = 8192;  // two 32-bit sums each in LDS

struct PageArgs {
  const int32_t* change;  // assign: new tokens; trim: tokens kept
  int32_t* lengths;
  int32_t* table;
  int32_t* free_pages;
  int32_t* free_count;
  int32_t* state;
  int64_t* slots;
  int64_t* positions;
  int32_t* cu;
  int requests, width, shift, pages, rows;
};

// Running sum of counts below 2^31 over a wave, in two 32-bit scans of 16 bits each.
DKV_DEVICE long wave_scan_long(long v) {
  return ((long)wave_scan((int)(v >> 16)) << 16) + wave_scan((int)(v & 0xffff));
}

DKV_DEVICE long pages_of(long tokens, int shift) { return (tokens + (1L << shift) - 1) >> shift; }

// Last request whose sum is at most x (requests without any share their sum with the next one).
DKV_DEVICE int owner_of(const int* sums, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// state: [0] why the last assign was refused (0: it was not), [1] arrivals of the running call, [2] the last trim's.
template <bool ASSIGN>
__global__ __launch_bounds__(kPageThreads) void pages_kernel(PageArgs a) {
  extern __shared__ int sums[];
  int* row_sum = sums;                // rows before request b
  int* page_sum = sums + a.requests;  // pages before request b
  __shared__ long wave_total[2][kPageThreads / 64];
  __shared__ int too_wide, last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) too_wide = 0;
  const int free_count = min(max(*a.free_count, 0), a.pages);
  long rows_before = 0, pages_before = 0;
  for (int b0 = 0; b0 < a.requests; b0 += kPageThreads) {
    const int b = b0 + tid;
    long rows = 0, pages = 0;
    bool wide = false;
    if (b < a.requests) {
      const long len = max(a.lengths[b], 0), change = max(a.change[b], 0);
      if (ASSIGN) {
        rows = change;
        const long after = pages_of(len + change, a.shift);
        pages = after - pages_of(len, a.shift);
        wide = after > a.width;
      } else {
        // a length past its table row is no length: nothing is taken from there
        pages = min(pages_of(len, a.shift), (long)a.width) - min(pages_of(min(len, change), a.shift), (long)a.width);
      }
    }
    const long rows_upto = ASSIGN ? wave_scan_long(rows) : 0, pages_upto = wave_scan_long(pages);
    __syncthreads();  // the sums of the block of requests before have been read
    if (lane == 63) {
      wave_total[0][wave] = rows_upto;
      wave_total[1][wave] = pages_upto;
    }
    if (wide) too_wide = 1;
    __syncthreads();
    long r = rows_before, p = pages_before;
    for (int w = 0; w < kPageThreads / 64; ++w) {
      if (w < wave) { r += wave_total[0][w]; p += wave_total[1][w]; }
      rows_before += wave_total[0][w];
      pages_before += wave_total[1][w];
    }
    if (b < a.requests) {
      if (ASSIGN) row_sum[b] = (int)min(r + rows_upto - rows, (long)INT32_MAX);
      page_sum[b] = (int)min(p + pages_upto - pages, (long)INT32_MAX);
    }
  }
  __syncthreads();
  int refused = 0;
  if (ASSIGN) {
    if (rows_before > a.rows) refused = DKV_PAGES_ROWS;
    else if (too_wide) refused = DKV_PAGES_WIDTH;
    else if (pages_before > free_count) refused = DKV_PAGES_FREE;
  } else if (pages_before > a.pages - free_count) {
    refused = DKV_PAGES_FREE;
  }
  const int total_rows = refused ? 0 : (int)rows_before, total_pages = refused ? 0 : (int)pages_before;
  const long step = (long)gridDim.x * kPageThreads, first = (long)blockIdx.x * kPageThreads + tid;
  if (ASSIGN) {
    const int mask = (1 << a.shift) - 1;
    for (long r = first; r < a.rows; r += step) {
      long slot = -1, position = -1;
      if (r < total_rows) {
        const int b = owner_of(row_sum, a.requests, (int)r);
        const long len = max(a.lengths[b], 0), held = pages_of(len, a.shift);
        position = len + (r - row_sum[b]);
        const long at = position >> a.shift;
        const int id = at < held ? a.table[(long)b * a.width + at]
                                 : a.free_pages[free_count - 1 - (page_sum[b] + (int)(at - held))];
        slot = ((long)id << a.shift) | (position & mask);
      }
      a.slots[r] = slot;
      a.positions[r] = position;
    }
  }
  for (long f = first; f < total_pages; f += step) {
    const int b = owner_of(page_sum, a.requests, (int)f);
    const long len = max(a.lengths[b], 0);
    if (ASSIGN) {
      a.table[(long)b * a.width + pages_of(len, a.shift) + (f - page_sum[b])] = a.free_pages[free_count - 1 - f];
    } else {
      const long left = pages_of(min(len, (long)max(a.change[b], 0)), a.shift);
      int32_t* entry = a.table + (long)b * a.width + left + (f - page_sum[b]);
      a.free_pages[free_count + total_pages - 1 - f] = *entry;
      *entry = -1;
    }
  }
  if (gridDim.x > 1) {
    // (what the last one must not overtake are the others' reads, and those have returned; nothing they wrote is read)
    __syncthreads();
    if (tid == 0) last = atomicAdd(a.state + 1, 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last) return;
  } else {
    __syncthreads();
  }
  for (int b = tid; b < a.requests; b += kPageThreads) {
    if (ASSIGN) a.cu[b] = refused ? 0 : row_sum[b];
    if (!refused) {
      const long len = max(a.lengths[b], 0), change = max(a.change[b], 0);
      a.lengths[b] = (int)(ASSIGN ? len + change : min(len, change));
    }
  }
  if (tid == 0) {
    if (ASSIGN) a.cu[a.requests] = total_rows;
    *a.free_count = ASSIGN ? free_count - total_pages : free_count + total_pages;
    a.state[ASSIGN ? 0 : 2] = refused;
    a.state[1] = 0;
  }
}

int check_pages(const dkv_pages_t* p, const char* what) {
  DKV_REQUIRE(p, DKV_EINVAL, "%s: null pages", what);
  DKV_REQUIRE(p->requests > 0 && p->requests <= kMaxRequests && p->width > 0 && p->pages > 0, DKV_ESHAPE,
              "%s: bad shape (requests=%d, at most %d; width=%d pages=%d)", what, p->requests, kMaxRequests, p->width, p->pages);
  DKV_REQUIRE(dkv::page_shift(p->page) >= 0, DKV_ESHAPE, "%s: page %d must be a power of two from 16 to 4096", what, p->page);
  DKV_REQUIRE((int64_t)p->width * p->page < dkv::kMostTokens, DKV_ESHAPE, "%s: %d pages of %d tokens pass 2^31 - 2^16 tokens a request",
              what, p->width, p->page);
  DKV_REQUIRE(p->lengths && p->table && p->free_pages && p->free_count && p->state, DKV_EINVAL, "%s: null pointer", what);
  return DKV_OK;
}

PageArgs page_args(const dkv_pages_t& p, const int32_t* change) {
  PageArgs a{};
  a.change = change;
  a.lengths = p.lengths; a.table = p.table; a.free_pages = p.free_pages; a.free_count = p.free_count; a.state = p.state;
  a.requests = p.requests; a.width = p.width; a.shift = dkv::page_shift(p.page); a.pages = p.pages;
  return a;
}

// ---------------------------------------------------------------------------
// Rows into the pages.  A lane takes 8 dimensions of one token and head (16 bytes of a 16-bit row, 4 bytes of codes);
// four lanes are a block of 32 and find its largest magnitude with two lane exchanges.  The exponent is read off that
// magnitude's bits, and the conversion rounds to the nearest code in one instruction for two values, so the pass is the
// memory's.  Consecutive lanes are a row's dimensions, then its next tokens: a wave writes whole lines of a page where
// the tokens are neighbours there.
// ---------------------------------------------------------------------------
struct StoreArgs {
  dkv_fp4_cache_t c;
  const void* rows[2];         // keys, values
  int64_t token[2], head[2];   // strides in elements
  const int64_t* slots;
  int n, shift;
};

// Magnitude bits of a block's largest value -> its exponent byte: e = floor(log2 amax) - 2, one more where amax would
// round past the largest code (1.75 * 2^floor(log2 amax) and above), clamped so that every value is an fp16 value.
// 255 for a block that holds an infinity or a NaN.
DKV_DEVICE uint32_t block_exponent(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return DKV_FP4_NAN;
  const int e = (int)(amax_bits >> 23) - 2 + ((amax_bits & 0x7fffffu) >= 0x600000u ? 1 : 0);
  return (uint32_t)min(max(e, 127 + DKV_FP4_EXP_MIN), 127 + DKV_FP4_EXP_MAX);
}

DKV_DEVICE uint32_t max_quad(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
}

template <typename T>
DKV_DEVICE void load8(const T* p, float (&x)[8]);
template <>
DKV_DEVICE void load8<float>(const float* p, float (&x)[8]) {
  const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <>
DKV_DEVICE void load8<half_t>(const half_t* p, float (&x)[8]) {
  const half8 h = *(const half8*)p;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
}
template <>
DKV_DEVICE void load8<dkv_bf16>(const dkv_bf16* p, float (&x)[8]) {
  const uint4 w = *(const uint4*)p;
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(v[i] << 16);
    x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
  }
}

// Where 8 dimensions (octet o) of a token's row lie in its page, in bytes: codes and the block's exponent.
template <int D>
DKV_DEVICE long code_at(bool value, long head_page, int at, int o, int page) {
  if (!value) return (head_page * page + at) * (D / 2) + o * 4;
  // inside a four of tokens: 16 lanes of D / 16 dimensions, each with four tokens' D / 32 bytes
  constexpr int kLane = D / 32;
  const int byte = o * 4, lane = byte / kLane, within = byte % kLane;
  return head_page * page * (D / 2) + (long)(at >> 2) * (2 * D) + lane * (4 * kLane) + (at & 3) * kLane + within;
}

template <int D>
DKV_DEVICE long scale_at(bool value, long head_page, int at, int block, int page) {
  if (!value) return (head_page * page + at) * (D / 32) + block;
  return head_page * page * (D / 32) + (long)(at >> 2) * (D / 8) + block * 4 + (at & 3);
}

template <int D, typename T>
__global__ __launch_bounds__(256) void fp4_store_kernel(StoreArgs a) {
  constexpr int kOct = D / 8, kTok = 256 / kOct;
  const int o = threadIdx.x % kOct, t = blockIdx.x * kTok + threadIdx.x / kOct;
  const int h = blockIdx.y;
  const bool value = blockIdx.z != 0;
  if (t >= a.n) return;
  const long slot = a.slots[t];
  if (slot < 0 || slot >= (long)a.c.pages << a.shift) return;  // the same for the four lanes of a block
  float x[8];
  load8<T>((const T*)a.rows[value] + t * a.token[value] + h * a.head[value] + o * 8, x);
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);
  const uint32_t e = block_exponent(max_quad(amax));
  uint32_t codes = 0;
  if (e != DKV_FP4_NAN) {
    const float scale = __uint_as_float(e << 23);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
  }
  const int page = a.c.page, at = (int)(slot & (page - 1));
  const long head_page = (slot >> a.shift) * a.c.kv_heads + h;
  uint8_t* code = (value ? a.c.value_codes : a.c.key_codes) + code_at<D>(value, head_page, at, o, page);
  if (D == 64 && value) {  // a lane's 4 dimensions are 2 bytes: an octet is two lanes, four tokens' bytes apart
    *(uint16_t*)code = (uint16_t)codes;
    *(uint16_t*)(code + 8) = (uint16_t)(codes >> 16);
  } else {
    *(uint32_t*)code = codes;
  }
  if ((o & 3) == 0) (value ? a.c.value_scales : a.c.key_scales)[scale_at<D>(value, head_page, at, o >> 2, page)] = (uint8_t)e;
}

// ---------------------------------------------------------------------------
// Raw projections into the pages: keys rotated on the way, and the queries rotated beside them.  A rotated key next to the
// border of two codes must fall on the right side, and float32 sums do not tell: so each sum of 16-bit rows is made in
// float32 with a bound on its error, and rounded from both ends of that.  Where the two agree the exact sum rounds to the same;
// where a wave's 512 hold one that does not, it makes them all again in float64: products of float32 are exact there, and
// what the sum loses, and its cut to float32, set the last bit, which keeps it on its side of every border of fewer bits.  Of
// rotated normal numbers that is one float16 query in 1,300 and one bfloat16 in 9,000 (a third and a twentieth of the
// waves), and one key in some 10^5 (less than a wave in a thousand).  Dimensions that are not rotated have no bound to fail.
// Float32 rows are summed in float64 at once.
// The pass is the memory's: 16,384 rows of 24 + 8 + 8 heads of 128 bfloat16 dimensions (294 MB) 64 us among other passes (4.6
// TB/s) and 57 where a graph repeats it (float16 55, 8,192 float32 rows 60), against 102 there with float64 for all and a head
// a thread.  With half of the dimensions rotated 77 and 82 (an octet a lane, whose partner is read twice), in neighbouring
// pairs 66 and 71.  64 rows of 32 + 8 + 8 heads of 64 float16 dimensions 4.5 us, which is latency.
// A lane takes an octet of dimensions, and the one it is rotated with where all dimensions are in halves, so that nothing
// is read twice; it keeps its angles for all the heads that it takes.
// ---------------------------------------------------------------------------
struct AppendArgs {
  dkv_fp4_cache_t c;
  const void* rows[3];        // queries, keys, values
  void* out;
  int64_t token[3], head[3];  // strides in elements
  int64_t out_token, out_head;
  const int64_t* slots;
  const int64_t* positions;
  const float* cos;
  const float* sin;
  int64_t cos_row, sin_row;
  int n, shift, q_heads, rotary, table_rows, fill;
  int each;  // heads that a thread takes, of the queries', the keys' and the values' in turn
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Eight floats rounded to a 16-bit type, as words.
DKV_DEVICE uint4 rounded(const float (&x)[8], half_t) {
  half8 y;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (half_t)x[i];
  uint4 w;
  __builtin_memcpy(&w, &y, 16);
  return w;
}
DKV_DEVICE uint4 rounded(const float (&x)[8], dkv_bf16) {
  bf16x8 y;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (__bf16)x[i];
  uint4 w;
  __builtin_memcpy(&w, &y, 16);
  return w;
}
DKV_DEVICE bool differ(uint4 a, uint4 b) { return ((a.x ^ b.x) | (a.y ^ b.y) | (a.z ^ b.z) | (a.w ^ b.w)) != 0; }

// One octet: x c + y s, y with its partners and s with the sign of its side.
struct Turn {
  float x[8], y[8], c[8], s[8];
  bool stays;  // the octet is not rotated: c is 1 (or NaN), y 0 and s -0, so that sums are x, the sign of a zero too
  // The sums in float32, and by how much their ends r - off and r + off have to lie apart from them: 2^-24 of the product that is
  // rounded, of the sum, and of the sum once more for the rounding of the end itself; 2^-20 of that more for the roundings in off.
  DKV_DEVICE void sums(float (&r)[8], float (&off)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float product = y[i] * s[i];
      r[i] = fmaf(x[i], c[i], product);
      off[i] = stays ? 0.0f : fmaf(fmaf(2.0f, fabsf(r[i]), fabsf(product)), 0x1.00001p-24f, 0x1p-140f);
    }
  }
  // What a sum in float64 lacks of its two products, which are exact there.
  DKV_DEVICE double lacks(int i, double sum) const {
    const double one = (double)x[i] * c[i], two = (double)y[i] * s[i], took = sum - one;
    return (one - (sum - took)) + (two - took);
  }
  // The exact sum cut to float32, its last bit set where that loses something: rounding the result once more to fewer bits, to
  // either side of a border of fewer bits, is rounding the exact one.  What float64 lacks is asked for only where float32 seems
  // to hold the sum: the five additions for all eight at once would take registers that there are not (16,384 rows 130 us
  // instead of 82, with their load).
  DKV_DEVICE float cut_to_odd(int i) const {
    const double sum = (double)x[i] * c[i] + (double)y[i] * s[i];
    const float f = (float)sum;
    double rest = sum - (double)f;
    if (__builtin_expect(rest == 0.0 && !stays, 0)) rest = lacks(i, sum);
    if (!(fabs(rest) > 0.0)) return f;  // (nor of infinities)
    return __uint_as_float((__float_as_uint(f) - (signbit(rest) != signbit(f) ? 1u : 0u)) | 1u);
  }
  // The exact sum rounded to float32.  A sum in float64 that lies between two floats is on its side of their middle, or on it
  // (the 28 last bits are zero), where a last bit that is set tells the side.
  DKV_DEVICE float nearest(int i) const {
    const double sum = (double)x[i] * c[i] + (double)y[i] * s[i];
    long bits = __double_as_longlong(sum);
    if (__builtin_expect(!(bits & 0xfffffff) && !stays, 0)) {
      const double rest = lacks(i, sum);
      if (fabs(rest) > 0.0) bits += (rest > 0.0) == (sum > 0.0) ? 1 : -1;
    }
    return (float)__longlong_as_double(bits);
  }
};

template <typename T>
DKV_DEVICE void put_query(T* p, const Turn& turn) {
  if constexpr (sizeof(T) == 2) {
    float r[8], off[8], low[8], high[8], most = 0.0f;
    turn.sums(r, off);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      low[i] = r[i] - off[i];
      high[i] = r[i] + off[i];
      most = __builtin_elementwise_maximum(most, off[i]);
    }
    uint4 w = rounded(low, T());
    // (An infinity beside a product past float32 may be NaN at both ends, and no bound tells.)
    if (__any(!turn.stays && (differ(w, rounded(high, T())) || !(most < INFINITY)))) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = turn.cut_to_odd(i);
      w = rounded(r, T());
    }
    *(uint4*)p = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i += 4)
      *(float4*)(p + i) = make_float4(turn.nearest(i), turn.nearest(i + 1), turn.nearest(i + 2), turn.nearest(i + 3));
  }
}

DKV_DEVICE uint32_t octet_codes(const float (&x)[8], uint32_t e) {
  const float scale = __uint_as_float(e << 23);
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
}

// An octet's codes and its block's exponent into their slot.
template <int D>
DKV_DEVICE void place_octet(const dkv_fp4_cache_t& c, int shift, bool value, long slot, int h, int o, uint32_t codes, uint32_t e) {
  const int page = c.page, at = (int)(slot & (page - 1));
  const long head_page = (slot >> shift) * c.kv_heads + h;
  uint8_t* code = (value ? c.value_codes : c.key_codes) + code_at<D>(value, head_page, at, o, page);
  if (D == 64 && value) {  // a lane's 4 dimensions are 2 bytes: an octet is two lanes, four tokens' bytes apart
    *(uint16_t*)code = (uint16_t)codes;
    *(uint16_t*)(code + 8) = (uint16_t)(codes >> 16);
  } else {
    *(uint32_t*)code = codes;
  }
  if ((o & 3) == 0) (value ? c.value_scales : c.key_scales)[scale_at<D>(value, head_page, at, o >> 2, page)] = (uint8_t)e;
}

template <int D>
DKV_DEVICE void put_octet(const dkv_fp4_cache_t& c, int shift, bool value, long slot, int h, int o, const float (&x)[8]) {
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);
  const uint32_t e = block_exponent(max_quad(amax));
  place_octet<D>(c, shift, value, slot, h, o, e == DKV_FP4_NAN ? 0u : octet_codes(x, e), e);
}

template <int D, typename T>
DKV_DEVICE void put_key(const dkv_fp4_cache_t& c, int shift, long slot, int h, int o, const Turn& turn) {
  float r[8];
  if constexpr (sizeof(T) == 2) {
    float off[8], low[8], high[8], least = 0.0f, most = 0.0f;  // (NaN and infinities: the ends differ, or are one's exponent)
    turn.sums(r, off);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      low[i] = r[i] - off[i];
      high[i] = r[i] + off[i];
      least = __builtin_elementwise_maximum(least, fabsf(r[i]) - off[i]);
      most = __builtin_elementwise_maximum(most, fabsf(r[i]) + off[i]);
    }
    const uint32_t e = block_exponent(max_quad(__float_as_uint(most) & 0x7fffffffu));
    const uint32_t codes = octet_codes(low, min(e, 254u));
    const bool certain = e != DKV_FP4_NAN && e == block_exponent(max_quad(__float_as_uint(least) & 0x7fffffffu)) &&
                         (turn.stays || codes == octet_codes(high, min(e, 254u)));
    if (!__any(!certain)) return place_octet<D>(c, shift, false, slot, h, o, codes, e);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = turn.cut_to_odd(i);
  put_octet<D>(c, shift, false, slot, h, o, r);
}

constexpr int kWholeHalves = 0, kHalves = 1, kPairs = 2;  // all dimensions in halves, some, neighbours

template <int D, typename T, int LAYOUT>
__global__ __launch_bounds__(256, 4) void fp4_append_kernel(AppendArgs a) {
  constexpr int kOctets = LAYOUT == kWholeHalves ? 2 : 1, kLanes = D / 8 / kOctets, kTok = 256 / kLanes;
  const int o = threadIdx.x % kLanes, t = blockIdx.x * kTok + threadIdx.x / kLanes;
  if (t >= a.n) return;
  const long slot = a.slots[t], position = a.positions[t];
  const bool kept = slot >= 0 && slot < (long)a.c.pages << a.shift;  // the same for a row's lanes
  const int keys = a.q_heads, values = a.q_heads + a.c.kv_heads;
  const int y0 = blockIdx.y * a.each, y1 = min(y0 + a.each, values + a.c.kv_heads);
  const int half = a.rotary / 2, first = o * 8;
  const bool turns = LAYOUT == kWholeHalves || first < a.rotary, low = LAYOUT == kWholeHalves || first < half;
  Turn turn;
  turn.stays = !turns;
  if (turns && y0 < values) {
    const bool known = position >= 0 && position < a.table_rows;  // (else the row becomes NaN)
    if constexpr (LAYOUT == kPairs) {
      float4 c = make_float4(__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")), s = c;
      if (known) {
        c = *(const float4*)(a.cos + position * a.cos_row + o * 4);
        s = *(const float4*)(a.sin + position * a.sin_row + o * 4);
      }
      const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) turn.c[i] = cs[i >> 1], turn.s[i] = i & 1 ? sn[i >> 1] : -sn[i >> 1];
    } else {
      const int pair = low ? first : first - half;
#pragma unroll
      for (int i = 0; i < 8; ++i) turn.c[i] = turn.s[i] = __builtin_nanf("");
      if (known) {
        load8<float>(a.cos + position * a.cos_row + pair, turn.c);
        load8<float>(a.sin + position * a.sin_row + pair, turn.s);
        if (low)
#pragma unroll
          for (int i = 0; i < 8; ++i) turn.s[i] = -turn.s[i];
      }
    }
  } else if (y0 < values) {
    const float stays = position >= 0 && position < a.table_rows ? 1.0f : __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < 8; ++i) turn.c[i] = stays, turn.s[i] = -0.0f;
  }
  for (int y = y0; y < y1; ++y) {
    const int kind = y < keys ? 0 : y < values ? 1 : 2, h = kind == 0 ? y : kind == 1 ? y - keys : y - values;
    if (kind && !kept) continue;
    const T* row = (const T*)a.rows[kind] + t * a.token[kind] + h * a.head[kind];
    T* out = (T*)a.out + t * a.out_token + h * a.out_head + first;
    if (kind == 0 && position < 0) {
      if (a.fill)
#pragma unroll
        for (int k = 0; k < kOctets; ++k) __builtin_memset(out + k * (D / 2), 0, 8 * sizeof(T));
      continue;
    }
    float x[8], other[8] = {};
    load8<T>(row + first, x);
    if constexpr (LAYOUT == kWholeHalves) load8<T>(row + first + D / 2, other);
    if (kind == 2) {
      put_octet<D>(a.c, a.shift, true, slot, h, o, x);
      if constexpr (LAYOUT == kWholeHalves) put_octet<D>(a.c, a.shift, true, slot, h, o + kLanes, other);
      continue;
    }
    if constexpr (LAYOUT == kHalves) {
      if (turns) load8<T>(row + (low ? first + half : first - half), other);
      __builtin_amdgcn_wave_barrier();  // a row is one wave's: in place, no lane writes before its partner has read
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) turn.x[i] = x[i], turn.y[i] = LAYOUT == kPairs ? (turns ? x[i ^ 1] : 0.0f) : other[i];
    if (kind == 0) put_query<T>(out, turn);
    else put_key<D, T>(a.c, a.shift, slot, h, o, turn);
    if constexpr (LAYOUT == kWholeHalves) {
      Turn back = turn;
#pragma unroll
      for (int i = 0; i < 8; ++i) back.x[i] = other[i], back.y[i] = x[i], back.s[i] = -turn.s[i];
      if (kind == 0) put_query<T>(out + D / 2, back);
      else put_key<D, T>(a.c, a.shift, slot, h, o + kLanes, back);
    }
  }
}

template <int D, typename T>
constexpr auto append_whole = fp4_append_kernel<D, T, kWholeHalves>;
template <int D, typename T>
constexpr auto append_halves = fp4_append_kernel<D, T, kHalves>;
template <int D, typename T>
constexpr auto append_pairs = fp4_append_kernel<D, T, kPairs>;

struct LoadArgs {
  dkv_fp4_cache_t c;
  void* rows[2];  // [n][kv_heads][D]
  const int64_t* slots;
  int n, shift;
};

template <typename T>
DKV_DEVICE void store8(T* p, const float (&x)[8]);
template <>
DKV_DEVICE void store8<float>(float* p, const float (&x)[8]) {
  ((float4*)p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  ((float4*)p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <>
DKV_DEVICE void store8<half_t>(half_t* p, const float (&x)[8]) {
  half8 h;
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = (half_t)x[i];
  *(half8*)p = h;
}
template <>
DKV_DEVICE void store8<dkv_bf16>(dkv_bf16* p, const float (&x)[8]) {
  // (every value has two significant bits, and a NaN's upper half is one)
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (__float_as_uint(x[2 * i]) >> 16) | (__float_as_uint(x[2 * i + 1]) & 0xffff0000u);
  *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows out of the pages, the same lanes the other way; rows without a slot become zeros.
template <int D, typename T>
__global__ __launch_bounds__(256) void fp4_load_kernel(LoadArgs a) {
  constexpr int kOct = D / 8, kTok = 256 / kOct;
  const int o = threadIdx.x % kOct, t = blockIdx.x * kTok + threadIdx.x / kOct;
  const int h = blockIdx.y;
  const bool value = blockIdx.z != 0;
  if (t >= a.n) return;
  const long slot = a.slots[t];
  float x[8] = {};
  if (slot >= 0 && slot < (long)a.c.pages << a.shift) {
    const int page = a.c.page, at = (int)(slot & (page - 1));
    const long head_page = (slot >> a.shift) * a.c.kv_heads + h;
    const uint8_t* code = (value ? a.c.value_codes : a.c.key_codes) + code_at<D>(value, head_page, at, o, page);
    uint32_t codes;
    if (D == 64 && value) codes = *(const uint16_t*)code | ((uint32_t)*(const uint16_t*)(code + 8) << 16);
    else codes = *(const uint32_t*)code;
    const uint32_t e = (value ? a.c.value_scales : a.c.key_scales)[scale_at<D>(value, head_page, at, o >> 2, page)];
    const float scale = __uint_as_float(e << 23);
    floatx2 p[4];
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = e == DKV_FP4_NAN ? __uint_as_float(0x7fc00000u) : p[i >> 1][i & 1];
  }
  store8<T>((T*)a.rows[value] + ((long)t * a.c.kv_heads + h) * D + o * 8, x);
}

// (head_dim, element type) -> the kernel's instance
#define DKV_FP4_BY_TYPE(kernel, D, dtype, ...)                                                           \
  do {                                                                                                   \
    if ((dtype) == DKV_F32) hipLaunchKernelGGL((kernel<D, float>), __VA_ARGS__);                         \
    else if ((dtype) == DKV_F16) hipLaunchKernelGGL((kernel<D, half_t>), __VA_ARGS__);                   \
    else hipLaunchKernelGGL((kernel<D, dkv_bf16>), __VA_ARGS__);                                         \
  } while (0)
#define DKV_FP4_BY_SHAPE(kernel, dim, dtype, ...)                                                        \
  do {                                                                                                   \
    if ((dim) == 64) DKV_FP4_BY_TYPE(kernel, 64, dtype, __VA_ARGS__);                                    \
    else if ((dim) == 128) DKV_FP4_BY_TYPE(kernel, 128, dtype, __VA_ARGS__);                             \
    else DKV_FP4_BY_TYPE(kernel, 256, dtype, __VA_ARGS__);                                               \
  } while (0)

int check_rows(const dkv_fp4_cache_t* c, const void* key, const void* value, int32_t dtype, const int64_t* slots, int32_t n,
               const char* what) {
  const int rc = dkv::check_fp4_cache(c, what);
  if (rc) return rc;
  DKV_REQUIRE(dtype == DKV_F32 || dtype == DKV_F16 || dtype == DKV_BF16, DKV_EINVAL, "%s: dtype %d not supported", what, dtype);
  DKV_REQUIRE(n >= 0 && n <= INT32_MAX - 65536, DKV_ESHAPE, "%s: %d rows", what, n);  // (a workgroup runs past the last)
  if (n == 0) return DKV_OK;
  DKV_REQUIRE(key && value && slots, DKV_EINVAL, "%s: null pointer", what);
  DKV_REQUIRE((((uintptr_t)key | (uintptr_t)value) & 15) == 0, DKV_EINVAL, "%s: rows must be 16-byte aligned", what);
  return DKV_OK;
}

}  // namespace

extern "C" int dkv_page_assign(const dkv_pages_t* p, const int32_t* new_tokens, int32_t rows, int64_t* slots,
                               int64_t* positions, int32_t* cu, void* stream) {
  const int rc = check_pages(p, "dkv_page_assign");
  if (rc) return rc;
  DKV_REQUIRE(rows >= 0 && rows <= INT32_MAX - 65536, DKV_ESHAPE, "dkv_page_assign: %d rows", rows);
  DKV_REQUIRE(new_tokens && cu && (rows == 0 || (slots && positions)), DKV_EINVAL, "dkv_page_assign: null pointer");
  PageArgs a = page_args(*p, new_tokens);
  a.slots = slots; a.positions = positions; a.cu = cu; a.rows = rows;
  const int blocks = min(max((rows + kPageThreads - 1) / kPageThreads, 1), 256);
  hipLaunchKernelGGL(pages_kernel<true>, dim3(blocks), dim3(kPageThreads), p->requests * 2 * sizeof(int), dkv::as_stream(stream), a);
  return dkv::check_launch("dkv_page_assign");
}

extern "C" int dkv_page_trim(const dkv_pages_t* p, const int32_t* keep, void* stream) {
  const int rc = check_pages(p, "dkv_page_trim");
  if (rc) return rc;
  DKV_REQUIRE(keep, DKV_EINVAL, "dkv_page_trim: null pointer");
  // a page a thread at the most: the pages the table can hold
  const long most = min((long)p->requests * p->width, (long)p->pages);
  const int blocks = (int)min(max((most + kPageThreads - 1) / kPageThreads, 1L), 16L);
  hipLaunchKernelGGL(pages_kernel<false>, dim3(blocks), dim3(kPageThreads), p->requests * 2 * sizeof(int),
                     dkv::as_stream(stream), page_args(*p, keep));
  return dkv::check_launch("dkv_page_trim");
}

extern "C" int dkv_fp4_store(const dkv_fp4_cache_t* c, const void* key, const void* value, int32_t dtype, int64_t key_token,
                             int64_t key_head, int64_t value_token, int64_t value_head, const int64_t* slots, int32_t n,
                             void* stream) {
  const int rc = check_rows(c, key, value, dtype, slots, n, "dkv_fp4_store");
  if (rc || n == 0) return rc;
  const int unit = dtype == DKV_F32 ? 4 : 8;
  DKV_REQUIRE(key_token % unit == 0 && key_head % unit == 0 && value_token % unit == 0 && value_head % unit == 0, DKV_EINVAL,
              "dkv_fp4_store: row strides must be multiples of 16 bytes");
  StoreArgs a{};
  a.c = *c;
  a.rows[0] = key; a.rows[1] = value;
  a.token[0] = key_token; a.token[1] = value_token; a.head[0] = key_head; a.head[1] = value_head;
  a.slots = slots; a.n = n; a.shift = dkv::page_shift(c->page);
  const int tok = 256 / (c->head_dim / 8);
  DKV_FP4_BY_SHAPE(fp4_store_kernel, c->head_dim, dtype, dim3((n + tok - 1) / tok, c->kv_heads, 2), dim3(256), 0,
                   dkv::as_stream(stream), a);
  return dkv::check_launch("dkv_fp4_store");
}

extern "C" int dkv_fp4_load(const dkv_fp4_cache_t* c, const int64_t* slots, int32_t n, void* key, void* value, int32_t dtype,
                            void* stream) {
  const int rc = check_rows(c, key, value, dtype, slots, n, "dkv_fp4_load");
  if (rc || n == 0) return rc;
  LoadArgs a{};
  a.c = *c;
  a.rows[0] = key; a.rows[1] = value;
  a.slots = slots; a.n = n; a.shift = dkv::page_shift(c->page);
  const int tok = 256 / (c->head_dim / 8);
  DKV_FP4_BY_SHAPE(fp4_load_kernel, c->head_dim, dtype, dim3((n + tok - 1) / tok, c->kv_heads, 2), dim3(256), 0,
                   dkv::as_stream(stream), a);
  return dkv::check_launch("dkv_fp4_load");
}

extern "C" int dkv_fp4_append(const dkv_fp4_append_args_t* p, void* stream) {
  const char* what = "dkv_fp4_append";
  DKV_REQUIRE(p, DKV_EINVAL, "%s: null arguments", what);
  const int rc = check_rows(&p->cache, p->key, p->value, p->dtype, p->slots, p->rows, what);
  if (rc) return rc;
  const int dim = p->cache.head_dim;
  DKV_REQUIRE(p->rotary >= 16 && p->rotary <= dim && p->rotary % 16 == 0, DKV_ESHAPE,
              "%s: %d rotated dimensions of %d (a multiple of 16)", what, p->rotary, dim);
  DKV_REQUIRE(p->table_rows > 0, DKV_ESHAPE, "%s: tables of %d rows", what, p->table_rows);
  DKV_REQUIRE(p->q_heads >= 0 && (p->query != nullptr || p->q_heads == 0), DKV_EINVAL, "%s: %d heads of null queries", what, p->q_heads);
  DKV_REQUIRE((int64_t)p->q_heads + 2 * p->cache.kv_heads <= 65535, DKV_ESHAPE, "%s: %d query heads and %d KV heads", what,
              p->q_heads, p->cache.kv_heads);
  if (p->rows == 0) return DKV_OK;
  DKV_REQUIRE(p->positions && p->cos && p->sin && (p->q_heads == 0 || p->out), DKV_EINVAL, "%s: null pointer", what);
  DKV_REQUIRE((((uintptr_t)p->query | (uintptr_t)p->out | (uintptr_t)p->cos | (uintptr_t)p->sin) & 15) == 0, DKV_EINVAL,
              "%s: rows and tables must be 16-byte aligned", what);
  const int unit = p->dtype == DKV_F32 ? 4 : 8;
  DKV_REQUIRE(p->key_token % unit == 0 && p->key_head % unit == 0 && p->value_token % unit == 0 && p->value_head % unit == 0 &&
                  p->cos_row % 4 == 0 && p->sin_row % 4 == 0,
              DKV_EINVAL, "%s: row strides must be multiples of 16 bytes", what);
  DKV_REQUIRE(p->q_heads == 0 || (p->query_token % unit == 0 && p->query_head % unit == 0 && p->out_token % unit == 0 &&
                                  p->out_head % unit == 0),
              DKV_EINVAL, "%s: row strides must be multiples of 16 bytes", what);
  AppendArgs a{};
  a.c = p->cache;
  a.rows[0] = p->query; a.rows[1] = p->key; a.rows[2] = p->value; a.out = p->out;
  a.token[0] = p->query_token; a.token[1] = p->key_token; a.token[2] = p->value_token;
  a.head[0] = p->query_head; a.head[1] = p->key_head; a.head[2] = p->value_head;
  a.out_token = p->out_token; a.out_head = p->out_head;
  a.slots = p->slots; a.positions = p->positions;
  a.cos = p->cos; a.sin = p->sin; a.cos_row = p->cos_row; a.sin_row = p->sin_row;
  a.n = p->rows; a.shift = dkv::page_shift(p->cache.page);
  a.q_heads = p->q_heads; a.rotary = p->rotary; a.table_rows = p->table_rows; a.fill = p->fill;
  const bool whole = !p->interleaved && p->rotary == dim;
  const int tok = 256 / (whole ? dim / 16 : dim / 8), heads = p->q_heads + 2 * p->cache.kv_heads;
  // A thread keeps its angles for up to sixteen heads where that leaves the card full: 53 us for the 16,384 rows above,
  // 83 a head a thread.
  const long blocks = (p->rows + tok - 1) / tok;
  a.each = (int)min(max(blocks * heads / 2048, 1L), 16L);
  const dim3 grid((unsigned)blocks, (heads + a.each - 1) / a.each), block(256);
  if (whole) DKV_FP4_BY_SHAPE(append_whole, dim, p->dtype, grid, block, 0, dkv::as_stream(stream), a);
  else if (p->interleaved) DKV_FP4_BY_SHAPE(append_pairs, dim, p->dtype, grid, block, 0, dkv::as_stream(stream), a);
  else DKV_FP4_BY_SHAPE(append_halves, dim, p->dtype, grid, block, 0, dkv::as_stream(stream), a);
  return dkv::check_launch(what);
}
