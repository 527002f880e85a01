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
