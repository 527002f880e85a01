// The logits of replies under penalties for repeated tokens, biases and a grammar's masks, and the token picked
// (include/dimmerkv.h states the arithmetic).
//
// One pass over the logits: a workgroup takes a stretch of a row's vocabulary, counts the history's tokens that fall into
// it in LDS (integer atomics: the order does not matter), and then streams the stretch once.  Every float32 operation is
// rounded on its own, in the stated order, so equal inputs stay equal and ties are ties.
#include <math.h>

#include "dkv_device.h"
#include "dkv_fp4.h"
#include "dkv_host.h"

namespace {

constexpr uint32_t kSeen = 0x80000000u;  // in a count: the prompt holds the token
constexpr int kThreads = 512;

struct LogitsArgs {
  dkv_logits_args_t p;
  uint64_t* partial;  // [rows][chunks] keys of the best token of each stretch; null when there is one stretch
  int chunk, chunks;  // elements of a stretch, and how many there are
};

// Float order as unsigned order; a NaN above all, both zeros the same.
DKV_DEVICE uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kNothing = 0x007fffffu;  // of -infinity

DKV_DEVICE uint64_t best_of(uint64_t a, uint64_t b) { return a > b ? a : b; }

DKV_DEVICE uint64_t wave_best(uint64_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = best_of(v, __shfl_xor(v, d));
  return v;
}

DKV_DEVICE int64_t picked(uint64_t best) {
  const uint32_t key = (uint32_t)(best >> 32);
  return key <= kNothing ? -1 : (int64_t)(uint32_t)~(uint32_t)best;
}

DKV_DEVICE float logit_value(float x) { return x; }
DKV_DEVICE float logit_value(half_t x) { return (float)x; }
DKV_DEVICE float logit_value(dkv_bf16 x) { return bf16_bits_to_float(x.bits); }
DKV_DEVICE void set_logit(float& y, float x) { y = x; }
DKV_DEVICE void set_logit(half_t& y, float x) { y = (half_t)x; }
DKV_DEVICE void set_logit(dkv_bf16& y, float x) { y.bits = float_to_bf16_bits(x); }

template <typename T, typename ID, bool BIAS>
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(LogitsArgs a) {
#pragma clang fp contract(off)
  constexpr int V = 16 / sizeof(T);
  extern __shared__ uint32_t lds[];
  uint32_t* counts = lds;           // [chunk]
  uint32_t* last = lds + a.chunk;   // [chunk] with biases: place in the row's list, from 1
  __shared__ uint64_t bests[kThreads / 64];
  const dkv_logits_args_t& p = a.p;
  const int row = blockIdx.y, tid = threadIdx.x, vocab = p.vocab;
  const T* logits = (const T*)p.logits + row * p.logits_row;
  T* out = (T*)p.out + row * p.out_row;
  // Elements are numbered from the 16-byte line the row begins in; a row of any alignment is read in whole lines if its
  // out row begins alike.
  const int shift = (int)((uintptr_t)logits / sizeof(T) % V);
  const bool alike = shift == (int)((uintptr_t)out / sizeof(T) % V);
  const long first = (long)blockIdx.x * a.chunk - shift;  // token of the stretch's element 0

  for (int x = tid * 4; x < a.chunk * (BIAS ? 2 : 1); x += kThreads * 4) *(uint4*)(lds + x) = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (p.tokens) {
    const int length = min(max(p.lengths[row], 0), p.history), reply = p.reply ? max(p.reply[row], 0) : 0;
    const ID* tokens = (const ID*)p.tokens + row * p.tokens_row;
    for (int j = tid; j < length; j += kThreads) {
      const long id = tokens[j], at = id - first;
      if (id >= 0 && id < vocab && at >= 0 && at < a.chunk) {
        if (j >= reply) atomicAdd(counts + at, 1u);
        else if (!(counts[at] & kSeen)) atomicOr(counts + at, kSeen);
      }
    }
  }
  if (BIAS) {
    const int lo = max(p.bias_cu[row], 0), hi = min(p.bias_cu[row + 1], p.biases);
    for (int j = lo + tid; j < hi; j += kThreads) {
      const long id = p.bias_ids[j], at = id - first;
      if (id >= 0 && id < vocab && at >= 0 && at < a.chunk) atomicMax(last + at, (uint32_t)(j - lo) + 1);
    }
  }
  __syncthreads();

  const float repetition = p.repetition ? p.repetition[row] : 1.0f, presence = p.presence ? p.presence[row] : 0.0f,
              frequency = p.frequency ? p.frequency[row] : 0.0f;
  const uint32_t* allowed = nullptr;
  if (p.allowed) {
    const int mask = p.allowed_row ? p.allowed_row[row] : row;
    if (mask >= 0 && mask < p.masks) allowed = (const uint32_t*)p.allowed + (long)mask * p.words;
  }
  uint64_t best = 0;
  auto adjust = [&](float x, int at, int token, bool allow) {
    const uint32_t count = counts[at];
    if (count) {
      x = x > 0.0f ? x / repetition : x * repetition;
      const uint32_t n = count & ~kSeen;
      if (n) {
        const float less = frequency * (float)n;
        x = x - (less + presence);
      }
    }
    if (BIAS) {
      const uint32_t place = last[at];
      if (place) x = x + p.bias_values[max(p.bias_cu[row], 0) + (int)place - 1];
    }
    if (!allow) x = -INFINITY;
    best = best_of(best, (uint64_t)order_key(x) << 32 | (uint32_t)~token);
    return x;
  };
  for (int at = tid * V; at < a.chunk; at += kThreads * V) {
    const long token = first + at;
    if (token >= vocab) break;
    if (token >= 0 && token + V <= vocab) {
      uint64_t bits = ~0ull;
      if (allowed) {
        const int word = (int)token >> 5, in = (int)token & 31;
        bits = allowed[word] >> in;
        if (in + V > 32) bits |= (uint64_t)allowed[word + 1] << (32 - in);
      }
      T x[V], y[V];
      __builtin_memcpy(x, __builtin_assume_aligned(logits + token, 16), 16);
#pragma unroll
      for (int k = 0; k < V; ++k) set_logit(y[k], adjust(logit_value(x[k]), at + k, (int)token + k, (bits >> k) & 1));
      if (alike) {
        __builtin_memcpy(__builtin_assume_aligned(out + token, 16), y, 16);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) out[token + k] = y[k];
      }
    } else {
      for (int k = 0; k < V; ++k) {
        const long t = token + k;
        if (t < 0 || t >= vocab) continue;
        const bool allow = !allowed || ((allowed[t >> 5] >> (t & 31)) & 1);
        set_logit(out[t], adjust(logit_value(logits[t]), at + k, (int)t, allow));
      }
    }
  }
  if (!p.pick) return;
  best = wave_best(best);
  if ((tid & 63) == 0) bests[tid >> 6] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kThreads / 64; ++w) best = best_of(best, bests[w]);
    if (a.partial) a.partial[(long)row * a.chunks + blockIdx.x] = best;
    else p.pick[row] = picked(best);
  }
}

// The best of a row's stretches: a wave per row.
__global__ __launch_bounds__(256) void pick_kernel(const uint64_t* partial, int chunks, int rows, int64_t* pick) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= rows) return;
  uint64_t best = 0;
  for (int c = lane; c < chunks; c += 64) best = best_of(best, partial[(long)row * chunks + c]);
  best = wave_best(best);
  if (lane == 0) pick[row] = picked(best);
}

// 32 KB of LDS either way
int chunk_of(const dkv_logits_args_t& p) { return p.biases ? 4096 : 8192; }

// one element of a line at the most in front of a row's first
int chunks_of(const dkv_logits_args_t& p, int chunk) { return (int)(((long)p.vocab + 8 + chunk - 1) / chunk); }

int check_logits(const dkv_logits_args_t* p, const char* what) {
  DKV_REQUIRE(p, DKV_EINVAL, "%s: null arguments", what);
  DKV_REQUIRE(p->dtype == DKV_F32 || p->dtype == DKV_F16 || p->dtype == DKV_BF16, DKV_EINVAL, "%s: dtype %d not supported", what, p->dtype);
  DKV_REQUIRE(p->rows >= 0 && p->rows <= 65535 && p->vocab > 0 && p->vocab <= INT32_MAX - 65536, DKV_ESHAPE,
              "%s: bad shape (rows=%d, at most 65535; vocab=%d)", what, p->rows, p->vocab);
  DKV_REQUIRE(p->history >= 0 && p->biases >= 0 && p->masks >= 0, DKV_ESHAPE, "%s: bad shape (history=%d biases=%d masks=%d)",
              what, p->history, p->biases, p->masks);
  DKV_REQUIRE(p->token_bytes == 4 || p->token_bytes == 8 || !p->tokens, DKV_EINVAL, "%s: tokens of %d bytes", what, p->token_bytes);
  DKV_REQUIRE(!p->tokens || p->lengths, DKV_EINVAL, "%s: tokens without lengths", what);
  DKV_REQUIRE(!p->biases || (p->bias_ids && p->bias_values && p->bias_cu), DKV_EINVAL, "%s: null bias pointer", what);
  DKV_REQUIRE(!p->allowed || p->words >= ((int64_t)p->vocab + 31) / 32, DKV_ESHAPE, "%s: %d mask words for %d tokens", what, p->words, p->vocab);
  DKV_REQUIRE(!p->allowed || p->allowed_row || p->masks >= p->rows, DKV_ESHAPE, "%s: %d masks for %d rows", what, p->masks, p->rows);
  return DKV_OK;
}

template <typename T, typename ID>
void launch(const LogitsArgs& a, hipStream_t st) {
  const dim3 grid(a.chunks, a.p.rows);
  if (a.p.biases)
    hipLaunchKernelGGL((adjust_logits_kernel<T, ID, true>), grid, dim3(kThreads), a.chunk * 8, st, a);
  else
    hipLaunchKernelGGL((adjust_logits_kernel<T, ID, false>), grid, dim3(kThreads), a.chunk * 4, st, a);
}

template <typename T>
void launch_type(const LogitsArgs& a, hipStream_t st) {
  if (a.p.token_bytes == 4) launch<T, int32_t>(a, st);
  else launch<T, int64_t>(a, st);
}

}  // namespace

extern "C" size_t dkv_adjust_logits_workspace_bytes(const dkv_logits_args_t* p) {
  if (check_logits(p, "dkv_adjust_logits_workspace_bytes")) return 0;
  return (size_t)p->rows * chunks_of(*p, chunk_of(*p)) * sizeof(uint64_t) + 16;
}

extern "C" int dkv_adjust_logits(const dkv_logits_args_t* p, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_logits(p, "dkv_adjust_logits");
  if (rc) return rc;
  if (p->rows == 0) return DKV_OK;
  DKV_REQUIRE(p->logits && p->out, DKV_EINVAL, "dkv_adjust_logits: null pointer");
  const int size = p->dtype == DKV_F32 ? 4 : 2;
  DKV_REQUIRE((uintptr_t)p->logits % size == 0 && (uintptr_t)p->out % size == 0, DKV_EINVAL, "dkv_adjust_logits: misaligned logits");
  DKV_REQUIRE(p->logits_row >= p->vocab && p->out_row >= p->vocab, DKV_ESHAPE, "dkv_adjust_logits: rows overlap");
  LogitsArgs a{};
  a.p = *p;
  a.chunk = chunk_of(*p);
  a.chunks = chunks_of(*p, a.chunk);
  if (p->pick && a.chunks > 1) {
    const size_t need = (size_t)p->rows * a.chunks * sizeof(uint64_t);
    DKV_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0, DKV_EINVAL, "dkv_adjust_logits: null or misaligned workspace");
    DKV_REQUIRE(need <= workspace_bytes, DKV_EWORKSPACE, "dkv_adjust_logits: workspace %zu < %zu bytes", workspace_bytes, need);
    a.partial = (uint64_t*)workspace;
  }
  hipStream_t st = dkv::as_stream(stream);
  if (p->dtype == DKV_F32) launch_type<float>(a, st);
  else if (p->dtype == DKV_F16) launch_type<half_t>(a, st);
  else launch_type<dkv_bf16>(a, st);
  if (a.partial)
    hipLaunchKernelGGL(pick_kernel, dim3((p->rows + 3) / 4), dim3(256), 0, st, a.partial, a.chunks, p->rows, p->pick);
  return dkv::check_launch("dkv_adjust_logits");
}
