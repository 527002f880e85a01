// The logits of replies under penalties for repeated tokens, biases and a grammar's masks, and the token picked
// (include/dimmerkv.h states the arithmetic).
//
// One pass over the logits: a workgroup takes a stretch of a row's vocabulary.  It loads the stretch into registers, counts
// meanwhile the history's tokens that fall into it in LDS (integer atomics that return nothing: the order does not matter and
// nothing waits for them), and writes the stretch once.  Every float32 operation is rounded on its own, in the stated order,
// so equal inputs stay equal and ties are ties.
// Measured: 128 replies of 128,256 bfloat16 logits 38 us with histories of up to 16K tokens, biases and masks, 22 us
// without any (66 MB: 13 us at a copy's rate): reading the history once for every stretch and dividing the logits it
// names are the difference.  Vector instructions issue in 78 % of the busy SIMDs' cycles; a wave waits for memory and LDS
// half of its time.  Stretches of 8,192 and 32,768 tokens cost 50 and 54 us, a list of the counted tokens worked off by full
// waves 43 to 56.
#include <math.h>

#include "dkv_device.h"
#include "dkv_fp4.h"
#include "dkv_stretch.h"
#include "dkv_host.h"

namespace {

using dkv::TokenRange;
using dkv::tokens_of_stretch;

constexpr int kThreads = 1024;

struct LogitsArgs {
  dkv_logits_args_t p;
  uint64_t* partial;  // [rows][chunks] keys of the best token of each stretch; null when there is one stretch
  int chunks;         // stretches of a row
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
DKV_DEVICE void set_logit(dkv_bf16& y, float x) {
  const __bf16 z = (__bf16)x;
  __builtin_memcpy(&y.bits, &z, 2);
}

// How often the stretch's tokens occur.  A token takes 16 bits where the history is short enough for 15 of count (the
// highest bit: the prompt holds it), 32 otherwise.
template <bool SHORT>
struct Counts {
  static constexpr uint32_t kSeen = SHORT ? 0x8000u : 0x80000000u;
  static DKV_DEVICE uint32_t get(const uint32_t* counts, int at) {
    return SHORT ? (counts[at >> 1] >> (16 * (at & 1))) & 0xffffu : counts[at];
  }
  static DKV_DEVICE void add(uint32_t* counts, int at, bool reply) {
    uint32_t* word = counts + (SHORT ? at >> 1 : at);
    const int shift = SHORT ? 16 * (at & 1) : 0;
    if (reply) atomicAdd(word, 1u << shift);
    else atomicOr(word, kSeen << shift);
  }
};

// A stretch is kThreads * N lines of 16 bytes.  LDS: counts, and a bit a token for those with a bias.
template <typename T, int N, bool SHORT>
struct Stretch {
  static constexpr int V = 16 / sizeof(T), kTokens = kThreads * N * V;
  static constexpr int kCountWords = SHORT ? kTokens / 2 : kTokens, kBitWords = kTokens / 32;
  static constexpr int kBytes = 4 * (kCountWords + kBitWords);
};

template <typename T, typename ID, int N, bool SHORT>
__global__ __launch_bounds__(kThreads, 8) void adjust_logits_kernel(LogitsArgs a) {
#pragma clang fp contract(off)
  using S = Stretch<T, N, SHORT>;
  using Count = Counts<SHORT>;
  constexpr int V = S::V, kTokens = S::kTokens;
  extern __shared__ uint32_t lds[];
  uint32_t* counts = lds;
  uint32_t* biased = lds + S::kCountWords;
  __shared__ uint64_t bests[kThreads / 64];
  const dkv_logits_args_t& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, vocab = p.vocab;
  // Eight rows at a time, so that a row's stretches run on one die and its second cache holds the history for all of them
  // (128 replies 37.7 us, 39.0 with the stretches on one die each).
  int stretch = blockIdx.x, row = 0;
  if (gridDim.y > 1) {  // (a single row does without the divisions)
    const uint32_t id_of = blockIdx.x + blockIdx.y * gridDim.x, eight = id_of / (8 * gridDim.x), in_eight = id_of - eight * 8 * gridDim.x;
    const uint32_t beside = min(8u, gridDim.y - 8 * eight);
    stretch = (int)(in_eight / beside);
    row = (int)(8 * eight + in_eight - stretch * beside);
  }
  const T* logits = (const T*)p.logits + row * p.logits_row;
  T* out = (T*)p.out + row * p.out_row;
  // Elements are numbered from the 16-byte line the row begins in; a row of any alignment is read in whole lines, and
  // written so if its out row begins alike.
  const int shift = (int)((uintptr_t)logits / sizeof(T) % V);
  const bool alike = shift == (int)((uintptr_t)out / sizeof(T) % V);
  const long first = (long)stretch * kTokens - shift;  // token of the stretch's element 0

  uint4 lines[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const long token = first + (k * kThreads + tid) * V;
    if (token >= 0 && token + V <= vocab) lines[k] = *(const uint4*)(logits + token);
  }
  // the history eight tokens a thread at a time, the first of them on their way while LDS is cleared
  const int length = p.tokens ? min(max(p.lengths[row], 0), p.history) : 0, reply = p.tokens && p.reply ? max(p.reply[row], 0) : 0;
  const ID* tokens = (const ID*)p.tokens + row * p.tokens_row;
  constexpr int kBatch = 8;
  ID id[kBatch];
  const auto fetch = [&](int j0) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int j = j0 + k * kThreads + tid;
      id[k] = j < length ? tokens[j] : (ID)-1;
    }
  };
  fetch(0);
  for (int x = tid * 4; x < S::kCountWords + (p.biases ? S::kBitWords : 0); x += kThreads * 4) *(uint4*)(lds + x) = make_uint4(0, 0, 0, 0);
  __syncthreads();
  // (in 32 bits, an id's upper half being 0: of 64, the comparisons of every id with every stretch would show)
  const TokenRange own = tokens_of_stretch((int)first, kTokens, vocab);
  for (int j0 = 0; j0 < length; j0 += kBatch * kThreads) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const uint32_t from = (uint32_t)id[k] - own.lowest;
      if ((sizeof(ID) == 4 || (uint32_t)((uint64_t)id[k] >> 32) == 0) && from < own.count)
        Count::add(counts, (int)(from + (uint32_t)(own.lowest - first)), j0 + k * kThreads + tid >= reply);
    }
    fetch(j0 + kBatch * kThreads);
  }
  const int bias0 = p.biases ? max(p.bias_cu[row], 0) : 0, bias1 = p.biases ? min(p.bias_cu[row + 1], p.biases) : 0;
  for (int j = bias0 + tid; j < bias1; j += kThreads) {
    const long token = p.bias_ids[j], at = token - first;
    if (token < 0 || token >= vocab || at < 0 || at >= kTokens) continue;
    atomicOr(biased + (at >> 5), 1u << (at & 31));
  }
  __syncthreads();

  const uint32_t* allowed = nullptr;
  bool limited = false;  // (a mask past the last one allows nothing)
  if (p.allowed) {
    const int mask = p.allowed_row ? p.allowed_row[row] : row;
    limited = mask >= 0;
    if (limited && mask < p.masks) allowed = (const uint32_t*)p.allowed + (long)mask * p.words;
  }
  const auto may = [&](int token) { return !limited || (allowed && ((allowed[token >> 5] >> (token & 31)) & 1)); };
  uint64_t best = 0;
  float highest = -INFINITY;  // of best; above it all once that is a NaN
  const auto seen = [&](float x, int token) {
    best = best_of(best, (uint64_t)order_key(x) << 32 | (uint32_t)~token);
    highest = x != x ? INFINITY : fmaxf(highest, x);
  };
  const float repetition = p.repetition ? p.repetition[row] : 1.0f, presence = p.presence ? p.presence[row] : 0.0f,
              frequency = p.frequency ? p.frequency[row] : 0.0f;
  const auto penalized = [&](float x, uint32_t count) {
    if (count) {
      x = x > 0.0f ? x / repetition : x * repetition;
      const uint32_t mentions = count & (Count::kSeen - 1);
      if (mentions) {
        const float less = frequency * (float)mentions;
        x = x - (less + presence);
      }
    }
    return x;
  };
  // Tokens with a bias keep their logit at first and are taken from there at the end (out may be the logits).
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int at = (k * kThreads + tid) * V;
    const long token = first + at;
    if (token >= vocab) break;
    const uint32_t with_bias = p.biases ? biased[at >> 5] >> (at & 31) : 0;
    if (token >= 0 && token + V <= vocab) {
      uint32_t held[SHORT ? V / 2 : V], any = 0, bits = ~0u;
#pragma unroll
      for (int v = 0; v < (SHORT ? V / 2 : V); ++v) any |= held[v] = counts[(SHORT ? at / 2 : at) + v];
      T x[V];
      float z[V];
      __builtin_memcpy(x, &lines[k], 16);
      if (limited) {
        const int word = (int)token >> 5, in = (int)token & 31;
        bits = allowed ? allowed[word] >> in : 0;
        if (allowed && in + V > 32) bits |= allowed[word + 1] << (32 - in);
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (!(((bits | with_bias) >> v) & 1)) set_logit(x[v], -INFINITY);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) z[v] = logit_value(x[v]);
      if (any) {
        const uint32_t free = bits & ~with_bias;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const uint32_t count = SHORT ? (held[v >> 1] >> (16 * (v & 1))) & 0xffffu : held[v];
          if (count && (free >> v) & 1) {
            z[v] = penalized(z[v], count);
            set_logit(x[v], z[v]);
          }
        }
      }
      if (with_bias) {
#pragma unroll
        for (int v = 0; v < V; ++v)
          if ((with_bias >> v) & 1) z[v] = -INFINITY;
      }
      float top = -INFINITY;  // of the line, whose tokens come after those of best: an equal one does not matter
      bool odd = false;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        top = fmaxf(top, z[v]);
        odd = odd || z[v] != z[v];
      }
      if (odd || top > highest) {
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (!(z[v] < highest)) seen(z[v], (int)token + v);
      }
      if (alike) {
        __builtin_memcpy(__builtin_assume_aligned(out + token, 16), x, 16);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) out[token + v] = x[v];
      }
    } else {
      for (int v = 0; v < V; ++v) {
        const long t = token + v;
        if (t < 0 || t >= vocab) continue;
        if ((with_bias >> v) & 1) {
          out[t] = logits[t];
          continue;
        }
        const float z = may((int)t) ? penalized(logit_value(logits[t]), Count::get(counts, at + v)) : -INFINITY;
        seen(z, (int)t);
        set_logit(out[t], z);
      }
    }
  }
  if (bias1 > bias0) {
    __syncthreads();
    for (int j = bias0 + tid; j < bias1; j += kThreads) {
      const long token = p.bias_ids[j], at = token - first;
      if (token < 0 || token >= vocab || at < 0 || at >= kTokens) continue;
      float x = penalized(logit_value(out[token]), Count::get(counts, (int)at));
      x = x + p.bias_values[j];
      if (!may((int)token)) x = -INFINITY;
      seen(x, (int)token);
      set_logit(out[token], x);
    }
  }
  if (!p.pick) return;
  best = wave_best(best);
  if (lane == 0) bests[tid >> 6] = best;
  __syncthreads();
  if (tid < 64) {
    best = wave_best(tid < kThreads / 64 ? bests[tid] : 0);
    if (!a.partial) {
      if (tid == 0) p.pick[row] = picked(best);
      return;
    }
    uint64_t* partial = a.partial + (long)row * a.chunks;
    if (!p.arrivals) {
      if (tid == 0) partial[stretch] = best;
      return;
    }
    bool last = false;
    if (tid == 0) {
      leave(partial + stretch, best);
      left_behind();
      last = last_of(p.arrivals + row, a.chunks);
    }
    if (!__any(last)) return;
    best = 0;
    for (int c = tid; c < a.chunks; c += 64) best = best_of(best, pick_up(partial + c));
    best = wave_best(best);
    if (tid == 0) p.pick[row] = picked(best);
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

// Stretches of 16,384 tokens (two or four lines a thread) where that makes two workgroups a CU, as each of them reads the
// whole history; one line a thread otherwise, for more workgroups.
struct Plan {
  bool counts16;
  int lines, chunks;
};

Plan plan_of(const dkv_logits_args_t& p) {
  Plan plan;
  const int line = p.dtype == DKV_F32 ? 4 : 8, most = 16 / line;  // elements of a line; lines of 16,384
  const auto chunks = [&](int lines) { return dkv::stretches_of_row(p.vocab, line, kThreads * lines * line); };
  plan.counts16 = !p.tokens || p.history < 0x8000;
  plan.lines = plan.counts16 && (long)chunks(most) * p.rows >= 512 ? most : 1;
  plan.chunks = chunks(plan.lines);
  return plan;
}

int check_logits(const dkv_logits_args_t* p, const char* what) {
  DKV_REQUIRE(p, DKV_EINVAL, "%s: null arguments", what);
  DKV_REQUIRE(p->dtype == DKV_F32 || p->dtype == DKV_F16 || p->dtype == DKV_BF16, DKV_EINVAL, "%s: dtype %d not supported", what, p->dtype);
  DKV_REQUIRE(p->rows >= 0 && p->rows <= 65535 && p->vocab > 0 && p->vocab <= INT32_MAX - 65536, DKV_ESHAPE,
              "%s: bad shape (rows=%d, at most 65535; vocab=%d)", what, p->rows, p->vocab);
  // (32-bit indexes that run a batch of the history and a workgroup of the biases past their ends)
  DKV_REQUIRE(p->history <= INT32_MAX - 65536 && p->biases <= INT32_MAX - 65536, DKV_ESHAPE, "%s: history=%d or biases=%d pass 2^31 - 2^16",
              what, p->history, p->biases);
  DKV_REQUIRE(p->history >= 0 && p->biases >= 0 && p->masks >= 0, DKV_ESHAPE, "%s: bad shape (history=%d biases=%d masks=%d)",
              what, p->history, p->biases, p->masks);
  DKV_REQUIRE(p->token_bytes == 4 || p->token_bytes == 8 || !p->tokens, DKV_EINVAL, "%s: tokens of %d bytes", what, p->token_bytes);
  DKV_REQUIRE((uintptr_t)p->arrivals % 4 == 0, DKV_EINVAL, "%s: misaligned arrivals", what);
  DKV_REQUIRE(!p->tokens || p->lengths, DKV_EINVAL, "%s: tokens without lengths", what);
  DKV_REQUIRE(!p->biases || (p->bias_ids && p->bias_values && p->bias_cu), DKV_EINVAL, "%s: null bias pointer", what);
  DKV_REQUIRE(!p->allowed || p->words >= ((int64_t)p->vocab + 31) / 32, DKV_ESHAPE, "%s: %d mask words for %d tokens", what, p->words, p->vocab);
  DKV_REQUIRE(!p->allowed || p->allowed_row || p->masks >= p->rows, DKV_ESHAPE, "%s: %d masks for %d rows", what, p->masks, p->rows);
  return DKV_OK;
}

template <typename T, typename ID, int N, bool SHORT>
void launch(const LogitsArgs& a, hipStream_t st) {
  using S = Stretch<T, N, SHORT>;  // (the bits come last: without biases they are not asked for)
  hipLaunchKernelGGL((adjust_logits_kernel<T, ID, N, SHORT>), dim3(a.chunks, a.p.rows), dim3(kThreads),
                     a.p.biases ? S::kBytes : 4 * S::kCountWords, st, a);
}

template <typename T, typename ID>
void launch_plan(const LogitsArgs& a, const Plan& plan, hipStream_t st) {
  if (plan.lines > 1) launch<T, ID, (int)sizeof(T), true>(a, st);
  else if (plan.counts16) launch<T, ID, 1, true>(a, st);
  else launch<T, ID, 1, false>(a, st);
}

template <typename T>
void launch_type(const LogitsArgs& a, const Plan& plan, hipStream_t st) {
  if (a.p.token_bytes == 4) launch_plan<T, int32_t>(a, plan, st);
  else launch_plan<T, int64_t>(a, plan, st);
}

}  // namespace

extern "C" size_t dkv_adjust_logits_workspace_bytes(const dkv_logits_args_t* p) {
  if (check_logits(p, "dkv_adjust_logits_workspace_bytes")) return 0;
  return (size_t)p->rows * plan_of(*p).chunks * sizeof(uint64_t) + 16;
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
  const Plan plan = plan_of(*p);
  a.chunks = plan.chunks;
  if (p->pick && a.chunks > 1) {
    const size_t need = (size_t)p->rows * a.chunks * sizeof(uint64_t);
    DKV_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0, DKV_EINVAL, "dkv_adjust_logits: null or misaligned workspace");
    DKV_REQUIRE(need <= workspace_bytes, DKV_EWORKSPACE, "dkv_adjust_logits: workspace %zu < %zu bytes", workspace_bytes, need);
    a.partial = (uint64_t*)workspace;
  }
  hipStream_t st = dkv::as_stream(stream);
  if (p->dtype == DKV_F32) launch_type<float>(a, plan, st);
  else if (p->dtype == DKV_F16) launch_type<half_t>(a, plan, st);
  else launch_type<dkv_bf16>(a, plan, st);
  if (a.partial && !p->arrivals)
    hipLaunchKernelGGL(pick_kernel, dim3((p->rows + 3) / 4), dim3(256), 0, st, a.partial, a.chunks, p->rows, p->pick);
  return dkv::check_launch("dkv_adjust_logits");
}
