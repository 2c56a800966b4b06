// What a request asks of its logits before a token is drawn, in one pass over the rows:
//   1. penalties for what its sequence holds: a token that occurs at all has its logit divided by `repetition` where that is positive,
//      multiplied elsewhere; one that was drawn n > 0 times loses frequency n + presence;
//   2. a bias per token is added;
//   3. a token whose bit in `allowed` is not set gets minus infinity.
// A sequence's tokens are its history: [places, longest] ids in the order of their positions, id for a token that was drawn, ~id for one that the prompt brought;
// ids outside the vocabulary count for nothing.  No table of counts is kept: a CTA owns a slice of a row's vocabulary, counts the
// history's ids of that slice in shared memory, and passes over its logits once.  Reading a history of thousands of ids once per slice
// (from L2) costs less than 4 bytes of counts per token of the vocabulary from memory, and there is nothing to reset or to keep right.
#include "common.cuh"
#include "logits.h"

LLM_DEFINE_LAST_ERROR(llm_logits_last_error)

namespace {

constexpr int MOST_SLICE = 4096;               // tokens of a CTA, at most: 16 KB of counters
constexpr unsigned SEEN = 0x80000000u;         // a counter's highest bit: the token occurs; the others: how often it was drawn

struct Rows {                                  // one number per row, or one for all
  const float *p;
  float v;
  __device__ __forceinline__ float at(long long b) const { return p ? p[b] : v; }
};

struct Adjust {
  const float *logits;
  float *out;
  long long ld, ldo;
  int V, slice;
  const int *history, *slots, *lengths;        // history null: no penalties; slots null: row b's place is b
  long long ldh;
  int places, longest;
  Rows repetition, presence, frequency;
  const float *bias;                           // null: none; ld_bias 0: one row for all
  long long ld_bias;
  const unsigned *allowed;                     // null: all; bit v % 32 of word v / 32
  long long ld_allowed;
};

// A row's penalties.  A division by `rep` is a product with 1 / rep in 64 bits, narrowed once: two roundings of 2^-53, where the quotient of two numbers of 24 bits lies
// 2^-49 of itself or more from every border between two others, so that what comes out is the nearest number of 32 bits as the division's would be.
// (With a product in 32 bits up to a sixth of the quotients were the next number to it, 64 rows of 128,256 took 14.9 us for 15.2; with the division itself, its
// registers and instructions, 16.6.)
struct Penalty {
  double inv;
  float rep, pres, freq;
  __device__ __forceinline__ Penalty(float r, float p, float f) : inv(1.0 / (double)r), rep(r), pres(p), freq(f) {}
};
__device__ __forceinline__ float adjusted(float x, unsigned c, const Penalty &p) {
  const float said = x > 0.f ? (float)((double)x * p.inv) : x * p.rep;
  const unsigned n = c & ~SEEN;
  x = c ? said : x;
  return n ? x - (p.freq * (float)n + p.pres) : x;
}

// The slice's ids among h[0 .. len).
__device__ __forceinline__ void count(unsigned *counts, int id, int v0, int n) {
  const unsigned at = (unsigned)(id < 0 ? ~id : id) - (unsigned)v0;
  if (at < (unsigned)n) {
    if (id >= 0) atomicAdd(&counts[at], 1u);             // any count but 0 says that the token occurs
    else if (!(counts[at] & SEEN)) atomicOr(&counts[at], SEEN);
  }
}

// AT threads to a slice.  Its logits are on their way while its history is counted: into shared memory where there are 256 threads (held in registers, 39
// for 32, they left six CTAs to an SM: 64 rows of 128,256 with everything 19.4 us for 16.6, with a mask alone 14.1 for 11.5, 5.9 TB/s, cold
// caches), into registers where there are 1,024 and time is what a load takes (7 rows of 50,257 with 5,000 ids 4.5 us for 5.0).
template <bool VEC, int AT>
__global__ void __launch_bounds__(AT, AT == 1024 ? 2 : VEC ? 7 : 6) adjust_kernel(Adjust a) {
  constexpr bool HELD = AT == 1024;
  extern __shared__ __align__(16) unsigned counts[];                     // [slice] with a history; then [slice] logits if not HELD
  float *ahead = reinterpret_cast<float *>(counts) + (a.history ? a.slice : 0);
  grid_dependents_launch();
  const long long b = blockIdx.y;
  const int v0 = blockIdx.x * a.slice, n = min(a.slice, a.V - v0);
  if (a.history)
    for (int i = threadIdx.x * 4; i < n; i += AT * 4) *reinterpret_cast<uint4 *>(counts + i) = make_uint4(0, 0, 0, 0);
  grid_dependency_wait();
  const float *x = a.logits + b * a.ld + v0, *bias = a.bias ? a.bias + b * a.ld_bias + v0 : nullptr;
  const unsigned *allowed = a.allowed ? a.allowed + b * a.ld_allowed : nullptr;
  float *out = a.out + b * a.ldo + v0;
  const int place = !a.history ? -1 : a.slots ? a.slots[b] : (int)b;
  const int said = a.history ? a.lengths[b] : 0;
  constexpr int AHEAD = MOST_SLICE / AT / 4;
  const unsigned ahead_at = (unsigned)__cvta_generic_to_shared(ahead);
  unsigned words[VEC ? AHEAD : 1];             // the mask's, in time: 12.6 -> 11.5 us for a mask alone
  float4 held[HELD ? AHEAD : 1];
  if (VEC) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int i = (threadIdx.x + j * AT) * 4;
      if (HELD && i + 4 <= n) held[HELD ? j : 0] = *reinterpret_cast<const float4 *>(x + i);
      if (!HELD && i + 4 <= n) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ahead_at + i * 4), "l"(x + i) : "memory");
      if (allowed && i < n) words[j] = allowed[(v0 + i) >> 5];
    }
  } else if (HELD) {
    float *v = reinterpret_cast<float *>(held);
#pragma unroll
    for (int j = 0; j < 4 * AHEAD; ++j) {
      const int i = threadIdx.x + j * AT;
      if (i < n) v[HELD ? j : 0] = x[i];
    }
  } else {
    for (int i = threadIdx.x; i < n; i += AT) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(ahead_at + i * 4), "l"(x + i) : "memory");
  }
  const Penalty pen = a.history ? Penalty(a.repetition.at(b), a.presence.at(b), a.frequency.at(b)) : Penalty(1.f, 0.f, 0.f);
  if (a.history) {
    const int len = place >= 0 && place < a.places ? min(max(said, 0), a.longest) : 0;
    const int *h = a.history + (long long)place * a.ldh;
    __syncthreads();
    int done = 0;
    if (((uintptr_t)h & 15) == 0) {
      done = len & ~3;
      for (int i = threadIdx.x * 4; i < done; i += AT * 8) {         // two loads on their way
        const int4 p = *reinterpret_cast<const int4 *>(h + i);
        const bool two = i + AT * 4 < done;
        const int4 q = two ? *reinterpret_cast<const int4 *>(h + i + AT * 4) : p;
        count(counts, p.x, v0, n);
        count(counts, p.y, v0, n);
        count(counts, p.z, v0, n);
        count(counts, p.w, v0, n);
        if (two) {
          count(counts, q.x, v0, n);
          count(counts, q.y, v0, n);
          count(counts, q.z, v0, n);
          count(counts, q.w, v0, n);
        }
      }
    }
#pragma unroll 4
    for (int i = done + threadIdx.x; i < len; i += AT) count(counts, h[i], v0, n);
    __syncthreads();
  }
  auto one = [&](int i, float v) {
    if (a.history) v = adjusted(v, counts[i], pen);
    if (bias) v += bias[i];
    if (allowed && !(allowed[(v0 + i) >> 5] >> ((v0 + i) & 31) & 1)) v = -INFINITY;
    return v;
  };
  if (!HELD) asm volatile("cp.async.wait_all;" ::: "memory");            // a thread reads what it copied itself
  if (VEC) {                                   // slices are multiples of 32 tokens
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int i = (threadIdx.x + j * AT) * 4;
      if (i + 4 > n) break;
      float4 v = HELD ? held[HELD ? j : 0] : *reinterpret_cast<const float4 *>(ahead + i);
      if (a.history) {
        const uint4 c = *reinterpret_cast<const uint4 *>(counts + i);
        if (c.x | c.y | c.z | c.w) {
          v.x = adjusted(v.x, c.x, pen);
          v.y = adjusted(v.y, c.y, pen);
          v.z = adjusted(v.z, c.z, pen);
          v.w = adjusted(v.w, c.w, pen);
        }
      }
      if (bias) {
        const float4 w = *reinterpret_cast<const float4 *>(bias + i);
        v.x += w.x;
        v.y += w.y;
        v.z += w.z;
        v.w += w.w;
      }
      if (allowed) {
        const unsigned bits = words[j] >> ((v0 + i) & 31);
        if (!(bits & 1)) v.x = -INFINITY;
        if (!(bits & 2)) v.y = -INFINITY;
        if (!(bits & 4)) v.z = -INFINITY;
        if (!(bits & 8)) v.w = -INFINITY;
      }
      *reinterpret_cast<float4 *>(out + i) = v;
    }
    const int i = (n & ~3) + threadIdx.x;
    if (i < n) out[i] = one(i, x[i]);
  } else if (HELD) {
    const float *v = reinterpret_cast<const float *>(held);
#pragma unroll
    for (int j = 0; j < 4 * AHEAD; ++j) {
      const int i = threadIdx.x + j * AT;
      if (i < n) out[i] = one(i, v[HELD ? j : 0]);
    }
  } else {
#pragma unroll 2
    for (int i = threadIdx.x; i < n; i += 2 * AT) {        // two at once: nothing is read ahead of a store
      const int second = i + AT < n ? i + AT : i;
      const float v = one(i, ahead[i]), w = one(second, ahead[second]);
      out[i] = v;
      if (second != i) out[second] = w;
    }
  }
}

// A step's tokens into their sequences' histories [places, longest], at their positions: a token that the last step drew (fed_rows[t] >= 0: row
// of fed_tokens) as its id; one that is brought as ~id, unless the sequence has this very token there already: then it was drawn before.
__global__ void __launch_bounds__(256) history_place_kernel(const int *tokens, const int *fed_tokens, const int *fed_rows, const int *tok_seq,
                                                            const int *tok_pos, const int *seq_slot, int T, int *history, int places, int longest) {
  grid_dependents_launch();
  grid_dependency_wait();
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= T) return;
  const int place = seq_slot[tok_seq[t]], pos = tok_pos[t], fed = fed_rows ? fed_rows[t] : -1;
  if (place < 0 || place >= places || pos < 0 || pos >= longest) return;
  int *at = history + (long long)place * longest + pos;
  if (fed >= 0) *at = fed_tokens[fed];
  else if (*at != tokens[t]) *at = ~tokens[t];
}
// Drawn tokens where they will stand: row r's at drawn_pos[r] of place row_slot[r]; a position of -1: nowhere.
__global__ void __launch_bounds__(256) history_drawn_kernel(const int *drawn, const int *row_slot, const int *drawn_pos, int n, int *history, int places,
                                                            int longest) {
  grid_dependents_launch();
  grid_dependency_wait();
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= n) return;
  const int place = row_slot[r], pos = drawn_pos[r];
  if (place >= 0 && place < places && pos >= 0 && pos < longest) history[(long long)place * longest + pos] = drawn[r];
}

}  // namespace

LLM_EXPORT int llm_history_place(const int *tokens, const int *fed_tokens, const int *fed_rows, const int *tok_seq, const int *tok_pos,
                                 const int *seq_slot, int T, int *history, int places, int longest, cudaStream_t stream) {
  if (T <= 0) return LLM_OK;
  LLM_REQUIRE(!fed_rows || fed_tokens, "history_place: rows of fed tokens without the tokens");
  LLM_CHECK_CUDA(llm_launch(history_place_kernel, dim3((T + 255) / 256), dim3(256), 0, stream, tokens, fed_tokens, fed_rows, tok_seq, tok_pos, seq_slot, T,
                            history, places, longest), "history_place launch");
  return LLM_OK;
}

LLM_EXPORT int llm_history_drawn(const int *drawn, const int *row_slot, const int *drawn_pos, int n, int *history, int places, int longest,
                                 cudaStream_t stream) {
  if (n <= 0) return LLM_OK;
  LLM_CHECK_CUDA(llm_launch(history_drawn_kernel, dim3((n + 255) / 256), dim3(256), 0, stream, drawn, row_slot, drawn_pos, n, history, places, longest),
                 "history_drawn launch");
  return LLM_OK;
}

LLM_EXPORT int llm_adjust_logits(const AdjustLogitsCall *call) {
  const AdjustLogitsCall &c = *call;
  LLM_REQUIRE(c.B >= 0 && c.V >= 0 && c.V <= (1 << 30), "adjust_logits: bad sizes %lld x %lld", c.B, c.V);
  if (c.B == 0 || c.V == 0) return LLM_OK;
  LLM_REQUIRE(c.B <= 65535, "adjust_logits: %lld rows, at most 65535 are taken", c.B);
  LLM_REQUIRE(!c.history || c.lengths, "adjust_logits: a history needs its rows' lengths");
  LLM_REQUIRE(!c.history || (c.places > 0 && c.longest > 0 && c.places < (1ll << 31) && c.longest < (1ll << 31)),
              "adjust_logits: a history of %lld places of %lld", c.places, c.longest);
  LLM_REQUIRE(!c.history || c.slots || c.B <= c.places, "adjust_logits: %lld rows, the history has %lld places", c.B, c.places);
  Adjust a{c.logits, c.out, c.ld, c.ldo, (int)c.V, 0, c.history, c.slots, c.lengths, c.ldh, (int)c.places, (int)c.longest,
           {c.repetition, (float)c.repetition_all}, {c.presence, (float)c.presence_all}, {c.frequency, (float)c.frequency_all}, c.bias, c.ld_bias,
           c.allowed, c.ld_allowed};
  // Slices as large as still make four CTAs of 256 threads to an SM; where there are more than six, of one size each: 128,256 tokens make 32 slices of
  // 4,032, of which seven fit an SM and not six (64 rows 19.3 -> 17.3 us; 16 rows of 151,936, 4.1 to an SM, 5.9 -> 6.4: a nearly empty last one is
  // less).  Few rows with long histories: CTAs of 1,024 threads, two to an SM, read a history in a quarter of the rounds (8 rows x 128,256, 2,048 ids
  // 4.6 -> 4.0 us, 16,384 12.9 -> 7.0; 1 row, 2,048 ids 2.7 -> 3.0, 32,768 13.1 -> 6.8).
  int slice = MOST_SLICE, wide = MOST_SLICE;
  while (slice > 1024 && (c.V + slice - 1) / slice * c.B < 4ll * sm_count()) slice /= 2;
  while (wide > 1024 && (c.V + wide / 2 - 1) / (wide / 2) * c.B <= 2ll * sm_count()) wide /= 2;
  const bool many = c.history && c.longest * c.B >= 8192 && (c.V + wide - 1) / wide * c.B <= 2ll * sm_count();
  if (many) slice = wide;
  const long long slices = (c.V + slice - 1) / slice;
  if (slices * c.B > 6ll * sm_count()) slice = (int)(((c.V + slices - 1) / slices + 31) / 32 * 32);
  a.slice = slice;
  const bool vec = ((uintptr_t)c.logits | (uintptr_t)c.out | (uintptr_t)c.bias) % 16 == 0 && (c.ld | c.ldo | (c.bias ? c.ld_bias : 0)) % 4 == 0;
  const dim3 grid((unsigned)((c.V + slice - 1) / slice), (unsigned)c.B);
  const size_t smem = (size_t)slice * sizeof(unsigned) * ((c.history ? 1 : 0) + (many ? 0 : 1));
  const cudaStream_t stream = (cudaStream_t)c.stream;
  auto kernel = vec ? (many ? adjust_kernel<true, 1024> : adjust_kernel<true, 256>) : (many ? adjust_kernel<false, 1024> : adjust_kernel<false, 256>);
  LLM_CHECK_CUDA(llm_launch(kernel, grid, dim3(many ? 1024 : 256), smem, stream, a), "adjust_logits launch");
  return LLM_OK;
}
