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

LLM_DEFINE_LAST_ERROR(llm_logits_last_error)

namespace {

constexpr int AT = 512;                        // threads of a CTA
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

__device__ __forceinline__ float adjusted(float x, unsigned c, float rep, float pres, float freq) {
  if (c == 0) return x;
  x = x > 0.f ? x / rep : x * rep;
  const unsigned n = c & ~SEEN;
  return n ? x - (freq * (float)n + pres) : x;
}

template <bool VEC>
__global__ void __launch_bounds__(AT) adjust_kernel(Adjust a) {
  extern __shared__ unsigned counts[];
  grid_dependents_launch();
  const long long b = blockIdx.y;
  const int v0 = blockIdx.x * a.slice, n = min(a.slice, a.V - v0);
  if (a.history)
    for (int i = threadIdx.x; i < n; i += AT) counts[i] = 0;
  grid_dependency_wait();
  float rep = 1.f, pres = 0.f, freq = 0.f;
  if (a.history) {
    rep = a.repetition.at(b);
    pres = a.presence.at(b);
    freq = a.frequency.at(b);
    __syncthreads();
    const int place = a.slots ? a.slots[b] : (int)b;
    const int len = place >= 0 && place < a.places ? min(max(a.lengths[b], 0), a.longest) : 0;
    const int *h = a.history + (long long)place * a.ldh;
    for (int i = threadIdx.x; i < len; i += AT) {
      const int id = h[i];
      const unsigned at = (unsigned)(id < 0 ? ~id : id) - (unsigned)v0;
      if (at < (unsigned)n) {
        if (id >= 0) atomicAdd(&counts[at], 1u);       // below, any count but 0 says that the token occurs
        else if (!(counts[at] & SEEN)) atomicOr(&counts[at], SEEN);
      }
    }
    __syncthreads();
  }
  const float *x = a.logits + b * a.ld + v0, *bias = a.bias ? a.bias + b * a.ld_bias + v0 : nullptr;
  const unsigned *allowed = a.allowed ? a.allowed + b * a.ld_allowed : nullptr;
  float *out = a.out + b * a.ldo + v0;
  auto one = [&](int i, float v) {
    if (a.history) v = adjusted(v, counts[i], rep, pres, freq);
    if (bias) v += bias[i];
    if (allowed && !(allowed[(v0 + i) >> 5] >> ((v0 + i) & 31) & 1)) v = -INFINITY;
    return v;
  };
  if (VEC) {                                   // slices are multiples of 32 tokens
    for (int i = threadIdx.x * 4; i + 4 <= n; i += AT * 4) {
      float4 v = *reinterpret_cast<const float4 *>(x + i);
      if (a.history) {
        const uint4 c = *reinterpret_cast<const uint4 *>(counts + i);
        v.x = adjusted(v.x, c.x, rep, pres, freq);
        v.y = adjusted(v.y, c.y, rep, pres, freq);
        v.z = adjusted(v.z, c.z, rep, pres, freq);
        v.w = adjusted(v.w, c.w, rep, pres, freq);
      }
      if (bias) {
        const float4 w = *reinterpret_cast<const float4 *>(bias + i);
        v.x += w.x;
        v.y += w.y;
        v.z += w.z;
        v.w += w.w;
      }
      if (allowed) {
        const unsigned bits = allowed[(v0 + i) >> 5] >> ((v0 + i) & 31);
        if (!(bits & 1)) v.x = -INFINITY;
        if (!(bits & 2)) v.y = -INFINITY;
        if (!(bits & 4)) v.z = -INFINITY;
        if (!(bits & 8)) v.w = -INFINITY;
      }
      *reinterpret_cast<float4 *>(out + i) = v;
    }
    const int i = (n & ~3) + threadIdx.x;
    if (i < n) out[i] = one(i, x[i]);
  } else {
    for (int i = threadIdx.x; i < n; i += AT) out[i] = one(i, x[i]);
  }
}

}  // namespace

// out [B, V] = logits [B, V] with the rows' penalties, bias and mask applied; out may be logits.  Row strides in elements (words for
// `allowed`); a row stride of 0 for bias or allowed: one row for all.  repetition, presence, frequency: [B], or null and the number beside.
LLM_EXPORT int llm_adjust_logits(const float *logits, long long ld, float *out, long long ldo, int B, int V, const int *history, long long ldh, int places,
                                 int longest, const int *slots, const int *lengths, const float *repetition, float repetition_all, const float *presence,
                                 float presence_all, const float *frequency, float frequency_all, const float *bias, long long ld_bias,
                                 const int *allowed, long long ld_allowed, cudaStream_t stream) {
  LLM_REQUIRE(B >= 0 && V >= 0, "adjust_logits: bad sizes %d x %d", B, V);
  if (B == 0 || V == 0) return LLM_OK;
  LLM_REQUIRE(B <= 65535, "adjust_logits: %d rows, at most 65535 are taken", B);
  LLM_REQUIRE(!history || lengths, "adjust_logits: a history needs its rows' lengths");
  LLM_REQUIRE(!history || slots || B <= places, "adjust_logits: %d rows, the history has %d", B, places);
  Adjust a{logits, out, ld, ldo, V, 0, history, slots, lengths, ldh, places, longest, {repetition, repetition_all}, {presence, presence_all},
           {frequency, frequency_all}, bias, ld_bias, (const unsigned *)allowed, ld_allowed};
  int slice = 8192;
  while (slice > 1024 && (long long)((V + slice - 1) / slice) * B < 4ll * sm_count()) slice /= 2;
  a.slice = slice;
  const bool vec = ((uintptr_t)logits | (uintptr_t)out | (uintptr_t)bias) % 16 == 0 && (ld | ldo | (bias ? ld_bias : 0)) % 4 == 0;
  const dim3 grid((unsigned)((V + slice - 1) / slice), (unsigned)B);
  const size_t smem = history ? (size_t)slice * sizeof(unsigned) : 0;
  LLM_CHECK_CUDA(vec ? llm_launch(adjust_kernel<true>, grid, dim3(AT), smem, stream, a) : llm_launch(adjust_kernel<false>, grid, dim3(AT), smem, stream, a),
                 "adjust_logits launch");
  return LLM_OK;
}
