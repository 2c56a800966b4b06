// Arguments of the kernel in logits.cu (plain C: the host library and the Python binding fill them alike).
#pragma once

// out [B, V] = logits [B, V] with the rows' penalties, bias and mask applied; out may be logits.  Row strides in elements (words for
// `allowed`); a row stride of 0 for bias or allowed: one row for all.  history null: no penalties; slots null: row b's place is b.  repetition,
// presence, frequency: [B], or null and the number beside them.
struct AdjustLogitsCall {
  const float *logits;
  long long ld;
  float *out;
  long long ldo, B, V;
  const int *history;
  long long ldh, places, longest;
  const int *slots, *lengths;
  const float *repetition, *presence, *frequency;
  double repetition_all, presence_all, frequency_all;
  const float *bias;
  long long ld_bias;
  const unsigned *allowed;
  long long ld_allowed;
  void *stream;
};
