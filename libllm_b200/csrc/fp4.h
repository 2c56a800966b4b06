// Arguments of the kernels in fp4.cu, one struct a call (plain C: the host library and the Python binding fill them alike).
#pragma once

// x [rows, cols] (dtype 0: 32-bit, 1: bfloat16; row stride ldx in elements) -> codes, scales, row_scale as fp4.cu lays them out; format 0:
// nvfp4, 1: mxfp4.
struct Fp4QuantizeCall {
  long long dtype;
  const void *x;
  long long ldx;
  void *codes, *scales;
  float *row_scale;
  long long rows, cols, format;
  void *stream;
};

// The other way: out [rows, cols] of `dtype`, row stride ldo in elements.
struct Fp4DequantizeCall {
  const void *codes, *scales;
  const float *row_scale;
  long long dtype;
  void *out;
  long long ldo, rows, cols, format;
  void *stream;
};

// out [M, N] of out_dtype (row stride ldo) = x [M, K] w [N, K]^T, both in `format`.  weights_first != 0: w was complete before the kernel in front of this
// one in the stream could start (a matrix that is held), and may be read while that one still runs.  A wait inside the kernel that runs out of
// time leaves a code in *status.
struct Fp4GemmCall {
  const void *x_codes, *x_scales;
  const float *x_row;
  const void *w_codes, *w_scales;
  const float *w_row;
  long long out_dtype;
  void *out;
  long long ldo, M, N, K, format, weights_first;
  int *status;
  void *stream;
};
