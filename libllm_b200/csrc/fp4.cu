// Microscaled 4-bit floating point: rows into four bits, back, and the product of two such matrices on the 5th-generation tensor cores.
//
// A value is a code of four bits, one of +-{0, .5, 1, 1.5, 2, 3, 4, 6} (e2m1), times its block's scale of eight bits, times a 32-bit
// scale of its row.  Two formats:
//   nvfp4   blocks of 16 along the row, scales e4m3; the row's scale is the power of two 2^(floor(log2 max|row|) - 10), which puts
//           the scale of its largest block, max|block| / 6 / row scale rounded to e4m3, between 170 and 342 of e4m3's 448; a block that
//           holds anything has a scale of at least 2^-9, e4m3's smallest.
//   mxfp4   blocks of 32, scales 2^(floor(log2 max|block|) - 2) (e8m0), row scale 1; what lies above 6 scales becomes 6.
// A code is the nearest one to value / scale, halves to the even code.  Row scales that are powers of two keep every step but that
// rounding exact.  A row that holds a NaN or an infinity gets the row scale NaN: whatever is made of it is NaN.
//
// Where things lie (a matrix of `rows` x `cols`):
//   codes      [rows, Kp / 2] bytes, Kp = cols rounded up to 32; the lower four bits hold the even element; zeros behind cols;
//   scales     tiles of 128 rows x 4 blocks, 512 bytes each, in the order in which tcgen05.cp takes them to tensor memory: row r, block j
//              at (r % 32) * 16 + (r / 32) * 4 + j; a row tile's tiles one behind the other, up to a multiple of 256 columns
//              (zeros behind cols);
//   row_scale  [rows] 32-bit.
#include "common.cuh"
#include "fp4.h"
#include "tc_common.cuh"
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

LLM_DEFINE_LAST_ERROR(llm_fp4_last_error)

namespace {

enum Fp4Format { NVFP4 = 0, MXFP4 = 1 };

constexpr int UNIT = 16;                       // values that a thread brings into four bits at once: 8 bytes of codes
constexpr int STAGE_K = 256;                   // of the product: 128 bytes of codes, one swizzle row
constexpr int SF_TILE = 512;                   // bytes of scales: 128 rows x 4 blocks

__host__ __device__ constexpr int stage_tiles(int format) { return format == NVFP4 ? 4 : 2; }         // scale tiles in 256 of K
__host__ __device__ inline long long k_stages(long long K) { return (K + STAGE_K - 1) / STAGE_K; }
__host__ __device__ inline long long code_bytes(long long K) { return (K + 31) / 32 * 16; }           // of a row

// ---------------------------------------------------------------- into four bits
// One pass: a row's values stay in registers between its maximum and its codes.  Memory bounds it (128,256 x 2,048 into nvfp4: bfloat16 96 us, 7.0 TB/s; 32-bit
// 170 us, 7.1 TB/s) since a lane has a whole block of nvfp4, so that its scale is worked out once and no lane asks another, and products and
// sums go in pairs; with half as many values to a lane instructions did (131 us).
// UNIT values of a row as they lie in memory, a lane's share: a block of nvfp4, half of one of mxfp4.
template <typename T>
struct Unit;
template <>
struct Unit<__nv_bfloat16> {
  unsigned w[UNIT / 2];
  __device__ __forceinline__ void load(const __nv_bfloat16 *p) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 raw = reinterpret_cast<const uint4 *>(p)[i];
      w[4 * i] = raw.x;
      w[4 * i + 1] = raw.y;
      w[4 * i + 2] = raw.z;
      w[4 * i + 3] = raw.w;
    }
  }
  __device__ __forceinline__ void gather(const __nv_bfloat16 *p, int n) {
#pragma unroll
    for (int i = 0; i < UNIT / 2; ++i) {
      const unsigned lo = 2 * i < n ? __bfloat16_as_ushort(p[2 * i]) : 0, hi = 2 * i + 1 < n ? __bfloat16_as_ushort(p[2 * i + 1]) : 0;
      w[i] = lo | hi << 16;
    }
  }
  __device__ __forceinline__ float2 two(int i) const { return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)); }
  // The largest magnitude's bits, as those of a 32-bit value: as whole numbers they are in the order of the values, and every infinity and NaN is
  // 0x7f800000 or more.
  __device__ __forceinline__ unsigned top() const {
    unsigned m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < UNIT / 2; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    return max(m << 16, m & 0xffff0000u);
  }
};
template <>
struct Unit<float> {
  float4 raw[UNIT / 4];
  __device__ __forceinline__ void load(const float *p) {
#pragma unroll
    for (int i = 0; i < UNIT / 4; ++i) raw[i] = reinterpret_cast<const float4 *>(p)[i];
  }
  __device__ __forceinline__ void gather(const float *p, int n) {
    float v[UNIT];
#pragma unroll
    for (int i = 0; i < UNIT; ++i) v[i] = i < n ? p[i] : 0.f;
#pragma unroll
    for (int i = 0; i < UNIT / 4; ++i) raw[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  }
  __device__ __forceinline__ float2 two(int i) const { return i % 2 ? make_float2(raw[i / 2].z, raw[i / 2].w) : make_float2(raw[i / 2].x, raw[i / 2].y); }
  __device__ __forceinline__ unsigned top() const {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < UNIT / 2; ++i) {
      const float2 v = two(i);
      m = max(m, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
    }
    return m;
  }
};

template <typename T>
__device__ __forceinline__ Unit<T> fetch_unit(const T *row, int u, int K) {
  Unit<T> x;
  if ((u + 1) * UNIT <= K) x.load(row + u * UNIT);
  else if (u * UNIT < K) x.gather(row + u * UNIT, K - u * UNIT);
  else x = Unit<T>{};
  return x;
}

// The units of G neighbouring lanes, u of lane 0 and those behind it, of a row that does not start on 16 bytes: lanes read neighbouring values and
// hand them over in shared memory, 1 KB of a warp's.  (Each lane on its own, value by value: 65,536 x 2,047 142 us for 82, of 32 bits 258 for
// 169.)  All lanes of a warp take part.
template <typename T, int G>
__device__ __forceinline__ Unit<T> fetch_unit_over(const T *row, int u, int K, unsigned *stage_raw) {
  constexpr int PASSES = sizeof(T) / 2, TURN = G / PASSES * UNIT;        // values of a turn
  T *stage = reinterpret_cast<T *>(stage_raw) + threadIdx.x % 32 / G * TURN;
  const int lane = threadIdx.x % G, k0 = (u - lane) * UNIT + lane;
  Unit<T> x;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    T v[TURN / G];
#pragma unroll
    for (int j = 0; j < TURN / G; ++j) {
      const int k = k0 + p * TURN + j * G;
      v[j] = k < K ? row[k] : T(0.f);
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < TURN / G; ++j) stage[j * G + lane] = v[j];
    __syncwarp();
    if (lane / (G / PASSES) == p) x.load(stage + lane % (G / PASSES) * UNIT);
  }
  return x;
}

// Two 32-bit products with a sum, or without, in one instruction.
__device__ __forceinline__ float2 fma_two(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
      "fma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add_two(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul_two(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ unsigned pack_codes(const float2 *v) {      // eight values, the first in the lowest four bits
  unsigned r;
  asm("{\n.reg .b8 a, b, c, d;\n"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      "mov.b32 %0, {a, b, c, d};\n}"
      : "=r"(r) : "f"(v[0].x), "f"(v[0].y), "f"(v[1].x), "f"(v[1].y), "f"(v[2].x), "f"(v[2].y), "f"(v[3].x), "f"(v[3].y));
  return r;
}

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }        // -126 .. 127

// The row's scale of nvfp4, from its largest magnitude's bits: its exponent.
__device__ __forceinline__ int row_exponent(unsigned top) { return top == 0 ? 0 : max((int)(top >> 23) - 137, -126); }

__device__ __forceinline__ float e4m3_value(unsigned byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}
__device__ __forceinline__ float reciprocal(float v) {        // off by 2^-22 of itself at most
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// The scale byte of a block whose largest magnitude has the bits `top`.
//
// nvfp4: largest / row scale / 6 to the nearest e4m3.  Halfway points t have five bits, so the argument of unit_codes() holds here too: 32-bit values
// are divided, and the quotient's rounding does not take them across t; a bfloat16 value (8 bits) and 6 t (7 bits) are equal or 2^-8 of
// themselves apart, so that the product with 1 / 6, rounded to 12 bits, is t exactly where the quotient is and on its side of t elsewhere.
template <typename T, int FORMAT>
__device__ __forceinline__ unsigned scale_byte(unsigned top, float row_up) {
  if (FORMAT == MXFP4) return top == 0 ? 0u : (unsigned)max((int)(top >> 23) - 2, 0);       // 253 at most
  float wanted = __uint_as_float(top) * row_up;
  if (sizeof(T) == 4) wanted = __fdiv_rn(fmaxf(wanted, 9.313226e-10f), 6.f);         // (see unit_codes; becomes the smallest scale either way)
  else wanted = __uint_as_float((__float_as_uint(wanted * (1.f / 6.f)) + 0x800u) & 0xfffff000u);
  const unsigned byte = __nv_cvt_float_to_fp8(wanted, __NV_SATFINITE, __NV_E4M3);
  return top == 0 ? 0u : max(byte, 1u);
}

// A unit's codes.  row_up: 1 / row scale.
//
// nvfp4: a = value / row scale is exact.  What has to be told is on which side of a halfway point t the quotient a / s by the block's scale lies, or
// that it is t.  a * (1 / s), off by 2^-21 of itself, is rounded to m, a multiple of 2^-13 (added to 1536, whose steps these are, and taken
// away again): t is one, and where m is not t the quotient is on m's side of it, also 2^-14 further.
//   Bfloat16 values (8 bits) and s t (4 + 3 bits) are equal or differ by 2^-8 of themselves, 2^-10 or more in the quotient: m is t exactly where the
// quotient is.
//   32-bit values: where m is t the sign of a - m s says it, which one instruction rounds once; m goes 2^-14 to that side.  (With divisions, which take
// a long way round for zeros, 65,536 rows of 1,024 took 52 us, of 768 and of 1,000, in which lanes have nothing, 91 and 94.)
// Above 0 for d > 0: 1; below: 0; 0: a half.  d is 0, or 2^-35 or more where a / s is near a halfway point.
__device__ __forceinline__ float side(float d) { return __saturatef(fmaf(d, 6.8719476736e10f, 0.5f)); }
template <typename T, int FORMAT>
__device__ __forceinline__ uint2 unit_codes(const Unit<T> &x, unsigned byte, float row_up) {
  float2 v[UNIT / 2];
#pragma unroll
  for (int i = 0; i < UNIT / 2; ++i) v[i] = x.two(i);
  if (FORMAT == MXFP4) {
    const float up = power_of_two(127 - (int)byte);
#pragma unroll
    for (int i = 0; i < UNIT / 2; ++i) v[i] = mul_two(v[i], make_float2(up, up));
  } else if (sizeof(T) == 4) {
    const float s = byte == 0 ? 1.f : e4m3_value(byte), by = reciprocal(s);          // an empty block is zeros by any scale
#pragma unroll
    for (int i = 0; i < UNIT / 2; ++i) {
      const float2 a = mul_two(v[i], make_float2(row_up, row_up));
      const float2 m = add_two(fma_two(a, make_float2(by, by), make_float2(1536.f, 1536.f)), make_float2(-1536.f, -1536.f));
      const float2 d = fma_two(m, make_float2(-s, -s), a);
      const float2 q = add_two(fma_two(make_float2(side(d.x), side(d.y)), make_float2(1.220703125e-4f, 1.220703125e-4f), m),
                               make_float2(-6.103515625e-5f, -6.103515625e-5f));
      v[i] = make_float2(copysignf(q.x, a.x), copysignf(q.y, a.y));
    }
  } else {
    if (row_up > 1.7e35f) {                    // 2^117: 1 / (row scale * s) would be beyond 32 bits, the row in two steps
      const float up = power_of_two(64);
#pragma unroll
      for (int i = 0; i < UNIT / 2; ++i) v[i] = mul_two(v[i], make_float2(up, up));
      row_up *= power_of_two(-64);
    }
    const float by = byte == 0 ? 0.f : reciprocal(e4m3_value(byte)) * row_up;
#pragma unroll
    for (int i = 0; i < UNIT / 2; ++i) v[i] = add_two(fma_two(v[i], make_float2(by, by), make_float2(1536.f, 1536.f)), make_float2(-1536.f, -1536.f));
  }
  return make_uint2(pack_codes(v), pack_codes(v + 4));
}

struct Fp4Out {
  unsigned char *codes, *scales;
  float *row_scale;
  long long ldc;                // bytes of a row of codes
  long long sf_tiles;           // scale tiles of 128 rows along K
};

// A unit into its codes, with its block's scale byte; a lane in 4 (nvfp4) or 8 (mxfp4) stores the scales of four blocks.  All lanes take part;
// the units of 256 of K lie within the row (`there`), or none does.
template <typename T, int FORMAT>
__device__ __forceinline__ void put_unit(const Fp4Out &o, long long row, int u, bool there, const Unit<T> &x, unsigned top, float row_up) {
  if (FORMAT == MXFP4) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  const unsigned byte = scale_byte<T, FORMAT>(top, row_up);
  const uint2 codes = unit_codes<T, FORMAT>(x, byte, row_up);
  if (there && u * 8 < o.ldc) *reinterpret_cast<uint2 *>(o.codes + row * o.ldc + u * 8) = codes;
  constexpr int LANES = FORMAT == NVFP4 ? 1 : 2, PER = 4 * LANES;     // lanes to a block, to four
  unsigned w = byte | __shfl_xor_sync(0xffffffffu, byte, LANES) << 8;
  w |= __shfl_xor_sync(0xffffffffu, w, 2 * LANES) << 16;
  if (there && u % PER == 0)
    *reinterpret_cast<unsigned *>(o.scales + ((row >> 7) * o.sf_tiles + u / PER) * SF_TILE + (row & 31) * 16 + (row >> 5 & 3) * 4) = w;
}
__device__ __forceinline__ float row_scale_of(int format, unsigned top) {
  return top >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : power_of_two(format == NVFP4 ? row_exponent(top) : 0);
}

// Short rows: LANES lanes to a row, ROWS rows of each such group at once, HELD units of each in a lane's registers between the row's maximum and
// the codes.
template <typename T, int FORMAT, bool VEC, int LANES, int ROWS, int HELD>
__global__ void __launch_bounds__(128)
fp4_quantize_warp_kernel(const T *x, long long ldx, Fp4Out o, long long rows, int K, int n_units) {
  grid_dependents_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x % LANES;
  const long long row0 = ((long long)blockIdx.x * (128 / LANES) + threadIdx.x / LANES) * ROWS;
  __shared__ __align__(16) unsigned stage[VEC ? 1 : 4][VEC ? 1 : 256];
  Unit<T> held[ROWS][HELD];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const T *from = x + (row0 + r) * ldx;
    const int end = row0 + r < rows ? K : 0;
    if (VEC && (lane + HELD * LANES - LANES + 1) * UNIT <= end) {        // asked once: in between the loads of a lane wait for one another
#pragma unroll
      for (int i = 0; i < HELD; ++i) held[r][i].load(from + (lane + i * LANES) * UNIT);
    } else {
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        held[r][i] = VEC ? fetch_unit(from, lane + i * LANES, end) : fetch_unit_over<T, LANES>(from, lane + i * LANES, end, stage[VEC ? 0 : threadIdx.x / 32]);
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    unsigned tu[HELD], top = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      tu[i] = held[r][i].top();
      top = max(top, tu[i]);
    }
    if (LANES == 32) {
      top = __reduce_max_sync(0xffffffffu, top);
    } else {
#pragma unroll
      for (int d = LANES / 2; d > 0; d /= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    }
    const bool there = row0 + r < rows;
    if (lane == 0 && there) o.row_scale[row0 + r] = row_scale_of(FORMAT, top);
    const float row_up = power_of_two(-row_exponent(top));
#pragma unroll
    for (int i = 0; i < HELD; ++i) put_unit<T, FORMAT>(o, row0 + r, lane + i * LANES, there && lane + i * LANES < n_units, held[r][i], tu[i], row_up);
  }
}

// A block of THREADS threads to a row: HELD units of it in a thread's registers, or (HELD 0) the row read twice.
template <typename T, int FORMAT, bool VEC, int THREADS, int HELD>
__global__ void __launch_bounds__(THREADS)
fp4_quantize_block_kernel(const T *x, long long ldx, Fp4Out o, long long rows, int K, int n_units) {
  grid_dependents_launch();
  grid_dependency_wait();
  __shared__ unsigned tops[THREADS / 32];
  __shared__ __align__(16) unsigned stage[VEC ? 1 : THREADS / 32][VEC ? 1 : 256];
  const int t = threadIdx.x;
  const long long row = blockIdx.x;
  const T *r = x + row * ldx;
  Unit<T> held[HELD ? HELD : 1];
  unsigned tu[HELD ? HELD : 1], top = 0;
  auto fetch = [&](int u) { return VEC ? fetch_unit(r, u, K) : fetch_unit_over<T, 32>(r, u, K, stage[VEC ? 0 : t / 32]); };
  if (HELD) {
    if (VEC && (t + HELD * THREADS - THREADS + 1) * UNIT <= K) {          // as above
#pragma unroll
      for (int i = 0; i < HELD; ++i) held[i].load(r + (t + i * THREADS) * UNIT);
    } else {
#pragma unroll
      for (int i = 0; i < HELD; ++i) held[i] = fetch(t + i * THREADS);
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      tu[i] = held[i].top();
      top = max(top, tu[i]);
    }
  } else {
#pragma unroll 4
    for (int u = t; u < (n_units + 31) / 32 * 32; u += THREADS) top = max(top, fetch(u).top());      // whole warps
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (t % 32 == 0) tops[t / 32] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) top = max(top, tops[w]);
  if (t == 0) o.row_scale[row] = row_scale_of(FORMAT, top);
  const float row_up = power_of_two(-row_exponent(top));
  if (HELD) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) put_unit<T, FORMAT>(o, row, t + i * THREADS, t + i * THREADS < n_units, held[i], tu[i], row_up);
  } else {
#pragma unroll 2
    for (int u = t; u < (n_units + 31) / 32 * 32; u += THREADS) {
      const Unit<T> v = fetch(u);
      put_unit<T, FORMAT>(o, row, u, u < n_units, v, v.top(), row_up);
    }
  }
}

template <typename T, int FORMAT, bool VEC>
int launch_quantize(const void *x, long long ldx, const Fp4Out &o, long long rows, int K, cudaStream_t stream) {
  const int n_units = (int)(k_stages(K) * (STAGE_K / UNIT));
#define FP4_GO(KERNEL, BLOCKS, THREADS)                                                                                                   \
  do {                                                                                                                                    \
    LLM_REQUIRE((BLOCKS) < (1ll << 31), "fp4_quantize: too many rows");                                                                  \
    LLM_CHECK_CUDA(llm_launch(KERNEL, dim3((unsigned)(BLOCKS)), dim3(THREADS), 0, stream, (const T *)x, ldx, o, rows, K, n_units),       \
                   "fp4_quantize launch");                                                                                               \
    return LLM_OK;                                                                                                                        \
  } while (0)
#define FP4_WARP(LANES, ROWS, HELD) \
  FP4_GO((fp4_quantize_warp_kernel<T, FORMAT, VEC, LANES, ROWS, HELD>), (rows + 128 / LANES * ROWS - 1) / (128 / LANES * ROWS), 128)
#define FP4_BLOCK(THREADS, HELD) FP4_GO((fp4_quantize_block_kernel<T, FORMAT, VEC, THREADS, HELD>), rows, THREADS)
  // us, bfloat16 into nvfp4.  Rows of up to 512 go in pairs, so that two rows' loads are on their way (128,256 x 256: 15.5, a row to a warp 35.8; 65,536 x
  // 512: 15.2, 18.9).  Up to 2,048 a row is a warp's (128,256 x 2,048: 96.6, a block of 128 threads 135), but where rows are too few to fill the chip
  // that way (beyond 1,024, 32-bit, 1,000 rows: 5.0, a block 4.2; bfloat16, 2,000 rows 4.4 and 4.0; 1,200 x 1,024: 2.7 and 3.0).  Longer rows: blocks as
  // small as hold two units a thread (65,536 x 4,096: 98.8, one unit 121, four 145), and beyond those of 1,024 threads the row is read twice.
  if (n_units <= 16) FP4_WARP(16, 2, 1);
  if (n_units <= 32) FP4_WARP(32, 2, 1);
  if (n_units <= 64) FP4_WARP(32, 1, 2);
  if (n_units <= 128 && rows <= 16 * sm_count()) FP4_BLOCK(128, 1);
  if (n_units <= 128) FP4_WARP(32, 1, 4);
  if (n_units <= 256) FP4_BLOCK(128, 2);
  if (n_units <= 512) FP4_BLOCK(256, 2);
  if (n_units <= 1024) FP4_BLOCK(512, 2);
  if (n_units <= 2048) FP4_BLOCK(1024, 2);
  FP4_BLOCK(1024, 0);
#undef FP4_WARP
#undef FP4_BLOCK
#undef FP4_GO
}

// ---------------------------------------------------------------- back
constexpr int EIGHT = 8;                       // values that a lane brings back at once: 16 bytes of bfloat16
__device__ __forceinline__ float scale_value(int format, unsigned byte) {
  if (format == NVFP4) return e4m3_value(byte & 0x7f);
  return byte == 0 ? __uint_as_float(0x00400000u) : byte == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte << 23);
}
__device__ __forceinline__ void store_unit(__nv_bfloat16 *p, const float (&v)[EIGHT]) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
}
__device__ __forceinline__ void store_unit(float *p, const float (&v)[EIGHT]) {
  reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// Memory bounds it (128,256 x 2,048 of nvfp4 into bfloat16 112 us, 6.0 TB/s, into 32 bits 191 us, 6.2; three quarters of the issue slots are
// taken).  32-bit results, and rows that do not start on 16 bytes, go through shared memory, so that lanes store neighbouring values (each its own:
// 269 us, and 65,536 x 2,047 of bfloat16 370 for 77).
//
// A warp to four times 32 units at a time: PER of them from one row, neighbouring lanes neighbouring units, the others from the rows behind it.
template <typename TO, int FORMAT, bool VEC, int PER>
__global__ void __launch_bounds__(256)
fp4_dequantize_kernel(const unsigned char *codes, const unsigned char *scales, const float *row_scale, TO *out, long long ldo, long long rows, int K,
                      int pieces, long long ldc, long long sf_tiles) {
  constexpr int LANES = FORMAT == NVFP4 ? 2 : 4, ROWS = 4 / PER;
  constexpr bool OVER = !VEC || sizeof(TO) == 4;                         // through shared memory
  __shared__ __align__(16) float stage_raw[OVER ? 8 : 1][OVER ? 32 * EIGHT * sizeof(TO) / 4 : 1];
  TO *stage = reinterpret_cast<TO *>(stage_raw[OVER ? threadIdx.x / 32 : 0]);
  grid_dependents_launch();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const long long n = (rows + ROWS - 1) / ROWS * pieces;
  for (long long job = (long long)blockIdx.x * 8 + threadIdx.x / 32; job < n; job += (long long)gridDim.x * 8) {
    const long long row0 = (PER < 4 ? job : job / pieces) * ROWS;
    const int u0 = (PER < 4 ? 0 : (int)(job - row0 * pieces) * 128) + lane;
    unsigned c[4], byte[4];
    float rs[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const long long row = row0 + r;
      const int end = ROWS == 1 || row < rows ? K : 0;
      const unsigned char *sf = scales + (row >> 7) * sf_tiles * SF_TILE + (row & 31) * 16 + (row >> 5 & 3) * 4;
      rs[r] = end ? row_scale[row] : 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int u = u0 + i * 32, block = u / LANES;
        c[r * PER + i] = u * EIGHT < end ? *reinterpret_cast<const unsigned *>(codes + row * ldc + u * 4) : 0;
        byte[r * PER + i] = u * EIGHT < end ? sf[(block / 4) * SF_TILE + block % 4] : 0;
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const long long row = row0 + r;
      if (ROWS > 1 && row >= rows) break;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int u = u0 + i * 32, k0 = (u - lane) * EIGHT;
        if ((OVER ? k0 : u * EIGHT) >= K) break;
        const float by = scale_value(FORMAT, byte[r * PER + i]) * rs[r];       // exact: a scale has four bits
        float v[EIGHT];
#pragma unroll
        for (int j = 0; j < EIGHT / 2; ++j) {
          const float2 f = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(c[r * PER + i] >> 8 * j & 0xff), __NV_E2M1)));
          v[2 * j] = f.x * by;
          v[2 * j + 1] = f.y * by;
        }
        TO *p = out + row * ldo;
        if (OVER) {
          __syncwarp();
          store_unit(stage + lane * EIGHT, v);
          __syncwarp();
        }
        if (VEC && OVER) {
#pragma unroll
          for (int j = 0; j < EIGHT / 4; ++j) {
            const int at = (j * 32 + lane) * 4;
            const float4 w = reinterpret_cast<const float4 *>(stage)[j * 32 + lane];
            if (k0 + at + 4 <= K) {
              *reinterpret_cast<float4 *>(p + k0 + at) = w;
            } else {
              if (k0 + at < K) p[k0 + at] = w.x;
              if (k0 + at + 1 < K) p[k0 + at + 1] = w.y;
              if (k0 + at + 2 < K) p[k0 + at + 2] = w.z;
            }
          }
        } else if (OVER) {
#pragma unroll
          for (int j = 0; j < EIGHT; ++j)
            if (k0 + j * 32 + lane < K) p[k0 + j * 32 + lane] = stage[j * 32 + lane];
        } else if ((u + 1) * EIGHT <= K) {
          store_unit(p + u * EIGHT, v);
        } else {
#pragma unroll
          for (int j = 0; j < EIGHT; ++j)
            if (u * EIGHT + j < K) p[u * EIGHT + j] = from_float<TO>(v[j]);
        }
      }
    }
  }
}

template <typename TO, int FORMAT, bool VEC, int PER>
int launch_dequantize(const Fp4DequantizeCall &c) {
  const long long K = c.cols, pieces = PER < 4 ? 1 : (K + 128 * EIGHT - 1) / (128 * EIGHT), jobs = (c.rows + 4 / PER - 1) / (4 / PER) * pieces;
  const long long blocks = (jobs + 7) / 8, most = 8ll * 4 * sm_count();
  LLM_CHECK_CUDA(llm_launch(fp4_dequantize_kernel<TO, FORMAT, VEC, PER>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, (cudaStream_t)c.stream,
                            (const unsigned char *)c.codes, (const unsigned char *)c.scales, c.row_scale, (TO *)c.out, c.ldo, c.rows, (int)K, (int)pieces,
                            code_bytes(K), k_stages(K) * stage_tiles(FORMAT)),
                 "fp4_dequantize launch");
  return LLM_OK;
}
// (128,256 x 256: 18.7 us, four from one row 35.3; 65,536 x 512: 16.9, 23.2.)
template <typename TO, int FORMAT, bool VEC>
int dispatch_dequantize_per(const Fp4DequantizeCall &c) {
  if (c.cols <= 32 * EIGHT) return launch_dequantize<TO, FORMAT, VEC, 1>(c);
  if (c.cols <= 64 * EIGHT) return launch_dequantize<TO, FORMAT, VEC, 2>(c);
  return launch_dequantize<TO, FORMAT, VEC, 4>(c);
}
template <typename TO, int FORMAT>
int dispatch_dequantize(const Fp4DequantizeCall &c) {
  const bool vec = ((uintptr_t)c.out | (unsigned long long)c.ldo * sizeof(TO)) % 16 == 0;
  return vec ? dispatch_dequantize_per<TO, FORMAT, true>(c) : dispatch_dequantize_per<TO, FORMAT, false>(c);
}

// ---------------------------------------------------------------- the product
// out[t, n] = Rx[t] Rw[n] sum over blocks b of sx[t, b] sw[n, b] sum over k of b of cx[t, k] cw[n, k]: tcgen05.mma with block scales takes codes
// from shared memory and scales from tensor memory and adds in 32 bits; the rows' scales are the epilogue's.
//
// The structure is gemm_tc.cu's: W's rows are the instruction's 128 rows, the tokens its N (16 to 128); a persistent CTA to an SM with a
// loader, an issuer and four epilogue warps, a ring of stages of 256 of K, two accumulators.  With the codes of a stage come its scales,
// as they lie in memory; the issuer has them copied to tensor memory (tcgen05.cp, in order with the products that read
// them) behind the accumulators.  Nothing orders a copy behind earlier products that read what was there, so every stage of the ring has its place: what
// says that the stage is free says so of the place.  (With two places and a wait for the products of two stages ago 8 x 28,672 x 4,096 took 15.0 us
// for 12.4.)
//
// Few tokens: W's bytes bound it (8 x 128,256 x 2,048: 27.4 us, 5.5 TB/s over seven rounds of tiles; 8 x 28,672 x 4,096: 12.4 us, 5.3 TB/s), and for small
// matrices the latency of one round, which parts of K in a cluster shorten (k_parts).
constexpr int FP_THREADS = 192;
constexpr int FP_ROWS = 128;

template <int TN, int FORMAT>
struct FpShape {
  static constexpr int TILES = stage_tiles(FORMAT);                       // scale tiles of 128 rows in a stage
  static constexpr int A_BYTES = FP_ROWS * 128, B_BYTES = TN * 128;
  static constexpr int SF_BYTES = TILES * SF_TILE;                        // of 128 rows
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + 2 * SF_BYTES;
  static constexpr int STAGES = 190 * 1024 / STAGE_BYTES;
  static constexpr int SF_COLS = TILES * 8;                               // columns of tensor memory of a stage's scales
  static constexpr int COLS = 2 * TN + STAGES * SF_COLS;
  static constexpr int TMEM_COLS = COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  static constexpr int ROW_BYTES = 4 * TN * 4;                            // row scales of the tile's tokens, for each epilogue warp
  static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE_BYTES + ROW_BYTES + 512;
  static_assert(STAGE_BYTES % 1024 == 0 && COLS <= 512 && (2 * STAGES + 6) * 8 + 8 <= 512, "a stage's parts do not fit");
};

// Instruction descriptor with block scales: A and B e2m1 (bits 7-9 and 10-12 = 1), both K-major, N >> 3 in bits 17-22, scales e8m0 (bit 23 = 1) or
// e4m3, M >> 4 in bits 24-28; which byte of a scale word is the first: B's in bits 4-5, A's in bits 29-30.
__host__ __device__ constexpr unsigned fp4_instr(int format, int m, int n, int sf) {
  return ((unsigned)sf << 4) | (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | ((unsigned)(format == MXFP4) << 23) | ((unsigned)(m >> 4) << 24) |
         ((unsigned)sf << 29);
}
template <int FORMAT>
__device__ __forceinline__ void fp4_mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned sfa, unsigned sfb,
                                        unsigned accumulate) {
  if (FORMAT == NVFP4)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// A scale tile to four columns of tensor memory, the same to each quarter of the lanes: 32 rows of 16 bytes, no swizzle, groups of 8 rows 128
// bytes apart.
__device__ __forceinline__ void scales_to_tmem(unsigned taddr, unsigned smem) {
  unsigned long long d = (unsigned long long)((smem & 0x3FFFF) >> 4);
  d |= 1ull << 16;
  d |= (unsigned long long)(128 >> 4) << 32;
  d |= 1ull << 46;
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}
__device__ __forceinline__ void bulk_load(unsigned dst, const void *src, unsigned bytes, unsigned bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned in_cta(unsigned addr, unsigned rank) {      // the same place in the shared memory of a CTA of the cluster
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A sum times its two rows' scales, which are powers of two (mxfp4: 1, so that the order does not matter; what its blocks' scales make of a sum has to lie within 32
// bits by itself).  nvfp4: codes are multiples of 1/2, block scales of 2^-9, so sums are multiples of 2^-20; a value is 6 x 352 at most, a sum below 2^23 K,
// 2^51 for the longest K.  Between 2^-63 and 2^64 (`near_one`) either order is safe: sum and first scale meet between 2^-83 and 2^115, without rounding, and the second
// scale rounds once, if the result leaves the ordinary numbers.  Beyond, scales at opposite ends of the range meet first (their product is in range where
// one step would leave it).  Scales whose product is out of range go one after the other: both above 1 (rows of 2^117 at most), where a first step that overflows
// would not have come back, or both below, where a first step that rounds is off by half of 2^-149 and the second makes that less.
__device__ __forceinline__ bool near_one(float scale) {
  const unsigned e = __float_as_uint(scale) >> 23;       // a NaN or a sign is not near
  return e >= 64 && e <= 190;
}
__device__ __forceinline__ float scaled_far(float v, float rw, float rx) {
  const float p = rw * rx;
  return fabsf(p) >= 1.17549435e-38f && fabsf(p) <= 3.40282347e38f ? v * p : v * rw * rx;
}

struct Fp4In {
  const unsigned char *x_scales, *w_scales;
  const float *x_row, *w_row;
};

template <int TN, int FORMAT, typename TO>
__global__ void __launch_bounds__(FP_THREADS, 1)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, Fp4In in, TO *out, long long ldo, int M, int N,
                int n_stages, int row_tiles, int tok_tiles, int parts, int weights_first, int *status) {
  using S = FpShape<TN, FORMAT>;
  constexpr int STAGES = S::STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float *row_raw = (float *)(smem + (size_t)STAGES * S::STAGE_BYTES);
  unsigned long long *bars = (unsigned long long *)((unsigned char *)row_raw + S::ROW_BYTES);
  const unsigned bar_full = smem_u32(bars), bar_empty = smem_u32(bars + STAGES);
  const unsigned bar_tfull = smem_u32(bars + 2 * STAGES), bar_tempty = smem_u32(bars + 2 * STAGES + 2);
  unsigned *tmem_slot = (unsigned *)(bars + 2 * STAGES + 4);
  volatile int *abort_flag = (volatile int *)(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  grid_dependents_launch();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(bar_tfull + 8 * a, 1);
      mbar_init(bar_tempty + 8 * a, 4);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tma_prefetch_map(&map_w);
    tma_prefetch_map(&map_x);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"((unsigned)S::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem_base = *tmem_slot;
  // this CTA's tiles, and of each its part of K (parts > 1: a cluster to a tile, which is the only one)
  const int n_tiles = row_tiles * tok_tiles, part = parts > 1 ? (int)cluster_rank() : 0;
  const int tile0 = blockIdx.x / parts, step = gridDim.x / parts;
  const int kb0 = n_stages * part / parts, kb1 = n_stages * (part + 1) / parts;
  const long long sf_row_tile = (long long)n_stages * S::SF_BYTES;        // bytes of 128 rows' scales

  bool near = true;                            // of the epilogue's tile: scales that may be applied one by one
  if (warp == 0) {
    // ------------------------------------------------------------ loader
    const bool leader = elect_one();
    struct Walk {
      int tile, kb;
      bool valid;
    };
    auto next = [&](Walk &w) {
      if (++w.kb >= kb1) {
        w.kb = kb0;
        w.tile += step;
        w.valid = w.tile < n_tiles;
      }
    };
    auto load_w = [&](const Walk &w, int stage) {
      if (!leader) return;
      const unsigned dst = smem_u32(smem + (size_t)stage * S::STAGE_BYTES), bar = bar_full + 8 * stage;
      const int row_tile = w.tile / tok_tiles;
      mbar_expect_tx(bar, S::STAGE_BYTES);
      tma_load_2d(dst, &map_w, w.kb * 128, row_tile * FP_ROWS, bar);
      bulk_load(dst + S::A_BYTES + S::B_BYTES, in.w_scales + row_tile * sf_row_tile + (long long)w.kb * S::SF_BYTES, S::SF_BYTES, bar);
    };
    auto load_x = [&](const Walk &w, int stage) {
      if (!leader) return;
      const unsigned dst = smem_u32(smem + (size_t)stage * S::STAGE_BYTES), bar = bar_full + 8 * stage;
      const int tok0 = w.tile % tok_tiles * TN;
      tma_load_2d(dst + S::A_BYTES, &map_x, w.kb * 128, tok0, bar);
      bulk_load(dst + S::A_BYTES + S::B_BYTES + S::SF_BYTES, in.x_scales + tok0 / 128 * sf_row_tile + (long long)w.kb * S::SF_BYTES, S::SF_BYTES, bar);
    };
    Walk w{tile0, kb0, tile0 < n_tiles}, w2 = w;
    if (!weights_first) grid_dependency_wait();
    int n_pre = 0;
    for (; w.valid && n_pre < STAGES; next(w), ++n_pre) load_w(w, n_pre);
    if (weights_first) grid_dependency_wait();
    for (int s = 0; s < n_pre; ++s, next(w2)) load_x(w2, s);
    int stage = n_pre % STAGES;
    unsigned phase = n_pre == STAGES ? 1u : 0u;
    bool ok = true;
    for (; w.valid; next(w)) {
      ok = __all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, status, 1));
      if (!ok) break;
      load_w(w, stage);
      load_x(w, stage);
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (leader && (!ok || *abort_flag)) {
      // given up: let the loads that are in flight land before the CTA goes away
      const unsigned long long t0 = globaltimer();
      for (int s = 0; s < STAGES; ++s)
        while (!mbar_try(bar_full + 8 * s, 0) && !mbar_try(bar_full + 8 * s, 1) && globaltimer() - t0 < 2000000ull) {
        }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ tensor-core issue
    const bool leader = elect_one();
    int stage = 0, iter = 0;
    unsigned phase = 0;
    bool ok = true;
    for (int tile = tile0; tile < n_tiles && ok; tile += step, ++iter) {
      const int acc = iter & 1, tok0 = tile % tok_tiles * TN;
      const unsigned shift = (unsigned)(tok0 % 128 / 32);                 // a tile of tokens may start within a scale tile
      ok = __all_sync(0xffffffffu, mbar_wait(bar_tempty + 8 * acc, ((iter >> 1) & 1) ^ 1, abort_flag, status, 2));
      if (!ok) break;
      tc_fence_after();
      const unsigned d_tmem = tmem_base + acc * TN;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_full + 8 * stage, phase, abort_flag, status, 3));
        if (!ok) break;
        tc_fence_after();
        const unsigned a_addr = smem_u32(smem + (size_t)stage * S::STAGE_BYTES);
        const unsigned long long a_desc = smem_desc(a_addr), b_desc = smem_desc(a_addr + S::A_BYTES);
        const unsigned sf = a_addr + S::A_BYTES + S::B_BYTES;
        const unsigned sfa = tmem_base + 2 * TN + stage * S::SF_COLS, sfb = sfa + S::TILES * 4;
        if (leader) {
#pragma unroll
          for (int j = 0; j < S::TILES; ++j) {
            scales_to_tmem(sfa + j * 4, sf + j * SF_TILE);
            scales_to_tmem(sfb + j * 4, sf + S::SF_BYTES + j * SF_TILE);
          }
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {           // 64 of K = 32 bytes further along the swizzled row
            const int j = kk * S::TILES / 4, first = FORMAT == NVFP4 ? 0 : kk % 2 * 2;
            fp4_mma<FORMAT>(d_tmem, a_desc + (unsigned long long)(kk * 2), b_desc + (unsigned long long)(kk * 2),
                            fp4_instr(FORMAT, FP_ROWS, TN, first), sfa + j * 4, sfb + j * 4 + shift, kk > 0 || kb > kb0 ? 1u : 0u);
          }
          tc_commit(bar_empty + 8 * stage);
        }
        __syncwarp();
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (ok && leader) tc_commit(bar_tfull + 8 * acc);
      __syncwarp();
    }
    grid_dependency_wait();
  } else {
    // ------------------------------------------------------------ epilogue (warps 2..5)
    grid_dependency_wait();
    const int quarter = warp & 3;
    int iter = 0;
    for (int tile = tile0; tile < n_tiles; tile += step, ++iter) {
      const int acc = iter & 1, tok0 = tile % tok_tiles * TN, f = tile / tok_tiles * FP_ROWS + quarter * 32 + lane;
      // the rows' scales, while the products run: from memory at each use they cost more than the rest of the epilogue
      const float rw = f < N ? in.w_row[f] : 0.f;
      float *rx = row_raw + (warp - 2) * TN;
      __syncwarp();
      near = near_one(rw) || f >= N;
      for (int i = lane; i < TN; i += 32) {
        const float r = tok0 + i < M ? in.x_row[tok0 + i] : 1.f;
        near = near && near_one(r);
        rx[i] = r;
      }
      near = __all_sync(0xffffffffu, near);
      const float rw1 = near ? rw : 1.f;
      __syncwarp();
      if (!__all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * acc, (iter >> 1) & 1, abort_flag, status, 4))) break;
      tc_fence_after();
      if (parts > 1) break;                    // the parts are added below
#pragma unroll 1
      for (int c0 = 0; c0 < TN && tok0 + c0 < M; c0 += 16) {
        float v[16], r[16];
        const int n = M - tok0 - c0;           // tokens from here on
#pragma unroll
        for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4 *>(r + i) = *reinterpret_cast<const float4 *>(rx + c0 + i);
        tc_ld16(tmem_base + ((unsigned)(quarter * 32) << 16) + (unsigned)(acc * TN + c0), v);
        if (!near) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            v[i] = scaled_far(v[i], rw, r[i]);
            r[i] = 1.f;
          }
        }
        if (f < N) {
          TO *p = out + (size_t)(tok0 + c0) * ldo + f;
#pragma unroll
          for (int i = 0; i < 16; ++i, p += ldo)
            if (i < n) *p = from_float<TO>(v[i] * rw1 * r[i]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_tempty + 8 * acc);
    }
  }

  if (parts > 1) {
    // ------------------------------------------------------------ the parts' sums: each CTA adds those of its share of the tokens, in order
    // The sums meet in the rings, which nobody needs any more once every CTA has come to the first barrier.
    const int quarter = warp & 3, row = quarter * 32 + lane, f = tile0 / tok_tiles * FP_ROWS + row;
    const int shift = 31 - __clz(TN / parts), share = 1 << shift, tok0 = tile0 % tok_tiles * TN + part * share;
    __syncwarp();
    cluster_sync();
    if (warp >= 2) {
      const unsigned mine = smem_u32(smem) + ((unsigned)(part * share) * FP_ROWS + (unsigned)row) * 4;      // of my part, in whosever ring
      float v[2][16];
#pragma unroll 1
      for (int c0 = 0; c0 < TN; c0 += 32) {
        const unsigned taddr = tmem_base + ((unsigned)(quarter * 32) << 16) + (unsigned)c0;
        tc_ld16(taddr, v[0]);
        if (TN > 16) tc_ld16(taddr + 16, v[1]);
#pragma unroll
        for (int i = 0; i < (TN > 16 ? 32 : 16); ++i)
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(in_cta(mine + (unsigned)(((c0 + i) & (share - 1)) * FP_ROWS * 4), (unsigned)((c0 + i) >> shift))),
                       "f"(v[i / 16][i % 16]) : "memory");
      }
    }
    __syncwarp();
    cluster_sync();
    if (warp >= 2 && f < N) {
      const float rw = in.w_row[f], *sums = (const float *)smem + row, *rx = row_raw + (warp - 2) * TN + part * share;
      TO *p = out + (size_t)tok0 * ldo + f;
#pragma unroll 4
      for (int c = 0; c < min(share, M - tok0); ++c, p += ldo) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < parts) v += sums[(q * share + c) * FP_ROWS];
        *p = from_float<TO>(near ? v * rw * rx[c] : scaled_far(v, rw, rx[c]));
      }
    }
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((unsigned)S::TMEM_COLS)
                 : "memory");
  }
}

// A map over rows of codes: boxes of 128 bytes (256 of K) x box_rows, 128-byte swizzle, zeros outside.
int get_code_map(const void *codes, long long rows, long long K, int box_rows, CUtensorMap *out) {
  EncodeTiledFn fn = encode_fn();
  LLM_REQUIRE(fn != nullptr, "tensor map: the driver does not offer cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {(cuuint64_t)code_bytes(K), (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)code_bytes(K)};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(codes), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  LLM_REQUIRE(r == CUDA_SUCCESS, "tensor map: cuTensorMapEncodeTiled failed (%d) for codes of %lld x %lld", (int)r, rows, K);
  return LLM_OK;
}

// Parts of K of a product of up to 128 tokens: as many as leave every CTA an SM of its own, eight only of matrices with 8 tiles or fewer (16
// clusters of 8 CTAs are not on the chip at once).  Handing sums over costs more the more tokens there are: up to 32 tokens, two stages to a part are
// enough; beyond, four parts or eight of 32 stages or more.  In 1 / 2 / 4 / 8 parts, us: 2,048 features, K = 2,048, 1 token 5.1 / 4.2 / 3.6 / 3.6, 64 tokens
// 5.5 / 7.3 / 5.7 / 5.7; K = 1,024, 8 tokens 3.5 / 4.0; K = 8,192, 8 tokens 11.5 / 8.5 / 6.2 / 8.7, 64 tokens 11.9 / 10.9 / 8.0 / 12.3, 128 tokens 13.1 / 14.2 /
// 10.7 / 17.1; 512 features, K = 16,384, 1 token 19.5 / 12.1 / 8.0 / 5.9; 8,192 features, K = 8,192, 8 tokens 11.9 / 10.4, 64 tokens 12.7 / 13.1.
// Other parts round their sums elsewhere: of matrices of up to 74 tiles (9,472 features) and K beyond 1,792 a token's result may differ in its last bits between calls of 32
// and 33 tokens, or of 128 and 129.  Elsewhere it has no part in what other tokens the call holds.
int k_parts(int M, int N, int K) {
  const long long tiles = (N + FP_ROWS - 1) / FP_ROWS, stages = k_stages(K);
  int parts = 1;
  while (parts < 8 && tiles * parts * 2 <= (parts == 4 ? 64 : sm_count()) && stages >= 8 && stages >= parts * 4) parts *= 2;
  return M <= 32 || (parts >= 4 && stages >= 32) ? parts : 1;
}

template <int TN, int FORMAT, typename TO>
int launch_fp4(const void *x_codes, const void *w_codes, const Fp4In &in, void *out, long long ldo, int M, int N, int K, int parts, int weights_first,
               int *status, cudaStream_t stream) {
  using S = FpShape<TN, FORMAT>;
  const int row_tiles = (N + FP_ROWS - 1) / FP_ROWS, tok_tiles = (M + TN - 1) / TN;
  CUtensorMap map_w, map_x;
  int rc = get_code_map(w_codes, N, K, FP_ROWS, &map_w);
  if (rc != LLM_OK) return rc;
  rc = get_code_map(x_codes, M, K, TN, &map_x);
  if (rc != LLM_OK) return rc;
  auto kern = fp4_gemm_kernel<TN, FORMAT, TO>;
  LLM_CHECK_CUDA(llm_allow_smem(kern, S::SMEM), "fp4_gemm attribute");
  const long long tiles = (long long)row_tiles * tok_tiles;
  LLM_REQUIRE(tiles < (1ll << 30), "fp4_gemm: too many tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts > 1 ? (unsigned)tiles * parts : (unsigned)(tiles < sm_count() ? tiles : sm_count()));
  cfg.blockDim = dim3(FP_THREADS);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (llm_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (parts > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)parts;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  LLM_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, map_w, map_x, in, (TO *)out, ldo, M, N, (int)k_stages(K), row_tiles, tok_tiles, parts, weights_first, status),
                 "fp4_gemm launch");
  return LLM_OK;
}

// ---------------------------------------------------------------- the product of prompts, two SMs to a tile
// At thousands of tokens the operands are what an SM cannot bring in fast enough: 128 rows x 192 take 46 KB (with their scales) for 384 cycles of
// products, 120 bytes a cycle where loads end at 64.  A cluster of two CTAs works on a tile of 256 tokens x 192 features (cta_group::2): each
// brings 128 tokens and 96 features, 34 KB, and holds the sums of its tokens; the instruction has them in its lanes and the features in its
// columns.  The CTA of even rank issues the products and the copies of scales for both; each CTA brings the scales of its tokens and of all 192
// features, in two places in turn.  The epilogue warps scale the sums, put boxes of 32 tokens x 128 bytes into buffers of their own and have TMA store
// them (a result whose rows do not start on 16 bytes, and the box that hangs over the last feature, the lanes store from there, row by row: 1,000 x
// 1,999 x 1,500 9.5 us, each lane a token's row 35).  With 64 bytes to a box, twice the fences, 2,048 x 16,384 x 2,048 took 41.5 us for 37, and the rows'
// scales, loaded a tile ahead, are part of that.
//
// 8,192 cubed: mxfp4 205 us, 5.4 PFLOP/s, nvfp4 220 us, 5.0; a stage takes 570 cycles for some 400 of products, 34 KB at 60 bytes a cycle.  2,048 x 16,384 x
// 2,048 nvfp4: 37 us (3.7 PFLOP/s), ten rounds of tiles of eight stages; with one stage to a tile 22, the epilogue's time, which hides behind eight stages
// and no fewer.  One SM to a tile took 242 us at 8,192 cubed; six stages in the ring, and eight epilogue warps for twelve, change nothing.
// Into 32 bits 2,048 x 16,384 x 2,048 takes 50 us, 23.7 of which its bytes take: eight epilogue warps, boxes of 32 features from two buffers in turn, four stages.
constexpr int PR_TOKENS = 256, PR_FEATURES = 192;
template <int FORMAT, typename TO>
struct PairShape {
  static constexpr int TILES = stage_tiles(FORMAT), SF_BYTES = TILES * SF_TILE;
  static constexpr int A_BYTES = PR_TOKENS / 2 * 128, B_BYTES = PR_FEATURES / 2 * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + 3 * SF_BYTES;
  static constexpr int STAGES = sizeof(TO) == 4 ? 4 : 5;
  static constexpr int SHARES = sizeof(TO) == 4 ? 2 : 3, SHARE = PR_FEATURES / SHARES;    // epilogue warps to a quarter of the lanes; their features
  static constexpr int WARPS = 4 * SHARES, THREADS = 64 + 32 * WARPS;
  static constexpr int SF_COLS = TILES * 12;                             // columns of a stage's scales: 4 of a tile for the tokens, 8 for the features
  static constexpr int BOX = 128 / (int)sizeof(TO), BOXES = SHARE / BOX, BUFFERS = BOXES > 1 ? 2 : 1;
  static constexpr int OUT_BYTES = 32 * 128;                             // 32 tokens x BOX features on their way out
  static constexpr int ROW_BYTES = WARPS * SHARE * 4;       // row scales of its features, for each epilogue warp
  static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE_BYTES + BUFFERS * WARPS * OUT_BYTES + ROW_BYTES + 256;
  static_assert(STAGE_BYTES % 1024 == 0 && 2 * PR_FEATURES + 2 * SF_COLS <= 512, "a stage's parts do not fit");
};
__device__ __forceinline__ void pair_load(unsigned dst, const CUtensorMap *map, int x, int y, unsigned bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void pair_scales_to_tmem(unsigned taddr, unsigned smem) {      // in both CTAs, each from its own shared memory
  unsigned long long d = (unsigned long long)((smem & 0x3FFFF) >> 4);
  d |= 1ull << 16;
  d |= (unsigned long long)(128 >> 4) << 32;
  d |= 1ull << 46;
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}
template <int FORMAT>
__device__ __forceinline__ void pair_mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned sfa, unsigned sfb,
                                         unsigned accumulate) {
  if (FORMAT == NVFP4)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// 16 bytes of a row of 128, the values from v on, into the box that TMA stores, swizzled as it takes them: piece ^ row % 8.
__device__ __forceinline__ void put_piece(unsigned box, int row, int piece, const float *v, float) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(box + row * 128 + ((piece ^ (row & 7)) << 4)), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3])
               : "memory");
}
__device__ __forceinline__ void put_piece(unsigned box, int row, int piece, const float *v, __nv_bfloat16) {
  unsigned w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    w[j] = *reinterpret_cast<const unsigned *>(&h);
  }
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + row * 128 + ((piece ^ (row & 7)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
               : "memory");
}

template <int FORMAT, typename TO>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__((PairShape<FORMAT, TO>::THREADS), 1)
fp4_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_xs,
                const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ CUtensorMap map_out, const float *x_row, const float *w_row, TO *out,
                long long ldo, int M, int N, int n_stages, int tok_tiles, int feature_tiles, int weights_first, int by_tma, int *status) {
  using S = PairShape<FORMAT, TO>;
  constexpr int STAGES = S::STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char *out_raw = smem + (size_t)STAGES * S::STAGE_BYTES;
  float *row_raw = (float *)(out_raw + S::BUFFERS * S::WARPS * S::OUT_BYTES);
  unsigned long long *bars = (unsigned long long *)((unsigned char *)row_raw + S::ROW_BYTES);
  const unsigned bar_full = smem_u32(bars), bar_empty = smem_u32(bars + STAGES);
  const unsigned bar_tfull = smem_u32(bars + 2 * STAGES), bar_tempty = smem_u32(bars + 2 * STAGES + 2);
  unsigned *tmem_slot = (unsigned *)(bars + 2 * STAGES + 4);
  volatile int *abort_flag = (volatile int *)(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const unsigned rank = cluster_rank();
  grid_dependents_launch();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);          // rank 0's: its loader, and the bytes of both
      mbar_init(bar_empty + 8 * s, 1);         // each CTA's own: the products that read the stage, committed to both
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(bar_tfull + 8 * a, 1);         // each CTA's own
      mbar_init(bar_tempty + 8 * a, 2 * S::WARPS);      // rank 0's: the epilogue warps of both
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tma_prefetch_map(&map_w);
    tma_prefetch_map(&map_x);
    tma_prefetch_map(&map_ws);
    tma_prefetch_map(&map_xs);
  }
  if (warp == 1) {                             // in both CTAs: the pair's tensor memory is allocated together
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();                              // both CTAs' barriers are there before anyone signals the other's
  tc_fence_after();
  const unsigned tmem_base = *tmem_slot;
  const int n_tiles = tok_tiles * feature_tiles, first = blockIdx.x / 2, step = gridDim.x / 2;      // this pair's tiles
  const int sf_tiles = n_stages * S::TILES;    // scale tiles of 128 rows

  if (warp == 0) {
    // ------------------------------------------------------------ loader: this CTA's half of both operands, and its scales
    const bool leader = elect_one();
    struct Walk {
      int tile, kb;
      bool valid;
    };
    auto next = [&](Walk &w) {
      if (++w.kb >= n_stages) {
        w.kb = 0;
        w.tile += step;
        w.valid = w.tile < n_tiles;
      }
    };
    auto load_w = [&](const Walk &w, int stage) {
      if (!leader) return;
      const unsigned full = in_cta(bar_full + 8 * stage, 0), dst = smem_u32(smem + (size_t)stage * S::STAGE_BYTES);
      const int f0 = w.tile / tok_tiles * PR_FEATURES, sf = f0 / 128 * sf_tiles + w.kb * S::TILES;
      if (rank == 0) mbar_expect_tx(bar_full + 8 * stage, 2 * S::STAGE_BYTES);
      pair_load(dst + S::A_BYTES, &map_w, w.kb * 128, f0 + (int)rank * (PR_FEATURES / 2), full);
      pair_load(dst + S::A_BYTES + S::B_BYTES + S::SF_BYTES, &map_ws, 0, sf, full);
      pair_load(dst + S::A_BYTES + S::B_BYTES + 2 * S::SF_BYTES, &map_ws, 0, sf + sf_tiles, full);     // behind the last row tile: zeros
    };
    auto load_x = [&](const Walk &w, int stage) {
      if (!leader) return;
      const unsigned full = in_cta(bar_full + 8 * stage, 0), dst = smem_u32(smem + (size_t)stage * S::STAGE_BYTES);
      const int half = w.tile % tok_tiles * 2 + (int)rank;
      pair_load(dst, &map_x, w.kb * 128, half * 128, full);
      pair_load(dst + S::A_BYTES + S::B_BYTES, &map_xs, 0, half * sf_tiles + w.kb * S::TILES, full);
    };
    Walk w{first, 0, first < n_tiles}, w2 = w;
    if (!weights_first) grid_dependency_wait();
    int n_pre = 0;
    for (; w.valid && n_pre < STAGES; next(w), ++n_pre) load_w(w, n_pre);
    if (weights_first) grid_dependency_wait();
    for (int s = 0; s < n_pre; ++s, next(w2)) load_x(w2, s);
    int stage = n_pre % STAGES;
    unsigned phase = n_pre == STAGES ? 1u : 0u;
    bool ok = true;
    for (; w.valid; next(w)) {
      ok = __all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, status, 1));
      if (!ok) break;
      load_w(w, stage);
      load_x(w, stage);
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (!ok) {                                 // given up: what is in flight lands within this time, whoever's barrier it signals
      const unsigned long long t0 = globaltimer();
      while (globaltimer() - t0 < 2000000ull) {
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ products and copies of scales in both CTAs, issued by rank 0
    auto commit = [&](unsigned bar) {          // arrives at this barrier in both CTAs when what was issued so far is done
      asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                   ::"r"(bar), "h"((unsigned short)3) : "memory");
    };
    // One lane alone: with the warp's votes behind every wait the wait for a place cost 5 %.
    if (elect_one() && rank == 0) {
      int stage = 0, iter = 0, issued = 0;
      unsigned phase = 0, turn = 0;
      bool ok = true;
      for (int tile = first; tile < n_tiles && ok; tile += step, ++iter) {
        const int acc = iter & 1;
        const unsigned shift = (unsigned)(tile / tok_tiles * PR_FEATURES % 128 / 32);     // a tile may start in the middle of a scale tile
        ok = mbar_wait(bar_tempty + 8 * acc, ((iter >> 1) & 1) ^ 1, abort_flag, status, 2);
        if (!ok) break;
        const unsigned d_tmem = tmem_base + acc * PR_FEATURES;
        for (int kb = 0; kb < n_stages; ++kb, turn ^= 1) {
          // Nothing orders a copy of scales behind the products that read what was in its place: those of two stages ago have to be done.  Asked before
          // the wait for the stage this costs nothing (8,192 cubed 219 us, without it 220), behind it 6 % (230).
          if (issued >= 2) {
            const int ago = stage >= 2 ? stage - 2 : stage - 2 + STAGES;
            ok = mbar_wait(bar_empty + 8 * ago, stage >= 2 ? phase : phase ^ 1, abort_flag, status, 2);
          }
          issued += issued < 2;
          ok = ok && mbar_wait(bar_full + 8 * stage, phase, abort_flag, status, 3);
          if (!ok) break;
          tc_fence_after();
          const unsigned a_addr = smem_u32(smem + (size_t)stage * S::STAGE_BYTES), sf = a_addr + S::A_BYTES + S::B_BYTES;
          const unsigned long long a_desc = smem_desc(a_addr), b_desc = smem_desc(a_addr + S::A_BYTES);
          const unsigned sfa = tmem_base + 2 * PR_FEATURES + turn * S::SF_COLS, sfb = sfa + S::TILES * 4;
#pragma unroll
          for (int j = 0; j < S::TILES; ++j) {
            pair_scales_to_tmem(sfa + j * 4, sf + j * SF_TILE);
            pair_scales_to_tmem(sfb + j * 8, sf + S::SF_BYTES + j * SF_TILE);
            pair_scales_to_tmem(sfb + j * 8 + 4, sf + 2 * S::SF_BYTES + j * SF_TILE);
          }
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {           // 64 of K = 32 bytes further along the swizzled row
            const int j = kk * S::TILES / 4, at = FORMAT == NVFP4 ? 0 : kk % 2 * 2;
            pair_mma<FORMAT>(d_tmem, a_desc + (unsigned long long)(kk * 2), b_desc + (unsigned long long)(kk * 2),
                             fp4_instr(FORMAT, PR_TOKENS, PR_FEATURES, at), sfa + j * 4, sfb + j * 8 + shift, kk > 0 || kb > 0 ? 1u : 0u);
          }
          commit(bar_empty + 8 * stage);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (ok) commit(bar_tfull + 8 * acc);
      }
    }
    __syncwarp();
    grid_dependency_wait();
  } else {
    // ------------------------------------------------------------ epilogue of this CTA's 128 tokens (warps 2 and up)
    grid_dependency_wait();
    const int quarter = warp & 3, from = (warp - 2) / 4 * S::SHARE;        // the lanes of tensor memory the warp may read; its first feature
    const unsigned box0 = smem_u32(out_raw) + (unsigned)(warp - 2) * S::BUFFERS * S::OUT_BYTES;
    float *rows = row_raw + (warp - 2) * S::SHARE;
    int iter = 0;
    unsigned turn = 0;
    // The rows' scales, a tile ahead: from memory at each use they cost more than the rest of the epilogue.
    float next_x = 0.f, next_w[S::SHARE / 32];
    auto fetch = [&](int tile) {
      const int f0 = tile / tok_tiles * PR_FEATURES + from + lane, t0 = tile % tok_tiles * PR_TOKENS + (int)rank * 128 + quarter * 32 + lane;
      next_x = t0 < M ? x_row[t0] : 1.f;
#pragma unroll
      for (int i = 0; i < S::SHARE / 32; ++i) next_w[i] = f0 + i * 32 < N ? w_row[f0 + i * 32] : 1.f;
    };
    if (first < n_tiles) fetch(first);
    for (int tile = first; tile < n_tiles; tile += step, ++iter) {
      const int acc = iter & 1, f0 = tile / tok_tiles * PR_FEATURES + from;
      const int tok0 = tile % tok_tiles * PR_TOKENS + (int)rank * 128 + quarter * 32;
      const float rx = next_x;
      __syncwarp();
      bool near = near_one(rx);
#pragma unroll
      for (int i = 0; i < S::SHARE / 32; ++i) {
        near = near && near_one(next_w[i]);
        rows[i * 32 + lane] = next_w[i];
      }
      near = __all_sync(0xffffffffu, near);
      __syncwarp();
      if (tile + step < n_tiles) fetch(tile + step);
      if (!__all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * acc, (iter >> 1) & 1, abort_flag, status, 4))) break;
      tc_fence_after();
      const unsigned taddr = tmem_base + ((unsigned)(quarter * 32) << 16) + (unsigned)(acc * PR_FEATURES + from);
#pragma unroll 1
      for (int b = 0; b < S::BOXES; ++b) {
        const int s0 = b * S::BOX;
        const bool there = f0 + s0 < N && tok0 < M;
        constexpr int HALVES = S::BOX / 32, PIECE = 16 / (int)sizeof(TO);                 // 32 features at a time
        const bool last = b == S::BOXES - 1;
        const unsigned box = box0 + turn * S::OUT_BYTES;
        if (there) {
          if (lane == 0) {                     // the buffer's last store has read it: with two, the newest store reads the other one
            if (S::BUFFERS == 2) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            else asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          }
          __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          float a[16], c[16];
          if (there) {
            tc_ld16_issue(taddr + s0 + h * 32, a);
            tc_ld16_issue(taddr + s0 + h * 32 + 16, c);
            tc_ld_wait();
            tc_ld_ready(a);
            tc_ld_ready(c);
          }
          // The sums are in registers: the accumulator is free.  Where nobody waits for it this is left out: it takes half a microsecond (a fence over
          // the cluster), 5 % of a product of one round of tiles.
          if (last && h == HALVES - 1 && tile + 2 * step < n_tiles) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
              asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_cta(bar_tempty + 8 * acc, 0)) : "memory");
          }
          if (!there) continue;
          if (near) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 w = *reinterpret_cast<const float4 *>(rows + s0 + h * 32 + i), q = *reinterpret_cast<const float4 *>(rows + s0 + h * 32 + 16 + i);
              a[i] = a[i] * w.x * rx;
              a[i + 1] = a[i + 1] * w.y * rx;
              a[i + 2] = a[i + 2] * w.z * rx;
              a[i + 3] = a[i + 3] * w.w * rx;
              c[i] = c[i] * q.x * rx;
              c[i + 1] = c[i + 1] * q.y * rx;
              c[i + 2] = c[i + 2] * q.z * rx;
              c[i + 3] = c[i + 3] * q.w * rx;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              a[i] = scaled_far(a[i], rows[s0 + h * 32 + i], rx);
              c[i] = scaled_far(c[i], rows[s0 + h * 32 + 16 + i], rx);
            }
          }
#pragma unroll
          for (int i = 0; i < 16 / PIECE; ++i) {
            put_piece(box, lane, h * (32 / PIECE) + i, a + i * PIECE, TO());
            put_piece(box, lane, h * (32 / PIECE) + 16 / PIECE + i, c + i * PIECE, TO());
          }
        }
        if (!there) continue;
        // what hangs over the last column the lanes store, as they do all of a result whose rows do not start on 16 bytes: TMA would round its end
        // up to 16 bytes, into what is not ours
        if (by_tma && f0 + s0 + S::BOX <= N) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                         ::"l"(&map_out), "r"(f0 + s0), "r"(tok0), "r"(box) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          // Only a store that TMA reads takes its buffer away.  A box that is not there, or that the lanes store, commits no group: with a turn for
          // each of them the wait above would let the store out of this very buffer stay open.
          if (S::BUFFERS == 2) turn ^= 1;
        } else {
          __syncwarp();
          const TO *from_box = reinterpret_cast<const TO *>(out_raw + (box - smem_u32(out_raw)));
          const int n = min(N - f0 - s0, S::BOX), m = min(M - tok0, 32);
          TO *p = out + (size_t)tok0 * ldo + f0 + s0;
          if (by_tma) {                        // rows start on 16 bytes
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int t = i * 4 + lane / 8, at = lane % 8 * PIECE;
              const TO *q = from_box + t * S::BOX + (lane % 8 ^ (t & 7)) * PIECE;
              TO *to = p + t * ldo + at;
              if (t < m && at + PIECE <= n) *reinterpret_cast<float4 *>(to) = *reinterpret_cast<const float4 *>(q);
              else if (t < m)
                for (int k = 0; at + k < n; ++k) to[k] = q[k];
            }
          } else {
            for (int t = 0; t < m; ++t, p += ldo)
#pragma unroll
              for (int i = lane; i < S::BOX; i += 32)
                if (i < n) p[i] = from_box[t * S::BOX + ((i / PIECE ^ (t & 7)) * PIECE) + i % PIECE];
          }
          __syncwarp();
        }
      }
    }
    if (by_tma && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  // ---------------------------------------------------------------- teardown: neither CTA leaves while the other may signal it
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// A map over scales: rows of 512 bytes (a tile of 128 rows x 4 blocks), boxes of a stage's tiles, zeros behind the last.
int get_scale_map(const void *scales, long long rows, long long K, int format, CUtensorMap *out) {
  EncodeTiledFn fn = encode_fn();
  LLM_REQUIRE(fn != nullptr, "tensor map: the driver does not offer cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {128, (cuuint64_t)((rows + 127) / 128 * k_stages(K) * stage_tiles(format))};
  const cuuint64_t strides[1] = {SF_TILE};
  const cuuint32_t box[2] = {128, (cuuint32_t)stage_tiles(format)};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void *>(scales), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  LLM_REQUIRE(r == CUDA_SUCCESS, "tensor map: cuTensorMapEncodeTiled failed (%d) for scales of %lld x %lld", (int)r, rows, K);
  return LLM_OK;
}
// A map over the result: boxes of 32 rows of 128 bytes, swizzled (put_piece); rows behind the last are not stored.
int get_out_map(void *out, long long M, long long N, long long ldo, bool f32, CUtensorMap *map) {
  EncodeTiledFn fn = encode_fn();
  LLM_REQUIRE(fn != nullptr, "tensor map: the driver does not offer cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
  const cuuint64_t strides[1] = {(cuuint64_t)ldo * (f32 ? 4 : 2)};
  const cuuint32_t box[2] = {f32 ? 32u : 64u, 32};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = fn(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, out, dims, strides, box, elem,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  LLM_REQUIRE(r == CUDA_SUCCESS, "tensor map: cuTensorMapEncodeTiled failed (%d) for a result of %lld x %lld", (int)r, M, N);
  return LLM_OK;
}

template <int FORMAT, typename TO>
int launch_pair(const void *x_codes, const void *w_codes, const Fp4In &in, void *out, long long ldo, int M, int N, int K, int weights_first, int *status,
                cudaStream_t stream) {
  using S = PairShape<FORMAT, TO>;
  CUtensorMap map_x, map_w, map_xs, map_ws, map_out;
  const bool by_tma = (uintptr_t)out % 16 == 0 && ldo * (long long)sizeof(TO) % 16 == 0;
  int rc = get_code_map(x_codes, M, K, PR_TOKENS / 2, &map_x);
  if (rc == LLM_OK) rc = get_code_map(w_codes, N, K, PR_FEATURES / 2, &map_w);
  if (rc == LLM_OK) rc = get_scale_map(in.x_scales, M, K, FORMAT, &map_xs);
  if (rc == LLM_OK) rc = get_scale_map(in.w_scales, N, K, FORMAT, &map_ws);
  if (rc == LLM_OK && by_tma) rc = get_out_map(out, M, N, ldo, sizeof(TO) == 4, &map_out);
  if (rc != LLM_OK) return rc;
  if (!by_tma) map_out = map_x;                // not used
  const int tok_tiles = (M + PR_TOKENS - 1) / PR_TOKENS, feature_tiles = (N + PR_FEATURES - 1) / PR_FEATURES;
  const long long tiles = (long long)tok_tiles * feature_tiles;
  LLM_REQUIRE(tiles < (1ll << 30), "fp4_gemm: too many tiles");
  const int pairs = (int)(tiles < sm_count() / 2 ? tiles : sm_count() / 2);
  auto kern = fp4_pair_kernel<FORMAT, TO>;
  LLM_CHECK_CUDA(llm_allow_smem(kern, S::SMEM), "fp4_gemm attribute");
  LLM_CHECK_CUDA(llm_launch(kern, dim3(2 * pairs), dim3(S::THREADS), S::SMEM, stream, map_x, map_w, map_xs, map_ws, map_out, in.x_row, in.w_row, (TO *)out,
                            ldo, M, N, (int)k_stages(K), tok_tiles, feature_tiles, weights_first, by_tma ? 1 : 0, status),
                 "fp4_gemm launch");
  return LLM_OK;
}

template <int FORMAT, typename TO>
int dispatch_fp4(const void *x_codes, const void *w_codes, const Fp4In &in, void *out, long long ldo, int M, int N, int K, int weights_first,
                 int *status, cudaStream_t stream) {
#define FP4_GO(TN, PARTS) return launch_fp4<TN, FORMAT, TO>(x_codes, w_codes, in, out, ldo, M, N, K, PARTS, weights_first, status, stream)
  if (M <= 128) {
    const int parts = k_parts(M, N, K);
    if (M <= 16) FP4_GO(16, parts);
    if (M <= 32) FP4_GO(32, parts);
    if (M <= 64) FP4_GO(64, parts);
    FP4_GO(128, parts);
  }
  // Tiles of 128 features x 64 tokens where one to an SM is enough, else two SMs to a tile of 256 x 192 (2,048 features, K = 2,048: 256 tokens 5.8
  // against 7.1 us, 1,024 tokens 8.9 against 7.7; 16,384 features, 256 tokens: 14.5 against 12.2).
  if ((long long)((N + FP_ROWS - 1) / FP_ROWS) * ((M + 63) / 64) <= sm_count()) FP4_GO(64, 1);
  return launch_pair<FORMAT, TO>(x_codes, w_codes, in, out, ldo, M, N, K, weights_first, status, stream);
#undef FP4_GO
}

}  // namespace

LLM_EXPORT int llm_fp4_quantize(const Fp4QuantizeCall *call) {
  const Fp4QuantizeCall &c = *call;
  LLM_REQUIRE(c.rows >= 0 && c.cols > 0 && c.cols <= (1 << 28), "fp4_quantize: bad sizes %lld x %lld", c.rows, c.cols);
  LLM_REQUIRE(c.format == NVFP4 || c.format == MXFP4, "fp4_quantize: unknown format %lld", c.format);
  LLM_REQUIRE(((uintptr_t)c.codes | (uintptr_t)c.scales) % 16 == 0, "fp4_quantize: codes and scales must be 16-byte aligned");
  LLM_REQUIRE(c.dtype == LLM_F32 || c.dtype == LLM_BF16, "fp4_quantize: unknown dtype %lld", c.dtype);
  if (c.rows == 0) return LLM_OK;
  const Fp4Out o{(unsigned char *)c.codes, (unsigned char *)c.scales, c.row_scale, code_bytes(c.cols), k_stages(c.cols) * stage_tiles((int)c.format)};
#define FP4_ARGS c.x, c.ldx, o, c.rows, (int)c.cols, (cudaStream_t)c.stream
#define FP4_TYPE(T, FORMAT) return vec ? launch_quantize<T, FORMAT, true>(FP4_ARGS) : launch_quantize<T, FORMAT, false>(FP4_ARGS)
  const bool vec = ((uintptr_t)c.x | (unsigned long long)c.ldx * (c.dtype == LLM_F32 ? 4 : 2)) % 16 == 0;
  if (c.dtype == LLM_F32) {
    if (c.format == NVFP4) FP4_TYPE(float, NVFP4);
    FP4_TYPE(float, MXFP4);
  }
  if (c.format == NVFP4) FP4_TYPE(__nv_bfloat16, NVFP4);
  FP4_TYPE(__nv_bfloat16, MXFP4);
#undef FP4_TYPE
#undef FP4_ARGS
}

LLM_EXPORT int llm_fp4_dequantize(const Fp4DequantizeCall *call) {
  const Fp4DequantizeCall &c = *call;
  LLM_REQUIRE(c.rows >= 0 && c.cols > 0 && c.cols <= (1 << 28), "fp4_dequantize: bad sizes %lld x %lld", c.rows, c.cols);
  LLM_REQUIRE(c.format == NVFP4 || c.format == MXFP4, "fp4_dequantize: unknown format %lld", c.format);
  LLM_REQUIRE(((uintptr_t)c.codes | (uintptr_t)c.scales) % 16 == 0, "fp4_dequantize: codes and scales must be 16-byte aligned");
  LLM_REQUIRE(c.dtype == LLM_F32 || c.dtype == LLM_BF16, "fp4_dequantize: unknown dtype %lld", c.dtype);
  if (c.rows == 0) return LLM_OK;
  if (c.dtype == LLM_F32) return c.format == NVFP4 ? dispatch_dequantize<float, NVFP4>(c) : dispatch_dequantize<float, MXFP4>(c);
  return c.format == NVFP4 ? dispatch_dequantize<__nv_bfloat16, NVFP4>(c) : dispatch_dequantize<__nv_bfloat16, MXFP4>(c);
}

LLM_EXPORT int llm_fp4_gemm(const Fp4GemmCall *call) {
  const Fp4GemmCall &c = *call;
  LLM_REQUIRE(c.M >= 0 && c.N >= 0 && c.M < (1 << 30) && c.N < (1 << 30) && c.K > 0 && c.K <= (1 << 28), "fp4_gemm: bad sizes %lld x %lld x %lld", c.M,
              c.N, c.K);
  LLM_REQUIRE(c.format == NVFP4 || c.format == MXFP4, "fp4_gemm: unknown format %lld", c.format);
  LLM_REQUIRE(c.out_dtype == LLM_F32 || c.out_dtype == LLM_BF16, "fp4_gemm: unknown output dtype %lld", c.out_dtype);
  LLM_REQUIRE(((uintptr_t)c.x_codes | (uintptr_t)c.x_scales | (uintptr_t)c.w_codes | (uintptr_t)c.w_scales) % 16 == 0,
              "fp4_gemm: operands must be 16-byte aligned");
  if (c.M == 0 || c.N == 0) return LLM_OK;
  const Fp4In in{(const unsigned char *)c.x_scales, (const unsigned char *)c.w_scales, c.x_row, c.w_row};
#define FP4_ARGS c.x_codes, c.w_codes, in, c.out, c.ldo, (int)c.M, (int)c.N, (int)c.K, c.weights_first != 0, c.status, (cudaStream_t)c.stream
  if (c.format == NVFP4) return c.out_dtype == LLM_F32 ? dispatch_fp4<NVFP4, float>(FP4_ARGS) : dispatch_fp4<NVFP4, __nv_bfloat16>(FP4_ARGS);
  return c.out_dtype == LLM_F32 ? dispatch_fp4<MXFP4, float>(FP4_ARGS) : dispatch_fp4<MXFP4, __nv_bfloat16>(FP4_ARGS);
#undef FP4_ARGS
}
