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
// 16 values of a row as they lie in memory
template <typename T>
struct Unit;
template <>
struct Unit<__nv_bfloat16> {
  uint4 raw[2];
  __device__ __forceinline__ void load(const __nv_bfloat16 *p) {
    raw[0] = reinterpret_cast<const uint4 *>(p)[0];
    raw[1] = reinterpret_cast<const uint4 *>(p)[1];
  }
  __device__ __forceinline__ void gather(const __nv_bfloat16 *p, int n) {
    unsigned w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned lo = 2 * i < n ? __bfloat16_as_ushort(p[2 * i]) : 0, hi = 2 * i + 1 < n ? __bfloat16_as_ushort(p[2 * i + 1]) : 0;
      w[i] = lo | hi << 16;
    }
    raw[0] = make_uint4(w[0], w[1], w[2], w[3]);
    raw[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
  __device__ __forceinline__ void values(float (&v)[UNIT]) const {
    const unsigned w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <>
struct Unit<float> {
  float4 raw[4];
  __device__ __forceinline__ void load(const float *p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = reinterpret_cast<const float4 *>(p)[i];
  }
  __device__ __forceinline__ void gather(const float *p, int n) {
    float v[UNIT];
#pragma unroll
    for (int i = 0; i < UNIT; ++i) v[i] = i < n ? p[i] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  }
  __device__ __forceinline__ void values(float (&v)[UNIT]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[4 * i] = raw[i].x;
      v[4 * i + 1] = raw[i].y;
      v[4 * i + 2] = raw[i].z;
      v[4 * i + 3] = raw[i].w;
    }
  }
};

template <typename T>
__device__ __forceinline__ Unit<T> fetch_unit(const T *row, int u, int K, bool vec) {
  Unit<T> x;
  if (vec && (u + 1) * UNIT <= K) x.load(row + u * UNIT);
  else x.gather(row + u * UNIT, K - u * UNIT);
  return x;
}

// The largest magnitude's bits: as integers they are in the order of the values, and every infinity and NaN is 0x7f800000 or more.
template <typename T>
__device__ __forceinline__ unsigned top_bits(const Unit<T> &x) {
  float v[UNIT];
  x.values(v);
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < UNIT; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  return top;
}

__device__ __forceinline__ unsigned pack_codes(const float *v) {      // eight values, the first in the lowest four bits
  unsigned r;
  asm("{\n.reg .b8 a, b, c, d;\n"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      "mov.b32 %0, {a, b, c, d};\n}"
      : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }        // -126 .. 127

// The row's scale of nvfp4, from its largest magnitude's bits: its exponent.
__device__ __forceinline__ int row_exponent(unsigned top) { return top == 0 ? 0 : max((int)(top >> 23) - 137, -126); }

__device__ __forceinline__ float e4m3_value(unsigned byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}

// The scale byte of a block whose largest magnitude has the bits `top`, and 16 of its values as codes.
//
// nvfp4: value / row scale is exact.  The quotient by the block's scale s may be rounded before it is rounded to a code, but not across a
// halfway point t: for 32-bit values the division's own rounding keeps the two apart (value and s t are 32-bit numbers, so they
// differ by a step of theirs, more than half a step of the quotient).  A bfloat16 value (8 bits) and s t (4 + 3 bits) differ by 2^-8 or
// are equal, so that value * (1 / s), off by 2^-23, rounded to 12 bits, is t exactly where the quotient is and on its side of t elsewhere.
template <typename T, int FORMAT>
__device__ __forceinline__ unsigned scale_byte(unsigned top, int row_e) {
  if (FORMAT == MXFP4) return top == 0 ? 0u : (unsigned)min(max((int)(top >> 23) - 2, 0), 254);
  const float wanted = __fdiv_rn(__uint_as_float(top) * power_of_two(-row_e), 6.f);
  const unsigned byte = __nv_cvt_float_to_fp8(wanted, __NV_SATFINITE, __NV_E4M3);
  return top == 0 ? 0u : max(byte, 1u);
}
template <typename T, int FORMAT>
__device__ __forceinline__ uint2 unit_codes(const Unit<T> &x, unsigned byte, int row_e) {
  float v[UNIT];
  x.values(v);
  if (FORMAT == MXFP4) {
    const float up = power_of_two(127 - (int)byte);
#pragma unroll
    for (int i = 0; i < UNIT; ++i) v[i] *= up;
  } else {
    const float up = power_of_two(-row_e), s = e4m3_value(byte), inv = byte == 0 ? 0.f : __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < UNIT; ++i) {
      const float y = v[i] * up;
      if (sizeof(T) == 4) v[i] = byte == 0 ? 0.f : __fdiv_rn(y, s);
      else v[i] = __uint_as_float((__float_as_uint(y * inv) + 0x800u) & 0xfffff000u);
    }
  }
  return make_uint2(pack_codes(v), pack_codes(v + 8));
}

struct Fp4Out {
  unsigned char *codes, *scales;
  float *row_scale;
  long long ldc;                // bytes of a row of codes
  long long sf_tiles;           // scale tiles of 128 rows along K
};

// Stores a unit's codes and, once per four blocks, their scales.  All lanes of the warp take part; `there`: the unit is one of the row's
// (of whole stages of 256).
template <int FORMAT>
__device__ __forceinline__ void store_unit(const Fp4Out &o, long long row, int u, bool there, uint2 codes, unsigned byte) {
  if (there && u * 8 < o.ldc) *reinterpret_cast<uint2 *>(o.codes + row * o.ldc + u * 8) = codes;
  constexpr int NEXT = FORMAT == NVFP4 ? 1 : 2, PER = 4 * NEXT;       // lanes to a block; units to four blocks
  unsigned w = byte | __shfl_xor_sync(0xffffffffu, byte, NEXT) << 8;
  w |= __shfl_xor_sync(0xffffffffu, w, 2 * NEXT) << 16;
  if (there && u % PER == 0)
    *reinterpret_cast<unsigned *>(o.scales + ((row >> 7) * o.sf_tiles + u / PER) * SF_TILE + (row & 31) * 16 + (row >> 5 & 3) * 4) = w;
}

// A group of G threads to a row (a warp, or the whole block), `HELD` units of a row in each thread's registers between the row's
// maximum and the codes; longer rows (HELD = 0) are read twice.
template <typename T, int FORMAT, int G, int HELD>
__global__ void __launch_bounds__(G == 32 ? 128 : G)
fp4_quantize_kernel(const T *x, long long ldx, Fp4Out o, long long rows, int K, int n_units, int vec) {
  grid_dependents_launch();
  grid_dependency_wait();
  __shared__ unsigned tops[32];
  const int t = threadIdx.x % G;
  const long long row = G == 32 ? (long long)blockIdx.x * 4 + threadIdx.x / 32 : blockIdx.x;
  if (row >= rows) return;                     // a whole group: no barrier behind it where G is a warp
  const T *r = x + row * ldx;
  Unit<T> held[HELD ? HELD : 1];
  unsigned tu[HELD ? HELD : 1], top = 0;
  if (HELD) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      held[i] = fetch_unit(r, t + i * G, K, vec);
      tu[i] = top_bits(held[i]);
      top = max(top, tu[i]);
    }
  } else {
    for (int u = t; u < n_units; u += G) top = max(top, top_bits(fetch_unit(r, u, K, vec)));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (G > 32) {
    if (t % 32 == 0) tops[t / 32] = top;
    __syncthreads();
    for (int w = 0; w < G / 32; ++w) top = max(top, tops[w]);
  }
  const int row_e = FORMAT == NVFP4 ? row_exponent(top) : 0;
  if (t == 0) o.row_scale[row] = top >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : power_of_two(row_e);
  auto put = [&](int u, const Unit<T> &v, unsigned unit_top) {
    if (FORMAT == MXFP4) unit_top = max(unit_top, __shfl_xor_sync(0xffffffffu, unit_top, 1));
    const unsigned byte = scale_byte<T, FORMAT>(unit_top, row_e);
    store_unit<FORMAT>(o, row, u, u < n_units, unit_codes<T, FORMAT>(v, byte, row_e), byte);
  };
  if (HELD) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) put(t + i * G, held[i], tu[i]);
  } else {
    for (int u = t; u < (n_units + 31) / 32 * 32; u += G) {
      const Unit<T> v = fetch_unit(r, u, K, vec);
      put(u, v, top_bits(v));
    }
  }
}

template <typename T, int FORMAT>
int launch_quantize(const void *x, long long ldx, const Fp4Out &o, long long rows, int K, cudaStream_t stream) {
  const int n_units = (int)(k_stages(K) * (STAGE_K / UNIT));
  const int vec = (uintptr_t)x % 16 == 0 && ldx * (long long)sizeof(T) % 16 == 0;
#define FP4_GO(G, HELD)                                                                                                                   \
  do {                                                                                                                                    \
    const long long blocks = G == 32 ? (rows + 3) / 4 : rows;                                                                            \
    LLM_REQUIRE(blocks < (1ll << 31), "fp4_quantize: too many rows");                                                                    \
    LLM_CHECK_CUDA(llm_launch(fp4_quantize_kernel<T, FORMAT, G, HELD>, dim3((unsigned)blocks), dim3(G == 32 ? 128 : G), 0, stream,       \
                              (const T *)x, ldx, o, rows, K, n_units, vec), "fp4_quantize launch");                                      \
    return LLM_OK;                                                                                                                        \
  } while (0)
  if (n_units <= 32) FP4_GO(32, 1);
  if (n_units <= 64) FP4_GO(32, 2);
  if (n_units <= 128) FP4_GO(32, 4);
  if (n_units <= 256) FP4_GO(256, 1);
  if (n_units <= 512) FP4_GO(256, 2);
  if (n_units <= 1024) FP4_GO(256, 4);
  FP4_GO(256, 0);
#undef FP4_GO
}

// ---------------------------------------------------------------- back
__device__ __forceinline__ float scale_value(int format, unsigned byte) {
  if (format == NVFP4) return e4m3_value(byte & 0x7f);
  return byte == 0 ? __uint_as_float(0x00400000u) : byte == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte << 23);
}

template <typename TO>
__global__ void __launch_bounds__(256)
fp4_dequantize_kernel(const unsigned char *codes, const unsigned char *scales, const float *row_scale, TO *out, long long ldo, long long rows,
                      int K, int format, long long ldc, long long sf_tiles, int vec) {
  grid_dependents_launch();
  grid_dependency_wait();
  const int per_row = (K + UNIT - 1) / UNIT;
  const long long n = rows * per_row;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long row = i / per_row;
    const int u = (int)(i - row * per_row), block = format == NVFP4 ? u : u / 2;
    const uint2 c = *reinterpret_cast<const uint2 *>(codes + row * ldc + u * 8);
    const unsigned byte = scales[((row >> 7) * sf_tiles + block / 4) * SF_TILE + (row & 31) * 16 + (row >> 5 & 3) * 4 + block % 4];
    const float s = scale_value(format, byte), rs = row_scale[row];
    float v[UNIT];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned two = (j < 4 ? c.x >> 8 * j : c.y >> 8 * (j - 4)) & 0xff;
      const float2 f = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)two, __NV_E2M1)));
      v[2 * j] = f.x * s * rs;
      v[2 * j + 1] = f.y * s * rs;
    }
    TO *p = out + row * ldo + u * UNIT;
    if (vec && (u + 1) * UNIT <= K) {
#pragma unroll
      for (int j = 0; j < UNIT; j += 4) st4(p + j, make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
    } else {
#pragma unroll
      for (int j = 0; j < UNIT; ++j)
        if (u * UNIT + j < K) p[j] = from_float<TO>(v[j]);
    }
  }
}

// ---------------------------------------------------------------- the product
// out[t, n] = Rx[t] Rw[n] sum over blocks b of sx[t, b] sw[n, b] sum over k of b of cx[t, k] cw[n, k]: tcgen05.mma with block scales takes codes
// from shared memory and scales from tensor memory and adds in 32 bits; the rows' scales are the epilogue's.
//
// The structure is gemm_tc.cu's: W's rows are the instruction's 128 rows, the tokens its N (16 to 192); a persistent CTA to an SM with a
// loader, an issuer and four epilogue warps, a ring of stages of 256 of K, two accumulators.  With the codes of a stage come its scales,
// as they lie in memory; the issuer has them copied to tensor memory (tcgen05.cp, in order with the products that read
// them) in two places in turn, behind the accumulators.
constexpr int FP_THREADS = 192;
constexpr int FP_ROWS = 128;

template <int TN, int FORMAT>
struct FpShape {
  static constexpr int TILES = stage_tiles(FORMAT);                       // scale tiles of 128 rows in a stage
  static constexpr int A_BYTES = FP_ROWS * 128, B_BYTES = TN * 128;
  static constexpr int SF_BYTES = TILES * SF_TILE;                        // of 128 rows
  static constexpr int B_PARTS = TN > 128 ? 2 : 1;                        // row tiles of scales that a tile of tokens touches
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + (1 + B_PARTS) * SF_BYTES;
  static constexpr int STAGES = 190 * 1024 / STAGE_BYTES;
  static constexpr int SF_COLS = TILES * 4 * (1 + B_PARTS);               // columns of tensor memory of a stage's scales
  static constexpr int COLS = 2 * TN + 2 * SF_COLS;
  static constexpr int TMEM_COLS = COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE_BYTES + 512;
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

struct Fp4In {
  const unsigned char *x_scales, *w_scales;
  const float *x_row, *w_row;
};

template <int TN, int FORMAT, typename TO>
__global__ void __launch_bounds__(FP_THREADS, 1)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, Fp4In in, TO *out, long long ldo, int M, int N,
                int n_stages, int row_tiles, int tok_tiles, int weights_first, int *status) {
  using S = FpShape<TN, FORMAT>;
  constexpr int STAGES = S::STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned long long *bars = (unsigned long long *)(smem + (size_t)STAGES * S::STAGE_BYTES);
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
  const int n_tiles = row_tiles * tok_tiles;
  const long long sf_row_tile = (long long)n_stages * S::SF_BYTES;        // bytes of 128 rows' scales
  const int x_row_tiles = (M + 127) / 128;

  if (warp == 0) {
    // ------------------------------------------------------------ loader
    const bool leader = elect_one();
    struct Walk {
      int tile, kb;
      bool valid;
    };
    auto next = [&](Walk &w) {
      if (++w.kb >= n_stages) {
        w.kb = 0;
        w.tile += gridDim.x;
        w.valid = w.tile < n_tiles;
      }
    };
    // how many row tiles of scales this tile's tokens lie in
    auto x_parts = [&](int tok0) { return S::B_PARTS == 2 && tok0 / 128 + 1 < x_row_tiles ? 2 : 1; };
    auto load_w = [&](const Walk &w, int stage) {
      if (!leader) return;
      const unsigned dst = smem_u32(smem + (size_t)stage * S::STAGE_BYTES), bar = bar_full + 8 * stage;
      const int row_tile = w.tile / tok_tiles, tok0 = w.tile % tok_tiles * TN;
      mbar_expect_tx(bar, S::A_BYTES + S::B_BYTES + (1 + x_parts(tok0)) * S::SF_BYTES);
      tma_load_2d(dst, &map_w, w.kb * 128, row_tile * FP_ROWS, bar);
      bulk_load(dst + S::A_BYTES + S::B_BYTES, in.w_scales + row_tile * sf_row_tile + (long long)w.kb * S::SF_BYTES, S::SF_BYTES, bar);
    };
    auto load_x = [&](const Walk &w, int stage) {
      if (!leader) return;
      const unsigned dst = smem_u32(smem + (size_t)stage * S::STAGE_BYTES), bar = bar_full + 8 * stage;
      const int tok0 = w.tile % tok_tiles * TN;
      tma_load_2d(dst + S::A_BYTES, &map_x, w.kb * 128, tok0, bar);
      for (int p = 0; p < x_parts(tok0); ++p)
        bulk_load(dst + S::A_BYTES + S::B_BYTES + (1 + p) * S::SF_BYTES, in.x_scales + (tok0 / 128 + p) * sf_row_tile + (long long)w.kb * S::SF_BYTES,
                  S::SF_BYTES, bar);
    };
    Walk w{(int)blockIdx.x, 0, (int)blockIdx.x < n_tiles}, w2 = w;
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
    unsigned phase = 0, turn = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x, ++iter) {
      const int acc = iter & 1, tok0 = tile % tok_tiles * TN;
      const int x_parts = S::B_PARTS == 2 && tok0 / 128 + 1 < x_row_tiles ? 2 : 1;
      const unsigned shift = (unsigned)(tok0 % 128 / 32);                 // a tile of 192 tokens may start in the middle of a scale tile
      ok = __all_sync(0xffffffffu, mbar_wait(bar_tempty + 8 * acc, ((iter >> 1) & 1) ^ 1, abort_flag, status, 2));
      if (!ok) break;
      tc_fence_after();
      const unsigned d_tmem = tmem_base + acc * TN;
      for (int kb = 0; kb < n_stages; ++kb, turn ^= 1) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_full + 8 * stage, phase, abort_flag, status, 3));
        if (!ok) break;
        tc_fence_after();
        const unsigned a_addr = smem_u32(smem + (size_t)stage * S::STAGE_BYTES);
        const unsigned long long a_desc = smem_desc(a_addr), b_desc = smem_desc(a_addr + S::A_BYTES);
        const unsigned sf = a_addr + S::A_BYTES + S::B_BYTES;
        const unsigned sfa = tmem_base + 2 * TN + turn * S::SF_COLS, sfb = sfa + S::TILES * 4;
        if (leader) {
#pragma unroll
          for (int j = 0; j < S::TILES; ++j) {
            scales_to_tmem(sfa + j * 4, sf + j * SF_TILE);
            scales_to_tmem(sfb + j * 4 * S::B_PARTS, sf + S::SF_BYTES + j * SF_TILE);
            if (S::B_PARTS == 2 && x_parts == 2) scales_to_tmem(sfb + j * 8 + 4, sf + 2 * S::SF_BYTES + j * SF_TILE);
          }
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {           // 64 of K = 32 bytes further along the swizzled row
            const int j = kk * S::TILES / 4, first = FORMAT == NVFP4 ? 0 : kk % 2 * 2;
            fp4_mma<FORMAT>(d_tmem, a_desc + (unsigned long long)(kk * 2), b_desc + (unsigned long long)(kk * 2),
                            fp4_instr(FORMAT, FP_ROWS, TN, first), sfa + j * 4, sfb + j * 4 * S::B_PARTS + shift, kk > 0 || kb > 0 ? 1u : 0u);
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
    for (int tile = blockIdx.x; tile < n_tiles; tile += gridDim.x, ++iter) {
      const int acc = iter & 1, tok0 = tile % tok_tiles * TN, f = tile / tok_tiles * FP_ROWS + quarter * 32 + lane;
      const float rw = f < N ? in.w_row[f] : 0.f;
      if (!__all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * acc, (iter >> 1) & 1, abort_flag, status, 4))) break;
      tc_fence_after();
#pragma unroll 1
      for (int c0 = 0; c0 < TN && tok0 + c0 < M; c0 += 16) {
        float v[16];
        tc_ld16(tmem_base + ((unsigned)(quarter * 32) << 16) + (unsigned)(acc * TN + c0), v);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int tok = tok0 + c0 + i;
          if (f < N && tok < M) out[(size_t)tok * ldo + f] = from_float<TO>(v[i] * rw * in.x_row[tok]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_tempty + 8 * acc);
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

template <int TN, int FORMAT, typename TO>
int launch_fp4(const void *x_codes, const void *w_codes, const Fp4In &in, void *out, long long ldo, int M, int N, int K, int weights_first, int *status,
               cudaStream_t stream) {
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
  const int grid = (int)(tiles < sm_count() ? tiles : sm_count());
  LLM_CHECK_CUDA(llm_launch(kern, dim3(grid), dim3(FP_THREADS), S::SMEM, stream, map_w, map_x, in, (TO *)out, ldo, M, N, (int)k_stages(K), row_tiles,
                            tok_tiles, weights_first, status),
                 "fp4_gemm launch");
  return LLM_OK;
}

template <int FORMAT, typename TO>
int dispatch_fp4(const void *x_codes, const void *w_codes, const Fp4In &in, void *out, long long ldo, int M, int N, int K, int weights_first,
                 int *status, cudaStream_t stream) {
#define FP4_GO(TN) return launch_fp4<TN, FORMAT, TO>(x_codes, w_codes, in, out, ldo, M, N, K, weights_first, status, stream)
  if (M <= 16) FP4_GO(16);
  if (M <= 32) FP4_GO(32);
  if (M <= 64) FP4_GO(64);
  if (M <= 128) FP4_GO(128);
  FP4_GO(192);
#undef FP4_GO
}

}  // namespace

// x [rows, cols] of `dtype`, row stride ldx (elements) -> codes, scales and row scales as they are laid out above.
LLM_EXPORT int llm_fp4_quantize(int dtype, const void *x, long long ldx, void *codes, void *scales, float *row_scale, long long rows, int cols,
                                int format, cudaStream_t stream) {
  LLM_REQUIRE(rows >= 0 && cols > 0 && cols <= (1 << 28), "fp4_quantize: bad sizes %lld x %d", rows, cols);
  LLM_REQUIRE(format == NVFP4 || format == MXFP4, "fp4_quantize: unknown format %d", format);
  LLM_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, "fp4_quantize: codes and scales must be 16-byte aligned");
  LLM_REQUIRE(dtype == LLM_F32 || dtype == LLM_BF16, "fp4_quantize: unknown dtype %d", dtype);
  if (rows == 0) return LLM_OK;
  const Fp4Out o{(unsigned char *)codes, (unsigned char *)scales, row_scale, code_bytes(cols), k_stages(cols) * stage_tiles(format)};
  if (dtype == LLM_F32)
    return format == NVFP4 ? launch_quantize<float, NVFP4>(x, ldx, o, rows, cols, stream) : launch_quantize<float, MXFP4>(x, ldx, o, rows, cols, stream);
  return format == NVFP4 ? launch_quantize<__nv_bfloat16, NVFP4>(x, ldx, o, rows, cols, stream)
                         : launch_quantize<__nv_bfloat16, MXFP4>(x, ldx, o, rows, cols, stream);
}

LLM_EXPORT int llm_fp4_dequantize(const void *codes, const void *scales, const float *row_scale, int dtype, void *out, long long ldo, long long rows,
                                  int cols, int format, cudaStream_t stream) {
  LLM_REQUIRE(rows >= 0 && cols > 0 && cols <= (1 << 28), "fp4_dequantize: bad sizes %lld x %d", rows, cols);
  LLM_REQUIRE(format == NVFP4 || format == MXFP4, "fp4_dequantize: unknown format %d", format);
  LLM_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, "fp4_dequantize: codes and scales must be 16-byte aligned");
  LLM_REQUIRE(dtype == LLM_F32 || dtype == LLM_BF16, "fp4_dequantize: unknown dtype %d", dtype);
  if (rows == 0) return LLM_OK;
  const long long units = rows * ((cols + UNIT - 1) / UNIT), blocks = (units + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 8ll * sm_count() * 4 ? blocks : 8ll * sm_count() * 4);
  const long long ldc = code_bytes(cols), tiles = k_stages(cols) * stage_tiles(format);
  const int vec = (uintptr_t)out % 16 == 0 && ldo % 4 == 0;
  if (dtype == LLM_F32)
    LLM_CHECK_CUDA(llm_launch(fp4_dequantize_kernel<float>, dim3(grid), dim3(256), 0, stream, (const unsigned char *)codes, (const unsigned char *)scales,
                              row_scale, (float *)out, ldo, rows, cols, format, ldc, tiles, vec), "fp4_dequantize launch");
  else
    LLM_CHECK_CUDA(llm_launch(fp4_dequantize_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, stream, (const unsigned char *)codes,
                              (const unsigned char *)scales, row_scale, (__nv_bfloat16 *)out, ldo, rows, cols, format, ldc, tiles, vec),
                   "fp4_dequantize launch");
  return LLM_OK;
}

// out [M, N] (row stride ldo) = x [M, K] w [N, K]^T, both in `format`.  `weights_first`: w was complete before the kernel in front of this one in
// the stream could start (a matrix that is held), and may be read while that one still runs.
LLM_EXPORT int llm_fp4_gemm(const void *x_codes, const void *x_scales, const float *x_row, const void *w_codes, const void *w_scales, const float *w_row,
                            int out_dtype, void *out, long long ldo, int M, int N, int K, int format, int weights_first, int *status,
                            cudaStream_t stream) {
  LLM_REQUIRE(M >= 0 && N >= 0 && K > 0 && K <= (1 << 28), "fp4_gemm: bad sizes %d x %d x %d", M, N, K);
  LLM_REQUIRE(format == NVFP4 || format == MXFP4, "fp4_gemm: unknown format %d", format);
  LLM_REQUIRE(out_dtype == LLM_F32 || out_dtype == LLM_BF16, "fp4_gemm: unknown output dtype %d", out_dtype);
  LLM_REQUIRE(((uintptr_t)x_codes | (uintptr_t)x_scales | (uintptr_t)w_codes | (uintptr_t)w_scales) % 16 == 0, "fp4_gemm: operands must be 16-byte aligned");
  if (M == 0 || N == 0) return LLM_OK;
  const Fp4In in{(const unsigned char *)x_scales, (const unsigned char *)w_scales, x_row, w_row};
#define FP4_ARGS x_codes, w_codes, in, out, ldo, M, N, K, weights_first, status, stream
  if (format == NVFP4) return out_dtype == LLM_F32 ? dispatch_fp4<NVFP4, float>(FP4_ARGS) : dispatch_fp4<NVFP4, __nv_bfloat16>(FP4_ARGS);
  return out_dtype == LLM_F32 ? dispatch_fp4<MXFP4, float>(FP4_ARGS) : dispatch_fp4<MXFP4, __nv_bfloat16>(FP4_ARGS);
#undef FP4_ARGS
}
