// Microscaled 4-bit tables: quantisation, its inverse, and the product of two packed tables on the matrix cores.
//
// A row is cut into blocks of 32 values that share a power of two s = 2^E, E = clamp(floor(log2(max |v|)) - 2, -127, 127);
// a value is held as the nearest of +-{0, .5, 1, 1.5, 2, 3, 4, 6} to v / s (ties to the even code, larger ones to 6): four
// bits (sign, two exponent bits, one mantissa bit), the lower of two columns in the low nibble.  E + 127 is a byte; 255 marks
// a block that held an infinity or NaN: all its values read as NaN.  Rows are padded with zeros to a multiple of 128 columns
// (64 bytes of codes, one dword of scales), so the product has no tail in its inner dimension.
//
// Dividing by s only moves the exponent, so quantisation has one rounding and is the same whatever the input's type.
#include "rowtypes.h"

namespace bkg {

constexpr int MX_K = 128;                       // columns a row is padded to a multiple of

typedef int mx_i32x8 __attribute__((ext_vector_type(8)));
typedef float mx_f32x16 __attribute__((ext_vector_type(16)));

// ---- 8 values of a row per lane, 4 lanes per block: 16-byte loads of a bf16 / fp16 row, a dword of codes out.
// ALIGNED: the rows' 8-value pieces are 16-byte aligned (fp32: two accesses).
template <typename T, bool ALIGNED>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int cols,
                                                           int pieces, uint32_t* __restrict__ codes,
                                                           uint32_t* __restrict__ scales) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = at / pieces;
  const int piece = (int)(at - row * pieces), c = piece * 8;
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = 0.f;
  if (row < rows) {
    const T* p = x + row * ldx + c;
    if (ALIGNED && c + 8 <= cols) {
      constexpr int N = 16 / sizeof(T);
#pragma unroll
      for (int h = 0; h < 8 / N; ++h) {
        const Pack<T, N> v = reinterpret_cast<const Pack<T, N>*>(p)[h];
#pragma unroll
        for (int j = 0; j < N; ++j) f[h * N + j] = widen(v.v[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < cols) f[j] = widen(p[j]);
    }
  }
  uint32_t top = 0;                             // largest magnitude's bits (infinities and NaN are the largest)
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
  const uint32_t field = top >> 23;             // floor(log2) + 127; 0 for zeros and denormals: their E is clamped anyway
  const uint32_t byte = field == 255u ? 255u : (field > 2u ? field - 2u : 0u);
  const float inv = __uint_as_float((254u - byte) << 23);               // 2^-E (255: unused)
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[0] * inv, f[1] * inv, 1.0f, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[2] * inv, f[3] * inv, 1.0f, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[4] * inv, f[5] * inv, 1.0f, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[6] * inv, f[7] * inv, 1.0f, 3);
  if (byte == 255u) q = 0;
  const uint32_t b1 = __shfl_down((int)byte, 4, 64), b2 = __shfl_down((int)byte, 8, 64), b3 = __shfl_down((int)byte, 12, 64);
  if (row < rows) {
    codes[row * pieces + piece] = q;
    if ((piece & 15) == 0) scales[row * (pieces >> 4) + (piece >> 4)] = byte | (b1 << 8) | (b2 << 16) | (b3 << 24);
  }
}

__device__ __forceinline__ float mx4_value(uint32_t code, int e, bool bad) {
  const uint32_t m = code & 7u;                 // 0 .5 1 1.5 2 3 4 6
  const float a = m < 2 ? 0.5f * m : ldexpf(1.f + 0.5f * (m & 1u), (int)(m >> 1) - 1);
  const float v = ldexpf(a, e);
  return bad ? __uint_as_float(0x7fc00000u) : (code & 8u) ? -v : v;
}

template <typename T, bool ALIGNED>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                             const unsigned char* __restrict__ scales, int64_t rows, int cols,
                                                             int pieces, T* __restrict__ out, int64_t ldo) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = at / pieces;
  if (row >= rows) return;
  const int piece = (int)(at - row * pieces), c = piece * 8;
  if (c >= cols) return;
  const uint32_t q = codes[row * pieces + piece];
  const int byte = scales[row * (pieces >> 2) + (piece >> 2)], e = byte - 127;
  T* p = out + row * ldo + c;
  T v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (T)mx4_value(q >> (4 * j), e, byte == 255);
  if (ALIGNED && c + 8 <= cols) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 8 / N; ++h) {
      Pack<T, N> o;
#pragma unroll
      for (int j = 0; j < N; ++j) o.v[j] = v[h * N + j];
      reinterpret_cast<Pack<T, N>*>(p)[h] = o;
    }
  } else {
    for (int j = 0; j < 8 && c + j < cols; ++j) p[j] = v[j];
  }
}

// ---- out[m, n] = sum_k A[m, k] B[n, k] (+ bias[n]).  v_mfma_scale_f32_32x32x64_f8f6f4: lane l holds 32 columns (16 bytes)
// of row l % 32, block l / 32, and that block's scale byte; the result's column is B's row l % 32.
struct Mx4Args {
  const uint32_t* ca; const uint32_t* sa; int64_t m;
  const uint32_t* cb; const uint32_t* sb; int64_t n;
  int steps;                                     // inner dimension / 128
  const float* bias;
  void* out; int64_t ldo;
};

__device__ __forceinline__ mx_i32x8 mx_operand(uint4 v) {
  return mx_i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_matmul_kernel(const Mx4Args a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, half = lane >> 5;
  const int64_t m0 = (int64_t)blockIdx.x * 128 + (wave & 1) * 64, n0 = (int64_t)blockIdx.y * 128 + (wave >> 1) * 64;
  const int pitch = a.steps * 16;                // dwords of codes per row
  mx_f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  int64_t ra[2], rb[2];                          // (rows behind the last one read the last one; their results are dropped)
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    ra[i] = min(m0 + i * 32 + l31, a.m - 1);
    rb[i] = min(n0 + i * 32 + l31, a.n - 1);
  }
  for (int st = 0; st < a.steps; ++st) {
    uint4 va[2][2], vb[2][2];
    uint32_t xa[2], xb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      xa[i] = a.sa[ra[i] * a.steps + st] >> (8 * half);
      xb[i] = a.sb[rb[i] * a.steps + st] >> (8 * half);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        va[i][h] = *reinterpret_cast<const uint4*>(a.ca + ra[i] * pitch + st * 16 + 8 * h + 4 * half);
        vb[i][h] = *reinterpret_cast<const uint4*>(a.cb + rb[i] * pitch + st * 16 + 8 * h + 4 * half);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(va[i][0]), mx_operand(vb[j][0]), acc[i][j], 4, 4,
                                                                    0, (int)xa[i], 0, (int)xb[j]);
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(va[i][1]), mx_operand(vb[j][1]), acc[i][j], 4, 4,
                                                                    2, (int)xa[i], 2, (int)xb[j]);
      }
  }
  T* out = (T*)a.out;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t n = n0 + j * 32 + l31;
    if (n >= a.n) continue;
    const float b = a.bias ? a.bias[n] : 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t m = m0 + i * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
        if (m < a.m) out[m * a.ldo + n] = (T)(acc[i][j][r] + b);
      }
  }
}

static int64_t mx4_steps(int64_t cols) { return (cols + MX_K - 1) / MX_K; }

}  // namespace bkg

using namespace bkg;

#define BKG_BY_TYPE(type, CALL)                          \
  do {                                                   \
    if ((type) == BKG_T_F32) { using T = float; CALL; }  \
    else if ((type) == BKG_T_BF16) { using T = __bf16; CALL; } \
    else { using T = _Float16; CALL; }                   \
  } while (0)

extern "C" int bkg_mx4_quantize(const void* x, int32_t type, int64_t ldx, int64_t rows, int64_t cols, void* codes, void* scales,
                                void* stream) {
  BKG_ARG(type >= 0 && type <= 2 && rows >= 0 && cols > 0 && cols <= (1 << 24) && rows < (1ll << 31),
          "bkg_mx4_quantize: bad sizes or type (1 to 2^24 columns, rows below 2^31)");
  if (rows == 0) return 0;
  BKG_ARG(x && codes && scales && (uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 4 == 0 && (uintptr_t)x % type_bytes(type) == 0,
          "bkg_mx4_quantize: null or misaligned buffer");
  const int pieces = (int)(mx4_steps(cols) * 16);
  const int64_t blocks = (rows * pieces + 255) / 256;
  BKG_ARG(blocks < (1ll << 31), "bkg_mx4_quantize: table too large for one launch");
  const bool al = access_bytes(x, 0, ldx * type_bytes(type)) == 16;
  hipStream_t s = (hipStream_t)stream;
#define BKG_MX4_Q(AL)                                                                                                       \
  BKG_BY_TYPE(type, hipLaunchKernelGGL((mx4_quantize_kernel<T, AL>), dim3((unsigned)blocks), dim3(256), 0, s, (const T*)x,  \
                                       ldx, rows, (int)cols, pieces, (uint32_t*)codes, (uint32_t*)scales))
  if (al) BKG_MX4_Q(true); else BKG_MX4_Q(false);
#undef BKG_MX4_Q
  return check_launch("bkg_mx4_quantize");
}

extern "C" int bkg_mx4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, void* out, int32_t type,
                                  int64_t ldo, void* stream) {
  BKG_ARG(type >= 0 && type <= 2 && rows >= 0 && cols > 0 && cols <= (1 << 24) && rows < (1ll << 31),
          "bkg_mx4_dequantize: bad sizes or type (1 to 2^24 columns, rows below 2^31)");
  if (rows == 0) return 0;
  BKG_ARG(out && codes && scales && ldo >= cols && (uintptr_t)codes % 4 == 0 && (uintptr_t)out % type_bytes(type) == 0,
          "bkg_mx4_dequantize: null or misaligned buffer");
  const int pieces = (int)(mx4_steps(cols) * 16);
  const int64_t blocks = (rows * pieces + 255) / 256;
  BKG_ARG(blocks < (1ll << 31), "bkg_mx4_dequantize: table too large for one launch");
  const bool al = access_bytes(out, 0, ldo * type_bytes(type)) == 16;
  hipStream_t s = (hipStream_t)stream;
#define BKG_MX4_D(AL)                                                                                                       \
  BKG_BY_TYPE(type, hipLaunchKernelGGL((mx4_dequantize_kernel<T, AL>), dim3((unsigned)blocks), dim3(256), 0, s,             \
                                       (const uint32_t*)codes, (const unsigned char*)scales, rows, (int)cols, pieces, (T*)out, ldo))
  if (al) BKG_MX4_D(true); else BKG_MX4_D(false);
#undef BKG_MX4_D
  return check_launch("bkg_mx4_dequantize");
}

extern "C" int bkg_mx4_matmul(const void* a_codes, const void* a_scales, int64_t m, const void* b_codes, const void* b_scales,
                              int64_t n, int64_t cols, const float* bias, void* out, int32_t type, int64_t ldo, void* stream) {
  BKG_ARG(type >= 0 && type <= 2 && m >= 0 && n >= 0 && cols > 0 && cols <= (1 << 24) && m < (1ll << 31) && n < (1ll << 31),
          "bkg_mx4_matmul: bad sizes or type (1 to 2^24 columns, rows below 2^31)");
  if (m == 0 || n == 0) return 0;
  BKG_ARG(a_codes && a_scales && b_codes && b_scales && out && ldo >= n, "bkg_mx4_matmul: null buffer or overlapping rows");
  BKG_ARG((uintptr_t)a_codes % 16 == 0 && (uintptr_t)b_codes % 16 == 0 && (uintptr_t)a_scales % 4 == 0 &&
              (uintptr_t)b_scales % 4 == 0 && (uintptr_t)out % type_bytes(type) == 0,
          "bkg_mx4_matmul: misaligned buffer");
  const Mx4Args a{(const uint32_t*)a_codes, (const uint32_t*)a_scales, m, (const uint32_t*)b_codes, (const uint32_t*)b_scales, n,
                  (int)mx4_steps(cols), bias, out, ldo};
  BKG_ARG((n + 127) / 128 < 65536, "bkg_mx4_matmul: table too long");
  const dim3 grid((unsigned)((m + 127) / 128), (unsigned)((n + 127) / 128));
  BKG_BY_TYPE(type, hipLaunchKernelGGL((mx4_matmul_kernel<T>), grid, dim3(256), 0, (hipStream_t)stream, a));
  return check_launch("bkg_mx4_matmul");
}
