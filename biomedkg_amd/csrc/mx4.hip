// Microscaled 4-bit tables: quantisation, its inverse, and the product of two packed tables on the matrix cores.
//
// A row is cut into blocks of 32 values that share a power of two s = 2^E, E = clamp(floor(log2(max |v|)) - 2, -127, 127);
// a value is held as the nearest of +-{0, .5, 1, 1.5, 2, 3, 4, 6} to v / s (ties to the even code, larger ones to 6): four
// bits (sign, two exponent bits, one mantissa bit), the lower of two columns in the low nibble.  E + 127 is a byte; 255 marks
// a block that held an infinity or NaN: all its values read as NaN.  Rows are padded with zeros to a multiple of 128 columns,
// and a table lies in PANELS of 128 columns: panel p holds the 64 bytes of codes of every row side by side (and one dword of
// scales per row), so the product has no tail in its inner dimension and reads neighbouring rows of a panel as one run.
//
// Dividing by s only moves the exponent, so quantisation has one rounding and is the same whatever the input's type.
#include <algorithm>
#include <atomic>

#include "rowtypes.h"

namespace bkg {

constexpr int MX_K = 128;                       // columns a row is padded to a multiple of

static int64_t mx4_steps(int64_t cols) { return (cols + MX_K - 1) / MX_K; }

typedef int mx_i32x4 __attribute__((ext_vector_type(4)));
typedef int mx_i32x8 __attribute__((ext_vector_type(8)));
typedef float mx_f32x4 __attribute__((ext_vector_type(4)));
typedef float mx_f32x16 __attribute__((ext_vector_type(16)));

// ---- 8 values of a row per lane, 4 lanes per block, 16 lanes per panel.  Every lane of the wave takes part; returns the
// lane's dword of codes and, in the first lane of 16, the panel's dword of scales.
struct Mx4Piece { uint32_t codes, scales; };
__device__ __forceinline__ Mx4Piece mx4_piece(const float (&f)[8]) {
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
  const uint32_t b1 = __shfl_down((int)byte, 4, 64), b2 = __shfl_down((int)byte, 8, 64), b3 = __shfl_down((int)byte, 12, 64);
  return Mx4Piece{byte == 255u ? 0u : q, byte | (b1 << 8) | (b2 << 16) | (b3 << 24)};
}

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
  const Mx4Piece q = mx4_piece(f);
  if (row < rows) {
    const int64_t at_row = (int64_t)(piece >> 4) * rows + row;                    // (panel, row)
    codes[at_row * 16 + (piece & 15)] = q.codes;
    if ((piece & 15) == 0) scales[at_row] = q.scales;
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
  const int64_t at_row = (int64_t)(piece >> 4) * rows + row;
  const uint32_t q = codes[at_row * 16 + (piece & 15)];
  const int byte = scales[at_row * 4 + ((piece >> 2) & 3)], e = byte - 127;
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
      store16(p + h * N, o);
    }
  } else {
    for (int j = 0; j < 8 && c + j < cols; ++j) p[j] = v[j];
  }
}

// ---- out[m, n] = sum_k A[m, k] B[n, k] (+ bias[n]).  v_mfma_scale_f32_32x32x64_f8f6f4: lane l holds 32 columns (16 bytes)
// of row l % 32, block l / 32, and that block's scale byte; the result's column is B's row l % 32.  A panel of 128 columns is
// two such products (h = 0, 1): lane half `half` takes the panel's 16-byte piece 2 h + half and byte 2 h + half of its dword
// of scales.
// 32 staged result rows of a wave (PITCH floats apart, 16-byte aligned), W columns, as 16-byte stores: LPR lanes a row.
template <typename T, int W, int PITCH, bool GUARD, bool STREAM>
__device__ __forceinline__ void mx_store_rows(const float* mine, const float* bias, T* dst, int64_t ldo, int64_t rows_left, int lane) {
  constexpr int VE = 16 / sizeof(T), LPR = W / VE, RPI = 64 / LPR, N = 32 / RPI;
  const int col = (lane % LPR) * VE, row0 = lane / LPR;
  mx_f32x4 v[N][VE / 4];
#pragma unroll
  for (int r = 0; r < N; ++r)
#pragma unroll
    for (int q = 0; q < VE / 4; ++q) v[r][q] = *reinterpret_cast<const mx_f32x4*>(mine + (r * RPI + row0) * PITCH + col + 4 * q);
#pragma unroll
  for (int r = 0; r < N; ++r) {
    Pack<T, VE> o;
#pragma unroll
    for (int e = 0; e < VE; ++e) o.v[e] = (T)(v[r][e / 4][e % 4] + bias[e]);
    if (!GUARD || r * RPI + row0 < rows_left) {
      if constexpr (STREAM) stream16(dst + (r * RPI + row0) * ldo + col, o);
      else store16(dst + (r * RPI + row0) * ldo + col, o);
    }
  }
}

struct Mx4Args {
  const unsigned char* ca; const uint32_t* sa; int64_t m;
  const unsigned char* cb; const uint32_t* sb; int64_t n;
  int steps;                                     // panels of 128 columns
  int m_tiles, n_tiles, band;                    // band: rows of tiles walked together / row tiles a streaming block walks
  const float* bias;
  void* out; int64_t ldo;
  int wide;                                      // the rows of `out` take aligned 16-byte stores
  int classes, stream;                           // see mx_class; the result is written past the caches
  int slices;                                    // (tiles) parts of the panels; more than one: fp32 sums [slice][m][ldo] in `out`
};

// Rows of the output whose starts lie at different places of a 128-byte line would be written with two partial lines for every
// tile's piece.  So a tile takes rows of ONE class r % classes -- `classes` rows further on the start lies at the same place of
// a line again -- and begins `shift` columns early, where a line does: its pieces are whole lines (1021 x 130000 x 256 in
// bf16, rows of 2031 lines and 32 bytes: 66 us, without classes 80).
struct MxClass { int64_t row, rows; int shift; };  // its first row, how many it has, columns a tile begins early
template <typename T>
__device__ __forceinline__ MxClass mx_class(const Mx4Args& a, int q) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(static_cast<T*>(a.out) + q * a.ldo);
  return MxClass{q, (a.m - q + a.classes - 1) / a.classes, a.wide ? (int)(at % 128 / sizeof(T)) : 0};
}

__device__ __forceinline__ mx_i32x8 mx_operand(mx_i32x4 v) {
  return mx_i32x8{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
}
template <int H>
__device__ __forceinline__ mx_f32x16 mx_mfma(mx_i32x4 a, mx_i32x4 b, mx_f32x16 c, uint32_t xa, uint32_t xb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(a), mx_operand(b), c, 4, 4, 2 * H, (int)xa, 2 * H, (int)xb);
}

// Tiled product.  Four waves (2 x 2) compute a block of 64 MT x 64 NT outputs, (32 MT) x (32 NT) per wave.  Panels travel
// through a ring of S LDS slots by LDS-DMA: a stage is the block's rows of one panel of A and of B (64 contiguous bytes a
// row: a wave-instruction copies 16 whole rows) and their dwords of scales.  Slot c' of row r holds piece c' ^ ((r / 4) & 3)
// (the swizzle is applied to the DMA's source address): the b128 fragment reads of 16 neighbouring rows then fall on all 64
// banks once.  One raw barrier per stage, placed between its two halves: behind it every wave has both halves of stage
// t in registers, so slot t is refilled with stage t + S, and the first fragments of stage t + 1 are read while the second
// half of stage t multiplies.  The ring is retired by counted vmcnt waits: the loop issues nothing but DMAs.
//
// The result goes through LDS once (32 rows of a wave at a time) so that rows leave in runs of 16-byte stores.
//
// At 256 x 256 an 8192^3 product takes 493 k cycles, 262 k of them products on every matrix unit (53 %), whatever the values; the
// clock is what power leaves: 1.81 GHz for random values (272 us), 2.28 for zeros (214).
template <typename T, int MT, int NT, int S>
__global__ __launch_bounds__(256, MT * NT >= 16 ? 1 : 2) void mx4_tile_kernel(const Mx4Args a) {
  constexpr int BM = 64 * MT, BN = 64 * NT;
  constexpr int A_BYTES = BM * 64, B_BYTES = BN * 64, STAGE = A_BYTES + B_BYTES + (BM + BN) * 4;
  constexpr int CH = 2 * MT, DMAS = CH + CH / 4;             // 16-row copies / all copies per wave and stage
  static_assert(MT == NT && MT % 2 == 0, "the waves share a stage's copies evenly, and a half has a product per fragment");
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l31 = lane & 31, half = lane >> 5;

  // tile order: each XCD takes a contiguous part of the list (slice after slice of the panels); the list runs through `band`
  // tiles of rows at a time, so the tiles in flight on one XCD share their panels in its L2
  const int64_t tiles = (int64_t)a.m_tiles * a.n_tiles, total = tiles * a.slices, per = (total + BKG_XCDS - 1) / BKG_XCDS;
  const int64_t ts = (int64_t)(blockIdx.x % BKG_XCDS) * per + blockIdx.x / BKG_XCDS;
  if (blockIdx.x / BKG_XCDS >= per || ts >= total) return;
  const int64_t slice = ts / tiles, t = ts - slice * tiles;
  const int per_slice = (a.steps + a.slices - 1) / a.slices, k0 = (int)slice * per_slice, steps = min(per_slice, a.steps - k0);
  const int64_t in_band = a.band * (int64_t)a.n_tiles, band = t / in_band, at = t - band * in_band;
  const int band_m = (int)min((int64_t)a.band, a.m_tiles - band * a.band);
  const int64_t m0 = (band * a.band + at % band_m) * BM, n0 = at / band_m * BN;

  // this wave's share of a stage's copies: waves 0 and 1 copy A's 4 MT chunks of 16 rows and MT chunks of 64 scales, waves 2
  // and 3 B's
  const bool of_a = wave < 2;
  const int64_t rows = of_a ? a.m : a.n, r0 = of_a ? m0 : n0;
  const unsigned char* const codes = of_a ? a.ca : a.cb;
  const uint32_t* const scales = of_a ? a.sa : a.sb;
  int64_t src[CH], ssrc[CH / 4];
#pragma unroll
  for (int j = 0; j < CH; ++j)
    src[j] = min(r0 + ((wave & 1) * CH + j) * 16 + (lane >> 2), rows - 1) * 64 + ((lane & 3) ^ ((lane >> 4) & 3)) * 16;
#pragma unroll
  for (int j = 0; j < CH / 4; ++j) ssrc[j] = min(r0 + ((wave & 1) * (CH / 4) + j) * 64 + lane, rows - 1);
  auto copy = [&](int stage, int slot, int j) {              // copy j of this wave's DMAS of a stage
    const int64_t k = min(k0 + stage, a.steps - 1);          // (past the end: valid memory, never used)
    unsigned char* base = lds + slot * STAGE;
    if (j < CH)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(codes + k * rows * 64 + src[j]),
                                       (__attribute__((address_space(3))) void*)(base + (wave * CH + j) * 1024), 16, 0, 0);
    else
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(scales + k * rows + ssrc[j - CH]),
          (__attribute__((address_space(3))) void*)(base + A_BYTES + B_BYTES + (wave * (CH / 4) + j - CH) * 256), 4, 0, 0);
  };

  const int wm = (wave & 1) * 32 * MT, wn = (wave >> 1) * 32 * NT;
  struct Frags { mx_i32x4 a[MT], b[NT]; };
  struct Scales { uint32_t a[MT], b[NT]; };
  const int swz = (l31 >> 2) & 3;
  auto read = [&](int slot, int h, Frags& f, int i) {        // fragment i of the MT + NT
    const unsigned char* base = lds + slot * STAGE + l31 * 64 + (((2 * h + half) ^ swz) * 16);
    if (i < MT) f.a[i] = *reinterpret_cast<const mx_i32x4*>(base + (wm + 32 * i) * 64);
    else f.b[i - MT] = *reinterpret_cast<const mx_i32x4*>(base + A_BYTES + (wn + 32 * (i - MT)) * 64);
  };
  auto read_scales = [&](int slot, Scales& s) {              // (as they lie: byte `half` is not yet in front)
    const unsigned char* base = lds + slot * STAGE + A_BYTES + B_BYTES + l31 * 4;
#pragma unroll
    for (int i = 0; i < MT; ++i) s.a[i] = *reinterpret_cast<const uint32_t*>(base + (wm + 32 * i) * 4);
#pragma unroll
    for (int j = 0; j < NT; ++j) s.b[j] = *reinterpret_cast<const uint32_t*>(base + (BM + wn + 32 * j) * 4);
  };
  // (hipcc would sink the reads that a later iteration uses in front of that use: this keeps them where they are written)
  auto pin = [&](Frags& f, Scales& s) {
#pragma unroll
    for (int i = 0; i < MT; ++i) asm volatile("" : "+v"(f.a[i]), "+v"(s.a[i]));
#pragma unroll
    for (int j = 0; j < NT; ++j) asm volatile("" : "+v"(f.b[j]), "+v"(s.b[j]));
  };

  mx_f32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int j = 0; j < DMAS; ++j) copy(s, s, j);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * DMAS) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  Frags f0, f1;
  Scales sc, sn;
#pragma unroll
  for (int i = 0; i < MT + NT; ++i) read(0, 0, f0, i);
  read_scales(0, sn);
  pin(f0, sn);
  int slot = 0;
  for (int st = 0; st < steps; ++st) {
#pragma unroll
    for (int i = 0; i < MT; ++i) sc.a[i] = sn.a[i] >> (8 * half);
#pragma unroll
    for (int j = 0; j < NT; ++j) sc.b[j] = sn.b[j] >> (8 * half);
    // first half: the second half's fragments are read between the products
#pragma unroll
    for (int x = 0; x < MT * NT; ++x) {
      const int i = x / NT, j = x % NT;
      acc[i][j] = mx_mfma<0>(f0.a[i], f0.b[j], acc[i][j], sc.a[i], sc.b[j]);
      if (x < MT + NT) read(slot, 1, f1, x);
      __builtin_amdgcn_sched_barrier(0);
    }
    // this wave's reads of stage st and its copies of stage st + 1 are complete; behind the barrier everyone's are
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_waitcnt vmcnt(%0)" ::"n"((S - 2) * DMAS) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    // second half: the next stage's first fragments are read and the freed slot's copies issued between the products
    const int next = slot + 1 == S ? 0 : slot + 1;
#pragma unroll
    for (int x = 0; x < MT * NT; ++x) {
      const int i = x / NT, j = x % NT;
      acc[i][j] = mx_mfma<1>(f1.a[i], f1.b[j], acc[i][j], sc.a[i], sc.b[j]);
#pragma unroll
      for (int y = x * (MT + NT) / (MT * NT); y < (x + 1) * (MT + NT) / (MT * NT); ++y) read(next, 0, f0, y);
      if (x == 0) read_scales(next, sn);
#pragma unroll
      for (int y = x * DMAS / (MT * NT); y < (x + 1) * DMAS / (MT * NT); ++y) copy(st + S, slot, y);
      __builtin_amdgcn_sched_barrier(0);
    }
    pin(f0, sn);
    slot = next;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the copies past the last panel
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");

  // ---- the wave's 32 MT rows of 32 NT columns, 32 rows at a time
  constexpr int WN = 32 * NT, PITCH = WN + 4;                  // floats
  float* mine = reinterpret_cast<float*>(lds) + wave * 32 * PITCH;
  static_assert(4 * 32 * PITCH * 4 <= S * STAGE, "the results' staging area lies in the ring");
  T* out = static_cast<T*>(a.out) + slice * a.m * a.ldo;
  constexpr int VE = 16 / sizeof(T), LPR = WN / VE;          // elements per store, lanes per row
  const int64_t nw = n0 + wn;                                  // the wave's first column
  const bool wide = a.wide && nw + WN <= a.n;
  const int col = wide ? (lane % LPR) * VE : lane;
  float bias[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) bias[e] = 0.f;
  if (a.bias) {
#pragma unroll
    for (int e = 0; e < VE; ++e) bias[e] = a.bias[min(nw + (wide ? col + e : col + 64 * e), a.n - 1)];
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[(8 * (r >> 2) + 4 * half + (r & 3)) * PITCH + 32 * j + l31] = acc[i][j][r];
    // (a wave's LDS operations complete in order and the area is its own: no barrier)
    const int64_t mr = m0 + wm + 32 * i;
    if (wide) {
      if (a.stream) mx_store_rows<T, WN, PITCH, true, true>(mine, bias, out + mr * a.ldo + nw, a.ldo, a.m - mr, lane);
      else mx_store_rows<T, WN, PITCH, true, false>(mine, bias, out + mr * a.ldo + nw, a.ldo, a.m - mr, lane);
    } else {                                                   // the last columns, or rows that are not 16-byte aligned
      const int rows_here = (int)min((int64_t)32, a.m - mr);
      for (int row = 0; row < rows_here; ++row)
#pragma unroll
        for (int e = 0; e < WN / 64; ++e)
          if (nw + col + 64 * e < a.n) out[(mr + row) * a.ldo + nw + col + 64 * e] = (T)(mine[row * PITCH + col + 64 * e] + bias[e]);
    }
  }
}

// Inner dimension of up to six panels (an entity table of up to 768 columns): the call is the writing of its outputs, or close
// to it.  A block keeps its rows of B in registers (a wave 128 of them, 64 from three panels on) and walks A's 32-row tiles:
// tile t + 1 travels into the other of two LDS slots while tile t multiplies and its results leave, so loads, products and
// stores overlap within a block too, and only A moves, out of the L2.  All blocks walk the rows of the output from the top,
// next to each other: what is written at one time is a band of whole rows, not a column of it -- whole DRAM pages, as far as
// they go, and few of them (1021 x 130000 x 256 in bf16, packed operands, outputs in turn: 66 us, 265 MB at 4.0 TB/s; with
// tiles of 128 rows 85; 4096 x 32768 54 us, 5 TB/s, where a fill of that size takes 40).
//
// (Dynamic LDS: reading a static array that LDS-DMAs write makes hipcc wait for every copy in flight.)
constexpr int MS_ROWS = 32, MS_PITCH = 64 + 4, MS_STEPS = 6;                      // pitch: floats of a staged result row
constexpr int ms_frags(int steps) { return steps <= 2 ? 4 : 2; }                  // fragments of 32 columns of B that a wave keeps
constexpr int ms_cols(int steps) { return 4 * 32 * ms_frags(steps); }
constexpr int ms_slot(int steps) { return steps * MS_ROWS * 64 + (steps + 1) / 2 * 256; }
constexpr int ms_lds(int steps) { return 2 * ms_slot(steps) + 4 * 32 * MS_PITCH * 4; }
template <typename T, int STEPS, bool STREAM>
__global__ __launch_bounds__(256, 2) void mx4_stream_kernel(const Mx4Args a) {
  constexpr int SLOT = ms_slot(STEPS), PITCH = MS_PITCH, NF = ms_frags(STEPS), NP = NF / 2;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  unsigned char* const ring = lds;
  float* const stage = reinterpret_cast<float*>(lds + 2 * SLOT);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l31 = lane & 31, half = lane >> 5;
  // block -> (a part of A's tiles, a tile of B, a class of rows, next to each other): the XCDs take contiguous runs of B's
  // tiles; few tiles go around
  const int64_t n_tiles = (int64_t)a.n_tiles * a.classes;
  int64_t bt, part;
  if (n_tiles >= 8 * BKG_XCDS) {
    const int64_t per_xcd = (n_tiles + BKG_XCDS - 1) / BKG_XCDS;
    bt = (int64_t)(blockIdx.x % BKG_XCDS) * per_xcd + blockIdx.x / BKG_XCDS % per_xcd;
    part = blockIdx.x / BKG_XCDS / per_xcd;
  } else {
    bt = blockIdx.x % n_tiles;
    part = blockIdx.x / n_tiles;
  }
  const int64_t t0 = part * a.band, t1 = min(t0 + a.band, (int64_t)a.m_tiles);
  if (bt >= n_tiles || t0 >= t1) return;
  const MxClass cl = mx_class<T>(a, (int)(bt % a.classes));
  const int64_t nw = bt / a.classes * ms_cols(STEPS) - cl.shift + wave * 32 * NF;       // the wave's first column

  // copies of a tile, dealt out to the waves: per panel 2 chunks of 16 rows, and the scales of 2 panels at a time side by side
  auto copy_tile = [&](int64_t tile, int slot) {
    const int64_t m0 = min(tile, (int64_t)a.m_tiles - 1) * MS_ROWS;
    unsigned char* base = ring + slot * SLOT;
#pragma unroll
    for (int u = 0; u < (2 * STEPS + (STEPS + 1) / 2 + 3) / 4; ++u) {
      const int i = u * 4 + wave;
      if (i < 2 * STEPS) {
        const int64_t r = cl.row + min(m0 + (i & 1) * 16 + (lane >> 2), cl.rows - 1) * a.classes;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(a.ca + ((i >> 1) * a.m + r) * 64 + ((lane & 3) ^ ((lane >> 4) & 3)) * 16),
            (__attribute__((address_space(3))) void*)(base + i * 1024), 16, 0, 0);
      } else if (i < 2 * STEPS + (STEPS + 1) / 2) {
        const int64_t r = cl.row + min(m0 + l31, cl.rows - 1) * a.classes, st = min(2 * (i - 2 * STEPS) + half, STEPS - 1);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.sa + st * a.m + r),
                                         (__attribute__((address_space(3))) void*)(base + STEPS * 2048 + (i - 2 * STEPS) * 256), 4, 0, 0);
      }
    }
  };

  mx_i32x4 fb[NF][STEPS][2];
  uint32_t xb[NF][STEPS];
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    const int64_t r = max((int64_t)0, min(nw + 32 * j + l31, a.n - 1));
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      xb[j][st] = a.sb[st * a.n + r] >> (8 * half);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        fb[j][st][h] = *reinterpret_cast<const mx_i32x4*>(a.cb + (st * a.n + r) * 64 + (2 * h + half) * 16);
    }
  }
  // the results leave in NP pieces of 64 columns
  constexpr int VE = 16 / sizeof(T), LPR = 64 / VE, RPI = 64 / LPR, STORES = NP * 32 / RPI;
  bool full[NP], all_full = true;
  int col[NP];
  float bias[NP][VE];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int64_t np = nw + 64 * p;
    full[p] = a.wide && np >= 0 && np + 64 <= a.n;
    all_full = all_full && full[p];
    col[p] = full[p] ? (lane % LPR) * VE : lane;
#pragma unroll
    for (int e = 0; e < VE; ++e) bias[p][e] = a.bias ? a.bias[max((int64_t)0, min(np + (full[p] ? col[p] + e : col[p]), a.n - 1))] : 0.f;
  }
  copy_tile(t0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int st = 0; st < STEPS; ++st)
      asm volatile("" : "+v"(fb[j][st][0]), "+v"(fb[j][st][1]), "+v"(xb[j][st]));
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int e = 0; e < VE; ++e) asm volatile("" : "+v"(bias[p][e]));

  float* mine = stage + wave * 32 * PITCH;
  T* out = static_cast<T*>(a.out) + cl.row * a.ldo;
  const int64_t ldo = a.ldo * a.classes;
  bool stores_known = false;                               // the last tile's STORES are behind the current tile's copies
  int slot = 0;
  for (int64_t t = t0; t < t1; ++t) {
    // this wave's copies of tile t have landed: only the last tile's stores were issued behind them (vmcnt retires in order;
    // where their number is not known -- a guarded tile -- wait for everything)
    if (stores_known) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(STORES) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();                          // everyone's have, and everyone is done with the other slot
    asm volatile("" ::: "memory");
    const int64_t mr = t * MS_ROWS;
    copy_tile(t + 1, slot ^ 1);                            // (past the range: valid memory, never read)
    const unsigned char* base = ring + slot * SLOT;
    mx_f32x16 acc[NF];
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][r] = 0.f;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const uint32_t xa = *reinterpret_cast<const uint32_t*>(base + STEPS * 2048 + st * 128 + l31 * 4) >> (8 * half);
      mx_i32x4 fa[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        fa[h] = *reinterpret_cast<const mx_i32x4*>(base + st * 2048 + l31 * 64 + (((2 * h + half) ^ ((l31 >> 2) & 3)) * 16));
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        acc[j] = mx_mfma<0>(fa[0], fb[j][st][0], acc[j], xa, xb[j][st]);
        acc[j] = mx_mfma<1>(fa[1], fb[j][st][1], acc[j], xa, xb[j][st]);
      }
    }
    const bool rows_full = mr + MS_ROWS <= cl.rows;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) mine[(8 * (r >> 2) + 4 * half + (r & 3)) * PITCH + 32 * j + l31] = acc[2 * p + j][r];
      const int64_t np = nw + 64 * p;
      if (full[p] && rows_full) {
        mx_store_rows<T, 64, PITCH, false, STREAM>(mine, bias[p], out + mr * ldo + np, ldo, MS_ROWS, lane);
      } else if (full[p]) {
        mx_store_rows<T, 64, PITCH, true, STREAM>(mine, bias[p], out + mr * ldo + np, ldo, cl.rows - mr, lane);
      } else {
        const int rows_here = (int)min((int64_t)MS_ROWS, cl.rows - mr);
        const int64_t c = np + col[p];
        for (int row = 0; row < rows_here; ++row)
          if (c >= 0 && c < a.n) out[(mr + row) * ldo + c] = (T)(mine[row * PITCH + col[p]] + bias[p][0]);
      }
    }
    stores_known = all_full && rows_full;
    slot ^= 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // the copies past the range
}

// A few rows (m <= 32): B streams from memory straight into the matrix cores, a 32-row tile of it per wave (KSPLIT: per
// block, the waves share the panels and add their sums in wave order).  PACKED: A lies packed in memory; else the block
// packs x itself (into LDS) while its first tiles are on their way: one launch, no scratch memory.
struct Mx4X { const void* x; int type; int64_t ldx; int cols; };
template <typename T, bool PACKED, bool KSPLIT>
__global__ __launch_bounds__(256) void mx4_few_kernel(const Mx4Args a, const Mx4X x) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];       // A: [panel][32 rows][64], [panel][32] scales
  __shared__ float sums[KSPLIT ? 3 * 16 * 64 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, half = lane >> 5;
  const int64_t n0 = (KSPLIT ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave) * 32;
  const int64_t rb = min(n0 + l31, a.n - 1), ra = min((int64_t)l31, a.m - 1);
  constexpr int D = KSPLIT ? 4 : 1, AHEAD = 2;
  const int first = KSPLIT ? wave : 0;
  mx_i32x4 vb[AHEAD][2];
  uint32_t xb[AHEAD];
  auto load = [&](int st, int at) {
    const int64_t s = min(st, a.steps - 1);
    xb[at] = a.sb[s * a.n + rb];
#pragma unroll
    for (int h = 0; h < 2; ++h) vb[at][h] = *reinterpret_cast<const mx_i32x4*>(a.cb + (s * a.n + rb) * 64 + (2 * h + half) * 16);
  };
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) load(first + u * D, u);
  if constexpr (!PACKED) {
    const int pieces = a.steps * 16;
    uint32_t* xs = reinterpret_cast<uint32_t*>(lds + a.steps * 2048);
    // (whole waves, at most 32 rows; what lies in the rows behind them ends in output rows that are not there)
    for (int p = threadIdx.x; p < (((int)a.m * pieces + 63) & ~63); p += 256) {
      const int row = p / pieces, piece = p - row * pieces, c = piece * 8;
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = 0.f;
        if (row < a.m && c + j < x.cols) {
          const int64_t at = row * x.ldx + c + j;
          f[j] = x.type == BKG_T_F32    ? static_cast<const float*>(x.x)[at]
                 : x.type == BKG_T_BF16 ? widen(static_cast<const __bf16*>(x.x)[at])
                                        : widen(static_cast<const _Float16*>(x.x)[at]);
        }
      }
      const Mx4Piece q = mx4_piece(f);
      const int st = piece >> 4, w = piece & 15;                            // word w of the row's 16: 16-byte piece w / 4, swizzled
      *reinterpret_cast<uint32_t*>(lds + st * 2048 + row * 64 + (((w >> 2) ^ ((row >> 2) & 3)) * 16) + (w & 3) * 4) = q.codes;
      if (w == 0) xs[st * 32 + row] = q.scales;
    }
    __syncthreads();
  }
  mx_f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  auto multiply = [&](int st, int at) {
    mx_i32x4 va[2];
    uint32_t xa;
    if constexpr (PACKED) {
      xa = a.sa[st * a.m + ra];
#pragma unroll
      for (int h = 0; h < 2; ++h) va[h] = *reinterpret_cast<const mx_i32x4*>(a.ca + (st * a.m + ra) * 64 + (2 * h + half) * 16);
    } else {
      xa = *reinterpret_cast<const uint32_t*>(lds + a.steps * 2048 + st * 128 + l31 * 4);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        va[h] = *reinterpret_cast<const mx_i32x4*>(lds + st * 2048 + l31 * 64 + (((2 * h + half) ^ ((l31 >> 2) & 3)) * 16));
    }
    acc = mx_mfma<0>(va[0], vb[at][0], acc, xa >> (8 * half), xb[at] >> (8 * half));
    acc = mx_mfma<1>(va[1], vb[at][1], acc, xa >> (8 * half), xb[at] >> (8 * half));
  };
  for (int st = first; st < a.steps; st += AHEAD * D) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (st + u * D < a.steps) {
        multiply(st + u * D, u);
        load(st + (u + AHEAD) * D, u);
      }
  }
  if constexpr (KSPLIT) {
    if (wave > 0)
#pragma unroll
      for (int r = 0; r < 16; ++r) sums[((wave - 1) * 16 + r) * 64 + lane] = acc[r];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < 3; ++w)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[r] += sums[(w * 16 + r) * 64 + lane];
  }
  const int64_t n = n0 + l31;
  if (n >= a.n) return;
  const float b = a.bias ? a.bias[n] : 0.f;
  T* out = static_cast<T*>(a.out);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int m = 8 * (r >> 2) + 4 * half + (r & 3);
    if (m < a.m) out[m * a.ldo + n] = (T)(acc[r] + b);
  }
}

// Whole lines of a result beyond STREAM_BYTES leave past the caches; a smaller one is found there by whoever reads it next (a
// 1536 x 130000 product in bf16 and the maximum of its rows: 189 us so, 215 through the caches; 768 rows: 96 and 76).
template <typename T>
static bool mx4_past_caches(const Mx4Args& a) {
  const int64_t row = a.ldo * (int64_t)sizeof(T);
  return a.wide && row * a.classes % 128 == 0 && a.m * row > STREAM_BYTES;
}

// The slices' sums, added in order, with the bias: a thread per four columns of a row (ld: the sums' rows, a multiple of 4).
template <typename T>
__global__ __launch_bounds__(256) void mx4_join_kernel(const float* __restrict__ sums, int slices, int64_t m, int64_t n, int64_t ld,
                                                       const float* __restrict__ bias, T* __restrict__ out, int64_t ldo) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, row = at / (ld / 4), c = (at - row * (ld / 4)) * 4;
  if (row >= m) return;
  mx_f32x4 s = *reinterpret_cast<const mx_f32x4*>(sums + row * ld + c);
#pragma unroll 4
  for (int i = 1; i < slices; ++i) s += *reinterpret_cast<const mx_f32x4*>(sums + (i * m + row) * ld + c);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c + j < n) out[row * ldo + c + j] = (T)(s[j] + (bias ? bias[c + j] : 0.f));
}

static const char* const MX_LDS = "bkg_mx4 product: dynamic LDS";
template <typename T, int MT, int NT, int S>
static int mx4_launch(Mx4Args a, hipStream_t s) {
  constexpr int LDS = S * (64 * (MT + NT) * 64 + 64 * (MT + NT) * 4);
  static std::atomic<uint64_t> granted{0};
  if (const int rc = grant_lds((const void*)mx4_tile_kernel<T, MT, NT, S>, LDS, granted, MX_LDS)) return rc;
  a.m_tiles = (int)((a.m + 64 * MT - 1) / (64 * MT));
  a.n_tiles = (int)((a.n + 64 * NT - 1) / (64 * NT));
  a.stream = mx4_past_caches<T>(a);
  // rows of tiles walked together: enough to share panels, few enough that what is written at one time is a few whole rows
  // (8192 x 16384 x 1024 in bf16: 133 us with 4 or 2, 155 with 8; 8192 x 8192 x 2048: 104 with 4, 108 with 2, 114 with 8)
  a.band = 4;
  const int64_t total = (int64_t)a.m_tiles * a.n_tiles * a.slices;
  const unsigned grid = (unsigned)((total + BKG_XCDS - 1) / BKG_XCDS * BKG_XCDS);
  hipLaunchKernelGGL((mx4_tile_kernel<T, MT, NT, S>), dim3(grid), dim3(256), LDS, s, a);
  return 0;
}

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
  BKG_ARG(blocks < (1ll << 24), "bkg_mx4_quantize: table too large for one launch");
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
  BKG_ARG(blocks < (1ll << 24), "bkg_mx4_dequantize: table too large for one launch");
  const bool al = access_bytes(out, 0, ldo * type_bytes(type)) == 16;
  hipStream_t s = (hipStream_t)stream;
#define BKG_MX4_D(AL)                                                                                                       \
  BKG_BY_TYPE(type, hipLaunchKernelGGL((mx4_dequantize_kernel<T, AL>), dim3((unsigned)blocks), dim3(256), 0, s,             \
                                       (const uint32_t*)codes, (const unsigned char*)scales, rows, (int)cols, pieces, (T*)out, ldo))
  if (al) BKG_MX4_D(true); else BKG_MX4_D(false);
#undef BKG_MX4_D
  return check_launch("bkg_mx4_dequantize");
}

static int mx4_check_product(int64_t m, int64_t n, int64_t cols, const void* b_codes, const void* b_scales, const float* bias,
                             const void* out, int32_t type, int64_t ldo) {
  BKG_ARG(type >= 0 && type <= 2 && m >= 0 && n >= 0 && cols > 0 && cols <= (1 << 24) && m < (1ll << 31) && n < (1ll << 31),
          "bkg_mx4 product: bad sizes or type (1 to 2^24 columns, rows below 2^31)");
  if (m == 0 || n == 0) return 0;
  BKG_ARG(b_codes && b_scales && out && ldo >= n, "bkg_mx4 product: null buffer or overlapping rows");
  BKG_ARG((uintptr_t)b_codes % 16 == 0 && (uintptr_t)b_scales % 4 == 0 && (uintptr_t)out % type_bytes(type) == 0 &&
              (uintptr_t)bias % 4 == 0,
          "bkg_mx4 product: misaligned buffer");
  BKG_ARG((m <= 32 ? 1 : (m + 127) / 128 + 8) * ((n + 127) / 128 + 1) < (1ll << 24) - 1024, "bkg_mx4 product: too many tiles for one launch");
  return 0;
}

template <typename T, bool PACKED, bool KSPLIT>
static int mx4_few_launch_as(const Mx4Args& a, const Mx4X& x, unsigned blocks, hipStream_t s) {
  const int lds = PACKED ? 0 : a.steps * (2048 + 128);
  constexpr int SUMS = KSPLIT ? 3 * 16 * 64 * 4 : 4;         // (the kernel's static LDS)
  if (lds + SUMS > (64 << 10)) {                             // (up to 64 panels, all granted at once)
    static std::atomic<uint64_t> granted{0};
    if (const int rc = grant_lds((const void*)mx4_few_kernel<T, PACKED, KSPLIT>, 64 * 2176, granted, MX_LDS)) return rc;
  }
  hipLaunchKernelGGL((mx4_few_kernel<T, PACKED, KSPLIT>), dim3(blocks), dim3(256), lds, s, a, x);
  return 0;
}
template <typename T, bool PACKED>
static int mx4_few_launch(const Mx4Args& a, const Mx4X& x, hipStream_t s) {
  const int64_t tiles = (a.n + 31) / 32;
  // a wave per tile keeps the chip busy from 2048 tiles on; below that, and with panels to share, the waves of a block
  if (tiles >= 2048 || a.steps < 4) return mx4_few_launch_as<T, PACKED, false>(a, x, (unsigned)((tiles + 3) / 4), s);
  return mx4_few_launch_as<T, PACKED, true>(a, x, (unsigned)tiles, s);
}

template <typename T, int STEPS, bool STREAM>
static int mx4_stream_launch_as(const Mx4Args& a, unsigned blocks, hipStream_t s) {
  static std::atomic<uint64_t> granted{0};
  if (const int rc = grant_lds((const void*)mx4_stream_kernel<T, STEPS, STREAM>, ms_lds(STEPS), granted, MX_LDS)) return rc;
  hipLaunchKernelGGL((mx4_stream_kernel<T, STEPS, STREAM>), dim3(blocks), dim3(256), ms_lds(STEPS), s, a);
  return 0;
}
template <typename T, int STEPS>
static int mx4_stream_launch(Mx4Args a, hipStream_t s) {
  // classes of rows (mx_class) where rows are long and every class fills a tile.  Blocks next to each other write the lines that
  // short rows share at about the same time: 130000 x 1000 in bf16, 256 inner columns, 93 us without classes and 110 with; in
  // fp32 162 and 132; 32768 x 4008 in bf16 96 and 62.
  constexpr int64_t LONG_ROW = 4000;                         // bytes
  const int64_t row = a.ldo * (int64_t)sizeof(T);
  if (a.wide && row >= LONG_ROW) {
    while (row * a.classes % 128) a.classes <<= 1;
    if (a.m < (int64_t)MS_ROWS * a.classes) a.classes = 1;
  }
  int64_t early = 0;                                         // columns that tiles begin early, at most
  for (int q = 0; q < a.classes && a.wide; ++q)
    early = std::max<int64_t>(early, (int64_t)((uintptr_t)(static_cast<T*>(a.out) + q * a.ldo) % 128 / sizeof(T)));
  a.stream = mx4_past_caches<T>(a);
  a.m_tiles = (int)(((a.m + a.classes - 1) / a.classes + MS_ROWS - 1) / MS_ROWS);
  a.n_tiles = (int)((a.n + early + ms_cols(STEPS) - 1) / ms_cols(STEPS));
  const int64_t n_tiles = (int64_t)a.n_tiles * a.classes;
  // parts of A's tiles: so many that two blocks per CU are there
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(a.m_tiles, 512 / n_tiles));
  a.band = (int)((a.m_tiles + parts - 1) / parts);
  const int64_t blocks = (int64_t)((a.m_tiles + a.band - 1) / a.band) *
                         (n_tiles >= 8 * BKG_XCDS ? (n_tiles + BKG_XCDS - 1) / BKG_XCDS * BKG_XCDS : n_tiles);
  return a.stream ? mx4_stream_launch_as<T, STEPS, true>(a, (unsigned)blocks, s)
                  : mx4_stream_launch_as<T, STEPS, false>(a, (unsigned)blocks, s);
}

// rows of x that a product packs within its one launch: at most 32, and few enough values that every block packs them anew
static bool mx4_packs_itself(int64_t m, int64_t cols) { return m <= 32 && m * mx4_steps(cols) * MX_K <= 8192; }

// Parts of a long inner dimension (32 panels or more) for a product of so few 128 x 128 tiles that most CUs would have none: as
// many as fill them, eight panels or more each; a second launch adds their sums in order.  33 x 5000 x 8192 in bf16: 15 us, 36 in
// one part; 8192 x 16 x 8192 20 and 39; 500 x 500 x 4096 15 and 19; 4096 x 64 x 4096 16 and 16.  1024 x 2048 x 2048 (128 tiles)
// took 20 instead of 11.  1: not worth it, or another kernel's (see mx4_product).
static int mx4_slices(int64_t m, int64_t n, int64_t cols) {
  const int64_t tiles = (m + 127) / 128 * ((n + 127) / 128), steps = mx4_steps(cols);
  if (m <= 32 || n <= 0 || steps < 32 || tiles > 64) return 1;
  const int64_t want = std::min<int64_t>(256 / tiles, steps / 8), per = (steps + want - 1) / want;
  return (int)((steps + per - 1) / per);                     // (every slice has a panel)
}
static int64_t mx4_sums_bytes(int64_t m, int64_t n, int64_t cols) {
  const int slices = mx4_slices(m, n, cols);
  return slices == 1 ? 0 : slices * m * ((n + 3) / 4 * 4) * 4;
}

template <typename T>
static int mx4_product(const Mx4Args& a, float* sums, int64_t cols, hipStream_t s) {
  const int slices = mx4_slices(a.m, a.n, cols);
  if (slices > 1) {
    Mx4Args b = a;
    b.bias = nullptr;
    b.out = sums;
    b.ldo = (a.n + 3) / 4 * 4;
    b.wide = 1;                                              // (the workspace is 16-byte aligned)
    b.slices = slices;
    if (const int rc = mx4_launch<float, 2, 2, 2>(b, s)) return rc;
    const int64_t threads = a.m * (b.ldo / 4);
    hipLaunchKernelGGL((mx4_join_kernel<T>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, sums, slices, a.m, a.n, b.ldo,
                       a.bias, (T*)a.out, a.ldo);
    return 0;
  }
  if (a.m <= 32) return mx4_few_launch<T, true>(a, Mx4X{}, s);
  // up to six panels: B in registers (1021 x 130000 x 768 in bf16 157 us with 128 x 128 tiles, 124 so; 8192 x 8192 x 768 68 and
  // 46; 4096 x 4096 x 768 17.4 and 16.5; 130000 x 256 x 768 37 and 29); each class of rows loads it anew.
  if (a.steps == 1) return mx4_stream_launch<T, 1>(a, s);
  if (a.steps == 2) return mx4_stream_launch<T, 2>(a, s);
  if (a.steps == 3) return mx4_stream_launch<T, 3>(a, s);
  if (a.steps == 4) return mx4_stream_launch<T, 4>(a, s);
  if (a.steps == 5) return mx4_stream_launch<T, 5>(a, s);
  if (a.steps == 6) return mx4_stream_launch<T, 6>(a, s);
  // More: 256 x 256 tiles, a block with a CU to itself, where they fill the chip and the inner dimension is long (8192 x 8192 x
  // 8192 in bf16: 271 us, 4 PFLOP/s, against 316 with 128 x 128; 4096 x 4096 x 4096 42 and 46; x 2048 31 and 31); else 128 x 128,
  // four blocks on a CU: one stores while others multiply (5000 x 6000 x 1024: 34 us, 256 x 256 44; 2048 x 2048 x 8192 39 and 52).
  if ((a.m + 255) / 256 * ((a.n + 255) / 256) >= 192 && a.steps >= 16) return mx4_launch<T, 4, 4, 4>(a, s);
  return mx4_launch<T, 2, 2, 2>(a, s);
}

extern "C" int64_t bkg_mx4_matmul_workspace_bytes(int64_t m, int64_t n, int64_t cols) {
  return m <= 0 || n <= 0 || cols <= 0 ? 0 : mx4_sums_bytes(m, n, cols);
}

extern "C" int bkg_mx4_matmul(const void* a_codes, const void* a_scales, int64_t m, const void* b_codes, const void* b_scales,
                              int64_t n, int64_t cols, const float* bias, void* out, int32_t type, int64_t ldo, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  if (const int rc = mx4_check_product(m, n, cols, b_codes, b_scales, bias, out, type, ldo)) return rc;
  if (m == 0 || n == 0) return 0;
  BKG_ARG(a_codes && a_scales && (uintptr_t)a_codes % 16 == 0 && (uintptr_t)a_scales % 4 == 0, "bkg_mx4_matmul: null or misaligned buffer");
  const int64_t need = mx4_sums_bytes(m, n, cols);
  BKG_ARG(need == 0 || (workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need),
          "bkg_mx4_matmul: workspace below bkg_mx4_matmul_workspace_bytes or misaligned");
  const Mx4Args a{(const unsigned char*)a_codes, (const uint32_t*)a_scales, m, (const unsigned char*)b_codes,
                  (const uint32_t*)b_scales, n, (int)mx4_steps(cols), 0, 0, 0, bias, out, ldo,
                  access_bytes(out, 0, ldo * type_bytes(type)) == 16, 1, 0, 1};
  int rc = 0;
  BKG_BY_TYPE(type, rc = mx4_product<T>(a, (float*)workspace, cols, (hipStream_t)stream));
  if (rc) return rc;
  return check_launch("bkg_mx4_matmul");
}

// the packed rows, then the slices' sums
static int64_t mx4_packed_bytes(int64_t m, int64_t cols) { return (mx4_steps(cols) * m * 68 + 255) & ~(int64_t)255; }
extern "C" int64_t bkg_mx4_linear_workspace_bytes(int64_t m, int64_t n, int64_t cols) {
  return m <= 0 || n <= 0 || cols <= 0 || mx4_packs_itself(m, cols) ? 0 : mx4_packed_bytes(m, cols) + mx4_sums_bytes(m, n, cols);
}

extern "C" int bkg_mx4_linear(const void* x, int32_t x_type, int64_t ldx, int64_t m, const void* b_codes, const void* b_scales,
                              int64_t n, int64_t cols, const float* bias, void* out, int32_t type, int64_t ldo, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  if (const int rc = mx4_check_product(m, n, cols, b_codes, b_scales, bias, out, type, ldo)) return rc;
  if (m == 0 || n == 0) return 0;
  BKG_ARG(x && x_type >= 0 && x_type <= 2 && (uintptr_t)x % type_bytes(x_type) == 0, "bkg_mx4_linear: null or misaligned x");
  if (!mx4_packs_itself(m, cols)) {
    BKG_ARG(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= bkg_mx4_linear_workspace_bytes(m, n, cols),
            "bkg_mx4_linear: workspace below bkg_mx4_linear_workspace_bytes or misaligned");
    unsigned char* codes = (unsigned char*)workspace;
    unsigned char* scales = codes + mx4_steps(cols) * m * 64;
    if (const int rc = bkg_mx4_quantize(x, x_type, ldx, m, cols, codes, scales, stream)) return rc;
    return bkg_mx4_matmul(codes, scales, m, b_codes, b_scales, n, cols, bias, out, type, ldo, codes + mx4_packed_bytes(m, cols),
                          workspace_bytes - mx4_packed_bytes(m, cols), stream);
  }
  const Mx4Args a{nullptr, nullptr, m, (const unsigned char*)b_codes, (const uint32_t*)b_scales, n, (int)mx4_steps(cols), 0, 0, 0,
                  bias, out, ldo, 0, 1, 0, 1};
  int rc = 0;
  BKG_BY_TYPE(type, rc = (mx4_few_launch<T, false>(a, Mx4X{x, x_type, ldx, (int)cols}, (hipStream_t)stream)));
  if (rc) return rc;
  return check_launch("bkg_mx4_linear");
}
