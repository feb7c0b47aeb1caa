// Distillation of a row of logits from a teacher's K best entries.
//
// x [R, V] student logits, (id, t) [R, K] the teacher's entries, temperature T.  An entry is usable if 0 <= id < V and t is
// not -inf.  With p = softmax(x / T) over all V columns and q = softmax(t / T) over the row's usable entries,
//     L_r = T^2 sum_j q_j (ln q_j - ln p_{id_j}),        dL_r / dx = T (p - q)
// (an id that occurs twice takes both entries' q).  A row without a usable entry, or whose logits are all -inf, is left out:
// loss 0, gradient 0.  K = 1 is cross entropy.
//
// Bound by HBM: x is read once for the running maximum and sum of exponentials (fp32, one pass), and once more where the
// gradient is written.  A training call writes the gradient of the mean / sum in the FORWARD, behind each row's (or the whole
// batch's) statistics, while the logits still lie in the caches: HBM sees them once.  That gradient is for an upstream
// factor of 1; the backward launch looks at the factor on the device and returns at once if it is 1, else it computes the
// gradient again from the logits (kd_regrad).
#include "rowtypes.h"

namespace bkg {

constexpr int KD_THREADS = 256;                  // blocks that share a row
constexpr int KD_MAX_K = 1024;
constexpr float KD_LOG2E = 1.4426950408889634f, KD_LN2 = 0.6931471805599453f;

struct KdTeacher {
  const void* ids; int ids_i32; int64_t ld_ids;
  const void* t; int t_type; int64_t ld_t;
  int k;
};
struct KdRow { float m, sum, tmax, tsum; };      // max of x and sum of exp2(c (x - max)), c = log2(e) / T; the same of the usable
                                                 // entries.  tsum = sum = 0: the row is left out
struct KdArgs {
  const void* x; int64_t ldx; int v, parts;
  float c, temp;
  KdTeacher te;
  float* part;                                   // [rows][parts][2]
  KdRow* rows; float* losses;
  void* d; int64_t ldd;                          // the gradient (null: none)
  const float* g; int g_step; float coef;        // d = g[row g_step] coef (p - q); g null: 1
  int64_t n_rows;
  int stream;                                    // the gradient is beyond STREAM_BYTES
  unsigned* done;                                // (parts) rows whose loss is there; the last one's block adds them up:
  float* loss; float sum_scale;                  // loss[0] = sum_scale * their sum (null: not wanted)
};

__device__ __forceinline__ float kd_exp2(float v) { return __builtin_amdgcn_exp2f(v); }

// (m, s) joined with (m2, s2): sums around the larger maximum.  -inf maxima carry s = 0 or NaN.
__device__ __forceinline__ void kd_join(float& m, float& s, float m2, float s2, float c) {
  const float mm = fmaxf(m, m2), ref = mm == -INFINITY ? 0.f : mm;
  s = s * kd_exp2((m - ref) * c) + s2 * kd_exp2((m2 - ref) * c);
  m = mm;
}

__device__ __forceinline__ float kd_block_sum(float v, float* red) {       // fixed order; every thread gets it
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < (int)blockDim.x / 64; ++w) s += red[w];
  return s;
}
__device__ __forceinline__ float kd_block_max(float v, float* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = red[0];
  for (int w = 1; w < (int)blockDim.x / 64; ++w) s = fmaxf(s, red[w]);
  return s;
}

// How a row's columns fall into 16-byte accesses: `head` single columns, n_vec accesses, the rest single columns.
template <typename T> struct KdSpan {
  static constexpr int VE = 16 / sizeof(T);
  int head, n_vec, v0, v1, tail0, tail1;         // this block's accesses [v0, v1) and its single columns [0, head) / [tail0, tail1)
  __device__ __forceinline__ KdSpan(const T* row, int n, int part, int parts) {
    const int off = (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T));
    const int h = off < n ? off : n;
    n_vec = (n - h) / VE;
    const int per = (n_vec + parts - 1) / parts;
    v0 = per * part < n_vec ? per * part : n_vec;
    v1 = v0 + per < n_vec ? v0 + per : n_vec;
    head = part == 0 ? h : 0;
    first = h;
    tail0 = part == parts - 1 ? h + n_vec * VE : n;
    tail1 = n;
  }
  int first;                                     // column of access 0
  __device__ __forceinline__ bool mine(int col) const {
    return (col < head) || (col >= first + v0 * VE && col < first + v1 * VE) || (col >= tail0 && col < tail1);
  }
};

// Running maximum and sum of this thread's columns.  exp2(c (x - m)), not exp2(c x - c m): the difference is exact near the
// maximum whatever the row's offset, and logits at the type's lowest or largest value do not overflow.
template <typename T, int THREADS>
__device__ __forceinline__ void kd_stats(const T* __restrict__ xr, const KdSpan<T>& sp, float c, float& m, float& s) {
  constexpr int VE = KdSpan<T>::VE, U = 4;
  const Pack<T, VE>* xv = reinterpret_cast<const Pack<T, VE>*>(xr + sp.first);
  float ref = 0.f;                                                    // m, 0 while m = -inf
  auto one = [&](float f) {
    if (f > m) { s *= kd_exp2((m - f) * c); m = ref = f; }            // (s = 0 while m = -inf)
    s += kd_exp2((f - ref) * c);
  };
  auto pack = [&](const Pack<T, VE>& r) {
    float f[VE], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < VE; ++j) { f[j] = widen(r.v[j]); top = fmaxf(top, f[j]); }
    if (top > m) { s *= kd_exp2((m - top) * c); m = ref = top; }
#pragma unroll
    for (int j = 0; j < VE; ++j) s += kd_exp2((f[j] - ref) * c);
  };
  int i = sp.v0 + threadIdx.x;
  for (; i + (U - 1) * THREADS < sp.v1; i += THREADS * U) {
    Pack<T, VE> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = xv[i + u * THREADS];
#pragma unroll
    for (int u = 0; u < U; ++u) pack(r[u]);
  }
  for (; i < sp.v1; i += THREADS) pack(xv[i]);
  for (int j = threadIdx.x; j < sp.head; j += THREADS) one(widen(xr[j]));
  for (int j = sp.tail0 + threadIdx.x; j < sp.tail1; j += THREADS) one(widen(xr[j]));
}

// The block's (m, s) from its threads'; every thread gets it.
template <int THREADS>
__device__ __forceinline__ void kd_block_join(float& m, float& s, float c, float* red) {        // red: 2 THREADS / 64 floats
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) kd_join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), c);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) { red[2 * (threadIdx.x >> 6)] = m; red[2 * (threadIdx.x >> 6) + 1] = s; }
  __syncthreads();
  m = red[0]; s = red[1];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) kd_join(m, s, red[2 * w], red[2 * w + 1], c);
}

// The row's teacher entries into LDS: id (-1 where not usable) and t.
__device__ __forceinline__ void kd_load_teacher(const KdTeacher& te, int64_t row, int v, int* __restrict__ id_lds,
                                                float* __restrict__ t_lds) {
  for (int j = threadIdx.x; j < te.k; j += blockDim.x) {
    const int64_t at = row * te.ld_ids + j;
    const int64_t id = te.ids_i32 ? (int64_t)static_cast<const int32_t*>(te.ids)[at] : static_cast<const int64_t*>(te.ids)[at];
    const int64_t tt = row * te.ld_t + j;
    const float t = te.t_type == BKG_T_F32    ? static_cast<const float*>(te.t)[tt]
                    : te.t_type == BKG_T_BF16 ? widen(static_cast<const __bf16*>(te.t)[tt])
                                              : widen(static_cast<const _Float16*>(te.t)[tt]);
    id_lds[j] = (id >= 0 && id < v && !(t == -INFINITY)) ? (int)id : -1;
    t_lds[j] = t;
  }
  __syncthreads();
}

// The usable entries' maximum and sum (the sum is 0 without one); t_lds becomes q.
__device__ __forceinline__ void kd_teacher_softmax(int k, float c, const int* __restrict__ id_lds, float* __restrict__ t_lds,
                                                   float* red, float& tm, float& ts) {
  tm = -INFINITY;
  bool any = false;
  for (int j = threadIdx.x; j < k; j += blockDim.x)
    if (id_lds[j] >= 0) { tm = fmaxf(tm, t_lds[j]); any = true; }
  tm = kd_block_max(tm, red);
  any = __syncthreads_or(any);
  ts = 0.f;
  for (int j = threadIdx.x; j < k; j += blockDim.x)
    if (id_lds[j] >= 0) ts += kd_exp2((t_lds[j] - tm) * c);
  ts = kd_block_sum(ts, red);
  if (!any) ts = 0.f;
}

// L = T sum_j q_j ((t_j - tm) - (x_j - m)) + T^2 (ln s - ln ts).  The sum runs over 2^-12 of the differences: logits masked with
// the type's lowest value are finite, and so is a loss over several of them, but not the sum of up to 1024 such differences, nor a
// difference divided by T < 1.  (Powers of two: the same digits.)
constexpr float KD_SMALL = 1.f / 4096, KD_LARGE = 4096.f;
__device__ __forceinline__ float kd_gap(float t, float tm, float x, float m) {
  return (t * KD_SMALL - tm * KD_SMALL) - (x * KD_SMALL - m * KD_SMALL);
}
__device__ __forceinline__ float kd_loss_of(float temp, float gap, float s, float ts) {
  const float ln_s = KD_LN2 * __builtin_amdgcn_logf(s), ln_ts = KD_LN2 * __builtin_amdgcn_logf(ts);
  return temp * KD_LARGE * gap + temp * temp * (ln_s - ln_ts);
}

// The row's loss from its statistics, in every thread (t_lds still holds t).
template <typename T>
__device__ __forceinline__ float kd_loss(const KdArgs& a, const T* __restrict__ xr, const int* __restrict__ id_lds,
                                         const float* __restrict__ t_lds, float m, float s, float tm, float ts, float* red) {
  const float inv_ts = 1.f / ts;
  float gap = 0.f;
  for (int j = threadIdx.x; j < a.te.k; j += blockDim.x) {
    if (id_lds[j] < 0) continue;
    const float q = kd_exp2((t_lds[j] - tm) * a.c) * inv_ts;
    if (!(q == 0.f)) gap += q * kd_gap(t_lds[j], tm, widen(xr[id_lds[j]]), m);
  }
  return kd_loss_of(a.temp, kd_block_sum(gap, red), s, ts);
}

// The teacher's columns of a row's gradient (the block's part of them) are written again, whole, once the others are there.
template <typename T>
__device__ __forceinline__ void kd_write_entries(const KdArgs& a, const T* __restrict__ xr, T* __restrict__ dr, const KdSpan<T>& sp,
                                                 const KdRow& rw, float scale, const int* __restrict__ id_lds,
                                                 float* __restrict__ t_lds) {
  const float c = a.c, ps = scale / rw.sum, ref = rw.m == -INFINITY ? 0.f : rw.m, inv_ts = 1.f / rw.tsum;
  for (int j = threadIdx.x; j < a.te.k; j += blockDim.x) t_lds[j] = kd_exp2((t_lds[j] - rw.tmax) * c) * inv_ts;
  __syncthreads();                                                    // (also orders the stores before it and those below)
  for (int j = threadIdx.x; j < a.te.k; j += blockDim.x) {
    const int id = id_lds[j];
    if (id < 0 || !sp.mine(id)) continue;
    bool first = true;                                                // (an id that occurs again is its first place's)
    float q = 0.f;
    for (int i = 0; i < a.te.k; ++i) {
      const bool same = id_lds[i] == id;
      first = first && (i >= j || !same);
      q += same ? t_lds[i] : 0.f;
    }
    if (first) dr[id] = (T)(kd_exp2((widen(xr[id]) - ref) * c) * ps - scale * q);
  }
}

// The block's part of the row's gradient, scale (p - q).  id_lds / t_lds hold the teacher's entries.
template <typename T, int THREADS>
__device__ __forceinline__ void kd_write_grad(const KdArgs& a, const T* __restrict__ xr, T* __restrict__ dr, const KdSpan<T>& sp,
                                              const KdRow& rw, float scale, const int* __restrict__ id_lds,
                                              float* __restrict__ t_lds) {
  constexpr int VE = KdSpan<T>::VE, U = 4;
  const bool off = rw.tsum == 0.f && rw.sum == 0.f;
  const float ps = off ? 0.f : scale / rw.sum, c = a.c, ref = rw.m == -INFINITY ? 0.f : rw.m;
  auto value = [&](float f) { return off ? 0.f : kd_exp2((f - ref) * c) * ps; };
  for (int i = threadIdx.x; i < sp.head; i += THREADS) dr[i] = (T)value(widen(xr[i]));
  for (int i = sp.tail0 + threadIdx.x; i < sp.tail1; i += THREADS) dr[i] = (T)value(widen(xr[i]));
  const Pack<T, VE>* xv = reinterpret_cast<const Pack<T, VE>*>(xr + sp.first);
  T* dv = dr + sp.first;
  auto pack = [&](Pack<T, VE> r, int i) {
#pragma unroll
    for (int j = 0; j < VE; ++j) r.v[j] = (T)value(widen(r.v[j]));
    if (a.stream) stream16(dv + (int64_t)i * VE, r);
    else store16(dv + (int64_t)i * VE, r);
  };
  if ((reinterpret_cast<uintptr_t>(dv) & 15) == 0) {
    int i = sp.v0 + threadIdx.x;
    for (; i + (U - 1) * THREADS < sp.v1; i += THREADS * U) {
      Pack<T, VE> r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) r[u] = xv[i + u * THREADS];
#pragma unroll
      for (int u = 0; u < U; ++u) pack(r[u], i + u * THREADS);
    }
    for (; i < sp.v1; i += THREADS) pack(xv[i], i);
  } else {                                                            // x and d begin at different places of 16 bytes
    for (int i = sp.v0 * VE + threadIdx.x; i < sp.v1 * VE; i += THREADS) dv[i] = (T)value(widen(xr[sp.first + i]));
  }
  if (!off) kd_write_entries(a, xr, dr, sp, rw, scale, id_lds, t_lds);
}

// What a block of N threads that has a row to itself makes of their (m, s) and teacher entries (t, t + N, ..: id -1 for none,
// its t and its logit xt): the row's statistics and loss, in every thread.  red: [4][waves].
struct KdDone { KdRow rw; float loss; };
template <int N> struct KdEntries { int id[KD_MAX_K / N]; float tv[KD_MAX_K / N], xt[KD_MAX_K / N], e[KD_MAX_K / N]; };
template <int N>
__device__ __forceinline__ KdDone kd_finish_row(const KdArgs& a, float m, float s, KdEntries<N>& te, float (*red)[N / 64]) {
  constexpr int W = N / 64, KD_E = KD_MAX_K / N;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float c = a.c;
  float tm = -INFINITY;
  bool some = false;
#pragma unroll
  for (int x = 0; x < KD_E; ++x)
    if (te.id[x] >= 0) { tm = fmaxf(tm, te.tv[x]); some = true; }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    kd_join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), c);
    tm = fmaxf(tm, __shfl_xor(tm, o, 64));
  }
  some = __ballot(some) != 0;
  if (lane == 0) { red[0][wave] = m; red[1][wave] = s; red[2][wave] = tm; red[3][wave] = some ? 1.f : 0.f; }
  __syncthreads();
  const bool any = __ballot(red[3][lane & (W - 1)] != 0.f) != 0;
  m = red[0][lane & (W - 1)]; s = red[1][lane & (W - 1)]; tm = red[2][lane & (W - 1)];
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    kd_join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), c);
    tm = fmaxf(tm, __shfl_xor(tm, o, 64));
  }
  // the teacher's sum and the loss: q = e / sum e
  float ts = 0.f, gap = 0.f;
#pragma unroll
  for (int x = 0; x < KD_E; ++x) {
    te.e[x] = te.id[x] >= 0 ? kd_exp2((te.tv[x] - tm) * c) : 0.f;
    ts += te.e[x];
    if (!(te.e[x] == 0.f)) gap += te.e[x] * kd_gap(te.tv[x], tm, te.xt[x], m);
  }
  ts = wave_sum(ts); gap = wave_sum(gap);
  __syncthreads();
  if (lane == 0) { red[0][wave] = ts; red[1][wave] = gap; }
  __syncthreads();
  ts = red[0][lane & (W - 1)]; gap = red[1][lane & (W - 1)];
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) { ts += __shfl_xor(ts, o, 64); gap += __shfl_xor(gap, o, 64); }
  const bool off = !any || (m == -INFINITY && s == 0.f);
  const float loss = off ? 0.f : kd_loss_of(a.temp, gap / ts, s, ts);
  return KdDone{KdRow{m, off ? 0.f : s, tm, off ? 0.f : ts}, loss};
}

// ---- a row per block: statistics, loss and (d given) the gradient of its own loss, for which the row is read again.  At 1024
// threads two blocks share a CU, and the rows in work (133 MB of 260 KB rows) stay in the Infinity Cache; more, smaller blocks
// push them out (4096 x 130000 in bf16: 1024 threads 547 us, 512 594, 256 699).  Rows up to KD_SHORT bytes take 512 threads
// (1021 x 32771 in fp16, loss only: 17 us against 21).  Keeping part of a row on the CU -- 272 KB of registers and LDS, one
// block per CU, each place filled with the next row's access as its gradient leaves -- took 595 us beside those 547 (nothing moves
// while it adds up), two smaller blocks with half a row kept 537: two percent, not worth a second kernel.
constexpr int64_t KD_SHORT = 128 << 10;
template <typename T, int N>
__global__ __launch_bounds__(N) void kd_row_kernel(const KdArgs a) {
  __shared__ int id_lds[KD_MAX_K];
  __shared__ float t_lds[KD_MAX_K], red[4][N / 64];
  const int64_t row = blockIdx.x;
  const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
  const KdSpan<T> sp(xr, a.v, 0, 1);
  float m = -INFINITY, s = 0.f;
  kd_load_teacher(a.te, row, a.v, id_lds, t_lds);
  kd_stats<T, N>(xr, sp, a.c, m, s);
  KdEntries<N> te;
#pragma unroll
  for (int x = 0; x < KD_MAX_K / N; ++x) {
    const int j = threadIdx.x + x * N;
    te.id[x] = j < a.te.k ? id_lds[j] : -1;
    te.tv[x] = te.id[x] >= 0 ? t_lds[j] : 0.f;
    te.xt[x] = te.id[x] >= 0 ? widen(xr[te.id[x]]) : 0.f;
  }
  const KdDone done = kd_finish_row<N>(a, m, s, te, red);
  if (threadIdx.x == 0) {
    a.losses[row] = done.loss;
    a.rows[row] = done.rw;
  }
  if (a.d) kd_write_grad<T, N>(a, xr, static_cast<T*>(a.d) + row * a.ldd, sp, done.rw, a.coef, id_lds, t_lds);
}

// scale * the sum of the rows' losses, in a fixed order (one block).  FRESH: written by other blocks of this launch, past the L2
template <int N, bool FRESH>
__device__ __forceinline__ void kd_sum(const float* losses, int64_t n, float scale, float* red, float* __restrict__ out) {
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += N)
    s += FRESH ? __hip_atomic_load(losses + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : losses[i];
  s = kd_block_sum(s, red);
  if (threadIdx.x == 0) out[0] = scale * s;
}
__global__ __launch_bounds__(1024) void kd_sum_kernel(const float* __restrict__ losses, int64_t n, float scale,
                                                      float* __restrict__ out) {
  __shared__ float red[16];
  kd_sum<1024, false>(losses, n, scale, red, out);
}

// ---- few rows: a.parts blocks share one.  First the parts' statistics ...
template <typename T>
__global__ __launch_bounds__(KD_THREADS) void kd_part_kernel(const KdArgs a) {
  __shared__ float red[2 * KD_THREADS / 64];
  const int64_t row = blockIdx.x / a.parts;
  const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
  const KdSpan<T> sp(xr, a.v, blockIdx.x % a.parts, a.parts);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.done = 0;      // (counted by the next launch)
  float m = -INFINITY, s = 0.f;
  kd_stats<T, KD_THREADS>(xr, sp, a.c, m, s);
  kd_block_join<KD_THREADS>(m, s, a.c, red);
  if (threadIdx.x == 0) { a.part[2 * (int64_t)blockIdx.x] = m; a.part[2 * (int64_t)blockIdx.x + 1] = s; }
}
// ... then, joined, the row's loss (part 0) and the parts' gradients (d given; else the grid is one block per row)
template <typename T>
__global__ __launch_bounds__(KD_THREADS) void kd_join_kernel(const KdArgs a) {
  __shared__ int id_lds[KD_MAX_K];
  __shared__ float t_lds[KD_MAX_K], red[2 * KD_THREADS / 64];
  const int64_t row = a.d ? blockIdx.x / a.parts : blockIdx.x;
  const int p = a.d ? blockIdx.x % a.parts : 0;
  const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
  kd_load_teacher(a.te, row, a.v, id_lds, t_lds);
  float m = -INFINITY, s = 0.f, tm, ts;
  for (int i = threadIdx.x; i < a.parts; i += KD_THREADS)
    kd_join(m, s, a.part[2 * (row * a.parts + i)], a.part[2 * (row * a.parts + i) + 1], a.c);
  kd_block_join<KD_THREADS>(m, s, a.c, red);
  kd_teacher_softmax(a.te.k, a.c, id_lds, t_lds, red, tm, ts);
  const bool off = ts == 0.f || (m == -INFINITY && s == 0.f);
  const KdRow rw{m, off ? 0.f : s, tm, off ? 0.f : ts};
  if (p == 0) {
    const float loss = kd_loss(a, xr, id_lds, t_lds, m, s, tm, ts, red);
    if (threadIdx.x == 0) {
      __hip_atomic_store(a.losses + row, off ? 0.f : loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      a.rows[row] = rw;
    }
  }
  // Which block is the last does not change the sum's order.  A row's loss goes past the L2 by itself and is waited for: a fence
  // for the device would write back all that the XCD's L2 holds of the gradients (128 x 130000 in fp32: this launch took 63 us with it, 30 without).
  if (p == 0 && a.loss) {
    __shared__ bool last;
    if (threadIdx.x == 0) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      last = __hip_atomic_fetch_add(a.done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)a.n_rows - 1;
      asm volatile("" ::: "memory");
    }
    __syncthreads();
    if (last) kd_sum<KD_THREADS, true>(a.losses, a.n_rows, a.sum_scale, red, a.loss);
  }
  if (a.d) {
    const KdSpan<T> sp(xr, a.v, p, a.parts);
    kd_write_grad<T, KD_THREADS>(a, xr, static_cast<T*>(a.d) + row * a.ldd, sp, rw, a.coef, id_lds, t_lds);
  }
}

// ---- the gradient from the kept row statistics.  unless_one: d already holds the gradient for g = 1.
template <typename T>
__global__ __launch_bounds__(KD_THREADS) void kd_regrad_kernel(const KdArgs a, int unless_one) {
  __shared__ int id_lds[KD_MAX_K];
  __shared__ float t_lds[KD_MAX_K];
  if (unless_one && a.g[0] == 1.f) return;
  for (int64_t b = blockIdx.x; b < a.n_rows * a.parts; b += gridDim.x) {
    const int64_t row = b / a.parts;
    const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
    const KdSpan<T> sp(xr, a.v, (int)(b % a.parts), a.parts);
    __syncthreads();                                                  // (the entries of the block's last row are done with)
    kd_load_teacher(a.te, row, a.v, id_lds, t_lds);
    kd_write_grad<T, KD_THREADS>(a, xr, static_cast<T*>(a.d) + row * a.ldd, sp, a.rows[row], a.g[row * a.g_step] * a.coef, id_lds,
                                 t_lds);
  }
}

// blocks per row: enough to give every CU a few, with at least 8 KB of a row each
static int kd_parts(int64_t rows, int64_t v, int e) {
  const int64_t want = (2048 + rows - 1) / rows, most = (v * e + 8191) / 8192;
  return (int)(want < 1 ? 1 : want < most ? want : most < 1 ? 1 : most);
}

static int kd_check(const char* who, const void* x, int32_t type, int64_t ldx, int64_t rows, int64_t v, int32_t k, int32_t t_type,
                    float temp) {
  BKG_ARG(x && type >= 0 && type <= 2 && t_type >= 0 && t_type <= 2, "bkg_distill: null logits or unknown type");
  BKG_ARG(rows > 0 && v > 0 && v < (1ll << 30) && ldx >= 0 && rows < (1ll << 22), "bkg_distill: rows in (0, 2^22), columns in (0, 2^30)");
  BKG_ARG(k > 0 && k <= KD_MAX_K, "bkg_distill: between 1 and 1024 teacher entries per row");
  BKG_ARG(temp >= 1e-18f && temp <= 1e18f, "bkg_distill: the temperature must lie between 1e-18 and 1e18");
  BKG_ARG((uintptr_t)x % type_bytes(type) == 0, "bkg_distill: misaligned logits");
  return 0;
}

}  // namespace bkg

using namespace bkg;

#define BKG_BY_TYPE(type, ...)                          \
  do {                                                   \
    if ((type) == BKG_T_F32) { using T = float; __VA_ARGS__; }  \
    else if ((type) == BKG_T_BF16) { using T = __bf16; __VA_ARGS__; } \
    else { using T = _Float16; __VA_ARGS__; }                   \
  } while (0)

extern "C" int64_t bkg_distill_workspace_floats(int64_t rows, int64_t v, int32_t type) {
  return rows <= 0 || v <= 0 ? 0 : 2 * rows * kd_parts(rows, v, type_bytes(type)) + 1;
}

// Few rows are shared by several blocks; from 192 rows on a block per row keeps three quarters of the CUs or more at work.
static bool kd_row_per_block(int64_t rows) { return rows >= 192; }

extern "C" int bkg_distill_forward(const void* x, int32_t type, int64_t ldx, int64_t rows, int64_t v, const void* ids,
                                   int32_t ids_i32, int64_t ld_ids, const void* t, int32_t t_type, int64_t ld_t, int32_t k,
                                   float temp, float sum_scale, float* workspace, float* row_stats, float* losses, float* loss,
                                   void* d, int64_t ldd, void* stream) {
  if (const int rc = kd_check("bkg_distill_forward", x, type, ldx, rows, v, k, t_type, temp)) return rc;
  BKG_ARG(ids && t && workspace && row_stats && losses, "bkg_distill_forward: null buffer");
  const int e = type_bytes(type);
  BKG_ARG(!d || (ldd >= v && (uintptr_t)d % e == 0), "bkg_distill_forward: misaligned gradient or overlapping rows");
  hipStream_t s = (hipStream_t)stream;
  KdArgs a{x, ldx, (int)v, kd_parts(rows, v, e), KD_LOG2E / temp, temp, {ids, ids_i32, ld_ids, t, t_type, ld_t, k},
           workspace, (KdRow*)row_stats, losses, d, ldd, nullptr, 0, temp * sum_scale, rows, rows * v * e > STREAM_BYTES,
           (unsigned*)(workspace + 2 * rows * kd_parts(rows, v, e)), loss, sum_scale};
  if (kd_row_per_block(rows) && v * e <= KD_SHORT) {
    BKG_BY_TYPE(type, hipLaunchKernelGGL((kd_row_kernel<T, 512>), dim3((unsigned)rows), dim3(512), 0, s, a));
  } else if (kd_row_per_block(rows)) {
    BKG_BY_TYPE(type, hipLaunchKernelGGL((kd_row_kernel<T, 1024>), dim3((unsigned)rows), dim3(1024), 0, s, a));
  } else {
    BKG_BY_TYPE(type, hipLaunchKernelGGL((kd_part_kernel<T>), dim3((unsigned)(rows * a.parts)), dim3(KD_THREADS), 0, s, a));
    BKG_BY_TYPE(type, hipLaunchKernelGGL((kd_join_kernel<T>), dim3((unsigned)(d ? rows * a.parts : rows)), dim3(KD_THREADS), 0, s, a));
  }
  if (loss && kd_row_per_block(rows)) hipLaunchKernelGGL(kd_sum_kernel, dim3(1), dim3(1024), 0, s, losses, rows, sum_scale, loss);
  return check_launch("bkg_distill_forward");
}

extern "C" int bkg_distill_backward(const void* x, int32_t type, int64_t ldx, int64_t rows, int64_t v, const void* ids,
                                    int32_t ids_i32, int64_t ld_ids, const void* t, int32_t t_type, int64_t ld_t, int32_t k,
                                    float temp, const float* row_stats, const float* g, int32_t g_step, float coef,
                                    int32_t unless_one, void* d, int64_t ldd, void* stream) {
  if (const int rc = kd_check("bkg_distill_backward", x, type, ldx, rows, v, k, t_type, temp)) return rc;
  const int e = type_bytes(type);
  BKG_ARG(ids && t && row_stats && g && d && ldd >= v && (uintptr_t)d % e == 0, "bkg_distill_backward: null or misaligned buffer");
  BKG_ARG(!unless_one || g_step == 0, "bkg_distill_backward: a kept gradient has one upstream factor");
  hipStream_t s = (hipStream_t)stream;
  KdArgs a{x, ldx, (int)v, kd_parts(rows, v, e), KD_LOG2E / temp, temp, {ids, ids_i32, ld_ids, t, t_type, ld_t, k},
           nullptr, (KdRow*)row_stats, nullptr, d, ldd, g, g_step, coef, rows, rows * v * e > STREAM_BYTES, nullptr, nullptr, 0.f};
  // (a launch that may have nothing to do keeps its grid small and loops)
  const int64_t all = rows * a.parts, grid = unless_one && all > 2048 ? 2048 : all;
  BKG_BY_TYPE(type, hipLaunchKernelGGL((kd_regrad_kernel<T>), dim3((unsigned)grid), dim3(KD_THREADS), 0, s, a, unless_one));
  return check_launch("bkg_distill_backward");
}
