// Distillation of a row of logits from a teacher's K best entries.
//
// x [R, V] student logits, (id, t) [R, K] the teacher's entries, temperature T.  An entry is usable if 0 <= id < V and t is
// not -inf.  With p = softmax(x / T) over all V columns and q = softmax(t / T) over the row's usable entries,
//     L_r = T^2 sum_j q_j (ln q_j - ln p_{id_j}),        dL_r / dx = T (p - q)
// (an id that occurs twice takes both entries' q).  A row without a usable entry, or whose logits are all -inf, is left out:
// loss 0, gradient 0.  K = 1 is cross entropy.
//
// Bound by HBM: the forward reads x once (running maximum and sum of exponentials in fp32, one pass), the backward reads x
// and writes its gradient.
#include "rowtypes.h"

namespace bkg {

constexpr int KD_THREADS = 256;
constexpr int KD_MAX_K = 1024;
constexpr float KD_LOG2E = 1.4426950408889634f, KD_LN2 = 0.6931471805599453f;

struct KdTeacher {
  const void* ids; int ids_i32; int64_t ld_ids;
  const void* t; int t_type; int64_t ld_t;
  int k;
};
struct KdRow { float m, sum, tmax, tsum; };      // max and sum of exp of x / T around it; the same of the usable entries.
                                                 // tsum = 0: no usable entry; sum = 0: the logits are all -inf

__device__ __forceinline__ float kd_exp(float v) { return __builtin_amdgcn_exp2f(v); }

// (m, s) joined with (m2, s2): s exp(m) + s2 exp(m2); c = log2(e) / T.  -inf maxima carry s = 0 or NaN.
__device__ __forceinline__ void kd_join(float& m, float& s, float m2, float s2, float c) {
  const float mm = fmaxf(m, m2), ref = mm == -INFINITY ? 0.f : mm;
  s = s * kd_exp((m - ref) * c) + s2 * kd_exp((m2 - ref) * c);
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

// per-row partial (max, sum): part[(row * parts + p) * 2]
template <typename T>
__global__ __launch_bounds__(KD_THREADS) void kd_stats_kernel(const T* __restrict__ x, int64_t ldx, int v, int parts, float c,
                                                              float* __restrict__ part) {
  constexpr int VE = KdSpan<T>::VE, U = 4;
  __shared__ float red_m[KD_THREADS / 64], red_s[KD_THREADS / 64];
  const int64_t row = blockIdx.x / parts;
  const int p = blockIdx.x % parts;
  const T* xr = x + row * ldx;
  const KdSpan<T> sp(xr, v, p, parts);
  const Pack<T, VE>* xv = reinterpret_cast<const Pack<T, VE>*>(xr + sp.first);
  float m = -INFINITY, s = 0.f;
  auto one = [&](float f) {
    if (f > m) { s *= kd_exp((m - f) * c); m = f; }                  // (s = 0 while m = -inf)
    s += kd_exp((f - (m == -INFINITY ? 0.f : m)) * c);
  };
  for (int i = threadIdx.x; i < sp.head; i += KD_THREADS) one(widen(xr[i]));
  for (int i = sp.tail0 + threadIdx.x; i < sp.tail1; i += KD_THREADS) one(widen(xr[i]));
  for (int i = sp.v0 + threadIdx.x; i < sp.v1; i += KD_THREADS * U) {
    Pack<T, VE> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * KD_THREADS < sp.v1) r[u] = xv[i + u * KD_THREADS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * KD_THREADS >= sp.v1) break;
      float f[VE], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < VE; ++j) { f[j] = widen(r[u].v[j]); top = fmaxf(top, f[j]); }
      if (top > m) { s *= kd_exp((m - top) * c); m = top; }
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int j = 0; j < VE; ++j) s += kd_exp((f[j] - ref) * c);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) kd_join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), c);
  if ((threadIdx.x & 63) == 0) { red_m[threadIdx.x >> 6] = m; red_s[threadIdx.x >> 6] = s; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < KD_THREADS / 64; ++w) kd_join(m, s, red_m[w], red_s[w], c);
    part[2 * (int64_t)blockIdx.x] = m;
    part[2 * (int64_t)blockIdx.x + 1] = s;
  }
}

// The row's teacher entries into LDS: id (or -1 where not usable) and t; returns (tmax, tsum).
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

// One block per row: the parts joined, the teacher's softmax, the loss; rows[row] keeps what the backward needs.
template <typename T>
__global__ __launch_bounds__(KD_THREADS) void kd_rows_kernel(const T* __restrict__ x, int64_t ldx, int v, int parts, float c,
                                                             float temp, const KdTeacher te, const float* __restrict__ part,
                                                             KdRow* __restrict__ rows, float* __restrict__ losses) {
  __shared__ int id_lds[KD_MAX_K];
  __shared__ float t_lds[KD_MAX_K], red[KD_THREADS / 64];
  const int64_t row = blockIdx.x;
  float m = -INFINITY, s = 0.f;
  for (int p = 0; p < parts; ++p) kd_join(m, s, part[2 * (row * parts + p)], part[2 * (row * parts + p) + 1], c);
  kd_load_teacher(te, row, v, id_lds, t_lds);
  float tm = -INFINITY;
  bool any = false;
  for (int j = threadIdx.x; j < te.k; j += KD_THREADS)
    if (id_lds[j] >= 0) { tm = fmaxf(tm, t_lds[j]); any = true; }
  tm = kd_block_max(tm, red);
  any = __syncthreads_or(any);
  float ts = 0.f;
  for (int j = threadIdx.x; j < te.k; j += KD_THREADS)
    if (id_lds[j] >= 0) ts += kd_exp((t_lds[j] - tm) * c);
  ts = kd_block_sum(ts, red);
  const float ln_s = KD_LN2 * __builtin_amdgcn_logf(s), ln_ts = KD_LN2 * __builtin_amdgcn_logf(ts);
  const float inv_t = c * KD_LN2, inv_ts = 1.f / ts;
  float loss = 0.f;
  for (int j = threadIdx.x; j < te.k; j += KD_THREADS) {
    if (id_lds[j] < 0) continue;
    const float q = kd_exp((t_lds[j] - tm) * c) * inv_ts;
    const float ln_q = (t_lds[j] - tm) * inv_t - ln_ts, ln_p = (widen(x[row * ldx + id_lds[j]]) - m) * inv_t - ln_s;
    if (!(q == 0.f)) loss += q * (ln_q - ln_p);
  }
  loss = kd_block_sum(loss, red);
  if (threadIdx.x == 0) {
    const bool off = !any || (m == -INFINITY && s == 0.f);
    losses[row] = off ? 0.f : temp * temp * loss;
    rows[row] = KdRow{m, off ? 0.f : s, tm, off ? 0.f : ts};
  }
}

// out[0] = scale * sum of the rows' losses, in a fixed order
__global__ __launch_bounds__(1024) void kd_sum_kernel(const float* __restrict__ losses, int64_t n, float scale,
                                                      float* __restrict__ out) {
  __shared__ float red[16];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += losses[i];
  s = kd_block_sum(s, red);
  if (threadIdx.x == 0) out[0] = scale * s;
}

// d[row, :] = g_row * coef * (p - q); g: one value per row (g_step = 1) or one for all (0)
template <typename T>
__global__ __launch_bounds__(KD_THREADS) void kd_grad_kernel(const T* __restrict__ x, int64_t ldx, int v, int parts, float c,
                                                             const KdTeacher te, const KdRow* __restrict__ rows,
                                                             const float* __restrict__ g, int g_step, float coef,
                                                             T* __restrict__ d, int64_t ldd, int same_phase) {
  constexpr int VE = KdSpan<T>::VE;
  __shared__ int id_lds[KD_MAX_K];
  __shared__ float q_lds[KD_MAX_K];
  const int64_t row = blockIdx.x / parts;
  const int p = blockIdx.x % parts;
  const T* xr = x + row * ldx;
  T* dr = d + row * ldd;
  const KdSpan<T> sp(xr, v, p, parts);
  const KdRow rw = rows[row];
  const bool off = rw.tsum == 0.f && rw.sum == 0.f;
  const float scale = g[row * g_step] * coef, ps = off ? 0.f : scale / rw.sum;
  auto value = [&](float f) { return off ? 0.f : kd_exp((f - rw.m) * c) * ps; };
  for (int i = threadIdx.x; i < sp.head; i += KD_THREADS) dr[i] = (T)value(widen(xr[i]));
  for (int i = sp.tail0 + threadIdx.x; i < sp.tail1; i += KD_THREADS) dr[i] = (T)value(widen(xr[i]));
  const Pack<T, VE>* xv = reinterpret_cast<const Pack<T, VE>*>(xr + sp.first);
  for (int i = sp.v0 + threadIdx.x; i < sp.v1; i += KD_THREADS) {
    Pack<T, VE> r = xv[i];
#pragma unroll
    for (int j = 0; j < VE; ++j) r.v[j] = (T)value(widen(r.v[j]));
    if (same_phase) *(reinterpret_cast<Pack<T, VE>*>(dr + sp.first) + i) = r;
    else
#pragma unroll
      for (int j = 0; j < VE; ++j) dr[sp.first + i * VE + j] = r.v[j];
  }
  if (off) return;
  kd_load_teacher(te, row, v, id_lds, q_lds);                         // (its barrier also orders the stores above)
  const float inv_ts = 1.f / rw.tsum;
  for (int j = threadIdx.x; j < te.k; j += KD_THREADS) q_lds[j] = kd_exp((q_lds[j] - rw.tmax) * c) * inv_ts;
  __syncthreads();
  for (int j = threadIdx.x; j < te.k; j += KD_THREADS) {              // the entries' columns are written again, whole
    const int id = id_lds[j];
    if (id < 0 || !sp.mine(id)) continue;
    bool first = true;
    for (int i = 0; i < j; ++i) first = first && id_lds[i] != id;
    if (!first) continue;
    float q = 0.f;
    for (int i = j; i < te.k; ++i) q += id_lds[i] == id ? q_lds[i] : 0.f;
    dr[id] = (T)(value(widen(xr[id])) - scale * q);
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
  BKG_ARG(rows > 0 && v > 0 && v < (1ll << 30) && ldx >= 0 && rows < (1ll << 24), "bkg_distill: rows in (0, 2^24), columns in (0, 2^30)");
  BKG_ARG(k > 0 && k <= KD_MAX_K, "bkg_distill: between 1 and 1024 teacher entries per row");
  BKG_ARG(temp > 0.f && temp < INFINITY, "bkg_distill: the temperature must be positive and finite");
  BKG_ARG((uintptr_t)x % type_bytes(type) == 0, "bkg_distill: misaligned logits");
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

extern "C" int64_t bkg_distill_workspace_floats(int64_t rows, int64_t v, int32_t type) {
  return rows <= 0 || v <= 0 ? 0 : 2 * rows * kd_parts(rows, v, type_bytes(type));
}

extern "C" int bkg_distill_forward(const void* x, int32_t type, int64_t ldx, int64_t rows, int64_t v, const void* ids,
                                   int32_t ids_i32, int64_t ld_ids, const void* t, int32_t t_type, int64_t ld_t, int32_t k,
                                   float temp, float sum_scale, float* workspace, float* row_stats, float* losses, float* loss,
                                   void* stream) {
  if (const int rc = kd_check("bkg_distill_forward", x, type, ldx, rows, v, k, t_type, temp)) return rc;
  BKG_ARG(ids && t && workspace && row_stats && losses, "bkg_distill_forward: null buffer");
  hipStream_t s = (hipStream_t)stream;
  const int parts = kd_parts(rows, v, type_bytes(type));
  const float c = KD_LOG2E / temp;
  const KdTeacher te{ids, ids_i32, ld_ids, t, t_type, ld_t, k};
  BKG_BY_TYPE(type, hipLaunchKernelGGL((kd_stats_kernel<T>), dim3((unsigned)(rows * parts)), dim3(KD_THREADS), 0, s, (const T*)x,
                                       ldx, (int)v, parts, c, workspace));
  BKG_BY_TYPE(type, hipLaunchKernelGGL((kd_rows_kernel<T>), dim3((unsigned)rows), dim3(KD_THREADS), 0, s, (const T*)x, ldx, (int)v,
                                       parts, c, temp, te, workspace, (KdRow*)row_stats, losses));
  if (loss) hipLaunchKernelGGL(kd_sum_kernel, dim3(1), dim3(1024), 0, s, losses, rows, sum_scale, loss);
  return check_launch("bkg_distill_forward");
}

extern "C" int bkg_distill_backward(const void* x, int32_t type, int64_t ldx, int64_t rows, int64_t v, const void* ids,
                                    int32_t ids_i32, int64_t ld_ids, const void* t, int32_t t_type, int64_t ld_t, int32_t k,
                                    float temp, const float* row_stats, const float* g, int32_t g_step, float coef, void* d,
                                    int64_t ldd, void* stream) {
  if (const int rc = kd_check("bkg_distill_backward", x, type, ldx, rows, v, k, t_type, temp)) return rc;
  const int e = type_bytes(type);
  BKG_ARG(ids && t && row_stats && g && d && ldd >= v && (uintptr_t)d % e == 0, "bkg_distill_backward: null or misaligned buffer");
  hipStream_t s = (hipStream_t)stream;
  const int parts = kd_parts(rows, v, e);
  const float c = KD_LOG2E / temp;
  const KdTeacher te{ids, ids_i32, ld_ids, t, t_type, ld_t, k};
  const int same = ((uintptr_t)x - (uintptr_t)d) % 16 == 0 && ((ldx - ldd) * e) % 16 == 0;
  BKG_BY_TYPE(type, hipLaunchKernelGGL((kd_grad_kernel<T>), dim3((unsigned)(rows * parts)), dim3(KD_THREADS), 0, s, (const T*)x,
                                       ldx, (int)v, parts, c, te, (const KdRow*)row_stats, g, g_step, coef, (T*)d, ldd, same));
  return check_launch("bkg_distill_backward");
}
