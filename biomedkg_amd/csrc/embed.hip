// Embedding lookup with scaling and the table's gradient by sorted ids.
//
//   out[i] = scale * W[id_i]                          (one rounding, from fp32)
//   dW[v]  = scale * sum over {i : id_i = v} of g[i]  (fp32 sums in a fixed order, one rounding; rows nobody looked up: 0)
//
// An id outside [0, V) reads as a row of zeros and gets no gradient (padded batches); `pad` reads its row and gets none.
// Both directions move bytes and compute nothing: bound by HBM (the lookup's random rows by the fabric).
//
// The gradient needs no atomics: the ids are sorted (stable, carrying positions), and every run of equal ids is summed in
// position order.  Runs are very uneven in a graph -- most entities occur a few times, a hub in a percent of all edges -- so
// the work is cut by ENTRIES, not by rows: a lane group takes the runs that start in its chunk of sorted entries.  A run
// longer than EG_LONG entries is left out there and summed by windows of EG_LONG entries (one lane group each) whose fp32
// partial rows a last launch adds in order.
#include "rowtypes.h"

namespace bkg {

constexpr int EG_LONG = 64;
constexpr int EG_PAD = EG_LONG + 2 * 8;             // words behind the sorted entries that steps of 8 and looks ahead reach
constexpr int64_t EMBED_MAX_D = 1 << 20;            // (column tiles are the grid's y extent)

__device__ __forceinline__ int64_t embed_id(const void* __restrict__ ids, int ids_i32, int64_t i) {
  return ids_i32 ? (int64_t)static_cast<const int32_t*>(ids)[i] : static_cast<const int64_t*>(ids)[i];
}

// A lane group of 2^lpr_log2 lanes copies a row's VEC-wide columns of tile blockIdx.y; UNROLL rows in flight per group.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_rows_kernel(const T* __restrict__ w, int64_t ldw, int64_t n_rows, int d,
                                                         const void* __restrict__ ids, int ids_i32, int64_t n, float scale,
                                                         T* __restrict__ out, int64_t ldo, int lpr_log2) {
  constexpr int UNROLL = 4;
  const int lig = threadIdx.x & ((1 << lpr_log2) - 1), groups = 256 >> lpr_log2;
  const int c = (((int)blockIdx.y << lpr_log2) + lig) * VEC;
  if (c >= d) return;
  const int64_t i0 = ((int64_t)blockIdx.x * groups + (threadIdx.x >> lpr_log2)) * UNROLL;
  Pack<T, VEC> r[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int64_t i = i0 + u;
#pragma unroll
    for (int j = 0; j < VEC; ++j) r[u].v[j] = (T)0.f;
    if (i < n) {
      const int64_t id = embed_id(ids, ids_i32, i);
      if (id >= 0 && id < n_rows) r[u] = *reinterpret_cast<const Pack<T, VEC>*>(w + id * ldw + c);
    }
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int64_t i = i0 + u;
    if (i >= n) break;
#pragma unroll
    for (int j = 0; j < VEC; ++j) r[u].v[j] = (T)(widen(r[u].v[j]) * scale);
    *reinterpret_cast<Pack<T, VEC>*>(out + i * ldo + c) = r[u];
  }
}

struct EmbedGradArgs {
  const uint32_t* keys; const uint32_t* perm;      // [n] sorted (key n_rows = no gradient), then EG_PAD all-ones words
  int64_t n, n_rows;
  float scale;
  int d, lpr_log2, chunk;
  int64_t n_chunks;                                // lane groups over entries; the rest of the grid are windows
  int64_t n_windows;
  float* part;                                     // [2 n_windows][d] partial rows of long runs (2 j: the run over window j's
};                                                 // first entry, 2 j + 1: the run that starts inside it and leaves it)

// Is the run of key k around entry p (keys[p] == k) longer than EG_LONG entries?  It is iff the entries of k within
// EG_LONG of p on either side are more than EG_LONG; the ends by binary search.
__device__ __forceinline__ bool run_is_long(const uint32_t* __restrict__ keys, int64_t n, int64_t p, uint32_t k) {
  int64_t lo = p - EG_LONG < 0 ? 0 : p - EG_LONG, hi = p;        // first entry of k in [p - EG_LONG, p]
  while (lo < hi) { const int64_t m = (lo + hi) >> 1; if (keys[m] < k) lo = m + 1; else hi = m; }
  const int64_t beg = lo;
  lo = p + 1; hi = p + EG_LONG + 1 > n ? n : p + EG_LONG + 1;    // first entry past k in (p, p + EG_LONG]
  while (lo < hi) { const int64_t m = (lo + hi) >> 1; if (keys[m] <= k) lo = m + 1; else hi = m; }
  return lo - beg > EG_LONG;
}

constexpr int EG_U = 8;                            // entries per step: their rows are in flight together
struct EgWords { uint32_t w[EG_U]; };
__device__ __forceinline__ EgWords eg_words(const uint32_t* __restrict__ p) {      // (32-byte aligned; reads into the pad)
  EgWords o;
  const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
  o.w[0] = a.x; o.w[1] = a.y; o.w[2] = a.z; o.w[3] = a.w;
  o.w[4] = b.x; o.w[5] = b.y; o.w[6] = b.z; o.w[7] = b.w;
  return o;
}

template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_grad_kernel(const EmbedGradArgs a, const T* __restrict__ g, int64_t ldg,
                                                         T* __restrict__ dw, int64_t ldw) {
  const int lig = threadIdx.x & ((1 << a.lpr_log2) - 1), groups = 256 >> a.lpr_log2;
  const int c = (((int)blockIdx.y << a.lpr_log2) + lig) * VEC;
  if (c >= a.d) return;
  const int64_t group = (int64_t)blockIdx.x * groups + (threadIdx.x >> a.lpr_log2);
  const T* gc = g + c;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  if (group < a.n_chunks) {                                     // ---- the runs that start in these entries
    const int64_t beg = group * a.chunk, last = beg + a.chunk < a.n ? beg + a.chunk : a.n;
    uint32_t cur = beg > 0 ? a.keys[beg - 1] : 0xFFFFFFFFu;
    bool mine = false;                                          // is `cur` a run of this group (and not a long one)?
    EgWords k = eg_words(a.keys + beg), pm = eg_words(a.perm + beg), kl = eg_words(a.keys + beg + EG_LONG);
    for (int64_t e = beg; e < last || mine; e += EG_U) {
      bool live[EG_U];
      Pack<T, VEC> r[EG_U];
      uint32_t run = cur;
      bool on = mine;
#pragma unroll
      for (int u = 0; u < EG_U; ++u) {
        if (k.w[u] != run) {
          run = k.w[u];
          on = e + u < last && run < (uint32_t)a.n_rows && kl.w[u] != run;
        }
        live[u] = on;
      }
#pragma unroll
      for (int u = 0; u < EG_U; ++u)
        if (live[u]) r[u] = *reinterpret_cast<const Pack<T, VEC>*>(gc + (int64_t)pm.w[u] * ldg);
      const EgWords kn = k;
      const int64_t en = e + EG_U < a.n ? e + EG_U : e;         // (a group that stops here reads its own entries again)
      k = eg_words(a.keys + en); pm = eg_words(a.perm + en); kl = eg_words(a.keys + en + EG_LONG);
      if (en == e)
#pragma unroll
        for (int u = 0; u < EG_U; ++u) k.w[u] = 0xFFFFFFFFu;
#pragma unroll
      for (int u = 0; u < EG_U; ++u) {
        if (kn.w[u] != cur) {
          if (mine) {
            Pack<T, VEC> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) { o.v[j] = (T)(acc[j] * a.scale); acc[j] = 0.f; }
            *reinterpret_cast<Pack<T, VEC>*>(dw + (int64_t)cur * ldw + c) = o;
          }
          cur = kn.w[u];
          mine = live[u];
        }
        if (live[u])
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += widen(r[u].v[j]);
      }
    }
    return;
  }
  // ---- a window of EG_LONG entries: the parts of long runs in it
  const int64_t j = group - a.n_chunks;
  if (j >= a.n_windows) return;
  const int64_t p = j * EG_LONG, q = p + EG_LONG < a.n ? p + EG_LONG : a.n;
  const uint32_t k0 = a.keys[p], k1 = a.keys[q - 1];
  // (candidates by one look each: a run longer than EG_LONG that covers the window's first entry either covers the whole
  // window or reaches back past it)
  const bool head = k0 < (uint32_t)a.n_rows && (k1 == k0 || (p > 0 && a.keys[p - 1] == k0)) && run_is_long(a.keys, a.n, p, k0);
  const bool tail = k1 != k0 && q < a.n && a.keys[q] == k1 && k1 < (uint32_t)a.n_rows && run_is_long(a.keys, a.n, q - 1, k1);
  for (int which = 0; which < 2; ++which) {
    if (!(which ? tail : head)) continue;
    const uint32_t key = which ? k1 : k0;
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
    EgWords k = eg_words(a.keys + p), pm = eg_words(a.perm + p);
    for (int64_t e = p; e < q; e += EG_U) {
      Pack<T, VEC> r[EG_U];
#pragma unroll
      for (int u = 0; u < EG_U; ++u)
        if (k.w[u] == key) r[u] = *reinterpret_cast<const Pack<T, VEC>*>(gc + (int64_t)pm.w[u] * ldg);
      const EgWords kn = k;
      k = eg_words(a.keys + e + EG_U); pm = eg_words(a.perm + e + EG_U);
#pragma unroll
      for (int u = 0; u < EG_U; ++u)
        if (kn.w[u] == key)
#pragma unroll
          for (int v = 0; v < VEC; ++v) acc[v] += widen(r[u].v[v]);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) a.part[(2 * j + which) * a.d + c + v] = acc[v];
  }
}

// Window j in which a long run starts adds that run's partial rows and writes the row: four waves take a quarter of the
// windows each, in order, and their sums are added in order.
template <typename T>
__global__ __launch_bounds__(256) void embed_grad_long_kernel(const EmbedGradArgs a, T* __restrict__ dw, int64_t ldw) {
  __shared__ float quarter[4][64];
  const int64_t j = blockIdx.x, p = j * EG_LONG, q = p + EG_LONG < a.n ? p + EG_LONG : a.n;
  const uint32_t k0 = a.keys[p], k1 = a.keys[q - 1];
  uint32_t k;
  int64_t slot;
  if (k0 < (uint32_t)a.n_rows && k1 == k0 && (p == 0 || a.keys[p - 1] != k0) && run_is_long(a.keys, a.n, p, k0)) {
    k = k0; slot = 2 * j;
  } else if (k1 != k0 && q < a.n && a.keys[q] == k1 && k1 < (uint32_t)a.n_rows && run_is_long(a.keys, a.n, q - 1, k1)) {
    k = k1; slot = 2 * j + 1;
  } else {
    return;
  }
  int64_t lo = q, hi = a.n;                                     // the run's end: the first entry past k
  while (lo < hi) { const int64_t m = (lo + hi) >> 1; if (a.keys[m] <= k) lo = m + 1; else hi = m; }
  const int64_t count = (lo - 1) / EG_LONG - j;                 // windows behind this one that it reaches
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t w0 = j + 1 + count * wave / 4, w1 = j + 1 + count * (wave + 1) / 4;
  for (int c0 = 0; c0 < a.d; c0 += 64) {
    const int c = c0 + lane;
    float s = 0.f;
    if (c < a.d) {
      if (wave == 0) s = a.part[slot * a.d + c];
#pragma unroll 8
      for (int64_t w = w0; w < w1; ++w) s += a.part[2 * w * a.d + c];
    }
    __syncthreads();
    quarter[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < a.d)
      dw[(int64_t)k * ldw + c] = (T)((((quarter[0][lane] + quarter[1][lane]) + quarter[2][lane]) + quarter[3][lane]) * a.scale);
  }
}

__global__ __launch_bounds__(256) void embed_zero_kernel(uint4* __restrict__ p, int64_t n16, unsigned char* __restrict__ tail,
                                                         int n_tail, uint32_t* __restrict__ pad_keys,
                                                         uint32_t* __restrict__ pad_perm) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (pad_keys && i < EG_PAD) { pad_keys[i] = 0xFFFFFFFFu; pad_perm[i] = 0u; }
  if (i < n16) p[i] = make_uint4(0u, 0u, 0u, 0u);
  if (i < n_tail) tail[i] = 0;
}

// lanes of a row group: the smallest power of two that covers a row's accesses, at most a wave
static int lanes_log2(int64_t d, int vec) {
  int l = 0;
  while (l < 6 && ((int64_t)vec << l) < d) ++l;
  return l;
}

template <typename T, int VEC>
static void embed_rows_launch(const void* w, int64_t ldw, int64_t n_rows, int64_t d, const void* ids, int ids_i32, int64_t n,
                              float scale, void* out, int64_t ldo, hipStream_t s) {
  const int lpr = lanes_log2(d, VEC);
  const int64_t per_block = (256 >> lpr) * 4;
  const dim3 grid((unsigned)((n + per_block - 1) / per_block), (unsigned)ceil_div(d, (int64_t)VEC << lpr));
  hipLaunchKernelGGL((embed_rows_kernel<T, VEC>), grid, dim3(256), 0, s, (const T*)w, ldw, n_rows, (int)d, ids, ids_i32, n, scale,
                     (T*)out, ldo, lpr);
}

template <typename T, int VEC>
static void embed_grad_launch(EmbedGradArgs a, const void* g, int64_t ldg, void* dw, int64_t ldw, hipStream_t s) {
  a.lpr_log2 = lanes_log2(a.d, VEC);
  const int groups = 256 >> a.lpr_log2, tiles = ceil_div(a.d, (int64_t)VEC << a.lpr_log2);
  // entries per group: 64 where that still gives every CU a few thousand lanes of work, down to 4 for short id lists
  a.chunk = 64;
  while (a.chunk > 4 && (a.n / a.chunk) * tiles < 8192) a.chunk >>= 1;
  a.n_chunks = (a.n + a.chunk - 1) / a.chunk;
  const int64_t all = a.n_chunks + a.n_windows;
  hipLaunchKernelGGL((embed_grad_kernel<T, VEC>), dim3((unsigned)((all + groups - 1) / groups), tiles), dim3(256), 0, s, a,
                     (const T*)g, ldg, (T*)dw, ldw);
  if (a.n_windows)
    hipLaunchKernelGGL((embed_grad_long_kernel<T>), dim3((unsigned)a.n_windows), dim3(256), 0, s, a, (T*)dw, ldw);
}

// FN<T, VEC>(args) for the type and the access width
#define BKG_EMBED_DISPATCH(FN, type, bytes, ...)                                  \
  do {                                                                            \
    if ((type) == BKG_T_F32) {                                                    \
      if ((bytes) == 16) FN<float, 4>(__VA_ARGS__);                               \
      else if ((bytes) == 8) FN<float, 2>(__VA_ARGS__);                           \
      else FN<float, 1>(__VA_ARGS__);                                             \
    } else if ((type) == BKG_T_BF16) {                                            \
      if ((bytes) == 16) FN<__bf16, 8>(__VA_ARGS__);                              \
      else if ((bytes) == 8) FN<__bf16, 4>(__VA_ARGS__);                          \
      else if ((bytes) == 4) FN<__bf16, 2>(__VA_ARGS__);                          \
      else FN<__bf16, 1>(__VA_ARGS__);                                            \
    } else {                                                                      \
      if ((bytes) == 16) FN<_Float16, 8>(__VA_ARGS__);                            \
      else if ((bytes) == 8) FN<_Float16, 4>(__VA_ARGS__);                        \
      else if ((bytes) == 4) FN<_Float16, 2>(__VA_ARGS__);                        \
      else FN<_Float16, 1>(__VA_ARGS__);                                          \
    }                                                                             \
  } while (0)

static int64_t n_windows_of(int64_t n) { return n > EG_LONG ? (n + EG_LONG - 1) / EG_LONG : 0; }
static int64_t round256(int64_t b) { return (b + 255) & ~(int64_t)255; }

}  // namespace bkg

using namespace bkg;

extern "C" int bkg_embed_rows(const void* w, int32_t type, int64_t ldw, int64_t n_rows, int64_t d, const void* ids,
                              int32_t ids_i32, int64_t n, float scale, void* out, int64_t ldo, void* stream) {
  BKG_ARG(type >= 0 && type <= 2 && n >= 0 && n < (1ll << 31) && d >= 0 && d <= EMBED_MAX_D && n_rows >= 0,
          "bkg_embed_rows: bad sizes or type (ids below 2^31, rows of at most 2^20 columns)");
  if (n == 0 || d == 0) return 0;
  BKG_ARG(ids && out && (w || n_rows == 0) && ldo >= d, "bkg_embed_rows: null buffer or overlapping rows");
  const int e = type_bytes(type);
  int bytes = access_bytes(w, d * e, ldw * e);
  const int ob = access_bytes(out, d * e, ldo * e);
  if (ob < bytes) bytes = ob;
  BKG_ARG(bytes >= e, "bkg_embed_rows: misaligned buffer");
  BKG_EMBED_DISPATCH(embed_rows_launch, type, bytes, w, ldw, n_rows, d, ids, ids_i32, n, scale, out, ldo, (hipStream_t)stream);
  return check_launch("bkg_embed_rows");
}

extern "C" int64_t bkg_embed_grad_workspace_bytes(int64_t n, int64_t d) {
  if (n <= 0 || d <= 0) return 0;
  return 2 * round256(4 * (n + EG_PAD)) + 2 * round256(4 * n) + round256(8 * n_windows_of(n) * d) + embed_sort_workspace_bytes(n) + 256;
}

extern "C" int bkg_embed_grad(const void* g, int32_t type, int64_t ldg, int64_t d, const void* ids, int32_t ids_i32, int64_t n,
                              int64_t n_rows, int64_t pad, float scale, void* dw, void* workspace, int64_t workspace_bytes,
                              void* stream) {
  BKG_ARG(type >= 0 && type <= 2 && n >= 0 && d >= 0 && n_rows >= 0 && n < (1ll << 31) && n_rows < (1ll << 31) && d <= EMBED_MAX_D,
          "bkg_embed_grad: bad sizes or type (ids and rows below 2^31, rows of at most 2^20 columns)");
  if (n_rows == 0 || d == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  const int e = type_bytes(type);
  BKG_ARG(dw && (uintptr_t)dw % 16 == 0, "bkg_embed_grad: dw must be 16-byte aligned");
  const int64_t total = n_rows * d * e, n16 = total / 16;
  BKG_ARG(n16 / 256 < (1ll << 31) - 1, "bkg_embed_grad: table too large for one launch");
  BKG_ARG(n == 0 || (workspace && (uintptr_t)workspace % 256 == 0 && workspace_bytes >= bkg_embed_grad_workspace_bytes(n, d)),
          "bkg_embed_grad: workspace below bkg_embed_grad_workspace_bytes or not 256-byte aligned");
  unsigned char* ws = (unsigned char*)workspace;
  uint32_t *keys = nullptr, *perm = nullptr;
  if (n) {
    keys = (uint32_t*)ws; ws += round256(4 * (n + EG_PAD));
    perm = (uint32_t*)ws; ws += round256(4 * (n + EG_PAD));
  }
  hipLaunchKernelGGL(embed_zero_kernel, dim3((unsigned)((n16 + 256) / 256)), dim3(256), 0, s, (uint4*)dw, n16,
                     (unsigned char*)dw + n16 * 16, (int)(total - n16 * 16), n ? keys + n : nullptr, n ? perm + n : nullptr);
  if (n == 0) return check_launch("bkg_embed_grad");
  BKG_ARG(g && ids, "bkg_embed_grad: null buffer");
  uint32_t* scratch = (uint32_t*)ws; ws += 2 * round256(4 * n);
  EmbedGradArgs a{};
  a.keys = keys; a.perm = perm; a.n = n; a.n_rows = n_rows; a.scale = scale; a.d = (int)d;
  a.n_windows = n_windows_of(n);
  a.part = (float*)ws; ws += round256(8 * a.n_windows * d);
  const int rc = embed_sort(ids, ids_i32, n, n_rows, pad, scratch, keys, perm, ws, embed_sort_workspace_bytes(n), s);
  if (rc) return rc;
  int bytes = access_bytes(g, d * e, ldg * e);
  const int ob = access_bytes(dw, d * e, d * e);
  if (ob < bytes) bytes = ob;
  BKG_ARG(bytes >= e, "bkg_embed_grad: misaligned gradient");
  BKG_EMBED_DISPATCH(embed_grad_launch, type, bytes, a, g, ldg, dw, d, s);
  return check_launch("bkg_embed_grad");
}
