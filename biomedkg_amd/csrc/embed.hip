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
// the work is cut by ENTRIES, not by rows: a lane group takes a chunk of the sorted entries, writes the rows of the runs that
// lie in it and leaves an fp32 partial row for a run that crosses either border; a last launch adds those in order (a million
// skewed ids, 256 columns in bf16: 229 us for the whole gradient; with a run given to the group it starts in, up to 64
// entries of it, 303).  Lists of up to 2048 ids take one launch in which a block sorts for itself.
#include <algorithm>

#include "rowtypes.h"

namespace bkg {

constexpr int EG_U = 8;                             // entries per step: their rows are in flight together
constexpr int EG_PAD = 4 * EG_U;                    // words behind the sorted entries that the steps ahead reach
constexpr int64_t EMBED_MAX_D = 1 << 20;            // (column tiles are the grid's y extent)

__device__ __forceinline__ int64_t embed_id(const void* __restrict__ ids, int ids_i32, int64_t i) {
  return ids_i32 ? (int64_t)static_cast<const int32_t*>(ids)[i] : static_cast<const int64_t*>(ids)[i];
}

// Memory the gradient clears beside its sort.
struct EmbedZero {
  uint4* p; int64_t n16;                           // whole 16-byte words
  unsigned char* tail; int n_tail;                 // < 16 bytes behind them
  uint32_t *pad_keys, *pad_perm; int n_pad;        // the words behind the sorted entries
};
__device__ __forceinline__ void embed_zero(int64_t i, const EmbedZero& z) {
  if (i < z.n_pad) { z.pad_keys[i] = 0xFFFFFFFFu; z.pad_perm[i] = 0u; }
  if (i < z.n16) z.p[i] = make_uint4(0u, 0u, 0u, 0u);
  if (i < z.n_tail) z.tail[i] = 0;
}
// The sort key of an id: the id, or n_rows for an entry whose gradient goes nowhere (those come last).
__device__ __forceinline__ uint32_t embed_key(const void* __restrict__ ids, int ids_i32, int64_t i, int64_t n_rows, int64_t pad) {
  const int64_t v = embed_id(ids, ids_i32, i);
  return (v < 0 || v >= n_rows || v == pad) ? (uint32_t)n_rows : (uint32_t)v;
}

constexpr int EMBED_UNROLL = 4;

// A lane group of 2^lpr_log2 lanes copies a row's VEC-wide columns of tile blockIdx.y; UNROLL rows in flight per group.
// STREAM: a result beyond STREAM_BYTES leaves past the L2s, so that the table's rows stay (a million rows of 512 bytes out of
// 130000: 172 us written through the L2s, 143 us past them; out of 5000, 1536 bytes each: 467 and 294).
template <typename T, int VEC, bool STREAM>
__global__ __launch_bounds__(256) void embed_rows_kernel(const T* __restrict__ w, int64_t ldw, int64_t n_rows, int d,
                                                         const void* __restrict__ ids, int ids_i32, int64_t n, float scale,
                                                         T* __restrict__ out, int64_t ldo, int lpr_log2) {
  constexpr int UNROLL = EMBED_UNROLL;
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
    if constexpr (STREAM && sizeof(T) * VEC == 16) stream16(out + i * ldo + c, r[u]);
    else *reinterpret_cast<Pack<T, VEC>*>(out + i * ldo + c) = r[u];
  }
}

struct EmbedGradArgs {
  const uint32_t* keys; const uint32_t* perm;      // [n] sorted (key n_rows = no gradient), then EG_PAD all-ones words
  int64_t n, n_rows;
  float scale;
  int d, lpr_log2;
  int chunk;                                       // entries per lane group, a multiple of EG_U
  int64_t n_chunks;
  float* part;                                     // [2 n_chunks][d] partial rows: 2 j: the run that comes into chunk j,
};                                                 // 2 j + 1: the run that starts in it and goes on behind it

struct EgWords { uint32_t w[EG_U]; };
__device__ __forceinline__ EgWords eg_words(const uint32_t* __restrict__ p) {      // (32-byte aligned; reads into the pad)
  EgWords o;
  const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
  o.w[0] = a.x; o.w[1] = a.y; o.w[2] = a.z; o.w[3] = a.w;
  o.w[4] = b.x; o.w[5] = b.y; o.w[6] = b.z; o.w[7] = b.w;
  return o;
}
template <typename T, int VEC> struct EgStep {
  EgWords key;
  Pack<T, VEC> row[EG_U];
};

template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_grad_kernel(const EmbedGradArgs a, const T* __restrict__ g, int64_t ldg,
                                                         T* __restrict__ dw, int64_t ldw) {
  const int lig = threadIdx.x & ((1 << a.lpr_log2) - 1), groups = 256 >> a.lpr_log2;
  const int c = (((int)blockIdx.y << a.lpr_log2) + lig) * VEC;
  if (c >= a.d) return;
  const int64_t j = (int64_t)blockIdx.x * groups + (threadIdx.x >> a.lpr_log2);
  if (j >= a.n_chunks) return;
  const int64_t beg = j * a.chunk, last = beg + a.chunk < a.n ? beg + a.chunk : a.n;
  const T* gc = g + c;
  const uint32_t none = (uint32_t)a.n_rows;
  const uint32_t before = beg > 0 ? a.keys[beg - 1] : 0xFFFFFFFFu, behind = a.keys[last];   // (all ones behind the last entry)
  float acc[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
  uint32_t cur = before;                           // the run being added; the one that comes in goes to a partial row
  bool came_in = true;
  // the sum of run `cur` leaves: a row, or a partial one (slot: -1 none)
  auto leave = [&](int64_t slot) {
    if (cur < none) {
      if (slot < 0) {
        Pack<T, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; ++v) o.v[v] = (T)(acc[v] * a.scale);
        *reinterpret_cast<Pack<T, VEC>*>(dw + (int64_t)cur * ldw + c) = o;
      } else {
        Pack<float, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; ++v) o.v[v] = acc[v];
        *reinterpret_cast<Pack<float, VEC>*>(a.part + slot * a.d + c) = o;
      }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
  };
  // two steps at work: step s + 1's rows are loaded while step s's are added, and the words of step s + 2 behind them
  EgWords k, pm;
  auto words = [&](int64_t e) { k = eg_words(a.keys + e); pm = eg_words(a.perm + e); };      // (e <= n + EG_U: into the pad)
  auto issue = [&](int64_t e, EgStep<T, VEC>& s) {
    s.key = k;
#pragma unroll
    for (int u = 0; u < EG_U; ++u)
      if (e + u < last && k.w[u] < none) s.row[u] = *reinterpret_cast<const Pack<T, VEC>*>(gc + (int64_t)pm.w[u] * ldg);
  };
  auto consume = [&](int64_t e, const EgStep<T, VEC>& s) {
#pragma unroll
    for (int u = 0; u < EG_U; ++u) {
      if (e + u >= last) break;
      if (s.key.w[u] != cur) {
        if (e + u > beg) leave(came_in ? 2 * j : -1);          // (nothing came in: `before` is not this chunk's)
        cur = s.key.w[u];
        came_in = false;
      }
      if (s.key.w[u] < none)
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] += widen(s.row[u].v[v]);
    }
  };
  EgStep<T, VEC> s0, s1;
  words(beg);
  issue(beg, s0);
  words(beg + EG_U);
  for (int64_t e = beg; e < last; e += 2 * EG_U) {
    issue(e + EG_U, s1);
    words(e + 2 * EG_U < a.n ? e + 2 * EG_U : beg);
    consume(e, s0);
    issue(e + 2 * EG_U, s0);
    words(e + 3 * EG_U < a.n ? e + 3 * EG_U : beg);
    consume(e + EG_U, s1);
  }
  leave(came_in ? 2 * j : behind == cur ? 2 * j + 1 : -1);
}

// The rows of runs that cross borders of chunks: the chunk a run starts in adds the run's partial rows.  A block looks after
// EG_FINISH chunks.  A run over few chunks is a wave's work, the waves side by side; for a longer one the block's eight waves
// take an eighth of its chunks each, in order, and their sums are added in order.  Columns: 4 per lane (d a multiple of 4) or 1.
constexpr int EG_FINISH = 32, EG_FEW = 8;
template <typename T, int VEC>
__device__ __forceinline__ Pack<float, VEC> eg_add_parts(const EmbedGradArgs& a, int64_t w0, int64_t w1, int c, Pack<float, VEC> s) {
#pragma unroll 8
  for (int64_t w = w0; w < w1; ++w) {
    const Pack<float, VEC> r = *reinterpret_cast<const Pack<float, VEC>*>(a.part + 2 * w * a.d + c);
#pragma unroll
    for (int v = 0; v < VEC; ++v) s.v[v] += r.v[v];
  }
  return s;
}
template <typename T, int VEC>
__global__ __launch_bounds__(512) void embed_grad_finish_kernel(const EmbedGradArgs a, T* __restrict__ dw, int64_t ldw) {
  __shared__ float eighth[8][64][VEC];
  __shared__ int n_few, n_many;
  __shared__ int few[EG_FINISH], few_count[EG_FINISH], many[EG_FINISH];
  if (threadIdx.x == 0) n_few = n_many = 0;
  __syncthreads();
  const int64_t j0 = (int64_t)blockIdx.x * EG_FINISH;
  if (threadIdx.x < EG_FINISH) {
    const int64_t j = j0 + threadIdx.x, beg = j * a.chunk, q = beg + a.chunk;
    if (q < a.n) {
      const uint32_t k1 = a.keys[q - 1];
      if (k1 < (uint32_t)a.n_rows && a.keys[q] == k1 && !(a.keys[beg] == k1 && beg > 0 && a.keys[beg - 1] == k1)) {
        int count = 1;                                          // chunks behind this one that the run reaches, as far as EG_FEW
        while (count < EG_FEW && q + (int64_t)count * a.chunk < a.n && a.keys[q + (int64_t)count * a.chunk] == k1) ++count;
        if (count < EG_FEW) {
          const int at = atomicAdd(&n_few, 1);                  // (their order does not matter: each writes a row of its own)
          few[at] = threadIdx.x; few_count[at] = count;
        } else {
          many[atomicAdd(&n_many, 1)] = threadIdx.x;
        }
      }
    }
  }
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, total_few = n_few, total_many = n_many;
  for (int i = wave; i < total_few; i += 8) {
    const int64_t j = j0 + few[i];
    const uint32_t k = a.keys[(j + 1) * a.chunk - 1];
    for (int c = lane * VEC; c < a.d; c += 64 * VEC) {
      const Pack<float, VEC> s = eg_add_parts<T, VEC>(a, j + 1, j + 1 + few_count[i], c,
                                                      *reinterpret_cast<const Pack<float, VEC>*>(a.part + (2 * j + 1) * a.d + c));
#pragma unroll
      for (int v = 0; v < VEC; ++v) dw[(int64_t)k * ldw + c + v] = (T)(s.v[v] * a.scale);
    }
  }
  for (int i = 0; i < total_many; ++i) {
    const int64_t j = j0 + many[i], q = (j + 1) * a.chunk;
    const uint32_t k = a.keys[q - 1];
    int64_t last = q, span = a.n - q;                           // the run's last entry lies in [last, last + span): 512 looks a round
    while (span > 1) {
      const int64_t step = (span + 511) / 512, at = last + threadIdx.x * step;
      last += (__syncthreads_count(at < last + span && a.keys[at < a.n ? at : a.n - 1] == k) - 1) * step;
      span = step;
      if (last + span > a.n) span = a.n - last;
    }
    const int64_t count = last / a.chunk - j;                   // chunks behind this one that it reaches
    const int64_t w0 = j + 1 + count * wave / 8, w1 = j + 1 + count * (wave + 1) / 8;
    for (int c0 = 0; c0 < a.d; c0 += 64 * VEC) {
      const int c = c0 + lane * VEC;
      Pack<float, VEC> s;
#pragma unroll
      for (int v = 0; v < VEC; ++v) s.v[v] = 0.f;
      if (c < a.d) {
        if (wave == 0) s = *reinterpret_cast<const Pack<float, VEC>*>(a.part + (2 * j + 1) * a.d + c);
        s = eg_add_parts<T, VEC>(a, w0, w1, c, s);
      }
      __syncthreads();
#pragma unroll
      for (int v = 0; v < VEC; ++v) eighth[wave][lane][v] = s.v[v];
      __syncthreads();
      if (wave == 0 && c < a.d) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          float sum = eighth[0][lane][v];
#pragma unroll
          for (int x = 1; x < 8; ++x) sum += eighth[x][lane][v];
          dw[(int64_t)k * ldw + c + v] = (T)(sum * a.scale);
        }
      }
    }
  }
}

// ---- up to EF_IDS ids: one launch.  A block owns some rows of the table and a tile of its columns: it looks through ALL ids,
// keeps those of its rows (in LDS, a word each: the row above the position), clears the rows meanwhile, sorts what it kept -- a
// few words, unless there is a hub -- and sums: its lane groups take equal parts of the sorted entries, and a run that crosses
// such parts is joined from partial rows in LDS, in order.  No scratch memory, no other launch.  Against the three launches
// below, on the chip: 13.0 us to 22.0 for 2048 ids of 5000 rows, 768 in fp32 (1021 ids: 11.2), 14.4 to 26.2 for 2048 ids of
// 130000 rows, 256 in bf16; all ids equal, the worst case: 24.5 to 28.2 and 30.3 to 29.4.  Tiles of 32 lanes (512 bytes of a
// row) spread a hub over more CUs than 64 (36.9 us), and clear whole pieces of rows better than 16 (uniform ids 14.9).
constexpr int EF_IDS = 2048, EF_POS = 11, EF_THREADS = 512, EF_ITEMS = EF_IDS / EF_THREADS, EF_WAVES = EF_THREADS / 64;
constexpr int EF_LPR = 5, EF_BITS = 5, EF_DIGITS = 1 << EF_BITS;
static_assert(EF_WAVES * EF_DIGITS <= EF_THREADS && EF_DIGITS <= 64, "a thread clears each counter, a lane of one wave adds each digit's");
struct EmbedFewArgs {
  const void* ids; int ids_i32, n;
  int64_t n_rows, pad;
  float scale;
  int d, lpr_log2, rows;                             // rows: per block
};
template <typename T, int VEC>
__global__ __launch_bounds__(EF_THREADS) void embed_grad_few_kernel(const EmbedFewArgs a, const T* __restrict__ g, int64_t ldg,
                                                                    T* __restrict__ dw, int64_t ldw) {
  __shared__ uint32_t list[EF_IDS];
  __shared__ int counts[EF_ITEMS][EF_WAVES], seen[EF_WAVES][EF_DIGITS];
  __shared__ float part[VEC][EF_THREADS];            // a lane's sums of the run that comes into its group's entries
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int lig = threadIdx.x & ((1 << a.lpr_log2) - 1), group = threadIdx.x >> a.lpr_log2, groups = EF_THREADS >> a.lpr_log2;
  const int c = (((int)blockIdx.y << a.lpr_log2) + lig) * VEC;
  const bool live = c < a.d;
  const int64_t r0 = (int64_t)blockIdx.x * a.rows, r1 = r0 + a.rows < a.n_rows ? r0 + a.rows : a.n_rows;

  uint32_t key[EF_ITEMS];
  int below[EF_ITEMS];
#pragma unroll
  for (int u = 0; u < EF_ITEMS; ++u) {
    const int i = u * EF_THREADS + threadIdx.x;
    const int64_t id = i < a.n ? embed_id(a.ids, a.ids_i32, i) : -1;
    const bool mine = id >= r0 && id < r1 && id != a.pad;
    const uint64_t all = __ballot(mine);
    key[u] = ((uint32_t)(id - r0) << EF_POS) | (uint32_t)i;
    below[u] = mine ? __popcll(all & ((1ull << lane) - 1)) : -1;
    if (lane == 0) counts[u][wave] = __popcll(all);
  }
  if (live) {
    Pack<T, VEC> zero;
#pragma unroll
    for (int v = 0; v < VEC; ++v) zero.v[v] = (T)0.f;
    for (int64_t r = r0 + group; r < r1; r += groups) *reinterpret_cast<Pack<T, VEC>*>(dw + r * ldw + c) = zero;
  }
  __syncthreads();                                   // (also orders the zeros before the sums)
  int total = 0;
#pragma unroll
  for (int u = 0; u < EF_ITEMS; ++u)
#pragma unroll
    for (int w = 0; w < EF_WAVES; ++w) {
      if (w == wave && below[u] >= 0) list[total + below[u]] = key[u];
      total += counts[u][w];
    }
  if (total == 0) return;
  __syncthreads();
  if (total <= 64) {                                 // a place per entry: how many are smaller (no two are equal)
    if (wave == 0) {
      const uint32_t x = lane < total ? list[lane] : 0xFFFFFFFFu;
      int place = 0;
      for (int i = 0; i < total; ++i) place += (uint32_t)__builtin_amdgcn_readlane((int)x, i) < x;
      if (lane < total) list[place] = x;
    }
  } else {                                           // stable passes over EF_BITS-bit digits of the row (they lie in position order)
    for (int shift = EF_POS; a.rows - 1 >> (shift - EF_POS) > 0; shift += EF_BITS) {
      uint32_t x[EF_ITEMS];
      int place[EF_ITEMS];
      if (threadIdx.x < EF_WAVES * EF_DIGITS) (&seen[0][0])[threadIdx.x] = 0;
      __syncthreads();
#pragma unroll
      for (int u = 0; u < EF_ITEMS; ++u) {           // a wave takes 64 EF_ITEMS neighbouring entries
        const int i = wave * 64 * EF_ITEMS + u * 64 + lane;
        x[u] = i < total ? list[i] : 0u;
        const uint32_t digit = (x[u] >> shift) & (EF_DIGITS - 1);
        uint64_t peers = __ballot(i < total);
#pragma unroll
        for (int b = 0; b < EF_BITS; ++b) {
          const uint64_t set = __ballot((digit >> b) & 1u);
          peers &= ((digit >> b) & 1u) ? set : ~set;
        }
        const int first = seen[wave][digit], ahead = __popcll(peers & ((1ull << lane) - 1));    // (a wave's LDS operations
        place[u] = first + ahead;                                                               // complete in order)
        asm volatile("" ::: "memory");
        if (i < total && ahead == 0) seen[wave][digit] = first + __popcll(peers);
        asm volatile("" ::: "memory");
      }
      __syncthreads();
      if (wave == 0) {                               // lane: a digit; what lies before its entries of each wave
        int count = 0;
        if (lane < EF_DIGITS)
          for (int w = 0; w < EF_WAVES; ++w) count += seen[w][lane];
        int at = count;
#pragma unroll
        for (int o = 1; o < EF_DIGITS; o <<= 1) {
          const int up = __shfl_up(at, o, 64);
          if (lane >= o) at += up;
        }
        at -= count;
        if (lane < EF_DIGITS)
          for (int w = 0; w < EF_WAVES; ++w) {
            const int n = seen[w][lane];
            seen[w][lane] = at;
            at += n;
          }
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < EF_ITEMS; ++u)
        if (wave * 64 * EF_ITEMS + u * 64 + lane < total) list[seen[wave][(x[u] >> shift) & (EF_DIGITS - 1)] + place[u]] = x[u];
      __syncthreads();
    }
  }
  __syncthreads();

  const int chunk = (total + groups - 1) / groups, beg = group * chunk, last = beg + chunk < total ? beg + chunk : total;
  const T* gc = g + c;
  auto row_of = [&](int e) { return list[e] >> EF_POS; };
  float acc[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
  auto write = [&](uint32_t row) {
    Pack<T, VEC> o;
#pragma unroll
    for (int v = 0; v < VEC; ++v) o.v[v] = (T)(acc[v] * a.scale);
    *reinterpret_cast<Pack<T, VEC>*>(dw + (r0 + row) * ldw + c) = o;
  };
  bool goes_on = false;                              // the last run starts in these entries and goes on behind them
  uint32_t cur = 0;
  if (live && beg < last) {
    bool came_in = beg > 0 && row_of(beg - 1) == row_of(beg);
    cur = row_of(beg);
    auto leave = [&]() {
      if (!came_in) write(cur);
      else
#pragma unroll
        for (int v = 0; v < VEC; ++v) part[v][threadIdx.x] = acc[v];
#pragma unroll
      for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
    };
    for (int e = beg; e < last; e += EG_U) {
      uint32_t k[EG_U];
      Pack<T, VEC> r[EG_U];
#pragma unroll
      for (int u = 0; u < EG_U; ++u) {
        k[u] = list[e + u < last ? e + u : last - 1];
        r[u] = *reinterpret_cast<const Pack<T, VEC>*>(gc + (int64_t)(k[u] & (EF_IDS - 1)) * ldg);
      }
#pragma unroll
      for (int u = 0; u < EG_U; ++u) {
        if (e + u >= last) break;
        if (k[u] >> EF_POS != cur) {
          leave();
          cur = k[u] >> EF_POS;
          came_in = false;
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] += widen(r[u].v[v]);
      }
    }
    goes_on = !came_in && last < total && row_of(last) == cur;
    if (!goes_on) leave();
  }
  __syncthreads();
  if (goes_on) {
    for (int w = group + 1; w * chunk < total && row_of(w * chunk) == cur; ++w)
#pragma unroll
      for (int v = 0; v < VEC; ++v) acc[v] += part[v][(w << a.lpr_log2) + lig];
    write(cur);
  }
}

// ---- up to ES_SMALL ids: one workgroup sorts in LDS, in stable passes over SS_BITS-bit digits -- its waves take neighbouring
// entries 64 at a time, lanes with equal digits find each other by ballots -- while the blocks behind it clear the gradient.
// (Positions behind n carry all-ones keys: they start last and stay last.)  Whole gradient of 8192 ids of 130000 rows, 256 in bf16: 33 us,
// 48 with the device library's block sort; with the launches of longer lists below 42.
constexpr int ES_SMALL = 8192, SS_THREADS = 1024, SS_WAVES = SS_THREADS / 64, SS_BITS = 6, SS_DIGITS = 1 << SS_BITS;
static_assert(SS_WAVES * SS_DIGITS == SS_THREADS, "a thread per counter");
template <int ITEMS>
__global__ __launch_bounds__(SS_THREADS) void embed_small_sort_kernel(const void* __restrict__ ids, int ids_i32, int n, int64_t n_rows,
                                                                      int64_t pad, int bits, uint32_t* __restrict__ sorted_keys,
                                                                      uint32_t* __restrict__ perm, const EmbedZero zero) {
  __shared__ uint32_t key_lds[SS_THREADS * ITEMS];
  __shared__ uint16_t val_lds[SS_THREADS * ITEMS];
  __shared__ uint32_t seen[SS_WAVES][SS_DIGITS], wave_sums[SS_WAVES];
  if (blockIdx.x > 0) {
    embed_zero((int64_t)(blockIdx.x - 1) * SS_THREADS + threadIdx.x, zero);
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i0 = wave * 64 * ITEMS + lane;
  uint32_t key[ITEMS], place[ITEMS];
  uint16_t val[ITEMS];
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const int i = i0 + u * 64;
    key[u] = i < n ? embed_key(ids, ids_i32, i, n_rows, pad) : 0xFFFFFFFFu;
    val[u] = (uint16_t)i;
  }
  for (int shift = 0; shift < bits; shift += SS_BITS) {
    (&seen[0][0])[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      const uint32_t digit = (key[u] >> shift) & (SS_DIGITS - 1);
      uint64_t peers = ~0ull;
#pragma unroll
      for (int b = 0; b < SS_BITS; ++b) {
        const uint64_t set = __ballot((digit >> b) & 1u);
        peers &= ((digit >> b) & 1u) ? set : ~set;
      }
      const uint32_t first = seen[wave][digit], ahead = __popcll(peers & ((1ull << lane) - 1));     // (a wave's LDS operations
      place[u] = first + ahead;                                                                     // complete in order)
      asm volatile("" ::: "memory");
      if (ahead == 0) seen[wave][digit] = first + __popcll(peers);
      asm volatile("" ::: "memory");
    }
    __syncthreads();
    // where each (digit, wave)'s entries go: exclusive prefix sums over the counters, a thread each
    const uint32_t count = seen[threadIdx.x % SS_WAVES][threadIdx.x / SS_WAVES];
    uint32_t at = count;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t up = __shfl_up((int)at, o, 64);
      if (lane >= o) at += up;
    }
    if (lane == 63) wave_sums[wave] = at;
    __syncthreads();
    at -= count;
    for (int w = 0; w < wave; ++w) at += wave_sums[w];
    seen[threadIdx.x % SS_WAVES][threadIdx.x / SS_WAVES] = at;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      const uint32_t to = seen[wave][(key[u] >> shift) & (SS_DIGITS - 1)] + place[u];
      key_lds[to] = key[u];
      val_lds[to] = val[u];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) { key[u] = key_lds[i0 + u * 64]; val[u] = val_lds[i0 + u * 64]; }
  }
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const int i = i0 + u * 64;
    if (i < n) { sorted_keys[i] = key[u]; perm[i] = val[u]; }
  }
}

// ---- the sort of longer id lists: stable radix passes over ES_BITS-bit digits, (key, position) pairs.  A block counts its
// ES_TILE entries' digits (the first pass makes the keys from the ids); a block per digit turns the counts into offsets; the
// third launch ranks the tile's entries -- its waves take 64 neighbouring entries at a time, lanes with equal digits find
// each other by ballots, a counter per wave and digit holds what came before -- and writes them where they belong.
// A million ids below 130001 take two passes: 68 us, the clearing of the 66 MB gradient in bf16 included.
constexpr int ES_BITS = 9, ES_DIGITS = 1 << ES_BITS, ES_THREADS = 1024, ES_WAVES = ES_THREADS / 64, ES_ITEMS = 2;
constexpr int ES_TILE = ES_THREADS * ES_ITEMS;     // (100003 ids: whole gradient of 8 columns 37 us, 43 with 4 items; 4M: 273, 260)
// Up to so many blocks, each adds up the counts of all by itself, without the launch between (whole gradient of 8 columns: 30000
// ids 30 us, 32 with it; 131072 ids 43 and 45; 500000 ids 97 and 81).
constexpr int ES_FEW_BLOCKS = 64;
static_assert(ES_THREADS >= ES_DIGITS, "a thread per digit computes where the digit begins");

struct EmbedSort {
  const void* ids; int ids_i32; int64_t n_rows, pad;   // first pass (ids not null): keys from the ids, positions 0 .. n - 1
  const uint32_t *key_in, *val_in;
  uint32_t *key_out, *val_out;
  int64_t n;
  int n_blocks, shift;
  uint32_t* counts;                                    // [ES_DIGITS][n_blocks]; few blocks: [n_blocks][ES_DIGITS]
  uint32_t* totals;                                    // [ES_DIGITS] (null: few blocks)
};
__device__ __forceinline__ uint32_t es_key(const EmbedSort& a, int64_t i) {
  return a.ids ? embed_key(a.ids, a.ids_i32, i, a.n_rows, a.pad) : a.key_in[i];
}

// (the blocks behind the sort's clear memory)
__global__ __launch_bounds__(ES_THREADS) void embed_count_kernel(const EmbedSort a, const EmbedZero z) {
  __shared__ uint32_t count[ES_DIGITS];
  if ((int)blockIdx.x >= a.n_blocks) {
    embed_zero((int64_t)(blockIdx.x - a.n_blocks) * ES_THREADS + threadIdx.x, z);
    return;
  }
  for (int d = threadIdx.x; d < ES_DIGITS; d += ES_THREADS) count[d] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * ES_TILE;
  uint32_t k[ES_ITEMS];
#pragma unroll
  for (int r = 0; r < ES_ITEMS; ++r) {
    const int64_t i = i0 + r * ES_THREADS + threadIdx.x;
    k[r] = i < a.n ? es_key(a, i) : 0u;
  }
#pragma unroll
  for (int r = 0; r < ES_ITEMS; ++r)
    if (i0 + r * ES_THREADS + threadIdx.x < a.n) atomicAdd(&count[(k[r] >> a.shift) & (ES_DIGITS - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < ES_DIGITS; d += ES_THREADS)
    a.counts[a.totals ? (int64_t)d * a.n_blocks + blockIdx.x : (int64_t)blockIdx.x * ES_DIGITS + d] = count[d];
}

// block d: the counts of digit d become their exclusive prefix sums over the blocks; totals[d] their sum
__global__ __launch_bounds__(256) void embed_offsets_kernel(uint32_t* __restrict__ counts, int n_blocks, uint32_t* __restrict__ totals) {
  __shared__ uint32_t wave_sums[4];
  uint32_t* row = counts + (int64_t)blockIdx.x * n_blocks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t carry = 0;
  for (int b0 = 0; b0 < n_blocks; b0 += 256) {
    const int b = b0 + threadIdx.x;
    const uint32_t v = b < n_blocks ? row[b] : 0u;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_up((int)s, o, 64);
      if (lane >= o) s += u;
    }
    if (lane == 63) wave_sums[wave] = s;
    __syncthreads();
    uint32_t before = carry, all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += wave_sums[w];
      all += wave_sums[w];
    }
    if (b < n_blocks) row[b] = before + s - v;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

__global__ __launch_bounds__(ES_THREADS) void embed_scatter_kernel(const EmbedSort a) {
  __shared__ uint32_t seen[ES_WAVES][ES_DIGITS];       // entries of the digit in this wave so far; then where the wave's first goes
  __shared__ uint32_t wave_sums[ES_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int d = threadIdx.x; d < ES_WAVES * ES_DIGITS; d += ES_THREADS) (&seen[0][0])[d] = 0;
  const int64_t i0 = (int64_t)blockIdx.x * ES_TILE + wave * (64 * ES_ITEMS) + lane;
  uint32_t key[ES_ITEMS], val[ES_ITEMS], rank[ES_ITEMS];
#pragma unroll
  for (int r = 0; r < ES_ITEMS; ++r) {
    const int64_t i = i0 + 64 * r;
    key[r] = i < a.n ? es_key(a, i) : 0u;
    val[r] = a.ids ? (uint32_t)i : i < a.n ? a.val_in[i] : 0u;
  }
  // where each digit begins: the totals' exclusive prefix sums (threads 0 .. ES_DIGITS - 1), plus this block's offset
  uint32_t start = 0;
  {
    uint32_t v = 0u, before = 0u;                      // the digit's total; its entries in the blocks before this one
    if (threadIdx.x < ES_DIGITS) {
      if (a.totals) {
        v = a.totals[threadIdx.x];
        before = a.counts[(int64_t)threadIdx.x * a.n_blocks + blockIdx.x];
      } else {
#pragma unroll 8
        for (int b = 0; b < a.n_blocks; ++b) {
          const uint32_t c = a.counts[b * ES_DIGITS + threadIdx.x];
          v += c;
          before += b < (int)blockIdx.x ? c : 0u;
        }
      }
    }
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_up((int)s, o, 64);
      if (lane >= o) s += u;
    }
    if (lane == 63) wave_sums[wave] = s;
    __syncthreads();
    for (int w = 0; w < wave; ++w) start += wave_sums[w];
    start += s - v + before;
  }
#pragma unroll
  for (int r = 0; r < ES_ITEMS; ++r) {
    const bool live = i0 + 64 * r < a.n;
    const uint32_t d = (key[r] >> a.shift) & (ES_DIGITS - 1);
    uint64_t peers = __ballot(live);
#pragma unroll
    for (int b = 0; b < ES_BITS; ++b) {
      const uint64_t set = __ballot((d >> b) & 1u);
      peers &= ((d >> b) & 1u) ? set : ~set;
    }
    const uint32_t below = __popcll(peers & ((1ull << lane) - 1));
    const uint32_t base = seen[wave][d];               // (a wave's LDS operations complete in order)
    rank[r] = base + below;
    asm volatile("" ::: "memory");
    if (live && below == 0) seen[wave][d] = base + __popcll(peers);
    asm volatile("" ::: "memory");
  }
  __syncthreads();
  if (threadIdx.x < ES_DIGITS) {
    uint32_t at = start;
#pragma unroll
    for (int w = 0; w < ES_WAVES; ++w) {
      const uint32_t c = seen[w][threadIdx.x];
      seen[w][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ES_ITEMS; ++r)
    if (i0 + 64 * r < a.n) {
      const uint32_t at = seen[wave][(key[r] >> a.shift) & (ES_DIGITS - 1)] + rank[r];
      a.key_out[at] = key[r];
      a.val_out[at] = val[r];
    }
}

static int64_t round256(int64_t b) { return (b + 255) & ~(int64_t)255; }
static int es_blocks(int64_t n) { return (int)((n + ES_TILE - 1) / ES_TILE); }
// two more pairs of arrays to pass through, the counts and the totals
static int64_t embed_sort_bytes(int64_t n) {
  return n <= ES_SMALL ? 0 : 2 * round256(4 * n) + round256(4 * (int64_t)ES_DIGITS * (es_blocks(n) + 1));
}

// Stable ascending sort of the ids' keys with their positions; `zero` is cleared beside it.
static int embed_sort(const void* ids, int ids_i32, int64_t n, int64_t n_rows, int64_t pad, uint32_t* keys, uint32_t* perm,
                      unsigned char* ws, const EmbedZero& zero, hipStream_t s) {
  int bits = 1;
  while (bits < 32 && (1ull << bits) <= (uint64_t)n_rows) ++bits;      // (keys go up to n_rows itself)
  if (n <= ES_SMALL) {
    const unsigned blocks = (unsigned)(1 + (zero.n16 + SS_THREADS) / SS_THREADS);
    if (n <= ES_SMALL / 2)
      hipLaunchKernelGGL(embed_small_sort_kernel<4>, dim3(blocks), dim3(SS_THREADS), 0, s, ids, ids_i32, (int)n, n_rows, pad, bits,
                         keys, perm, zero);
    else
      hipLaunchKernelGGL(embed_small_sort_kernel<8>, dim3(blocks), dim3(SS_THREADS), 0, s, ids, ids_i32, (int)n, n_rows, pad, bits,
                         keys, perm, zero);
    return check_launch("bkg_embed_grad: sort");
  }
  uint32_t* other_keys = (uint32_t*)ws;
  uint32_t* other_perm = (uint32_t*)(ws + round256(4 * n));
  uint32_t* counts = (uint32_t*)(ws + 2 * round256(4 * n));
  EmbedSort a{ids, ids_i32, n_rows, pad, nullptr, nullptr, nullptr, nullptr, n, es_blocks(n), 0, counts,
              counts + (int64_t)ES_DIGITS * es_blocks(n)};
  if (a.n_blocks <= ES_FEW_BLOCKS) a.totals = nullptr;
  const int passes = (bits + ES_BITS - 1) / ES_BITS;
  for (int p = 0; p < passes; ++p) {                                   // the last pass ends in keys / perm
    const bool to_result = (passes - 1 - p) % 2 == 0;
    a.key_out = to_result ? keys : other_keys;
    a.val_out = to_result ? perm : other_perm;
    a.shift = p * ES_BITS;
    const unsigned clear = p == 0 ? (unsigned)((zero.n16 + ES_THREADS) / ES_THREADS) : 0u;
    hipLaunchKernelGGL(embed_count_kernel, dim3(a.n_blocks + clear), dim3(ES_THREADS), 0, s, a, zero);
    if (a.totals) hipLaunchKernelGGL(embed_offsets_kernel, dim3(ES_DIGITS), dim3(256), 0, s, a.counts, a.n_blocks, a.totals);
    hipLaunchKernelGGL(embed_scatter_kernel, dim3(a.n_blocks), dim3(ES_THREADS), 0, s, a);
    a.ids = nullptr;
    a.key_in = a.key_out;
    a.val_in = a.val_out;
  }
  return check_launch("bkg_embed_grad: sort");
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
  const int64_t per_block = (256 >> lpr) * EMBED_UNROLL, most = per_block << 23;     // (a launch has below 2^32 threads)
  if (n > most) {
    embed_rows_launch<T, VEC>(w, ldw, n_rows, d, ids, ids_i32, most, scale, out, ldo, s);
    return embed_rows_launch<T, VEC>(w, ldw, n_rows, d, (const char*)ids + most * (ids_i32 ? 4 : 8), ids_i32, n - most, scale,
                                     (T*)out + most * ldo, ldo, s);
  }
  const dim3 grid((unsigned)((n + per_block - 1) / per_block), (unsigned)ceil_div(d, (int64_t)VEC << lpr));
  if (sizeof(T) * VEC == 16 && n * d * (int64_t)sizeof(T) > STREAM_BYTES)
    hipLaunchKernelGGL((embed_rows_kernel<T, VEC, sizeof(T) * VEC == 16>), grid, dim3(256), 0, s, (const T*)w, ldw, n_rows, (int)d,
                       ids, ids_i32, n, scale, (T*)out, ldo, lpr);
  else
    hipLaunchKernelGGL((embed_rows_kernel<T, VEC, false>), grid, dim3(256), 0, s, (const T*)w, ldw, n_rows, (int)d, ids, ids_i32, n,
                       scale, (T*)out, ldo, lpr);
}

template <typename T, int VEC>
static void embed_grad_launch(EmbedGradArgs a, const void* g, int64_t ldg, void* dw, int64_t ldw, hipStream_t s) {
  a.lpr_log2 = lanes_log2(a.d, VEC);
  const int groups = 256 >> a.lpr_log2, tiles = ceil_div(a.d, (int64_t)VEC << a.lpr_log2);
  hipLaunchKernelGGL((embed_grad_kernel<T, VEC>), dim3((unsigned)((a.n_chunks + groups - 1) / groups), tiles), dim3(256), 0, s, a,
                     (const T*)g, ldg, (T*)dw, ldw);
  if (a.n_chunks > 1) {
    const dim3 grid((unsigned)ceil_div(a.n_chunks, EG_FINISH));
    if (a.d % 4 == 0) hipLaunchKernelGGL((embed_grad_finish_kernel<T, 4>), grid, dim3(512), 0, s, a, (T*)dw, ldw);
    else hipLaunchKernelGGL((embed_grad_finish_kernel<T, 1>), grid, dim3(512), 0, s, a, (T*)dw, ldw);
  }
}

// Rows per block: blocks for the chip, each with 16 rows or more (a block looks through all ids whatever it owns), at most the
// 2^21 that fit above a position.
template <typename T, int VEC>
static void embed_grad_few_launch(EmbedFewArgs a, const void* g, int64_t ldg, void* dw, int64_t ldw, hipStream_t s) {
  a.lpr_log2 = std::min(lanes_log2(a.d, VEC), EF_LPR);
  const int64_t tiles = ceil_div(a.d, (int64_t)VEC << a.lpr_log2);
  a.rows = (int)std::min<int64_t>(std::max<int64_t>((a.n_rows * tiles + 1023) / 1024, 16), 1 << (32 - EF_POS));
  hipLaunchKernelGGL((embed_grad_few_kernel<T, VEC>), dim3((unsigned)((a.n_rows + a.rows - 1) / a.rows), (unsigned)tiles),
                     dim3(EF_THREADS), 0, s, a, (const T*)g, ldg, (T*)dw, ldw);
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

// Entries per lane group: 64 from a quarter of a million entries on (a chunk writes up to two partial rows of 4 bytes a column
// and they are read back: with 64 they cost a few percent of the entries' own bytes); fewer where the list is short, so that
// there are groups for the chip.
static int embed_chunk(int64_t n) {
  int chunk = 64;
  while (chunk > EG_U && n / chunk < 4096) chunk >>= 1;
  return chunk;
}
static int64_t embed_chunks(int64_t n) { return (n + embed_chunk(n) - 1) / embed_chunk(n); }
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
  if (n <= EF_IDS || d <= 0) return 0;
  return 2 * round256(4 * (n + EG_PAD)) + round256(8 * embed_chunks(n) * d) + embed_sort_bytes(n);
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
  int bytes = n ? access_bytes(g, d * e, ldg * e) : 16;
  const int ob = access_bytes(dw, d * e, d * e);
  if (ob < bytes) bytes = ob;
  BKG_ARG(n == 0 || (g && ids), "bkg_embed_grad: null buffer");
  BKG_ARG(bytes >= e, "bkg_embed_grad: misaligned gradient");
  if (n <= EF_IDS) {
    const EmbedFewArgs a{ids, ids_i32, (int)n, n_rows, pad, scale, (int)d, 0, 0};
    BKG_EMBED_DISPATCH(embed_grad_few_launch, type, bytes, a, g, ldg, dw, d, s);
    return check_launch("bkg_embed_grad");
  }
  const int64_t total = n_rows * d * e, n16 = total / 16;
  BKG_ARG(n16 + n < (1ll << 32) - (1 << 20), "bkg_embed_grad: gradient too large for one launch (64 GB)");
  BKG_ARG(workspace && (uintptr_t)workspace % 256 == 0 && workspace_bytes >= bkg_embed_grad_workspace_bytes(n, d),
          "bkg_embed_grad: workspace below bkg_embed_grad_workspace_bytes or not 256-byte aligned");
  unsigned char* ws = (unsigned char*)workspace;
  uint32_t* keys = (uint32_t*)ws; ws += round256(4 * (n + EG_PAD));
  uint32_t* perm = (uint32_t*)ws; ws += round256(4 * (n + EG_PAD));
  const EmbedZero z{(uint4*)dw, n16, (unsigned char*)dw + n16 * 16, (int)(total - n16 * 16), keys + n, perm + n, EG_PAD};
  EmbedGradArgs a{};
  a.keys = keys; a.perm = perm; a.n = n; a.n_rows = n_rows; a.scale = scale; a.d = (int)d;
  a.chunk = embed_chunk(n);
  a.n_chunks = embed_chunks(n);
  a.part = (float*)ws; ws += round256(8 * a.n_chunks * d);
  const int rc = embed_sort(ids, ids_i32, n, n_rows, pad, keys, perm, ws, z, s);
  if (rc) return rc;
  BKG_EMBED_DISPATCH(embed_grad_launch, type, bytes, a, g, ldg, dw, d, s);
  return check_launch("bkg_embed_grad");
}
