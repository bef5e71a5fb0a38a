// Embedding lookup with scaling, and the gradient of the table.
//
//   out[i]  = scale * table[id_i]                                   (a row of NaN where id_i is outside [0, vocab))
//   grad[v] = scale * sum over i with id_i = v, v != padding, of g[i]   in increasing order of i, fp32 sums, zero rows where no i is
//
// Both are bound by memory: rows gathered and rows written, no arithmetic to speak of.  The gradient's order of summation is fixed
// by sorting the positions by token, without atomics on values, so it repeats bit for bit:
//   k_embed_sort  one block per range of table rows.  Its waves each read their part of the ids twice: once to count what is smaller than
//                 the range (this gives the block's place among the sorted positions) and what falls on each row of it (counters in
//                 LDS, one set a wave), and once to put the positions in place, in order.  So the sort is one launch with no exchange
//                 between blocks, for n ids read (rows / range) times from the L2.  Rows that got no token are zeroed here.
//   k_embed_sum   chunks of sorted positions x column slabs: sums each run of equal tokens.  A run inside its chunk is written to the table's
//                 gradient, a run across chunk borders as fp32 parts to the workspace: work is even however often one token occurs.
//   k_embed_tail  joins those parts in their order.
#include "token_vec.h"

namespace omnihd {
namespace {
using namespace tok;

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kMaxRange = 896;                     // table rows of one sorting block: 16 sets of counters, 56 KB of LDS

template <typename ID> __device__ __forceinline__ bool usable(ID id, long long vocab, long long padding) {
  return id >= 0 && (long long)id < vocab && (long long)id != padding;
}

template <typename TT, typename TO, typename ID, int TPR, bool ODD>
__global__ __launch_bounds__(256) void k_embed_fwd(const ID* __restrict__ ids, const TT* __restrict__ table, long long pitch, long long vocab,
                                                   long long n, int dim, float scale, TO* __restrict__ out) {
  constexpr int RPB = 256 / TPR;
  const int t = threadIdx.x % TPR;
  for (long long i = (long long)blockIdx.x * RPB + threadIdx.x / TPR; i < n; i += (long long)gridDim.x * RPB) {
    const long long id = (long long)ids[i];
    const bool ok = id >= 0 && id < vocab;
    for (int c = t * 8; c < dim; c += TPR * 8) {
      float v[8];
      if (ok) {
        load8<ODD>(table + id * pitch + c, dim - c, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= scale;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = __builtin_nanf("");
      }
      store8<ODD>(out + i * dim + c, dim - c, v);
    }
  }
}

template <typename TT, typename ID, bool ODD>
__global__ __launch_bounds__(kSortThreads) void k_embed_sort(const ID* __restrict__ ids, long long n, long long vocab, long long padding,
                                                             int range, int dim, int* __restrict__ keys, int* __restrict__ pos,
                                                             int* __restrict__ used, TT* __restrict__ grad) {
  extern __shared__ int hist[];                    // [waves][range]
  __shared__ int wave_sum[kSortWaves], empty_rows, smaller[kSortWaves];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long long r0 = (long long)blockIdx.x * range;
  const int rows = (int)(vocab - r0 < range ? vocab - r0 : range);
  for (int i = threadIdx.x; i < kSortWaves * range; i += kSortThreads) hist[i] = 0;
  __syncthreads();
  // each wave has a run of the ids, a multiple of 64
  const long long part = ((n + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const long long lo = part * w < n ? part * w : n, hi = lo + part < n ? lo + part : n;
  int* mine = hist + w * range;
  int less = 0;
  long long i = lo + lane;
  for (; i + 448 < hi; i += 512) {                 // eight loads in flight a lane
    ID v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = ids[i + 64 * k];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (usable(v[k], vocab, padding)) {
        const long long d = (long long)v[k] - r0;
        less += d < 0;
        if (d >= 0 && d < rows) atomicAdd(mine + d, 1);
      }
  }
  for (; i < hi; i += 64) {
    const ID v = ids[i];
    if (usable(v, vocab, padding)) {
      const long long d = (long long)v - r0;
      less += d < 0;
      if (d >= 0 && d < rows) atomicAdd(mine + d, 1);
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) less += __shfl_xor(less, o, 64);
  if (lane == 0) smaller[w] = less;
  __syncthreads();
  // where each row's and wave's positions begin
  int total = 0;
  if ((int)threadIdx.x < rows)
    for (int k = 0; k < kSortWaves; ++k) total += hist[k * range + threadIdx.x];
  int scan = total;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(scan, o, 64);
    if (lane >= o) scan += up;
  }
  if (lane == 63) wave_sum[w] = scan;
  __syncthreads();
  int begin = scan - total, all = 0;
  for (int k = 0; k < kSortWaves; ++k) {
    begin += smaller[k] + (k < w ? wave_sum[k] : 0);
    all += wave_sum[k];
  }
  if (threadIdx.x == 0 && r0 + range >= vocab) *used = begin + all;            // positions that count
  if ((int)threadIdx.x < rows)
    for (int k = 0; k < kSortWaves; ++k) {
      const int c = hist[k * range + threadIdx.x];
      hist[k * range + threadIdx.x] = begin;
      begin += c;
    }
  // rows without a token: their numbers, in LDS behind the counters
  int* empty = hist + kSortWaves * range;
  if (threadIdx.x == 0) empty_rows = 0;
  __syncthreads();
  if ((int)threadIdx.x < rows && total == 0) empty[atomicAdd(&empty_rows, 1)] = threadIdx.x;   // (their order does not matter)
  __syncthreads();
  if (all > 0) {
    int bits = 0;
    while ((1 << bits) < rows) ++bits;
    for (long long b = lo; b < hi; b += 64) {
      const long long at = b + lane;
      const ID v = at < hi ? ids[at] : (ID)-1;
      const long long d = (long long)v - r0;
      const bool in = usable(v, vocab, padding) && d >= 0 && d < rows;
      unsigned long long same = __ballot(in);
      if (same == 0) continue;
      for (int k = 0; k < bits; ++k) {             // the lanes with this lane's row
        const unsigned long long set = __ballot(in && ((d >> k) & 1));
        same &= ((d >> k) & 1) ? set : ~set;
      }
      if (in) {
        const int place = __popcll(same & ((1ull << lane) - 1));
        const int from = mine[d];
        __builtin_amdgcn_wave_barrier();
        if (place == 0) mine[d] = from + __popcll(same);
        __builtin_amdgcn_wave_barrier();
        keys[from + place] = (int)v;
        pos[from + place] = (int)at;
      }
    }
  }
  for (int e = w; e < empty_rows; e += kSortWaves) {
    TT* row = grad + (r0 + empty[e]) * dim;
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int c = lane * 8; c < dim; c += 512) store8<ODD>(row + c, dim - c, zero);
  }
}

// LANES lanes own one chunk x slab of LANES * 8 columns.
template <typename TT, typename TO, int LANES, bool ODD>
__global__ __launch_bounds__(256) void k_embed_sum(const TO* __restrict__ g, long long pitch, const int* __restrict__ keys,
                                                   const int* __restrict__ pos, const int* __restrict__ used, int chunk, int slabs, int dim,
                                                   float scale, TT* __restrict__ grad, float* __restrict__ parts) {
  const int n = *used;
  const long long unit = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const long long c = unit / slabs;
  const int col = (int)(unit % slabs) * LANES * 8 + (threadIdx.x % LANES) * 8, left = dim - col;
  const long long lo = c * chunk;
  if (lo >= n || left <= 0) return;
  const int hi = (int)(lo + chunk < n ? lo + chunk : n);
  const bool open = lo > 0 && keys[lo - 1] == keys[lo];     // the first run began in an earlier chunk
  bool first = true;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  int i = (int)lo;
  while (i < hi) {
    // four rows ahead: the loads of one step do not wait for one another
    const int m = hi - i < 4 ? hi - i : 4;
    int key[4];
    float v[4][8];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < m) {
        key[k] = keys[i + k];
        load8<ODD>(g + (long long)pos[i + k] * pitch + col, left, v[k]);
      }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k >= m) break;
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] += v[k][q];
      const int at = i + k;
      const bool more = at + 1 < n && keys[at + 1] == key[k];
      if (more && at + 1 < hi) continue;
      if ((first && open) || more) {               // a part of a run across chunks: its end (0) or its beginning (1)
        store8<ODD>(parts + (2 * c + (first && open ? 0 : 1)) * dim + col, left, acc);
      } else {
        float o[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) o[q] = acc[q] * scale;
        store8<ODD>(grad + (long long)key[k] * dim + col, left, o);
      }
      first = false;
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] = 0.f;
    }
    i += m;
  }
}

// One block a chunk x slab of 512 columns, for the chunks in which a run begins that ends in a later one.
template <typename TT, bool ODD>
__global__ __launch_bounds__(256) void k_embed_tail(const int* __restrict__ keys, const int* __restrict__ used, int chunk, int slabs, int dim,
                                                    float scale, TT* __restrict__ grad, const float* __restrict__ parts) {
  __shared__ float sums[4][64][9];
  const int n = *used;
  const long long c = blockIdx.x / slabs;
  const long long lo = c * chunk, hi = lo + chunk;
  if (hi >= n) return;
  const int key = keys[hi - 1];
  if (keys[hi] != key || (keys[lo] == key && lo > 0 && keys[lo - 1] == key)) return;     // nothing crosses, or it began before
  long long a = hi, b = n;                         // the run's end: first place in (hi, n] with another key
  while (a < b) {
    const long long m = (a + b) / 2;
    if (keys[m] == key) a = m + 1; else b = m;
  }
  const long long last = (a - 1) / chunk;          // chunks c + 1 .. last hold the run's further parts
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, col = (int)(blockIdx.x % slabs) * 512 + lane * 8, left = dim - col;
  const long long count = last - c, each = (count + 3) / 4;
  const long long from = c + 1 + w * each, to = from + each < last + 1 ? from + each : last + 1;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (left > 0) {
    if (w == 0) load8<ODD>(parts + (2 * c + 1) * dim + col, left, acc);
#pragma unroll 8
    for (long long k = from; k < to; ++k) {
      float v[8];
      load8<ODD>(parts + 2 * k * dim + col, left, v);
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] += v[q];
    }
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) sums[w][lane][q] = acc[q];
  __syncthreads();
  if (w == 0 && left > 0) {
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[q] = (acc[q] + sums[1][lane][q] + sums[2][lane][q] + sums[3][lane][q]) * scale;
    store8<ODD>(grad + (long long)key * dim + col, left, acc);
  }
}

int lanes_for(int dim, int most) {
  int l = 8;
  while (l < most && l * 8 < dim) l *= 2;
  return l;
}

// rows of a sorting block: one block a CU, until the counters fill the LDS
int range_for(long long vocab) {
  long long r = (vocab + kCUs - 1) / kCUs;
  return (int)(r > kMaxRange ? kMaxRange : r < 1 ? 1 : r);
}
// sorted positions of one chunk: short ones while few, so that they fill the card; at most some thousands of parts to join
int chunk_for(long long n) {
  int c = 16;
  while (c < 256 && n / c > 1024) c *= 2;
  return c;
}

struct BwdWs { size_t keys, pos, used, parts, total; long long chunks; };
BwdWs bwd_ws(long long n, int dim) {
  BwdWs w;
  w.chunks = (n + chunk_for(n) - 1) / chunk_for(n);
  w.keys = 0;
  w.pos = align_up((size_t)n * 4, 256);
  w.used = w.pos + align_up((size_t)n * 4, 256);
  w.parts = w.used + 256;
  w.total = w.parts + (w.chunks > 1 ? (size_t)w.chunks * 2 * dim * sizeof(float) : 0);
  return w;
}

template <typename TT, typename TO, typename ID, bool ODD>
int fwd(const void* ids, const void* table, long long pitch, long long vocab, long long n, int dim, float scale, void* out, hipStream_t st) {
  const int tpr = lanes_for(dim, 256);
  const long long rpb = 256 / tpr, g = (n + rpb - 1) / rpb, most = 64ll * kMaxBlocks;
  const dim3 grid((unsigned)(g < most ? g : most)), block(256);
#define OMNIHD_EMBED_FWD(L) hipLaunchKernelGGL((k_embed_fwd<TT, TO, ID, L, ODD>), grid, block, 0, st, static_cast<const ID*>(ids), \
                                               static_cast<const TT*>(table), pitch, vocab, n, dim, scale, static_cast<TO*>(out))
  switch (tpr) {
    case 8: OMNIHD_EMBED_FWD(8); break;
    case 16: OMNIHD_EMBED_FWD(16); break;
    case 32: OMNIHD_EMBED_FWD(32); break;
    case 64: OMNIHD_EMBED_FWD(64); break;
    case 128: OMNIHD_EMBED_FWD(128); break;
    default: OMNIHD_EMBED_FWD(256); break;
  }
#undef OMNIHD_EMBED_FWD
  return check_launch("token_embed_fwd");
}

template <typename TT, typename TO, typename ID, bool ODD>
int bwd(const void* ids, const void* g, long long pitch, long long vocab, long long n, int dim, float scale, long long padding, void* grad,
        char* ws, const BwdWs& at, hipStream_t st) {
  int *keys = reinterpret_cast<int*>(ws + at.keys), *pos = reinterpret_cast<int*>(ws + at.pos), *used = reinterpret_cast<int*>(ws + at.used);
  float* parts = reinterpret_cast<float*>(ws + at.parts);
  const int range = range_for(vocab), chunk = chunk_for(n);
  hipLaunchKernelGGL((k_embed_sort<TT, ID, ODD>), dim3((unsigned)((vocab + range - 1) / range)), dim3(kSortThreads),
                     (size_t)(kSortWaves + 1) * range * sizeof(int), st, static_cast<const ID*>(ids), n, vocab, padding, range, dim, keys,
                     pos, used, static_cast<TT*>(grad));
  if (n > 0) {
    const int l = lanes_for(dim, 64), slabs = (dim + l * 8 - 1) / (l * 8);
    const long long units = at.chunks * slabs, per = 256 / l;
    const dim3 grid((unsigned)((units + per - 1) / per)), block(256);
#define OMNIHD_EMBED_SUM(L) hipLaunchKernelGGL((k_embed_sum<TT, TO, L, ODD>), grid, block, 0, st, static_cast<const TO*>(g), pitch, keys, pos, \
                                               used, chunk, slabs, dim, scale, static_cast<TT*>(grad), parts)
    switch (l) {
      case 8: OMNIHD_EMBED_SUM(8); break;
      case 16: OMNIHD_EMBED_SUM(16); break;
      case 32: OMNIHD_EMBED_SUM(32); break;
      default: OMNIHD_EMBED_SUM(64); break;
    }
#undef OMNIHD_EMBED_SUM
    if (at.chunks > 1) {
      const int wide = (dim + 511) / 512;
      hipLaunchKernelGGL((k_embed_tail<TT, ODD>), dim3((unsigned)(at.chunks * wide)), dim3(256), 0, st, keys, used, chunk, wide, dim, scale,
                         static_cast<TT*>(grad), parts);
    }
  }
  return check_launch("token_embed_bwd");
}

bool row_vec(const void* p, long long pitch, int dim, int type) {
  return dim % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (pitch * type_size(type)) % 16 == 0;
}

#define OMNIHD_EMBED_TYPES(call)                                                                                   \
  (out_type == kF32 ? OMNIHD_EMBED_ID(call, float, float)                                                            \
   : out_type == kBF16 ? (table_type == kF32 ? OMNIHD_EMBED_ID(call, float, __bf16) : OMNIHD_EMBED_ID(call, __bf16, __bf16)) \
                       : (table_type == kF32 ? OMNIHD_EMBED_ID(call, float, _Float16) : OMNIHD_EMBED_ID(call, _Float16, _Float16)))
#define OMNIHD_EMBED_ID(call, TT, TO) (wide_ids ? OMNIHD_EMBED_ODD(call, TT, TO, long long) : OMNIHD_EMBED_ODD(call, TT, TO, int))

}  // namespace
}  // namespace omnihd

using namespace omnihd;

#define OMNIHD_EMBED_CHECKS                                                                                                          \
  OMNIHD_REQUIRE(n >= 0 && n < (1ll << 31) && vocab >= 1 && vocab < (1ll << 31) && dim >= 1, "0 <= n < 2^31, 1 <= vocab < 2^31, dim >= 1"); \
  OMNIHD_REQUIRE(type_ok(table_type) && type_ok(out_type) && (table_type == out_type || table_type == kF32), "types: the table has the output's type or fp32")

extern "C" int omnihd_token_embed_fwd(const void* ids, int wide_ids, long long n, const void* table, int table_type, long long table_stride,
                                      long long vocab, int dim, float scale, void* out, int out_type, void* stream) {
  OMNIHD_EMBED_CHECKS;
  if (n == 0) return OMNIHD_OK;
  OMNIHD_REQUIRE(ids && table && out && table_stride >= dim, "null pointer or short rows");
  hipStream_t st = (hipStream_t)stream;
  const bool vec = row_vec(table, table_stride, dim, table_type) && row_vec(out, dim, dim, out_type);
#define OMNIHD_EMBED_ODD(call, TT, TO, ID) (vec ? fwd<TT, TO, ID, false>(ids, table, table_stride, vocab, n, dim, scale, out, st) \
                                                : fwd<TT, TO, ID, true>(ids, table, table_stride, vocab, n, dim, scale, out, st))
  return OMNIHD_EMBED_TYPES(fwd);
#undef OMNIHD_EMBED_ODD
}

extern "C" size_t omnihd_token_embed_bwd_workspace_bytes(long long n, int dim) {
  return n < 0 || dim < 1 ? 0 : bwd_ws(n, dim).total;
}

extern "C" int omnihd_token_embed_bwd(const void* ids, int wide_ids, long long n, const void* g, int out_type, long long g_stride,
                                      long long vocab, int dim, float scale, long long padding, void* grad, int table_type,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  OMNIHD_EMBED_CHECKS;
  OMNIHD_REQUIRE(grad && workspace && (n == 0 || (ids && g && g_stride >= dim)), "null pointer or short rows");
  const BwdWs at = bwd_ws(n, dim);
  if (workspace_bytes < at.total) { set_error("token_embed_bwd: workspace %zu < required %zu", workspace_bytes, at.total); return OMNIHD_ERR_WORKSPACE; }
  OMNIHD_REQUIRE(at.chunks * ((dim + 63) / 64) < (1ll << 31), "grid");
  hipStream_t st = (hipStream_t)stream;
  char* ws = static_cast<char*>(workspace);
  const bool vec = row_vec(g, g_stride, dim, out_type) && row_vec(grad, dim, dim, table_type) && (reinterpret_cast<uintptr_t>(ws) & 15u) == 0;
#define OMNIHD_EMBED_ODD(call, TT, TO, ID) (vec ? bwd<TT, TO, ID, false>(ids, g, g_stride, vocab, n, dim, scale, padding, grad, ws, at, st) \
                                                : bwd<TT, TO, ID, true>(ids, g, g_stride, vocab, n, dim, scale, padding, grad, ws, at, st))
  return OMNIHD_EMBED_TYPES(bwd);
#undef OMNIHD_EMBED_ODD
}
