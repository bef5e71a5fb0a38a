// Embedding lookup with scaling, and the gradient of the table.
//
//   out[i]  = scale * table[id_i]                                   (a row of NaN where id_i is outside [0, vocab))
//   grad[v] = scale * sum over i with id_i = v, v != padding, of g[i]   in increasing order of i, fp32 sums, zero rows where no i is
//
// Both are bound by memory: rows gathered and rows written, no arithmetic to speak of.  The gradient's order of summation is fixed
// by sorting the positions by token, without atomics on values, so it repeats bit for bit:
//   k_embed_sort  one block per range of table rows.  Its waves each read their part of the ids, count what is smaller than the range (this
//                 gives the block's place among the sorted positions) and what falls on each row of it (counters in LDS, one set a
//                 wave), keep the latter, and put their positions in place, in order; where a wave has no room for them it reads its ids
//                 again.  So the sort is one launch with no exchange between blocks, for n ids read once or twice by each of them
//                 from the L2.  Rows that got no token are zeroed here.  Many ids go into buckets first (k_embed_count, _offsets,
//                 _place), and each block reads its bucket's.
//   k_embed_sum   chunks of sorted positions x column slabs: sums each run of equal tokens.  A run inside its chunk is written to the table's
//                 gradient, a run across chunk borders as fp32 parts to the workspace: work is even however often one token occurs.
//   k_embed_tail  joins those parts in their order.
// Measured (copy rate 5.1 TB/s): 65536 x 2048 bf16 of 100000 rows, frequent-word ids: lookup 59 us (5.9 TB/s), gradient 164 us (sort with zero rows
// 76, sums 74, tail 9; 4.1 TB/s); all ids the same 171 us; 8192 x 1024, fp32 table of 32000 rows: 8 and 42 us; a million ids x 256: 86 and 332 us (count,
// offsets and place 46, sort 116, sums 130, tail 44).
#include "token_vec.h"

namespace omnihd {
namespace {
using namespace tok;

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kMaxWidth = 1 << 24;                 // (columns are counted in int)
constexpr int kMaxRange = 896;                     // table rows of one sorting block: 16 sets of counters, 56 KB of LDS

template <typename ID> __device__ __forceinline__ bool usable(ID id, long long vocab, long long padding) {
  return id >= 0 && (long long)id < vocab && (long long)id != padding;
}

// The output is written past the caches: 65536 x 2048 bf16 of random tokens 75 us, 89 through them.  With the norm that reads it next the two take 180
// and 183 us there, 43.4 and 41.7 at 32768 x 1024, and as long up to 2048 x 4096 and 8192 x 1024.
template <typename TT, typename TO, typename ID, int TPR, bool ODD>
__global__ __launch_bounds__(256) void k_embed_fwd(const ID* __restrict__ ids, const TT* __restrict__ table, long long pitch, long long vocab,
                                                   long long n, int dim, float scale, TO* __restrict__ out) {
  constexpr int RPB = 256 / TPR;
  const int t = threadIdx.x % TPR;
  for (long long i = (long long)blockIdx.x * RPB + threadIdx.x / TPR; i < n; i += (long long)gridDim.x * RPB) {
    const long long id = (long long)ids[i];
    const bool ok = id >= 0 && id < vocab;
    for (int c = t * 8; c < dim; c += 4 * TPR * 8) {         // up to four loads in flight a lane: two in rows up to 4096 columns (fwd)
      float v[4][8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = c + j * TPR * 8;
        if (at < dim && ok) load8<ODD>(table + id * pitch + at, dim - at, v[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = c + j * TPR * 8;
        if (at >= dim) continue;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[j][k] = ok ? v[j][k] * scale : __builtin_nanf("");
        store8<ODD, true>(out + i * dim + at, dim - at, v[j]);   // past the caches (below)
      }
    }
  }
}

// LISTED: `ids` are those of the block's bucket alone (`span` rows of the table, a multiple of `range`), with their positions
template <typename TT, typename ID, bool LISTED, bool ODD>
__global__ __launch_bounds__(kSortThreads) void k_embed_sort(const ID* __restrict__ ids, const int* __restrict__ where,
                                                             const int* __restrict__ starts, long long n, long long vocab, long long padding,
                                                             int span, int range, int cap, int dim, int stream, int* __restrict__ keys, int* __restrict__ pos,
                                                             int* __restrict__ used, TT* __restrict__ grad) {
  extern __shared__ int hist[];                    // [waves][range] counters, [range] empty rows, [waves][cap] positions, [waves][cap] rows
  __shared__ int wave_sum[kSortWaves], empty_rows, smaller[kSortWaves];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const unsigned long long before = (1ull << lane) - 1;
  const long long r0 = (long long)blockIdx.x * range;
  const int rows = (int)(vocab - r0 < range ? vocab - r0 : range);
  int* empty = hist + kSortWaves * range;
  int* found_pos = empty + range + w * cap;        // this wave's tokens of the range, in order, as far as there is room
  short* found_row = reinterpret_cast<short*>(empty + range + kSortWaves * cap) + w * cap;
  for (int i = threadIdx.x; i < kSortWaves * range; i += kSortThreads) hist[i] = 0;
  if (threadIdx.x == 0) empty_rows = 0;
  __syncthreads();
  int smaller_buckets = 0;
  if (LISTED) {
    const int b = (int)(r0 / span);
    smaller_buckets = starts[b];
    n = starts[b + 1] - smaller_buckets;
    ids += smaller_buckets;
    where += smaller_buckets;
  }
  // each wave has a run of the ids, a multiple of 64
  const long long part = ((n + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const long long lo = part * w < n ? part * w : n, hi = lo + part < n ? lo + part : n;
  int* mine = hist + w * range;
  int less = 0, found = 0;                         // (the same in all lanes: counted from ballots)
  // An id as 32 bits (all ones: none), so that one comparison each tells whether it is smaller than the range, or in it
  const unsigned pad32 = padding < 0 ? ~0u : (unsigned)padding, vocab32 = (unsigned)vocab, first32 = (unsigned)r0, rows32 = (unsigned)rows;
  auto narrow = [&](ID v) { const unsigned u = (unsigned)v; return v >= 0 && (sizeof(ID) == 4 || (unsigned long long)v >> 32 == 0) && u < vocab32 && u != pad32 ? u : ~0u; };
  auto look = [&](ID v, long long at) {
    const unsigned u = narrow(v), d = u - first32;
    less += __popcll(__ballot(u < first32));
    const unsigned long long who = __ballot(d < rows32);         // (no range ends at all ones: vocab < 2^31)
    if (who == 0) return;
    if (d < rows32) {
      atomicAdd(mine + d, 1);
      const int to = found + __popcll(who & before);
      if (to < cap) { found_pos[to] = (int)at; found_row[to] = (short)d; }
    }
    found += __popcll(who);
  };
  long long b0 = lo;
  for (; b0 + 512 <= hi; b0 += 512) {              // eight loads in flight a lane
    ID v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = ids[b0 + 64 * k + lane];
#pragma unroll
    for (int k = 0; k < 8; ++k) look(v[k], b0 + 64 * k + lane);
  }
  for (; b0 < hi; b0 += 64) look(b0 + lane < hi ? ids[b0 + lane] : (ID)-1, b0 + lane);
  if (lane == 0) smaller[w] = less;
  __syncthreads();
  // where each row's and wave's positions begin
  int total = 0;
  if ((int)threadIdx.x < rows)
    for (int k = 0; k < kSortWaves; ++k) total += hist[k * range + threadIdx.x];
  if ((int)threadIdx.x < rows && total == 0) empty[atomicAdd(&empty_rows, 1)] = threadIdx.x;   // (their order does not matter)
  int scan = total;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(scan, o, 64);
    if (lane >= o) scan += up;
  }
  if (lane == 63) wave_sum[w] = scan;
  __syncthreads();
  int begin = smaller_buckets + scan - total, all = 0;
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
  __syncthreads();
  int bits = 0;
  while ((1 << bits) < rows) ++bits;
  // 64 tokens of this wave in order: each to the place that its row has reached
  auto place = [&](bool in, int d, int at) {
    unsigned long long same = 0, todo = __ballot(in);
    for (int k = 0; k < 3 && todo; ++k) {          // a frequent token or two, one comparison each ...
      const unsigned long long like = __ballot(in && d == __builtin_amdgcn_readlane(d, __builtin_ctzll(todo)));
      if (like >> lane & 1) same = like;
      todo &= ~like;
    }
    if (todo) {                                    // ... and the rest by the bits of their rows: the lanes with this lane's row
      const bool rest = todo >> lane & 1;
      unsigned long long mine_too = todo;
      for (int k = 0; k < bits; ++k) {
        const unsigned long long set = __ballot(rest && ((d >> k) & 1));
        mine_too &= ((d >> k) & 1) ? set : ~set;
      }
      if (rest) same = mine_too;
    }
    if (in) {
      const int nth = __popcll(same & before), from = mine[d];
      __builtin_amdgcn_wave_barrier();
      if (nth == 0) mine[d] = from + __popcll(same);
      __builtin_amdgcn_wave_barrier();
      keys[from + nth] = (int)(r0 + d);
      pos[from + nth] = at;
    }
  };
  if (found <= cap) {
    for (int b = 0; b < found; b += 64) {
      const bool in = b + lane < found;
      const int at = in ? found_pos[b + lane] : 0;
      place(in, in ? found_row[b + lane] : 0, LISTED && in ? where[at] : at);
    }
  } else {                                         // a crowded range: the ids once more
    for (long long b = lo; b < hi; b += 512) {
      ID v[8];
      int at[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const long long i = b + 64 * k + lane;
        v[k] = i < hi ? ids[i] : (ID)-1;
        at[k] = LISTED && i < hi ? where[i] : (int)i;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const unsigned d = narrow(v[k]) - first32;
        const bool in = d < rows32;
        if (__ballot(in) != 0) place(in, in ? (int)d : 0, at[k]);
      }
    }
  }
  for (int e = w; e < empty_rows; e += kSortWaves) {
    TT* row = grad + (r0 + empty[e]) * dim;
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (stream)
      for (int c = lane * 8; c < dim; c += 512) store8<ODD, true>(row + c, dim - c, zero);
    else
      for (int c = lane * 8; c < dim; c += 512) store8<ODD>(row + c, dim - c, zero);
  }
}

// Many ids: first into buckets of `span` table rows, in order, so that each sorting block reads its bucket's alone.  Blocks of 4 waves, a
// chunk of ids each: count, offsets (one block a bucket: where each chunk's share of it begins), place.
constexpr int kChunkIds = 4096, kMaxBuckets = 2048;

template <typename ID>
__global__ __launch_bounds__(256) void k_embed_count(const ID* __restrict__ ids, long long n, long long vocab, long long padding, int span,
                                                     int buckets, int chunks, int* __restrict__ counts) {
  __shared__ int hist[kMaxBuckets];
  for (int b = threadIdx.x; b < buckets; b += 256) hist[b] = 0;
  __syncthreads();
  const long long lo = (long long)blockIdx.x * kChunkIds;
#pragma unroll 4
  for (int i = threadIdx.x; i < kChunkIds; i += 256) {
    const ID v = lo + i < n ? ids[lo + i] : (ID)-1;
    if (usable(v, vocab, padding)) atomicAdd(hist + (unsigned)v / (unsigned)span, 1);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < buckets; b += 256) counts[(long long)b * chunks + blockIdx.x] = hist[b];
}

__global__ __launch_bounds__(256) void k_embed_offsets(int chunks, int* __restrict__ counts, int* __restrict__ totals) {
  __shared__ int wave_sum[4];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int* mine = counts + (long long)blockIdx.x * chunks;
  int run = 0;
  for (int b = 0; b < chunks; b += 256) {
    const int i = b + threadIdx.x, v = i < chunks ? mine[i] : 0;
    int scan = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(scan, o, 64);
      if (lane >= o) scan += up;
    }
    if (lane == 63) wave_sum[w] = scan;
    __syncthreads();
    int at = run + scan - v;
    for (int k = 0; k < 4; ++k) {
      at += k < w ? wave_sum[k] : 0;
      run += wave_sum[k];
    }
    if (i < chunks) mine[i] = at;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = run;
}

template <typename ID>
__global__ __launch_bounds__(256) void k_embed_place(const ID* __restrict__ ids, long long n, long long vocab, long long padding, int span,
                                                     int buckets, int chunks, const int* __restrict__ offsets, const int* __restrict__ totals,
                                                     int* __restrict__ starts, int* __restrict__ out_ids, int* __restrict__ out_pos) {
  __shared__ int hist[4][kMaxBuckets], wave_sum[4];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const unsigned long long before = (1ull << lane) - 1;
  for (int b = threadIdx.x; b < 4 * kMaxBuckets; b += 256) (&hist[0][0])[b] = 0;
  __syncthreads();
  const long long lo = (long long)blockIdx.x * kChunkIds + w * (kChunkIds / 4);
#pragma unroll 4
  for (int i = lane; i < kChunkIds / 4; i += 64) {
    const ID v = lo + i < n ? ids[lo + i] : (ID)-1;
    if (usable(v, vocab, padding)) atomicAdd(&hist[w][(unsigned)v / (unsigned)span], 1);
  }
  __syncthreads();
  // eight neighbouring buckets a thread: where each begins, this chunk's and each wave's share of it
  constexpr int PER = kMaxBuckets / 256;
  int total[PER], sum = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = threadIdx.x * PER + k;
    total[k] = b < buckets ? totals[b] : 0;
    sum += total[k];
  }
  int scan = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(scan, o, 64);
    if (lane >= o) scan += up;
  }
  if (lane == 63) wave_sum[w] = scan;
  __syncthreads();
  int begin = scan - sum;
  for (int k = 0; k < w; ++k) begin += wave_sum[k];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = threadIdx.x * PER + k;
    if (b < buckets) {
      if (blockIdx.x == 0) {
        starts[b] = begin;
        if (b == buckets - 1) starts[buckets] = begin + total[k];
      }
      int at = begin + offsets[(long long)b * chunks + blockIdx.x];
      for (int q = 0; q < 4; ++q) {
        const int c = hist[q][b];
        hist[q][b] = at;
        at += c;
      }
    }
    begin += total[k];
  }
  __syncthreads();
  int bits = 0;
  while ((1 << bits) < buckets) ++bits;
  for (int i = lane; i < kChunkIds / 4; i += 64) {
    const ID v = lo + i < n ? ids[lo + i] : (ID)-1;
    const bool in = usable(v, vocab, padding);
    const unsigned b = in ? (unsigned)v / (unsigned)span : 0;
    unsigned long long same = __ballot(in);
    for (int k = 0; k < bits; ++k) {
      const unsigned long long set = __ballot(in && ((b >> k) & 1));
      same &= ((b >> k) & 1) ? set : ~set;
    }
    if (in) {
      const int nth = __popcll(same & before), from = hist[w][b];
      __builtin_amdgcn_wave_barrier();
      if (nth == 0) hist[w][b] = from + __popcll(same);
      __builtin_amdgcn_wave_barrier();
      out_ids[from + nth] = (int)v;
      out_pos[from + nth] = (int)(lo + i);
    }
  }
}

// LANES lanes own one chunk x slab of LANES * 8 columns.  They hold LANES sorted positions at a time, one each, so the rows' addresses
// are there before the rows are asked for: eight row loads in flight.
template <typename TT, typename TO, int LANES, bool ODD>
__global__ __launch_bounds__(256) void k_embed_sum(const TO* __restrict__ g, long long pitch, const int* __restrict__ keys,
                                                   const int* __restrict__ pos, const int* __restrict__ used, int chunk, int slabs, int dim,
                                                   float scale, TT* __restrict__ grad, float* __restrict__ parts) {
  const int n = *used, lane = threadIdx.x % LANES;
  const long long unit = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const long long c = unit / slabs;
  const int col = (int)(unit % slabs) * LANES * 8 + lane * 8, left = dim - col;
  const long long lo = c * chunk;
  if (lo >= n) return;                             // (the same in all lanes of a unit)
  const int len = (int)(lo + chunk < n ? chunk : n - lo);        // places are counted from the chunk's first: n may end at 2^31 - 1
  const int earlier = lo > 0 ? keys[lo - 1] : -1, later = lo + len < n ? keys[lo + len] : -1;
  keys += lo;
  pos += lo;
  bool first = true, open = false;                 // open: the chunk's first run began in an earlier one
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto at = [&](int v, int i) { return LANES == 64 ? __builtin_amdgcn_readlane(v, i) : __shfl(v, i, LANES); };
  for (int b = 0; b < len; b += LANES) {
    const int m = len - b < LANES ? len - b : LANES;
    const int mykey = lane < m ? keys[b + lane] : -1, mypos = lane < m ? pos[b + lane] : 0;
    const int beyond = b + m < len ? keys[b + m] : later;     // the key behind these
    if (b == 0) open = at(mykey, 0) == earlier;
    for (int i = 0; i < m; i += 8) {
      float v[8][8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + k < m) {
          const long long p = at(mypos, i + k);
          if (left > 0) load8<ODD>(g + p * pitch + col, left, v[k]);
        }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (i + k >= m) break;
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] += v[k][q];
        const int key = at(mykey, i + k), next = i + k + 1 < m ? at(mykey, i + k + 1) : beyond;
        const bool ends = b + i + k + 1 == len;
        if (key == next && !ends) continue;
        if ((first && open) || key == next) {      // a part of a run across chunks: its end (0) or its beginning (1)
          if (left > 0) store8<ODD>(parts + (2 * c + (first && open ? 0 : 1)) * dim + col, left, acc);
        } else {
          float o[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) o[q] = acc[q] * scale;
          if (left > 0) store8<ODD>(grad + (long long)key * dim + col, left, o);
        }
        first = false;
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] = 0.f;
      }
    }
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

// rows of a sorting block: two blocks a CU, until the counters fill the LDS
int range_for(long long vocab) {
  long long r = (vocab + 2 * kCUs - 1) / (2 * kCUs);
  return (int)(r > kMaxRange ? kMaxRange : r < 1 ? 1 : r);
}
// tokens that a wave of a sorting block can keep: what is left of 64 KB (two blocks a CU)
int cap_for(int range) { return (64000 - (kSortWaves + 1) * range * 4) / (kSortWaves * 6) & ~1; }
// sorted positions of one chunk: as many chunks x slabs as give 4096 waves where the row is wide, no fewer than 8 positions, no more than 256
// (72946 positions of 52 columns: 135 us in chunks of 128, whose 570 groups of 8 lanes fill 18 blocks)
int chunk_for(long long n, int dim) {
  const int l = lanes_for(dim, 64), slabs = (dim + l * 8 - 1) / (l * 8);
  int c = 8;
  while (c < 256 && (n / (2 * c)) * slabs * l >= 4096ll * 64) c *= 2;
  return c;
}
// From here on the ids are put into buckets first: three more launches, but no block reads all of them (frequent-word ids, 131072 x 512: 102 us so, 92
// to 119 without; 160000 x 256: 107 us, 147 without; 262144 x 256: 118, 201).
constexpr long long kBucketIds = 144 << 10;
int span_for(long long vocab) {
  const long long range = range_for(vocab), ranges = (vocab + range - 1) / range;
  return (int)(range * ((ranges + kMaxBuckets - 1) / kMaxBuckets));
}

struct BwdWs { size_t keys, pos, used, parts, ids, where, starts, totals, counts, total; long long chunks, buckets, id_chunks; };
BwdWs bwd_ws(long long n, long long vocab, int dim) {
  BwdWs w{};
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t from = at; at += align_up(bytes, 256); return from; };
  const int chunk = chunk_for(n, dim);
  w.chunks = (n + chunk - 1) / chunk;
  w.keys = take((size_t)n * 4);
  w.pos = take((size_t)n * 4);
  w.used = take(4);
  w.parts = take(w.chunks > 1 ? (size_t)w.chunks * 2 * dim * sizeof(float) : 0);
  if (n >= kBucketIds) {
    w.buckets = (vocab + span_for(vocab) - 1) / span_for(vocab);
    w.id_chunks = (n + kChunkIds - 1) / kChunkIds;
    w.ids = take((size_t)n * 4);
    w.where = take((size_t)n * 4);
    w.starts = take((size_t)(w.buckets + 1) * 4);
    w.totals = take((size_t)w.buckets * 4);
    w.counts = take((size_t)w.buckets * w.id_chunks * 4);
  }
  w.total = at;
  return w;
}

template <typename TT, typename TO, typename ID, bool ODD>
int fwd(const void* ids, const void* table, long long pitch, long long vocab, long long n, int dim, float scale, void* out, hipStream_t st) {
  // two loads a lane and row in flight: 65536 x 2048 bf16 in training 238 us a pass with two, 247 with one, 236 with four (and 64 lanes); alone 59
  // with each
  const int tpr = lanes_for((dim + 1) / 2, 256);
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
  const int range = range_for(vocab), cap = cap_for(range), chunk = chunk_for(n, dim);
  const dim3 sorters((unsigned)((vocab + range - 1) / range));
  const size_t lds = (size_t)(kSortWaves + 1) * range * sizeof(int) + (size_t)kSortWaves * cap * 6;
  const int stream = (size_t)vocab * dim * sizeof(TT) > kCacheBytes;
  if (at.buckets) {
    const int span = span_for(vocab), buckets = (int)at.buckets, chunks = (int)at.id_chunks;
    int *listed = reinterpret_cast<int*>(ws + at.ids), *where = reinterpret_cast<int*>(ws + at.where), *starts = reinterpret_cast<int*>(ws + at.starts);
    int *totals = reinterpret_cast<int*>(ws + at.totals), *counts = reinterpret_cast<int*>(ws + at.counts);
    const ID* from = static_cast<const ID*>(ids);
    hipLaunchKernelGGL((k_embed_count<ID>), dim3(chunks), dim3(256), 0, st, from, n, vocab, padding, span, buckets, chunks, counts);
    hipLaunchKernelGGL(k_embed_offsets, dim3(buckets), dim3(256), 0, st, chunks, counts, totals);
    hipLaunchKernelGGL((k_embed_place<ID>), dim3(chunks), dim3(256), 0, st, from, n, vocab, padding, span, buckets, chunks, counts, totals, starts,
                       listed, where);
    hipLaunchKernelGGL((k_embed_sort<TT, int, true, ODD>), sorters, dim3(kSortThreads), lds, st, listed, where, starts, n, vocab, padding, span, range,
                       cap, dim, stream, keys, pos, used, static_cast<TT*>(grad));
  } else {
    hipLaunchKernelGGL((k_embed_sort<TT, ID, false, ODD>), sorters, dim3(kSortThreads), lds, st, static_cast<const ID*>(ids), nullptr, nullptr, n, vocab,
                       padding, 1, range, cap, dim, stream, keys, pos, used, static_cast<TT*>(grad));
  }
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
  OMNIHD_REQUIRE(n >= 0 && n < (1ll << 31) && vocab >= 1 && vocab < (1ll << 31) && dim >= 1 && dim <= kMaxWidth,                         \
                 "0 <= n < 2^31, 1 <= vocab < 2^31, 1 <= dim <= 2^24");                                                                      \
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

extern "C" size_t omnihd_token_embed_bwd_workspace_bytes(long long n, long long vocab, int dim) {
  return n < 0 || n >= (1ll << 31) || vocab < 1 || vocab >= (1ll << 31) || dim < 1 || dim > kMaxWidth ? 0 : bwd_ws(n, vocab, dim).total;
}

extern "C" int omnihd_token_embed_bwd(const void* ids, int wide_ids, long long n, const void* g, int out_type, long long g_stride,
                                      long long vocab, int dim, float scale, long long padding, void* grad, int table_type,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  OMNIHD_EMBED_CHECKS;
  OMNIHD_REQUIRE(grad && workspace && (n == 0 || (ids && g && g_stride >= dim)), "null pointer or short rows");
  if (padding >= vocab) padding = -1;              // no row of the table (ids are compared as 32 bits below)
  const BwdWs at = bwd_ws(n, vocab, dim);
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
