// Norms before and after a block of a residual stream, fused with the block's gate and the residual scale.
//
//   norm(v; w) = v * rsqrt(mean(v^2) + eps) * w
//   join:  x' = r * x + gate * norm(y; post),  h = norm(x'; next)          (post, gate, next may each be absent)
//   alone: h = norm(x; next)                                              (y == NULL)
//
// Backward, with nh = y * ry, xh = x' * rx (ry, rx kept from the forward, 8 bytes a row), a = dh * next:
//   t  = dx' + rx * (a - xh * mean(a * xh)),      dx = r * t,             dnext = sum_rows dh * xh
//   m  = t * gate * post,  dy = ry * (m - nh * mean(m * nh)),             dpost = sum_rows t * gate * nh,  dgate = sum t * nh * post
// x' is computed again in fp32 from x and y (which have to be read anyway) and not read back: its stored form is rounded, and weight
// gradients in fp32 would carry that rounding (1e-3 of them for bf16 rows).
//
// Bound by HBM: 4 rows of D forward, 6 backward, about 50 operations an element in all.  So each row is read once into registers
// (8 elements a lane and step, TPR lanes a row, the next row asked for while one is worked on), its one or two sums go over the
// lanes by DPP (over LDS beyond a wave), and the column sums of the weight gradients stay in registers over all rows that a block
// walks; only their block sums go through memory ([blocks][2][D] fp32), joined in a fixed order by a second launch.
// Measured (copy rate 5.1 TB/s): 16384 x 4096 bf16 forward 92 us (5.8 TB/s, reads past the cache), backward 191 us (4.2); 76800 x 256 fp16 norm
// alone 12.7 / 27 us; 20000 x 512 fp32 32 / 54 us; 8 x 4096 one launch of 3.8 us.  Rows beyond 8192 columns: backward 2.6 TB/s.  A gate a token as a
// gate a channel; a full gate 128 / 253 us (5.2, 4.2 TB/s); a gate for every four rows 123 / 323 us (a block and its two sums for each: 2.9).
// With a gate per channel (or per sample and channel) S = sum_rows t * nh serves both gradients: dgate = S * post, dpost = sum S * gate.
#include "token_vec.h"

namespace omnihd {
namespace {
using namespace tok;

enum { kGateNone = 0, kGateRows = 1, kGateToken = 2, kGateFull = 3 };

struct BlockArgs {
  const void *x, *y, *post, *gate, *next;
  const void *dxo, *dh;                  // backward: gradients of x' and h (either may be NULL)
  void *xo, *ho, *gx, *gy, *ggate;
  float *stats, *part;
  long long rows, xs, ys, gs, dxos, dhs; // row strides in elements (outputs are dense)
  long long per_gate, per_split;         // rows of one gate row, of one block
  unsigned first;                        // backward: the launch's first block of (gate row, split)
  int splits, dim, post_type, gate_type, next_type, gate_kind, stream;
  float r, eps;
};

template <int TPR> constexpr int threads_of() { return TPR > 256 ? TPR : 256; }

template <typename TA, typename TX, int TPR, int NV, bool ODD, bool HASY, bool STREAM>
__global__ __launch_bounds__(threads_of<TPR>()) void k_block_fwd(BlockArgs a) {
  constexpr int TPB = threads_of<TPR>(), RPB = TPB / TPR;
  __shared__ float red[32];
  int turn = 0;
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, D = a.dim;
  const float inv_d = 1.f / (float)D;
  const bool post = HASY && a.post, one_gate = a.gate_kind == kGateRows && a.per_gate >= a.rows;
  float gp[NV][8], wn[NV][8];            // post (times the gate, where one serves all rows) and next
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + t) * 8, left = D - c;
#pragma unroll
    for (int k = 0; k < 8; ++k) gp[j][k] = wn[j][k] = 1.f;
    if (left <= 0) continue;
    if (post) load8_any<ODD>(a.post, a.post_type, c, left, gp[j]);
    if (a.next) load8_any<ODD>(a.next, a.next_type, c, left, wn[j]);
    if (HASY && one_gate) {
      float g[8];
      load8_any<ODD>(a.gate, a.gate_type, c, left, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) gp[j][k] *= g[k];
    }
  }
  typename Raw<TX>::V xr[NV];            // the next row, asked for while this one is worked on
  typename Raw<TA>::V yr[NV];
  auto ask = [&](long long row) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + t) * 8, left = D - c;
      xr[j] = typename Raw<TX>::V{};
      if (HASY) yr[j] = typename Raw<TA>::V{};
      if (row >= a.rows || left <= 0) continue;
      const TX* x = static_cast<const TX*>(a.x) + row * a.xs + c;
      const TA* y = static_cast<const TA*>(a.y) + (HASY ? row * a.ys + c : 0);
      xr[j] = raw8<ODD, STREAM>(x, left);
      if (HASY) yr[j] = raw8<ODD, STREAM>(y, left);
    }
  };
  const long long step = (long long)gridDim.x * RPB;
  ask((long long)blockIdx.x * RPB + sub);
  for (long long base = (long long)blockIdx.x * RPB; base < a.rows; base += step) {
    const long long row = base + sub;
    const bool act = row < a.rows;
    float x[NV][8], y[NV][8], ry = 1.f, rx = 1.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[j][k] = (float)xr[j][k];
        y[j][k] = HASY ? (float)yr[j][k] : 0.f;
      }
    ask(row + step);
    if (HASY) {
      if (post) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int k = 0; k < 8; ++k) s = fmaf(y[j][k], y[j][k], s);
        ry = __builtin_amdgcn_rsqf(fmaf(group<TPR>(s, Add(), red, turn), inv_d, a.eps));
      }
      float scalar = ry;
      if (a.gate_kind == kGateToken && act) scalar *= load1_any(a.gate, a.gate_type, row);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + t) * 8, left = D - c;
        if (!act || left <= 0) continue;
        float g[8];
        const bool own_gate = a.gate_kind == kGateFull || (a.gate_kind == kGateRows && !one_gate);
        if (own_gate) load8_any<ODD>(a.gate, a.gate_type, a.gate_kind == kGateFull ? row * a.gs + c : (row / a.per_gate) * a.gs + c, left, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float w = own_gate ? gp[j][k] * g[k] : gp[j][k];
          x[j][k] = fmaf(y[j][k] * scalar, w, a.r * x[j][k]);
        }
        if (ODD) {                       // what the row does not have stays out of the sums
#pragma unroll
          for (int k = 0; k < 8; ++k) x[j][k] = k < left ? x[j][k] : 0.f;
        }
        if (a.xo) store8<ODD>(static_cast<TX*>(a.xo) + row * D + c, left, x[j]);
      }
    }
    if (a.next) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < 8; ++k) s = fmaf(x[j][k], x[j][k], s);
      rx = __builtin_amdgcn_rsqf(fmaf(group<TPR>(s, Add(), red, turn), inv_d, a.eps));
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + t) * 8, left = D - c;
        if (!act || left <= 0) continue;
        float h[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) h[k] = x[j][k] * rx * wn[j][k];
        store8<ODD>(static_cast<TA*>(a.ho) + row * D + c, left, h);
      }
    }
    if (a.stats && act && t == 0) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(ry, rx);
  }
}

// One block: `per_split` rows of one gate row (unit = gate row * splits + split).  With two vectors a lane (rows beyond 8192) there are
// not registers for all of it: the weights are read when they are used, no row is asked for ahead, and the column sums are kept in
// LDS (128 KB) - 2048 rows of 16384 bf16: 312 us with them in registers, which spill.
template <typename TA, typename TX, int TPR, int NV, bool ODD, bool HASY>
__global__ __launch_bounds__(threads_of<TPR>()) void k_block_bwd(BlockArgs a) {
  constexpr int TPB = threads_of<TPR>(), RPB = TPB / TPR;
  constexpr bool LEAN = NV > 1;
  constexpr int DEPTH = TPR == 512 ? 2 : 1;         // rows asked for ahead: one block of 512 a CU has room (and need) for two
  __shared__ float red[32];
  __shared__ float fold[RPB > 1 ? TPB * 8 : 1];
  int turn = 0;
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, D = a.dim;
  const float inv_d = 1.f / (float)D;
  const bool post = HASY && a.post;
  const unsigned unit = a.first + blockIdx.x;
  const long long grp = unit / (unsigned)a.splits, first = grp * a.per_gate, lo = first + (unit % (unsigned)a.splits) * a.per_split;
  long long hi = lo + a.per_split;
  if (hi > first + a.per_gate) hi = first + a.per_gate;
  if (hi > a.rows) hi = a.rows;
  auto weights = [&](int j, float (&gp)[8], float (&wn)[8]) {     // post (times the gate row), next
    const int c = (j * TPR + t) * 8, left = D - c;
#pragma unroll
    for (int k = 0; k < 8; ++k) gp[k] = wn[k] = 1.f;
    if (left <= 0) return;
    if (post) load8_any<ODD>(a.post, a.post_type, c, left, gp);
    if (a.next) load8_any<ODD>(a.next, a.next_type, c, left, wn);
    if (HASY && a.gate_kind == kGateRows) {
      float g[8];
      load8_any<ODD>(a.gate, a.gate_type, grp * a.gs + c, left, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) gp[k] *= g[k];
    }
  };
  float gph[LEAN ? 1 : NV][8], wnh[LEAN ? 1 : NV][8], awr[LEAN ? 1 : NV][8], aur[LEAN ? 1 : NV][8];
  extern __shared__ float wide[];        // [2][NV * 8][TPB]
  auto aw = [&](int j, int k) -> float& { return LEAN ? wide[(j * 8 + k) * TPB + threadIdx.x] : awr[LEAN ? 0 : j][k]; };
  auto au = [&](int j, int k) -> float& { return LEAN ? wide[(NV * 8 + j * 8 + k) * TPB + threadIdx.x] : aur[LEAN ? 0 : j][k]; };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if constexpr (!LEAN) weights(j, gph[j], wnh[j]);
#pragma unroll
    for (int k = 0; k < 8; ++k) aw(j, k) = au(j, k) = 0.f;
  }
  struct Ahead { typename Raw<TX>::V xr[NV], dr[NV]; typename Raw<TA>::V yr[NV], hr[NV]; float2 stat; };
  auto ask = [&](Ahead& r, long long row) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + t) * 8, left = D - c;
      r.xr[j] = r.dr[j] = typename Raw<TX>::V{};
      r.yr[j] = r.hr[j] = typename Raw<TA>::V{};
      if (row >= hi || left <= 0) continue;
      if (a.dh) r.xr[j] = raw8<ODD>(static_cast<const TX*>(a.x) + row * a.xs + c, left);
      if (HASY) r.yr[j] = raw8<ODD>(static_cast<const TA*>(a.y) + row * a.ys + c, left);
      if (HASY && a.dxo) r.dr[j] = raw8<ODD>(static_cast<const TX*>(a.dxo) + row * a.dxos + c, left);
      if (a.dh) r.hr[j] = raw8<ODD>(static_cast<const TA*>(a.dh) + row * a.dhs + c, left);
    }
    r.stat = make_float2(1.f, 1.f);
    if (row < hi) r.stat = *reinterpret_cast<const float2*>(a.stats + 2 * row);
  };
  // one row: what was asked for of it, and the row to ask for in its place
  auto work = [&](Ahead& r, long long row) {
    const bool act = row < hi;
    if (LEAN) ask(r, row);
    const float ry = r.stat.x, rx = r.stat.y;
    float x[NV][8], y[NV][8], d[NV][8], h[NV][8], tok = 1.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[j][k] = (float)r.xr[j][k];
        y[j][k] = HASY ? (float)r.yr[j][k] * ry : 0.f;             // nh
        d[j][k] = HASY ? (float)r.dr[j][k] : 0.f;
        h[j][k] = (float)r.hr[j][k];
      }
    if (HASY && a.gate_kind == kGateToken && act) tok = load1_any(a.gate, a.gate_type, row);
    if (!LEAN) ask(r, row + DEPTH * RPB);
    auto row_gate = [&](int j, float (&g)[8]) {                  // what multiplies post and a gate row here: a gate of this very row
      const int c = (j * TPR + t) * 8, left = D - c;
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = a.gate_kind == kGateFull ? 0.f : tok;
      if (HASY && a.gate_kind == kGateFull && act && left > 0) load8_any<ODD>(a.gate, a.gate_type, row * a.gs + c, left, g);
    };
    if (a.dh) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float gl[8], wl[8], g[8];
        if constexpr (LEAN) weights(j, gl, wl);
        const float(&gp)[8] = *(LEAN ? &gl : &gph[LEAN ? 0 : j]);
        const float(&wn)[8] = *(LEAN ? &wl : &wnh[LEAN ? 0 : j]);
        if (HASY) row_gate(j, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float xn = HASY ? fmaf(y[j][k], gp[k] * g[k], a.r * x[j][k]) : x[j][k];
          x[j][k] = xn * rx;                                     // xh
          au(j, k) = fmaf(h[j][k], x[j][k], au(j, k));
          h[j][k] *= wn[k];                                      // a
          s = fmaf(h[j][k], x[j][k], s);
        }
      }
      s = group<TPR>(s, Add(), red, turn) * inv_d;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < 8; ++k) d[j][k] = fmaf(rx, h[j][k] - x[j][k] * s, d[j][k]);       // t
    }
    if (a.gx) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + t) * 8, left = D - c;
        if (!act || left <= 0) continue;
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = (HASY ? a.r : 1.f) * d[j][k];
        store8<ODD>(static_cast<TX*>(a.gx) + row * D + c, left, o);
      }
    }
    if (!HASY) return;
    float s = 0.f;                       // sum of t * nh * post (* gate, unless the gate is the token's): mean(m * nh), a token gate's gradient
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + t) * 8, left = D - c;
      float dg[8], gl[8], wl[8], g[8];
      if constexpr (LEAN) weights(j, gl, wl);
      const float(&gp)[8] = *(LEAN ? &gl : &gph[LEAN ? 0 : j]);
      row_gate(j, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float tn = d[j][k] * y[j][k];
        aw(j, k) = a.gate_kind == kGateRows ? aw(j, k) + tn : fmaf(tn, g[k], aw(j, k));
        dg[k] = tn * gp[k];
        s = fmaf(dg[k], a.gate_kind == kGateFull ? g[k] : 1.f, s);
        d[j][k] *= gp[k] * g[k];                                 // m
      }
      if (a.gate_kind == kGateFull && a.ggate && act && left > 0) store8_any<ODD>(a.ggate, a.gate_type, row * D + c, left, dg);
    }
    float mean = 0.f;
    if (post || (a.gate_kind == kGateToken && a.ggate)) {
      s = group<TPR>(s, Add(), red, turn);
      if (a.gate_kind == kGateToken && a.ggate && act && t == 0) store1_any(a.ggate, a.gate_type, row, s);
      if (post) mean = s * tok * inv_d;
    }
    if (a.gy) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + t) * 8, left = D - c;
        if (!act || left <= 0) continue;
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = ry * (d[j][k] - y[j][k] * mean);
        store8<ODD>(static_cast<TA*>(a.gy) + row * D + c, left, o);
      }
    }
  };
  Ahead r0, r1;
  if (!LEAN) ask(r0, lo + sub);
  if (DEPTH > 1) ask(r1, lo + RPB + sub);
  for (long long base = lo; base < hi; base += DEPTH * RPB) {
    work(r0, base + sub);
    if (DEPTH > 1 && base + RPB < hi) work(r1, base + RPB + sub);
  }
  if (!a.part) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (which == 0 && !HASY) continue;
    if (which == 1 && !a.next) continue;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + t) * 8, left = D - c;
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = which ? au(j, k) : aw(j, k);
      if constexpr (RPB > 1) {           // the block's rows side by side: added in the order of their places
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) fold[k * TPB + threadIdx.x] = v[k];
        __syncthreads();
        if (sub == 0) {
          for (int o = 1; o < RPB; ++o)
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] += fold[k * TPB + o * TPR + t];
        }
      }
      if (sub == 0 && left > 0) store8<ODD>(a.part + ((long long)unit * 2 + which) * D + c, left, v);
    }
  }
}

// Block sums -> dnext, dpost (grp -1) and the gradient of each gate row.  16 columns by 64 places of the blocks, whose sums are joined in a
// fixed order; four loads in flight a lane.  Gate rows of one block sum each have nothing to join: the blocks behind the first tiles walk
// over them, `lanes` columns at a time (there may be as many of them as rows: one block each and 16 columns would not fit a grid).
__global__ __launch_bounds__(1024) void k_block_cols(const float* __restrict__ part, long long blocks, int splits, int dim, int lanes, const void* post,
                                                     int post_type, const void* gate, int gate_type, long long gs, int gate_kind,
                                                     void* gpost, void* ggate, void* gnext, int next_type) {
  __shared__ float s0[64][17], s1[64][17];
  const int tiles = (dim + 15) / 16;
  if (splits == 1 && (int)blockIdx.x >= tiles) {
    const int each = 1024 / lanes;
    for (long long grp = (long long)(blockIdx.x - tiles) * each + threadIdx.x / lanes; grp < blocks; grp += (long long)(gridDim.x - tiles) * each)
      for (int c = threadIdx.x % lanes; c < dim; c += lanes) {
        const float w = part[grp * 2 * dim + c];
        store1_any(ggate, gate_type, grp * dim + c, post ? w * load1_any(post, post_type, c) : w);
      }
    return;
  }
  const int c = (blockIdx.x % tiles) * 16 + (threadIdx.x & 15), place = threadIdx.x >> 4;
  const long long grp = (long long)(blockIdx.x / tiles) - 1;
  const bool gated = gate_kind == kGateRows, many = gated && blocks > splits;
  float w = 0.f, u = 0.f;
  if (c < dim) {
    if (grp < 0) {
      for (long long b = place; b < blocks; b += 256) {
        float v[4], q[4], f[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const long long i = b + 64 * k;
          v[k] = gpost && i < blocks ? part[i * 2 * dim + c] : 0.f;
          q[k] = gnext && i < blocks ? part[(i * 2 + 1) * dim + c] : 0.f;
          f[k] = many && gpost && i < blocks ? load1_any(gate, gate_type, (long long)((unsigned)i / (unsigned)splits) * gs + c) : 1.f;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) { w = fmaf(v[k], f[k], w); u += q[k]; }
      }
    } else {
      for (int b = place; b < splits; b += 64) w += part[(grp * splits + b) * 2 * dim + c];
    }
  }
  s0[place][threadIdx.x & 15] = w;
  s1[place][threadIdx.x & 15] = u;
  __syncthreads();
  if (place == 0 && c < dim) {
    for (int o = 1; o < 64; ++o) w += s0[o][threadIdx.x], u += s1[o][threadIdx.x];
    if (grp >= 0) store1_any(ggate, gate_type, grp * dim + c, post ? w * load1_any(post, post_type, c) : w);
    else {
      if (gpost) store1_any(gpost, post_type, c, gated && !many ? w * load1_any(gate, gate_type, c) : w);
      if (gnext) store1_any(gnext, next_type, c, u);
    }
  }
}

constexpr int kMaxDim = 16384;

// lanes of a row: 8 elements a lane, 16 beyond 8192 columns
int lanes_of(int dim) {
  int l = 8;
  while (l < 1024 && l * 8 < dim) l *= 2;
  return l;
}

// Rows of one gate row are cut into as many blocks as are on the card at once (with a block's output a backward lane needs 120 to 150
// registers: three blocks of 256 a CU, one of 512 or 1024; four of 256 without), but no block gets fewer rows than it has places for.  More of
// them cost their sums: 16384 x 4096 bf16, 256 / 512 / 768 blocks of 512: 195 / 202 / 236 us; 76800 x 256, 512 / 768 / 1024 of 256: 63 / 57 / 67.
void split_of(long long rows, int dim, int gate_kind, long long per_gate, bool has_y, long long* groups, int* splits, long long* per_split) {
  const long long per = gate_kind == kGateRows ? per_gate : rows;
  *groups = rows > 0 ? (rows + per - 1) / per : 0;
  const int tpr = lanes_of(dim), tpb = tpr > 256 ? tpr : 256, rpb = tpb / tpr, want = kCUs * (tpb > 256 ? 1 : has_y ? 3 : 4);
  long long s = (want + *groups - 1) / (*groups > 0 ? *groups : 1), most = (per + rpb - 1) / rpb;
  if (s > most) s = most;
  if (s < 1) s = 1;
  *per_split = ((per + s - 1) / s + rpb - 1) / rpb * rpb;
  *splits = per > 0 ? (int)((per + *per_split - 1) / *per_split) : 1;
}

// A launch takes fewer than 2^32 threads
constexpr long long most_blocks(int threads) { return 0xffffffffll / threads; }

template <typename TA, typename TX, int TPR, int NV, bool ODD, bool HASY>
void launch(const BlockArgs& a, bool bwd, long long blocks, hipStream_t st) {
  constexpr int TPB = threads_of<TPR>(), RPB = TPB / TPR;
  if (bwd) {
    const size_t wide = NV > 1 ? 2 * NV * 8 * TPB * sizeof(float) : 0;
    if (wide) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k_block_bwd<TA, TX, TPR, NV, ODD, HASY>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)wide);
    constexpr long long most = most_blocks(TPB);
    for (long long first = 0; first < blocks; first += most) {
      BlockArgs part = a;
      part.first = (unsigned)first;
      hipLaunchKernelGGL((k_block_bwd<TA, TX, TPR, NV, ODD, HASY>), dim3((unsigned)(blocks - first < most ? blocks - first : most)), dim3(TPB), wide, st, part);
    }
  } else {
    long long g = (a.rows + RPB - 1) / RPB, most = (long long)kMaxBlocks * 256 / TPB;
    const dim3 grid((unsigned)(g < most ? g : most)), block(TPB);
    if (!ODD && a.stream) hipLaunchKernelGGL((k_block_fwd<TA, TX, TPR, NV, ODD, HASY, !ODD>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_block_fwd<TA, TX, TPR, NV, ODD, HASY, false>), grid, block, 0, st, a);
  }
}
template <typename TA, typename TX, bool ODD, bool HASY>
void launch_dim(const BlockArgs& a, bool bwd, long long blocks, hipStream_t st) {
  switch (lanes_of(a.dim)) {
    case 8: return launch<TA, TX, 8, 1, ODD, HASY>(a, bwd, blocks, st);
    case 16: return launch<TA, TX, 16, 1, ODD, HASY>(a, bwd, blocks, st);
    case 32: return launch<TA, TX, 32, 1, ODD, HASY>(a, bwd, blocks, st);
    case 64: return launch<TA, TX, 64, 1, ODD, HASY>(a, bwd, blocks, st);
    case 128: return launch<TA, TX, 128, 1, ODD, HASY>(a, bwd, blocks, st);
    case 256: return launch<TA, TX, 256, 1, ODD, HASY>(a, bwd, blocks, st);
    case 512: return launch<TA, TX, 512, 1, ODD, HASY>(a, bwd, blocks, st);
    default: return a.dim <= 8192 ? launch<TA, TX, 1024, 1, ODD, HASY>(a, bwd, blocks, st) : launch<TA, TX, 1024, 2, ODD, HASY>(a, bwd, blocks, st);
  }
}
template <typename TA, typename TX>
void launch_types(const BlockArgs& a, bool odd, bool bwd, long long blocks, hipStream_t st) {
  if (a.y) return odd ? launch_dim<TA, TX, true, true>(a, bwd, blocks, st) : launch_dim<TA, TX, false, true>(a, bwd, blocks, st);
  return odd ? launch_dim<TA, TX, true, false>(a, bwd, blocks, st) : launch_dim<TA, TX, false, false>(a, bwd, blocks, st);
}

bool vec_ok(const void* p, long long stride, int type) {
  return !p || ((reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (stride * type_size(type)) % 16 == 0);
}

int run_block(const BlockArgs& a, int x_type, int act_type, bool bwd, long long blocks, hipStream_t st) {
  const int D = a.dim;
  const bool vec = D % 8 == 0 && vec_ok(a.x, a.xs, x_type) && vec_ok(a.y, a.ys, act_type) && vec_ok(a.post, 0, 0) && vec_ok(a.next, 0, 0) &&
                   (a.gate_kind == kGateToken || vec_ok(a.gate, a.gs, a.gate_type)) && vec_ok(a.dxo, a.dxos, x_type) &&
                   vec_ok(a.dh, a.dhs, act_type) && vec_ok(a.xo, D, x_type) && vec_ok(a.ho, D, act_type) && vec_ok(a.gx, D, x_type) &&
                   vec_ok(a.gy, D, act_type) && (a.gate_kind != kGateFull || vec_ok(a.ggate, D, a.gate_type)) && vec_ok(a.part, D, kF32);
  if (act_type == kF32) launch_types<float, float>(a, !vec, bwd, blocks, st);
  else if (act_type == kBF16 && x_type == kBF16) launch_types<__bf16, __bf16>(a, !vec, bwd, blocks, st);
  else if (act_type == kBF16) launch_types<__bf16, float>(a, !vec, bwd, blocks, st);
  else if (x_type == kF16) launch_types<_Float16, _Float16>(a, !vec, bwd, blocks, st);
  else launch_types<_Float16, float>(a, !vec, bwd, blocks, st);
  return check_launch(bwd ? "block_join_bwd" : "block_join_fwd");
}

}  // namespace
}  // namespace omnihd

using namespace omnihd;

#define OMNIHD_BLOCK_CHECKS                                                                                                             \
  OMNIHD_REQUIRE(rows >= 0 && rows < (1ll << 31) && dim >= 1 && dim <= kMaxDim, "0 <= rows < 2^31, 1 <= dim <= 16384");                  \
  OMNIHD_REQUIRE(type_ok(x_type) && type_ok(act_type) && (x_type == act_type || x_type == kF32), "types: the stream has the block's type or fp32"); \
  OMNIHD_REQUIRE((!post || type_ok(post_type)) && (!next || type_ok(next_type)) && (!gate || type_ok(gate_type)), "weight types");       \
  OMNIHD_REQUIRE(gate_kind >= kGateNone && gate_kind <= kGateFull && (gate != nullptr) == (gate_kind != kGateNone), "gate and its kind"); \
  OMNIHD_REQUIRE(gate_kind != kGateRows || rows_per_gate >= 1, "rows per gate");                                                        \
  OMNIHD_REQUIRE(y || (!post && !gate && next), "without a block's output there is the next norm alone")

extern "C" int omnihd_block_join_fwd(const void* x, long long x_stride, int x_type, const void* y, long long y_stride, int act_type,
                                     const void* post, int post_type, const void* gate, int gate_type, int gate_kind,
                                     long long gate_stride, long long rows_per_gate, const void* next, int next_type,
                                     float residual_scale, float eps, long long rows, int dim, void* x_out, void* h_out, float* stats,
                                     void* stream) {
  OMNIHD_BLOCK_CHECKS;
  if (rows == 0) return OMNIHD_OK;
  OMNIHD_REQUIRE(x && (!y || x_out) && (!next || h_out), "null pointer");
  BlockArgs a{};
  a.x = x; a.y = y; a.post = post; a.gate = gate; a.next = next; a.xo = y ? x_out : nullptr; a.ho = h_out; a.stats = stats;
  a.rows = rows; a.xs = x_stride; a.ys = y_stride; a.gs = gate_stride; a.per_gate = rows_per_gate;
  a.dim = dim; a.post_type = post_type; a.gate_type = gate_type; a.next_type = next_type; a.gate_kind = gate_kind;
  a.r = residual_scale; a.eps = eps;
  // inputs that the Infinity Cache cannot hold are read past it: 16384 x 4096 bf16 108 -> 92 us; below that they may well be there (8192 x 1024:
  // 13.4 us, 16.3 past it)
  a.stream = (size_t)rows * dim * (type_size(x_type) + (y ? type_size(act_type) : 0)) >= kCacheBytes;
  return run_block(a, x_type, act_type, false, 0, (hipStream_t)stream);
}

extern "C" size_t omnihd_block_join_bwd_workspace_bytes(long long rows, int dim, int gate_kind, long long rows_per_gate, int has_y) {
  if (rows <= 0 || dim < 1 || (gate_kind == kGateRows && rows_per_gate < 1)) return 256;
  long long groups, per_split;
  int splits;
  split_of(rows, dim, gate_kind, rows_per_gate, has_y, &groups, &splits, &per_split);
  return (size_t)groups * splits * 2 * dim * sizeof(float);
}

extern "C" int omnihd_block_join_bwd(const void* x, long long x_stride, int x_type, const void* y, long long y_stride, int act_type,
                                     const void* post, int post_type, const void* gate, int gate_type, int gate_kind,
                                     long long gate_stride, long long rows_per_gate, const void* next, int next_type,
                                     float residual_scale, long long rows, int dim, const float* stats, const void* dx_out,
                                     long long dx_out_stride, const void* dh, long long dh_stride, void* gx, void* gy, void* g_post,
                                     void* g_gate, void* g_next, void* workspace, size_t workspace_bytes, void* stream) {
  OMNIHD_BLOCK_CHECKS;
  OMNIHD_REQUIRE((g_post == nullptr || post) && (g_gate == nullptr || gate) && (g_next == nullptr || next), "a gradient without its input");
  OMNIHD_REQUIRE((gy == nullptr || y) && (dh == nullptr || next), "a gradient without its input");
  hipStream_t st = (hipStream_t)stream;
  long long groups = 0, per_split = 1;
  int splits = 1;
  split_of(rows, dim, gate_kind, rows_per_gate, y != nullptr, &groups, &splits, &per_split);
  const long long blocks = groups * splits, tiles = (dim + 15) / 16;
  const bool rows_gate = gate_kind == kGateRows && g_gate;
  const bool cols = g_post || g_next || rows_gate;
  // Several blocks a gate row come with fewer gate rows than blocks on the card at once (split_of): a column block for each of them and 16
  // columns.  One block a gate row: as many column blocks as fill the card, `lanes` columns of a gate row side by side.
  int lanes = 1;
  while (lanes < dim && lanes < 1024) lanes *= 2;
  const long long each = 1024 / lanes, walk = (groups + each - 1) / each;
  const long long col_blocks = tiles + (!rows_gate ? 0 : splits > 1 ? tiles * groups : walk < kMaxBlocks ? walk : kMaxBlocks);
  OMNIHD_REQUIRE(blocks < (1ll << 31) && col_blocks <= most_blocks(1024), "grid");
  if (rows > 0) {
    OMNIHD_REQUIRE(x && stats, "null pointer");
    if (cols) {
      OMNIHD_REQUIRE(workspace, "null pointer");
      const size_t need = (size_t)blocks * 2 * dim * sizeof(float);
      if (workspace_bytes < need) { set_error("block_join_bwd: workspace %zu < required %zu", workspace_bytes, need); return OMNIHD_ERR_WORKSPACE; }
    }
    BlockArgs a{};
    a.x = x; a.y = y; a.post = post; a.gate = gate; a.next = next; a.dxo = dx_out; a.dh = dh; a.gx = gx; a.gy = gy;
    a.ggate = gate_kind == kGateRows ? nullptr : g_gate; a.stats = const_cast<float*>(stats);
    a.part = cols ? static_cast<float*>(workspace) : nullptr;
    a.rows = rows; a.xs = x_stride; a.ys = y_stride; a.gs = gate_stride; a.dxos = dx_out_stride; a.dhs = dh_stride;
    a.per_gate = gate_kind == kGateRows ? rows_per_gate : rows; a.per_split = per_split; a.splits = splits;
    a.dim = dim; a.post_type = post_type; a.gate_type = gate_type; a.next_type = next_type; a.gate_kind = gate_kind; a.r = residual_scale;
    const int rc = run_block(a, x_type, act_type, true, blocks, st);
    if (rc != OMNIHD_OK) return rc;
  }
  if (cols)                              // with no rows the weights' gradients are zero: no block, no gate row
    hipLaunchKernelGGL(k_block_cols, dim3((unsigned)col_blocks), dim3(1024), 0, st,
                       static_cast<const float*>(workspace), blocks, splits, dim, lanes, post, post_type, gate, gate_type, gate_stride,
                       gate_kind, g_post, g_gate, g_next, next_type);
  return check_launch("block_join_bwd");
}
