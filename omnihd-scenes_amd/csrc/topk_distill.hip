// Distillation from a teacher's top logits: the loss and its gradient in one pass over the student's logits.
//
//   p = softmax over the filled slots of t_k / T          (K slots a row, id < 0: an empty slot)
//   q = softmax(z / T) over the V entries of the row
//   row  = T^2 * sum_k p_k (ln p_k - ln q[id_k])          loss = factor * sum_rows w * row      (or factor * w * row, row by row)
//   dz_v = factor * w * T * (q_v - sum_{k: id_k = v} p_k) (* up: the gradient that arrives at the loss)
//
// A row with no teacher mass (no filled slot, or all of them -inf) or of weight 0 adds exactly 0 and gets a zero gradient, whatever
// its logits hold; an id >= V makes its row NaN (nothing outside the row is read or written).
//
// Bound by HBM at large V: V read, V written; about 15 operations an element (two exponentials among them) take half as long.  So a row
// is read once into registers (16 bytes a lane and step), its maximum and its sum of exponentials go over the lanes that share it, and the
// gradient is written from the registers.  Rows beyond 128 K (16-bit) entries are read twice, the second time out of the caches.  All in base 2:
// exp2(z * c - m * c), c = log2(e) / T, one fused multiply-add with a single rounding of the difference; sums in fp32.  Rows whose maximum lies far
// from 0 are moved there first (Base).
// The few entries that the teacher names are written again behind the row's own stores, from their own p sums (slots with the same id are
// summed by the first of them, so an id may stand in a row more than once).
// Rows of up to 16 entries (the classes of a detection or occupancy head) take a lane each.
// Measured, loss and gradient (copy rate 5.1 TB/s): 4096 x 131072 bf16 453 us (4.7 TB/s), 4096 x 32000 111 us (4.8), 4096 x 50001 185 us
// (4.4), 60000 x 1000 70 us (3.6: the teacher's part of each row), 614400 x 12 fp32 30 us (2.9: 1000 instructions a wave, half of it arithmetic).
#include "token_vec.h"

namespace omnihd {
namespace {
using namespace tok;

constexpr int kLaneVocab = 16, kMaxTop = 256, kMaxVocab = 1 << 30;      // (places in a row are counted in int)
constexpr float kLn2 = 0.69314718055994531f;

struct DistillArgs {
  const void *z, *t, *ids;
  const float *w, *up, *avg;             // row weights, gradient of the loss (up_step 0: one for all rows), divisor on the device: each may be NULL
  void* g;                               // gradient of z (NULL: not asked for)
  float *rows_out, *sums;                // per-row losses, or one sum a block; both may be NULL
  long long rows, zs, gs, ts, is;        // rows and row strides in elements
  int vocab, top, t_type, wide_ids, up_step, skip_if_one;
  float temperature, factor;
};

__device__ __forceinline__ long long id_at(const DistillArgs& a, long long at) {
  return a.wide_ids ? static_cast<const long long*>(a.ids)[at] : (long long)static_cast<const int*>(a.ids)[at];
}
__device__ __forceinline__ float factor_of(const DistillArgs& a) { return a.avg ? a.factor / *a.avg : a.factor; }

// 16 bytes of logits, kept as they are
template <typename T> struct Pack { static constexpr int n = 16 / (int)sizeof(T); typedef T V __attribute__((ext_vector_type(16 / sizeof(T)))); };
// `first` of them (if positive) and those from `left` on are not the row's: they read as -inf, and are not written
template <bool ODD, typename T>
__device__ __forceinline__ typename Pack<T>::V load_pack(const T* __restrict__ p, int left, int first = 0) {
  typedef typename Pack<T>::V V;
  typedef V W __attribute__((aligned(ODD ? sizeof(T) : 16)));
  if (!ODD || (left >= Pack<T>::n && first <= 0)) return *reinterpret_cast<const W*>(p);
  V v;
#pragma unroll
  for (int k = 0; k < Pack<T>::n; ++k) v[k] = k < left && k >= first ? p[k] : (T)-__builtin_inff();
  return v;
}
// Past the caches: 1021 x 50021 fp16 44.4 us, 46.2 through them; 2048 x 32000 48 and 51; 614400 x 12 31 and 32.  An operation that reads the gradient
// at once changes that where the caches would hold it: both together 110 and 95 us at 60000 x 1000, 101 and 95 at 2048 x 32000; 82 each at
// 1021 x 50021, 42 each at 614400 x 12, 770 each at 4096 x 131072.
template <bool ODD, typename T>
__device__ __forceinline__ void store_pack(T* __restrict__ p, int left, const typename Pack<T>::V& v, int first = 0) {
  typedef typename Pack<T>::V V;
  typedef V W __attribute__((aligned(ODD ? sizeof(T) : 16)));
  if (!ODD || (left >= Pack<T>::n && first <= 0)) { __builtin_nontemporal_store(v, reinterpret_cast<W*>(p)); return; }
#pragma unroll
  for (int k = 0; k < Pack<T>::n; ++k)
    if (k < left && k >= first) p[k] = v[k];
}

// NaN where either is NaN (fmaxf drops it: a NaN logit has to reach the loss)
struct MaxNan { __device__ __forceinline__ float operator()(float a, float b) const { return (a != a || b != b) ? __builtin_nanf("") : fmaxf(a, b); } };

// a product as it was rounded: the compiler may not take it into a fused multiply-add
__device__ __forceinline__ float rounded(float v) { asm volatile("" : "+v"(v)); return v; }

// What a row's entries are shifted by: exp2(fma(v - off, c, -mc)).  The product m * c is rounded, which shifts all of them alike by half a step of it
// and does no harm up to 2^24; beyond, the shift would leave exp2's range and masks of the type's lowest value overflow in it, so m itself is
// taken off first (what is still in exp2's range then lies within a factor of two of m: that difference is exact, in the entries' own type too).
// `off` is 0 elsewhere, and the entries are moved in a branch of their own: a subtraction for every one of them costs 17 % at 614400 x 12.
struct Base { float off, mc; };
constexpr float kFar = 16777216.f;
__device__ __forceinline__ Base base_of(float m, float c) {
  const float off = fabsf(m * c) < kFar ? 0.f : m;
  return {off, rounded((m - off) * c)};            // (NaN for a maximum that is infinite, or of a row with nothing but -inf)
}
__device__ __forceinline__ float below(float v, const Base& b, float c) { return fmaf(v - b.off, c, -b.mc); }
// how far one shift lies below another
__device__ __forceinline__ float between(const Base& a, const Base& b, float c) { return fmaf(a.off - b.off, c, a.mc - b.mc); }
template <typename T> __device__ __forceinline__ void move(typename Pack<T>::V& v, float off) {
#pragma unroll
  for (int k = 0; k < Pack<T>::n; ++k) v[k] = (T)((float)v[k] - off);
}

// Which of this lane's ids (bit i: slot t + i * SL) stand in the row once.  Every slot is compared with up to four of the lane's own at a
// time: two instructions a pair (34830 rows of 172 slots: 508 us with a search for each slot).
template <int SL, int N>
__device__ __forceinline__ unsigned alone_of(const int* sid, int K, int at) {
  int mine[N], seen[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    mine[j] = at + j * SL < K ? sid[at + j * SL] : -2;
    seen[j] = 0;
  }
#pragma unroll 4
  for (int o = 0; o < K; ++o) {
    const int other = sid[o];
#pragma unroll
    for (int j = 0; j < N; ++j) seen[j] += mine[j] == other;
  }
  unsigned once = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) once |= (seen[j] == 1 ? 1u : 0u) << j;
  return once;
}
template <int SL>
__device__ __forceinline__ unsigned alone_in_row(const int* sid, int K, int t) {
  unsigned once = 0;
  for (int b = 0; b < K; b += 4 * SL) {
    const int left = (K - b + SL - 1) / SL;        // (kMaxTop / 8 lanes: 32 slots a lane at most)
    const unsigned some = left == 1 ? alone_of<SL, 1>(sid, K, b + t) : left == 2 ? alone_of<SL, 2>(sid, K, b + t)
                        : left == 3 ? alone_of<SL, 3>(sid, K, b + t) : alone_of<SL, 4>(sid, K, b + t);
    once |= some << (b / SL);
  }
  return once;
}

// TPR lanes a row; NV steps of 16 bytes a lane in registers, or (NV = 0) the row is read twice.
template <typename T, int TPR, int NV, bool ODD>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256, TPR > 256 ? 4 : 1) void k_distill_rows(DistillArgs a) {
  constexpr int TPB = TPR > 256 ? TPR : 256, RPB = TPB / TPR, VE = Pack<T>::n, KEEP = NV ? NV : 1;
  constexpr int SL = TPR < 64 ? TPR : 64, FL = TPR > 64 ? kMaxTop : SL;      // lanes that share sums of slots, lanes with slots
  static_assert(TPR <= 64 || TPR >= kMaxTop, "a thread a slot");
  typedef typename Pack<T>::V V;
  __shared__ float red[32], row_sum[RPB], wave_max[4], wave_sum[4], wave_part[4];
  __shared__ bool wave_bad[4];
  extern __shared__ float slots[];       // [RPB][3][K]: ids, teacher's and student's values
  if (a.skip_if_one && *a.up == 1.f) return;
  int turn = 0;
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, K = a.top;
  int* sid = reinterpret_cast<int*>(slots) + sub * 3 * K;
  float *st = slots + sub * 3 * K + K, *sz = st + K;
  const float c = 1.44269504088896341f / a.temperature, base = factor_of(a);
  float total = 0.f;
  for (long long first = (long long)blockIdx.x * RPB; first < a.rows; first += (long long)gridDim.x * RPB) {
    const long long row = first + sub;
    const bool act = row < a.rows;
    const T* z = static_cast<const T*>(a.z) + (act ? row : 0) * a.zs;
    // Rows that start anywhere: packs are counted from the 16-byte border before the row (4096 x 50001 bf16: 225 us from its first entry)
    const int skip = ODD ? (int)(reinterpret_cast<uintptr_t>(z) / sizeof(T) % VE) : 0, end = a.vocab + skip;
    const T* zb = z - skip;
    const float w = !act ? 0.f : a.w ? a.w[row] : 1.f;
    // the row is asked for first: the teacher's slots are worked on while it is on its way
    V keep[KEEP];
    if constexpr (NV > 0) {
      if (w != 0.f) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int at = (j * TPR + t) * VE, left = end - at;
          if (left > 0) keep[j] = load_pack<ODD>(zb + at, left, skip - at);
        }
      }
    }
    // The teacher.  Where a row has a block, a thread a slot, the waves' maxima and sums exchanged behind the barriers of the row's own; else
    // the row's lanes walk over the slots.
    float coef = 0.f, mt = -__builtin_inff(), ls = 0.f, value = -__builtin_inff();
    bool bad = false;
    if (t < FL && w != 0.f)
      for (int k = t; k < K; k += FL) {
        const long long id = id_at(a, row * a.is + k);
        value = id < 0 ? -__builtin_inff() : load1_any(a.t, a.t_type, row * a.ts + k);
        bad |= id >= a.vocab;
        const bool fits = id >= 0 && id < a.vocab;
        sid[k] = fits ? (int)id : -1;
        st[k] = value;
        sz[k] = fits ? (float)z[id] : 0.f;
        mt = MaxNan()(mt, value);
      }
    mt = lanes<SL>(mt, MaxNan());
    bad = (bool)lanes<SL>(bad ? 1.f : 0.f, Max());
    if constexpr (TPR > 64) {
      if (t < FL && (t & 63) == 0) { wave_max[t >> 6] = mt; wave_bad[t >> 6] = bad; }
    } else {
      const bool some = w != 0.f && mt != -__builtin_inff();
      const Base tb = base_of(mt, c);
      float e = 0.f;
      if (some)
        for (int k = t; k < K; k += SL) {
          const float d = below(st[k], tb, c);
          st[k] = d;                               // log2 of p, short of the sum's
          e += __builtin_amdgcn_exp2f(d);
        }
      e = lanes<SL>(e, Add());
      ls = some ? __builtin_amdgcn_logf(e) : 0.f;        // base 2
      coef = bad ? __builtin_nanf("") : some ? w : 0.f;
    }
    // the row's maximum and sum
    float m = -__builtin_inff(), s = 0.f;
    Base at_base{0.f, 0.f};                        // what this lane's terms are shifted by so far (rows read twice)
    if (w != 0.f) {
      if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if ((j * TPR + t) * VE < end)
#pragma unroll
            for (int k = 0; k < VE; ++k) m = fmaxf(m, (float)keep[j][k]);
      } else {
        for (int at = t * VE; at < end; at += 4 * TPR * VE) {        // four loads in flight a lane
          V v[4];
          float big = -__builtin_inff();
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (at + j * TPR * VE < end) v[j] = load_pack<ODD>(zb + at + j * TPR * VE, end - at - j * TPR * VE, skip - at - j * TPR * VE);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (at + j * TPR * VE < end)
#pragma unroll
              for (int k = 0; k < VE; ++k) big = fmaxf(big, (float)v[j][k]);
          if (big > m) {
            const Base to = base_of(big, c);
            s = m == -__builtin_inff() ? s : s * __builtin_amdgcn_exp2f(between(at_base, to, c));
            m = big;
            at_base = to;
          }
          if (at_base.off != 0.f)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (at + j * TPR * VE < end) move<T>(v[j], at_base.off);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (at + j * TPR * VE < end)
#pragma unroll
              for (int k = 0; k < VE; ++k) s += __builtin_amdgcn_exp2f(fmaf((float)v[j][k], c, -at_base.mc));
        }
      }
    }
    const float own = m;
    m = group<TPR>(m, Max(), red, turn);
    const Base zbase = base_of(m, c);
    const float mc = zbase.mc;
    if constexpr (NV > 0) {
      if (w != 0.f && zbase.off != 0.f)
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if ((j * TPR + t) * VE < end) move<T>(keep[j], zbase.off);
    }
    bool some = false;
    if constexpr (TPR > 64) {
#pragma unroll
      for (int i = 0; i < FL / 64; ++i) {
        mt = i ? MaxNan()(mt, wave_max[i]) : wave_max[0];
        bad = i ? bad || wave_bad[i] : wave_bad[0];
      }
      some = w != 0.f && mt != -__builtin_inff();
      float e = 0.f;
      if (some && t < FL && t < K) {
        const float d = below(value, base_of(mt, c), c);
        st[t] = d;
        e = __builtin_amdgcn_exp2f(d);
      }
      if (t < FL) {
        e = lanes<64>(e, Add());
        if ((t & 63) == 0) wave_sum[t >> 6] = e;
      }
    }
    if (w != 0.f) {
      if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if ((j * TPR + t) * VE < end)
#pragma unroll
            for (int k = 0; k < VE; ++k) s += __builtin_amdgcn_exp2f(fmaf((float)keep[j][k], c, -mc));
      } else if (own == -__builtin_inff()) {
        if (m == own && t * VE < end) s = __builtin_nanf("");   // nothing but -inf in the row
      } else {
        s *= __builtin_amdgcn_exp2f(between(at_base, zbase, c));
      }
    }
    s = group<TPR>(s, Add(), red, turn);
    if constexpr (TPR > 64) {
      float e = wave_sum[0];
#pragma unroll
      for (int i = 1; i < FL / 64; ++i) e += wave_sum[i];
      ls = some ? __builtin_amdgcn_logf(e) : 0.f;
      coef = bad ? __builtin_nanf("") : some ? w : 0.f;
    }
    const float scale = base * coef * a.temperature;
    float up = 1.f;
    if (a.up) up = act ? a.up[a.up_step ? row : 0] : 0.f;
    const float k1 = coef == 0.f ? 0.f : scale * up, kq = k1 / s;
    if (a.g && act) {
      T* g = static_cast<T*>(a.g) + row * a.gs - skip;
      if (k1 == 0.f) {                             // nothing to learn from this row
        V zero;
#pragma unroll
        for (int k = 0; k < VE; ++k) zero[k] = (T)0.f;
        for (int at = t * VE; at < end; at += TPR * VE) store_pack<ODD>(g + at, end - at, zero, skip - at);
      } else if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int at = (j * TPR + t) * VE, left = end - at;
          if (left <= 0) continue;
          V o;
#pragma unroll
          for (int k = 0; k < VE; ++k) o[k] = (T)(__builtin_amdgcn_exp2f(fmaf((float)keep[j][k], c, -mc)) * kq);
          store_pack<ODD>(g + at, left, o, skip - at);
        }
      } else {
        for (int at = t * VE; at < end; at += 4 * TPR * VE) {
          V v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (at + j * TPR * VE < end) v[j] = load_pack<ODD>(zb + at + j * TPR * VE, end - at - j * TPR * VE, skip - at - j * TPR * VE);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int left = end - at - j * TPR * VE;
            if (left <= 0) continue;
            if (zbase.off != 0.f) move<T>(v[j], zbase.off);
            V o;
#pragma unroll
            for (int k = 0; k < VE; ++k) o[k] = (T)(__builtin_amdgcn_exp2f(fmaf((float)v[j][k], c, -mc)) * kq);
            store_pack<ODD>(g + at + j * TPR * VE, left, o, skip - at - j * TPR * VE);
          }
        }
      }
    }
    const bool learns = a.g && act && k1 != 0.f;
    unsigned alone = 0;
    if (t < FL && learns) alone = alone_in_row<FL>(sid, K, t);
    // the teacher's entries, behind the stores of the whole row
    if (TPR > 64) __syncthreads();
    else {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    float part = 0.f;
    if (t < FL && coef != 0.f && act) {
      const float lq = __builtin_amdgcn_logf(s);
      for (int k = t; k < K; k += FL) {
        const int id = sid[k];
        if (id < 0) continue;
        const float lp = st[k] - ls, p = __builtin_amdgcn_exp2f(lp), zk = below(sz[k], zbase, c);
        if (!(p == 0.f)) part = fmaf(p, lp - (zk - lq), part);
        if (!learns) continue;
        float sum = 0.f;                           // p of every slot with this id; only the first of them writes
        bool leads = true;
        if (alone >> ((k - t) / FL) & 1) sum = p;
        else
          for (int b = 0; b < K; b += 8) {         // (eight reads in flight)
            unsigned same = 0;
#pragma unroll
            for (int o = 0; o < 8; ++o) same |= (b + o < K && sid[b + o < K ? b + o : 0] == id ? 1u : 0u) << o;
            for (; same; same &= same - 1) {
              const int o = b + __builtin_ctz(same);
              leads &= o >= k;
              sum += __builtin_amdgcn_exp2f(st[o] - ls);
            }
          }
        if (leads) static_cast<T*>(a.g)[row * a.gs + id] = (T)fmaf(__builtin_amdgcn_exp2f(zk), kq, -k1 * sum);
      }
    }
    part = lanes<SL>(part, Add());
    if (TPR > 64 && t < FL && (t & 63) == 0) wave_part[t >> 6] = part;
    if (TPR > 64) __syncthreads();                 // (the slots are written again)
    else {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    if (t == 0 && act) {
      if constexpr (TPR > 64) part = (wave_part[0] + wave_part[1]) + (wave_part[2] + wave_part[3]);
      const float loss = coef == 0.f ? 0.f : base * coef * a.temperature * a.temperature * kLn2 * part;
      if (a.rows_out) a.rows_out[row] = loss;
      total += loss;
    }
  }
  if (a.sums) {
    if (t == 0) row_sum[sub] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int o = 1; o < RPB; ++o) total += row_sum[o];
      a.sums[blockIdx.x] = total;
    }
  }
}

// A lane a row, up to VM entries in registers; the first KR slots too.  Rows that lie side by side go through LDS, 64 of a wave at a time
// in whole lines (a lane's own 16-byte pieces of a row of 48 bytes touch every line three times, and store parts of lines).
template <typename T, int VM>
__global__ __launch_bounds__(256) void k_distill_lanes(DistillArgs a) {
  constexpr int VE = Pack<T>::n, NP = VM / VE, KR = 8;
  typedef typename Pack<T>::V V;
  constexpr int PITCH = VM + 1;
  __shared__ float wave_sum[4], staged[4][64 * PITCH];
  float* tile = staged[threadIdx.x >> 6];
  const int lane = threadIdx.x & 63;
  const unsigned by_vocab = ((1u << 20) + a.vocab - 1) / a.vocab;          // e / vocab = e * this >> 20 for e < 64 * 16
  const bool in_dense = a.zs == a.vocab, out_dense = a.g && a.gs == a.vocab;
  if (a.skip_if_one && *a.up == 1.f) return;
  const float c = 1.44269504088896341f / a.temperature, base = factor_of(a);
  float total = 0.f;
  for (long long first = (long long)blockIdx.x * 256 + (threadIdx.x & ~63); first < a.rows; first += (long long)gridDim.x * 256) {
    const bool act = first + lane < a.rows;
    const long long row = act ? first + lane : a.rows - 1;        // (a lane beyond the last row repeats it and writes nothing)
    const float w = !act ? 0.f : a.w ? a.w[row] : 1.f;
    const T* z = static_cast<const T*>(a.z) + row * a.zs;
    const int held = (int)(a.rows - first < 64 ? a.rows - first : 64) * a.vocab;      // elements of this wave's rows
    const int K = a.top, V_ = a.vocab;
    long long raw_id[KR];                          // the teacher's slots are asked for before the rows
    float raw_t[KR];
#pragma unroll
    for (int k = 0; k < KR; ++k) {
      raw_id[k] = k < K ? id_at(a, row * a.is + k) : -1;
      raw_t[k] = k < K ? load1_any(a.t, a.t_type, row * a.ts + k) : 0.f;
    }
    if (in_dense) {
      for (int e = lane * VE; e < held; e += 64 * VE) {
        const V v = load_pack<true>(static_cast<const T*>(a.z) + first * a.vocab + e, held - e);
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          const unsigned r = (unsigned)(e + k) * by_vocab >> 20;
          if (e + k < held) tile[r * PITCH + (e + k) - r * a.vocab] = (float)v[k];
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    float x[VM], m = -__builtin_inff(), s = 0.f;
    int id[KR];
    float tv[KR], mt = -__builtin_inff();
    bool bad = false;
    if (!in_dense) {
#pragma unroll
      for (int j = 0; j < NP; ++j)
        if (j * VE < V_) {
          const V v = load_pack<true>(z + j * VE, V_ - j * VE);
#pragma unroll
          for (int k = 0; k < VE; ++k) tile[lane * PITCH + j * VE + k] = (float)v[k];
        }
    }
    if (!act && in_dense)                          // (the last row's copy: its entries in this lane's own place)
      for (int k = 0; k < V_; ++k) tile[lane * PITCH + k] = 0.f;
#pragma unroll
    for (int k = 0; k < VM; ++k) x[k] = k < V_ ? tile[lane * PITCH + k] : -__builtin_inff();
    auto take = [&](long long full, float value, int& i, float& v) {
      v = full < 0 ? -__builtin_inff() : value;
      bad |= full >= V_;
      i = full < 0 || full >= V_ ? -1 : (int)full;
    };
    auto slot = [&](int k, int& i, float& v) { take(id_at(a, row * a.is + k), load1_any(a.t, a.t_type, row * a.ts + k), i, v); };
#pragma unroll
    for (int k = 0; k < KR; ++k) take(raw_id[k], raw_t[k], id[k], tv[k]);
#pragma unroll
    for (int k = 0; k < KR; ++k) mt = MaxNan()(mt, tv[k]);
    for (int k = KR; k < K; ++k) {
      int i; float v;
      slot(k, i, v);
      mt = MaxNan()(mt, v);
    }
#pragma unroll
    for (int k = 0; k < VM; ++k) m = fmaxf(m, x[k]);
    float* own = tile + lane * PITCH;              // this lane's row: logits here, its gradient below
    const Base xb = base_of(m, c);
    const float mc = xb.mc;
    if (xb.off != 0.f) {
#pragma unroll
      for (int k = 0; k < VM; ++k)
        if (k < V_) own[k] = x[k] -= xb.off;
    }
#pragma unroll
    for (int k = 0; k < VM; ++k) {
      if (k < V_) { x[k] = fmaf(x[k], c, -mc); s += __builtin_amdgcn_exp2f(x[k]); }
    }
    const bool some = mt != -__builtin_inff();
    const Base tb = base_of(mt, c);
    if (tb.off != 0.f) {
#pragma unroll
      for (int k = 0; k < KR; ++k) tv[k] -= tb.off;
    }
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < KR; ++k) if (k < K) sum += __builtin_amdgcn_exp2f(fmaf(tv[k], c, -tb.mc));
    for (int k = KR; k < K; ++k) {
      int i; float v;
      slot(k, i, v);
      sum += __builtin_amdgcn_exp2f(below(v, tb, c));
    }
    float coef = w != 0.f && some ? w : 0.f;
    if (bad && w != 0.f) coef = __builtin_nanf("");
    const float ls = __builtin_amdgcn_logf(sum), lq = __builtin_amdgcn_logf(s);
    float up = 1.f;
    if (a.up) up = a.up[a.up_step ? row : 0];
    const float k1 = coef == 0.f ? 0.f : base * coef * a.temperature * up, kq = k1 / s;
    float part = 0.f;
    auto use = [&](int i, float d) {               // (d: below(value, tb, c))
      if (i < 0) return;
      const float lp = d - ls, p = __builtin_amdgcn_exp2f(lp), zk = fmaf(own[i], c, -mc);
      if (!(p == 0.f)) part = fmaf(p, lp - (zk - lq), part);
    };
    auto learn = [&](int i, float d) {
      if (i >= 0) own[i] -= k1 * __builtin_amdgcn_exp2f(d - ls);
    };
    if (coef != 0.f) {
#pragma unroll
      for (int k = 0; k < KR; ++k) if (k < K) use(id[k], fmaf(tv[k], c, -tb.mc));
      for (int k = KR; k < K; ++k) {
        int i; float v;
        slot(k, i, v);
        use(i, below(v, tb, c));
      }
    }
    if (a.g) {
      T* g = static_cast<T*>(a.g) + row * a.gs;
#pragma unroll
      for (int k = 0; k < VM; ++k)
        if (k < V_) own[k] = k1 == 0.f ? 0.f : __builtin_amdgcn_exp2f(x[k]) * kq;
      if (k1 != 0.f) {
#pragma unroll
        for (int k = 0; k < KR; ++k) if (k < K) learn(id[k], fmaf(tv[k], c, -tb.mc));
        for (int k = KR; k < K; ++k) {
          int i; float v;
          slot(k, i, v);
          learn(i, below(v, tb, c));
        }
      }
      if (!out_dense && act) {
        for (int k = 0; k < V_; ++k) g[k] = (T)own[k];
      }
      if (out_dense) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        for (int e = lane * VE; e < held; e += 64 * VE) {
          V o;
#pragma unroll
          for (int k = 0; k < VE; ++k) {
            const unsigned r = (unsigned)(e + k) * by_vocab >> 20;
            o[k] = (T)(e + k < held ? tile[r * PITCH + (e + k) - r * a.vocab] : 0.f);
          }
          store_pack<true>(static_cast<T*>(a.g) + first * a.vocab + e, held - e, o);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
    const float loss = coef == 0.f ? 0.f : base * coef * a.temperature * a.temperature * kLn2 * part;
    if (a.rows_out && act) a.rows_out[row] = loss;
    total += loss;
  }
  if (a.sums) {
    total = lanes<64>(total, Add());
    if ((threadIdx.x & 63) == 0) wave_sum[threadIdx.x >> 6] = total;
    __syncthreads();
    if (threadIdx.x == 0) a.sums[blockIdx.x] = (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);
  }
}

__global__ __launch_bounds__(1024) void k_distill_total(const float* __restrict__ sums, int n, float* __restrict__ loss) {
  __shared__ double wave_sum[16];
  double s = 0;
  for (int i = threadIdx.x; i < n; i += 1024) s += sums[i];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) wave_sum[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) s += wave_sum[i];
    *loss = (float)s;
  }
}

struct Geometry { int tpr, nv; };       // nv 0: the row is read twice
// A lane holds up to eight packs, sixteen in the longest rows.  Short rows share a wave, so that the teacher's part, much the same for any
// vocabulary, is paid once for several (60000 x 1000 bf16: 96 us with a wave a row, 70 so).
template <typename T> Geometry geometry(int vocab, int top, bool odd) {
  const long long packs = odd ? (vocab + 2ll * (Pack<T>::n - 1)) / Pack<T>::n : vocab / Pack<T>::n;       // (odd: at any start of the row)
  int tpr = 8;
  while (tpr < 64 && (packs > 8 * tpr || (256 / tpr) * 12 * top > 32768)) tpr *= 2;
  if (tpr == 8 && packs <= 8 * 2) return {8, 2};
  if (packs <= 8 * tpr) return {tpr, 8};
  if (packs <= 256 * 4) return {256, 4};
  if (packs <= 256 * 8) return {256, 8};
  if (packs <= 512 * 8) return {512, 8};
  if (packs <= 512 * 16) return {512, 16};
  if (packs <= 1024 * 16) return {1024, 16};
  return {1024, 0};
}
// (600000 rows of 12 entries, 4 slots: 31 us with a lane a row, 53 with eight; 300000 of 20: 33.4 and 29.5, with 12 slots 56 and 40)
bool by_lanes(int vocab) { return vocab <= kLaneVocab; }
template <typename T> int blocks_of(long long rows, int vocab, int top, bool odd) {
  if (by_lanes(vocab)) return (int)(rows <= 16384 * 256 ? (rows + 255) / 256 : 16384);
  const int tpr = geometry<T>(vocab, top, odd).tpr, tpb = tpr > 256 ? tpr : 256;
  const long long g = (rows + tpb / tpr - 1) / (tpb / tpr), most = (long long)kMaxBlocks * 256 / tpb;
  return (int)(g < most ? g : most);
}
template <typename T> int most_blocks(long long rows, int vocab, int top) {
  if (rows <= 0) return 1;
  const int odd = blocks_of<T>(rows, vocab, top, true);
  if (vocab % Pack<T>::n) return odd;
  const int even = blocks_of<T>(rows, vocab, top, false);
  return odd > even ? odd : even;
}

template <typename T, bool ODD>
int launch_rows(const DistillArgs& a, hipStream_t st) {
  const Geometry g = geometry<T>(a.vocab, a.top, ODD);
  const int blocks = blocks_of<T>(a.rows, a.vocab, a.top, ODD);
  const int tpb = g.tpr > 256 ? g.tpr : 256;
  const size_t lds = (size_t)(tpb / g.tpr) * 3 * a.top * sizeof(float);
#define OMNIHD_DISTILL(R, N) hipLaunchKernelGGL((k_distill_rows<T, R, N, ODD>), dim3(blocks), dim3(tpb), lds, st, a)
  if (g.tpr == 8 && g.nv == 2) OMNIHD_DISTILL(8, 2);
  else if (g.tpr == 8) OMNIHD_DISTILL(8, 8);
  else if (g.tpr == 16) OMNIHD_DISTILL(16, 8);
  else if (g.tpr == 32) OMNIHD_DISTILL(32, 8);
  else if (g.tpr == 64) OMNIHD_DISTILL(64, 8);
  else if (g.tpr == 256 && g.nv == 4) OMNIHD_DISTILL(256, 4);
  else if (g.tpr == 256) OMNIHD_DISTILL(256, 8);
  else if (g.nv == 8) OMNIHD_DISTILL(512, 8);
  else if (g.tpr == 512) OMNIHD_DISTILL(512, 16);
  else if (g.nv == 16) OMNIHD_DISTILL(1024, 16);
  else OMNIHD_DISTILL(1024, 0);
#undef OMNIHD_DISTILL
  return blocks;
}
// the number of blocks, each of which leaves a sum
template <typename T>
int launch_distill(const DistillArgs& a, hipStream_t st) {
  if (by_lanes(a.vocab)) {
    const int blocks = blocks_of<T>(a.rows, a.vocab, a.top, true);
    hipLaunchKernelGGL((k_distill_lanes<T, kLaneVocab>), dim3(blocks), dim3(256), 0, st, a);
    return blocks;
  }
  auto fits = [&](const void* p, long long stride) { return !p || ((reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % Pack<T>::n == 0); };
  if (a.vocab % Pack<T>::n == 0 && fits(a.z, a.zs) && fits(a.g, a.gs)) return launch_rows<T, false>(a, st);
  return launch_rows<T, true>(a, st);
}

}  // namespace
}  // namespace omnihd

using namespace omnihd;

extern "C" size_t omnihd_topk_distill_workspace_bytes(long long rows, int vocab, int top, int z_type) {
  if (rows < 0 || vocab < 1 || vocab > kMaxVocab || top < 1 || top > kMaxTop || !type_ok(z_type)) return 0;
  const int blocks = z_type == kF32 ? most_blocks<float>(rows, vocab, top) : most_blocks<__bf16>(rows, vocab, top);
  return align_up((size_t)blocks * sizeof(float), 256);
}

extern "C" int omnihd_topk_distill(const void* z, int z_type, long long z_stride, const void* t, int t_type, long long t_stride,
                                   const void* ids, int wide_ids, long long ids_stride, const float* row_weight, long long rows, int vocab,
                                   int top, float temperature, float factor, const float* avg_factor, const float* up, int up_per_row,
                                   int skip_if_one, void* grad, long long grad_stride, float* row_loss, float* loss, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  OMNIHD_REQUIRE(rows >= 0 && rows < (1ll << 31) && vocab >= 1 && vocab <= kMaxVocab && top >= 1 && top <= kMaxTop,
                 "0 <= rows < 2^31, 1 <= vocab <= 2^30, 1 <= top <= 256");
  OMNIHD_REQUIRE(type_ok(z_type) && type_ok(t_type), "types");
  OMNIHD_REQUIRE(temperature > 0.f, "temperature > 0");
  OMNIHD_REQUIRE(!skip_if_one || (up && !up_per_row && !loss && !row_loss), "skip_if_one goes with one gradient for all rows");
  hipStream_t st = (hipStream_t)stream;
  int blocks = 0;
  float* sums = nullptr;
  if (loss) {
    const size_t need = omnihd_topk_distill_workspace_bytes(rows, vocab, top, z_type);
    OMNIHD_REQUIRE(workspace, "null pointer");
    if (workspace_bytes < need) { set_error("topk_distill: workspace %zu < required %zu", workspace_bytes, need); return OMNIHD_ERR_WORKSPACE; }
    sums = static_cast<float*>(workspace);
  }
  if (rows > 0) {
    OMNIHD_REQUIRE(z && t && ids && z_stride >= vocab && t_stride >= top && ids_stride >= top && (!grad || grad_stride >= vocab), "null pointer or short rows");
    DistillArgs a{};
    a.z = z; a.t = t; a.ids = ids; a.w = row_weight; a.up = up; a.avg = avg_factor; a.g = grad; a.rows_out = row_loss; a.sums = sums;
    a.rows = rows; a.zs = z_stride; a.gs = grad_stride; a.ts = t_stride; a.is = ids_stride;
    a.vocab = vocab; a.top = top; a.t_type = t_type; a.wide_ids = wide_ids; a.up_step = up_per_row; a.skip_if_one = skip_if_one;
    a.temperature = temperature; a.factor = factor;
    blocks = z_type == kF32 ? launch_distill<float>(a, st) : z_type == kBF16 ? launch_distill<__bf16>(a, st) : launch_distill<_Float16>(a, st);
  }
  if (loss) hipLaunchKernelGGL(k_distill_total, dim3(1), dim3(1024), 0, st, sums, blocks, loss);
  return check_launch("topk_distill");
}
