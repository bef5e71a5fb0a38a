// Rows of token operators: eight elements at a time as fp32 values, for fp32, bf16 and IEEE-half rows, and sums over the lanes that
// share a row.  A row whose width or address fits no 16-byte vector is read with the same 16-byte instructions at its element's
// alignment (gfx950 reads and writes global memory at any alignment) and its last, partial vector element by element: nothing outside
// the row is touched.
#pragma once
#include "common.h"

namespace omnihd {
namespace tok {

enum { kF32 = 0, kBF16 = 1, kF16 = 2 };          // omnihd_hip.h: element type codes
constexpr size_t kCacheBytes = 256u << 20;       // the Infinity Cache
inline bool type_ok(int t) { return t == kF32 || t == kBF16 || t == kF16; }
inline int type_size(int t) { return t == kF32 ? 4 : 2; }

// eight elements from p; `left` (> 0) elements of the row remain from p on.  Missing ones read as `fill`.
template <bool ODD, typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, int left, float (&v)[8], float fill = 0.f) {
  if (!ODD || left >= 8) {
    typedef T V __attribute__((ext_vector_type(8)));
    typedef V W __attribute__((aligned(ODD ? sizeof(T) : 16)));
    const V raw = *reinterpret_cast<const W*>(p);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = (float)raw[k];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < left ? (float)p[k] : fill;
  }
}

// the same kept as they are (a row that is asked for ahead of its use), missing ones 0
template <typename T> struct Raw { typedef T V __attribute__((ext_vector_type(8))); };
template <bool ODD, bool STREAM = false, typename T>
__device__ __forceinline__ typename Raw<T>::V raw8(const T* __restrict__ p, int left) {
  typedef typename Raw<T>::V V;
  typedef V W __attribute__((aligned(ODD ? sizeof(T) : 16)));
  if (!ODD || left >= 8) return STREAM ? __builtin_nontemporal_load(reinterpret_cast<const W*>(p)) : *reinterpret_cast<const W*>(p);
  V v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = k < left ? p[k] : (T)0.f;
  return v;
}

// STREAM: past the caches, for what they would not hold anyway
template <bool ODD, bool STREAM = false, typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, int left, const float (&v)[8]) {
  if (!ODD || left >= 8) {
    typedef T V __attribute__((ext_vector_type(8)));
    typedef V W __attribute__((aligned(ODD ? sizeof(T) : 16)));
    V raw;
#pragma unroll
    for (int k = 0; k < 8; ++k) raw[k] = (T)v[k];      // round to nearest even
    if (STREAM) __builtin_nontemporal_store(raw, reinterpret_cast<W*>(p));
    else *reinterpret_cast<W*>(p) = raw;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) p[k] = (T)v[k];
  }
}

// the same for an array whose type is known at run time only (weights, gates): the branch is uniform
template <bool ODD>
__device__ __forceinline__ void load8_any(const void* p, int type, long long at, int left, float (&v)[8]) {
  if (type == kF32) load8<ODD>(static_cast<const float*>(p) + at, left, v);
  else if (type == kBF16) load8<ODD>(static_cast<const __bf16*>(p) + at, left, v);
  else load8<ODD>(static_cast<const _Float16*>(p) + at, left, v);
}
template <bool ODD>
__device__ __forceinline__ void store8_any(void* p, int type, long long at, int left, const float (&v)[8]) {
  if (type == kF32) store8<ODD>(static_cast<float*>(p) + at, left, v);
  else if (type == kBF16) store8<ODD>(static_cast<__bf16*>(p) + at, left, v);
  else store8<ODD>(static_cast<_Float16*>(p) + at, left, v);
}
__device__ __forceinline__ float load1_any(const void* p, int type, long long at) {
  if (type == kF32) return static_cast<const float*>(p)[at];
  if (type == kBF16) return (float)static_cast<const __bf16*>(p)[at];
  return (float)static_cast<const _Float16*>(p)[at];
}
__device__ __forceinline__ void store1_any(void* p, int type, long long at, float v) {
  if (type == kF32) static_cast<float*>(p)[at] = v;
  else if (type == kBF16) static_cast<__bf16*>(p)[at] = (__bf16)v;
  else static_cast<_Float16*>(p)[at] = (_Float16)v;
}

struct Add { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct Max { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };

// Every lane of each run of N neighbouring lanes (N a power of two up to 64) gets the run's combined value.  Within 16 lanes by DPP
// (swap pairs, swap pairs of pairs, mirror 8, mirror 16), beyond by the lane swaps of gfx950: no LDS.  The order is symmetric, so all
// lanes hold the same bits.
template <int N, typename F>
__device__ __forceinline__ float lanes(float v, F f) {
#define OMNIHD_DPP(ctrl) __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(v), ctrl, 0xf, 0xf, true))
  if (N >= 2) v = f(v, OMNIHD_DPP(0xb1));
  if (N >= 4) v = f(v, OMNIHD_DPP(0x4e));
  if (N >= 8) v = f(v, OMNIHD_DPP(0x141));
  if (N >= 16) v = f(v, OMNIHD_DPP(0x140));
#undef OMNIHD_DPP
  if (N >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if (N >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}

// The same over N lanes that may span waves of the block.  `buf` is shared memory for 32 floats, `turn` (same in all threads, 0 at
// first) picks its halves in turn, so that one barrier a call is enough: a thread writes a half again only behind the barrier of the
// call in between, which every thread reaches after it has read that half.  All threads of the block call it.
template <int N, typename F>
__device__ __forceinline__ float group(float v, F f, float* buf, int& turn) {
  if constexpr (N <= 64) {
    return lanes<N>(v, f);
  } else {
    constexpr int waves = N / 64;
    v = lanes<64>(v, f);
    float* half = buf + turn * 16;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) half[threadIdx.x >> 6] = v;
    __syncthreads();
    const float* mine = half + (threadIdx.x / N) * waves;
    v = mine[0];
#pragma unroll
    for (int i = 1; i < waves; ++i) v = f(v, mine[i]);
    return v;
  }
}

}  // namespace tok
}  // namespace omnihd
