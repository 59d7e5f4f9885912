// row_io.h -- what the row kernels share: eight columns of a row in and out of a lane's registers, at 16-byte and at element
// alignment, and sums over the lanes of a row.
#pragma once

#include "device_io.h"

namespace {

constexpr int WG = 256;

// ---------------------------------------------------------------------------------------------------------------
// eight columns of a row at `col`: zeros past the row's end (a lane of no columns gets zeros). AL: rows of a multiple of 8
// elements, 16-byte aligned (unconditional loads, from a clamped column); else at element alignment, the last columns of
// a row one by one
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint4 select(bool ok, uint4 a) {
  return make_uint4(ok ? a.x : 0u, ok ? a.y : 0u, ok ? a.z : 0u, ok ? a.w : 0u);
}
template <typename T> __device__ __forceinline__ typename IO<T>::Raw zero_unless(bool ok, const typename IO<T>::Raw& r) {
  if constexpr (std::is_same<T, float>::value) {
    typename IO<T>::Raw z = r;
    z.a = make_float4(ok ? r.a.x : 0.f, ok ? r.a.y : 0.f, ok ? r.a.z : 0.f, ok ? r.a.w : 0.f);
    z.b = make_float4(ok ? r.b.x : 0.f, ok ? r.b.y : 0.f, ok ? r.b.z : 0.f, ok ? r.b.w : 0.f);
    return z;
  } else {
    typename IO<T>::Raw z = r;
    z.u = select(ok, r.u);
    return z;
  }
}
// the same values, looked at anew: what is unpacked from them in a loop is not kept in twice the registers outside it
template <typename T> __device__ __forceinline__ void anew(typename IO<T>::Raw& r) {
  if constexpr (!std::is_same<T, float>::value) asm volatile("" : "+v"(r.u.x), "+v"(r.u.y), "+v"(r.u.z), "+v"(r.u.w));
  else asm volatile("" : "+v"(r.a.x), "+v"(r.a.y), "+v"(r.a.z), "+v"(r.a.w), "+v"(r.b.x), "+v"(r.b.y), "+v"(r.b.z), "+v"(r.b.w));
}
template <typename T> struct Eight { T e[8]; };
template <typename T, bool AL> __device__ __forceinline__ typename IO<T>::Raw load8(const T* p, int col, int d) {
  if constexpr (AL) {
    return zero_unless<T>(col < d, IO<T>::raw(p + min(col, d - 8)));
  } else {
    if (col + 8 <= d) return UIO<T>::raw(p + col);
    Eight<T> v;
#pragma unroll
    for (int k = 0; k < 8; ++k) v.e[k] = col + k < d ? p[col + k] : (T)0;
    return __builtin_bit_cast(typename IO<T>::Raw, v);
  }
}
template <typename T, bool AL> __device__ __forceinline__ void store8(T* p, int col, int d, const float (&o)[8]) {
  if constexpr (AL) {
    if (col < d) IO<T>::store(p + col, o);
  } else {
    if (col + 8 <= d) {
      UIO<T>::store(p + col, o);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (col + k < d) st1(p + col + k, o[k]);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// LPR lanes share a row, eight columns each; the workgroup's lanes / LPR rows go side by side.
// ---------------------------------------------------------------------------------------------------------------
constexpr int lanes_of(int lpr) { return lpr > WG ? lpr : WG; }

// which of the workgroup's rows this lane has a share of; the same for a whole wave where rows are at least that wide, so that
// the rows' addresses are scalar
template <int LPR> __device__ __forceinline__ int group_of() {
  const int g = (int)threadIdx.x / LPR;
  return LPR >= 64 ? __builtin_amdgcn_readfirstlane(g) : g;
}

// sums over the lanes of a row; rows wider than a wave meet in LDS. The two slots take turns: a slot is written again only
// after the barrier of the other one, which every wave reaches past its reads
template <int LPR> struct RowSum {
  static constexpr int WAVES = lanes_of(LPR) / 64;
  float (*red)[WAVES];
  int slot = 0;
  __device__ __forceinline__ float operator()(float v) {
    v = lanes_reduce(v, LPR < 64 ? LPR : 64, AddOp());
    if constexpr (LPR > 64) {
      const int wave = (int)threadIdx.x >> 6;
      if (((int)threadIdx.x & 63) == 0) red[slot][wave] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int k = 0; k < LPR / 64; ++k) v += red[slot][(wave / (LPR / 64)) * (LPR / 64) + k];
      slot ^= 1;
    }
    return v;
  }
};

}  // namespace
