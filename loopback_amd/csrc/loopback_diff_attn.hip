// loopback_diff_attn.hip -- MI355X (gfx950, CDNA4) kernels of differential attention, bf16 and fp16, forward and backward:
//
//   y = (P1 - lam P2) v,   Pi = softmax(c qi ki^T) over the keys that a query sees
//
// Both maps of a head go through one pass over its keys, each with its own running maximum and sum (fp32 scores, statistics
// and accumulators; the probabilities and score gradients enter the matrix cores in 16 bits, the probabilities of few queries and
// of chunks in two parts of 16). The difference is taken of the two fp32 results. Backward, with D1 = dy . (P1 v), D2 = dy . (P2 v)
// and dA = dy v^T, which both maps share:
//
//   dS1 = P1 (dA - D1),  dS2 = -lam P2 (dA - D2),  dqi = c dSi ki,  dki = c dSi^T qi,  dv = (P1 - lam P2)^T dy,
//   dlam = -sum over the keys of P2 dA (from the fp32 values: D2 has the rounding of the saved P2 v)
//
// Operands go through v_mfma_f32_32x32x16 (dk and dv: 16x16x32): lane l holds row (A) or column (B) l mod 32 at k = 8 (l / 32) .. + 8; of the
// 32 x 32 result it holds column l mod 32 and, in register r, row 4 (l / 32) + r mod 4 + 8 (r / 4). Scores are formed so that
// the next product sums over their rows: a result is then the next one's B operand as it lies in the registers, its k order
// that of Cols32. What a wave keeps in registers are its 32 queries (forward, dq) or keys (dk, dv); the others come through
// LDS in tiles of 32 or 64 rows, two buffers, filled by direct loads. A tile's rows are unpadded and its 16-byte pieces permuted
// (swizzle), so that neither the reads of rows nor the transposing reads of columns meet in a bank.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include <type_traits>

#include "loopback_model.h"
#include "loopback_read.h"
#include "device_io.h"
#include "lds_limit.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void global_void;

constexpr int WG = 256, QB = 128, TILE = 64;      // lanes, rows kept per workgroup (32 a wave), rows per LDS tile of dq's kernel
constexpr float LAZY = 8.f;                        // the maximum moves when it grows by 2^8 or more
constexpr float NONE = -1e30f;                     // the maximum of no scores: finite, so that differences from it are
constexpr float LOG2E = 1.4426950408889634f;

template <typename T> struct Mat;
template <> struct Mat<bf16_t> {
  typedef Bf16Cvt Cvt;
  static __device__ __forceinline__ f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
struct F16Pair : F16Cvt {   // both at once; a multiplication that goes into the conversion rounds once instead of twice
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
  }
};
template <> struct Mat<_Float16> {
  typedef F16Pair Cvt;
  static __device__ __forceinline__ f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}
// registers 8 s .. 8 s + 7 of a result as the B operand of the next product's 16-row step s
template <typename T> __device__ __forceinline__ uint4 operand(const f32x16& x, int s) {
  typedef typename Mat<T>::Cvt C;
  return make_uint4(C::pack2(x[8 * s], x[8 * s + 1]), C::pack2(x[8 * s + 2], x[8 * s + 3]), C::pack2(x[8 * s + 4], x[8 * s + 5]),
                    C::pack2(x[8 * s + 6], x[8 * s + 7]));
}
template <typename T> __device__ __forceinline__ uint2 packed4(const f32x4& x) {
  typedef typename Mat<T>::Cvt C;
  return make_uint2(C::pack2(x[0], x[1]), C::pack2(x[2], x[3]));
}
__device__ __forceinline__ float other_half(float x, bool sum) {   // x joined with the other lane half's
  const unsigned u = __float_as_uint(x);
  const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const float a = __uint_as_float((unsigned)sw[0]), b = __uint_as_float((unsigned)sw[1]);
  return sum ? a + b : fmaxf(a, b);
}
// keeps the compiler from loading operands ahead across it: they would not fit the registers
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }
// the row of a result's register r in lane half h
__device__ __forceinline__ int row_of(int r, int h) { return 4 * h + (r & 3) + 8 * (r >> 2); }

// ---------------------------------------------------------------------------------------------------------------
// rows in LDS, of W elements (64, 128 or 256) in pieces of 16 bytes, piece p of row r in place p ^ swizzle(r). What reads them
// together then meets in no bank (64 of 4 bytes): 16 rows at one piece; four rows, aligned, at four pieces; eight at two.
// Addresses are bytes from the start of LDS (a kernel has one block of it): a few offsets of a lane, formed once, and what is
// known at compile time, which goes into the instruction. (Arrays of their own cost an address register for each of them and
// each offset: 100 spilled registers in the kernel of dk and dv.)
// ---------------------------------------------------------------------------------------------------------------
template <int W> __device__ __forceinline__ int swizzle(int r) {
  return (W == 64 ? (r >> 1 & 1) << 2 : (r & 1) << 3 | (r >> 1 & 1) << 2) | ((r >> 2 ^ r >> 3) & 1) << 1 | (r >> 3 & 1);
}
__device__ __forceinline__ int kept(int x) {   // held as it is, not formed again from what it was formed from
  asm volatile("" : "+v"(x));
  return x;
}
template <typename V> __device__ __forceinline__ V lds_at(int at) { return *reinterpret_cast<__attribute__((address_space(3))) const V*>(at); }
__device__ __forceinline__ uint4 sixteen(int at) { return __builtin_bit_cast(uint4, lds_at<u32x4>(at)); }
__device__ __forceinline__ uint4 four_and_four(int p, int q) {   // a column's elements of two times four rows
  typedef __attribute__((address_space(3))) s16x4* lds4;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds4>(p));
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds4>(q));
  const uint2 ua = __builtin_bit_cast(uint2, a), ub = __builtin_bit_cast(uint2, b);
  return make_uint4(ua.x, ua.y, ub.x, ub.y);
}
// operands of v_mfma_f32_32x32x16
template <int W> struct Rows32 {   // A: rows r0 + l mod 32, columns 16 ks + 8 (l / 32) .. + 8
  int o[W == 64 ? 4 : 8];
  __device__ __forceinline__ explicit Rows32(int ks0 = 0) {   // ks counted from ks0, 0 or half the row's
    const int lane = (int)threadIdx.x & 63, r = lane & 31;
#pragma unroll
    for (int v = 0; v < (W == 64 ? 4 : 8); ++v)
      o[v] = kept(2 * (r * W + 8 * ((2 * (v + ks0) & 15) ^ ((lane >> 5) ^ swizzle<W>(r))) + 128 * (ks0 >> 3)));
  }
  __device__ __forceinline__ uint4 at(int tile, int r0, int ks) const {   // r0 a multiple of 32
    return sixteen(o[W == 64 ? ks & 3 : ks & 7] + tile + 2 * (r0 * W + 128 * (ks >> 3)));
  }
};
template <int W> struct Cols32 {   // A: columns c0 + l mod 32, rows r0 + {4 h + 0..3, 8 + 4 h + 0..3}, h = l / 32
  static constexpr int V = W == 64 ? 2 : 4;
  int o[V];   // of the first four rows; for the others the swizzle turns the two lowest bits of the piece
  __device__ __forceinline__ Cols32() {
    const int lane = (int)threadIdx.x & 63, j = lane & 15, r = 4 * (lane >> 5) + (j >> 2);
    const int piece = (lane >> 4 & 1) * 2 + ((j & 3) >> 1), half = 4 * (j & 1);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      o[v] = kept(2 * (r * W + 8 * ((4 * v) ^ (piece ^ swizzle<W>(r))) + half));
    }
  }
  __device__ __forceinline__ uint4 at(int tile, int r0, int c0) const {   // r0 a multiple of 16, c0 of 32
    const int v = (c0 >> 5) & (V - 1), more = tile + 2 * (r0 * W + 128 * (c0 >> 7));
    return four_and_four(o[v] + more, (o[v] ^ 48) + more + 16 * W);
  }
};
// operands of v_mfma_f32_16x16x32
template <int W> struct Rows16 {   // A: rows r0 + l mod 16, columns 32 ks + 8 (l / 16) .. + 8
  int o[W == 64 ? 2 : 4];
  __device__ __forceinline__ Rows16() {
    const int lane = (int)threadIdx.x & 63, r = lane & 15;
#pragma unroll
    for (int v = 0; v < (W == 64 ? 2 : 4); ++v) o[v] = kept(2 * (r * W + 8 * ((4 * v) ^ ((lane >> 4) ^ swizzle<W>(r)))));
  }
  __device__ __forceinline__ uint4 at(int tile, int r0, int ks) const {   // r0 a multiple of 16
    return sixteen(o[W == 64 ? ks & 1 : ks & 3] + tile + 2 * (r0 * W + 128 * (ks >> 2)));
  }
};
template <int W> struct Cols16 {   // A: columns c0 + l mod 16, rows r0 + {4 g + 0..3, 16 + 4 g + 0..3}, g = l / 16
  int o[W == 64 ? 2 : 4];   // of every other 16 columns: the others are 32 bytes from them, forward or back
  __device__ __forceinline__ Cols16() {
    const int lane = (int)threadIdx.x & 63, j = lane & 15, r = 4 * (lane >> 4) + (j >> 2);
#pragma unroll
    for (int v = 0; v < (W == 64 ? 2 : 4); ++v) o[v] = kept(2 * (r * W + 8 * ((4 * v) ^ (((j & 3) >> 1) ^ swizzle<W>(r))) + 4 * (j & 1)));
  }
  __device__ __forceinline__ uint4 at(int tile, int r0, int c0) const {   // r0 a multiple of 32, c0 of 16
    const int v = (c0 >> 4) & (W == 64 ? 3 : 7), p = (v & 1 ? o[v >> 1] ^ 32 : o[v >> 1]) + tile + 2 * (r0 * W + 128 * (c0 >> 7));
    return four_and_four(p, p + 32 * W);
  }
};

// the offsets for rows of W elements: the given ones, where they are
template <template <int> class R, int W, typename O> __device__ __forceinline__ auto of_width(const O& given) {
  if constexpr (std::is_same<O, R<W>>::value) return given;
  else return R<W>();
}

// 16 bytes (or 4) of memory for each lane, at base + off, to LDS at `to` and what follows it in the lanes' order. In assembly:
// the compiler would wait for it before any read of LDS, of the other buffer too. The data is there past filled().
// ONCE: data that no one reads again soon, past the caches
template <bool ONCE = false> __device__ __forceinline__ void load_lds16(const void* base, uint32_t off, int to) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(to), "v"(off), "s"(base) : "m0", "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "m0", "memory");
}
__device__ __forceinline__ void load_lds4(const void* base, uint32_t off, int to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(off), "s"(base) : "m0", "memory");
}

// Fills N rows of LDS from memory by LANES lanes (whole waves). MAPS rows of memory of W / MAPS elements (`width` of them
// exist, the columns past them repeat the first piece: what they meet is zero) lie side by side in a row of LDS. Rows past
// row `last` repeat it.
template <typename T, int W, int MAPS, int N, int LANES, bool ONCE = false> struct Fill {
  static constexpr int P = W / 8, PASSES = N * P / LANES, PM = P / MAPS, ROWS = LANES / P, VAR = ROWS >= 16 ? 1 : 16 / ROWS;
  static_assert(N * P % LANES == 0 && N % 16 == 0, "whole passes, whole turns of the swizzle");
  const T* base;      // row 0
  int64_t stride;     // elements between rows
  uint32_t off[VAR];  // bytes, of a pass's rows from its first
  // the piece that is stored in this lane's place, in elements from the row's start
  static __device__ __forceinline__ uint32_t col(int lane, int v, int64_t map_stride, int width) {
    const int p = (lane % P) ^ swizzle<W>(lane / P + ROWS * v), m = p / PM, c = 8 * (p % PM);
    return (uint32_t)(m * (int)map_stride) + (uint32_t)(c < width ? c : 0);
  }
  __device__ __forceinline__ Fill(const T* base_, int64_t stride_, int64_t map_stride, int width) : base(base_), stride(stride_) {
    const int lane = (int)threadIdx.x % LANES;
#pragma unroll
    for (int v = 0; v < VAR; ++v) off[v] = (uint32_t)kept(2u * ((uint32_t)(lane / P) * (uint32_t)stride + col(lane, v, map_stride, width)));
  }
  __device__ __forceinline__ void fetch(int row0, int last, int to) const {   // asynchronous: done when vmcnt says so
    to += LANES == 64 ? 0 : 1024 * __builtin_amdgcn_readfirstlane((int)(threadIdx.x % LANES) >> 6);
    const char* b = reinterpret_cast<const char*>(base + (int64_t)row0 * stride);
    if (row0 + N - 1 <= last) {
#pragma unroll
      for (int i = 0; i < PASSES; ++i) load_lds16<ONCE>(b + 2 * i * ROWS * stride, off[i % VAR], to + 16 * i * LANES);
    } else {
      const int r = kept((int)(threadIdx.x % LANES) / P);   // formed here, where it is rarely needed, and not kept
#pragma unroll
      for (int i = 0; i < PASSES; ++i)
        load_lds16<ONCE>(b, off[i % VAR] + 2u * (uint32_t)(min(r + ROWS * i, last - row0) - r) * (uint32_t)stride, to + 16 * i * LANES);
    }
  }
};
__device__ __forceinline__ void filled() {   // this wave's loads are in LDS; then every wave's
  __builtin_amdgcn_s_waitcnt(0x0f70);        // vmcnt(0)
  __syncthreads();
}

// ---------------------------------------------------------------------------------------------------------------
struct Strided { const void* p; int64_t b, t, h; };   // elements between batches, tokens and heads; columns lie side by side
struct Diff {
  Strided q, k, v, lam;
  const int *lengths, *starts;   // NULL: tk, and tk - tq
  void *out, *second;            // y and P2 v [b, tq, h, dv]; second NULL: no backward follows
  float* lse;                    // [2][b h][tq]: base-2 logarithms of the sums of exponentials
  int b, tq, tk, h, hk, dh, dv;
  int causal, lam32;             // lam32: lam is fp32, else the rows' type
  float c, scale;                // scale log2(e), and scale
  // backward
  const void* dy;
  void *dq, *dk, *dval;
  float *delta, *dlam;           // four or, where lam has queries, five numbers [b h][tq] for k_diff_bwd_kv; dlam's parts
  // fp16: the largest |v| of 128 keys [b hk][tk / 128], and |dy| max(1, |lam|) and max(1, |lam|) of 32 queries [b h][tq / 32]
  float* norms;
  float2* sizes;
  int lam_rows;                  // lam has queries; dlam is per query, else per workgroup
  // keys in chunks (few queries), or tiles of queries in parts (dk and dv)
  int splits, chunk;
  float* part;
};

template <typename T> __device__ __forceinline__ float lam_at(const Diff& a, int b, int t, int h) {
  const int64_t o = b * a.lam.b + t * a.lam.t + h * a.lam.h;
  return a.lam32 ? static_cast<const float*>(a.lam.p)[o] : ld1(static_cast<const T*>(a.lam.p) + o);
}
__device__ __forceinline__ int length_of(const Diff& a, int b) { return a.lengths ? min(max(a.lengths[b], 0), a.tk) : a.tk; }
__device__ __forceinline__ int start_of(const Diff& a, int b) {   // far positions all mean every key or none
  const int far = (1 << 30) - 1;
  return a.starts ? min(max(a.starts[b], -far), far) : a.tk - a.tq;
}
// the keys that query i sees: those before this one
__device__ __forceinline__ int seen_by(const Diff& a, int i, int start, int len) {
  return a.causal ? min(max(start + i + 1, 0), len) : len;   // start and i below 2^30
}

// Which block of which head a workgroup takes: `items` (batches times heads of keys) go to the eight XCDs in turn where they
// divide by eight, so that a head's keys are read from one L2; the blocks with the most work first.
struct Work { int item, g, block; };
__device__ __forceinline__ bool work_of(int id, int items, int groups, int blocks, Work& w) {
  int unit;
  if (items % 8 == 0) {
    const int i = id >> 3, per = items >> 3;
    w.item = (id & 7) + 8 * (i % per);
    unit = i / per;
  } else {
    w.item = id % items;
    unit = id / items;
  }
  w.g = unit % groups;
  w.block = unit / groups;
  return w.block < blocks;
}

__device__ __forceinline__ uint4 only(bool ok, const uint4& a) {   // a, or zeros
  return make_uint4(ok ? a.x : 0u, ok ? a.y : 0u, ok ? a.z : 0u, ok ? a.w : 0u);
}
// a wave's 32 rows as B operands: row r, columns 16 ks + 8 (l / 32) .. + 8, zeros past `width`
template <typename T, int W> struct Kept {
  uint4 f[W / 16];
  __device__ __forceinline__ void load(const T* row, int width) {
    const int h = ((int)threadIdx.x & 63) >> 5;
#pragma unroll
    for (int ks = 0; ks < W / 16; ++ks) {
      const int c = 16 * ks + 8 * h;
      f[ks] = only(c < width, *reinterpret_cast<const uint4*>(row + min(c, width - 8)));
    }
  }
};

// One map's running softmax of a query (a lane pair's column)
struct Soft {
  float m = NONE, l[4] = {0.f, 0.f, 0.f, 0.f};   // four sums: no chain of dependent adds
  __device__ __forceinline__ float sum() const { return other_half((l[0] + l[1]) + (l[2] + l[3]), true); }
};
// a tile's scores of one map, as probabilities relative to the running maximum, packed: p[4 i' ...]; o, and l, are rescaled
template <typename T, int NB, int DB>
__device__ __forceinline__ void soft_step(f32x16 (&s)[NB], Soft& st, f32x16 (&o)[DB], uint4 (&p)[2 * NB], float c) {
  float mx = s[0][0];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[i][r]);
  mx = other_half(mx, false) * c;
  if (__any(mx > st.m + LAZY)) {
    const float mn = fmaxf(st.m, mx), a = st.m == mn ? 1.f : __builtin_amdgcn_exp2f(st.m - mn);
    st.m = mn;
#pragma unroll
    for (int k = 0; k < 4; ++k) st.l[k] *= a;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] *= a;
  }
#pragma unroll
  for (int i = 0; i < NB; ++i) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[i][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][r], c, -st.m));
      st.l[r & 3] += s[i][r];
    }
    p[2 * i] = operand<T>(s[i], 0);
    p[2 * i + 1] = operand<T>(s[i], 1);
  }
}

// what the 16 bits of a tile's probabilities leave of them, s as soft_step left it: the products' second part, where their rounding is
// not to be added to the result's
template <typename T> __device__ __forceinline__ void rest_of(const f32x16& s, const uint4 (&p)[2], uint4 (&rest)[2]) {
  typedef typename Mat<T>::Cvt C;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w[4] = {p[i].x, p[i].y, p[i].z, p[i].w};
    uint32_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float u, v;
      C::unpack2(w[k], u, v);
      x[k] = C::pack2(s[8 * i + 2 * k] - u, s[8 * i + 2 * k + 1] - v);
    }
    rest[i] = make_uint4(x[0], x[1], x[2], x[3]);
  }
}

template <int DH, int DV> constexpr int waves_bwd() { return DH + DV <= 192 ? 2 : 1; }   // waves to a SIMD, by their registers

// ---------------------------------------------------------------------------------------------------------------
// The score gradients P (dA - D) enter the matrix cores in 16 bits. fp16 holds 2^-14 to 2^16 in full; from upstreams of 1e-4 dq and dk
// were 6.3e-3 and 7.2e-3 off for that (2048 tokens; their own rounding 2.0e-3 and 1.4e-3, and now no more), and from some of 1e4 infinite,
// though both are in range. So the gradients are taken times a power of two that brings their bound, |dA - D| <= 2 |dy| |v|, to 2^LIFT,
// and the fp32 sums by as much back: each query's own power in dq, whose columns are queries; that of all the queries that a workgroup
// meets in dk and dv, which sum over them. What is below 2^(-24 - LIFT) of the bound is lost. dv's combined map, whose probabilities of
// 32768 keys are about 2^-15, is lifted the same way from its bound (4.4e-4 off, now 2.9e-4 as of 4096 keys). bf16 has fp32's range.
// The norms of v are a launch before: 8 x 2048 tokens, 6 heads of 128: 6 us of the backward's 260 (25 MB at 4 TB/s); 3 x 683, 2 of 256: 4.
// ---------------------------------------------------------------------------------------------------------------
template <typename T> constexpr bool LIFTED = std::is_same<T, _Float16>::value;
constexpr int LIFT = 13;   // three binades are left for what D's own rounding adds
__device__ __forceinline__ int lift_of(float bound) { return LIFT - __builtin_amdgcn_frexp_expf(bound); }   // bound < 2^frexp_exp; 0: any
__device__ __forceinline__ float power_of_2(int n) { return __uint_as_float((unsigned)(127 + n) << 23); }   // within +-126, as a lift is
__device__ __forceinline__ float finite_or_0(float x) { return x < INFINITY ? x : 0.f; }   // of x >= 0 or NaN
// the largest |v| of the first n keys of an item, to every lane of a wave
__device__ __forceinline__ float norm_of(const Diff& a, int item, int n) {
  const float* of = a.norms + (int64_t)item * ((a.tk + QB - 1) / QB);
  float most = 0.f;
  for (int i = (int)threadIdx.x & 63; i * QB < n; i += 64) most = fmaxf(most, of[i]);
  return lanes_reduce(most, 64, MaxOp());
}
// |v|, the largest of QB keys, those that are finite (a result that another one enters is not): DV / 8 lanes to a row
template <typename T, int DV> __global__ __launch_bounds__(WG) void k_diff_bwd_norms(const Diff a) {
  constexpr int P = DV / 8, N = QB * P / WG;
  __shared__ float s_most[WG / 64];
  const int tid = (int)threadIdx.x, blocks = (a.tk + QB - 1) / QB, item = (int)blockIdx.x / blocks, k0 = ((int)blockIdx.x - item * blocks) * QB;
  const int b = item / a.hk, hk = item - b * a.hk, end = min(k0 + QB, length_of(a, b)), col = 8 * (tid % P);
  const T* v = static_cast<const T*>(a.v.p) + b * a.v.b + hk * a.v.h + col;
  typename IO<T>::Raw x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {   // all in flight at once
    const int r = k0 + tid / P + i * (WG / P);
    x[i] = IO<T>::zero();
    if (r < end && col < a.dv) x[i] = IO<T>::raw(v + r * a.v.t);
  }
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float e[8], sum = 0.f;
    IO<T>::unpack(x[i], e);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum = __builtin_fmaf(e[k], e[k], sum);
    most = fmaxf(most, finite_or_0(lanes_reduce(sum, P, AddOp())));
  }
  most = lanes_reduce(most, 64, MaxOp());
  if ((tid & 63) == 0) s_most[tid >> 6] = most;
  __syncthreads();
  if (tid == 0) a.norms[blockIdx.x] = sqrtf(fmaxf(fmaxf(s_most[0], s_most[1]), fmaxf(s_most[2], s_most[3])));
}

// ---------------------------------------------------------------------------------------------------------------
// forward: 64 queries of a head per workgroup, two waves for each 32 of them, one for each map. (Both maps in one wave read
// the values once for both, but hold 256 registers, so two waves to a SIMD, in which the vector units, a wave's softmax, wait
// for its products and the other way round; so it is three here.) Vector units and matrix cores bound it: per 32 x 32 scores of a
// map 16 exponentials of 8 cycles and some 80 operations of 4, 490 cycles with what the issue of products costs, and 384 of
// products; the two overlap little (counters: 0.47 and 0.37 of the time). 8 x 2048 tokens, 6 heads of 64|128 in bf16: 101 us, 77 GFLOP
// done at 0.77 PFLOP/s; 2 x 4096, 16 heads: 235 us, 0.88. A tile's scores formed between the exponentials of the tile before, so
// that one wave's products and softmax overlap: 107 us. Tiles of 64 keys: 111, eight waves to a workgroup: 218.
// The probabilities enter the products rounded to the type, which is added to the results' own rounding (1.4 to 1.5 of it in the norm):
// as two parts, 125 us for 92 without gradients. SPLIT, few blocks of queries over long keys, takes the two parts: there they cost 20.3 ->
// 22.7 us (3 x 333 new tokens over 1001 keys) to 75 -> 100 (500 over 16384), and the results are rounded once.
// ---------------------------------------------------------------------------------------------------------------
constexpr int FW = 4, FQ = 16 * FW, FT = 32, FL = 64 * FW;   // waves and queries of a workgroup, keys of a tile, lanes
template <int DH, int DV> constexpr int waves_fwd() { return DH <= 64 && DV <= 128 ? 3 : 2; }
template <int DH, int DV> constexpr int fwd_lds() {   // two tiles; at the end a map's results
  const int tiles = 2 * FT * (2 * DH + DV) * 2, results = FQ * DV * 4;
  return tiles > results ? tiles : results;
}
template <int DV> constexpr int partial_row() { return 2 * DV + 4; }   // floats of a row's partial result: o1, o2, m1, l1, m2, l2
template <typename T, int DH, int DV, bool SPLIT>
__global__ __launch_bounds__(FL) __attribute__((amdgpu_waves_per_eu((waves_fwd<DH, DV>())))) void k_diff_fwd(const Diff a) {
  extern __shared__ __align__(16) char lds_block[];   // two tiles of keys, two of values
  constexpr int KT = FT * 2 * DH, VT = FT * DV, DB = DV / 32, K0 = 0, K1 = 2 * KT, V0 = 4 * KT, V1 = 4 * KT + 2 * VT;
  const int lane = (int)threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), map = wave & 1;
  const int groups = a.h / a.hk, blocks = (a.tq + FQ - 1) / FQ;
  const int all = a.b * a.h * blocks, split = SPLIT ? (int)blockIdx.x / all : 0;
  Work wk;
  if (!work_of((int)blockIdx.x - split * all, a.b * a.hk, groups, blocks, wk)) return;
  const int q0 = (blocks - 1 - wk.block) * FQ, b = wk.item / a.hk, hk = wk.item - b * a.hk, head = hk * groups + wk.g;
  const int len = length_of(a, b), start = start_of(a, b);
  const int w0 = q0 + 32 * (wave >> 1), query = w0 + (lane & 31), qrow = min(query, a.tq - 1);
  Kept<T, DH> q;
  q.load(static_cast<const T*>(a.q.p) + b * a.q.b + qrow * a.q.t + (2 * head + map) * a.q.h, a.dh);
  const int seen = seen_by(a, qrow, start, len);
  const int most = seen_by(a, min(q0 + FQ, a.tq) - 1, start, len);             // of the workgroup's queries
  const int wmost = w0 < a.tq ? seen_by(a, min(w0 + 32, a.tq) - 1, start, len) : 0, wleast = seen_by(a, min(w0, a.tq - 1), start, len);
  const Rows32<2 * DH> krows(map * (DH / 16));
  const Cols32<DV> vcols;
  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = zero16();
  Soft sm;
  const int first = SPLIT ? split * a.chunk / FT : 0, last = (most + FT - 1) / FT;   // a chunk has whole tiles
  const int ntiles = SPLIT ? min(last, first + a.chunk / FT) : last;
  const Fill<T, 2 * DH, 2, FT, FL> kf(static_cast<const T*>(a.k.p) + b * a.k.b + 2 * hk * a.k.h, a.k.t, a.k.h, a.dh);
  const Fill<T, DV, 1, FT, FL> vf(static_cast<const T*>(a.v.p) + b * a.v.b + hk * a.v.h, a.v.t, 0, a.dv);
  if (ntiles > first) {
    kf.fetch(first * FT, len - 1, K0);
    vf.fetch(first * FT, len - 1, V0);
  }
  filled();   // in every case: a wait for what was loaded above, left to the loop, would wait there for the tiles too
  auto tile = [&](int j, auto buffer) {
    constexpr int cur = decltype(buffer)::value, kt = cur ? K1 : K0, vt = cur ? V1 : V0;   // known: they go into the reads' offsets
    const int k0 = j * FT;
    if (j + 1 < ntiles) {   // the other buffer's readers are past the barrier below
      kf.fetch(k0 + FT, len - 1, cur ? K0 : K1);
      vf.fetch(k0 + FT, len - 1, cur ? V0 : V1);
    }
#pragma unroll
    for (int n = 0; n < FT / 32; ++n) {
      const int k1 = k0 + 32 * n;
      if (k1 >= wmost) break;
      f32x16 s[1];
      s[0] = zero16();
      uint4 x[DH / 16], v[DB];   // operands, read before they are needed
      constexpr bool AHEAD = DB <= 4;   // wider: the registers do not hold them
#pragma unroll
      for (int ks = 0; ks < DH / 16; ++ks) x[ks] = krows.at(kt, 32 * n, ks);
      if (AHEAD) {
#pragma unroll
        for (int d = 0; d < DB; ++d) v[d] = vcols.at(vt, 32 * n, 32 * d);
      }
      in_order();
#pragma unroll
      for (int ks = 0; ks < DH / 16; ++ks) s[0] = Mat<T>::mfma(x[ks], q.f[ks], s[0]);
      if (k1 + 32 > wleast) {   // wave-uniform: keys that some query of the wave does not see
        const int left = seen - k1 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (row_of(r, 0) >= left) s[0][r] = -INFINITY;
      }
      uint4 p[2], rest[2];
      soft_step<T>(s, sm, o, p, a.c);
      if (SPLIT) rest_of<T>(s[0], p, rest);
      auto product = [&](int i, int d, const uint4& v) {
        o[d] = Mat<T>::mfma(v, p[i], o[d]);
        if (SPLIT) o[d] = Mat<T>::mfma(v, rest[i], o[d]);
      };
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        product(0, d, AHEAD ? v[d] : vcols.at(vt, 32 * n, 32 * d));
        if (AHEAD) v[d] = vcols.at(vt, 32 * n + 16, 32 * d);
      }
      if (AHEAD) in_order();
#pragma unroll
      for (int d = 0; d < DB; ++d) product(1, d, AHEAD ? v[d] : vcols.at(vt, 32 * n + 16, 32 * d));
    }
    if (j + 1 < ntiles) filled();
  };
  for (int j = first; j < ntiles; j += 2) {
    tile(j, std::integral_constant<int, 0>());
    if (j + 1 < ntiles) tile(j + 1, std::integral_constant<int, 1>());
  }
  if constexpr (SPLIT) {
    const float l = sm.sum();
    if (query >= a.tq) return;
    float* p = a.part + (((int64_t)wk.item * a.tq * groups + query * groups + wk.g) * a.splits + split) * partial_row<DV>();
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int col = 32 * d + 8 * g + 4 * half;
        if (col < a.dv) *reinterpret_cast<f32x4*>(p + map * DV + col) = f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
      }
    if (half == 0) *reinterpret_cast<float2*>(p + 2 * DV + 2 * map) = make_float2(sm.m, l);
    return;
  }
  // a query that sees no key: zeros, and an infinite logarithm, which makes every probability 0
  const float l = sm.sum(), inv = l > 0.f || l != l ? 1.f / l : 0.f;
  if (a.lse && half == 0 && query < a.tq)
    a.lse[(((int64_t)map * a.b + b) * a.h + head) * a.tq + query] = inv != 0.f ? sm.m + __builtin_amdgcn_logf(l) : INFINITY;
  const int64_t orow = (((int64_t)b * a.tq + query) * a.h + head) * a.dv;
  T* op = static_cast<T*>(a.out) + orow;
  T* sp = static_cast<T*>(a.second) + orow;
  float* mine = reinterpret_cast<float*>(lds_block) + (wave >> 1) * 32 * DV + 4 * lane;   // [register / 4][lane][4]
  __syncthreads();   // the last tile has been read
  if (map) {
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 z = f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]} * inv;
        *reinterpret_cast<f32x4*>(mine + (4 * d + g) * 256) = z;
        const int col = 32 * d + 8 * g + 4 * half;
        if (a.second && col < a.dv && query < a.tq) *reinterpret_cast<uint2*>(sp + col) = packed4<T>(z);
      }
  }
  __syncthreads();
  if (map || query >= a.tq) return;
  const float lam = lam_at<T>(a, b, query, head);
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = 32 * d + 8 * g + 4 * half;
      const f32x4 z = *reinterpret_cast<const f32x4*>(mine + (4 * d + g) * 256);
      const f32x4 y = f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]} * inv - lam * z;
      if (col < a.dv) *reinterpret_cast<uint2*>(op + col) = packed4<T>(y);
    }
}

// ---------------------------------------------------------------------------------------------------------------
// few queries: the (query, head of the group) pairs of a head of keys are the 32 rows of one block (tq times the group at
// most 32). A workgroup takes a chunk of its keys, in tiles of 64: two waves for each map, each with 32 keys of a tile. The
// keys' and values' stream bounds it, so the probabilities enter the products as two 16-bit parts: their rounding is not added to
// the result's. The waves' results meet in LDS, and those of the chunks in k_diff_join. One token each over 32 caches of up to 8192
// keys, 8 heads on 2 of 64|128 in bf16: 41 us, 201 MB at 4.9 TB/s past the caches (44 through them), and 4 for the join. (A wave for
// both maps and a quarter of a tile's keys held too many registers: 60 where this took 44. Two and a half times as many chunks: 45.)
// ---------------------------------------------------------------------------------------------------------------
constexpr int FEW = 32, NT = 64;   // rows, keys of a tile
template <int DH, int DV> constexpr int few_lds() {   // two tiles; at the end the four waves' results
  const int tiles = 2 * NT * (2 * DH + DV) * 2, results = 4 * FEW * (DV + 2) * 4;
  return tiles > results ? tiles : results;
}

template <typename T, int DH, int DV>
__global__ __launch_bounds__(WG) __attribute__((amdgpu_waves_per_eu(2))) void k_diff_few(const Diff a) {
  extern __shared__ __align__(16) char lds_block[];
  constexpr int KT = NT * 2 * DH, VT = NT * DV, DB = DV / 32, K0 = 0, K1 = 2 * KT, V0 = 4 * KT, V1 = 4 * KT + 2 * VT, ROW = partial_row<DV>();
  typedef typename Mat<T>::Cvt C;
  const int lane = (int)threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), map = wave & 1, part = wave >> 1;
  const int groups = a.h / a.hk, rows = a.tq * groups;
  const int item = (int)blockIdx.x / a.splits, split = (int)blockIdx.x - item * a.splits, b = item / a.hk, hk = item - b * a.hk;
  const int len = length_of(a, b), start = start_of(a, b);
  const int row = min(lane & 31, rows - 1), query = row / groups, head = hk * groups + row - query * groups;
  Kept<T, DH> q;
  q.load(static_cast<const T*>(a.q.p) + b * a.q.b + query * a.q.t + (2 * head + map) * a.q.h, a.dh);
  const int seen = seen_by(a, query, start, len);
  const int c0 = split * a.chunk, c1 = min(c0 + a.chunk, seen_by(a, a.tq - 1, start, len)), least = seen_by(a, 0, start, len);
  const Rows32<2 * DH> krows(map * (DH / 16));
  const Cols32<DV> vcols;
  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = zero16();
  Soft sm;
  const Fill<T, 2 * DH, 2, NT, WG, true> kf(static_cast<const T*>(a.k.p) + b * a.k.b + 2 * hk * a.k.h, a.k.t, a.k.h, a.dh);
  const Fill<T, DV, 1, NT, WG, true> vf(static_cast<const T*>(a.v.p) + b * a.v.b + hk * a.v.h, a.v.t, 0, a.dv);
  if (c0 < c1) {
    kf.fetch(c0, len - 1, K0);
    vf.fetch(c0, len - 1, V0);
  }
  filled();
  auto tile = [&](int k0, auto buffer) {
    constexpr int cur = decltype(buffer)::value;
    if (k0 + NT < c1) {
      kf.fetch(k0 + NT, len - 1, cur ? K0 : K1);
      vf.fetch(k0 + NT, len - 1, cur ? V0 : V1);
    }
    const int k1 = k0 + 32 * part, kt = (cur ? K1 : K0) + 64 * part * 2 * DH, vt = (cur ? V1 : V0) + 64 * part * DV;
    if (k1 < c1) {
      f32x16 s[1];
      s[0] = zero16();
#pragma unroll
      for (int ks = 0; ks < DH / 16; ++ks) s[0] = Mat<T>::mfma(krows.at(kt, 0, ks), q.f[ks], s[0]);
      if (k1 + 32 > min(least, c1)) {   // past the chunk too: those keys are the next one's
        const int left = min(seen, c1) - k1 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (row_of(r, 0) >= left) s[0][r] = -INFINITY;
      }
      uint4 p[2], rest[2];
      soft_step<T>(s, sm, o, p, a.c);
      rest_of<T>(s[0], p, rest);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const uint4 v = vcols.at(vt, 16 * i, 32 * d);
          o[d] = Mat<T>::mfma(v, p[i], o[d]);
          o[d] = Mat<T>::mfma(v, rest[i], o[d]);
        }
    }
    if (k0 + NT < c1) filled();
  };
  for (int k0 = c0; k0 < c1; k0 += 2 * NT) {
    tile(k0, std::integral_constant<int, 0>());
    if (k0 + NT < c1) tile(k0 + NT, std::integral_constant<int, 1>());
  }
  const float l = sm.sum();
  __syncthreads();   // the last tile has been read
  float* mine = reinterpret_cast<float*>(lds_block);   // [wave][32 rows][DV + 2]: o, m, l
  if ((lane & 31) < rows) {
    float* p = mine + (wave * FEW + (lane & 31)) * (DV + 2);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) p[32 * d + row_of(r, half)] = o[d][r];
    if (half == 0) {
      p[DV] = sm.m;
      p[DV + 1] = l;
    }
  }
  __syncthreads();
  for (int i = (int)threadIdx.x; i < rows * DV; i += WG) {
    const int r = i / DV, col = i - r * DV, qi = r / groups, hd = hk * groups + r - qi * groups;
    float y[2], m[2], sum[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {   // the map's two waves
      const float *p0 = mine + (e * FEW + r) * (DV + 2), *p1 = p0 + 2 * FEW * (DV + 2);
      m[e] = fmaxf(p0[DV], p1[DV]);
      const float f0 = __builtin_amdgcn_exp2f(p0[DV] - m[e]), f1 = __builtin_amdgcn_exp2f(p1[DV] - m[e]);
      sum[e] = p0[DV + 1] * f0 + p1[DV + 1] * f1;
      y[e] = p0[col] * f0 + p1[col] * f1;
    }
    if (a.splits == 1) {
#pragma unroll
      for (int e = 0; e < 2; ++e) y[e] = sum[e] > 0.f || sum[e] != sum[e] ? y[e] / sum[e] : 0.f;
      if (col < a.dv)
        st1(static_cast<T*>(a.out) + (((int64_t)b * a.tq + qi) * a.h + hd) * a.dv + col, y[0] - lam_at<T>(a, b, qi, hd) * y[1]);
    } else {
      float* out = a.part + ((int64_t)(item * rows + r) * a.splits + split) * ROW;
      out[col] = y[0];
      out[DV + col] = y[1];
      if (col == 0) *reinterpret_cast<float4*>(out + 2 * DV) = make_float4(m[0], sum[0], m[1], sum[1]);
    }
  }
}

// The chunks' partial rows [batch and head of keys][query][head of its group] as one, relative to the running maxima: DV / 4 lanes to
// a row, four columns of both maps each, four chunks' loads in flight. SHARED, few rows: the workgroup's groups of lanes take the
// chunks of one row in turn, and meet in LDS.
constexpr int MOST_CHUNKS = 256, SHARED_ROWS = 4096;
struct Joined {
  float m[2] = {NONE, NONE}, l[2] = {0.f, 0.f};
  f32x4 o[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  // N chunks' maxima and sums (m1, l1, m2, l2) and values
  template <int N> __device__ __forceinline__ void add(const float4 (&e)[N], const f32x4 (&x)[2][N]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float most = m[k];
#pragma unroll
      for (int u = 0; u < N; ++u) most = fmaxf(most, k ? e[u].z : e[u].x);
      const float f = __builtin_amdgcn_exp2f(m[k] - most);
      m[k] = most;
      l[k] *= f;
      o[k] *= f;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const float w = __builtin_amdgcn_exp2f((k ? e[u].z : e[u].x) - most);
        l[k] = __builtin_fmaf(k ? e[u].w : e[u].y, w, l[k]);
        o[k] += x[k][u] * w;
      }
    }
  }
};
template <typename T, int DV, bool SHARED> __global__ __launch_bounds__(WG) void k_diff_join(const Diff a) {
  constexpr int ROW = partial_row<DV>(), L = DV / 4, G = WG / L, U = 4;
  __shared__ __align__(16) float s_part[SHARED ? G * ROW : 4];
  const int tid = (int)threadIdx.x, lane = tid % L, grp = tid / L, groups = a.h / a.hk, rows = a.tq * groups, n = a.splits;
  const int64_t at = SHARED ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * G + grp;
  if (at >= (int64_t)a.b * a.hk * rows) return;   // SHARED: the grid is the rows
  const int item = (int)(at / rows), r = (int)(at - (int64_t)item * rows);
  const int b = item / a.hk, hk = item - b * a.hk, query = r / groups, head = hk * groups + r - query * groups;
  const float* p = a.part + at * n * ROW;
  const float lam = lam_at<T>(a, b, query, head);
  Joined s;
  auto take = [&](auto many, int i, int step) {
    constexpr int N = decltype(many)::value;
    float4 e[N];
    f32x4 x[2][N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const float* c = p + (int64_t)(i + u * step) * ROW;
      e[u] = *reinterpret_cast<const float4*>(c + 2 * DV);
      x[0][u] = *reinterpret_cast<const f32x4*>(c + 4 * lane);
      x[1][u] = *reinterpret_cast<const f32x4*>(c + DV + 4 * lane);
    }
    s.template add<N>(e, x);
  };
  constexpr int step = SHARED ? G : 1;
  int i = SHARED ? grp : 0;
  for (; i + (U - 1) * step < n; i += U * step) take(std::integral_constant<int, U>(), i, step);
  for (; i < n; i += step) take(std::integral_constant<int, 1>(), i, step);
  if constexpr (SHARED) {
    float* mine = s_part + grp * ROW;
    *reinterpret_cast<f32x4*>(mine + 4 * lane) = s.o[0];
    *reinterpret_cast<f32x4*>(mine + DV + 4 * lane) = s.o[1];
    if (lane == 0) *reinterpret_cast<float4*>(mine + 2 * DV) = make_float4(s.m[0], s.l[0], s.m[1], s.l[1]);
    __syncthreads();
    if (grp) return;
    for (int g = 1; g < G; ++g) {
      const float* c = s_part + g * ROW;
      const float4 e[1] = {*reinterpret_cast<const float4*>(c + 2 * DV)};
      const f32x4 x[2][1] = {{*reinterpret_cast<const f32x4*>(c + 4 * lane)}, {*reinterpret_cast<const f32x4*>(c + DV + 4 * lane)}};
      s.add<1>(e, x);
    }
  }
  bool sees[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    sees[k] = s.l[k] > 0.f || s.l[k] != s.l[k];
    s.o[k] *= sees[k] ? 1.f / s.l[k] : 0.f;
    if (a.lse && lane == 0)
      a.lse[(((int64_t)k * a.b + b) * a.h + head) * a.tq + query] = sees[k] ? s.m[k] + __builtin_amdgcn_logf(s.l[k]) : INFINITY;
  }
  if (4 * lane >= a.dv) return;
  const int64_t o = (((int64_t)b * a.tq + query) * a.h + head) * a.dv + 4 * lane;
  if (a.second) *reinterpret_cast<uint2*>(static_cast<T*>(a.second) + o) = packed4<T>(s.o[1]);
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + o) = packed4<T>(s.o[0] - lam * s.o[1]);
}

// ---------------------------------------------------------------------------------------------------------------
// backward: dq, the deltas and dlam's parts. 128 queries of a head per workgroup, both maps in a wave, which share dA. Bound as the
// forward is, by vector units (0.39 of the time) and matrix cores (0.30) that overlap little, at two waves to a SIMD: 8 x 2048 tokens, 6
// heads of 64|128: 122 us, 77 GFLOP at 0.63 PFLOP/s; 2 x 4096, 16 heads: 281 us, 0.73. Operands read a step ahead spill: 141.
// D1 and D2 come from the rounded y and P2 v, where many keys share them; for the queries that see at most two tiles, where dA - D is a
// small part of both, a pass over these before sums P dA in fp32 (the first block of a causal sequence, short ones: no time). Of a single
// key's probability the gradient is zero, and exactly that.
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int DH, int DV>
__global__ __launch_bounds__(WG) __attribute__((amdgpu_waves_per_eu((waves_bwd<DH, DV>())))) void k_diff_bwd_q(const Diff a) {
  constexpr int KT = TILE * 2 * DH, VT = TILE * DV, QB_ = DH / 32;
  extern __shared__ __align__(16) char lds_block[];   // two tiles of keys, two of values; four floats
  constexpr int K0 = 0, K1 = 2 * KT, V0 = 4 * KT, V1 = 4 * KT + 2 * VT;
  const int lane = (int)threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int groups = a.h / a.hk, blocks = (a.tq + QB - 1) / QB;
  Work wk;
  if (!work_of((int)blockIdx.x, a.b * a.hk, groups, blocks, wk)) return;
  const int qblock = blocks - 1 - wk.block, q0 = qblock * QB, b = wk.item / a.hk, hk = wk.item - b * a.hk, head = hk * groups + wk.g;
  const int len = length_of(a, b), start = start_of(a, b);
  const int w0 = q0 + 32 * wave, query = w0 + (lane & 31), qrow = min(query, a.tq - 1);
  const T* qp = static_cast<const T*>(a.q.p) + b * a.q.b + qrow * a.q.t + 2 * head * a.q.h;
  const int64_t orow = (((int64_t)b * a.tq + qrow) * a.h + head) * a.dv;
  Kept<T, DH> q[2];
  Kept<T, DV> g;
  q[0].load(qp, a.dh);
  q[1].load(qp + a.q.h, a.dh);
  g.load(static_cast<const T*>(a.dy) + orow, a.dv);
  const float lam = lam_at<T>(a, b, qrow, head);
  float d1 = 0.f, d2 = 0.f;   // dy . y, dy . (P2 v)
#pragma unroll
  for (int ks = 0; ks < DV / 16; ++ks) {
    const int col = 16 * ks + 8 * half;
    if (col < a.dv) {
      float u[8], y[8], z[8];
      IO<T>::unpack(typename IO<T>::Raw{g.f[ks]}, u);
      IO<T>::load(static_cast<const T*>(a.out) + orow + col, y);
      IO<T>::load(static_cast<const T*>(a.second) + orow + col, z);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        d1 = __builtin_fmaf(u[k], y[k], d1);
        d2 = __builtin_fmaf(u[k], z[k], d2);
      }
    }
  }
  d2 = other_half(d2, true);
  d1 = __builtin_fmaf(lam, d2, other_half(d1, true));
  const int64_t n = ((int64_t)b * a.h + head) * a.tq + qrow, all = (int64_t)a.b * a.h * a.tq;
  const float ls1 = a.lse[n], ls2 = a.lse[n + all];
  const int seen = seen_by(a, qrow, start, len);
  const int most = seen_by(a, min(q0 + QB, a.tq) - 1, start, len), least = seen_by(a, q0, start, len);
  const int wmost = w0 < a.tq ? seen_by(a, min(w0 + 32, a.tq) - 1, start, len) : 0, wleast = seen_by(a, min(w0, a.tq - 1), start, len);
  const Rows32<2 * DH> krows;
  const auto vrows = of_width<Rows32, DV>(krows);
  const Cols32<2 * DH> kcols;
  f32x16 dq[2][QB_];
#pragma unroll
  for (int d = 0; d < QB_; ++d) dq[0][d] = dq[1][d] = zero16();
  float dlam = 0.f;
  int lift = 0;
  if constexpr (LIFTED<T>) {
    float sum = 0.f;
#pragma unroll
    for (int ks = 0; ks < DV / 16; ++ks) {
      float u[8];
      IO<T>::unpack(typename IO<T>::Raw{g.f[ks]}, u);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum = __builtin_fmaf(u[k], u[k], sum);
    }
    const float size = finite_or_0(sqrtf(other_half(sum, true)));
    lift = lift_of(2.f * size * norm_of(a, wk.item, most));
    const float factor = fmaxf(1.f, finite_or_0(fabsf(lam)));
    const float largest = lanes_reduce(query < a.tq ? finite_or_0(size * factor) : 0.f, 64, MaxOp());
    const float most_lam = lanes_reduce(factor, 64, MaxOp());
    if (lane == 0) a.sizes[(((int64_t)b * a.h + head) * blocks + qblock) * (QB / 32) + wave] = make_float2(largest, most_lam);
  }
  const int ntiles = (most + TILE - 1) / TILE;
  const Fill<T, 2 * DH, 2, TILE, WG> kf(static_cast<const T*>(a.k.p) + b * a.k.b + 2 * hk * a.k.h, a.k.t, a.k.h, a.dh);
  const Fill<T, DV, 1, TILE, WG> vf(static_cast<const T*>(a.v.p) + b * a.v.b + hk * a.v.h, a.v.t, 0, a.dv);
  if (ntiles > 0) {
    kf.fetch(0, len - 1, K0);
    vf.fetch(0, len - 1, V0);
  }
  filled();   // in every case: a wait for what was loaded above, left to the loop, would wait there for the tiles too
  if (least <= 2 * TILE) {   // workgroup-uniform: some of its queries' keys all lie in the first two tiles
    if (ntiles > 1) {
      kf.fetch(TILE, len - 1, K1);
      vf.fetch(TILE, len - 1, V1);
      filled();
    }
    float e[2] = {0.f, 0.f};
    auto terms = [&](int k0, int kt, int vt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x16 da = zero16();
#pragma unroll
        for (int ks = 0; ks < DV / 16; ++ks) da = Mat<T>::mfma(vrows.at(vt, 32 * i, ks), g.f[ks], da);
        const int left = seen - k0 - 32 * i - 4 * half;
#pragma unroll
        for (int map = 0; map < 2; ++map) {
          f32x16 x = zero16();
#pragma unroll
          for (int ks = 0; ks < DH / 16; ++ks) x = Mat<T>::mfma(krows.at(kt, 32 * i, map * (DH / 16) + ks), q[map].f[ks], x);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (row_of(r, 0) < left) e[map] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(x[r], a.c, map ? -ls2 : -ls1)), da[r], e[map]);
        }
      }
    };
    if (0 < wmost) terms(0, K0, V0);
    if (TILE < wmost) terms(TILE, K1, V1);
    const float sum1 = other_half(e[0], true), sum2 = other_half(e[1], true);
    d1 = seen <= 2 * TILE ? sum1 : d1;
    d2 = seen <= 2 * TILE ? sum2 : d2;
    __syncthreads();   // the second tile, which the loop fetches again, has been read
  }
  if (query < a.tq && half == 0) {   // what the kernel of dk and dv reads: see there
    const float sign = lam < 0.f ? -1.f : 1.f;
    a.delta[n] = ls1;
    a.delta[n + all] = ls2 - __builtin_amdgcn_logf(fabsf(lam));
    a.delta[n + 2 * all] = -d1;
    a.delta[n + 3 * all] = seen == 1 ? 0.f : sign * (d2 - d1);
    if (a.lam_rows) a.delta[n + 4 * all] = -sign;
  }
  const float up = power_of_2(lift), d1up = d1 * up, d2up = d2 * up;
  auto tile = [&](int j, auto buffer) {
    constexpr int cur = decltype(buffer)::value;   // known: the buffers' offsets go into the reads' own
    const int k0 = j * TILE;
    if (j + 1 < ntiles) {
      kf.fetch(k0 + TILE, len - 1, cur ? K0 : K1);
      vf.fetch(k0 + TILE, len - 1, cur ? V0 : V1);
    }
    if (k0 < wmost) {
      constexpr int kt = cur ? K1 : K0;
      constexpr int vt = cur ? V1 : V0;
      const bool edge = k0 + TILE > wleast;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x16 da = zero16();
#pragma unroll
        for (int ks = 0; ks < DV / 16; ++ks) da = Mat<T>::mfma(vrows.at(vt, 32 * i, ks), g.f[ks], da);
#pragma unroll
        for (int map = 0; map < 2; ++map) {
          f32x16 s = zero16();
#pragma unroll
          for (int ks = 0; ks < DH / 16; ++ks) s = Mat<T>::mfma(krows.at(kt, 32 * i, map * (DH / 16) + ks), q[map].f[ks], s);
          if (edge) {
            const int left = seen - k0 - 4 * half;
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (32 * i + row_of(r, 0) >= left) s[r] = -INFINITY;
          }
          const float ls = map ? ls2 : ls1, d = map ? d2 : d1, dup = map ? d2up : d1up;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -ls));
            if (map) dlam = __builtin_fmaf(p, da[r], dlam);
            s[r] = p * (LIFTED<T> ? __builtin_fmaf(da[r], up, -dup) : da[r] - d);
          }
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const uint4 ds = operand<T>(s, st);
#pragma unroll
            for (int e = 0; e < QB_; ++e)
              dq[map][e] = Mat<T>::mfma(kcols.at(kt, 32 * i + 16 * st, map * DH + 32 * e), ds, dq[map][e]);
          }
        }
      }
    }
    if (j + 1 < ntiles) filled();
  };
  for (int j = 0; j < ntiles; j += 2) {
    tile(j, std::integral_constant<int, 0>());
    if (j + 1 < ntiles) tile(j + 1, std::integral_constant<int, 1>());
  }
  typedef typename Mat<T>::Cvt C;
  if (query < a.tq) {
    T* row = static_cast<T*>(a.dq) + (((int64_t)b * a.tq + query) * 2 * a.h + 2 * head) * a.dh;
#pragma unroll
    for (int map = 0; map < 2; ++map) {
      const float back = LIFTED<T> ? a.scale * power_of_2(-lift) : a.scale, f = seen == 1 ? 0.f : map ? -lam * back : back;
#pragma unroll
      for (int e = 0; e < QB_; ++e)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int col = 32 * e + 8 * k + 4 * half;
          const f32x16& v = dq[map][e];
          if (col < a.dh)
            *reinterpret_cast<uint2*>(row + map * a.dh + col) =
                make_uint2(C::pack2(v[4 * k] * f, v[4 * k + 1] * f), C::pack2(v[4 * k + 2] * f, v[4 * k + 3] * f));
        }
    }
  }
  if (!a.dlam) return;
  dlam = query < a.tq ? -other_half(dlam, true) : 0.f;
  if (a.lam_rows) {
    if (query < a.tq && half == 0) a.dlam[((int64_t)b * a.tq + query) * a.h + head] = dlam;
    return;
  }
  dlam = lanes_reduce(dlam, 32, AddOp());
  float* s_dlam = reinterpret_cast<float*>(lds_block);
  __syncthreads();   // the last tile has been read
  if (lane == 0) s_dlam[wave] = dlam;
  __syncthreads();
  if (threadIdx.x == 0) a.dlam[(int64_t)head * (a.b * blocks) + b * blocks + qblock] = (s_dlam[0] + s_dlam[1]) + (s_dlam[2] + s_dlam[3]);
}

// dlam: `n` parts of each of `outs` results in a row, summed in order by 256 lanes, then a tree; or (n 1) only converted
template <typename T> __global__ __launch_bounds__(WG) void k_diff_dlam(const float* __restrict__ part, int64_t n, int64_t outs, T* __restrict__ out) {
  __shared__ float s[WG];
  const int tid = (int)threadIdx.x;
  if (n == 1) {
    for (int64_t i = (int64_t)blockIdx.x * WG + tid; i < outs; i += (int64_t)gridDim.x * WG) st1(out + i, part[i]);
    return;
  }
  float acc = 0.f;
  for (int64_t i = tid; i < n; i += WG) acc += part[blockIdx.x * n + i];
  s[tid] = acc;
  __syncthreads();
  for (int w = WG / 2; w > 0; w >>= 1) {
    if (tid < w) s[tid] += s[tid + w];
    __syncthreads();
  }
  if (tid == 0) st1(out + blockIdx.x, s[0]);
}

// ---------------------------------------------------------------------------------------------------------------
// backward: dk and dv. 128 keys of a head of keys per workgroup, 32 a wave, over the queries of its group's heads one after
// another, or a part of them: the first keys of a causal sequence have the most queries, and a group's heads add to them; parts of
// at most `limit` tiles, their fp32 results summed by k_diff_kv_sum, leave no CU behind the others.
// Here the scores' rows are queries, whose four or five numbers come from LDS for every row a lane has: by
// v_mfma_f32_16x16x32 a lane has 4 of 16 rows, not 16 of 32, and half as much is read for them, and held. With s = -1 where lam < 0,
// else 1, and P2' = |lam| P2 = exp2(c s2 - (lse2 - log2 |lam|)), the numbers are lse1, lse2 - log2 |lam|, -D1 (where the product
// for dA begins), s (D2 - D1) and -s, so that
//   P = P1 - s P2',   dS1 = P1 (dA - D1),   dS2 = P2' (s (D2 - D1) - s (dA - D1))
// 8 x 2048 tokens, 6 heads of 64|128: 148 us, 103 GFLOP at 0.70 PFLOP/s (vector units 0.36 of the time, matrix cores 0.32); 2 x 4096, 16
// heads on 4: 437 us and 13 for the parts' sum. The values in LDS, not in registers, leave two waves to a SIMD without spills; 64 keys
// to a wave at one wave took 285 us, scratch loads between the tiles' loads, which they wait for, 188 to 221.
// ---------------------------------------------------------------------------------------------------------------
constexpr int KVT = 32;   // queries of a tile
template <typename T, int W> struct Kept16 {   // a wave's 32 rows as B operands: row 16 n + l mod 16, columns 32 ks + 8 (l / 16) .. + 8
  uint4 f[2][W / 32];
  __device__ __forceinline__ void load(int n, const T* row, int width, bool there) {   // zeros past `width`, and for no row
    const int g = ((int)threadIdx.x & 63) >> 4;
#pragma unroll
    for (int ks = 0; ks < W / 32; ++ks) {
      const int c = 32 * ks + 8 * g;
      f[n][ks] = only(c < width && there, *reinterpret_cast<const uint4*>(row + min(c, width - 8)));
    }
  }
};

// the tiles of queries that a block of keys has in one head, from which on, and its parts
struct KvTiles { int first, n, parts; };
__device__ __forceinline__ KvTiles kv_tiles(const Diff& a, int b, int kb) {
  const int first_q = a.causal ? max(kb - start_of(a, b), 0) : 0, first = first_q / KVT;
  const int n = kb < length_of(a, b) && first_q < a.tq ? (a.tq + KVT - 1) / KVT - first : 0;
  return {first, n, min(a.splits, max(1, (n * (a.h / a.hk) + a.chunk - 1) / a.chunk))};
}

template <typename T, int DH, int DV, bool TOKEN>   // TOKEN: lam differs between queries
__global__ __launch_bounds__(WG) __attribute__((amdgpu_waves_per_eu((waves_bwd<DH, DV>())))) void k_diff_bwd_kv(const Diff a) {
  extern __shared__ __align__(16) char lds_block[];
  constexpr int QT = KVT * 2 * DH, GT = KVT * DV, KB = DH / 16, VB = DV / 16, NUMBERS = TOKEN ? 5 : 4;
  // two tiles of queries and of dy, this workgroup's values, and twice lse1, lse2, D1, D2, lam of the tile's queries
  constexpr int Q0 = 0, Q1 = 2 * QT, G0 = 4 * QT, G1 = 4 * QT + 2 * GT, VALUES = 4 * (QT + GT), R0 = VALUES + 2 * QB * DV, R1 = R0 + 4 * NUMBERS * KVT;
  const int tid = (int)threadIdx.x, lane = tid & 63, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = a.h / a.hk, blocks = (a.tk + QB - 1) / QB;
  Work wk;
  if (!work_of((int)blockIdx.x, a.b * a.hk, a.splits, blocks, wk)) return;
  const int kb = wk.block * QB, b = wk.item / a.hk, hk = wk.item - b * a.hk;
  const KvTiles kv = kv_tiles(a, b, kb);
  if (wk.g >= kv.parts) return;
  const int len = length_of(a, b), start = start_of(a, b);
  const int w0 = kb + 32 * wave;
  Kept16<T, DH> k[2];
  int from[2];   // the first query that sees the lane's keys
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int key = w0 + 16 * n + (lane & 15), krow = min(key, a.tk - 1);
    const bool there = key < len;   // what is past the length is not read into anything: a NaN would reach a product of zeros
    const T* kp = static_cast<const T*>(a.k.p) + b * a.k.b + krow * a.k.t + 2 * hk * a.k.h;
    k[0].load(n, kp, a.dh, there);
    k[1].load(n, kp + a.k.h, a.dh, there);
    from[n] = !there ? 0x7fffffff : a.causal ? max(key - start, 0) : 0;
  }
  const Rows16<2 * DH> qrows;
  const Cols16<2 * DH> qcols;
  const auto grows = of_width<Rows16, DV>(qrows);
  const auto gcols = of_width<Cols16, DV>(qcols);
  f32x4 dk[2][KB][2], dv[VB][2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
#pragma unroll
    for (int d = 0; d < KB; ++d) dk[0][d][n] = dk[1][d][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < VB; ++d) dv[d][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int per = (kv.n * groups + kv.parts - 1) / kv.parts, it0 = wk.g * per, it1 = min(it0 + per, kv.n * groups);
  const int64_t all = (int64_t)a.b * a.h * a.tq;
  const T* qbase = static_cast<const T*>(a.q.p) + b * a.q.b + 2 * hk * groups * a.q.h;
  const T* gbase = static_cast<const T*>(a.dy) + ((int64_t)b * a.tq * a.h + hk * groups) * a.dv;
  Fill<T, 2 * DH, 2, KVT, WG> qf(qbase, a.q.t, a.q.h, a.dh);
  Fill<T, DV, 1, KVT, WG> gf(gbase, (int64_t)a.h * a.dv, 0, a.dv);
  auto fetch = [&](int row0, int head, int s_q, int s_g, int s_row) {   // a tile of one of the group's heads
    qf.base = qbase + 2 * head * a.q.h;
    gf.base = gbase + head * a.dv;
    qf.fetch(row0, a.tq - 1, s_q);
    gf.fetch(row0, a.tq - 1, s_g);
    // a wave loads 32 of two of the numbers
    const float* of = a.delta + ((int64_t)b * a.h + hk * groups + head) * a.tq + row0;
    const uint32_t row = 4u * (uint32_t)min(lane & 31, a.tq - 1 - row0);
    if (wave < 2) load_lds4(of + 2 * wave * all, row + (lane & 32 ? (uint32_t)(4 * all) : 0u), s_row + wave * 8 * KVT);
    if (TOKEN && wave == 2 && lane < 32) load_lds4(of + 4 * all, row, s_row + 16 * KVT);
  };
  const int mine = kept(wave * 64 * DV);   // the offset of the wave's values
  const int numbers = kept(16 * grp);
  int head = kv.n ? it0 / kv.n : 0, at = kv.first + it0 - head * kv.n;
  auto minus_of = [&](int head) {   // -s of a head, waited for here and not where it is used
    const float lam = TOKEN || head >= groups ? 0.f : lam_at<T>(a, b, 0, hk * groups + head);
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(lam < 0.f ? 1.f : -1.f)));
  };
  float next_minus = minus_of(head);
  float up = 1.f, back = 1.f, up_p = 1.f, back_p = 1.f;   // what dA - D and the combined map are multiplied by, and the sums back
  if constexpr (LIFTED<T>) {
    float size = 0.f, lam = 1.f;
    const int tiles = (a.tq + QB - 1) / QB * (QB / KVT);
    for (int it = it0 + lane; it < it1; it += 64) {
      const int of = it / kv.n;
      const float2 e = a.sizes[((int64_t)b * a.h + hk * groups + of) * tiles + kv.first + it - of * kv.n];
      size = fmaxf(size, e.x);
      lam = fmaxf(lam, e.y);
    }
    const int n = __builtin_amdgcn_readfirstlane(lift_of(2.f * lanes_reduce(size, 64, MaxOp()) * norm_of(a, wk.item, len)));
    const int n_p = __builtin_amdgcn_readfirstlane(lift_of(2.f * lanes_reduce(lam, 64, MaxOp())));   // |P1 - lam P2| <= 2 max(1, |lam|)
    up = power_of_2(n);
    back = power_of_2(-n);
    up_p = power_of_2(n_p);
    back_p = power_of_2(-n_p);
  }
  if (it0 < it1) {
    const Fill<T, DV, 1, QB, WG> vf(static_cast<const T*>(a.v.p) + b * a.v.b + hk * a.v.h, a.v.t, 0, a.dv);
    vf.fetch(kb, len - 1, VALUES);
    fetch(at * KVT, head, Q0, G0, R0);
  }
  filled();
  if (a.dv < DV) {   // the values' columns past the last repeat some, as dy's do: zeros in their place
    for (int i = tid; i < QB * (DV / 8); i += WG) {
      const int r = i / (DV / 8), p = i % (DV / 8);
      if (8 * p >= a.dv) *reinterpret_cast<uint4*>(lds_block + VALUES + 2 * (r * DV + 8 * (p ^ swizzle<DV>(r)))) = make_uint4(0u, 0u, 0u, 0u);
    }
    __syncthreads();
  }
  auto tile = [&](int it, auto buffer) {
    constexpr int cur = decltype(buffer)::value;
    const int q0 = at * KVT;
    const float minus = next_minus;
    if (++at == kv.first + kv.n) {
      at = kv.first;
      ++head;
      next_minus = minus_of(head);
    }
    if (it + 1 < it1) fetch(at * KVT, head, cur ? Q0 : Q1, cur ? G0 : G1, cur ? R0 : R1);
    // the keys that the tile's last and first queries see: whether any of this wave's is among them, and whether all are
    if (w0 < seen_by(a, min(q0 + KVT, a.tq) - 1, start, len)) {
      constexpr int qt = cur ? Q1 : Q0, gt = cur ? G1 : G0, rt = cur ? R1 : R0;
      const bool edge = w0 + 32 > seen_by(a, q0, start, len) || q0 + KVT > a.tq;
      uint2 pd[2][2], p1[2][2], p2[2][2];   // [16 queries][16 keys]: P1 - lam P2, dS1, dS2
      f32x4 da[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) da[u][0] = da[u][1] = lds_at<f32x4>(numbers + rt + 4 * (2 * KVT + 16 * u));
#pragma unroll
      for (int ks = 0; ks < DV / 32; ++ks) {
        uint4 x[2], y[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[e] = grows.at(gt, 16 * e, ks);
          y[e] = grows.at(mine + VALUES, 16 * e, ks);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int n = 0; n < 2; ++n) da[u][n] = Mat<T>::mfma16(x[u], y[n], da[u][n]);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r0 = 16 * u;
        f32x4 s1[2], s2[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) s1[n] = s2[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < DH / 32; ++ks) {
          const uint4 x = qrows.at(qt, r0, ks), y = qrows.at(qt, r0, DH / 32 + ks);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            s1[n] = Mat<T>::mfma16(x, k[0].f[n][ks], s1[n]);
            s2[n] = Mat<T>::mfma16(y, k[1].f[n][ks], s2[n]);
          }
        }
        if (edge) {
          const int here = q0 + 4 * grp, left = a.tq - here;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (r0 + r >= left || here + r0 + r < from[n]) s1[n][r] = s2[n][r] = -INFINITY;
#pragma unroll
          for (int r = 0; r < 4; ++r)   // the probability of a query's only key does not change
            if (seen_by(a, here + r0 + r, start, len) == 1) da[u][0][r] = da[u][1][r] = 0.f;
        }
        auto number = [&](int e) { return lds_at<f32x4>(numbers + rt + 4 * (e * KVT + r0)); };
        const f32x4 ls1 = number(0), ls2 = number(1);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s1[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s1[n][r], a.c, -ls1[r]));
            s2[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s2[n][r], a.c, -ls2[r]));
          }
        f32x4 sg;
        if (TOKEN) sg = number(NUMBERS - 1);
        f32x4 d = number(3);
        if (LIFTED<T>) d *= up;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float q1 = s1[n][r], q2 = s2[n][r], x = LIFTED<T> ? da[u][n][r] * up : da[u][n][r], m = TOKEN ? sg[r] : minus;
            da[u][n][r] = __builtin_fmaf(m, q2, q1);
            s1[n][r] = q1 * x;
            s2[n][r] = q2 * __builtin_fmaf(m, x, d[r]);
          }
          pd[u][n] = packed4<T>(LIFTED<T> ? da[u][n] * up_p : da[u][n]);
          p1[u][n] = packed4<T>(s1[n]);
          p2[u][n] = packed4<T>(s2[n]);
        }
      }
      in_order();
      auto both = [](const uint2 (&p)[2][2], int n) { return make_uint4(p[0][n].x, p[0][n].y, p[1][n].x, p[1][n].y); };
#pragma unroll
      for (int d = 0; d < VB; ++d) {
        const uint4 x = gcols.at(gt, 0, 16 * d);
#pragma unroll
        for (int n = 0; n < 2; ++n) dv[d][n] = Mat<T>::mfma16(x, both(pd, n), dv[d][n]);
      }
#pragma unroll
      for (int d = 0; d < KB; ++d) {
        const uint4 x = qcols.at(qt, 0, 16 * d), y = qcols.at(qt, 0, DH + 16 * d);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          dk[0][d][n] = Mat<T>::mfma16(x, both(p1, n), dk[0][d][n]);
          dk[1][d][n] = Mat<T>::mfma16(y, both(p2, n), dk[1][d][n]);
        }
      }
    }
    if (it + 1 < it1) filled();
  };
  for (int it = it0; it < it1; it += 2) {
    tile(it, std::integral_constant<int, 0>());
    if (it + 1 < it1) tile(it + 1, std::integral_constant<int, 1>());
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int key = w0 + 16 * n + (lane & 15);
    if (key >= a.tk) continue;
    if (kv.parts > 1) {   // [dk1 | dk2 | dv] of a key, not scaled
      float* row = a.part + ((((int64_t)wk.item * blocks + wk.block) * a.splits + wk.g) * QB + (key - kb)) * (2 * a.dh + a.dv);
#pragma unroll
      for (int d = 0; d < KB; ++d) {
        const int col = 16 * d + 4 * grp;
        if (col < a.dh) {
          *reinterpret_cast<f32x4*>(row + col) = LIFTED<T> ? dk[0][d][n] * back : dk[0][d][n];
          *reinterpret_cast<f32x4*>(row + a.dh + col) = LIFTED<T> ? dk[1][d][n] * back : dk[1][d][n];
        }
      }
#pragma unroll
      for (int d = 0; d < VB; ++d) {
        const int col = 16 * d + 4 * grp;
        if (col < a.dv) *reinterpret_cast<f32x4*>(row + 2 * a.dh + col) = LIFTED<T> ? dv[d][n] * back_p : dv[d][n];
      }
      continue;
    }
    const float scale = LIFTED<T> ? a.scale * back : a.scale;
    T* krow = static_cast<T*>(a.dk) + (((int64_t)b * a.tk + key) * 2 * a.hk + 2 * hk) * a.dh;
    T* vrow = static_cast<T*>(a.dval) + (((int64_t)b * a.tk + key) * a.hk + hk) * a.dv;
#pragma unroll
    for (int d = 0; d < KB; ++d) {
      const int col = 16 * d + 4 * grp;
      if (col < a.dh) {
        *reinterpret_cast<uint2*>(krow + col) = packed4<T>(dk[0][d][n] * scale);
        *reinterpret_cast<uint2*>(krow + a.dh + col) = packed4<T>(dk[1][d][n] * scale);
      }
    }
#pragma unroll
    for (int d = 0; d < VB; ++d) {
      const int col = 16 * d + 4 * grp;
      if (col < a.dv) *reinterpret_cast<uint2*>(vrow + col) = packed4<T>(LIFTED<T> ? dv[d][n] * back_p : dv[d][n]);
    }
  }
}

// the parts of a block of keys, in order, scaled and rounded: SUM_ROWS keys of a block per workgroup, four columns a lane
constexpr int SUM_ROWS = 8;
template <typename T> __global__ __launch_bounds__(WG) void k_diff_kv_sum(const Diff a) {
  const int blocks = (a.tk + QB - 1) / QB, item = (int)blockIdx.x / blocks, kb = ((int)blockIdx.x - item * blocks) * QB;
  const int b = item / a.hk, hk = item - b * a.hk, parts = kv_tiles(a, b, kb).parts, row = 2 * a.dh + a.dv, per = row / 4;
  if (parts == 1) return;
  const float* p = a.part + (int64_t)blockIdx.x * a.splits * QB * row;
  const int k0 = (int)blockIdx.y * SUM_ROWS, k1 = min(min(k0 + SUM_ROWS, QB), a.tk - kb);
  for (int i = k0 * per + (int)threadIdx.x; i < k1 * per; i += WG) {
    const int key = i / per, col = 4 * (i - key * per);
    const float* x = p + (int64_t)key * row + col;
    f32x4 t = *reinterpret_cast<const f32x4*>(x);
    for (int s = 1; s < parts; ++s) t += *reinterpret_cast<const f32x4*>(x + (int64_t)s * QB * row);
    if (col < 2 * a.dh)
      *reinterpret_cast<uint2*>(static_cast<T*>(a.dk) + (((int64_t)b * a.tk + kb + key) * 2 * a.hk + 2 * hk) * a.dh + col) = packed4<T>(t * a.scale);
    else
      *reinterpret_cast<uint2*>(static_cast<T*>(a.dval) + (((int64_t)b * a.tk + kb + key) * a.hk + hk) * a.dv + col - 2 * a.dh) = packed4<T>(t);
  }
}

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int launched() { return (int)hipGetLastError(); }

#define DIFF_SWITCH(DT, DHS, DVS, ...)                                                                                        \
  if ((DT) == LDR_BF16) { typedef bf16_t T; DIFF_SIZES(DHS, DVS, __VA_ARGS__) }                                                \
  else { typedef _Float16 T; DIFF_SIZES(DHS, DVS, __VA_ARGS__) }
#define DIFF_SIZES(DHS, DVS, ...)                                                                                             \
  if ((DHS) <= 64 && (DVS) <= 64) { constexpr int DH = 64, DV = 64; __VA_ARGS__; }                                             \
  else if ((DHS) <= 64 && (DVS) <= 128) { constexpr int DH = 64, DV = 128; __VA_ARGS__; }                                      \
  else if ((DVS) <= 128) { constexpr int DH = 128, DV = 128; __VA_ARGS__; }                                                    \
  else { constexpr int DH = 128, DV = 256; __VA_ARGS__; }

constexpr int64_t MOST = 0x7fffff;
int diff_args(const lmo_diff_shape* s, const lmo_strides* q, const lmo_strides* k, const lmo_strides* v, int dtype) {
  if (dtype != LDR_BF16 && dtype != LDR_F16) return LDR_E_DTYPE;
  if (!s || !q || !k || !v) return LDR_E_ARG;
  if (s->b < 0 || s->tq < 0 || s->tk < 1 || s->hk < 1 || s->h < s->hk || s->h % s->hk || s->b * s->h > MOST || s->tq >= (1 << 30) ||
      s->tk >= (1 << 30))
    return LDR_E_ARG;
  if (s->b * s->h * s->tq >= (1 << 29)) return LDR_E_SHAPE;   // a number of each within 32 bits of bytes
  if (s->dh < 8 || s->dh > 128 || s->dh % 8 || s->dv < 8 || s->dv > 256 || s->dv % 8) return LDR_E_SHAPE;
  if (!(s->scale > 0.f) || !(s->scale < INFINITY)) return LDR_E_ARG;
  for (const lmo_strides* t : {q, k, v}) {
    if (!t->p && s->b * s->tq > 0) return LDR_E_ARG;
    if (!al16(t->p) || t->b % 8 || t->t % 8 || t->h % 8) return LDR_E_ALIGN;
    if (t->b < 0 || t->t < 0 || t->h < 0 || t->t > (1 << 23) || t->h > (1 << 23)) return LDR_E_SHAPE;   // 64 rows within 32 bits
  }
  return LDR_OK;
}
Diff diff_of(const lmo_diff_shape* s, const lmo_strides* q, const lmo_strides* k, const lmo_strides* v, const lmo_strides* lam, int lam32,
             const int32_t* lengths, const int32_t* starts) {
  Diff a{};
  a.q = {q->p, q->b, q->t, q->h};
  a.k = {k->p, k->b, k->t, k->h};
  a.v = {v->p, v->b, v->t, v->h};
  a.lam = {lam->p, lam->b, lam->t, lam->h};
  a.lengths = lengths;
  a.starts = starts;
  a.b = (int)s->b;
  a.tq = (int)s->tq;
  a.tk = (int)s->tk;
  a.h = (int)s->h;
  a.hk = (int)s->hk;
  a.dh = (int)s->dh;
  a.dv = (int)s->dv;
  a.causal = s->causal;
  a.lam32 = lam32;
  a.scale = s->scale;
  a.c = s->scale * LOG2E;
  return a;
}
inline int64_t blocks_of(int64_t t) { return (t + QB - 1) / QB; }
inline bool few(const lmo_diff_shape* s) { return s->tq * (s->h / s->hk) <= FEW; }
// Chunks of the keys: enough workgroups for the CUs twice over, chunks of 256 keys at least. Blocks of 64 queries (not `few`: the rows
// of the kernel of few queries) are split where that makes three chunks at least: 3 x 333 new tokens over 1001 keys, 6 heads, 26.5 us
// whole and 19.4 + 4.8 for the join in three; 3 x 683 tokens, 4 heads of 128|256, 33.2 whole and 23.2 + 9.7 in two (in one part).
struct Chunks { int64_t splits, chunk; };
inline Chunks chunks_of(const lmo_diff_shape* s, bool few) {
  const int64_t items = few ? s->b * s->hk : s->b * s->h * ((s->tq + FQ - 1) / FQ), most = s->tk / 256;
  const int64_t want = few ? (512 + items - 1) / (items > 0 ? items : 1) : items > 0 ? 512 / items : 1;
  int64_t n = want < most ? want : most;
  n = n < (few ? 1 : 3) ? 1 : n > MOST_CHUNKS ? MOST_CHUNKS : n;
  const int64_t chunk = ((s->tk + n - 1) / n + NT - 1) / NT * NT;
  return {s->tk < 1 ? 1 : (s->tk + chunk - 1) / chunk, chunk};
}
// parts of the tiles of queries for dk and dv: those of a causal sequence (positions and lengths are the kernel's to know), so that
// the longest takes little more than its share of what the CUs hold at once
struct Parts { int64_t splits, limit; };
inline Parts kv_parts(const lmo_diff_shape* s) {
  const int64_t blocks = blocks_of(s->tk), tiles = (s->tq + KVT - 1) / KVT, groups = s->h / s->hk, slots = s->dh <= 64 && s->dv <= 128 ? 512 : 256;
  int64_t all = 0, most = 0;
  for (int64_t i = 0; i < blocks; ++i) {
    const int64_t from = s->causal ? i * QB - (s->tk - s->tq) : 0, n = from < s->tq ? (tiles - (from > 0 ? from / KVT : 0)) * groups : 0;
    all += n;
    most = n > most ? n : most;
  }
  const int64_t share = (all * s->b * s->hk + slots - 1) / slots;
  int64_t limit = share + (share + 2) / 3;
  limit = limit < 16 ? 16 : limit;
  const int64_t splits = (most + limit - 1) / limit;
  return {splits < 1 ? 1 : splits > 16 ? 16 : splits, limit};
}
// the backward's scratch memory, in floats from its start
struct BwdScratch { int64_t dlam, norms, sizes, part, all; };
inline BwdScratch bwd_scratch(const lmo_diff_shape* s, int lam_kind, const Parts& kv) {
  const bool token = lam_kind == LMO_LAM_TOKEN;
  BwdScratch at;
  at.dlam = (token ? 5 : 4) * s->b * s->h * s->tq;
  at.norms = at.dlam + s->b * s->h * (token ? s->tq : blocks_of(s->tq));
  at.sizes = (at.norms + s->b * s->hk * blocks_of(s->tk) + 3) / 4 * 4;
  at.part = at.sizes + s->b * s->h * blocks_of(s->tq) * (QB / KVT) * 2;   // 8 floats a block of queries
  at.all = at.part + (kv.splits > 1 ? s->b * s->hk * blocks_of(s->tk) * kv.splits * QB * (2 * s->dh + s->dv) : 0);
  return at;
}
inline int padded_dv(const lmo_diff_shape* s) { return s->dv <= 64 && s->dh <= 64 ? 64 : s->dv <= 128 ? 128 : 256; }

}  // namespace

extern "C" {

int64_t lmo_diff_attn_scratch(const lmo_diff_shape* s, int record) {
  if (!s || s->hk < 1 || s->b < 1 || s->tq < 1) return 0;
  const Chunks n = chunks_of(s, !record && few(s));
  return n.splits == 1 ? 0 : s->b * s->h * s->tq * n.splits * (2 * padded_dv(s) + 4);
}

int lmo_diff_attn_fwd(const lmo_strides* q, const lmo_strides* k, const lmo_strides* v, const lmo_strides* lam, int lam32,
                      const int32_t* lengths, const int32_t* starts, void* out, void* second, float* lse, float* scratch,
                      const lmo_diff_shape* s, int dtype, void* stream) {
  int e = diff_args(s, q, k, v, dtype);
  if (e) return e;
  if (s->b * s->tq == 0) return LDR_OK;
  if (!lam || !lam->p || !out || !second != !lse) return LDR_E_ARG;
  if (!al16(out) || !al16(second) || !al16(scratch)) return LDR_E_ALIGN;
  Diff a = diff_of(s, q, k, v, lam, lam32, lengths, starts);
  a.out = out;
  a.second = second;
  a.lse = lse;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool fewer = !lse && few(s);
  const Chunks n = chunks_of(s, fewer);
  if (n.splits > 1 && !scratch) return LDR_E_ARG;
  a.splits = (int)n.splits;
  a.chunk = (int)n.chunk;
  a.part = scratch;
  const int64_t grid = (fewer ? s->b * s->hk : s->b * s->h * ((s->tq + FQ - 1) / FQ)) * n.splits;
  if (grid > 0x7fffffff) return LDR_E_SHAPE;
  DIFF_SWITCH(dtype, s->dh, s->dv, {
    if (fewer) {
      constexpr int bytes = few_lds<DH, DV>();
      if ((e = ALLOW_LDS(bytes, k_diff_few<T, DH, DV>))) return e;
      hipLaunchKernelGGL((k_diff_few<T, DH, DV>), dim3((unsigned)grid), dim3(WG), bytes, st, a);
    } else if (n.splits > 1) {
      constexpr int bytes = fwd_lds<DH, DV>();
      if ((e = ALLOW_LDS(bytes, k_diff_fwd<T, DH, DV, true>))) return e;
      hipLaunchKernelGGL((k_diff_fwd<T, DH, DV, true>), dim3((unsigned)grid), dim3(FL), bytes, st, a);
    } else {
      constexpr int bytes = fwd_lds<DH, DV>();
      if ((e = ALLOW_LDS(bytes, k_diff_fwd<T, DH, DV, false>))) return e;
      hipLaunchKernelGGL((k_diff_fwd<T, DH, DV, false>), dim3((unsigned)grid), dim3(FL), bytes, st, a);
    }
    if ((e = launched())) return e;
    const int64_t rows = s->b * s->h * s->tq;
    if (n.splits > 1 && rows <= SHARED_ROWS) {
      hipLaunchKernelGGL((k_diff_join<T, DV, true>), dim3((unsigned)rows), dim3(WG), 0, st, a);
    } else if (n.splits > 1) {
      hipLaunchKernelGGL((k_diff_join<T, DV, false>), dim3((unsigned)((rows * (DV / 4) + WG - 1) / WG)), dim3(WG), 0, st, a);
    }
  })
  return launched();
}

int64_t lmo_diff_attn_bwd_scratch(const lmo_diff_shape* s, int lam_kind) {
  if (!s || s->b < 1 || s->tq < 1 || s->tk < 1 || s->hk < 1 || s->h < s->hk) return 0;
  return bwd_scratch(s, lam_kind, kv_parts(s)).all;
}

int lmo_diff_attn_bwd(const lmo_strides* q, const lmo_strides* k, const lmo_strides* v, const lmo_strides* lam, int lam32,
                      const int32_t* lengths, const int32_t* starts, const void* out, const void* second, const float* lse,
                      const void* dy, void* dq, void* dk, void* dv, void* dlam, int lam_kind, float* scratch,
                      const lmo_diff_shape* s, int dtype, void* stream) {
  int e = diff_args(s, q, k, v, dtype);
  if (e) return e;
  if (lam_kind < LMO_LAM_LAYER || lam_kind > LMO_LAM_TOKEN) return LDR_E_ARG;
  if (s->tq > 1 && s->h * s->dv > (1 << 26)) return LDR_E_SHAPE;   // 32 rows of dy within 32 bits of bytes
  if (s->b * s->tq == 0) return LDR_OK;
  if (!lam || !lam->p || !out || !second || !lse || !dy || !dq || !scratch || !dk != !dv) return LDR_E_ARG;
  for (const void* p : {out, second, dy, (const void*)dq, (const void*)dk, (const void*)dv, (const void*)scratch})
    if (!al16(p)) return LDR_E_ALIGN;
  Diff a = diff_of(s, q, k, v, lam, lam32, lengths, starts);
  a.out = const_cast<void*>(out);
  a.second = const_cast<void*>(second);
  a.lse = const_cast<float*>(lse);
  a.dy = dy;
  a.dq = dq;
  a.dk = dk;
  a.dval = dv;
  a.delta = scratch;
  const Parts kv = kv_parts(s);
  const BwdScratch at = bwd_scratch(s, lam_kind, kv);
  a.dlam = dlam ? scratch + at.dlam : nullptr;
  a.norms = scratch + at.norms;
  a.sizes = reinterpret_cast<float2*>(scratch + at.sizes);
  a.splits = (int)kv.splits;
  a.chunk = (int)kv.limit;
  a.part = scratch + at.part;
  a.lam_rows = lam_kind == LMO_LAM_TOKEN;
  const int64_t qblocks = blocks_of(s->tq), grid_q = s->b * s->h * qblocks, grid_k = s->b * s->hk * blocks_of(s->tk) * kv.splits;
  if (grid_q > 0x7fffffff || grid_k > 0x7fffffff) return LDR_E_SHAPE;
  hipStream_t st = static_cast<hipStream_t>(stream);
  DIFF_SWITCH(dtype, s->dh, s->dv, {
    if constexpr (LIFTED<T>) {
      hipLaunchKernelGGL((k_diff_bwd_norms<T, DV>), dim3((unsigned)(grid_k / kv.splits)), dim3(WG), 0, st, a);
      if ((e = launched())) return e;
    }
    constexpr int bytes = 2 * TILE * (2 * DH + DV) * 2;
    if ((e = ALLOW_LDS(bytes, k_diff_bwd_q<T, DH, DV>))) return e;
    hipLaunchKernelGGL((k_diff_bwd_q<T, DH, DV>), dim3((unsigned)grid_q), dim3(WG), bytes, st, a);
    if ((e = launched())) return e;
    if (dlam) {
      const int64_t all = s->b * s->tq * s->h, outs = lam_kind == LMO_LAM_TOKEN ? all : lam_kind == LMO_LAM_HEAD ? s->h : 1;
      const int64_t n = lam_kind == LMO_LAM_TOKEN ? 1 : lam_kind == LMO_LAM_HEAD ? s->b * qblocks : s->h * s->b * qblocks;
      const int64_t grid = lam_kind == LMO_LAM_TOKEN || n == 1 ? (outs + WG - 1) / WG : outs;
      const unsigned g = (unsigned)(grid < 4096 || n != 1 ? grid : 4096);
      if (lam32) hipLaunchKernelGGL(k_diff_dlam<float>, dim3(g), dim3(WG), 0, st, a.dlam, n, outs, static_cast<float*>(dlam));
      else hipLaunchKernelGGL(k_diff_dlam<T>, dim3(g), dim3(WG), 0, st, a.dlam, n, outs, static_cast<T*>(dlam));
      if ((e = launched())) return e;
    }
    constexpr int kv_bytes = 2 * (2 * KVT * (2 * DH + DV) + QB * DV) + 2 * 5 * KVT * 4;
    if (dk && lam_kind == LMO_LAM_TOKEN) {
      if ((e = ALLOW_LDS(kv_bytes, k_diff_bwd_kv<T, DH, DV, true>))) return e;
      hipLaunchKernelGGL((k_diff_bwd_kv<T, DH, DV, true>), dim3((unsigned)grid_k), dim3(WG), kv_bytes, st, a);
    } else if (dk) {
      if ((e = ALLOW_LDS(kv_bytes, k_diff_bwd_kv<T, DH, DV, false>))) return e;
      hipLaunchKernelGGL((k_diff_bwd_kv<T, DH, DV, false>), dim3((unsigned)grid_k), dim3(WG), kv_bytes, st, a);
    }
    if (dk && kv.splits > 1) {
      if ((e = launched())) return e;
      hipLaunchKernelGGL(k_diff_kv_sum<T>, dim3((unsigned)(grid_k / kv.splits), QB / SUM_ROWS), dim3(WG), 0, st, a);
    }
  })
  return launched();
}

}  // extern "C"
