// loopback_ffn.hip -- MI355X (gfx950, CDNA4) kernels of the gated feed-forward block on the matrix cores: one tiled product
// with the block's epilogues.
//
// A product is C[q][p] = sum_k P(p, k) Q(q, k): p the contiguous dimension of the result, q its rows (tokens, or a weight's
// output rows). Each operand lies in memory either by rows of k ("ROW": index i at i * ld, k contiguous) or by rows of the
// index ("COL": k at k * ld, the index contiguous), so the forward (x W^T), the input gradient (dy W) and the weight
// gradient (dy^T x) are the same kernel without a transposed copy of anything.
//
// Operands go through v_mfma_f32_32x32x16 (bf16 or fp16): lane l holds row (P) or column (Q) l mod 32 at k = 8 (l / 32) .. + 8;
// of the 32 x 32 result it holds column l mod 32 and, in register r, row 4 (l / 32) + r mod 4 + 8 (r / 4): four consecutive p of
// one q, which one exchange of lane halves makes eight (a 16-byte store). Tiles of 64 k sit in LDS twice, the next one filled
// by direct global -> LDS loads while one is worked on. Such loads write 64 lanes' 16 bytes in order, so the tiles have no
// padding; instead the 16-byte pieces of a row are permuted: ROW tiles (128-byte rows) by (row / 2) mod 8, so that 16 rows at
// one k cover the 64 banks once, COL tiles (rows of the tile's width) by 4 (k mod 4), or 4 (k / 2 mod 2), so that the four rows a transposing read
// (ds_read_b64_tr_b16) takes together do (SQ_LDS_BANK_CONFLICT: 0 for both kinds).
//
// The matrix cores bound it: 2 q p k operations, and a 256 x 256 tile reads 64 KiB for each 64 k it multiplies. 8192 x 2048 x 5632
// in bf16: gate and up projection 314 us (1202 TFLOP/s; a library's product without the activation 352), down 151 us (125),
// input gradient 289 us (273), weight gradients 317 and 157 us (339 and 171). Smaller tiles with more workgroups to a CU took
// 5-11 % longer (the projections' gradient apart: dgated_shape), 32 k per tile in three or four buffers 4-15 % (a barrier for half the work), four waves of 128 x 128 12-17 %,
// a raised wave priority around the products 0-14 %; reloading one tile throughout, without memory traffic, only 3-5 % less.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include "loopback_block.h"
#include "loopback_read.h"
#include "device_io.h"

namespace {

constexpr int BK = 64;   // k per tile

enum Kind { ROW, COL };
enum Epi { STORE, PARTIAL, GATED, DGATED };

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

__device__ __forceinline__ f32x16 mfma(bf16_t, uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(_Float16, uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <typename T> struct CvtOf { typedef Bf16Cvt type; };
template <> struct CvtOf<_Float16> { typedef F16Cvt type; };

// ---------------------------------------------------------------------------------------------------------------
// one operand: where it lies, and its tile of ROWS indices (ROW) or columns (COL) x 64 k
// ---------------------------------------------------------------------------------------------------------------
struct Operand {   // 16-byte aligned, ld a multiple of 8; COL: every row's ld elements can be read
  const void* base;
  int64_t ld;      // elements between rows of memory
  int64_t size;    // indices
  int64_t half;    // GATED: indices per half (tile indices past its middle are those of the second half); else 0
};

template <typename T, Kind KIND, int ROWS, int LANES, bool GATED_P> struct Tile {
  static constexpr int PER = (KIND == ROW ? BK : ROWS) / 8;   // 16-byte pieces per row of the tile
  static constexpr int PASSES = ROWS * BK / 8 / LANES;
  static_assert(ROWS * BK / 8 % LANES == 0 && (KIND == ROW ? LANES / PER % 16 == 0 : ROWS % 64 == 0 && ROWS >= 128) &&
                (!GATED_P || PASSES % 2 == 0), "tile shape");

  static __device__ __forceinline__ int swizzle(int r) { return (r >> 1) & 7; }
  // COL: the block of 32 columns that row r has in the place of block 0 (rows of 192 columns begin 32 banks apart by themselves)
  static __device__ __forceinline__ int block(int r) { return ROWS % 128 ? (r >> 1) & 1 : r & 3; }
  // this lane's piece of pass i: the tile's row it is in, and which piece of memory's row is stored there
  static __device__ __forceinline__ int row(int i) { return (int)((i * LANES + threadIdx.x) / PER); }
  static __device__ __forceinline__ int piece(int i) {
    const int r = row(i), c = (int)((i * LANES + threadIdx.x) % PER);
    return KIND == ROW ? c ^ swizzle(r) : c ^ (4 * block(r));
  }
  // the operand's index of tile row r (ROW) from the tile's first index i0; past the end: the last one
  static __device__ __forceinline__ int64_t index(const Operand& o, int64_t i0, int r) {
    if (o.half) return r < ROWS / 2 ? min(i0 + r, o.half - 1) : o.half + min(i0 + r - ROWS / 2, o.half - 1);
    return min(i0 + r, o.size - 1);
  }

  // whole tiles of k from k0 on: a base that all lanes share and moves on by a tile, and each lane's byte offsets from it
  const T *base, *base2;   // GATED: of the first and the second half's indices
  uint32_t off[PASSES];
  int64_t step;
  __device__ __forceinline__ void start(const Operand& o, int64_t i0, int64_t k0) {
    const T* b = static_cast<const T*>(o.base);
    if (KIND == ROW) {
      base = b + i0 * o.ld + k0;
      base2 = base + o.half * o.ld;
      const int last = (int)min((o.half ? o.half : o.size) - 1 - i0, (int64_t)ROWS);
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int r = GATED_P && i >= PASSES / 2 ? row(i - PASSES / 2) : row(i);
        off[i] = 2 * ((uint32_t)min(r, last) * (uint32_t)o.ld + 8 * piece(i));
      }
    } else {
      base = b + k0 * o.ld + i0;
      const int last = (int)min((o.size - 1 - i0) & ~(int64_t)7, (int64_t)ROWS);
#pragma unroll
      for (int i = 0; i < PASSES; ++i) off[i] = 2 * ((uint32_t)row(i) * (uint32_t)o.ld + min(8 * piece(i), last));
    }
    step = KIND == ROW ? BK : BK * o.ld;
  }
  __device__ __forceinline__ void fetch(T* lds) {   // asynchronous: done when vmcnt says so
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const T* b = GATED_P && i >= PASSES / 2 ? base2 : base;
      __builtin_amdgcn_global_load_lds((global_void*)(reinterpret_cast<const char*>(b) + off[i]),
                                       (lds_void*)(lds + 8 * (i * LANES + wave * 64)), 16, 0, 0);
    }
    base += step;
    base2 += step;
  }
  // k from k0 to k1, fewer than BK of them: zeros past k1 and past the operand's indices
  static __device__ __forceinline__ void copy(const Operand& o, int64_t i0, int64_t k0, int64_t k1, T* lds) {
    const T* base = static_cast<const T*>(o.base);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const T* p;
      int64_t left;   // elements of this piece that exist
      if (KIND == ROW) {
        p = base + index(o, i0, row(i)) * o.ld + k0 + 8 * piece(i);
        left = k1 - k0 - 8 * piece(i);
      } else {
        p = base + (k0 + row(i)) * o.ld + i0 + 8 * piece(i);
        left = k0 + row(i) < k1 ? o.size - i0 - 8 * piece(i) : 0;
      }
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (left >= 8) {
        v = *reinterpret_cast<const uint4*>(p);
      } else if (left > 0) {
        struct { T e[8]; } e;
#pragma unroll
        for (int k = 0; k < 8; ++k) e.e[k] = k < left ? p[k] : (T)0;
        v = __builtin_bit_cast(uint4, e);
      }
      *reinterpret_cast<uint4*>(lds + 8 * (i * LANES + (int)threadIdx.x)) = v;
    }
  }
  // the matrix cores' operand: indices r0 .. r0 + 31 (r0 a multiple of 32) at k = 16 s .. 16 s + 15
  static __device__ __forceinline__ uint4 frag(const T* lds, int r0, int s) {
    const int lane = (int)threadIdx.x & 63, h = lane >> 5;
    if constexpr (KIND == ROW) {
      const int r = lane & 31;
      return *reinterpret_cast<const uint4*>(lds + (r0 + r) * BK + 8 * ((2 * s + h) ^ swizzle(r)));
    } else {
      typedef __attribute__((address_space(3))) s16x4* lds4;
      const int j = lane & 15, kr = j >> 2;
      const int col = 32 * ((r0 >> 5) ^ block(kr)) + (lane & 16) + 4 * (j & 3);
      const T* p = lds + (16 * s + 8 * h + kr) * ROWS + col;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(const_cast<T*>(p)));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(const_cast<T*>(p + 4 * ROWS)));
      const uint2 ua = __builtin_bit_cast(uint2, a), ub = __builtin_bit_cast(uint2, b);
      return make_uint4(ua.x, ua.y, ub.x, ub.y);
    }
  }
};

// ---------------------------------------------------------------------------------------------------------------
// what the backward needs of the gate and up projections: (u a'(g), a(g)) of each (token, inner column), which the
// activation's gradient is multiplied by. Kept as the upper 24 bits of their fp32 values, the rest cut off (less than 2^-15 of the
// value): 16 would double the input and
// gate/up weight gradients' squared error (three roundings instead of two). In blocks of 32 tokens x 32 columns in the
// matrix cores' own order, so both kernels move them as whole vectors: 64 lanes x 16 values, upper 16 bits as two planes of
// eight values a lane, then the next eight bits: half a block's bytes for each of the two. Stores and loads past the
// caches: gate and up projection of 8192 x 2048 x 5632 382 -> 342 us, the gradient that reads them 266 -> 238.
// ---------------------------------------------------------------------------------------------------------------
constexpr int64_t SAVED_BLOCK = 6144;
struct Saved {
  static __device__ __forceinline__ unsigned hi2(float a, float b) {   // upper halves of two words
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
  // past the caches: what is written here is not read before the backward, and then once
  static __device__ __forceinline__ void put16(uint4* p, unsigned a, unsigned b, unsigned c, unsigned d) {
    __builtin_nontemporal_store(u32x4{a, b, c, d}, reinterpret_cast<u32x4*>(p));
  }
  static __device__ __forceinline__ void put(char* block, const f32x16& v) {
    const int lane = (int)threadIdx.x & 63;
    unsigned lo[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      lo[q] = ((__float_as_uint(v[4 * q]) >> 8) & 0xffu) | (__float_as_uint(v[4 * q + 1]) & 0xff00u) |
              ((__float_as_uint(v[4 * q + 2]) & 0xff00u) << 8) | ((__float_as_uint(v[4 * q + 3]) & 0xff00u) << 16);
    uint4* p = reinterpret_cast<uint4*>(block) + lane;
    put16(p, hi2(v[0], v[1]), hi2(v[2], v[3]), hi2(v[4], v[5]), hi2(v[6], v[7]));
    put16(p + 64, hi2(v[8], v[9]), hi2(v[10], v[11]), hi2(v[12], v[13]), hi2(v[14], v[15]));
    put16(p + 128, lo[0], lo[1], lo[2], lo[3]);
  }
  struct Raw { uint4 v[6]; };   // both values of a block
  static __device__ __forceinline__ void load(const char* block, Raw& r) {
    const uint4* p = reinterpret_cast<const uint4*>(block) + ((int)threadIdx.x & 63);
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + 64 * i));
      r.v[i] = make_uint4(v.x, v.y, v.z, v.w);
    }
  }
  static __device__ __forceinline__ void get(const Raw& r, int which, float (&v)[16]) {
    const uint4 a = r.v[3 * which], b = r.v[3 * which + 1], c = r.v[3 * which + 2];
    const unsigned hi[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, lo[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const unsigned h = r & 1 ? hi[r >> 1] & 0xffff0000u : hi[r >> 1] << 16;
      const unsigned l = (r & 3) == 0 ? (lo[r >> 2] & 0xffu) << 8 : (r & 3) == 1 ? lo[r >> 2] & 0xff00u
                       : (r & 3) == 2 ? (lo[r >> 2] >> 8) & 0xff00u : (lo[r >> 2] >> 16) & 0xff00u;
      v[r] = __uint_as_float(h | l);
    }
  }
};

// ---------------------------------------------------------------------------------------------------------------
// the product
// ---------------------------------------------------------------------------------------------------------------
struct Product {
  Operand p, q;
  int64_t k, run;          // k in all, and per split
  void* out;               // [q][ldo]; PARTIAL: fp32 [split][q][ldo], ldo a multiple of 4
  int64_t ldo;
  bool out16;              // whole 16-byte vectors of the result are aligned
  void* saved;             // GATED: written (NULL: not wanted); DGATED: read
  int64_t saved_cols;      // its blocks of columns
  int tiles_p, tiles, splits, per;
  int act;                 // 0 silu, 1 gelu (tanh form)
};

// 16 registers of a result tile (column q = this lane's, rows p0 + 4 h + r mod 4 + 8 (r / 4)) to out[p0 ..], rounded:
// exchanged between the lane halves so that each lane has eight consecutive p, twice
template <typename T>
__device__ __forceinline__ void store_tile(T* row, int64_t p0, int64_t np, bool ok, bool al, const f32x16& v) {
  typedef typename CvtOf<T>::type Cvt;
  const int h = ((int)threadIdx.x >> 5) & 1;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    unsigned u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = Cvt::pack2(v[8 * g + 2 * e], v[8 * g + 2 * e + 1]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const auto sw = __builtin_amdgcn_permlane32_swap(u[e], u[2 + e], false, false);
      u[e] = (unsigned)sw[0];
      u[2 + e] = (unsigned)sw[1];
    }
    const int64_t p = p0 + 16 * g + 8 * h;
    if (!ok) continue;
    if (p + 8 <= np) {
      if (al) *reinterpret_cast<uint4*>(row + p) = make_uint4(u[0], u[1], u[2], u[3]);
      else *reinterpret_cast<u32x4_u16*>(row + p) = u32x4{u[0], u[1], u[2], u[3]};
    } else if (p < np) {
      struct { T e[8]; } e = __builtin_bit_cast(decltype(e), make_uint4(u[0], u[1], u[2], u[3]));
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (p + k < np) row[p + k] = e.e[k];
    }
  }
}

// a(g) and a'(g): silu (ACT 0), or gelu in its tanh form (1), g s(2 sqrt(2/pi) (g + 0.044715 g^3)). The fast exponential and
// reciprocal are off by some 2^-23 |q| and 2^-23, far below the results' rounding; where |q| is large the sigmoid is 0 or 1.
template <int ACT> __device__ __forceinline__ void activation(float g, float& a, float& da) {
  const float g2 = g * g;
  const float q = ACT ? g * __builtin_fmaf(0.07135481282553433f, g2, 1.5957691216057308f) : g;
  const float dq = ACT ? __builtin_fmaf(0.21406443847660298f, g2, 1.5957691216057308f) : 1.f;
  const float s = __builtin_amdgcn_rcpf(1.f + __expf(-q));
  a = g * s;
  da = __builtin_fmaf(a * dq, 1.f - s, s);
  if (ACT && !(g2 < 1e4f)) da = g != g ? g : s;   // far out, where q' overflows: a is 0 or g
}

// the order of a step: N matrix instructions, after the first of them the next step's READS (two each, so that the last
// have arrived when the step ends), and LOADS tile loads spread over all
template <int N, int READS, int LOADS, int M = 0> __device__ __forceinline__ void interleave() {
  if constexpr (M < N) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    constexpr int r = READS - 2 * M > 2 ? 2 : READS - 2 * M, l = (M + 1) * LOADS / N - M * LOADS / N;
    if constexpr (r > 0) __builtin_amdgcn_sched_group_barrier(0x100, r, 0);
    if constexpr (l > 0) __builtin_amdgcn_sched_group_barrier(0x010, l, 0);
    interleave<N, READS, LOADS, M + 1>();
  }
}

// WP x WQ waves of FP x FQ results of 32 x 32. Two waves to a SIMD: eight of 256 x 256 (128 KiB of LDS, one workgroup to a CU), or
// two workgroups of four of 128 x 128; which one: tiling_of.
template <typename T, Kind KP, Kind KQ, int WP, int WQ, int FP, int FQ, Epi EPI>
__global__ __launch_bounds__(WP * WQ * 64) __attribute__((amdgpu_waves_per_eu(2))) void k_product(const Product a) {
  constexpr int LANES = WP * WQ * 64, TP = WP * FP * 32, TQ = WQ * FQ * 32;
  typedef Tile<T, KP, TP, LANES, EPI == GATED> PT;
  typedef Tile<T, KQ, TQ, LANES, false> QT;
  // objects of their own: what is read is seen not to be what is being filled
  __shared__ __align__(16) T sp0[TP * BK], sq0[TQ * BK], sp1[TP * BK], sq1[TQ * BK];
  // XCD x (workgroups go to XCDs in turn) takes `per` consecutive tiles, in groups of eight rows of tiles: the tiles worked
  // on at a time then share their operands' rows in that XCD's L2
  const int id = ((int)blockIdx.x & 7) * a.per + ((int)blockIdx.x >> 3);
  if (id >= a.tiles * a.splits || ((int)blockIdx.x >> 3) >= a.per) return;
  const int split = id / a.tiles, tile = id - split * a.tiles;
  const int tiles_q = a.tiles / a.tiles_p, group = tile / (8 * a.tiles_p), first = 8 * group, rows = min(8, tiles_q - first);
  const int in = tile - first * a.tiles_p, tp = in / rows, tq = first + in - tp * rows;
  const int64_t p0 = (int64_t)tp * (EPI == GATED ? TP / 2 : TP), q0 = (int64_t)tq * TQ;
  const int64_t k0 = split * a.run, k1 = min(a.k, k0 + a.run);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wp = wave % WP, wq = wave / WP;
  // GATED: a wave's P tiles are the gate's and then the up projection's of the same columns
  constexpr int FH = FP / 2;
  auto p_row = [&](int i) { return EPI == GATED ? i / FH * (TP / 2) + 32 * (wp * FH + i % FH) : 32 * (wp * FP + i); };

  f32x16 acc[FP][FQ];
#pragma unroll
  for (int i = 0; i < FP; ++i)
#pragma unroll
    for (int j = 0; j < FQ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  constexpr int STEPS = BK / 16, READS = (KP == COL ? 2 : 1) * FP + (KQ == COL ? 2 : 1) * FQ;
  struct Frags { uint4 p[FP], q[FQ]; };
  auto read = [&](const T* sp, const T* sq, int s, Frags& f) {
#pragma unroll
    for (int i = 0; i < FP; ++i) f.p[i] = PT::frag(sp, p_row(i), s);
#pragma unroll
    for (int j = 0; j < FQ; ++j) f.q[j] = QT::frag(sq, 32 * (wq * FQ + j), s);
  };
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int i = 0; i < FP; ++i)
#pragma unroll
      for (int j = 0; j < FQ; ++j) acc[i][j] = mfma(T{}, f.p[i], f.q[j], acc[i][j]);
  };
  auto copy = [&](int64_t k, T* sp, T* sq) {   // fewer than BK of k
    PT::copy(a.p, p0, k, min(k1, k + BK), sp);
    QT::copy(a.q, q0, k, min(k1, k + BK), sq);
  };
  {
    // Each step's operands are read while the step before it is multiplied. A tile's last step is multiplied after the
    // barrier: every wave is past its reads of this tile, whose buffer is filled with the tile after the next one, and the
    // next tile's loads have arrived, whose first step is read. What is left of k past the whole tiles is the first tile.
    const int whole = (int)((k1 - k0) / BK), left = k0 + (int64_t)whole * BK < k1 ? 1 : 0, tiles = whole + left;
    PT pt;
    QT qt;
    auto fetch = [&](T* sp, T* sq) {
      pt.fetch(sp);
      qt.fetch(sq);
    };
    Frags f[2];
    auto steps = [&](const T* sp, const T* sq) {   // all but the last
#pragma unroll
      for (int s = 0; s + 1 < STEPS; ++s) {
        read(sp, sq, s + 1, f[(s + 1) & 1]);
        multiply(f[s & 1]);
        interleave<FP * FQ, READS, 0>();
      }
    };
    auto arrived = [&]() {
      __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
      __syncthreads();
    };
    auto tile = [&](T* sp, T* sq, const T* np, const T* nq) {   // another after the next one
      steps(sp, sq);
      arrived();
      read(np, nq, 0, f[0]);
      fetch(sp, sq);
      multiply(f[(STEPS - 1) & 1]);
      interleave<FP * FQ, READS, PT::PASSES + QT::PASSES>();
    };
    if (left) copy(k0 + (int64_t)whole * BK, sp0, sq0);
    pt.start(a.p, p0, k0);
    qt.start(a.q, q0, k0);
    if (!left && tiles) fetch(sp0, sq0);
    arrived();
    if (tiles > 1) fetch(sp1, sq1);
    read(sp0, sq0, 0, f[0]);
    int t = tiles;   // tiles to do
    for (; t >= 4; t -= 2) {
      tile(sp0, sq0, sp1, sq1);
      tile(sp1, sq1, sp0, sq0);
    }
    const T *cp = sp0, *cq = sq0, *np = sp1, *nq = sq1;
    if (t == 3) {
      tile(sp0, sq0, sp1, sq1);
      cp = sp1, cq = sq1, np = sp0, nq = sq0;
    }
    if (t >= 2) {
      steps(cp, cq);
      arrived();
      read(np, nq, 0, f[0]);
      multiply(f[(STEPS - 1) & 1]);
      cp = np, cq = nq;
    }
    if (t) {
      steps(cp, cq);
      multiply(f[(STEPS - 1) & 1]);
    }
  }

  const int64_t np = EPI == GATED ? a.p.half : a.p.size;
  // DGATED: the saved values of the next AHEAD blocks are in flight while one is worked on (what is stored could be what is
  // loaded, for all the compiler knows: it would load each block after the stores of the one before)
  constexpr int AHEAD = 2, BLOCKS = FP * FQ;
  Saved::Raw raw[AHEAD];
  auto load_saved = [&](int n) {   // block n = j FP + i; past the result: its last one
    const int64_t qb = min(q0 + 32 * (wq * FQ + n / FP), a.q.size - 1) >> 5, pb = min(p0 + p_row(n % FP), np - 1) >> 5;
    Saved::load(static_cast<const char*>(a.saved) + (qb * a.saved_cols + pb) * SAVED_BLOCK, raw[n % AHEAD]);
  };
  if constexpr (EPI == DGATED) {
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) load_saved(n);
  }
#pragma unroll
  for (int j = 0; j < FQ; ++j) {
    const int64_t qt = q0 + 32 * (wq * FQ + j), q = qt + (lane & 31);
    const bool ok = q < a.q.size;
    if constexpr (EPI == GATED) {
#pragma unroll
      for (int i = 0; i < FH; ++i) {
        const int64_t p = p0 + p_row(i);
        if (qt >= a.q.size || p >= np) continue;   // wave-uniform
        f32x16 x, y, z;
        auto gated = [&](auto act) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float u = acc[FH + i][j][r];
            float av, da;
            activation<decltype(act)::value>(acc[i][j][r], av, da);
            z[r] = av * u;
            x[r] = u * da;
            y[r] = av;
          }
        };
        if (a.act) gated(std::integral_constant<int, 1>());   // uniform
        else gated(std::integral_constant<int, 0>());
        store_tile<T>(static_cast<T*>(a.out) + q * a.ldo, p, np, ok, a.out16, z);
        if (a.saved) {
          char* block = static_cast<char*>(a.saved) + ((qt >> 5) * a.saved_cols + (p >> 5)) * SAVED_BLOCK;
          Saved::put(block, x);
          Saved::put(block + SAVED_BLOCK / 2, y);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < FP; ++i) {
        const int64_t p = p0 + p_row(i);
        if constexpr (EPI == DGATED) {
          const int n = j * FP + i;
          const Saved::Raw saved = raw[n % AHEAD];
          if (n + AHEAD < BLOCKS) load_saved(n + AHEAD);
          if (qt >= a.q.size || p >= np) continue;   // wave-uniform
          float m[16];
          f32x16 o;
          T* row = static_cast<T*>(a.out) + q * a.ldo;
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            Saved::get(saved, which, m);
#pragma unroll
            for (int r = 0; r < 16; ++r) o[r] = acc[i][j][r] * m[r];
            store_tile<T>(row + which * np, p, np, ok, a.out16, o);
          }
          continue;
        }
        if (qt >= a.q.size || p >= np) continue;
        if constexpr (EPI == STORE) {
          store_tile<T>(static_cast<T*>(a.out) + q * a.ldo, p, np, ok, a.out16, acc[i][j]);
        } else {
          float* row = static_cast<float*>(a.out) + ((int64_t)split * a.q.size + q) * a.ldo;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int64_t pp = p + 8 * g + 4 * (lane >> 5);
            if (ok && pp < np)   // ldo is np rounded up to a multiple of 4
              *reinterpret_cast<float4*>(row + pp) =
                  make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
          }
        }
      }
    }
  }
}

// out [nq][ldo] = round(sum of the splits' products [nq][ldp], in order: the same bits every time), four columns per lane. Its
// reads bound it, mostly out of the caches: 9.7 us for the weight gradients of 16384 x 768 x 2048.
template <typename T>
__global__ __launch_bounds__(256) void k_split_sum(const float* __restrict__ part, int splits, int64_t nq, int64_t np, int64_t ldp,
                                                   T* __restrict__ out, int64_t ldo, bool al) {
  const int64_t per = ldp / 4, all = nq * per, step = nq * ldp;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t q = i / per, p = 4 * (i - q * per);
    const float* src = part + q * ldp + p;
    float4 acc = *reinterpret_cast<const float4*>(src);
    int s = 1;
    for (; s + 4 <= splits; s += 4) {   // four splits' loads in flight
      float4 e[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) e[u] = *reinterpret_cast<const float4*>(src + (s + u) * step);
#pragma unroll
      for (int u = 0; u < 4; ++u) acc = make_float4(acc.x + e[u].x, acc.y + e[u].y, acc.z + e[u].z, acc.w + e[u].w);
    }
    for (; s < splits; ++s) {
      const float4 e = *reinterpret_cast<const float4*>(src + s * step);
      acc = make_float4(acc.x + e.x, acc.y + e.y, acc.z + e.z, acc.w + e.w);
    }
    T* o = out + q * ldo + p;
    const float v[4] = {acc.x, acc.y, acc.z, acc.w};
    if (al && p + 4 <= np) {
      typedef typename CvtOf<T>::type Cvt;
      *reinterpret_cast<uint2*>(o) = make_uint2(Cvt::pack2(v[0], v[1]), Cvt::pack2(v[2], v[3]));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (p + k < np) st1(o + k, v[k]);
    }
  }
}

// out [rows][ld] = x [rows][cols], zeros past the columns, for operands whose rows are not aligned; eight columns per lane. 3 to 6 us for each
// operand of 1001 x 1001 x 2731; the products on unaligned rows, element by element, took 708 us a pass there and take 217 so.
template <typename T>
__global__ __launch_bounds__(256) void k_pad_rows(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t ld,
                                                  T* __restrict__ out) {
  const int64_t per = ld / 8, all = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per, c = 8 * (i - r * per);
    const T* src = x + r * cols + c;
    uint4 v;
    if (c + 8 <= cols) {
      v = UIO<T>::raw(src).u;
    } else {
      struct { T e[8]; } e;
#pragma unroll
      for (int k = 0; k < 8; ++k) e.e[k] = c + k < cols ? src[k] : (T)0;
      v = __builtin_bit_cast(uint4, e);
    }
    *reinterpret_cast<uint4*>(out + r * ld + c) = v;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// few tokens (a serving step): y = x W^T, or the gated pair, for up to 16 MT tokens. The weights' stream bounds it, so they go
// from memory to the matrix cores' registers (v_mfma_f32_16x16x32: lane l has row l mod 16): a workgroup takes 16 rows (of the
// gate's and of the up projection's), its waves the columns in turns of 128, each load instruction 64 consecutive bytes of 16
// rows, all loads of a few turns in flight together. The waves' sums meet in LDS, in order. Any alignment. One token at 2048 x
// 5632 in bf16: 11 to 13 us for gate and up projection (3.6 TB/s of weights) and 8 to 9 us for the down projection (2.6).
// LBK_FEW_TOKENS is one limit for both products. us here and on the tiles, bf16: gate and up projection 32 x 768 x 2048 5.1 and 7.9,
// 32 x 2048 x 5632 18 and 22, 32 x 4096 x 11008 46 and 45; down 32 x 768 x 2048 7.5 and 8.6, but 8 x 2048 x 5632 10.1 and 11.1,
// 16 x 2048 x 5632 11.9 and 11.5, 32 x 2048 x 5632 21 and 13, 1 x 4096 x 11008 22 and 21, 32 x 4096 x 11008 32 and 22.
// ---------------------------------------------------------------------------------------------------------------
typedef float f32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mfma16(bf16_t, uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(_Float16, uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <typename T, int MT, int PAIR, int WAVES, int U>
__global__ __launch_bounds__(64 * WAVES) void k_few_tokens(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw,
                                                           T* __restrict__ y, int64_t ldy, int t, int64_t n, int64_t k, int act) {
  __shared__ f32x4 s_acc[WAVES][PAIR][MT][64];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, r = lane & 15, quad = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16, row = min(n0 + r, n - 1);
  const T* wp[PAIR];
  const T* xp[MT];
#pragma unroll
  for (int g = 0; g < PAIR; ++g) wp[g] = w + (g * n + row) * ldw + 8 * quad;
#pragma unroll
  for (int m = 0; m < MT; ++m) xp[m] = x + (int64_t)min(16 * m + r, t - 1) * ldx + 8 * quad;
  f32x4 acc[PAIR][MT];
#pragma unroll
  for (int g = 0; g < PAIR; ++g)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[g][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t whole = k / 128;
  // a wave takes consecutive turns, the loads of U of them before the first is used (past its last one: that again, as zeros)
  const int64_t each = (whole + WAVES - 1) / WAVES, end = min(whole, (wave + 1) * each);
  for (int64_t c = wave * each; c < end; c += U) {
    uint4 wf[U][PAIR][4], xf[U][MT][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = 128 * min(c + u, end - 1);
#pragma unroll
      for (int g = 0; g < PAIR; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j) wf[u][g][j] = UIO<T>::raw(wp[g] + at + 32 * j).u;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) xf[u][m][j] = UIO<T>::raw(xp[m] + at + 32 * j).u;
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = c + u < end;   // wave-uniform
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4 xv = there ? xf[u][m][j] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int g = 0; g < PAIR; ++g) {
            const uint4 wv = there ? wf[u][g][j] : make_uint4(0u, 0u, 0u, 0u);
            acc[g][m] = mfma16(T{}, wv, xv, acc[g][m]);
          }
        }
    }
  }
  if (k % 128 && wave == WAVES - 1) {   // the last columns, zeros past them
    auto piece = [&](const T* p, int64_t c) {
      if (c + 8 <= k) return UIO<T>::raw(p + c - 8 * quad).u;
      struct { T e[8]; } e;
#pragma unroll
      for (int i = 0; i < 8; ++i) e.e[i] = c + i < k ? p[c - 8 * quad + i] : (T)0;
      return __builtin_bit_cast(uint4, e);
    };
    for (int j = 0; j < 4; ++j) {
      const int64_t c = 128 * whole + 32 * j + 8 * quad;
      uint4 wf[PAIR], xf[MT];
#pragma unroll
      for (int g = 0; g < PAIR; ++g) wf[g] = piece(wp[g], c);
#pragma unroll
      for (int m = 0; m < MT; ++m) xf[m] = piece(xp[m], c);
#pragma unroll
      for (int g = 0; g < PAIR; ++g)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[g][m] = mfma16(T{}, wf[g], xf[m], acc[g][m]);
    }
  }
#pragma unroll
  for (int g = 0; g < PAIR; ++g)
#pragma unroll
    for (int m = 0; m < MT; ++m) s_acc[wave][g][m][lane] = acc[g][m];
  __syncthreads();
  // element e of a 16 x 16 result: row e / 16 of the weights (register e / 16 mod 4 of lane 16 (e / 64) + token)
  for (int i = (int)threadIdx.x; i < 256 * MT; i += 64 * WAVES) {
    const int m = i >> 8, token = (i >> 4) & 15, rr = i & 15, from = 16 * (rr >> 2) + token;
    float v[PAIR];
#pragma unroll
    for (int g = 0; g < PAIR; ++g) {
      v[g] = 0.f;
      for (int q = 0; q < WAVES; ++q) v[g] += s_acc[q][g][m][from][rr & 3];
    }
    float o = v[0];
    if constexpr (PAIR == 2) {
      float da;
      if (act) activation<1>(v[0], o, da);
      else activation<0>(v[0], o, da);
      o *= v[1];
    }
    if (16 * m + token < t && n0 + rr < n) st1(y + (int64_t)(16 * m + token) * ldy + n0 + rr, o);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------
inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool al2(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }
inline int launched() { return (int)hipGetLastError(); }
inline unsigned grid_of(int64_t n, int64_t cap) { return (unsigned)((n + 255) / 256 < cap ? (n + 255) / 256 : cap); }
constexpr int64_t MAX_SIZE = 0x7fffffff;   // of one dimension
constexpr int64_t MAX_LD = 1 << 22;        // rows of memory up to which a tile's byte offsets fit 32 bits (256 rows)

template <typename T, Kind KP, Kind KQ, int WP, int WQ, int FP, int FQ, Epi EPI> int launch_tiles(Product a, hipStream_t st) {
  constexpr int TP = (EPI == GATED ? WP * FP * 16 : WP * FP * 32), TQ = WQ * FQ * 32;
  const int64_t np = EPI == GATED ? a.p.half : a.p.size;
  const int64_t tp = (np + TP - 1) / TP, tq = (a.q.size + TQ - 1) / TQ, tiles = tp * tq;
  if (tiles * a.splits > 0xfffffff) return LDR_E_SHAPE;
  a.tiles_p = (int)tp;
  a.tiles = (int)tiles;
  a.per = (int)((tiles * a.splits + 7) / 8);
  hipLaunchKernelGGL((k_product<T, KP, KQ, WP, WQ, FP, FQ, EPI>), dim3((unsigned)(8 * a.per)), dim3(WP * WQ * 64), 0, st, a);
  return launched();
}

// Which tiles, and in how many splits of k, by the time they take: 128 x 128 ones of four waves, two to a CU; 256 x 256 ones of
// eight waves, one to a CU; 192 (of P) x 256 likewise, which divide some sizes better (768: 256 tiles instead of 192 at 16384
// tokens, 50.0 -> 47.2 and 94.8 -> 90.0 us; 8192 x 2048 x 5632: 348 -> 321 and 167 -> 160 for the weight gradients, but 152 -> 200
// for the down product). A round of tiles takes a step per 64 k, the shorter the fewer of them the GPU holds (less contention, a
// higher clock), and what surrounds the steps; splits are written and read as fp32. The constants are a fit to 59 products
// of sides from 250 to 16384, in bf16; over 48 others the choice is 0.9 % behind the fastest of the three in the mean, 16 % at
// most.
enum Shape { SMALL, BIG, WIDE };
struct Tiling { Shape shape; int splits; };
inline Tiling tiling_of(int64_t np, int64_t nq, int64_t k, bool plain) {   // plain: may be split, and of any shape
  constexpr int64_t CUS = 256;
  constexpr struct { double least, fixed, filled, around; } US[] = {{0.5, 0.43, 0.66, 4.3}, {1.0, 0.48, 1.1, 8.6}, {1.0, 0.46, 0.74, 6.7}};
  Tiling best{SMALL, 1};
  double least = 1e30;
  for (int shape = SMALL; shape <= (plain ? WIDE : BIG); ++shape) {
    const int64_t tp = shape == SMALL ? 128 : shape == BIG ? 256 : 192, tq = shape == SMALL ? 128 : 256;
    const int64_t tiles = ((np + tp - 1) / tp) * ((nq + tq - 1) / tq), at_once = shape == SMALL ? 2 * CUS : CUS;
    auto round = [&](double part, int64_t steps) {   // of so many steps, that holds `part` of what the GPU does
      const double step = US[shape].fixed + US[shape].filled * part;
      return steps * (step < US[shape].least ? US[shape].least : step) + US[shape].around;
    };
    const int64_t ks = (k + 63) / 64, most = plain ? (ks / 4 < 32 ? ks / 4 : 32) : 1;
    for (int64_t s = 1; s <= (most < 1 ? 1 : most); ++s) {
      const int64_t full = tiles * s / at_once, rest = tiles * s % at_once, each = (ks + s - 1) / s;
      const double us = full * round(1.0, each) + (rest ? round((double)rest / at_once, each) : 0.0) +
                        (s > 1 ? 1.4 + (double)s * np * nq * 8 / 4e6 : 0.0);
      if (us < least) least = us, best = Tiling{(Shape)shape, (int)s};
    }
  }
  return best;
}
// the gated products' shapes: gate and up projection of t tokens, d -> 2 n, and their gradients, n columns summed over d. The first
// by the plain products' model: of 27 sizes, d from 512 to 8192, it chose the slower one once (2048 x 2048 x 5632: 104 us, 100)
inline Shape gated_shape(int64_t t, int64_t d, int64_t n) { return tiling_of(2 * n, t, d, false).shape; }
// a short sum beside ten bytes moved per element: two workgroups to a CU, one's loads and stores beside the other's products.
// us with the small and the large tiles: 16384 x 512 x 1408 65 and 79, 16384 x 768 x 2048 103 and 114, 16384 x 1024 x 2816 154
// and 169, 16384 x 1280 x 3456 215 and 237, 16384 x 1536 x 4096 288 and 310, 8192 x 2048 x 5632 234 and 240; 8192 x 2560 x 6912 369
// and 362, 4096 x 2816 x 7680 207 and 198, 8192 x 4096 x 11008 881 and 837, 8192 x 6144 x 5632 626 and 537. Past 2048 the time
// model of the plain products chooses, which is not fitted to this kernel (2048 x 4096 x 11008: 229, where the small ones take 213)
inline Shape dgated_shape(int64_t t, int64_t d, int64_t n) { return d > 2048 ? tiling_of(n, t, d, false).shape : SMALL; }
inline int64_t scratch_ld(int64_t np) { return (np + 3) / 4 * 4; }

template <typename T, Kind KP, Kind KQ, Epi EPI> int launch_product(const Product& a, Shape shape, hipStream_t st) {
  if constexpr (EPI == STORE || EPI == PARTIAL)
    if (shape == WIDE) return launch_tiles<T, KP, KQ, 2, 4, 3, 2, EPI>(a, st);
  return shape == SMALL ? launch_tiles<T, KP, KQ, 2, 2, 2, 2, EPI>(a, st) : launch_tiles<T, KP, KQ, 4, 2, 2, 4, EPI>(a, st);
}
template <typename T, Kind KP, Kind KQ> int plain_product(Product a, float* scratch, hipStream_t st) {
  const int64_t np = a.p.size, nq = a.q.size;
  const Tiling tl = tiling_of(np, nq, a.k, true);
  const bool al = np % 8 == 0 && a.ldo % 8 == 0 && al16(a.out);
  if (tl.splits == 1) {
    a.out16 = al;
    return launch_product<T, KP, KQ, STORE>(a, tl.shape, st);
  }
  if (!scratch) return LDR_E_ARG;
  void* const out = a.out;
  const int64_t ldo = a.ldo, ldp = scratch_ld(np);
  a.run = ((a.k + tl.splits - 1) / tl.splits + 63) / 64 * 64;
  a.splits = (int)((a.k + a.run - 1) / a.run);
  a.out = scratch;
  a.ldo = ldp;
  const int e = launch_product<T, KP, KQ, PARTIAL>(a, tl.shape, st);
  if (e) return e;
  hipLaunchKernelGGL(k_split_sum<T>, dim3(grid_of(nq * ldp / 4, 4096)), dim3(256), 0, st, scratch, a.splits, nq, np, ldp,
                     static_cast<T*>(out), ldo, al);
  return launched();
}

template <typename T, int MT, int PAIR>
int few(const void* x, int64_t ldx, const void* w, int64_t ldw, void* y, int64_t ldy, int64_t t, int64_t n, int64_t k, int act,
        hipStream_t st) {
  const int64_t blocks = (n + 15) / 16;
  if (blocks > MAX_SIZE) return LDR_E_SHAPE;
#define FEW(W, U) hipLaunchKernelGGL((k_few_tokens<T, MT, PAIR, W, U>), dim3((unsigned)blocks), dim3(64 * W), 0, st,                   \
                                     static_cast<const T*>(x), ldx, static_cast<const T*>(w), ldw, static_cast<T*>(y), ldy, (int)t, n,  \
                                     k, act)
  // waves that share a workgroup's columns: more where there are few workgroups; as many turns' loads in flight as each has, up
  // to what its registers hold (one token at 2048 x 5632: 13 and 9 us; with one turn's 21 and 14)
  constexpr int MANY = PAIR > 1 ? 8 : 16, MOST = MT > 1 ? 2 : PAIR > 1 ? 4 : 3;
  const int64_t turns = k / 128;
  if (blocks >= 256) {
    if (turns <= 4) FEW(4, 1);
    else FEW(4, MOST);
  } else {
    if (turns <= MANY) FEW(MANY, 1);
    else FEW(MANY, (MOST > 2 && PAIR > 1 ? 2 : MOST));
  }
#undef FEW
  return launched();
}
template <typename T, int PAIR>
int few_tokens(const void* x, int64_t ldx, const void* w, int64_t ldw, void* y, int64_t ldy, int64_t t, int64_t n, int64_t k, int act,
               hipStream_t st) {
  if (t <= 16) return few<T, 1, PAIR>(x, ldx, w, ldw, y, ldy, t, n, k, act, st);
  return few<T, 2, PAIR>(x, ldx, w, ldw, y, ldy, t, n, k, act, st);
}

#define FFN_TYPE_SWITCH(DT, ...)                                 \
  if ((DT) == LDR_BF16) { typedef bf16_t T; __VA_ARGS__; }       \
  else { typedef _Float16 T; __VA_ARGS__; }

// sizes of a product with t tokens: dtype, dimensions, and the rows' lengths
inline int sizes(int64_t t, int64_t a, int64_t b, int dtype) {
  if (dtype != LDR_BF16 && dtype != LDR_F16) return LDR_E_DTYPE;
  if (t < 0 || a < 1 || b < 1) return LDR_E_ARG;
  return t > MAX_SIZE || a > MAX_SIZE || b > MAX_SIZE ? LDR_E_SHAPE : LDR_OK;
}
// an operand of the tiled kernels: rows of `cols` elements, ld apart
inline int operand(const void* p, int64_t cols, int64_t ld) {
  if (!p) return LDR_E_ARG;
  if (ld < cols || ld > MAX_LD) return LDR_E_SHAPE;
  return ld % 8 || !al16(p) ? LDR_E_ALIGN : LDR_OK;
}
inline Product product(Operand p, Operand q, int64_t k, void* out, int64_t ldo) {
  Product a{};
  a.p = p, a.q = q, a.k = a.run = k, a.out = out, a.ldo = ldo, a.splits = 1;
  return a;
}

}  // namespace

extern "C" {

int lbk_pad_rows(const void* x, int64_t rows, int64_t cols, int64_t ld, void* out, int dtype, void* stream) {
  const int e = sizes(rows, cols, ld, dtype);
  if (e || rows == 0) return e;
  if (!x || !out) return LDR_E_ARG;
  if (ld < cols) return LDR_E_SHAPE;
  if (ld % 8 || !al16(out) || !al2(x)) return LDR_E_ALIGN;
  FFN_TYPE_SWITCH(dtype, hipLaunchKernelGGL(k_pad_rows<T>, dim3(grid_of(rows * (ld / 8), 8192)), dim3(256), 0,
                                            static_cast<hipStream_t>(stream), static_cast<const T*>(x), rows, cols, ld,
                                            static_cast<T*>(out)))
  return launched();
}

int64_t lbk_ffn_saved_bytes(int64_t t, int64_t n) {
  return t < 1 || n < 1 ? 0 : ((t + 31) / 32) * ((n + 31) / 32) * SAVED_BLOCK;
}

int lbk_ffn_gate_up(const void* x, int64_t ldx, const void* w, int64_t ldw, void* act, int64_t ld_act, void* saved, int64_t t,
                    int64_t d, int64_t n, int activation, int dtype, void* stream) {
  int e = sizes(t, d, n, dtype);
  if (e) return e;
  if ((activation != 0 && activation != 1) || ld_act < n) return LDR_E_ARG;
  if (t == 0) return LDR_OK;
  if (!x || !w || !act) return LDR_E_ARG;
  if (!al2(x) || !al2(w) || !al2(act) || !al16(saved)) return LDR_E_ALIGN;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (t <= LBK_FEW_TOKENS && !saved) {
    if (ldx < d || ldw < d) return LDR_E_SHAPE;
    FFN_TYPE_SWITCH(dtype, return (few_tokens<T, 2>(x, ldx, w, ldw, act, ld_act, t, n, d, activation, st)))
  }
  if ((e = operand(x, d, ldx)) || (e = operand(w, d, ldw))) return e;
  Product a = product({w, ldw, 2 * n, n}, {x, ldx, t, 0}, d, act, ld_act);
  a.out16 = ld_act % 8 == 0 && al16(act);
  a.saved = saved;
  a.saved_cols = (n + 31) / 32;
  a.act = activation;
  FFN_TYPE_SWITCH(dtype, return (launch_product<T, ROW, ROW, GATED>(a, gated_shape(t, d, n), st)))
}

int lbk_ffn_dgate_up(const void* dy, int64_t ld_dy, const void* w_down, int64_t ldw, const void* saved, void* dgate_up, int64_t ld_dgu,
                     int64_t t, int64_t n, int64_t d, int dtype, void* stream) {
  int e = sizes(t, d, n, dtype);
  if (e) return e;
  if (ld_dgu < 2 * n) return LDR_E_ARG;
  if (t == 0) return LDR_OK;
  if (!saved || !dgate_up) return LDR_E_ARG;
  if (!al2(dgate_up) || !al16(saved)) return LDR_E_ALIGN;
  if ((e = operand(dy, d, ld_dy)) || (e = operand(w_down, n, ldw))) return e;
  Product a = product({w_down, ldw, n, 0}, {dy, ld_dy, t, 0}, d, dgate_up, ld_dgu);
  a.out16 = n % 8 == 0 && ld_dgu % 8 == 0 && al16(dgate_up);
  a.saved = const_cast<void*>(saved);
  a.saved_cols = (n + 31) / 32;
  FFN_TYPE_SWITCH(dtype, return (launch_product<T, COL, ROW, DGATED>(a, dgated_shape(t, d, n), static_cast<hipStream_t>(stream))))
}

int64_t lbk_linear_scratch(int64_t np, int64_t nq, int64_t k) {
  if (np < 1 || nq < 1 || k < 1) return 0;
  const Tiling tl = tiling_of(np, nq, k, true);
  return tl.splits > 1 ? tl.splits * nq * scratch_ld(np) : 0;
}

int lbk_product_tiling(int product, int64_t columns, int64_t rows, int64_t summed, int* splits) {
  if (product < 0 || product > 2 || !splits) return LDR_E_ARG;
  if (columns < 1 || rows < 1 || summed < 1 || (product == 1 && columns % 2)) return LDR_E_SHAPE;
  *splits = 1;
  if (product == 1) return gated_shape(rows, summed, columns / 2);
  if (product == 2) return dgated_shape(rows, summed, columns);
  const Tiling tl = tiling_of(columns, rows, summed, true);
  *splits = tl.splits;
  return tl.shape;
}

int lbk_linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, void* y, int64_t ldy, float* scratch, int64_t t, int64_t k,
                   int64_t n, int dtype, void* stream) {
  int e = sizes(t, k, n, dtype);
  if (e || t == 0) return e;
  if (!x || !w || !y || ldy < n) return LDR_E_ARG;
  if (!al2(x) || !al2(w) || !al2(y) || !al16(scratch)) return LDR_E_ALIGN;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (t <= LBK_FEW_TOKENS) {
    if (ldx < k || ldw < k) return LDR_E_SHAPE;
    FFN_TYPE_SWITCH(dtype, return (few_tokens<T, 1>(x, ldx, w, ldw, y, ldy, t, n, k, 0, st)))
  }
  if ((e = operand(x, k, ldx)) || (e = operand(w, k, ldw))) return e;
  const Product a = product({w, ldw, n, 0}, {x, ldx, t, 0}, k, y, ldy);
  FFN_TYPE_SWITCH(dtype, return (plain_product<T, ROW, ROW>(a, scratch, st)))
}

int lbk_linear_dx(const void* dy, int64_t ld_dy, const void* w, int64_t ldw, void* dx, int64_t ld_dx, float* scratch, int64_t t, int64_t n,
                  int64_t k, int dtype, void* stream) {
  int e = sizes(t, k, n, dtype);
  if (e || t == 0) return e;
  if (!dx || ld_dx < k) return LDR_E_ARG;
  if (!al2(dx) || !al16(scratch)) return LDR_E_ALIGN;
  if ((e = operand(dy, n, ld_dy)) || (e = operand(w, k, ldw))) return e;
  const Product a = product({w, ldw, k, 0}, {dy, ld_dy, t, 0}, n, dx, ld_dx);
  FFN_TYPE_SWITCH(dtype, return (plain_product<T, COL, ROW>(a, scratch, static_cast<hipStream_t>(stream))))
}

int lbk_linear_dw(const void* dy, int64_t ld_dy, const void* x, int64_t ldx, float* scratch, void* dw, int64_t t, int64_t n, int64_t k,
                  int dtype, void* stream) {
  int e = sizes(t, k, n, dtype);
  if (e) return e;
  if (!dw || t < 1) return LDR_E_ARG;
  if (!al2(dw) || !al16(scratch)) return LDR_E_ALIGN;
  if ((e = operand(dy, n, ld_dy)) || (e = operand(x, k, ldx))) return e;
  const Product a = product({x, ldx, k, 0}, {dy, ld_dy, n, 0}, t, dw, k);
  FFN_TYPE_SWITCH(dtype, return (plain_product<T, COL, COL>(a, scratch, static_cast<hipStream_t>(stream))))
}

}  // extern "C"
