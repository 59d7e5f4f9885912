// loopback_block.hip -- MI355X (gfx950, CDNA4) kernels that bring a block's output back on the residual stream, and
// dropout. Both are bound by the HBM stream of their rows: each is one pass over them, with fp32 statistics, one rounding
// per result, and dropout's mask formed from its counter in the registers where it is applied. Every sum has a fixed
// order: results are deterministic.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include "loopback_block.h"
#include "loopback_read.h"
#include "row_io.h"

namespace {

// ---------------------------------------------------------------------------------------------------------------
// Philox-4x32-10 (Salmon, Moraes, Dror, Shaw, 2011): ten rounds of two 32 x 32 -> 64 bit products over a 128-bit counter
// ---------------------------------------------------------------------------------------------------------------
struct Rng { uint32_t k0, k1, step; };
__device__ __forceinline__ Rng rng_of(const int64_t* rng) {
  const uint64_t seed = (uint64_t)rng[0];
  return Rng{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)(uint64_t)rng[1]};
}
__device__ __forceinline__ uint4 philox(uint32_t block, uint32_t row, uint32_t site, const Rng& r) {
  uint32_t c0 = block, c1 = row, c2 = site, c3 = r.step, k0 = r.k0, k1 = r.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}
// v = kept ? v * s : 0, eight columns from one block w of the generator
__device__ __forceinline__ void drop8(float (&v)[8], const uint4& w, uint32_t drop, float s) {
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t bits = k & 1 ? words[k >> 1] >> 16 : words[k >> 1] & 0xffffu;
    v[k] = bits >= drop ? v[k] * s : 0.f;
  }
}
// The generator is two 32 x 32 -> 64 bit products a round, ten rounds for eight columns: it stays behind the rows' stream, which
// bounds the kernel where there are rows enough: 16384 x 5632 in bf16 66 us (5.6 TB/s), 16384 x 768 12 us (4.2 TB/s).
inline float keep_scale(int drop) { return drop >= 65536 ? 0.f : 65536.f / (float)(65536 - drop); }

template <typename T, bool AL>
__global__ __launch_bounds__(WG) void k_dropout(const T* __restrict__ x, const int64_t* __restrict__ rng, uint32_t site,
                                                uint32_t drop, float s, T* __restrict__ out, int64_t rows, int64_t d,
                                                int64_t nb) {
  const Rng r = rng_of(rng);
  const int64_t n = rows * nb;
  for (int64_t i = (int64_t)blockIdx.x * WG + threadIdx.x; i < n; i += (int64_t)gridDim.x * WG) {
    const int64_t row = i / nb, b = i - row * nb;
    const int left = (int)min((int64_t)8, d - 8 * b);   // columns of this block
    const int64_t o = row * d + 8 * b;
    float v[8];
    IO<T>::unpack(load8<T, AL>(x + o, 0, left), v);
    drop8(v, philox((uint32_t)b, (uint32_t)row, site, r), drop, s);
    store8<T, AL>(out + o, 0, left, v);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// block join. LPR lanes share a row, eight columns each (row_io.h).
// ---------------------------------------------------------------------------------------------------------------
template <typename T> struct JoinFwd {
  const T *x, *y, *post, *gate, *pre;
  const int64_t* rng;
  T *h, *n;
  float *r_post, *r_pre;
  int rows, d, gate_rows;
  uint32_t site, drop;
  float scale, keep, eps;
};

// Reads x and y, writes h and n and two statistics a row: the rows' stream bounds it, beside the vector units (0.7 of the time with
// the generator, 0.46 without). 16384 x 768 in bf16 with all parts 19 to 21 us (4.8 to 5.2 TB/s), 6825 x 2048 in fp16 18 to 23 us (4.9
// to 5.8 TB/s). LPR lanes to a row of LPR x 8 columns at most, so that a lane holds its
// eight in registers.
// PARTS: which parts the call has, known when the kernel is compiled (1 the norm before the next block, 2 the norm after this
// one, 4 dropout), or ANY: looked up as it runs (rows that take the narrow loads)
constexpr int ANY = -1;
template <typename T, int LPR, bool AL, int PARTS>
__global__ __launch_bounds__(lanes_of(LPR)) void k_join_fwd(const JoinFwd<T> a) {
  const bool has_pre = PARTS < 0 ? a.pre != nullptr : PARTS & 1, has_post = PARTS < 0 ? a.post != nullptr : PARTS & 2,
             drops = PARTS < 0 ? a.drop != 0 : PARTS & 4;
  constexpr int LANES = lanes_of(LPR), R = LANES / LPR;
  __shared__ float s_red[2][LANES / 64];
  RowSum<LPR> row_sum{s_red};
  const int d = a.d, lane = (int)threadIdx.x % LPR, col = 8 * lane, grp = group_of<LPR>();
  const float inv_d = 1.f / (float)d;
  const typename IO<T>::Raw post = has_post ? load8<T, AL>(a.post, col, d) : IO<T>::zero(),
                            pre = has_pre ? load8<T, AL>(a.pre, col, d) : IO<T>::zero();
  typename IO<T>::Raw gate = IO<T>::zero();
  Rng rng{0, 0, 0};
  if (drops) rng = rng_of(a.rng);
  int gate_row = -1;
  for (int64_t row0 = (int64_t)blockIdx.x * R; row0 < a.rows; row0 += (int64_t)gridDim.x * R) {
    const int64_t mine = row0 + grp;
    const bool ok = mine < a.rows;
    const int row = (int)(ok ? mine : a.rows - 1);
    const int64_t ro = (int64_t)row * d;
    const typename IO<T>::Raw xr = load8<T, AL>(a.x + ro, col, d), yr = load8<T, AL>(a.y + ro, col, d);
    if (a.gate && row / a.gate_rows != gate_row) {
      gate_row = row / a.gate_rows;
      gate = load8<T, AL>(a.gate + (int64_t)gate_row * d, col, d);
    }
    float r1 = 1.f;
    if (has_post) {
      float e[8], ss = 0.f;
      IO<T>::unpack(yr, e);
#pragma unroll
      for (int k = 0; k < 8; ++k) ss = __builtin_fmaf(e[k], e[k], ss);
      r1 = rsqrtf(row_sum(ss) * inv_d + a.eps);
      if (a.r_post && lane == 0 && ok) a.r_post[row] = r1;
    }
    float h[8], z[8], e[8], ss = 0.f;
    IO<T>::unpack(yr, z);
    if (has_post) {
      IO<T>::unpack(post, e);
#pragma unroll
      for (int k = 0; k < 8; ++k) z[k] *= r1 * e[k];
    }
    if (a.gate) {
      IO<T>::unpack(gate, e);
#pragma unroll
      for (int k = 0; k < 8; ++k) z[k] *= e[k];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) z[k] *= a.scale;
    if (drops) drop8(z, philox((uint32_t)lane, (uint32_t)row, a.site, rng), a.drop, a.keep);
    IO<T>::unpack(xr, h);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      h[k] += z[k];
      ss = __builtin_fmaf(h[k], h[k], ss);
    }
    if (ok) store8<T, AL>(a.h + ro, col, d, h);
    if (has_pre) {
      const float r2 = rsqrtf(row_sum(ss) * inv_d + a.eps);
      if (a.r_pre && lane == 0 && ok) a.r_pre[row] = r2;
      IO<T>::unpack(pre, e);
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] *= h[k] * r2;
      if (ok) store8<T, AL>(a.n + ro, col, d, e);
    }
  }
}

template <typename T> struct JoinBwd {
  const T *dh, *dn, *x, *y, *post, *gate, *pre;
  const float *r_post, *r_pre;
  const int64_t* rng;
  T *dx, *dy, *dgate;
  float *part_post, *part_pre, *part_gate;   // [parts][d], [parts][d], [parts][2][d]; NULL: not wanted
  int rows, d, gate_rows, per;
  uint32_t site, drop;
  float scale, keep;
};

// The next norm's gradient is formed at the sum before it was rounded, from x, y and the mask: at the rounded one, which would be read
// in x's place, dpre has up to 7.5 times the error of its own rounding (few rows), so 1.0.
// A workgroup takes `per` consecutive rows and keeps the column sums of the three weight gradients in registers. The gate's
// belong to runs of gate_rows rows: a run that lies inside the workgroup's rows is finished here, a share of a longer one
// goes to part_gate, first slot where the run began before this workgroup's rows, second where it ends after them.
// gate_rows 1: each element's own. Nothing is saturated: counters at 16384 x 768 in bf16 with all parts have the vector units issue
// for 0.64 of the time, the rows move at 4.4 TB/s and the waves wait for 0.45 of their cycles, at 2.9 waves to a SIMD (148 registers);
// without dropout at 6825 x 2048 in fp16 0.43, 5.6 TB/s and 0.59. 36 to 42 us and 33 to 36 us by machine (two vectors a lane on half
// the lanes took 72, held to fewer registers 121 to 210 with spills; loading the next row ahead changed nothing, 43.4 against 43.7).
// Rows wider than 4096 take 16 waves of 128 registers: with both norms some are spilled (12 to 108 bytes a lane). 512 lanes of two
// vectors spill nothing and are slower: 16384 x 5001 in bf16 394 -> 470 us, 8192 x 8192 226 -> 255.
template <typename T, int LPR, bool AL, int PARTS>
__global__ __launch_bounds__(lanes_of(LPR)) void k_join_bwd(const JoinBwd<T> a) {
  const bool has_dn = PARTS < 0 ? a.dn != nullptr : PARTS & 1, has_post = PARTS < 0 ? a.post != nullptr : PARTS & 2,
             drops = PARTS < 0 ? a.drop != 0 : PARTS & 4;
  constexpr int LANES = lanes_of(LPR), R = LANES / LPR, W = 8 * LPR;
  __shared__ float s_red[2][LANES / 64];
  __shared__ float s_sum[R > 1 ? R * W : 1];
  RowSum<LPR> row_sum{s_red};
  const int d = a.d, lane = (int)threadIdx.x % LPR, col = 8 * lane, grp = group_of<LPR>();
  const float inv_d = 1.f / (float)d;
  typename IO<T>::Raw post = has_post ? load8<T, AL>(a.post, col, d) : IO<T>::zero(),
                      pre = has_dn ? load8<T, AL>(a.pre, col, d) : IO<T>::zero(), gate = IO<T>::zero();
  float d_post[8], d_pre[8], d_gate[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) d_post[k] = d_pre[k] = d_gate[k] = 0.f;
  Rng rng{0, 0, 0};
  if (drops) rng = rng_of(a.rng);
  int gate_row = -1;

  // the row groups' column sums, added in order, to out (fp32) or out_t (rounded)
  auto flush = [&](float (&acc)[8], float* out, T* out_t) {
    if constexpr (R == 1) {
      if (out) store8<float, AL>(out, col, d, acc);
      else store8<T, AL>(out_t, col, d, acc);
    } else {
      __syncthreads();
      IO<float>::store(s_sum + grp * W + col, acc);
      __syncthreads();
      for (int c = (int)threadIdx.x; c < d; c += LANES) {
        float t = s_sum[c];
        for (int g = 1; g < R; ++g) t += s_sum[g * W + c];
        if (out) out[c] = t;
        else st1(out_t + c, t);
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.f;
  };

  const bool runs = a.dgate && a.gate_rows > 1;   // gate sums over runs of rows
  const int64_t r0 = (int64_t)blockIdx.x * a.per, r1 = min((int64_t)a.rows, r0 + a.per);
  for (int64_t s0 = r0; s0 < r1;) {
    const int64_t g0 = runs ? s0 / a.gate_rows * a.gate_rows : r0;                  // the run's first row
    const int64_t g1 = runs ? min((int64_t)a.rows, g0 + a.gate_rows) : r1;          // and its end
    const int64_t s1 = min(r1, g1);
    for (int64_t row0 = s0; row0 < s1; row0 += R) {
      const bool ok = row0 + grp < s1;
      const int row = (int)(ok ? row0 + grp : s1 - 1);
      const int64_t ro = (int64_t)row * d;
      typename IO<T>::Raw xr, yr, dhr, dnr;
      if (has_dn) {
        dnr = load8<T, AL>(a.dn + ro, col, d);
        xr = load8<T, AL>(a.x + ro, col, d);
      }
      dhr = a.dh ? load8<T, AL>(a.dh + ro, col, d) : IO<T>::zero();
      yr = load8<T, AL>(a.y + ro, col, d);
      // a row that is not there (its lanes work on the last one again) adds nothing to the column sums: not zeros either, which
      // would be NaN beside an infinite factor
      const bool there = R == 1 || ok;
      if (a.gate && row / a.gate_rows != gate_row) {
        gate_row = row / a.gate_rows;
        gate = load8<T, AL>(a.gate + (int64_t)gate_row * d, col, d);
      }
      anew<T>(post);
      anew<T>(pre);
      anew<T>(gate);
      const float q2 = has_dn ? a.r_pre[row] : 0.f, q1 = has_post ? a.r_post[row] : 1.f;
      const uint4 words = drops ? philox((uint32_t)lane, (uint32_t)row, a.site, rng) : make_uint4(0u, 0u, 0u, 0u);
      float g[8];   // the gradient of h
      if (has_dn) {
        float h[8], e[8], z[8], c = 0.f;   // h before its rounding; sum dn pre h
        IO<T>::unpack(yr, z);
        if (has_post) {
          IO<T>::unpack(post, e);
#pragma unroll
          for (int k = 0; k < 8; ++k) z[k] *= q1 * e[k];
        }
        if (a.gate) {
          IO<T>::unpack(gate, e);
#pragma unroll
          for (int k = 0; k < 8; ++k) z[k] *= e[k];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) z[k] *= a.scale;
        if (drops) drop8(z, words, a.drop, a.keep);
        IO<T>::unpack(xr, h);
        IO<T>::unpack(dnr, g);
        IO<T>::unpack(pre, e);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          h[k] += z[k];
          if (there) d_pre[k] = __builtin_fmaf(g[k], h[k] * q2, d_pre[k]);
          g[k] *= e[k];
          c = __builtin_fmaf(g[k], h[k], c);
        }
        c = row_sum(c) * q2 * q2 * inv_d;
        if constexpr (LPR > 512) {   // 128 registers a lane: fewer unpacked values kept (bf16 8192 x 8192 251 -> 197 us)
          anew<T>(yr);
          anew<T>(post);
          anew<T>(gate);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] = q2 * (g[k] - c * h[k]);
        IO<T>::unpack(dhr, e);
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] += e[k];
      } else {
        IO<T>::unpack(dhr, g);
      }
      float c = 0.f;       // sum of the normed row's gradient times y
      if (a.dx && ok) store8<T, AL>(a.dx + ro, col, d, g);
      float e[8], w[8], gt[8];
      IO<T>::unpack(yr, e);
      IO<T>::unpack(post, w);
      IO<T>::unpack(gate, gt);
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] *= a.scale;
      if (drops) drop8(g, words, a.drop, a.keep);
      if (a.gate) {
        float og[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          og[k] = g[k] * (has_post ? e[k] * q1 * w[k] : e[k]);
          if (there) d_gate[k] += og[k];
          g[k] *= gt[k];
        }
        if (a.dgate && a.gate_rows == 1 && ok) store8<T, AL>(a.dgate + ro, col, d, og);
      }
      if (has_post) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (there) d_post[k] = __builtin_fmaf(g[k], e[k] * q1, d_post[k]);
          g[k] *= w[k];
          c = __builtin_fmaf(g[k], e[k], c);
        }
      }
      if (a.dy) {
        if (has_post) {
          c = row_sum(c) * q1 * q1 * inv_d;
#pragma unroll
          for (int k = 0; k < 8; ++k) g[k] = q1 * (g[k] - c * e[k]);
        }
        if (ok) store8<T, AL>(a.dy + ro, col, d, g);
      }
    }
    if (runs) {
      if (s0 == g0 && s1 == g1) flush(d_gate, nullptr, a.dgate + g0 / a.gate_rows * d);
      else flush(d_gate, a.part_gate + ((int64_t)blockIdx.x * 2 + (s0 == g0 ? 1 : 0)) * d, nullptr);
    }
    s0 = s1;
  }
  if (a.part_post) flush(d_post, a.part_post + (int64_t)blockIdx.x * d, nullptr);
  if (a.part_pre) flush(d_pre, a.part_pre + (int64_t)blockIdx.x * d, nullptr);
}

// The workgroups' shares summed in order and rounded: job 0 dpost, 1 dpre, 2 + j the gate's run j where several workgroups have
// a share of it. COLS columns and 1024 / COLS groups of shares per workgroup. 5 us at 16384 x 768, 10 us at five runs of 1365 x 2048
// (162 us with a job for every share).
constexpr int SUM_LANES = 1024;
template <typename T, int COLS>
__global__ __launch_bounds__(SUM_LANES) void k_join_sum(const JoinBwd<T> a, T* __restrict__ d_post, T* __restrict__ d_pre, int parts,
                                                        int job0) {
  constexpr int GROUPS = SUM_LANES / COLS;
  __shared__ float s[SUM_LANES];
  const int job = job0 + (int)blockIdx.y, d = a.d, c = (int)blockIdx.x * COLS + (int)threadIdx.x % COLS;
  const float *first, *rest;   // share 0, and share i > 0 at rest + i * step
  int64_t step = d;
  int count = parts;
  T* out;
  if (job == 0) {
    if (!a.part_post) return;
    first = rest = a.part_post;
    out = d_post;
  } else if (job == 1) {
    if (!a.part_pre) return;
    first = rest = a.part_pre;
    out = d_pre;
  } else {
    const int64_t run = job - 2, g0 = run * a.gate_rows, g1 = min((int64_t)a.rows, g0 + a.gate_rows), b = g0 / a.per;
    count = (int)((g1 - 1) / a.per - b + 1);
    if (count == 1) return;
    first = a.part_gate + (2 * b + 1) * d;
    rest = a.part_gate + 2 * b * d;
    step = 2 * (int64_t)d;
    out = a.dgate + run * d;
  }
  const int grp = (int)threadIdx.x / COLS;
  float acc = 0.f;
  if (c < d) {
    int i = grp;
    if (i == 0) {
      acc = first[c];
      i = GROUPS;
    }
    for (; i + 3 * GROUPS < count; i += 4 * GROUPS) {   // four shares' loads in flight
      float e[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) e[u] = rest[(i + u * GROUPS) * step + c];
#pragma unroll
      for (int u = 0; u < 4; ++u) acc += e[u];
    }
    for (; i < count; i += GROUPS) acc += rest[i * step + c];
  }
  s[threadIdx.x] = acc;
  __syncthreads();
  for (int w = GROUPS / 2; w > 0; w >>= 1) {
    if (grp < w) s[threadIdx.x] += s[threadIdx.x + COLS * w];
    __syncthreads();
  }
  if (grp == 0 && c < d) st1(out + c, s[threadIdx.x]);
}

// ---------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------
inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool al_of(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == LDR_F32 ? 3u : 1u)) == 0; }
inline bool dtype_ok(int dt) { return dt == LDR_F32 || dt == LDR_BF16 || dt == LDR_F16; }
inline unsigned grid_of(int64_t blocks, int64_t cap) { return (unsigned)(blocks < cap ? blocks : cap); }
inline int launched() { return (int)hipGetLastError(); }

// lanes per row, eight columns each: 4, 16 or 64 of a wave, or 2 to 16 waves
inline int lanes_per_row(int64_t d) {
  return d <= 32 ? 4 : d <= 128 ? 16 : d <= 512 ? 64 : d <= 1024 ? 128 : d <= 2048 ? 256 : d <= 4096 ? 512 : 1024;
}

// workgroups of the backward and the consecutive rows each takes: three workgroups per CU of 256 lanes where there are rows
// for them. Gate runs no longer than that are not cut.
struct Plan { int64_t per, parts; };
inline Plan plan_of(int64_t rows, int64_t d, int64_t gate_rows) {
  const int lpr = lanes_per_row(d), r = lpr > WG ? 1 : WG / lpr;
  const int64_t most = lpr > 512 ? 256 : lpr > WG ? 384 : 768;
  int64_t per = (rows + most - 1) / most;
  per = (per + r - 1) / r * r;
  if (gate_rows > 1 && gate_rows <= per) per = per / gate_rows * gate_rows;
  return Plan{per, (rows + per - 1) / per};
}

#define LBK_TYPE_SWITCH(DT, ...)                                 \
  if ((DT) == LDR_BF16) { typedef bf16_t T; __VA_ARGS__; }       \
  else if ((DT) == LDR_F16) { typedef _Float16 T; __VA_ARGS__; } \
  else { typedef float T; __VA_ARGS__; }
#define LBK_LANES_SWITCH(N, ...)                                      \
  switch (N) {                                                        \
    case 4: { constexpr int LPR = 4; __VA_ARGS__; } break;            \
    case 16: { constexpr int LPR = 16; __VA_ARGS__; } break;          \
    case 64: { constexpr int LPR = 64; __VA_ARGS__; } break;          \
    case 128: { constexpr int LPR = 128; __VA_ARGS__; } break;        \
    case 256: { constexpr int LPR = 256; __VA_ARGS__; } break;        \
    case 512: { constexpr int LPR = 512; __VA_ARGS__; } break;        \
    default: { constexpr int LPR = 1024; __VA_ARGS__; } break;        \
  }

#define LBK_PARTS_SWITCH(P, ...)                                 \
  switch (P) {                                                   \
    case 0: { constexpr int PARTS = 0; __VA_ARGS__; } break;     \
    case 1: { constexpr int PARTS = 1; __VA_ARGS__; } break;     \
    case 2: { constexpr int PARTS = 2; __VA_ARGS__; } break;     \
    case 3: { constexpr int PARTS = 3; __VA_ARGS__; } break;     \
    case 4: { constexpr int PARTS = 4; __VA_ARGS__; } break;     \
    case 5: { constexpr int PARTS = 5; __VA_ARGS__; } break;     \
    case 6: { constexpr int PARTS = 6; __VA_ARGS__; } break;     \
    default: { constexpr int PARTS = 7; __VA_ARGS__; } break;    \
  }

}  // namespace

extern "C" {

int lbk_abi_version(void) { return LBK_ABI_VERSION; }

int lbk_dropout(const void* x, const int64_t* rng, uint32_t site, int drop, void* out, int64_t rows, int64_t d, int dtype,
                void* stream) {
  if (!dtype_ok(dtype)) return LDR_E_DTYPE;
  if (rows < 0 || d < 1 || drop < 0 || drop > 65536) return LDR_E_ARG;
  if (rows > 0x7fffffff || d > ((int64_t)1 << 35)) return LDR_E_SHAPE;
  if (rows == 0) return LDR_OK;
  if (!x || !rng || !out) return LDR_E_ARG;
  if (!al_of(x, dtype) || !al_of(out, dtype) || (reinterpret_cast<uintptr_t>(rng) & 7u)) return LDR_E_ALIGN;
  const int64_t nb = (d + 7) / 8;
  const bool al = d % 8 == 0 && al16(x) && al16(out);
  const unsigned grid = grid_of((rows * nb + WG - 1) / WG, 8192);
  hipStream_t st = static_cast<hipStream_t>(stream);
  LBK_TYPE_SWITCH(dtype, {
    if (al)
      hipLaunchKernelGGL((k_dropout<T, true>), dim3(grid), dim3(WG), 0, st, static_cast<const T*>(x), rng, site,
                         (uint32_t)drop, keep_scale(drop), static_cast<T*>(out), rows, d, nb);
    else
      hipLaunchKernelGGL((k_dropout<T, false>), dim3(grid), dim3(WG), 0, st, static_cast<const T*>(x), rng, site,
                         (uint32_t)drop, keep_scale(drop), static_cast<T*>(out), rows, d, nb);
  })
  return launched();
}

static int join_shape(int64_t rows, int64_t d, int64_t gate_rows, const void* gate, int drop, const int64_t* rng, int dtype) {
  if (!dtype_ok(dtype)) return LDR_E_DTYPE;
  if (rows < 0 || d < 1 || drop < 0 || drop > 65536 || (gate && gate_rows < 1)) return LDR_E_ARG;
  if (rows > 0x7fffffff || d > LBK_JOIN_MAX_WIDTH) return LDR_E_SHAPE;
  if (drop && (!rng || (reinterpret_cast<uintptr_t>(rng) & 7u))) return rng ? LDR_E_ALIGN : LDR_E_ARG;
  return LDR_OK;
}

int lbk_join_fwd(const void* x, const void* y, const void* post, const void* gate, int64_t gate_rows, const void* pre,
                 const int64_t* rng, uint32_t site, int drop, float scale, float eps, void* h, void* n, float* r_post,
                 float* r_pre, int64_t rows, int64_t d, int dtype, void* stream) {
  if (rows == 0) drop = 0;
  const int e = join_shape(rows, d, gate_rows, gate, drop, rng, dtype);
  if (e || rows == 0) return e;
  if (!x || !y || !h || (pre && !n)) return LDR_E_ARG;
  bool al = d % 8 == 0;
  for (const void* p : {x, y, post, gate, pre, (const void*)h, (const void*)n}) {
    if (!al_of(p, dtype)) return LDR_E_ALIGN;
    al = al && al16(p);
  }
  const int lpr = lanes_per_row(d), r = lpr > WG ? 1 : WG / lpr;
  const unsigned grid = grid_of((rows + r - 1) / r, lpr > WG ? 1024 : 2048);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t gr = !gate || gate_rows > rows ? rows : gate_rows;
  LBK_TYPE_SWITCH(dtype, {
    const JoinFwd<T> a{static_cast<const T*>(x), static_cast<const T*>(y), static_cast<const T*>(post),
                       static_cast<const T*>(gate), static_cast<const T*>(pre), rng, static_cast<T*>(h),
                       static_cast<T*>(n), r_post, r_pre, (int)rows, (int)d, (int)gr, site, (uint32_t)drop, scale,
                       keep_scale(drop), eps};
    LBK_LANES_SWITCH(lpr, {
      if (al) {
        LBK_PARTS_SWITCH((pre ? 1 : 0) + (post ? 2 : 0) + (drop ? 4 : 0),
                         hipLaunchKernelGGL((k_join_fwd<T, LPR, true, PARTS>), dim3(grid), dim3(lanes_of(LPR)), 0, st, a))
      } else {
        hipLaunchKernelGGL((k_join_fwd<T, LPR, false, ANY>), dim3(grid), dim3(lanes_of(LPR)), 0, st, a);
      }
    })
  })
  return launched();
}

int64_t lbk_join_scratch(int64_t rows, int64_t d, int64_t gate_rows) {
  if (rows < 1 || d < 1 || d > LBK_JOIN_MAX_WIDTH) return 0;
  return plan_of(rows, d, gate_rows).parts * 4 * d;
}

int lbk_join_bwd(const void* dh, const void* dn, const void* x, const void* y, const void* post, const void* gate,
                 int64_t gate_rows, const void* pre, const float* r_post, const float* r_pre, const int64_t* rng,
                 uint32_t site, int drop, float scale, void* dx, void* dy, void* dpost, void* dgate, void* dpre,
                 float* scratch, int64_t rows, int64_t d, int dtype, void* stream) {
  if (rows == 0) drop = 0;
  const int e = join_shape(rows, d, gate_rows, gate, drop, rng, dtype);
  if (e || rows == 0) return e;
  if ((!dh && !dn) || !y || (dn && (!x || !pre || !r_pre)) || (post && !r_post)) return LDR_E_ARG;
  if ((dpost && !post) || (dgate && !gate) || (dpre && !dn)) return LDR_E_ARG;
  if (!dx && !dy && !dpost && !dgate && !dpre) return LDR_OK;
  if ((dpost || dgate || dpre) && !scratch) return LDR_E_ARG;
  bool al = d % 8 == 0;
  for (const void* p : {dh, dn, x, y, post, gate, pre, (const void*)dx, (const void*)dy, (const void*)dgate,
                        (const void*)scratch}) {
    if (!al_of(p, dtype)) return LDR_E_ALIGN;
    al = al && al16(p);
  }
  if (!al_of(scratch, LDR_F32) || !al_of(dpost, dtype) || !al_of(dpre, dtype)) return LDR_E_ALIGN;
  const int64_t gr = !gate || gate_rows > rows ? rows : gate_rows;
  const Plan plan = plan_of(rows, d, gate ? gate_rows : rows);
  const int parts = (int)plan.parts;
  hipStream_t st = static_cast<hipStream_t>(stream);
  LBK_TYPE_SWITCH(dtype, {
    const JoinBwd<T> a{static_cast<const T*>(dh), static_cast<const T*>(dn), static_cast<const T*>(x),
                       static_cast<const T*>(y), static_cast<const T*>(post), static_cast<const T*>(gate),
                       static_cast<const T*>(pre), r_post, r_pre, rng, static_cast<T*>(dx), static_cast<T*>(dy),
                       static_cast<T*>(dgate), dpost ? scratch : nullptr, dpre ? scratch + parts * d : nullptr,
                       scratch + 2 * parts * d, (int)rows, (int)d, (int)gr, (int)plan.per, site, (uint32_t)drop, scale,
                       keep_scale(drop)};
    LBK_LANES_SWITCH(lanes_per_row(d), {
      if (al) {
        LBK_PARTS_SWITCH((dn ? 1 : 0) + (post ? 2 : 0) + (drop ? 4 : 0),
                         hipLaunchKernelGGL((k_join_bwd<T, LPR, true, PARTS>), dim3(parts), dim3(lanes_of(LPR)), 0, st, a))
      } else if constexpr (LPR == 1024) {   // 128 registers a lane: looked up, 108 spill (16384 x 5001 with all parts: 999 us, 390 so)
        LBK_PARTS_SWITCH((dn ? 1 : 0) + (post ? 2 : 0) + (drop ? 4 : 0),
                         hipLaunchKernelGGL((k_join_bwd<T, LPR, false, PARTS>), dim3(parts), dim3(lanes_of(LPR)), 0, st, a))
      } else {
        hipLaunchKernelGGL((k_join_bwd<T, LPR, false, ANY>), dim3(parts), dim3(lanes_of(LPR)), 0, st, a);
      }
    })
    const int err = launched();
    if (err) return err;
    // a gate's runs that several workgroups have a share of: none where they are not cut. One over many workgroups is summed
    // beside the weights' sums, in groups of shares; short ones with more columns to a workgroup
    const int64_t runs = !dgate || gr == 1 || plan.per % gr == 0 ? 0 : (rows + gr - 1) / gr;
    const bool beside = runs > 0 && (gr >= 32 * plan.per);
    const unsigned jobs = beside ? 2 + (unsigned)runs : 2;
    if (dpost || dpre || beside)
      hipLaunchKernelGGL((k_join_sum<T, 16>), dim3((unsigned)((d + 15) / 16), jobs), dim3(SUM_LANES), 0, st, a,
                         static_cast<T*>(dpost), static_cast<T*>(dpre), parts, 0);
    if (runs && !beside)
      hipLaunchKernelGGL((k_join_sum<T, 256>), dim3((unsigned)((d + 255) / 256), (unsigned)runs), dim3(SUM_LANES), 0, st, a,
                         static_cast<T*>(dpost), static_cast<T*>(dpre), parts, 2);
  })
  return launched();
}

}  // extern "C"
