// loopback_model.hip -- MI355X (gfx950, CDNA4) kernels of layer norm and of the distillation loss from a teacher's highest
// logits, forward and backward. All are bound by the HBM stream of their rows: fp32 statistics, one rounding per result.
// Every sum has a fixed order: results are deterministic.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include <type_traits>

#include "loopback_model.h"
#include "loopback_read.h"
#include "lds_limit.h"
#include "row_io.h"

namespace {

// ---------------------------------------------------------------------------------------------------------------
// layer norm. LPR lanes to a row, VPT times eight columns each, the whole row in registers: the mean, then the squares of
// the differences from it (not the mean of squares, which would cancel where the mean is large), then the result. Bound by the
// rows' stream: 16384 x 768 bf16 with the add 18.5 us (101 MB, 5.4 TB/s), 8192 x 8192 49 (268 MB, 5.4 TB/s).
// ---------------------------------------------------------------------------------------------------------------
template <typename T> struct NormFwd {
  const T *x, *add, *w, *b;
  T *h, *y;
  float* stats;
  int rows, d;
  float eps;
};

template <typename T, int LPR, int VPT, bool AL>
__global__ __launch_bounds__(lanes_of(LPR)) void k_layer_norm_fwd(const NormFwd<T> a) {
  constexpr int LANES = lanes_of(LPR), R = LANES / LPR;
  __shared__ float s_red[2][LANES / 64];
  RowSum<LPR> row_sum{s_red};
  const int d = a.d, lane = (int)threadIdx.x % LPR, grp = group_of<LPR>();
  const float inv_d = 1.f / (float)d;
  for (int64_t row0 = (int64_t)blockIdx.x * R; row0 < a.rows; row0 += (int64_t)gridDim.x * R) {
    const bool ok = row0 + grp < a.rows;
    const int64_t row = ok ? row0 + grp : a.rows - 1, ro = row * d;
    typename IO<T>::Raw xr[VPT], ar[VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      xr[v] = load8<T, AL>(a.x + ro, 8 * (lane + LPR * v), d);
      if (a.add) ar[v] = load8<T, AL>(a.add + ro, 8 * (lane + LPR * v), d);
    }
    float h[VPT][8], m = 0.f, ss = 0.f;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      IO<T>::unpack(xr[v], h[v]);
      if (a.add) {
        float e[8];
        IO<T>::unpack(ar[v], e);
#pragma unroll
        for (int k = 0; k < 8; ++k) h[v][k] = IO<T>::round(h[v][k] + e[k]);
        if (ok) store8<T, AL>(a.h + ro, 8 * (lane + LPR * v), d, h[v]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) m += h[v][k];   // zeros past the row's end
    }
    m = row_sum(m) * inv_d;
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        h[v][k] -= m;
        const bool in = 8 * (lane + LPR * v) + (AL ? 0 : k) < d;
        ss = in ? __builtin_fmaf(h[v][k], h[v][k], ss) : ss;
      }
    const float r = rsqrtf(row_sum(ss) * inv_d + a.eps);
    if (a.stats && lane == 0 && ok) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(m, r);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int col = 8 * (lane + LPR * v);
      float e[8];
      if (a.w) {
        IO<T>::unpack(load8<T, AL>(a.w, col, d), e);
#pragma unroll
        for (int k = 0; k < 8; ++k) h[v][k] *= r * e[k];
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) h[v][k] *= r;
      }
      if (a.b) {
        IO<T>::unpack(load8<T, AL>(a.b, col, d), e);
#pragma unroll
        for (int k = 0; k < 8; ++k) h[v][k] += e[k];
      }
      if (ok) store8<T, AL>(a.y + ro, col, d, h[v]);
    }
  }
}

template <typename T> struct NormBwd {
  const T *dy, *h, *w;
  const float* stats;
  const T* dres;
  T* dx;
  float *part_w, *part_b;   // [workgroups][d]; NULL: not wanted
  int rows, d, per;
};

// A workgroup takes `per` consecutive rows and keeps the columns' sums of dy hat and dy in registers; its row groups' sums
// meet in LDS, one partial row a workgroup. Bound by the rows' stream and the few waves that the sums' registers leave: 16384 x 768
// bf16 with the residual's gradient 21.6 us (101 MB, 4.7 TB/s), 8192 x 8192 84 (403 MB, 4.8 TB/s); the next row's loads ahead spill
// in wide rows (118 us) and gain nothing in narrow ones.
template <typename T, int LPR, int VPT, bool AL>
__global__ __launch_bounds__(lanes_of(LPR)) void k_layer_norm_bwd(const NormBwd<T> a) {
  constexpr int LANES = lanes_of(LPR), R = LANES / LPR, W = 8 * LPR * VPT;
  __shared__ float s_red[2][LANES / 64];
  __shared__ float s_sum[R > 1 ? R * W : 1];
  RowSum<LPR> row_sum{s_red};
  const int d = a.d, lane = (int)threadIdx.x % LPR, grp = group_of<LPR>();
  const float inv_d = 1.f / (float)d;
  typename IO<T>::Raw wr[VPT];
  float dw[VPT][8], db[VPT][8];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    wr[v] = a.w ? load8<T, AL>(a.w, 8 * (lane + LPR * v), d) : IO<T>::zero();
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[v][k] = db[v][k] = 0.f;
  }
  const int64_t r0 = (int64_t)blockIdx.x * a.per, r1 = min((int64_t)a.rows, r0 + a.per);
  for (int64_t row0 = r0; row0 < r1; row0 += R) {
    const bool ok = row0 + grp < r1, there = R == 1 || ok;   // a row that is not there adds nothing to the sums
    const int64_t row = ok ? row0 + grp : r1 - 1, ro = row * d;
    typename IO<T>::Raw yr[VPT], hr[VPT], rr[VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int col = 8 * (lane + LPR * v);
      yr[v] = load8<T, AL>(a.dy + ro, col, d);
      hr[v] = load8<T, AL>(a.h + ro, col, d);
      if (a.dres) rr[v] = load8<T, AL>(a.dres + ro, col, d);
      anew<T>(wr[v]);
    }
    const float2 st = *reinterpret_cast<const float2*>(a.stats + 2 * row);
    float t[VPT][8], hat[VPT][8], c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float w[8];
      IO<T>::unpack(yr[v], t[v]);
      IO<T>::unpack(hr[v], hat[v]);
      if (a.w) IO<T>::unpack(wr[v], w);
      const int left = d - 8 * (lane + LPR * v);
      const float rstd = left > 0 ? st.y : 0.f;   // past the row's end: -m r can be infinite, and is multiplied by a zero
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float g = t[v][k], x = AL || k < left ? (hat[v][k] - st.x) * rstd : 0.f;
        hat[v][k] = x;
        if (there) {
          dw[v][k] = __builtin_fmaf(g, x, dw[v][k]);
          db[v][k] += g;
        }
        const float u = a.w ? g * w[k] : g;   // zeros past the row's end
        t[v][k] = u;
        c1 += u;
        c2 = __builtin_fmaf(u, x, c2);
      }
    }
    if (!a.dx) continue;
    c1 = row_sum(c1) * inv_d;
    c2 = row_sum(c2) * inv_d;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float e[8];
      if (a.dres) IO<T>::unpack(rr[v], e);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        t[v][k] = st.y * (t[v][k] - c1 - hat[v][k] * c2);
        if (a.dres) t[v][k] += e[k];
      }
      if (ok) store8<T, AL>(a.dx + ro, 8 * (lane + LPR * v), d, t[v]);
    }
  }
  auto flush = [&](float (&acc)[VPT][8], float* out) {
    if constexpr (R == 1) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) store8<float, AL>(out, 8 * (lane + LPR * v), d, acc[v]);
    } else {
      __syncthreads();
#pragma unroll
      for (int v = 0; v < VPT; ++v) IO<float>::store(s_sum + grp * W + 8 * (lane + LPR * v), acc[v]);
      __syncthreads();
      for (int c = (int)threadIdx.x; c < d; c += LANES) {
        float s = s_sum[c];
        for (int g = 1; g < R; ++g) s += s_sum[g * W + c];
        out[c] = s;
      }
    }
  };
  if (a.part_w) flush(dw, a.part_w + (int64_t)blockIdx.x * d);
  if (a.part_b) flush(db, a.part_b + (int64_t)blockIdx.x * d);
}

// dw (blockIdx.y 0) and db (1): the workgroups' partial rows summed in order by a workgroup's groups of COLS lanes, then the groups.
// Wide rows take whole lines of 256 bytes (512 x 8192: 6.5 us, 11.6 by 64); of narrow ones the workgroups would be too few
constexpr int SUM_LANES = 1024;
template <typename T, int SUM_COLS>
__global__ __launch_bounds__(SUM_LANES) void k_layer_norm_sum(const float* __restrict__ part_w, const float* __restrict__ part_b,
                                                              T* __restrict__ dw, T* __restrict__ db, int parts, int d) {
  constexpr int GROUPS = SUM_LANES / SUM_COLS;
  __shared__ float s[SUM_LANES];
  const float* part = blockIdx.y ? part_b : part_w;
  T* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int tid = (int)threadIdx.x, c = (int)blockIdx.x * SUM_COLS + tid % SUM_COLS, grp = tid / SUM_COLS;
  float acc = 0.f;
  if (c < d) {
    int i = grp;
    for (; i + 3 * GROUPS < parts; i += 4 * GROUPS) {   // four partial rows' loads in flight
      float e[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) e[u] = part[(int64_t)(i + u * GROUPS) * d + c];
#pragma unroll
      for (int u = 0; u < 4; ++u) acc += e[u];
    }
    for (; i < parts; i += GROUPS) acc += part[(int64_t)i * d + c];
  }
  s[tid] = acc;
  __syncthreads();
  for (int w = GROUPS / 2; w > 0; w >>= 1) {
    if (grp < w) s[tid] += s[tid + SUM_COLS * w];
    __syncthreads();
  }
  if (grp == 0 && c < d) st1(out + c, s[tid]);
}

// ---------------------------------------------------------------------------------------------------------------
// distillation. One workgroup per row of logits. The forward streams it once: a running maximum m and the sums of
// exp((x - m) / tau) and, with labels at a temperature, of exp(x - m); with a teacher_lse the named classes, marked in a
// bitmap in LDS (a byte for the eight logits of a vector), are summed apart from the others, so that the others' share
// q_rest never comes from a difference. The backward streams the row again and writes the gradient as if no class were
// named, then, past a barrier, the row's k named elements and the label's once more with theirs. 16384 x 32000 bf16, 64 classes, labels
// at temperature 2: forward 195 us (1.05 GB, 5.4 TB/s; the vector units are busy for some two thirds of it), gradient 388 (2.1 GB,
// 5.4 TB/s; a copy of these sizes takes 335 to 405).
// ---------------------------------------------------------------------------------------------------------------
constexpr float LOG2E = 1.4426950408889634f;

// what the forward keeps of a row: its terms (all rows' first, side by side for their mean), and what its gradient needs
struct DistillTerms {
  float kl, ce;
  float counts, labelled; // 1 or 0
};
struct alignas(16) DistillRow {
  float m, l, l1;         // the maximum, and the logs of the sums of exp((x - m) / tau) and exp(x - m)
  float mr, lr;           // the same of the classes that are not named
  float all, rest;        // P + rest, and rest
  float teacher;          // p_i = exp(top_i / tau - teacher)
};
static_assert(sizeof(DistillTerms) + sizeof(DistillRow) == LMO_DISTILL_SAVED * sizeof(float), "saved row");

struct Sums {   // running maximum, sum of exp((x - m) / tau) and, HARD, of exp(x - m)
  float m = -INFINITY, s = 0.f, s1 = 0.f;
};
template <bool HARD> __device__ __forceinline__ void grow(Sums& a, float mx, float c, float c1) {   // the maximum, to mx at least
  if (mx > a.m) {
    a.s *= __builtin_amdgcn_exp2f((a.m - mx) * c);
    if (HARD) a.s1 *= __builtin_amdgcn_exp2f((a.m - mx) * c1);
    a.m = mx;
  }
}
template <bool HARD> __device__ __forceinline__ void take(Sums& a, float x, float c, float c1) {
  if (x != x) {
    a.s = a.s1 = x;
    if (a.m == -INFINITY) a.m = 0.f;
    return;
  }
  grow<HARD>(a, x, c, c1);
  if (a.m == -INFINITY) return;
  a.s += __builtin_amdgcn_exp2f((x - a.m) * c);
  if (HARD) a.s1 += __builtin_amdgcn_exp2f((x - a.m) * c1);
}
// two sets of sums as one
template <bool HARD> __device__ __forceinline__ Sums joined(const Sums& a, const Sums& b, float c, float c1) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float fa = a.m == r.m ? 1.f : exp2f((a.m - r.m) * c), fb = b.m == r.m ? 1.f : exp2f((b.m - r.m) * c);
  r.s = a.s * fa + b.s * fb;
  if (HARD) {
    const float ga = a.m == r.m ? 1.f : exp2f((a.m - r.m) * c1), gb = b.m == r.m ? 1.f : exp2f((b.m - r.m) * c1);
    r.s1 = a.s1 * ga + b.s1 * gb;
  }
  return r;
}
template <typename Op, int WAVES> __device__ __forceinline__ float wg_reduce(float v, float* red, Op op) {   // to every lane
  v = lanes_reduce(v, 64, op);
  __syncthreads();   // red may still be read from the reduction before
  if (((int)threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int k = 1; k < WAVES; ++k) v = op(v, red[k]);
  return v;
}
// the lanes' sums as the workgroup's (fmaxf skips a NaN maximum; sums carry it)
template <bool HARD, int WAVES> __device__ __forceinline__ Sums wg_joined(Sums a, float* red, float c, float c1) {
  Sums r;
  r.m = wg_reduce<MaxOp, WAVES>(a.m, red, MaxOp());
  r.s = wg_reduce<AddOp, WAVES>(a.m == r.m ? a.s : a.s * exp2f((a.m - r.m) * c), red, AddOp());
  if (HARD) r.s1 = wg_reduce<AddOp, WAVES>(a.m == r.m ? a.s1 : a.s1 * exp2f((a.m - r.m) * c1), red, AddOp());
  return r;
}

__device__ __forceinline__ float ld_as(const void* p, int64_t i, int dtype) {
  return dtype == LDR_F32 ? static_cast<const float*>(p)[i]
         : dtype == LDR_BF16 ? ld1(static_cast<const bf16_t*>(p) + i) : ld1(static_cast<const _Float16*>(p) + i);
}
// a named class as an int: -1 names nothing, vocab stands for any past the last
__device__ __forceinline__ int id_of(const void* ids, int wide, int64_t i, int vocab) {
  const int64_t v = wide ? static_cast<const int64_t*>(ids)[i] : (int64_t) static_cast<const int32_t*>(ids)[i];
  return v < 0 ? -1 : v >= vocab ? vocab : (int)v;
}

struct Distill {
  const void *logits, *top, *ids;
  const float* teacher_lse;
  const int64_t* labels;
  DistillTerms* terms;
  DistillRow* saved;
  const float *coef, *dloss;
  void* dlogits;
  int vocab, k, top_dtype, wide;
  float tau;
  int64_t row0;   // of this launch's first row
  int parts;      // the backward's workgroups of a row
};

// U vectors of eight that a lane takes at a time, NT: past the caches (16384 x 32000 bf16: forward 195 us, 204 through them, gradient
// 387, 461; 1001 x 50257 fp16, which the caches hold: 31 and 42 past them, 26 and 35 through)
template <typename T, int LANES, int U, bool NT> struct Vectors {
  typename IO<T>::Raw r[U];
  __device__ __forceinline__ void load(const T* x, int v0, int nv) {   // past the end: the last one again
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const T* p = x + 8 * (int64_t)min(v0 + (int)threadIdx.x + u * LANES, nv - 1);
      r[u] = NT ? UIO<T>::raw_nt(p) : UIO<T>::raw(p);
    }
  }
};
template <typename T, bool NT> __device__ __forceinline__ void store_stream(T* p, const float (&o)[8]) {
  if constexpr (!NT) {
    UIO<T>::store(p, o);
  } else if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 8; i += 4)
      __builtin_nontemporal_store(u32x4{__float_as_uint(o[i]), __float_as_uint(o[i + 1]), __float_as_uint(o[i + 2]), __float_as_uint(o[i + 3])},
                                  reinterpret_cast<u32x4_u32*>(p + i));
  } else {
    typedef typename std::conditional<std::is_same<T, bf16_t>::value, Bf16Cvt, F16Cvt>::type Cvt;
    __builtin_nontemporal_store(u32x4{Cvt::pack2(o[0], o[1]), Cvt::pack2(o[2], o[3]), Cvt::pack2(o[4], o[5]), Cvt::pack2(o[6], o[7])},
                                reinterpret_cast<u32x4_u16*>(p));
  }
}

// POW: 0 no second sum (no labels, or temperature 1, where it is the first); 2 and 4 temperatures whose exp((x - m) / tau), squared
// once or twice, is the second sum's exponential (16384 x 32000: 239 -> 195 us, with the maximum once for 16 logits); 1 any other
template <typename T, int LANES, bool TAIL, int POW, bool NT>
__global__ __launch_bounds__(LANES) void k_distill_fwd(const Distill a) {
  constexpr int WAVES = LANES / 64, U = sizeof(T) == 4 ? 1 : 2, STEP = U * LANES;
  constexpr bool HARD = POW != 0;
  extern __shared__ unsigned s_map[];   // TAIL: the named classes' bits, 32 to a word
  __shared__ float red[WAVES];
  const int64_t row = a.row0 + blockIdx.x;
  const int vocab = a.vocab, k = a.k, tid = (int)threadIdx.x, nv = vocab >> 3;
  const T* x = static_cast<const T*>(a.logits) + row * vocab;
  const float c = LOG2E / a.tau, c1 = LOG2E;
  const int64_t label = a.labels ? a.labels[row] : -100;
  // the teacher: which classes count, its maximum and sum
  float zm = -INFINITY, named = 0.f;   // named: 1 with a class that counts, 2 with one past the last
  for (int i = tid; i < k; i += LANES) {
    const int id = id_of(a.ids, a.wide, row * k + i, vocab);
    if (id < 0) continue;
    named = fmaxf(named, id >= vocab ? 2.f : 1.f);
    zm = fmaxf(zm, ld_as(a.top, row * k + i, a.top_dtype) * c);
  }
  named = wg_reduce<MaxOp, WAVES>(named, red, MaxOp());
  const bool counts = named > 0.f;
  const bool labelled = label != -100;
  DistillRow out{};
  DistillTerms terms{};
  if (!counts && !labelled) {   // workgroup-uniform
    if (tid == 0) {
      a.terms[row] = terms;
      a.saved[row] = out;
    }
    return;
  }
  if (TAIL) {
    const int words = (vocab + 31) >> 5;
    for (int i = tid; i < words; i += LANES) s_map[i] = 0u;
    __syncthreads();
    for (int i = tid; i < k; i += LANES) {
      const int id = id_of(a.ids, a.wide, row * k + i, vocab);
      if (id >= 0 && id < vocab) atomicOr(s_map + (id >> 5), 1u << (id & 31));   // bits: no order to depend on
    }
    __syncthreads();
  }
  float others = 1.f;   // whether a class is left that is not named
  if (TAIL && k >= vocab) {
    float n = 0.f;
    for (int i = tid; i < (vocab + 31) >> 5; i += LANES) n += (float)__popc(s_map[i]);
    others = wg_reduce<AddOp, WAVES>(n, red, AddOp()) < (float)vocab ? 1.f : 0.f;
  }
  Sums s, sn;   // of the classes (TAIL: those not named), and of the named ones
  auto use = [&](const Vectors<T, LANES, U, NT>& from, int v0) {
    float e[U][8], mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + tid + u * LANES;
      IO<T>::unpack(from.r[u], e[u]);
      if (v >= nv) {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[u][j] = -INFINITY;
      } else if (TAIL) {
        const unsigned bits = reinterpret_cast<const unsigned char*>(s_map)[v];
        if (bits) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (bits >> j & 1u) {
              take<HARD>(sn, e[u][j], c, c1);
              e[u][j] = -INFINITY;
            }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) mx = fmaxf(mx, e[u][j]);   // passes a NaN over, which the sums keep
    }
    grow<HARD>(s, mx, c, c1);
    const float m = s.m == -INFINITY ? 0.f : s.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float t = 0.f, t1 = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = e[u][j] - m, x1 = __builtin_amdgcn_exp2f(d * c), x2 = x1 * x1;
        t += x1;
        if (POW == 1) t1 += __builtin_amdgcn_exp2f(d * c1);
        else if (POW == 2) t1 = __builtin_fmaf(x1, x1, t1);
        else if (POW == 4) t1 = __builtin_fmaf(x2, x2, t1);
      }
      s.s += t;
      if (HARD) s.s1 += t1;
    }
  };
  if (nv > 0) {   // the next vectors' loads are in flight while these are summed
    Vectors<T, LANES, U, NT> r0, r1;
    r0.load(x, 0, nv);
    for (int v0 = 0; v0 < nv; v0 += 2 * STEP) {   // the same for every lane
      if (v0 + STEP < nv) r1.load(x, v0 + STEP, nv);
      use(r0, v0);
      if (v0 + 2 * STEP < nv) r0.load(x, v0 + 2 * STEP, nv);
      if (v0 + STEP < nv) use(r1, v0 + STEP);
    }
  }
  if (tid < (vocab & 7)) {
    const int i = 8 * nv + tid;
    if (TAIL && (s_map[i >> 5] >> (i & 31) & 1u)) take<HARD>(sn, ld1(x + i), c, c1);
    else take<HARD>(s, ld1(x + i), c, c1);
  }
  s = wg_joined<HARD, WAVES>(s, red, c, c1);
  if (TAIL) {
    out.mr = s.m;
    out.lr = logf(s.s);
    s = joined<HARD>(s, wg_joined<HARD, WAVES>(sn, red, c, c1), c, c1);
  }
  out.m = s.m;
  out.l = logf(s.s);   // kept apart from the maximum: their sum would lose it beside large logits
  out.l1 = HARD ? logf(s.s1) : out.l;
  if (counts) {
    // p_i = exp(z_i - teacher) of z = top / tau
    float teacher;
    if (TAIL) {
      teacher = a.teacher_lse[row];
    } else {
      zm = wg_reduce<MaxOp, WAVES>(zm, red, MaxOp());
      float zs = 0.f;
      for (int i = tid; i < k; i += LANES)
        if (id_of(a.ids, a.wide, row * k + i, vocab) >= 0) zs += exp2f(ld_as(a.top, row * k + i, a.top_dtype) * c - zm);
      zs = wg_reduce<AddOp, WAVES>(zs, red, AddOp());
      teacher = (zm + log2f(zs)) * (1.f / LOG2E);
    }
    const float inv_tau = 1.f / a.tau;
    float kl = 0.f, P = 0.f;
    for (int i = tid; i < k; i += LANES) {
      const int id = id_of(a.ids, a.wide, row * k + i, vocab);
      if (id < 0 || id >= vocab) continue;
      const float lp = ld_as(a.top, row * k + i, a.top_dtype) * inv_tau - teacher, p = expf(lp);
      P += p;
      if (!(p <= 0.f)) kl += p * (lp - ((ld1(x + id) - s.m) * inv_tau - out.l));
    }
    kl = wg_reduce<AddOp, WAVES>(kl, red, AddOp());
    P = wg_reduce<AddOp, WAVES>(P, red, AddOp());
    if (TAIL) {
      out.rest = P != P ? P : others * fmaxf(0.f, 1.f - P);
      if (out.rest > 0.f) kl += out.rest * (logf(out.rest) - ((out.mr - out.m) * inv_tau + out.lr - out.l));
    }
    terms.kl = named > 1.f ? NAN : kl;
    out.all = P + out.rest;
    terms.counts = 1.f;
    out.teacher = teacher;
  }
  if (labelled) {
    terms.ce = label >= 0 && label < vocab ? out.l1 + (out.m - ld1(x + label)) : NAN;
    terms.labelled = 1.f;
  }
  if (tid == 0) {
    a.terms[row] = terms;
    a.saved[row] = out;
  }
}

// the loss, and what the rows' gradients are multiplied by, by one workgroup: lane sums in order, then a fixed tree
constexpr int MEAN_LANES = 1024;
__global__ __launch_bounds__(MEAN_LANES) void k_distill_mean(const DistillTerms* __restrict__ terms, int64_t rows, float tau,
                                                             float hard, float* __restrict__ coef, float* __restrict__ loss) {
  __shared__ float4 s[MEAN_LANES];
  const int tid = (int)threadIdx.x;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [](float4& p, const float4& q) {
    p.x += q.x;
    p.y += q.y;
    p.z += q.z;
    p.w += q.w;
  };
  int64_t i = tid;
  const float4* row = reinterpret_cast<const float4*>(terms);
  for (; i + 7 * MEAN_LANES < rows; i += 8 * MEAN_LANES) {   // eight rows' loads in flight
    float4 e[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) e[u] = row[i + u * MEAN_LANES];
#pragma unroll
    for (int u = 0; u < 8; ++u) add(a, e[u]);
  }
  for (; i < rows; i += MEAN_LANES) add(a, row[i]);
  s[tid] = a;
  __syncthreads();
  for (int w = MEAN_LANES / 2; w > 0; w >>= 1) {
    if (tid < w) add(s[tid], s[tid + w]);
    __syncthreads();
  }
  if (tid == 0) {
    // exact up to 2^24 rows that count; past them, as the other sums, to the tree's ten roundings
    const float n = fmaxf(s[0].z, 1.f), m = fmaxf(s[0].w, 1.f);
    const float soft = (1.f - hard) * tau;
    coef[0] = soft / n;
    coef[1] = hard / m;
    *loss = soft * tau * (s[0].x / n) + hard * (s[0].y / m);
  }
}

// A class that is neither named nor the label gets F softmax(x / tau) + gb softmax(x). TAIL: its share of the teacher's rest
// goes with the softmax of the classes that are not named, of which softmax(x / tau) is the 2^-D'th part (D >= 0), so one exponential
// carries both. HARD: the labels' softmax is another one; at temperature 1 it is the same and in F too.
// A workgroup takes U vectors a lane of one row, a.parts workgroups in turn a row: what all of them have in flight lies close together.
template <typename T> constexpr int BWD_AT_ONCE = sizeof(T) == 4 ? 2 : 4;
template <typename T, bool TAIL, bool HARD, bool NT> __global__ __launch_bounds__(WG) void k_distill_bwd(const Distill a) {
  constexpr int U = BWD_AT_ONCE<T>, STEP = U * WG;
  extern __shared__ unsigned s_dyn[];   // k ids, k probabilities
  int* s_id = reinterpret_cast<int*>(s_dyn);
  float* s_p = reinterpret_cast<float*>(s_dyn) + a.k;
  const int64_t row = a.row0 + blockIdx.x / a.parts;
  const int vocab = a.vocab, tid = (int)threadIdx.x, nv = vocab >> 3, part = (int)blockIdx.x % a.parts;
  const int v0 = part * STEP, c0 = 8 * v0, c1 = part == a.parts - 1 ? vocab : c0 + 8 * STEP;   // vectors from v0, classes c0 to c1
  const T* x = static_cast<const T*>(a.logits) + row * vocab;
  T* o = static_cast<T*>(a.dlogits) + row * vocab;
  Vectors<T, WG, U, NT> raw;
  if (nv > 0) raw.load(x, v0, nv);
  const DistillTerms n = a.terms[row];
  const DistillRow r = a.saved[row];
  const float g = *a.dloss, zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const bool labelled = a.labels && n.labelled != 0.f;
  if (n.counts == 0.f && !labelled) {   // workgroup-uniform
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + tid + u * WG < nv) store_stream<T, NT>(o + 8 * (int64_t)(v0 + tid + u * WG), zero);
    if (c1 == vocab && tid < (vocab & 7)) st1(o + 8 * (int64_t)nv + tid, 0.f);
    return;
  }
  const int k = n.counts != 0.f ? a.k : 0;
  const float inv_tau = 1.f / a.tau, c = LOG2E / a.tau;
  const float ga = k ? g * a.coef[0] : 0.f, gb = labelled ? g * a.coef[1] : 0.f;
  const float qa = ga * r.all, l2 = r.l * LOG2E, l12 = r.l1 * LOG2E, lr2 = r.lr * LOG2E;
  const bool rest = TAIL && r.rest > 0.f;
  const float share = rest ? __builtin_amdgcn_exp2f((r.mr - r.m) * c + (lr2 - l2)) : 1.f;   // 2^-D
  const float base = rest ? r.mr : r.m, lb = rest ? lr2 : l2, minus = rest ? ga * r.rest : 0.f;
  const float unnamed = qa * share - minus, F = HARD ? unnamed : (qa + gb) * share - minus;
  const int64_t label = labelled ? a.labels[row] : -1;
  for (int i = tid; i < k; i += WG) {
    const int id = id_of(a.ids, a.wide, row * k + i, vocab);
    const bool here = id >= c0 && id < c1;
    s_id[i] = here ? id : -1;
    s_p[i] = here ? expf(ld_as(a.top, row * k + i, a.top_dtype) * inv_tau - r.teacher) : 0.f;
  }
  auto grad = [&](float e) {
    float t = F * __builtin_amdgcn_exp2f((e - base) * c - lb);
    if (HARD) t = __builtin_fmaf(gb, __builtin_amdgcn_exp2f((e - r.m) * LOG2E - l12), t);
    return t;
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v = v0 + tid + u * WG;
    float e[8];
    IO<T>::unpack(raw.r[u], e);
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = grad(e[j]);
    if (v < nv) store_stream<T, NT>(o + 8 * (int64_t)v, e);
  }
  if (c1 == vocab && tid < (vocab & 7)) {
    const int64_t i = 8 * (int64_t)nv + tid;
    st1(o + i, grad(ld1(x + i)));
  }
  __syncthreads();   // orders the row's stores before those below, and the named classes in LDS
  for (int i = tid; i <= k; i += WG) {   // the named classes, and the label
    const int64_t id = i < k ? s_id[i] : label;
    if (id < c0 || id >= c1) continue;
    float p = 0.f;
    bool named = false;
    for (int j = 0; j < k; ++j)   // a class named twice, or the label named: all write the same value
      if (s_id[j] == id) {
        p += s_p[j];
        named = true;
      }
    const float e = ld1(x + id);
    float t = named ? qa * __builtin_amdgcn_exp2f((e - r.m) * c - l2) - ga * p : unnamed * __builtin_amdgcn_exp2f((e - base) * c - lb);
    if (labelled) t += gb * (__builtin_amdgcn_exp2f((e - r.m) * LOG2E - l12) - (id == label ? 1.f : 0.f));
    st1(o + id, t);
  }
}

inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool al_of(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == LDR_F32 ? 3u : 1u)) == 0; }
inline bool dtype_ok(int dt) { return dt == LDR_F32 || dt == LDR_BF16 || dt == LDR_F16; }
constexpr int64_t MOST_GROUPS = 1 << 22;   // of a launch: its lanes are counted in 32 bits
inline unsigned grid_of(int64_t blocks, int64_t cap) { return (unsigned)(blocks < cap ? blocks : cap); }
inline int launched() { return (int)hipGetLastError(); }

#define LMO_TYPE_SWITCH(DT, ...)                                 \
  if ((DT) == LDR_BF16) { typedef bf16_t T; __VA_ARGS__; }       \
  else if ((DT) == LDR_F16) { typedef _Float16 T; __VA_ARGS__; } \
  else { typedef float T; __VA_ARGS__; }
#define LMO_BOOL_SWITCH(V, NAME, ...)                            \
  if (V) { constexpr bool NAME = true; __VA_ARGS__; }            \
  else { constexpr bool NAME = false; __VA_ARGS__; }
#define LMO_POW_SWITCH(P, ...)                         \
  switch (P) {                                         \
    case 0: { constexpr int POW = 0; __VA_ARGS__; } break; \
    case 2: { constexpr int POW = 2; __VA_ARGS__; } break; \
    case 4: { constexpr int POW = 4; __VA_ARGS__; } break; \
    default: { constexpr int POW = 1; __VA_ARGS__; } break; \
  }
#define LMO_CASE(L, V, ...) case 8 * L + V: { constexpr int LPR = L, VPT = V; __VA_ARGS__; } break;
#define LMO_LANES_SWITCH(S, ...)                                                                                           \
  switch (8 * (S).lpr + (S).vpt) {                                                                                         \
    LMO_CASE(4, 1, __VA_ARGS__) LMO_CASE(16, 1, __VA_ARGS__) LMO_CASE(64, 1, __VA_ARGS__) LMO_CASE(128, 2, __VA_ARGS__)    \
    LMO_CASE(256, 2, __VA_ARGS__) LMO_CASE(512, 4, __VA_ARGS__)

// Lanes to a row, and vectors of eight columns to a lane. Few lanes with several loads each in flight beat many lanes with one, whose
// rows are a load and two barriers long (30000 x 2048 bf16 backward: 128 lanes 71 us, 256 100; 4096 x 16384: 512 lanes 97 us, 1024 250),
// until the backward's column sums leave too few waves. Rows of up to 1024 columns are one wave's in the backward (no barriers: 21.5 us
// for 16384 x 768, 26 with two); the forward, which has no sums to keep, is faster with two (18.4 and 19.5).
struct Lanes { int lpr, vpt; };
inline Lanes lanes_of_row(int64_t rows, int64_t d, bool backward) {
  if (d <= 32) return {4, 1};
  if (d <= 128) return {16, 1};
  if (d <= 512) return {64, 1};
  if (d <= 1024) return backward ? Lanes{64, 2} : Lanes{128, 1};
  if (d <= 2048) return backward || rows > 256 ? Lanes{128, 2} : Lanes{256, 1};   // 1 x 2048: 3.0 and 2.2 us
  if (d <= 4096) return {256, 2};
  if (d <= 8192) return backward ? Lanes{256, 4} : Lanes{512, 2};
  return {512, 4};
}
// The backward's consecutive rows of a workgroup, and its workgroups: as many as run at once (3 to a CU, 2 of the wider rows, whose
// partial sums cost more too, 1 of the widest).
struct Plan { int64_t per, parts; };
inline Plan plan_of(int64_t rows, int64_t d) {
  const int lpr = lanes_of_row(rows, d, true).lpr, r = lpr > WG ? 1 : WG / lpr;
  const int64_t most = d <= 1024 ? 768 : d <= 8192 ? 512 : 256;
  int64_t per = (rows + most - 1) / most;
  per = (per + r - 1) / r * r;
  return Plan{per, (rows + per - 1) / per};
}
int norm_shape(int64_t rows, int64_t d, int dtype) {
  if (!dtype_ok(dtype)) return LDR_E_DTYPE;
  if (d < 1 || d > LMO_NORM_MAX_WIDTH) return LDR_E_SHAPE;
  if (rows < 0 || rows > 0x7fffffff) return LDR_E_ARG;
  return LDR_OK;
}

// logits that the 256 MB of the last cache do not hold beside their gradient go past the caches
inline bool past_caches(int64_t rows, int64_t vocab, int dtype) {
  return rows * vocab > (int64_t)(dtype == LDR_F32 ? 32 : 64) << 20;
}
// workgroups of 1024 lanes where there are too few rows for the CUs, of 256 otherwise
inline bool wide_workgroups(int64_t rows) { return rows <= 512; }

int distill_args(const Distill& a, int64_t rows, int64_t vocab, int64_t k, int dtype, bool tail) {
  if (!dtype_ok(dtype) || !dtype_ok(a.top_dtype)) return LDR_E_DTYPE;
  if (vocab < 1 || vocab > 0x7fffffff - 8 || k < 1 || k > LMO_DISTILL_MAX_TOP || (tail && vocab > LMO_DISTILL_MAX_TAIL))
    return LDR_E_SHAPE;
  if (rows < 0 || rows > 0x7fffffff || !(a.tau > 0.f) || !(a.tau < INFINITY)) return LDR_E_ARG;
  if (rows > 0 && (!a.logits || !a.top || !a.ids || !a.saved)) return LDR_E_ARG;
  if (!al_of(a.logits, dtype) || !al_of(a.dlogits, dtype) || !al_of(a.top, a.top_dtype) || !al16(a.saved) ||
      (reinterpret_cast<uintptr_t>(a.ids) & (a.wide ? 7u : 3u)) || (reinterpret_cast<uintptr_t>(a.labels) & 7u) ||
      !al_of(a.teacher_lse, LDR_F32))
    return LDR_E_ALIGN;
  return LDR_OK;
}

}  // namespace

extern "C" {

int lmo_abi_version(void) { return LMO_ABI_VERSION; }

int lmo_layer_norm_fwd(const void* x, const void* add, const void* w, const void* b, void* h_out, void* y, float* stats,
                       int64_t rows, int64_t d, float eps, int dtype, void* stream) {
  const int e = norm_shape(rows, d, dtype);
  if (e || rows == 0) return e;
  if (!x || !y || (add && !h_out)) return LDR_E_ARG;
  bool al = d % 8 == 0;
  for (const void* p : {x, add, w, b, (const void*)(add ? h_out : nullptr), (const void*)y}) {
    if (!al_of(p, dtype)) return LDR_E_ALIGN;
    al = al && al16(p);
  }
  if (reinterpret_cast<uintptr_t>(stats) & 7u) return LDR_E_ALIGN;
  const Lanes lanes = lanes_of_row(rows, d, false);
  const int lpr = lanes.lpr, r = lpr > WG ? 1 : WG / lpr;
  const unsigned grid = grid_of((rows + r - 1) / r, MOST_GROUPS / 4);
  hipStream_t st = static_cast<hipStream_t>(stream);
  LMO_TYPE_SWITCH(dtype, {
    const NormFwd<T> a{static_cast<const T*>(x), static_cast<const T*>(add), static_cast<const T*>(w), static_cast<const T*>(b),
                       static_cast<T*>(h_out), static_cast<T*>(y), stats, (int)rows, (int)d, eps};
    LMO_BOOL_SWITCH(al, AL, {
      LMO_LANES_SWITCH(lanes, hipLaunchKernelGGL((k_layer_norm_fwd<T, LPR, VPT, AL>), dim3(grid), dim3(lanes_of(LPR)), 0, st, a))
      LMO_CASE(128, 1, hipLaunchKernelGGL((k_layer_norm_fwd<T, LPR, VPT, AL>), dim3(grid), dim3(lanes_of(LPR)), 0, st, a))
      LMO_CASE(256, 1, hipLaunchKernelGGL((k_layer_norm_fwd<T, LPR, VPT, AL>), dim3(grid), dim3(lanes_of(LPR)), 0, st, a))
      LMO_CASE(512, 2, hipLaunchKernelGGL((k_layer_norm_fwd<T, LPR, VPT, AL>), dim3(grid), dim3(lanes_of(LPR)), 0, st, a))
      }
    })
  })
  return launched();
}

int64_t lmo_layer_norm_scratch(int64_t rows, int64_t d) {
  return rows < 1 || d < 1 ? 0 : 2 * d * plan_of(rows, d).parts;
}

int lmo_layer_norm_bwd(const void* dy, const void* h, const void* w, const float* stats, const void* dres, void* dx,
                       void* dw, void* db, float* scratch, int64_t rows, int64_t d, int dtype, void* stream) {
  const int e = norm_shape(rows, d, dtype);
  if (e || rows == 0) return e;
  if (!dy || !h || !stats || ((dw || db) && !scratch)) return LDR_E_ARG;
  if (!dx && !dw && !db) return LDR_OK;
  bool al = d % 8 == 0;
  for (const void* p : {dy, h, w, dres, (const void*)dx, (const void*)scratch}) {
    if (!al_of(p, dtype)) return LDR_E_ALIGN;
    al = al && al16(p);
  }
  if (!al_of(scratch, LDR_F32) || !al_of(dw, dtype) || !al_of(db, dtype) || (reinterpret_cast<uintptr_t>(stats) & 7u))
    return LDR_E_ALIGN;
  const Plan plan = plan_of(rows, d);
  const int parts = (int)plan.parts;
  hipStream_t st = static_cast<hipStream_t>(stream);
  LMO_TYPE_SWITCH(dtype, {
    const NormBwd<T> a{static_cast<const T*>(dy), static_cast<const T*>(h), static_cast<const T*>(w), stats,
                       static_cast<const T*>(dres), static_cast<T*>(dx), dw ? scratch : nullptr,
                       db ? scratch + parts * d : nullptr, (int)rows, (int)d, (int)plan.per};
    LMO_BOOL_SWITCH(al, AL, {
      LMO_LANES_SWITCH(lanes_of_row(rows, d, true), hipLaunchKernelGGL((k_layer_norm_bwd<T, LPR, VPT, AL>), dim3(parts), dim3(lanes_of(LPR)), 0, st, a))
      LMO_CASE(64, 2, hipLaunchKernelGGL((k_layer_norm_bwd<T, LPR, VPT, AL>), dim3(parts), dim3(lanes_of(LPR)), 0, st, a))
      LMO_CASE(256, 4, hipLaunchKernelGGL((k_layer_norm_bwd<T, LPR, VPT, AL>), dim3(parts), dim3(lanes_of(LPR)), 0, st, a))
      }
    })
    const int err = launched();
    if (err) return err;
    if (dw || db) {
      LMO_BOOL_SWITCH(d > 2048, WIDE, {
        constexpr int COLS = WIDE ? 64 : 16;
        hipLaunchKernelGGL((k_layer_norm_sum<T, COLS>), dim3((unsigned)((d + COLS - 1) / COLS), 2), dim3(SUM_LANES), 0, st, a.part_w,
                           a.part_b, static_cast<T*>(dw), static_cast<T*>(db), parts, (int)d);
      })
    }
  })
  return launched();
}

int lmo_distill_fwd(const void* logits, const void* top, int top_dtype, const void* ids, int wide_ids,
                    const float* teacher_lse, const int64_t* labels, float tau, float hard, float* saved, float* coef,
                    float* loss, int64_t rows, int64_t vocab, int64_t k, int dtype, void* stream) {
  Distill a{logits, top, ids, teacher_lse, labels, reinterpret_cast<DistillTerms*>(saved),
            reinterpret_cast<DistillRow*>(saved + 4 * rows), nullptr, nullptr, nullptr,
                  (int)vocab, (int)k, top_dtype, wide_ids, tau, 0, 1};
  const int e = distill_args(a, rows, vocab, k, dtype, teacher_lse != nullptr);
  if (e) return e;
  if (!coef || !loss || !(hard >= 0.f && hard <= 1.f)) return LDR_E_ARG;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t map = teacher_lse ? ((size_t)vocab + 31) / 32 * 4 : 0;
  const int pow = !labels || tau == 1.f ? 0 : tau == 2.f ? 2 : tau == 4.f ? 4 : 1;
  for (; a.row0 < rows; a.row0 += MOST_GROUPS) {
    const unsigned grid = (unsigned)(rows - a.row0 < MOST_GROUPS ? rows - a.row0 : MOST_GROUPS);
    int err = 0;
    LMO_TYPE_SWITCH(dtype, LMO_BOOL_SWITCH(teacher_lse != nullptr, TAIL, LMO_POW_SWITCH(pow, {
      const auto run = [&](auto lanes, auto nt) {   // the waves' sums lie beside the map: together they can be past 64 KiB
        constexpr int LANES = decltype(lanes)::value, BESIDE = LANES / 64 * 4;
        constexpr bool NT = decltype(nt)::value;
        const int most = map + BESIDE > 65536 ? LMO_DISTILL_MAX_TAIL / 8 : 0;
        if (const int err = ALLOW_LDS_BESIDE(BESIDE, most, k_distill_fwd<T, LANES, TAIL, POW, NT>)) return err;
        hipLaunchKernelGGL((k_distill_fwd<T, LANES, TAIL, POW, NT>), dim3(grid), dim3(LANES), map, st, a);
        return launched();
      };
      if (wide_workgroups(rows)) err = run(std::integral_constant<int, 1024>(), std::false_type());
      else if (past_caches(rows, vocab, dtype)) err = run(std::integral_constant<int, WG>(), std::true_type());
      else err = run(std::integral_constant<int, WG>(), std::false_type());
    })))
    if (err) return err;
  }
  hipLaunchKernelGGL(k_distill_mean, dim3(1), dim3(MEAN_LANES), 0, st, a.terms, rows, tau, hard,
                     coef, loss);
  return launched();
}

int lmo_distill_bwd(const void* logits, const void* top, int top_dtype, const void* ids, int wide_ids,
                    const int64_t* labels, float tau, const float* saved, const float* coef, const float* dloss,
                    void* dlogits, int64_t rows, int64_t vocab, int64_t k, int tail, int dtype, void* stream) {
  Distill a{logits, top, ids, nullptr, labels, reinterpret_cast<DistillTerms*>(const_cast<float*>(saved)),
            reinterpret_cast<DistillRow*>(const_cast<float*>(saved) + 4 * rows), coef, dloss,
                  dlogits, (int)vocab, (int)k, top_dtype, wide_ids, tau, 0, 1};
  const int e = distill_args(a, rows, vocab, k, dtype, tail != 0);
  if (e || rows == 0) return e;
  if (!coef || !dloss || !dlogits) return LDR_E_ARG;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t lds = 8 * (size_t)k;
  const int64_t step = 8 * WG * (dtype == LDR_F32 ? BWD_AT_ONCE<float> : BWD_AT_ONCE<bf16_t>);
  a.parts = (int)((vocab + step - 1) / step);
  for (const int64_t most = MOST_GROUPS / a.parts > 0 ? MOST_GROUPS / a.parts : 1; a.row0 < rows; a.row0 += most) {
    const unsigned grid = (unsigned)(rows - a.row0 < most ? rows - a.row0 : most) * (unsigned)a.parts;
    LMO_TYPE_SWITCH(dtype, LMO_BOOL_SWITCH(tail != 0, TAIL, LMO_BOOL_SWITCH(labels != nullptr && tau != 1.f, HARD,
        LMO_BOOL_SWITCH(past_caches(rows, vocab, dtype), NT,
            hipLaunchKernelGGL((k_distill_bwd<T, TAIL, HARD, NT>), dim3(grid), dim3(WG), lds, st, a)))))
    const int err = launched();
    if (err) return err;
  }
  return LDR_OK;
}

}  // extern "C"
