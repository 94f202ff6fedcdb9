// The state-free part of every chunk: T = (I + A)^{-1}, P and the row factors, and
// the tiles of K and Q where the caller's rows are not copied as they are
// (delta_common.hpp).  One workgroup of four waves a (value
// sequence, chunk); wave w owns token rows 16 w .. 16 w + 15.
//
// T.  Wave w inverts diagonal block w by substitution (a lane a column, 120 steps
// in registers against broadcast LDS rows); the blocks below follow from
// [[X, 0], [Y, Z]]^{-1} = [[X', 0], [-Z' Y X', Z']] at 16 and at 32, on fp32 MFMA:
// substitution's accuracy without its 64-step chain.
// L is summed and subtracted in fp64, so that a decay that has cost the chunk
// hundreds of nats leaves the differences of later tokens exact; logA below -1e5
// (a = 0 many times over) counts as -1e5, which keeps -inf - -inf out.
//
// Bound by HBM, what it writes above all (T and P in three terms, 30 KB): 196 us for 8
// sequences of 131072 tokens, r = 128 in bf16, 5.3 TB/s.
#pragma once

#include "delta_common.hpp"

namespace smat {
namespace dl {

constexpr int kLd = 68;            // floats a row of the 64 x 64 LDS tiles

// acc += A B for 16 x 16 fp32 blocks, A row-major in LDS, B as a result tile in
// registers (row 4g + i in element i): instruction i contracts rows 4g + i.
__device__ __forceinline__ f32x4 mm16(f32x4 acc, const float* A, const f32x4& B) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(A + (lane_id() & 15) * kLd + 4 * (lane_id() >> 4));
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], B[i], acc, 0, 0, 0);
  return acc;
}
__device__ __forceinline__ f32x4 tile_of(const float* B) {
  f32x4 b;
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = B[(4 * (lane_id() >> 4) + i) * kLd + (lane_id() & 15)];
  return b;
}
__device__ __forceinline__ void put_tile(float* B, const f32x4& b, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) B[(4 * (lane_id() >> 4) + i) * kLd + (lane_id() & 15)] = s * b[i];
}

// Am (strictly lower, zero elsewhere) -> Tm = (I + Am)^{-1}, lower tiles only.
// Called by four waves; ends with a barrier.
__device__ __forceinline__ void unit_lower_inverse(const float* Am, float* Tm) {
  const int w = wave_id(), lane = lane_id(), c = lane & 15;
  auto at = [](const float* M, int a, int b) { return M + (16 * a) * kLd + 16 * b; };
  {
    const float* A = at(Am, w, w);
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = (i == c) ? 1.f : 0.f;
#pragma unroll
      for (int j4 = 0; j4 < (i + 3) / 4; ++j4) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(A + i * kLd + 4 * j4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (4 * j4 + j < i) s -= a[j] * x[4 * j4 + j];
      }
      x[i] = s;
    }
    if (lane < 16) {
      float* Tw = Tm + (16 * w) * kLd + 16 * w;
#pragma unroll
      for (int i = 0; i < 16; ++i) Tw[i * kLd + c] = x[i];
    }
  }
  __syncthreads();
  if (w < 2) {                                     // blocks (1, 0) and (3, 2)
    const int a = 2 * w + 1, b = 2 * w;
    f32x4 y = mm16(zero4(), at(Am, a, b), tile_of(at(Tm, b, b)));
    y = mm16(zero4(), at(Tm, a, a), y);
    put_tile(Tm + (16 * a) * kLd + 16 * b, y, -1.f);
  }
  __syncthreads();
  {                                                // rows 2, 3 x columns 0, 1
    const int a = 2 + (w >> 1), b = w & 1;
    f32x4 y2 = zero4(), y3 = zero4(), t;
    const f32x4 t1 = tile_of(at(Tm, 1, b));
    y2 = mm16(y2, at(Am, 2, 1), t1);
    if (a == 3) y3 = mm16(y3, at(Am, 3, 1), t1);
    if (b == 0) {
      const f32x4 t0 = tile_of(at(Tm, 0, 0));
      y2 = mm16(y2, at(Am, 2, 0), t0);
      if (a == 3) y3 = mm16(y3, at(Am, 3, 0), t0);
    }
    t = mm16(zero4(), at(Tm, a, 2), y2);
    if (a == 3) t = mm16(t, at(Tm, 3, 3), y3);
    put_tile(Tm + (16 * a) * kLd + 16 * b, t, -1.f);
  }
  __syncthreads();
}

// Running sum of the chunk's logA in fp64, in units of log 2, into Ls (wave 0), beta
// into bs.  Tokens past the chunk's end count as logA = 0, beta = 0.  The loads are a
// call of their own, to be issued ahead.
struct Gates {
  float a, b;
};
__device__ __forceinline__ Gates load_gates(const Geo& g, const float* logA, const float* beta,
                                            int s, int t0, int len) {
  const int64_t t = t0 + min(lane_id(), len - 1);
  return {logA[s * g.a_sb + t * g.a_st], beta[s * g.b_sb + t * g.b_st]};
}
__device__ __forceinline__ void chunk_decays(const Gates& gt, int len, double* Ls, float* bs) {
  const int t = threadIdx.x;
  if (t < C) {
    const bool ok = t < len;
    // NaN stays NaN
    double x = ok ? (gt.a < -1e5f ? -1e5 : (double)gt.a) * 1.4426950408889634 : 0.0;
    bs[t] = ok ? gt.b : 0.f;
#pragma unroll
    for (int d = 1; d < C; d <<= 1) {
      const double y = __shfl_up(x, d);
      if (t >= d) x += y;
    }
    Ls[t] = x;
  }
}
// 2^x of a difference of them: v_exp_f32, within an ulp and zero below 2^-126.
__device__ __forceinline__ float decay(double x) { return __builtin_amdgcn_exp2f((float)x); }

// The eight values (slots of contraction block kb) of token row m as terms.  Rows that
// are read whole (a full bf16 chunk of 32 RB features) skip the checks.
template <typename In, int N>
__device__ __forceinline__ Frag<N> row_frag(const In* row, bool ok, int c0, int r, bool vec) {
  const f32x4 a = ok ? load4(row + c0, r - c0, vec) : zero4();
  const f32x4 b = ok ? load4(row + c0 + 16, r - c0 - 16, vec) : zero4();
  return split<N>(a, b);
}
__device__ __forceinline__ Frag<1> whole_frag(const bf16* row, int c0) {
  const bf16x4 a = *reinterpret_cast<const bf16x4*>(row + c0);
  const bf16x4 b = *reinterpret_cast<const bf16x4*>(row + c0 + 16);
  Frag<1> f;
  f.t[0] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  return f;
}
template <typename In, int RB, int N>
__device__ __forceinline__ void row_frags(Frag<N>* f, const In* row, bool ok, int r, bool vec,
                                          int len) {
  const int gq = lane_id() >> 4;
  if constexpr (__is_same(In, bf16)) {
    if (vec && len == C && r == 32 * RB) {
#pragma unroll
      for (int kb = 0; kb < RB; ++kb) f[kb] = whole_frag(row, 32 * kb + 4 * gq);
      return;
    }
  }
#pragma unroll
  for (int kb = 0; kb < RB; ++kb) f[kb] = row_frag<In, N>(row, ok, 32 * kb + 4 * gq, r, vec);
}

// A lower triangle's fragment of row tile mt and block kb into its place, or its half.
__device__ __forceinline__ void store_tri(bf16* p, int mt, int kb, const Frag<kMid>& f) {
  if (half_tri(mt, kb)) {
#pragma unroll
    for (int n = 0; n < kMid; ++n)
      *reinterpret_cast<bf16x4*>(p + n * kLow * kFrag + lane_id() * 8 + 4 * kb) =
          __builtin_shufflevector(f.t[n], f.t[n], 0, 1, 2, 3);
  } else {
    store_frag<kMid>(p + tri(mt, kb) * kFrag, kLow * kFrag, f);
  }
}

// A token's slots of contraction block kb into its row of a tile (a tile a term).
template <int RB, int N>
__device__ __forceinline__ void store_row(bf16* tile, int t, int kb, const Frag<N>& f) {
  constexpr int RS = row_chunks(RB);
  const int g = lane_id() >> 4;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = (4 * kb + 2 * h + (g >> 1)) ^ swz<RS>(t);
      bf16* p = tile + n * tile_elems(RB) + (t * RS + k) * 8 + 4 * (g & 1);
      *reinterpret_cast<bf16x4*>(p) =
          h ? __builtin_shufflevector(f.t[n], f.t[n], 4, 5, 6, 7)
            : __builtin_shufflevector(f.t[n], f.t[n], 0, 1, 2, 3);
    }
}

// LDS: the row fragments of K (BWD: then of Q), with T's tile in their place once they
// are read, and A's tile.
template <typename In, int RB, bool BWD> constexpr int prep_rows() {
  constexpr int rows = Terms<In>::in * 4 * RB * kFrag * 2;
  return BWD || rows < C * kLd * 4 ? (BWD ? rows + C * kLd * 4 : C * kLd * 4) : rows;
}

template <typename In, int RB, bool BWD>
__global__ __launch_bounds__(256) void delta_prep_kernel(
    const In* __restrict__ q, const In* __restrict__ k, const float* __restrict__ logA,
    const float* __restrict__ beta, Geo g, Ops o, bool qvec, bool kvec) {
  constexpr int NT = Terms<In>::in, NI = kMid;
  constexpr int KB = 4 * RB * kFrag;               // elements of one term of a chunk's rows
  __shared__ __align__(16) char mem[prep_rows<In, RB, BWD>()];
  __shared__ __align__(16) float Am[C * kLd];
  __shared__ double Ls[C];
  __shared__ float bs[C];
  bf16* rows = reinterpret_cast<bf16*>(mem);
  float* Tm = reinterpret_cast<float*>(mem + (BWD ? NT * KB * 2 : 0));
  const int c = blockIdx.x, s = blockIdx.y;
  const int w = uniform_wave(), m = lane_id() & 15, gq = lane_id() >> 4;
  int t0, len;
  chunk_of(g, c, t0, len);
  const int64_t ks = key_of(g, s);
  const bool tiles = o.kw && s % (g.nb / g.nbk) == 0;   // this workgroup stores K's and Q's tiles
  const int tok = 16 * w + m;
  const bool live = tok < len;
  const In* krow = k + ks * g.k_sb + (int64_t)(t0 + (live ? tok : 0)) * g.k_st;
  const In* qrow = q + ks * g.q_sb + (int64_t)(t0 + (live ? tok : 0)) * g.q_st;
  const int64_t kc = (ks * g.nch + c) * (int64_t)NT * tile_elems(RB), sc = (int64_t)s * g.nch + c;
  const Gates gates = load_gates(g, logA, beta, s, t0, len);
  Frag<NT> kf[RB], qf[RB];
  row_frags<In, RB, NT>(kf, krow, live, g.r, kvec, len);
  row_frags<In, RB, NT>(qf, qrow, live, g.r, qvec, len);
  chunk_decays(gates, len, Ls, bs);
#pragma unroll
  for (int kb = 0; kb < RB; ++kb) store_frag<NT>(rows + (w * RB + kb) * kFrag, KB, kf[kb]);
  if (tiles) {
#pragma unroll
    for (int kb = 0; kb < RB; ++kb) {
      store_row<RB, NT>(o.kw + kc, tok, kb, kf[kb]);
      store_row<RB, NT>(o.qw + kc, tok, kb, qf[kb]);
    }
  }
  __syncthreads();
  const double Lt = Ls[tok];
  f32x4 pacc[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) pacc[t] = zero4();
  if (!BWD) {
    // token i = 16 w + m in the lane, tile jt's rows j = 16 jt + 4 gq + i in registers: A
    // below the diagonal (row i of it in vectors) and P by rows from one set of decays
    const float b = bs[tok];
#pragma unroll
    for (int jt = 0; jt < 4; ++jt)
      if (jt <= w) {
        f32x4 a = zero4(), P = zero4();
#pragma unroll
        for (int kb = 0; kb < RB; ++kb) {
          const Frag<NT> kj = load_frag<NT>(rows + (jt * RB + kb) * kFrag, KB);
          a = mul_inputs(a, kj, kf[kb]);
          P = mul_inputs(P, kj, qf[kb]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = 16 * jt + 4 * gq + i;
          const float D = decay(Lt - Ls[j]);
          a[i] = j < tok ? b * (D * a[i]) : 0.f;
          pacc[jt][i] = j <= tok ? g.scale * (D * P[i]) : 0.f;
        }
        *reinterpret_cast<f32x4*>(Am + tok * kLd + 16 * jt + 4 * gq) = a;
      }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
      if (kb <= w / 2)
        store_tri(o.pm + sc * NI * kLow * kFrag, w, kb, split<NI>(pacc[2 * kb], pacc[2 * kb + 1]));
    __syncthreads();                               // Am whole; the rows are read
  } else {
    // token j = 16 w + m in the lane, rows i = 16 it + 4 gq + .. in registers: the same
    // decays serve column j of A and of P, whose queries come through LDS
    f32x4 D[4];
#pragma unroll
    for (int it = 0; it < 4; ++it)
      if (it >= w) {
        f32x4 a = zero4();
#pragma unroll
        for (int kb = 0; kb < RB; ++kb)
          a = mul_inputs(a, load_frag<NT>(rows + (it * RB + kb) * kFrag, KB), kf[kb]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ti = 16 * it + 4 * gq + i;
          D[it][i] = tok <= ti ? decay(Ls[ti] - Lt) : 0.f;
          Am[ti * kLd + tok] = tok < ti ? bs[ti] * (D[it][i] * a[i]) : 0.f;
        }
      }
    __syncthreads();                               // Am whole; K's rows are read
#pragma unroll
    for (int kb = 0; kb < RB; ++kb) store_frag<NT>(rows + (w * RB + kb) * kFrag, KB, qf[kb]);
    __syncthreads();
#pragma unroll
    for (int it = 0; it < 4; ++it)
      if (it >= w) {
#pragma unroll
        for (int kb = 0; kb < RB; ++kb)
          pacc[it] = mul_inputs(pacc[it], load_frag<NT>(rows + (it * RB + kb) * kFrag, KB), kf[kb]);
        // selected, not multiplied: a query that is not finite stays in its own row
#pragma unroll
        for (int i = 0; i < 4; ++i)
          pacc[it][i] = tok <= 16 * it + 4 * gq + i ? g.scale * (D[it][i] * pacc[it][i]) : 0.f;
      }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
      if (kb >= w / 2)
        store_frag<NI>(o.pt + (sc * NI * kTri + tri_t(w, kb)) * kFrag, kTri * kFrag,
                       split<NI>(pacc[2 * kb], pacc[2 * kb + 1]));
  }
  unit_lower_inverse(Am, Tm);
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    if (BWD && kb >= w / 2) {
      f32x4 x[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ti = 32 * kb + 16 * h + 4 * gq + i;
          x[h][i] = ti >= 16 * w ? Tm[ti * kLd + tok] : 0.f;
        }
      store_frag<NI>(o.tt + (sc * NI * kTri + tri_t(w, kb)) * kFrag, kTri * kFrag,
                     split<NI>(x[0], x[1]));
    }
    if (!BWD && kb <= w / 2) {
      const float* row = Tm + tok * kLd + 32 * kb + 4 * gq;
      const f32x4 x0 = *reinterpret_cast<const f32x4*>(row);
      const f32x4 x1 = 2 * kb + 1 <= w ? *reinterpret_cast<const f32x4*>(row + 16) : zero4();
      store_tri(o.tm + sc * NI * kLow * kFrag, w, kb, split<NI>(x0, x1));
    }
  }
  if (threadIdx.x < C) {
    const int t = threadIdx.x;
    float* v = o.vec + sc * kVec;
    const double Lc = Ls[C - 1];
    v[t] = decay(Ls[t]);
    v[C + t] = decay(Lc - Ls[t]);
    v[2 * C + t] = bs[t];
    v[3 * C + t] = t == 0 ? decay(Lc) : 0.f;
  }
}

}  // namespace dl
}  // namespace smat
