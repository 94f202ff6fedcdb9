// The gradient of the gated delta rule over whole sequences.  With the notation of
// delta_common.hpp, the gradient dO of the output and dS' of the state leaving a
// chunk:
//
//   dU = P^T dO + w K dS'            Z = T^T dU              dV = b Z
//   dS = exp(L_C) dS' + Q^T (scale e dO) - K^T (e b Z)
//   G  = D . (scale dO U^T) (j <= i)     N = -D . (Z U^T) (j < i)
//   dQ = scale e dO S^T + G K
//   y  = N K - e Z S^T                   dK = b y + w U dS'^T + G^T Q + (b N)^T K
//   db_i = Z_i.V_i + k_i.y_i
//   dlogA_t = sum_{i >= t} (q_i.dQ_i + b_i k_i.y_i - k_i.(dK_i - b_i y_i)) + <dS', S'>
//
// Where the state entering a chunk is zero, dlogA of its first token is zero, and is
// stored as that: its terms cancel only up to their roundings.
//
// (L_i enters as q_i e^{L_i}, as the e^{L_i} of the reading k_i and as the e^{-L_i}
// of the writing one, and everything behind the chunk as e^{L_C} in S'.)
//
// Two kernels after the chunks' operands: delta_rchain_kernel walks the chunks
// backwards through dS as the forward's chain walks them through S (16 columns a
// wave, operands shared in LDS), storing dS' and Z of every chunk (runs: their
// transitions are the forward's transposed, which it keeps); delta_grad_kernel,
// one workgroup a (key sequence, chunk), forms the rest for the group's value heads
// one after another, so the gradients of a shared key head are sums in registers, in
// the heads' order.
//
// Both move fp32 states and rows of every chunk through HBM and are bound by that: 96 x
// 4096 tokens, r = p = 64 in bf16: the walk 140 us at 4.5 TB/s (its first pass 84), the
// rest 225 us for 113 KB a chunk, 3.1 TB/s, its loads one step of 32 columns ahead.
#include "delta_prep.hpp"

namespace smat {
namespace dl {

struct RChainIO {
  const void* dout;       // (nb, T, p), strides d_sb, d_st
  int64_t d_sb, d_st;
  const float* start;     // dS behind run i of sequence s: start + (i nb + s) r p; or null
  float* end;             // first pass: dS before it, same layout
  float* fin;             // dS before segment j: fin + (j nb + s) r p; or null
  float *save_d, *z;      // dS' of every chunk (R x p32) and Z (64 x p32)
  void* dv;               // (nb, T, p) contiguous
  int ptiles;
};

// Bytes of LDS: KD buffers of K and the factors, Q, T^T and P^T.
template <typename In, int RB> constexpr int rchain_lds(int KD) {
  constexpr int NT = Terms<In>::in;
  return KD * (2 * NT * tile_elems(RB) + kVec * 4) +
         2 * (NT * tile_elems(RB) + 2 * kTri * kFrag * kMid);
}
template <typename In, int RB> constexpr int rchain_bufs() {
  return rchain_lds<In, RB>(2) <= kMaxLds ? 2 : 1;
}

template <typename In, int RB> constexpr int rchain_waves() {
  return 2 * rchain_lds<In, RB>(rchain_bufs<In, RB>()) <= kMaxLds ? 4 : 8;
}

template <typename In, int RB, bool OUT>
__global__ __launch_bounds__((64 * rchain_waves<In, RB>()), 2) void delta_rchain_kernel(
    Geo g, Ops o, RChainIO io, int tiles) {
  constexpr int NT = Terms<In>::in, NI = kMid, R = 32 * RB;
  constexpr int TL = NT * tile_elems(RB), TB = kTri * kFrag;
  constexpr int KD = rchain_bufs<In, RB>();
  extern __shared__ __align__(1024) bf16 lds[];
  bf16 *kl = lds, *ql = lds + KD * TL, *tl = ql + TL, *pl = tl + NI * TB;
  float* vl = reinterpret_cast<float*>(pl + NI * TB);
  constexpr int W = rchain_waves<In, RB>();
  const int w = uniform_wave();
  const int ct = blockIdx.y * W + w;
  const bool on = ct < tiles;                      // else: copies and barriers only
  const int s = blockIdx.x;                        // sequences first, as in the forward
  const int m = lane_id() & 15, gq = lane_id() >> 4;
  int run, c0, c1, seg;
  bool head, tail;
  run_of(g, blockIdx.z, run, c0, c1, seg, head, tail);
  if (!OUT && head) return;                        // nothing is carried past a segment's first run
  const int col = 16 * ct + m;
  const int64_t ks = key_of(g, s);
  const int64_t rp = (int64_t)g.r * g.p, sn = (int64_t)run * g.nb + s;
  const int ld = (g.p + 31) / 32 * 32;

  f32x4 S[2 * RB];                                 // dS
#pragma unroll
  for (int mt = 0; mt < 2 * RB; ++mt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int a = 16 * mt + 4 * gq + i;
      S[mt][i] = (io.start && a < g.r && col < g.p) ? io.start[sn * rp + (int64_t)a * g.p + col]
                                                    : 0.f;
    }
  const In* ds = (const In*)io.dout + s * io.d_sb;
  const uint32_t soff = (4 * gq * ld + col) * 4;    // in fp32 rows of ld
  const bool dlive = col < g.p;
  uint32_t dv[16];
  auto load_d = [&](int t0, int len) {
    load_column(dv, ds, io.d_st, t0, len, col, g.p);
  };
  const TileStage<RB, NT, W> kstage(o.k, g.r, w), qstage(o.q, g.r, w);
  auto vec_of = [&](int c) { return o.vec + ((int64_t)s * g.nch + c) * kVec; };
  auto stage_k = [&](int c, int t0, int len, int buf) {
    kstage(kl + buf * TL, o.k, ks, g.nch, c, t0, len, g.r, vec_of(c), w);
    stage<1, W>(vl + buf * kVec, vec_of(c), W - 1 - w);
  };
  auto stage_tp = [&](int c) {
    const int64_t sc = (int64_t)s * g.nch + c;
    stage<NI * kTri, W>(tl, o.tt + sc * NI * TB, w);
    stage<NI * kTri, W>(pl, o.pt + sc * NI * TB, w);
  };

  int t0 = 0, len = 0, t1 = 0, len1 = 0;
  if (c0 < c1) {
    chunk_of(g, c1 - 1, t0, len);
    load_d(t0, len);
    stage_k(c1 - 1, t0, len, 0);
    stage_tp(c1 - 1);
  }
  Frag<NI> sb[RB];                                 // dS as the next products' operand
#pragma unroll
  for (int kb = 0; kb < RB; ++kb) sb[kb] = split<NI>(S[2 * kb], S[2 * kb + 1]);
  for (int c = c1 - 1; c >= c0; --c) {
    const int buf = KD == 2 ? (c1 - 1 - c) & 1 : 0;
    const bool more = c > c0;
    const int64_t sc = (int64_t)s * g.nch + c;
    const bf16* kt = kl + buf * TL;
    const float* vec = vl + buf * kVec;
    const int lane = RB >= 3 ? fresh_lane() : lane_id(), f4 = 4 * (lane >> 4);
    chunk_of(g, more ? c - 1 : c, t1, len1);
    wait_vmcnt<0>();
    lds_barrier();
    // ---- K, T^T, P^T and the factors of chunk c are in LDS
    f32x4 d[4], x[4];
    column_values<In>(d, dv, dlive, len);
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) asm volatile("" : "+v"(d[mt]));   // their wait is here
    qstage(ql, o.q, ks, g.nch, c, t0, len, g.r, vec_of(c), w);
    if (KD == 2 && more) stage_k(c - 1, t1, len1, 1 - buf);
    Frag<NI> f[2];
    if (on) {
      if (OUT) {
#pragma unroll
        for (int mt = 0; mt < 2 * RB; ++mt)
          put_rows(io.save_d + (sc * R + 16 * mt) * ld, soff, ld, S[mt]);
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) x[mt] = zero4();                // dU
      constexpr int U = row_step(NT, RB);
      pipelined<4 / U * RB, Rows<NT, U>>(
          [&](int st, Rows<NT, U>& b) {
#pragma unroll
            for (int u = 0; u < U; ++u)
              b.k[u] = rows_of<RB, NT>(kt, st * U % 4 + u, st * U / 4, lane);
          },
          [&](int st, Rows<NT, U>& b) {
            const int m0 = st * U % 4, kb = st * U / 4;
            f32x4 ca[U];
            Frag<NI> sa[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              ca[u] = x[m0 + u];
              sa[u] = sb[kb];
            }
            mul_each(ca, b.k, sa);
#pragma unroll
            for (int u = 0; u < U; ++u) x[m0 + u] = ca[u];
          });
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
        x[mt] *= *reinterpret_cast<const f32x4*>(vec + C + 16 * mt + f4);
      Frag<NT> df[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) df[kb] = split<NT>(d[2 * kb], d[2 * kb + 1]);
      triangle_t<NI>(x, pl, df, lane);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) f[kb] = split<NI>(x[2 * kb], x[2 * kb + 1]);
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) x[mt] = zero4();
      triangle_t<NI>(x, tl, f, lane);              // Z
    }
    wait_vmcnt<0>();
    lds_barrier();
    // ---- Q of chunk c and the next K are in LDS; T^T and P^T are free
    load_d(t1, len1);                              // (the last chunk's once more: no branch)
    if (more) stage_tp(c - 1);
    if (on) {
      if (OUT) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) put_rows(io.z + (sc * C + 16 * mt) * ld, soff, ld, x[mt]);
      }
      const uint32_t voff = (f4 * g.p + col) * sizeof(In);
      Frag<NI> fd[2];
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const f32x4 e = *reinterpret_cast<const f32x4*>(vec + 16 * mt + f4);
        x[mt] *= *reinterpret_cast<const f32x4*>(vec + 2 * C + 16 * mt + f4);     // b Z
        if (OUT && dlive) {
          In* row = (In*)io.dv + ((int64_t)s * g.T + t0 + 16 * mt) * g.p;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (len == C || 16 * mt + f4 + i < len)
              *reinterpret_cast<In*>(reinterpret_cast<char*>(row + (int64_t)i * g.p) + voff) =
                  from_f32<In>(x[mt][i]);
        }
        x[mt] *= -e;
        d[mt] *= g.scale * e;
      }
      const float aC = vec[3 * C];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        f[kb] = split<NI>(x[2 * kb], x[2 * kb + 1]);
        fd[kb] = split<NI>(d[2 * kb], d[2 * kb + 1]);
      }
      update_state<RB, NT, true>(S, sb, aC, kt, f, ql, fd, lane);
    }
    if (KD == 1 && more) {
      lds_barrier();                               // K is read
      stage_k(c - 1, t1, len1, 0);
    }
    t0 = t1;
    len = len1;
  }
  if (!on) return;
  float* out = OUT ? (io.fin && head ? io.fin + ((int64_t)seg * g.nb + s) * rp : nullptr)
                   : io.end + sn * rp;
  if (out) {
#pragma unroll
    for (int mt = 0; mt < 2 * RB; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int a = 16 * mt + 4 * gq + i;
        if (a < g.r && col < g.p) out[(int64_t)a * g.p + col] = S[mt][i];
      }
  }
}

struct GradIO {
  const void *v, *dout;
  const float *logA, *beta;
  int64_t d_sb, d_st;
  const float *save_s, *save_u, *save_d, *z;
  void *dq, *dk;          // (nbk, T, r) contiguous
  float *dlogA, *dbeta;   // (nb, T) contiguous
  bool vvec, dvec, ovec;
};

__device__ __forceinline__ float dot4(const f32x4& a, const f32x4& b) {
  return a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3];
}
// Sum over the four lane groups (lanes m, m + 16, m + 32, m + 48).
__device__ __forceinline__ float sum_groups(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}
// Eight consecutive elements; those at and past nv are zero.  vec: groups of four.
template <typename In>
__device__ __forceinline__ void load8f(f32x4* x, const In* p, int nv, bool vec) {
  x[0] = load4(p, nv, vec);
  x[1] = load4(p + 4, nv - 4, vec);
}

// Feature tiles are shared by H waves a token tile: two for more than 64 features, to
// keep the sums of a wave within half of its SIMD's registers.
constexpr int grad_split(int RB) { return RB >= 3 ? 2 : 1; }
constexpr int most(int a, int b) { return a > b ? a : b; }
// K's and Q's tiles beside the fragments, or, where that is too much (fp32 of more than
// 64 features), behind G and N once the fragments are read, for each head anew.
template <typename In, int RB> constexpr bool grad_late() {
  return 4 * Terms<In>::in * tile_elems(RB) + (4 * RB + 8) * kMid * kFrag * 2 + 8192 > kMaxLds;
}
template <typename In, int RB> constexpr int grad_lds() {
  const int frags = (4 * RB + 8) * kMid * kFrag * 2, gn = 8 * C * kLd;
  const int tiles = 4 * Terms<In>::in * tile_elems(RB);
  return grad_late<In, RB>() ? most(frags, gn + tiles) : tiles + most(frags, gn);
}

// Wave (token tile tt, half hf).  The products over the value columns take S, dS', U and
// Z in steps of 32 columns, split into terms once, by the wave that loaded them, and
// shared as fragments in LDS; the next step's are loaded while one computes.  G and N
// then take the fragments' place.
// Keeps the operands of one group of products from being fetched during another's: the
// sums take most registers.
__device__ __forceinline__ void hold() { __builtin_amdgcn_sched_barrier(0); }

// SHARED: key heads shared by value heads, whose sums take registers of their own.  FULL:
// rows of V and dO in whole aligned groups, loaded without a branch (at a join the
// compiler waits for the loads of either side, a step ahead of their use).
template <typename In, int RB, bool SHARED, bool FULL>
__global__ __launch_bounds__(256 * grad_split(RB), 2) void delta_grad_kernel(Geo g, Ops o,
                                                                              GradIO io) {
  constexpr int NT = Terms<In>::in, NI = kMid, R = 32 * RB, TL = NT * tile_elems(RB);
  constexpr int H = grad_split(RB), W = 4 * H, RT = 2 * RB / H;   // feature tiles a wave
  constexpr int FS = 0, FD = 2 * RB, FU = 4 * RB, FZ = FU + 4, NF = FZ + 4, FP = NF * kFrag;
  extern __shared__ __align__(1024) bf16 lds[];
  constexpr bool LATE = grad_late<In, RB>();
  bf16 *kl = lds + (LATE ? 4 * C * kLd : 0), *ql = kl + TL, *fr = LATE ? lds : ql + TL;
  float *G = reinterpret_cast<float*>(fr), *N = G + C * kLd;
  __shared__ double Ls[C];
  __shared__ float bs[C], zvs[C], pair[W], sums[H][4][C];
  __shared__ bool holds[W];
  const int c = blockIdx.x, ks = blockIdx.y, group = SHARED ? g.nb / g.nbk : 1;
  const int w = uniform_wave(), tt = w & 3, hf = w >> 2;
  const int ld = (g.p + 31) / 32 * 32, rt0 = hf * RT;
  int t0, len;
  chunk_of(g, c, t0, len);
  auto stage_tiles = [&]() {
    const float* vec = o.vec + ((int64_t)ks * group * g.nch + c) * kVec;
    TileStage<RB, NT, W>(o.k, g.r, w)(kl, o.k, ks, g.nch, c, t0, len, g.r, vec, w);
    TileStage<RB, NT, W>(o.q, g.r, w)(ql, o.q, ks, g.nch, c, t0, len, g.r, vec, w);
  };
  if (!LATE) stage_tiles();
  // token in the lane, features 16 rt + 4 gq + i in registers, throughout
  f32x4 dQ[SHARED ? RT : 1], dK[SHARED ? RT : 1];
  if (SHARED) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) dQ[rt] = dK[rt] = zero4();
  }
  auto put = [&](int tok, int rt, const f32x4& q, const f32x4& k) {
    const int f0 = 16 * (rt0 + rt) + 4 * (lane_id() >> 4);
    const int64_t at = ((int64_t)ks * g.T + t0 + tok) * g.r + f0;
    store4((In*)io.dq + at, q, g.r - f0, io.ovec);
    store4((In*)io.dk + at, k, g.r - f0, io.ovec);
  };

  for (int h = 0; h < group; ++h) {
    // the lane's place, new to the compiler in every pass: what is built from it would
    // otherwise be kept in registers across the heads
    int lane = lane_id();
    asm("" : "+v"(lane));
    const int m = lane & 15, gq = lane >> 4, tok = 16 * tt + m;
    const bool live = tok < len;
    const int64_t row = t0 + (live ? tok : 0);
    const int s = ks * group + h;
    const int64_t sc = (int64_t)s * g.nch + c;
    const float* vec = o.vec + sc * kVec;
    const In* drow = (const In*)io.dout + s * io.d_sb + row * io.d_st;
    const In* vrow = (const In*)io.v + s * g.v_sb + row * g.v_st;
    // this wave's loads of a step: tile w of S and dS' (the last one again where there is
    // no tile w), and rows of U (waves of half 0) and Z (waves of the last half)
    constexpr bool both = H == 1;
    const bool pairs = w < 2 * RB, has_u = hf == 0, has_z = hf == H - 1;
    const int64_t lane_row = (int64_t)m * ld + 8 * gq;
    const int tile = min(w, 2 * RB - 1);
    const float* Sp = io.save_s + (sc * R + 16 * tile) * ld + lane_row;
    const float* Dp = io.save_d + (sc * R + 16 * tile) * ld + lane_row;
    const float* Up = (has_u ? io.save_u : io.z) + (sc * C + 16 * tt) * ld + lane_row;
    const float* Zp = io.z + (sc * C + 16 * tt) * ld + lane_row;
    f32x4 sx[2], ex[2], ux[2], zx[2], dx[2], vx[2];   // both = false: ux is U's or Z's rows
    typedef In In4 __attribute__((ext_vector_type(4)));
    In4 dr[2], vr[2];
    auto get = [&](f32x4* x, const float* p) {
      x[0] = *reinterpret_cast<const f32x4*>(p);
      x[1] = *reinterpret_cast<const f32x4*>(p + 4);
    };
    auto load_step = [&](int pb) {
      get(sx, Sp + pb);
      get(ex, Dp + pb);
      get(ux, Up + pb);
      if (both) get(zx, Zp + pb);
      const int pc = pb + 8 * gq;
      if constexpr (FULL) {
#pragma unroll
        for (int h4 = 0; h4 < 2; ++h4) {
          dr[h4] = *reinterpret_cast<const In4*>(drow + pc + 4 * h4);
          vr[h4] = *reinterpret_cast<const In4*>(vrow + pc + 4 * h4);
        }
      } else {
        load8f(dx, drow + pc, live ? g.p - pc : 0, io.dvec);
        load8f(vx, vrow + pc, live ? g.p - pc : 0, io.vvec);
      }
    };
    const Gates gates = load_gates(g, io.logA, io.beta, s, t0, len);
    load_step(0);
    __syncthreads();                               // the last head's LDS is read
    chunk_decays(gates, len, Ls, bs);

    f32x4 a[RT], y[RT], kw[RT], gp[4], np[4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) a[rt] = y[rt] = kw[rt] = zero4();
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) gp[jt] = np[jt] = zero4();
    float zv = 0.f, dots = 0.f;
    uint32_t held = 0;                             // whether the state entering holds anything
    for (int pb = 0; pb < ld; pb += 32) {
      if constexpr (FULL) {
#pragma unroll
        for (int h4 = 0; h4 < 2; ++h4)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dx[h4][i] = live ? to_f32(dr[h4][i]) : 0.f;
            vx[h4][i] = live ? to_f32(vr[h4][i]) : 0.f;
          }
      }
      if (pairs) {
        dots += dot4(sx[0], ex[0]) + dot4(sx[1], ex[1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) held |= __float_as_uint(sx[0][i]) | __float_as_uint(sx[1][i]);
        store_frag<NI>(fr + (FS + w) * kFrag, FP, split<NI>(sx[0], sx[1]));
        store_frag<NI>(fr + (FD + w) * kFrag, FP, split<NI>(ex[0], ex[1]));
      }
      store_frag<NI>(fr + ((has_u ? FU : FZ) + tt) * kFrag, FP, split<NI>(ux[0], ux[1]));
      if (both) {
        zv += dot4(zx[0], vx[0]) + dot4(zx[1], vx[1]);
        store_frag<NI>(fr + (FZ + tt) * kFrag, FP, split<NI>(zx[0], zx[1]));
      } else if (has_z) {
        zv += dot4(ux[0], vx[0]) + dot4(ux[1], vx[1]);
      }
      const Frag<NT> df = split<NT>(dx[0], dx[1]);
      __syncthreads();
      load_step(min(pb + 32, ld - 32));            // (the last step's once more: no branch)
      {
        const Frag<NI> zf = load_frag<NI>(fr + (FZ + tt) * kFrag, FP);
        const Frag<NI> uf = load_frag<NI>(fr + (FU + tt) * kFrag, FP);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const Frag<NI> sf = load_frag<NI>(fr + (FS + rt0 + rt) * kFrag, FP);
          a[rt] = mul(a[rt], sf, df);
          y[rt] = mul(y[rt], sf, zf);
          kw[rt] = mul(kw[rt], load_frag<NI>(fr + (FD + rt0 + rt) * kFrag, FP), uf);
        }
        hold();
#pragma unroll
        for (int jt = 0; jt < 4; ++jt)
          if (jt <= tt) {                          // column j in the lane, rows i in registers
            const Frag<NI> uj = load_frag<NI>(fr + (FU + jt) * kFrag, FP);
            if (has_u) gp[jt] = mul(gp[jt], df, uj);
            if (has_z) np[jt] = mul(np[jt], zf, uj);
          }
      }
      lds_barrier();                               // the fragments are read
    }
    if (LATE) stage_tiles();
    if (pairs) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) dots += __shfl_xor(dots, d);
    }
    const bool any = __any((held << 1) != 0);      // (a zero may have a sign)
    if (lane_id() == 0) {
      pair[w] = dots;
      holds[w] = any;
    }
    if (has_z) {
      zv = sum_groups(zv);
      if (gq == 0) zvs[tok] = zv;
    }
#pragma unroll
    for (int jt = 0; jt < 4; ++jt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ti = 16 * tt + 4 * gq + i, j = 16 * jt + m;
        const float D = jt <= tt && j <= ti ? decay(Ls[ti] - Ls[j]) : 0.f;
        if (has_u) G[ti * kLd + j] = j <= ti ? g.scale * (D * gp[jt][i]) : 0.f;
        if (has_z) N[ti * kLd + j] = j < ti ? -(D * np[jt][i]) : 0.f;
      }
    if (LATE || h == 0) wait_vmcnt<0>();           // K's and Q's tiles
    __syncthreads();
    const float e = vec[tok], wt = vec[C + tok], b = bs[tok];
    float qd = 0.f, ky = 0.f, kk = 0.f, kint = 0.f;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      a[rt] *= g.scale * e;
      y[rt] *= -e;
      kw[rt] *= wt;
      kint += dot4(tile_values<RB, NT>(kl, tok, 16 * (rt0 + rt) + 4 * gq), kw[rt]);
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int j0 = 32 * kb + 4 * gq;
      hold();
      if (kb <= tt / 2) {                          // rows i = tok, over j
        const float *Gr = G + tok * kLd + j0, *Nr = N + tok * kLd + j0;
        const Frag<NI> gf = split<NI>(*reinterpret_cast<const f32x4*>(Gr),
                                      *reinterpret_cast<const f32x4*>(Gr + 16));
        const Frag<NI> nf = split<NI>(*reinterpret_cast<const f32x4*>(Nr),
                                      *reinterpret_cast<const f32x4*>(Nr + 16));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const Frag<NT> kf = cols_of<RB, NT>(kl, rt0 + rt, kb);
          a[rt] = mul(a[rt], kf, gf);
          y[rt] = mul(y[rt], kf, nf);
        }
      }
      hold();
      if (kb >= tt / 2) {                          // columns j = tok, over i
        f32x4 gx[2], nx[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int ti = j0 + 16 * t + i;
            gx[t][i] = G[ti * kLd + tok];
            nx[t][i] = bs[ti] * N[ti * kLd + tok];
          }
        const Frag<NI> gf = split<NI>(gx[0], gx[1]), nf = split<NI>(nx[0], nx[1]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          kw[rt] = mul(kw[rt], cols_of<RB, NT>(ql, rt0 + rt, kb), gf);
          kw[rt] = mul(kw[rt], cols_of<RB, NT>(kl, rt0 + rt, kb), nf);
        }
      }
    }
    hold();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const f32x4 kv = tile_values<RB, NT>(kl, tok, 16 * (rt0 + rt) + 4 * gq);
      qd += dot4(tile_values<RB, NT>(ql, tok, 16 * (rt0 + rt) + 4 * gq), a[rt]);
      ky += dot4(kv, y[rt]);
      kk += dot4(kv, kw[rt]);
      const f32x4 dk = b * y[rt] + kw[rt];
      if constexpr (SHARED) {
        dQ[rt] += a[rt];
        dK[rt] += dk;
      } else if (live) {
        put(tok, rt, a[rt], dk);
      }
    }
    hold();
    qd = sum_groups(qd);
    ky = sum_groups(ky);
    kk = sum_groups(kk);
    kint = sum_groups(kint);
    if (gq == 0) {
      sums[hf][0][tok] = qd;
      sums[hf][1][tok] = ky;
      sums[hf][2][tok] = kk;
      sums[hf][3][tok] = kint;
    }
    __syncthreads();
    if (w == 0) {
      const int t = lane_id();
      float v4[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) v4[n] = H == 2 ? sums[0][n][t] + sums[H - 1][n][t] : sums[0][n][t];
      float x = v4[0] + bs[t] * v4[1] - v4[2], sum = v4[3], ds = 0.f;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const float up = __shfl_down(x, d);
        if (t + d < 64) x += up;
        sum += __shfl_xor(sum, d);
      }
#pragma unroll
      for (int n = 0; n < W; ++n) ds += pair[n];
      sum += vec[3 * C] * ds;                      // <dS', S'>
      bool enters = false;
#pragma unroll
      for (int n = 0; n < W; ++n) enters |= holds[n];
      if (t < len) {
        io.dlogA[(int64_t)s * g.T + t0 + t] = t > 0 || enters ? x + sum : 0.f;
        io.dbeta[(int64_t)s * g.T + t0 + t] = zvs[t] + v4[1];
      }
    }
  }
  const int tok = 16 * tt + (lane_id() & 15);
  if (SHARED && tok < len) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) put(tok, rt, dQ[rt], dK[rt]);
  }
}

template <typename In, int RB, bool OUT>
static void rchain(const Geo& g, const Ops& o, const RChainIO& io, int tiles, hipStream_t st) {
  constexpr int lds = rchain_lds<In, RB>(rchain_bufs<In, RB>()), W = rchain_waves<In, RB>();
  static_assert(lds <= kMaxLds, "");
  auto kern = delta_rchain_kernel<In, RB, OUT>;
  static uint64_t done;
  allow_lds(kern, lds, done);
  hipLaunchKernelGGL(kern, dim3(g.nb, (tiles + W - 1) / W, g.nruns), dim3(64 * W), lds, st, g, o,
                     io, tiles);
}

template <typename In, int RB>
static int backward(int dtype, const Geo& g, const In* q, const In* k, GradIO gr, void* dv,
                    const float* dstate_out, float* dstate, const bf16* save_m, void* ws,
                    hipStream_t st) {
  constexpr int eb = sizeof(In);
  Arena ar{(char*)ws};
  const Ops o = place_ops(ar, dtype, g, q, k, true);
  const bool qvec = vec4_ok(q, g.q_sb, g.q_st, eb), kvec = vec4_ok(k, g.k_sb, g.k_st, eb);
  gr.vvec = vec4_ok(gr.v, g.v_sb, g.v_st, eb);
  gr.dvec = vec4_ok(gr.dout, gr.d_sb, gr.d_st, eb);
  gr.ovec = vec4_ok(gr.dq, 0, g.r, eb) && vec4_ok(gr.dk, 0, g.r, eb);
  if (g.nch > 0)
    hipLaunchKernelGGL((delta_prep_kernel<In, RB, true>), dim3(g.nch, g.nb), dim3(256), 0, st, q,
                       k, gr.logA, gr.beta, g, o, qvec, kvec);
  RChainIO io = {};
  io.dout = gr.dout;
  io.d_sb = gr.d_sb;
  io.d_st = gr.d_st;
  io.dv = dv;
  io.start = dstate_out;
  io.fin = dstate;
  io.ptiles = (g.p + 15) / 16;
  if (g.nruns > g.nseg) {
    Carry c = take_carry(ar, g.nb, g.nruns, g.r, g.p, false);
    c.M = save_m;
    RChainIO first = io;
    first.start = nullptr;
    first.end = c.E;
    rchain<In, RB, false>(g, o, first, io.ptiles, st);
    const int rc = launch_carry(g, dstate_out, c, true, st);
    if (rc) return rc;
    io.start = c.start;
  }
  float* save_d = ar.take<float>((int64_t)g.nb * g.nch * 32 * RB * p32(g.p));
  float* z = ar.take<float>((int64_t)g.nb * g.nch * C * p32(g.p));
  io.save_d = save_d;
  io.z = z;
  io.ptiles = p32(g.p) / 16;
  rchain<In, RB, true>(g, o, io, io.ptiles, st);
  gr.save_d = save_d;
  gr.z = z;
  if (g.nch > 0) {
    constexpr int lds = grad_lds<In, RB>();
    static_assert(lds + 4096 <= kMaxLds, "");
    const bool full = g.p % 32 == 0 && gr.vvec && gr.dvec, shared = g.nb > g.nbk;
    auto kern = shared ? (full ? delta_grad_kernel<In, RB, true, true>
                               : delta_grad_kernel<In, RB, true, false>)
                       : (full ? delta_grad_kernel<In, RB, false, true>
                               : delta_grad_kernel<In, RB, false, false>);
    static uint64_t done[4];
    allow_lds(kern, lds, done[2 * shared + full]);
    hipLaunchKernelGGL(kern, dim3(g.nch, g.nbk), dim3(256 * grad_split(RB)), lds, st, g, o, gr);
  }
  return launch_status("smat_delta_scan_backward");
}

}  // namespace dl
}  // namespace smat

extern "C" int smat_delta_scan_backward(
    int dtype, const void* q, const void* k, const void* v, const float* logA, const float* beta,
    const void* dout, const float* dstate_out, const float* save_s, const float* save_u,
    const void* save_m, void* dq, void* dk, void* dv, float* dlogA, float* dbeta, float* dstate,
    const int32_t* chunks, const int32_t* runs, const int32_t* segrun, int nb, int nbk, int T,
    int nseg, int nch, int nruns, int K, int r, int p, float scale, int64_t q_sb, int64_t q_st,
    int64_t k_sb, int64_t k_st, int64_t v_sb, int64_t v_st, int64_t a_sb, int64_t a_st,
    int64_t b_sb, int64_t b_st, int64_t d_sb, int64_t d_st, void* workspace,
    int64_t workspace_bytes, void* stream) {
  using namespace smat;
  using namespace smat::dl;
  clear_error();
  const char* who = "smat_delta_scan_backward";
  const Geo g = {chunks, runs, segrun, nb, nbk, T, nseg, nch, nruns, K, r, p, scale,
                 q_sb, q_st, k_sb, k_st, v_sb, v_st, a_sb, a_st, b_sb, b_st};
  int rc = check_geo(who, dtype, g);
  if (rc == SMAT_OK) rc = check_grid(who, g);
  if (rc) return rc;
  if (nb == 0) return SMAT_OK;
  SMAT_REQUIRE(nch == 0 || (q && k && v && logA && beta && dout && save_s && save_u && dq && dk &&
                            dv && dlogA && dbeta && (save_m || nruns == nseg)),
               SMAT_EINVAL, "%s: null pointer", who);
  SMAT_REQUIRE(near_rows(v_st) && near_rows(d_st), SMAT_EUNSUPPORTED,
               "%s: rows of v or dout %lld and %lld elements apart, beyond 2^23", who,
               (long long)v_st, (long long)d_st);
  const int64_t need = smat_delta_workspace_bytes(dtype, nb, nbk, nch, nseg, nruns, r, p, 1);
  SMAT_REQUIRE(workspace_bytes >= need && (workspace || need == 0) &&
                   ((uintptr_t)workspace & 255) == 0,
               SMAT_EINVAL, "%s: workspace of %lld bytes, %lld needed (256-byte aligned)", who,
               (long long)workspace_bytes, (long long)need);
  GradIO gr = {};
  gr.v = v;
  gr.dout = dout;
  gr.logA = logA;
  gr.beta = beta;
  gr.d_sb = d_sb;
  gr.d_st = d_st;
  gr.save_s = save_s;
  gr.save_u = save_u;
  gr.dq = dq;
  gr.dk = dk;
  gr.dlogA = dlogA;
  gr.dbeta = dbeta;
  return dispatch(dtype, r, [&](auto in, auto rb) {
    typedef decltype(in) In;
    return backward<In, decltype(rb)::value>(dtype, g, (const In*)q, (const In*)k, gr, dv,
                                             dstate_out, dstate, (const bf16*)save_m, workspace,
                                             (hipStream_t)stream);
  });
}
