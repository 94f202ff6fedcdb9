// The gated delta rule over whole sequences (gated_delta_scan): the mathematics, the
// operand splits and the fragment layout are in delta_common.hpp, the state-free
// part of a chunk in delta_prep.hpp.
//
// delta_chain_kernel walks the chunks.  The columns of the state do not mix, so a
// wave takes 16 of them with all r rows in registers (fp32) and needs nothing of
// any other wave: K S and Q S from the state, U = T b (V - e K S), O, and the new
// state, each product's result tiles being the next one's operand as they lie.  The
// waves of a workgroup share the chunk's operands in LDS, copied there two phases
// ahead of their use: while K S, Q S and T run, the chunk's P and the next K land;
// while P U and K^T U run, the next Q and T.
//
// One wave walks a whole segment where sequences and columns give enough waves.
// Where they do not, segments are cut into runs: a first pass takes every run from
// the zero state for its end state E and from the identity for its transition M
// (its columns are more columns of the same recurrence, with V = 0), a kernel
// carries the states across the runs, S <- M S + E, and the second pass takes every
// run from its own state.
//
// What bounds it: the vector ALUs, which split every product's result into terms (eight
// operations a value), with the reloads of addresses spilled to vector lanes, and MFMA
// issue beside them.  8 sequences of 131072 tokens, r = p = 128 in bf16: 699 us for the
// first pass, 65 for the carry over 32 runs, 588 for the second, 0.76 PFLOP/s of issued
// products.  In training the second pass also writes S and U and runs at 4.7 TB/s (96 x
// 4096, r = p = 64: 127 us).
#include "delta_prep.hpp"

namespace smat {
namespace dl {

struct ChainIO {
  const void* v;
  void* o;
  const float* start;     // state entering run i of sequence s: start + (i nb + s) r p; or null
  float* end;             // first pass: the state leaving it, same layout
  bf16* trans;            // first pass: M of run i as fragments (trans_at, index i nb + s)
  bf16* save_m;           // training, first pass: M transposed, same layout; or null
  bool first_m, last_m;   // first pass: whether M of a segment's first, last run is wanted
  float* fin;             // state leaving segment j: fin + (j nb + s) r p; or null
  float *save_s, *save_u; // training: states entering chunks, and U, rows padded to p32; or null
  int ptiles;             // value tiles of 16 columns (tiles behind them are M's)
  bool ovec;              // out's rows in groups of four
};

// Bytes of LDS: KD buffers of K and the factors, T; and Q and P with the outputs.
template <typename In, int RB, bool OUT> constexpr int chain_lds(int KD) {
  constexpr int NT = Terms<In>::in, TB = kLow * kFrag * kMid;
  return KD * (2 * NT * tile_elems(RB) + kVec * 4) +
         2 * (TB + (OUT ? NT * tile_elems(RB) + TB : 0));
}
// fp32 tiles of more than 64 features fit once only: their next K is copied between
// the chunks.
template <typename In, int RB, bool OUT> constexpr int chain_bufs() {
  return chain_lds<In, RB, OUT>(2) <= kMaxLds ? 2 : 1;
}

// Two workgroups of four waves a CU where their LDS allows, else one of eight.
template <typename In, int RB, bool OUT> constexpr int chain_waves() {
  return 2 * chain_lds<In, RB, OUT>(chain_bufs<In, RB, OUT>()) <= kMaxLds ? 4 : 8;
}

template <typename In, int RB, bool OUT>
__global__ __launch_bounds__((64 * chain_waves<In, RB, OUT>()), 2) void delta_chain_kernel(
    Geo g, Ops o, ChainIO io, int tiles) {
  constexpr int NT = Terms<In>::in, NI = kMid, R = 32 * RB;
  constexpr int TL = NT * tile_elems(RB), TB = NI * kLow * kFrag;
  constexpr int KD = chain_bufs<In, RB, OUT>();
  extern __shared__ __align__(1024) bf16 lds[];
  bf16 *kl = lds, *tl = lds + KD * TL, *ql = tl + TB, *pl = ql + (OUT ? TL : 0);
  float* vl = reinterpret_cast<float*>(pl + (OUT ? TB : 0));
  constexpr int W = chain_waves<In, RB, OUT>();
  const int w = uniform_wave();
  const int ct = blockIdx.y * W + w;
  const int s = blockIdx.x;                        // sequences first: see below
  const int m = lane_id() & 15, gq = lane_id() >> 4;
  int run, c0, c1, seg;
  bool head, tail;
  run_of(g, blockIdx.z, run, c0, c1, seg, head, tail);
  const bool values = ct < io.ptiles;              // else columns of the transition
  bool on = ct < tiles;                            // else: copies and barriers only
  if (!OUT) {                                      // E of all runs but a segment's last, and M
    const bool e = !tail, t = !(head && tail) && (!head || io.first_m) && (!tail || io.last_m);
    const int w0 = blockIdx.y * W;
    if (!(e && w0 < io.ptiles) && !(t && w0 + W > io.ptiles)) return;
    on = on && (values ? e : t);
  }
  const int col = 16 * (values ? ct : ct - io.ptiles) + m;
  const int64_t ks = key_of(g, s);
  const int64_t rp = (int64_t)g.r * g.p, sn = (int64_t)run * g.nb + s;
  const int ld = (g.p + 31) / 32 * 32;

  f32x4 S[2 * RB];
#pragma unroll
  for (int mt = 0; mt < 2 * RB; ++mt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int a = 16 * mt + 4 * gq + i;
      if (!values)
        S[mt][i] = a == col ? 1.f : 0.f;
      else
        S[mt][i] = (io.start && a < g.r && col < g.p) ? io.start[sn * rp + (int64_t)a * g.p + col]
                                                      : 0.f;
    }
  const In* vs = (const In*)io.v + s * g.v_sb;
  const uint32_t soff = (4 * gq * ld + col) * 4;    // in fp32 rows of ld
  const bool vlive = values && col < g.p;
  uint32_t v[16];
  auto load_v = [&](int t0, int len) {
    load_column(v, vs, g.v_st, t0, len, values ? col : 0, g.p);
  };
  const TileStage<RB, NT, W> kstage(o.k, g.r, w), qstage(o.q, g.r, w);
  auto vec_of = [&](int c) { return o.vec + ((int64_t)s * g.nch + c) * kVec; };
  auto stage_k = [&](int c, int t0, int len, int buf) {
    kstage(kl + buf * TL, o.k, ks, g.nch, c, t0, len, g.r, vec_of(c), w);
    stage<1, W>(vl + buf * kVec, vec_of(c), W - 1 - w);
  };
  auto stage_qt = [&](int c, int t0, int len) {
    stage<NI * kLow, W>(tl, o.tm + ((int64_t)s * g.nch + c) * TB, w);
    if (OUT) qstage(ql, o.q, ks, g.nch, c, t0, len, g.r, vec_of(c), w);
  };

  int t0 = 0, len = 0, t1 = 0, len1 = 0;
  if (c0 < c1) {
    chunk_of(g, c0, t0, len);
    load_v(t0, len);
    stage_k(c0, t0, len, 0);
    stage_qt(c0, t0, len);
  }
  Frag<NI> sb[RB];                                 // S as the next products' operand
#pragma unroll
  for (int kb = 0; kb < RB; ++kb) sb[kb] = split<NI>(S[2 * kb], S[2 * kb + 1]);
  for (int c = c0; c < c1; ++c) {
    const int buf = KD == 2 ? (c - c0) & 1 : 0;
    const bool more = c + 1 < c1;
    const int64_t sc = (int64_t)s * g.nch + c;
    const bf16* kt = kl + buf * TL;
    const float* vec = vl + buf * kVec;
    const int lane = RB >= 3 ? fresh_lane() : lane_id(), fm = lane & 15, f4 = 4 * (lane >> 4);
    chunk_of(g, more ? c + 1 : c, t1, len1);
    wait_vmcnt<0>();
    lds_barrier();
    // ---- K, Q, T and the factors of chunk c are in LDS
    f32x4 x[4];
    column_values<In>(x, v, vlive, len);
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) asm volatile("" : "+v"(x[mt]));   // their wait is here
    if (OUT) stage<NI * kLow, W>(pl, o.pm + sc * TB, w);
    if (KD == 2 && more) stage_k(c + 1, t1, len1, 1 - buf);

    f32x4 ot[4];
    Frag<NI> f[2];
    if (on) {
      if (OUT && io.save_s) {
#pragma unroll
        for (int mt = 0; mt < 2 * RB; ++mt)
          put_rows(io.save_s + (sc * R + 16 * mt) * ld, soff, ld, S[mt]);
      }
      // K S, and Q S transposed (columns in registers, token in the lane)
      f32x4 ks4[4];
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) ks4[mt] = ot[mt] = zero4();
      constexpr int U = row_step(NT, RB);
      pipelined<4 / U * RB, Rows<NT, U>>(
          [&](int st, Rows<NT, U>& b) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int mt = st * U % 4 + u, kb = st * U / 4;
              b.k[u] = rows_of<RB, NT>(kt, mt, kb, lane);
              if (OUT) b.q[u] = rows_of<RB, NT>(ql, mt, kb, lane);
            }
          },
          [&](int st, Rows<NT, U>& b) {
            const int m0 = st * U % 4, kb = st * U / 4;
            f32x4 ca[U], co[U];
            Frag<NI> sa[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              ca[u] = ks4[m0 + u];
              co[u] = ot[m0 + u];
              sa[u] = sb[kb];
            }
            mul_each(ca, b.k, sa);
            if (OUT) mul_each(co, sa, b.q);
#pragma unroll
            for (int u = 0; u < U; ++u) {
              ks4[m0 + u] = ca[u];
              ot[m0 + u] = co[u];
            }
          });
      // b (V - e K S)
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const f32x4 e = *reinterpret_cast<const f32x4*>(vec + 16 * mt + f4);
        const f32x4 b = *reinterpret_cast<const f32x4*>(vec + 2 * C + 16 * mt + f4);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[mt][i] = b[i] * (x[mt][i] - e[i] * ks4[mt][i]);
        if (OUT) ot[mt] *= g.scale * vec[16 * mt + fm];
      }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) f[kb] = split<NI>(x[2 * kb], x[2 * kb + 1]);
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) x[mt] = zero4();
      triangle<false, NI>(x, tl, f, lane);         // U, in place of x
    }
    wait_vmcnt<0>();
    lds_barrier();
    // ---- P of chunk c and the next K are in LDS; Q and T are free
    load_v(t1, len1);                              // (the last chunk's once more: no branch)
    if (more) stage_qt(c + 1, t1, len1);
    if (on) {
      if (OUT && io.save_u) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
          put_rows(io.save_u + (sc * C + 16 * mt) * ld, soff, ld, x[mt]);
      }
      Frag<NI> fo[2];
      if (OUT) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) fo[kb] = split<NI>(x[2 * kb], x[2 * kb + 1]);
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
        x[mt] *= *reinterpret_cast<const f32x4*>(vec + C + 16 * mt + f4);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) f[kb] = split<NI>(x[2 * kb], x[2 * kb + 1]);
      if (OUT) {
        const uint32_t ooff = (fm * g.p + f4) * sizeof(In);
        const int left = g.p - 16 * ct - f4;
        triangle<true, NI>(ot, pl, fo, lane);
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          In* row = (In*)io.o + ((int64_t)s * g.T + t0 + 16 * mt) * g.p + 16 * ct;
          if (16 * mt + fm < len && left > 0)
            store4(reinterpret_cast<In*>(reinterpret_cast<char*>(row) + ooff), ot[mt],
                   io.ovec ? 4 : left, io.ovec);
        }
      }
      const float aC = vec[3 * C];
      update_state<RB, NT, false>(S, sb, aC, kt, f, kt, f, lane);
    }
    if (KD == 1 && more) {
      lds_barrier();                               // K is read
      stage_k(c + 1, t1, len1, 0);
    }
    t0 = t1;
    len = len1;
  }
  if (!OUT) lds_barrier();                         // the tiles are read: their place is free
  if (!on) return;
  if (!OUT && !values) {                           // sb: columns of M, the rows in the slots
    const int tile = ct - io.ptiles;
    if (io.save_m) {                               // which makes them rows of M transposed
#pragma unroll
      for (int kb = 0; kb < RB; ++kb)
        store_frag<NI>(io.save_m + trans_at<RB>(sn, tile, kb), kFrag, sb[kb]);
    }
    // rows of M, their 16 columns half a contraction block: transposed a term at a time in
    // the wave's part of LDS
    constexpr int LD = R + 4;
    static_assert(W * 16 * LD * 2 <= chain_lds<In, RB, OUT>(KD), "");
    bf16* part = lds + w * 16 * LD;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
#pragma unroll
      for (int kb = 0; kb < RB; ++kb) {
        const bf16x8 x = sb[kb].t[n];
        bf16* p = part + m * LD + 32 * kb + 4 * gq;
        *reinterpret_cast<bf16x4*>(p) = bf16x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<bf16x4*>(p + 16) = bf16x4{x[4], x[5], x[6], x[7]};
      }
      asm volatile("" ::: "memory");               // between lanes: a wave's LDS is in order
#pragma unroll
      for (int rt = 0; rt < 2 * RB; ++rt) {
        bf16x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = part[(4 * gq + i) * LD + 16 * rt + m];
        *reinterpret_cast<bf16x4*>(io.trans + trans_at<RB>(sn, rt, tile >> 1) + n * kFrag +
                                   lane_id() * 8 + 4 * (tile & 1)) = x;
      }
      asm volatile("" ::: "memory");
    }
    return;
  }
  float* out = OUT ? (io.fin && tail ? io.fin + ((int64_t)seg * g.nb + s) * rp : nullptr)
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

// The states entering the runs of a segment (start): S <- M_i S + E_i past each but
// the last, from init or from zero (then the first M is not used and need not exist);
// `rev` walks the runs backwards (the gradient's direction).  Every step waits on the
// last one, so a step is made short: a workgroup takes 16 columns only, wave w the rows
// [16 w, 16 w + 16) of them, M's rows and E's are loaded two steps ahead of their use,
// and the waves meet once, over their parts of S.  The sequences come first in the
// grid: the workgroups that read one M then mostly share an XCD's L2.
template <int RB>
__global__ __launch_bounds__(128 * RB) void delta_carry_kernel(Geo g,
                                                               const float* __restrict__ init,
                                                               const float* __restrict__ E,
                                                               const bf16* __restrict__ M,
                                                               float* __restrict__ start,
                                                               bool rev) {
  constexpr int NI = kMid;
  __shared__ __align__(16) bf16 parts[2][NI * RB * kFrag];
  const int w = uniform_wave(), m = lane_id() & 15, gq = lane_id() >> 4;
  const int col = 16 * blockIdx.y + m, seg = blockIdx.z, s = blockIdx.x;
  const int64_t rp = (int64_t)g.r * g.p;
  const int r0 = g.segrun ? g.segrun[seg] : 0, r1 = g.segrun ? g.segrun[seg + 1] : g.nruns;
  if (r0 >= r1) return;
  auto at = [&](int n) { return (int64_t)(rev ? r0 + r1 - 1 - n : n) * g.nb + s; };
  // element i is row 16 w + 4 gq + i; rows and columns past the end read the last one
  // there is
  uint32_t off[4];
  bool live[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int a = 16 * w + 4 * gq + i;
    live[i] = a < g.r && col < g.p;
    off[i] = (uint32_t)(min(a, g.r - 1) * g.p + min(col, g.p - 1));
  }
  struct Run {
    Frag<NI> m[RB];
    f32x4 e;
  };
  Run a, b, c;                                     // this step's, the next one's, and past it
  auto load = [&](const float* p) {
    f32x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = p[off[i]];
    return y;
  };
  auto keep = [&](f32x4 y) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = live[i] ? y[i] : 0.f;
    return y;
  };
  auto store = [&](float* p, const f32x4& y) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (live[i]) p[off[i]] = y[i];
  };
  const int last = max(r1 - 2, r0);                // (read once more at the end: no branch)
  auto load_run = [&](Run& x, int n) {
    const int64_t sn = at(min(n, last));
#pragma unroll
    for (int kb = 0; kb < RB; ++kb) x.m[kb] = load_frag<NI>(M + trans_at<RB>(sn, w, kb), kFrag);
    x.e = load(E + sn * rp);
  };
  f32x4 S = zero4();
  if (init) S = keep(load(init + ((int64_t)seg * g.nb + s) * rp));
  load_run(a, r0);
  load_run(b, r0 + 1);
  auto step = [&](int n, const Run& x, Run& behind) {
    bf16* part = parts[(n - r0) & 1];
    const Frag<NI> f = split<NI>(S, zero4());
#pragma unroll
    for (int t = 0; t < NI; ++t)                   // half a fragment: the wave's 16 rows
      *reinterpret_cast<bf16x4*>(part + (t * RB + (w >> 1)) * kFrag + lane_id() * 8 +
                                 4 * (w & 1)) =
          bf16x4{f.t[t][0], f.t[t][1], f.t[t][2], f.t[t][3]};
    store(start + at(n) * rp, S);
    load_run(behind, n + 2);
    lds_barrier();                                 // one a step: the parts alternate
    S = keep(x.e);
    if (n > r0 || init) {
#pragma unroll
      for (int kb = 0; kb < RB; ++kb)
        S = mul(S, x.m[kb], load_frag<NI>(part + kb * kFrag, RB * kFrag));
    }
  };
  for (int n = r0; n + 1 < r1; n += 3) {
    step(n, a, c);
    if (n + 2 >= r1) break;
    step(n + 1, b, a);
    if (n + 3 >= r1) break;
    step(n + 2, c, b);
  }
  store(start + at(r1 - 1) * rp, S);
}

int check_geo(const char* who, int dtype, const Geo& g) {
  SMAT_REQUIRE(dtype == SMAT_BF16 || dtype == SMAT_F16 || dtype == SMAT_F32, SMAT_EINVAL,
               "%s: unknown dtype %d", who, dtype);
  SMAT_REQUIRE(g.nb >= 0 && g.nbk >= 1 && g.T >= 0 && g.nseg >= 1 && g.nch >= 0, SMAT_EINVAL,
               "%s: bad sizes (nb=%d nbk=%d T=%d nseg=%d nch=%d)", who, g.nb, g.nbk, g.T, g.nseg,
               g.nch);
  SMAT_REQUIRE(g.nb % g.nbk == 0, SMAT_EINVAL, "%s: nbk=%d does not divide nb=%d", who, g.nbk,
               g.nb);
  SMAT_REQUIRE(g.r >= 1 && g.r <= kMaxR && g.p >= 1 && g.p <= kMaxP, SMAT_EUNSUPPORTED,
               "%s: r=%d p=%d beyond r<=%d, p<=%d", who, g.r, g.p, kMaxR, kMaxP);
  if (g.chunks || g.runs || g.segrun) {
    SMAT_REQUIRE(g.chunks && g.runs && g.segrun && g.nruns >= g.nseg, SMAT_EINVAL,
                 "%s: segments need the chunk, run and segment tables", who);
  } else {
    SMAT_REQUIRE(g.nseg == 1 && g.nch == (g.T + C - 1) / C, SMAT_EINVAL,
                 "%s: %d chunks for T=%d", who, g.nch, g.T);
    SMAT_REQUIRE(g.K >= 1 && g.nruns == (g.nch > 0 ? (g.nch + g.K - 1) / g.K : 1), SMAT_EINVAL,
                 "%s: %d runs of %d chunks for %d chunks", who, g.nruns, g.K, g.nch);
  }
  return SMAT_OK;
}

// The chunks' kernels have sequences, segments and runs along a grid's second and third axes.
int check_grid(const char* who, const Geo& g) {
  SMAT_REQUIRE(g.nb <= kMaxGrid && g.nruns <= kMaxGrid && g.nseg <= kMaxGrid, SMAT_EUNSUPPORTED,
               "%s: nb=%d, %d segments and %d runs must stay within %d", who, g.nb, g.nseg,
               g.nruns, kMaxGrid);
  return SMAT_OK;
}

template <int RB>
static void carry_kernel(const Geo& g, const float* init, const Carry& c, bool rev,
                         hipStream_t st) {
  hipLaunchKernelGGL(delta_carry_kernel<RB>, dim3(g.nb, (g.p + 15) / 16, g.nseg), dim3(128 * RB), 0,
                     st, g, init, c.E, c.M, c.start, rev);
}

int launch_carry(const Geo& g, const float* init, const Carry& c, bool rev, hipStream_t st) {
  switch (rblocks(g.r)) {
    case 1: carry_kernel<1>(g, init, c, rev, st); break;
    case 2: carry_kernel<2>(g, init, c, rev, st); break;
    case 3: carry_kernel<3>(g, init, c, rev, st); break;
    default: carry_kernel<4>(g, init, c, rev, st); break;
  }
  return launch_status("smat_delta_scan: carry");
}

template <typename In, int RB, bool OUT>
static void chain(const Geo& g, const Ops& o, const ChainIO& io, int tiles, hipStream_t st) {
  constexpr int lds = chain_lds<In, RB, OUT>(chain_bufs<In, RB, OUT>());
  constexpr int W = chain_waves<In, RB, OUT>();
  static_assert(lds <= kMaxLds, "");
  auto kern = delta_chain_kernel<In, RB, OUT>;
  static uint64_t done;
  allow_lds(kern, lds, done);
  // workgroups go to the XCDs in turn: with the sequences first, runs that are shorter or
  // not wanted leave every XCD as much; the runs table has the longest go first
  hipLaunchKernelGGL(kern, dim3(g.nb, (tiles + W - 1) / W, g.nruns), dim3(64 * W), lds, st, g, o,
                     io, tiles);
}

template <typename In, int RB>
static int scan(int dtype, const Geo& g, const In* q, const In* k, const void* v,
                const float* logA, const float* beta, const float* state, void* out,
                float* state_out, float* save_s, float* save_u, bf16* save_m, void* ws,
                hipStream_t st) {
  constexpr int eb = sizeof(In);
  Arena ar{(char*)ws};
  const Ops o = place_ops(ar, dtype, g, q, k, false);
  const bool qvec = vec4_ok(q, g.q_sb, g.q_st, eb), kvec = vec4_ok(k, g.k_sb, g.k_st, eb);
  if (g.nch > 0)
    hipLaunchKernelGGL((delta_prep_kernel<In, RB, false>), dim3(g.nch, g.nb), dim3(256), 0, st, q,
                       k, logA, beta, g, o, qvec, kvec);
  ChainIO io = {};
  io.v = v;
  io.o = out;
  io.start = state;
  io.fin = state_out;
  io.ovec = vec4_ok(out, 0, g.p, eb);
  io.ptiles = (g.p + 15) / 16;
  if (g.nruns > g.nseg) {
    const Carry c = take_carry(ar, g.nb, g.nruns, g.r, g.p, true);
    ChainIO first = io;
    first.o = nullptr;
    first.start = nullptr;
    first.end = c.E;
    first.trans = c.trans;
    first.save_m = save_m;
    first.first_m = state != nullptr;
    first.last_m = save_m && state_out;            // else nothing comes from behind it
    chain<In, RB, false>(g, o, first, io.ptiles + 2 * RB, st);
    const int rc = launch_carry(g, state, c, false, st);
    if (rc) return rc;
    io.start = c.start;
  }
  io.save_s = save_s;
  io.save_u = save_u;
  if (save_s) io.ptiles = p32(g.p) / 16;
  chain<In, RB, true>(g, o, io, io.ptiles, st);
  return launch_status("smat_delta_scan");
}

}  // namespace dl
}  // namespace smat

// Run length: of the lengths that cut the longest segment into 1 to 256 runs, the one
// whose passes take least by what their steps measure, in microseconds a chunk with a
// workgroup on every CU: 3.4 + 0.375 RB with outputs, 1.9 + 0.24 RB in the first pass,
// 1.9 times that where inputs have several terms (measured in fp16; fp32, with three and
// one buffer of K from 96 features on, is taken for the same); 0.55 RB a run of the carry
// and 10 for the two launches more.  Workgroups of four waves share a CU in pairs, which then take
// 1.64 times as long; more than are resident follow one another, the last ones alone.
// (8 sequences of 2048 chunks, r = p = 128: 10915 whole, 1446 in 32 runs, 1496 in 64,
// 1648 in 128; 12 of 5 segments and 158 chunks, r = p = 96 in fp16: 734 whole, 242 in
// runs of 9, 247 of 8, 294 of 16.)  A step with outputs takes 4.0 + 0.43 RB by now; priced
// so, the rule cuts finer, which suits forwards alone (32 x 128 chunks, r = p = 64: 188,
// not 198) and costs training, whose backward walks the same runs (79 x 18 chunks, r = 64,
// p = 128: 365, not 337): over the ten of 123 sizes that it moves, 2 % lost.
extern "C" int smat_delta_run_chunks(int dtype, int nb, int nch, const int32_t* lengths,
                                     const int32_t* times, int n, int r, int p) {
  using namespace smat::dl;
  const bool packed = lengths && times && n > 0;
  int longest = packed ? 0 : nch;
  for (int i = 0; packed && i < n; ++i) longest = lengths[i] > longest ? lengths[i] : longest;
  if (longest < 1 || nb < 1 || r < 1 || p < 1 || r > kMaxR || dtype < SMAT_BF16 ||
      dtype > SMAT_F32)
    return 1;
  const int RB = rblocks(r), tiles = (p + 15) / 16;
  int wout = 4, wfirst = 4;
  dispatch(dtype, r, [&](auto in, auto rb) {
    wout = chain_waves<decltype(in), decltype(rb)::value, true>();
    wfirst = chain_waves<decltype(in), decltype(rb)::value, false>();
    return 0;
  });
  const double terms = dtype == SMAT_BF16 ? 1.0 : 1.9;
  // a pass of wgs workgroups of up to K chunks, `steps` chunks in all
  auto pass = [&](double wgs, double steps, int K, int waves, double cost) {
    const double share = waves == 4 ? 0.82 : 1.0;
    if (wgs <= 256) return K * cost;
    if (waves == 4 && wgs <= 512) return 2 * share * K * cost;
    return (share * steps / 256 + 0.4 * K) * cost;
  };
  int best = longest;
  double least = 0;
  for (int G = 1; G <= 256 && (G == 1 || longest / G >= 2); ++G) {
    const int K = (longest + G - 1) / G;
    double runs = 0, chunks = 0, ends = 0;         // `ends`: runs with one behind them
    for (int i = 0; i < (packed ? n : 1); ++i) {
      const double len = packed ? lengths[i] : nch, t = packed ? times[i] : 1;
      const double cut = len > K ? (int)((len + K - 1) / K) : 1;
      runs += t * cut;
      ends += t * (cut - 1);
      chunks += t * len;
    }
    if (G > 1 && runs > kMaxGrid) continue;        // more than a grid holds
    const double out = (double)nb * ((tiles + wout - 1) / wout);
    const double first = (double)nb * ((tiles + 2 * RB + wfirst - 1) / wfirst);
    double us = pass(runs * out, chunks * out, K, wout, terms * (3.4 + 0.375 * RB));
    if (ends > 0)
      us += pass(ends * first, ends * K * first, K, wfirst, terms * (1.9 + 0.24 * RB)) +
            G * 0.55 * RB + 10;
    if (G == 1 || us < least) {
      least = us;
      best = K;
    }
  }
  return best;
}

extern "C" int64_t smat_delta_workspace_bytes(int dtype, int nb, int nbk, int nch, int nseg,
                                              int nruns, int r, int p, int backward) {
  using namespace smat::dl;
  Arena ar{nullptr};
  take_ops(ar, dtype, nb, nbk, nch, r, backward != 0, false);
  if (nruns > nseg) take_carry(ar, nb, nruns, r, p, backward == 0);
  if (backward) {
    ar.take<float>((int64_t)nb * nch * 32 * rblocks(r) * p32(p));   // dS' of every chunk
    ar.take<float>((int64_t)nb * nch * C * p32(p));                 // Z
  }
  return ar.used;
}

extern "C" int smat_delta_scan(int dtype, const void* q, const void* k, const void* v,
                               const float* logA, const float* beta, const float* state, void* out,
                               float* state_out, float* save_s, float* save_u, void* save_m,
                               const int32_t* chunks, const int32_t* runs, const int32_t* segrun,
                               int nb, int nbk, int T, int nseg, int nch, int nruns, int K, int r,
                               int p, float scale, int64_t q_sb, int64_t q_st, int64_t k_sb,
                               int64_t k_st, int64_t v_sb, int64_t v_st, int64_t a_sb,
                               int64_t a_st, int64_t b_sb, int64_t b_st, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  using namespace smat;
  using namespace smat::dl;
  clear_error();
  const char* who = "smat_delta_scan";
  const Geo g = {chunks, runs, segrun, nb, nbk, T, nseg, nch, nruns, K, r, p, scale,
                 q_sb, q_st, k_sb, k_st, v_sb, v_st, a_sb, a_st, b_sb, b_st};
  const int rc = check_geo(who, dtype, g);
  if (rc) return rc;
  if (nb == 0) return SMAT_OK;
  SMAT_REQUIRE(nch == 0 || (q && k && v && logA && beta && out), SMAT_EINVAL, "%s: null pointer",
               who);
  SMAT_REQUIRE(!save_s == !save_u && (save_s && nruns > nseg ? save_m != nullptr : !save_m),
               SMAT_EINVAL, "%s: save_s, save_u and (with more runs than segments) save_m go "
               "together", who);
  SMAT_REQUIRE(state_out != state || !state, SMAT_EINVAL, "%s: state_out must not be state", who);
  hipStream_t st = (hipStream_t)stream;
  if (!chunks && !save_s && T >= 1 && T <= kFewTokens)
    return launch_tokens(who, dtype, g, q, k, v, logA, beta, state, state_out, out, st);
  const int fits = check_grid(who, g);
  if (fits) return fits;
  SMAT_REQUIRE(near_rows(v_st), SMAT_EUNSUPPORTED, "%s: rows of v %lld elements apart, beyond 2^23",
               who, (long long)v_st);
  const int64_t need = smat_delta_workspace_bytes(dtype, nb, nbk, nch, nseg, nruns, r, p, 0);
  SMAT_REQUIRE(workspace_bytes >= need && (workspace || need == 0) &&
                   ((uintptr_t)workspace & 255) == 0,
               SMAT_EINVAL, "%s: workspace of %lld bytes, %lld needed (256-byte aligned)", who,
               (long long)workspace_bytes, (long long)need);
  auto go = [&](auto in, auto rb) {
    typedef decltype(in) In;
    return scan<In, decltype(rb)::value>(dtype, g, (const In*)q, (const In*)k, v, logA, beta,
                                         state, out, state_out, save_s, save_u,
                                         (bf16*)save_m, workspace, st);
  };
  return dispatch(dtype, r, go);
}
