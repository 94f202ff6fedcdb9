// Linear attention with a decay for each head (head_decay_scan and its gradient): the walk
// over a sequence's chunks that all of its passes are.
//
//   S_t = a S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t,   a = exp(logA) of the head.
//
// Over a chunk of n <= 64 tokens entered with state S, with e_i = a^(i+1),
// w_j = a^(n-1-j) and D_ij = a^(i-j) (j <= i, else 0):
//
//   O  = scale (e (Q S) + ((Q K^T) o D) V)
//   S' = a^n S + K^T (w V)
//
// The gradient is three walks of the same form.  With Y_t the gradient of S_t from the
// tokens behind t, Y_{t-1} = a (Y_t + scale q_t do_t^T):
//
//   dq_i = scale S_i do_i:                       forward over (dO, V, K), state S^T
//   dv_j = (Y_j + scale q_j do_j^T)^T k_j:       backward over (K, Q, dO), state Y
//   dk_j = (Y_j + scale q_j do_j^T) v_j:         backward over (V, dO, Q), state Y^T
//
// A walk backwards takes the tokens in turned order; then its in-chunk part is the forward
// one's, and its factors are e_i = a^i, w_j = a^(n-j).
//
// The columns of the state do not mix, so a wave takes 16 of them with all key rows in
// registers (fp32).  A workgroup has all columns of a sequence: its waves share the
// chunk's rows in LDS and one P = (Q K^T) o D, of which each forms a few tiles.
//
// Operands: every product runs on v_mfma_f32_16x16x32_bf16, values held in fewer than
// their own bits as sums of bf16 terms (delta_common.hpp): bf16 inputs one term, fp16 two,
// fp32 and what is computed in fp32 (P, the state, w V) three, 24 bits.  Results are
// rounded once, where they are stored.
#pragma once

#include "delta_common.hpp"
#include "row_groups.hpp"

namespace smat {
namespace hd {

using dl::C;
using dl::Frag;
using dl::Terms;
using dl::kFrag;
using dl::kLow;
using dl::kMid;

constexpr int kMaxD = 128;         // features and value columns
constexpr int kMinD = 8;           // narrower rows come padded: rows are read eight at a time
constexpr int kTiles = 10;         // 16 x 16 tiles of a chunk's lower triangle

// Rows of one operand: sequence s reads those of s / div.
struct Side {
  const void* p;
  int64_t sb, st;
  int div;
};

// What a walk with LEARN sums of the decay's gradient:
//   d loss / d logA = sum_ij (i - j) P_ij (do_i . v_j)  +  sum_i (i + 1) q_i . (inter of dq_i)
//                   + sum_j (n - 1 - j) k_j . (inter of dk_j)  +  n a^n <S, Y>
// over the chunks, every term with a factor of at most 64, so that nothing cancels that does
// not cancel in the sum itself.
enum Learn { kNone = 0, kDq = 1, kDk = 2, kDv = 3 };

struct Walk {
  const int32_t *chunks, *runs, *segrun;   // as the gated delta rule's (delta_common.hpp)
  int nb, T, nseg, nch, nruns, K;
  int r, p;                // key and value columns of this walk
  Side q, k, v;
  const float* logA;       // (heads), sequence s has head s % heads
  int heads;
  bool rev;
  float upd, inter, intra; // factors of the state's update and of the output's two parts
  const float* start;      // state entering run i of sequence s: start + (i nb + s) r p; or null
  float* fin;              // state leaving segment j (first pass: run j), same layout; or null
  int s_row, s_col;        // element strides in a state of start and fin
  void* o;                 // (nb, T, p) contiguous
  bool wide;               // o is fp32
  float* save_s;           // states entering chunks in the kernel's layout; or null
  const float* load_s;     // LEARN kDv: what save_s received
  Side x;                  // LEARN kDq: Q; kDk: K
  int learn;
  float* part;             // LEARN: (nruns, nb, W)
};

// One operand's rows of a chunk on their way to LDS: loaded a chunk ahead into registers,
// then written as a tile (delta_common.hpp), a tile a term.  B: 32-column blocks.
template <typename In, int B, int W> struct Rows {
  static constexpr int LC = 4 * B, RS = dl::row_chunks(B), UNITS = C * LC;
  static constexpr int U = (UNITS + 64 * W - 1) / (64 * W);
  Raw<In> x[U];

  __device__ __forceinline__ static void place(int u, int& t, int& k) {
    const int i = u * 64 * W + (int)threadIdx.x;
    t = i / LC;
    k = i % LC;
  }
  // base: the walk's first row of the chunk, st: to the next one in the walk's order.  Rows
  // past the last are the last one's, and a group that would pass the row's end is read
  // earlier in it (cols >= 8): every address lies in the operand.
  __device__ __forceinline__ void load(const In* base, int64_t st, int len, int cols) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      int t, k;
      place(u, t, k);
      x[u].load(base + min(t, len - 1) * st + min(8 * k, cols - 8));
    }
  }
  __device__ __forceinline__ void put(bf16* tile, int len, int cols) {
    const int over = cols & 7;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      int t, k;
      place(u, t, k);
      if (UNITS % (64 * W) && t >= C) break;
      if (over && 8 * k + 8 > cols && 8 * k < cols) x[u].drop(8 - over);
      if (t >= len || 8 * k >= cols) x[u].zero();
      bf16* at = tile + (t * RS + (k ^ dl::swz<RS>(t))) * 8;
      if constexpr (__is_same(In, bf16)) {
        *reinterpret_cast<typename Raw<In>::u4*>(at) = x[u].x[0];
      } else {
        f32x4 a, b;
        x[u].values(a, b);
        const Frag<Terms<In>::in> f = dl::split<Terms<In>::in>(a, b);
#pragma unroll
        for (int n = 0; n < Terms<In>::in; ++n)
          *reinterpret_cast<bf16x8*>(at + n * dl::tile_elems(B)) = f.t[n];
      }
    }
  }
};

template <int W> __device__ __host__ constexpr int value_blocks() { return W / 2; }

// Elements of a set of tiles, Q (where there are outputs), K and V, and bytes of LDS.
template <typename In, int RB, int W, bool OUT> constexpr int set_elems() {
  return Terms<In>::in *
         ((OUT ? 2 : 1) * dl::tile_elems(RB) + dl::tile_elems(value_blocks<W>()));
}
constexpr int kTab = C + 4 + 2 * C;   // floats: a^0 .. a^64; the update's factors, zeros behind
template <typename In, int RB, int W, bool OUT> constexpr int walk_lds(int KD) {
  return KD * set_elems<In, RB, W, OUT>() * 2 + (OUT ? kMid * kLow * kFrag * 2 : 0) +
         kTab * 4;
}
// Two sets, so that the next chunk's rows are written beside this one's use, where that
// fits half (W = 4) or all of a CU's LDS.
template <typename In, int RB, int W, bool OUT> constexpr int walk_sets() {
  return walk_lds<In, RB, W, OUT>(2) <= (W == 4 ? dl::kMaxLds / 2 : dl::kMaxLds) ? 2 : 1;
}

// Rows fragment of a tile at a row tile known at run time only.
template <int B, int N>
__device__ __forceinline__ Frag<N> row_frag(const bf16* tile, int mt, int kb) {
  constexpr int RS = dl::row_chunks(B);
  const int m = lane_id() & 15, g = lane_id() >> 4;
  const int k0 = (4 * kb + (g >> 1)) ^ dl::swz<RS>(m), k1 = (4 * kb + 2 + (g >> 1)) ^ dl::swz<RS>(m);
  const bf16* p = tile + (16 * mt + m) * RS * 8 + 4 * (g & 1);
  Frag<N> f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(p + n * dl::tile_elems(B) + k0 * 8);
    const bf16x4 b = *reinterpret_cast<const bf16x4*>(p + n * dl::tile_elems(B) + k1 * 8);
    f.t[n] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return f;
}

// The same fragment from the caller's rows: row tile mt of the chunk, 32-column block kb.
template <typename In>
__device__ __forceinline__ Frag<Terms<In>::in> global_frag(const In* base, int64_t st, int len,
                                                           int cols, int mt, int kb) {
  const int t = 16 * mt + (lane_id() & 15), g = lane_id() >> 4;
  const In* row = base + min(t, len - 1) * st;
  f32x4 h[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 32 * kb + 16 * i + 4 * g + j;
      const float x = to_f32(row[min(c, cols - 1)]);
      h[i][j] = t < len && c < cols ? x : 0.f;
    }
  return dl::split<Terms<In>::in>(h[0], h[1]);
}

template <int N> __device__ __forceinline__ void values_of(const Frag<N>& f, f32x4& a, f32x4& b) {
  a = b = zero4();
#pragma unroll
  for (int n = N - 1; n >= 0; --n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] += to_f32(f.t[n][i]);
      b[i] += to_f32(f.t[n][i + 4]);
    }
}

// A product rounded here, not fused into what reads it: results keep their bits whichever
// variant of the kernel forms them.
__device__ __forceinline__ f32x4 rounded(f32x4 x) {
  asm("" : "+v"(x));
  return x;
}

__device__ __forceinline__ void tile_of(int i, int& mt, int& jt) {
  mt = i < 1 ? 0 : i < 3 ? 1 : i < 6 ? 2 : 3;
  jt = i - mt * (mt + 1) / 2;
}

template <typename In, int RB, int W, bool OUT, bool LEARN>
__global__ __launch_bounds__(64 * W, 2) void decay_walk_kernel(Walk g) {
  constexpr int NT = Terms<In>::in, NI = kMid, VB = value_blocks<W>();
  constexpr int KT = NT * dl::tile_elems(RB), SET = set_elems<In, RB, W, OUT>();
  constexpr int KD = walk_sets<In, RB, W, OUT>(), TP = (kTiles + W - 1) / W;
  extern __shared__ __align__(1024) bf16 lds[];
  bf16* pl = lds + KD * SET;
  float* tab = reinterpret_cast<float*>(pl + (OUT ? NI * kLow * kFrag : 0));   // a^0 .. a^64
  float* wt = tab + C + 4;                         // wt[64 - n + j] = w_j of a chunk of n
  const int w = dl::uniform_wave(), s = blockIdx.x;
  const int m = lane_id() & 15, gq = lane_id() >> 4;
  int run, c0, c1, seg;
  bool head, tail;
  {
    dl::Geo geo = {};
    geo.chunks = g.chunks;
    geo.runs = g.runs;
    geo.segrun = g.segrun;
    geo.T = g.T;
    geo.nch = g.nch;
    geo.nruns = g.nruns;
    geo.K = g.K;
    dl::run_of(geo, blockIdx.y, run, c0, c1, seg, head, tail);
  }
  if (!OUT && (g.rev ? head : tail)) return;       // no run follows it
  auto chunk_at = [&](int i, int& t0, int& len) {
    const int c = g.rev ? c1 - 1 - i : c0 + i;
    if (g.chunks) {
      t0 = g.chunks[2 * c];
      len = g.chunks[2 * c + 1];
    } else {
      t0 = c * C;
      len = min(C, g.T - t0);
    }
  };
  const int chunks = c1 - c0, col = 16 * w + m;
  const bool on = 16 * w < g.p;                    // else: copies, tiles of P and barriers only
  const int64_t sn = (int64_t)run * g.nb + s, rp = (int64_t)g.r * g.p;
  {
    // powers from 64 bits: a^i is then rounded once, however long the product
    const double la = g.logA[s % g.heads];
    const int i = threadIdx.x;
    if (i <= C) tab[i] = i == 0 ? 1.f : (float)exp(la * i);
    if (i < 2 * C) {
      const int e = C - 1 - i + (g.rev ? 1 : 0);
      wt[i] = i < C ? (e == 0 ? 1.f : (float)exp(la * e)) * g.upd : 0.f;
    }
  }
  f32x4 S[2 * RB];
#pragma unroll
  for (int mt = 0; mt < 2 * RB; ++mt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int a = 16 * mt + 4 * gq + i;
      S[mt][i] = g.start && a < g.r && col < g.p
                     ? g.start[sn * rp + (int64_t)a * g.s_row + (int64_t)col * g.s_col]
                     : 0.f;
    }
  const In *qs = (const In*)g.q.p + s / g.q.div * g.q.sb, *ks = (const In*)g.k.p + s / g.k.div * g.k.sb,
           *vs = (const In*)g.v.p + s / g.v.div * g.v.sb;
  auto first_row = [&](const In* p, int64_t st, int t0, int len) {
    return p + (int64_t)(g.rev ? t0 + len - 1 : t0) * st;
  };
  auto step_of = [&](int64_t st) { return g.rev ? -st : st; };
  Rows<In, RB, W> rq, rk;
  Rows<In, VB, W> rv;
  auto load = [&](int t0, int len) {
    if (OUT) rq.load(first_row(qs, g.q.st, t0, len), step_of(g.q.st), len, g.r);
    rk.load(first_row(ks, g.k.st, t0, len), step_of(g.k.st), len, g.r);
    rv.load(first_row(vs, g.v.st, t0, len), step_of(g.v.st), len, g.p);
  };
  auto put = [&](bf16* set, int len) {
    rk.put(set, len, g.r);
    rv.put(set + KT, len, g.p);
    if (OUT) rq.put(set + KT + NT * dl::tile_elems(VB), len, g.r);
  };
  int t0 = 0, len = 0;
  if (chunks > 0) {
    chunk_at(0, t0, len);
    load(t0, len);
    put(lds, len);
  }
  Frag<NI> sb[OUT ? RB : 1];                       // S as the next product's operand
  if (OUT) {
#pragma unroll
    for (int kb = 0; kb < RB; ++kb) sb[kb] = dl::split<NI>(S[2 * kb], S[2 * kb + 1]);
  }
  lds_barrier();
  float e[4];
  f32x4 D[OUT ? TP : 1];
  if (OUT) {
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) e[mt] = g.inter * tab[16 * mt + m + (g.rev ? 0 : 1)];
#pragma unroll
    for (int u = 0; u < TP; ++u) {
      int mt, jt;
      tile_of(min(w + u * W, kTiles - 1), mt, jt);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 16 * (mt - jt) + m - 4 * gq - i;
        D[u][i] = d >= 0 ? g.intra * tab[d] : 0.f;
      }
    }
  }
  float acc = 0.f;                                 // LEARN: this lane's part of the gradient

  for (int c = 0; c < chunks; ++c) {
    bf16* set = lds + (KD == 2 ? (c & 1) * SET : 0);
    const bf16 *kt = set, *vt = set + KT, *qt = vt + NT * dl::tile_elems(VB);
    const bool more = c + 1 < chunks;
    int t1 = t0, len1 = len;
    if (c > 0) lds_barrier();
    // ---- the chunk's rows are in LDS
    if (more) {
      chunk_at(c + 1, t1, len1);
      load(t1, len1);
    }
    const float aC = tab[len];
    f32x4 ot[OUT ? 4 : 1];
    if constexpr (OUT) {
#pragma unroll
      for (int u = 0; u < TP; ++u) {
        if (w + u * W >= kTiles) break;
        int mt, jt;
        tile_of(w + u * W, mt, jt);
        // transposed: rows are tokens j, columns i
        f32x4 x = zero4();
#pragma unroll
        for (int kb = 0; kb < RB; ++kb)
          x = dl::mul_inputs(x, row_frag<RB, NT>(kt, jt, kb), row_frag<RB, NT>(qt, mt, kb));
        x = rounded(x * D[u]);
        if constexpr (LEARN) {
          if (g.learn == kDq) {                    // here i: dO, j: V; and V's place has K
            const In* xs = (const In*)g.x.p + s / g.x.div * g.x.sb;
            f32x4 z = zero4();
            for (int kb = 0; kb < VB; ++kb)
              z = dl::mul_inputs(z, row_frag<VB, NT>(vt, jt, kb),
                                 global_frag(first_row(xs, g.x.st, t0, len), step_of(g.x.st), len,
                                             g.p, mt, kb));
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc += (float)(16 * (mt - jt) + m - 4 * gq - i) * (x[i] * z[i]);
          }
        }
        const Frag<NI> f = dl::split<NI>(x, zero4());
        const int half = mt == 2 && jt == 2 ? 1 : jt & 1;
        bf16* at = pl + dl::tri(mt, jt >> 1) * kFrag + lane_id() * 8 + 4 * half;
#pragma unroll
        for (int n = 0; n < NI; ++n)
          *reinterpret_cast<bf16x4*>(at + n * kLow * kFrag) = dl::low_half(f.t[n]);
      }
      if (on) {
        if (g.save_s) {
          f32x4* to = reinterpret_cast<f32x4*>(g.save_s) +
                      (((int64_t)s * g.nch + c0 + c) * W + w) * (2 * RB * 64) + lane_id();
#pragma unroll
          for (int mt = 0; mt < 2 * RB; ++mt) to[mt * 64] = S[mt];
        }
        // (Q S)^T: columns in registers, the token in the lane
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) ot[mt] = zero4();
#pragma unroll
        for (int kb = 0; kb < RB; ++kb)
#pragma unroll
          for (int mt = 0; mt < 4; ++mt)
            ot[mt] = dl::mul(ot[mt], sb[kb], dl::rows_of<RB, NT>(qt, mt, kb));
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) ot[mt] = rounded(ot[mt] * e[mt]);
        if constexpr (LEARN) {
          if (g.learn == kDq || g.learn == kDk) {  // (i + 1) q . dq, and i k . dk in turned order
            const In* xs = (const In*)g.x.p + s / g.x.div * g.x.sb;
            const In* base = first_row(xs, g.x.st, t0, len);
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
              const int t = 16 * mt + m;
              const In* row = base + min(t, len - 1) * step_of(g.x.st);
              float dot = 0.f;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int cc = 16 * w + 4 * gq + i;
                const float x = to_f32(row[min(cc, g.p - 1)]);
                dot += cc < g.p ? x * ot[mt][i] : 0.f;
              }
              if (t < len) acc += (float)(t + (g.rev ? 0 : 1)) * dot;
            }
          } else if (g.learn == kDv) {             // n a^n <S, Y>
            const f32x4* from = reinterpret_cast<const f32x4*>(g.load_s) +
                                (((int64_t)s * g.nch + c1 - 1 - c) * W + w) * (2 * RB * 64) +
                                lane_id();
            float dot = 0.f;
#pragma unroll
            for (int mt = 0; mt < 2 * RB; ++mt) {
              const f32x4 x = from[mt * 64];
#pragma unroll
              for (int i = 0; i < 4; ++i) dot += x[i] * S[mt][i];
            }
            acc += (float)len * aC * dot;
          }
        }
      }
      lds_barrier();
      // ---- P is in LDS
    }
    if (on) {
      Frag<NT> vf[2];
      Frag<NI> f[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        vf[kb] = dl::cols_of<VB, NT>(vt, w, kb);
        f32x4 a, b, wa, wb;
        values_of(vf[kb], a, b);
        const float* wp = wt + C - len + 32 * kb + 4 * gq;
        if (len == C) {
          wa = *reinterpret_cast<const f32x4*>(wp);
          wb = *reinterpret_cast<const f32x4*>(wp + 16);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            wa[i] = wp[i];
            wb[i] = wp[16 + i];
          }
        }
        f[kb] = dl::split<NI>(rounded(wa * a), rounded(wb * b));
      }
      if constexpr (OUT) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int kb = 0; kb <= mt / 2; ++kb) {
            Frag<NI> pf;
            const bf16* at = pl + dl::tri(mt, kb) * kFrag + lane_id() * 8;
#pragma unroll
            for (int n = 0; n < NI; ++n) {
              if (dl::half_tri(mt, kb)) {
                const bf16x4 h =
                    *reinterpret_cast<const bf16x4*>(at + n * kLow * kFrag + (mt == 2 ? 4 : 0));
                const bf16x4 no = {(bf16)0.f, (bf16)0.f, (bf16)0.f, (bf16)0.f};
                pf.t[n] = __builtin_shufflevector(h, no, 0, 1, 2, 3, 4, 5, 6, 7);
              } else {
                pf.t[n] = *reinterpret_cast<const bf16x8*>(at + n * kLow * kFrag);
              }
            }
            ot[mt] = dl::mul(ot[mt], vf[kb], pf);
          }
        const int c4 = 16 * w + 4 * gq;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          const int t = 16 * mt + m;
          if (t >= len || c4 >= g.p) continue;
          const int64_t at = ((int64_t)s * g.T + (g.rev ? t0 + len - 1 - t : t0 + t)) * g.p + c4;
          auto store = [&](auto* o) {
            typedef typename std::remove_pointer<decltype(o)>::type Out;
            typedef Out out4u __attribute__((ext_vector_type(4), aligned(sizeof(Out))));
            if (c4 + 4 <= g.p) {
              out4u y;
#pragma unroll
              for (int i = 0; i < 4; ++i) y[i] = from_f32<Out>(ot[mt][i]);
              *reinterpret_cast<out4u*>(o + at) = y;
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (c4 + i < g.p) o[at + i] = from_f32<Out>(ot[mt][i]);
            }
          };
          if (!__is_same(In, float) && g.wide)
            store((float*)g.o);
          else
            store((In*)g.o);
        }
      }
      // S <- a^n S + K^T (w V)
#pragma unroll
      for (int mt = 0; mt < 2 * RB; ++mt) {
        f32x4 x = S[mt] * aC;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) x = dl::mul(x, dl::cols_of<RB, NT>(kt, mt, kb), f[kb]);
        S[mt] = x;
      }
      if constexpr (OUT) {
#pragma unroll
        for (int kb = 0; kb < RB; ++kb) sb[kb] = dl::split<NI>(S[2 * kb], S[2 * kb + 1]);
      }
    }
    if (more) {
      if (KD == 1) lds_barrier();                  // the tiles are read
      put(lds + (KD == 2 ? ((c + 1) & 1) * SET : 0), len1);
    }
    t0 = t1;
    len = len1;
  }
  if (LEARN && g.learn) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) acc += __shfl_xor(acc, d);
    if (lane_id() == 0) g.part[sn * W + w] = acc;
  }
  if (!on || !g.fin || (OUT && !(g.rev ? head : tail))) return;
  float* out = g.fin + (OUT ? (int64_t)seg * g.nb + s : sn) * rp;
#pragma unroll
  for (int mt = 0; mt < 2 * RB; ++mt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int a = 16 * mt + 4 * gq + i;
      if (a < g.r && col < g.p)
        out[(int64_t)a * g.s_row + (int64_t)col * g.s_col] = S[mt][i];
    }
}

inline int waves_of(int p) { return p <= 64 ? 4 : 8; }

template <typename In, int RB, int W, bool OUT, bool LEARN>
static void walk(const Walk& g, hipStream_t st) {
  constexpr int lds = walk_lds<In, RB, W, OUT>(walk_sets<In, RB, W, OUT>());
  static_assert(lds <= dl::kMaxLds, "");
  auto kern = decay_walk_kernel<In, RB, W, OUT, LEARN>;
  static uint64_t done;
  dl::allow_lds(kern, lds, done);
  hipLaunchKernelGGL(kern, dim3(g.nb, g.nruns), dim3(64 * W), lds, st, g);
}

// One file a type instantiates it.
template <typename In> int launch_walk(const Walk& g, bool out, hipStream_t st) {
  auto go = [&](auto rb, auto wv) {
    constexpr int RB = decltype(rb)::value, W = decltype(wv)::value;
    if (!out)
      walk<In, RB, W, false, false>(g, st);
    else if (g.learn)
      walk<In, RB, W, true, true>(g, st);
    else
      walk<In, RB, W, true, false>(g, st);
    return launch_status("smat_head_decay_scan");
  };
  auto rows = [&](auto wv) {
    switch (dl::rblocks(g.r)) {
      case 1: return go(std::integral_constant<int, 1>(), wv);
      case 2: return go(std::integral_constant<int, 2>(), wv);
      case 3: return go(std::integral_constant<int, 3>(), wv);
      default: return go(std::integral_constant<int, 4>(), wv);
    }
  };
  return waves_of(g.p) == 4 ? rows(std::integral_constant<int, 4>())
                            : rows(std::integral_constant<int, 8>());
}
extern template int launch_walk<bf16>(const Walk&, bool, hipStream_t);
extern template int launch_walk<f16>(const Walk&, bool, hipStream_t);
extern template int launch_walk<float>(const Walk&, bool, hipStream_t);

}  // namespace hd
}  // namespace smat
