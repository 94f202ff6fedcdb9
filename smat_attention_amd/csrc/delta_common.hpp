// The gated delta rule's chunked form (delta.hip, delta_bwd.hip): sizes, operand
// splits, and the layout of a chunk's operands in the workspace.
//
//   S_t = a_t S_{t-1} + k_t u_t^T,   u_t = b_t (v_t - a_t S_{t-1}^T k_t),
//   o_t = scale S_t^T q_t,           a_t = exp(logA_t).
//
// Over a chunk of C = 64 tokens entered with state S, with L the running sum of
// logA inside it, e_i = exp(L_i), w_i = exp(L_C - L_i) and D_ij = exp(L_i - L_j):
//
//   (I + A) U = b (V - e K S),   A_ij = b_i D_ij k_i.k_j  (j < i)
//   O  = scale e Q S + P U,      P_ij = scale D_ij q_i.k_j  (j <= i)
//   S' = exp(L_C) S + (w K)^T U
//
// T = (I + A)^{-1}, P and the row factors do not depend on S, so one kernel forms
// them for every chunk at once; what remains along the sequence is the chain of
// products through S.
//
// Operands.  Every product runs on v_mfma_f32_16x16x32_bf16.  A value held in
// fewer than its own bits is a sum of bf16 terms: bf16 inputs are one term, fp16
// inputs two (exact: 11 bits), fp32 inputs and everything that is computed in fp32
// on the way three (24 bits), so that states, gradients and outputs have fp32's
// accuracy and 16-bit ones are rounded once, at the end.  A product keeps the terms
// whose orders sum below the larger count.  (fp32 MFMA needs 16 times the cycles of
// one bf16 product, these forms three to six.)
//
// Contraction slots.  A 16x16 result has its column in lane & 15 and rows 4g + i
// (g = lane >> 4) in registers.  Slot (g, j) of a 32-long contraction stands for
// index 4g + j (j < 4) or 16 + 4g + j - 4: then two stacked result tiles are an
// operand of the next product as they lie in registers, and the chain needs no
// exchange between lanes.  T and P are stored as fragments in that order, 16 x 32
// in 1 KB, lane by lane.  Of a lower triangle's six the first and the fifth have
// values in the first half of their slots only; they share a place, 15 KB in three
// terms, so that two workgroups of four waves still fit a CU where the tiles take 8 KB
// a term and two of them are copied ahead.
//
// K and Q are read both by rows (contraction over features) and transposed (over
// tokens).  Both reads come from one LDS tile of 64 rows: 8-byte reads of a row's
// slots, and transposing reads.  The tile's rows hold RS 16-byte chunks, chunk k of
// row t at k ^ swz(t), which keeps both reads free of bank conflicts (64 banks;
// 32 lanes a phase: 16 rows x 16 bytes one way, 8 rows x 32 bytes the other).
// Tiles are copied to LDS by the DMA path straight from the caller's rows where
// those are bf16 in 16-byte groups; otherwise delta_prep_kernel writes them to the
// workspace, a tile a term, padded and swizzled.
#pragma once

#include <type_traits>

#include "smat_host.hpp"

namespace smat {
namespace dl {

constexpr int C = 64;              // tokens a chunk
constexpr int kFrag = 512;         // elements a 16 x 32 fragment
constexpr int kVec = 256;          // floats a chunk: e[64], w[64], b[64], exp(L_C), zeros
constexpr int kZero = 3 * C + 4;   // where 16 bytes of zeros lie in it
constexpr int kLow = 5;            // places of a 64 x 64 lower triangle's fragments
constexpr int kTri = 6;            // and of an upper one's
constexpr int kMaxR = 128, kMaxP = 256;

template <typename In> struct Terms;
template <> struct Terms<bf16> { static constexpr int in = 1; };
template <> struct Terms<f16> { static constexpr int in = 2; };
template <> struct Terms<float> { static constexpr int in = 3; };
constexpr int kMid = 3;            // terms of what is computed in fp32

template <int N> struct Frag { bf16x8 t[N]; };

// Eight fp32 values as N bf16 terms each.  Values that would round to infinity (beyond
// (2 - 2^-8) 2^127) take bf16's largest as their first term, and the others make up the
// rest.  (Two terms are fp16 values', which end at 65504.)
template <int N>
__device__ __forceinline__ Frag<N> split(const f32x4& a, const f32x4& b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  Frag<N> f;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    f32x2 v = q < 2 ? f32x2{a[2 * q], a[2 * q + 1]} : f32x2{b[2 * q - 4], b[2 * q - 3]};
#pragma unroll
    for (int n = 0; n < N; ++n) {
      bf16x2 h;
      if (N == 3 && n == 0) {
        constexpr float most = 0x1.fefffep127f;    // rounds to bf16's largest
        h = __builtin_convertvector((f32x2{__builtin_amdgcn_fmed3f(v[0], -most, most),
                                           __builtin_amdgcn_fmed3f(v[1], -most, most)}),
                                    bf16x2);
      } else {
        h = __builtin_convertvector(v, bf16x2);
      }
      f.t[n][2 * q] = h[0];
      f.t[n][2 * q + 1] = h[1];
      if (n + 1 < N) {
        const unsigned u = __builtin_bit_cast(unsigned, h);
        v[0] -= __uint_as_float(u << 16);
        v[1] -= __uint_as_float(u & 0xffff0000u);
      }
    }
  }
  return f;
}

// c += a b over the terms of order below M, by default max(NA, NB), small ones first.
// Two fp16 inputs want order 2 as well: their second terms are 2^-9 of the first, and
// where fp32 accuracy is due their product counts.
template <int M, int NA, int NB>
__device__ __forceinline__ f32x4 mul_below(f32x4 c, const Frag<NA>& a, const Frag<NB>& b) {
#pragma unroll
  for (int o = M - 1; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (o - i >= 0 && o - i < NB) c = mma(c, a.t[i], b.t[o - i]);
  return c;
}

template <int NA, int NB>
__device__ __forceinline__ f32x4 mul(f32x4 c, const Frag<NA>& a, const Frag<NB>& b) {
  return mul_below<(NA > NB ? NA : NB)>(c, a, b);
}
template <int N>
__device__ __forceinline__ f32x4 mul_inputs(f32x4 c, const Frag<N>& a, const Frag<N>& b) {
  return mul_below<(N == 1 ? 1 : 3)>(c, a, b);
}

// The same for U products at once, term by term across them, so that consecutive
// instructions do not wait for each other's sums.
template <int U, int NA, int NB>
__device__ __forceinline__ void mul_each(f32x4 (&c)[U], const Frag<NA> (&a)[U],
                                         const Frag<NB> (&b)[U]) {
  constexpr int M = NA > NB ? NA : NB;
#pragma unroll
  for (int o = M - 1; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (o - i >= 0 && o - i < NB)
#pragma unroll
        for (int u = 0; u < U; ++u) c[u] = mma(c[u], a[u].t[i], b[u].t[o - i]);
}

// Steps whose operands come from LDS: the next step's reads are issued before a step's
// products, and stay there.
template <int STEPS, typename Buf, typename Load, typename Use>
__device__ __forceinline__ void pipelined(Load load, Use use) {
  Buf buf[2];
  load(0, buf[0]);
#pragma unroll
  for (int st = 0; st < STEPS; ++st) {
    if (st + 1 < STEPS) load(st + 1, buf[(st + 1) & 1]);
    __builtin_amdgcn_sched_barrier(0);
    use(st, buf[st & 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Terms of a stored fragment: term n lies `ts` elements behind term n - 1.
template <int N>
__device__ __forceinline__ Frag<N> load_frag(const bf16* p, int64_t ts, int lane = lane_id()) {
  Frag<N> f;
#pragma unroll
  for (int n = 0; n < N; ++n) f.t[n] = *reinterpret_cast<const bf16x8*>(p + n * ts + lane * 8);
  return f;
}
template <int N>
__device__ __forceinline__ void store_frag(bf16* p, int64_t ts, const Frag<N>& f) {
#pragma unroll
  for (int n = 0; n < N; ++n) *reinterpret_cast<bf16x8*>(p + n * ts + lane_id() * 8) = f.t[n];
}

// Place of a lower triangle's fragment: row tile mt, contraction block kb (kb <= mt / 2).
// (0, 0) has the first half of each lane's eight elements of place 0, (2, 1) the second.
__device__ __forceinline__ constexpr int tri(int mt, int kb) {
  return mt < 2 ? mt : mt == 2 ? (kb == 0 ? 2 : 0) : 3 + kb;
}
__device__ __forceinline__ constexpr bool half_tri(int mt, int kb) { return mt == 2 * kb; }
// and of its transpose's (kb >= mt / 2), each a place of its own.
__device__ __forceinline__ constexpr int tri_t(int mt, int kb) {
  return mt < 2 ? 2 * mt + kb : mt + 2;
}

// 16-byte chunks a tile row, and elements a tile.
constexpr int row_chunks(int RB) { return RB == 1 ? 4 : RB == 2 ? 8 : 16; }
constexpr int tile_elems(int RB) { return C * row_chunks(RB) * 8; }
template <int RS> __device__ __forceinline__ int swz(int t) {
  if (RS == 16) return (((t & 7) << 1) | ((t >> 3) & 1)) ^ (t & 8);
  if (RS == 8) return (t & 6) | ((t >> 3) & 1);
  return ((t >> 1) & 2) | ((t >> 3) & 1);
}

// Row fragment: token 16 mt + (lane & 15), feature slots of block kb.
template <int RB, int N>
__device__ __forceinline__ Frag<N> rows_of(const bf16* tile, int mt, int kb,
                                           int lane = lane_id()) {
  constexpr int RS = row_chunks(RB);
  const int m = lane & 15, g = lane >> 4;
  const int k0 = (4 * kb + (g >> 1)) ^ swz<RS>(m), k1 = (4 * kb + 2 + (g >> 1)) ^ swz<RS>(m);
  int at = (16 * mt + m) * RS * 8 + 4 * (g & 1);
  // odd row tiles take an address the compiler cannot relate to the even ones': fused
  // into ds_read2st64_b64 the pair would be read at half the rate (with two and three
  // terms it still fuses the terms of one tile)
  if (mt & 1) asm("" : "+v"(at));
  const bf16* p = tile + at;
  Frag<N> f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(p + n * tile_elems(RB) + k0 * 8);
    const bf16x4 b = *reinterpret_cast<const bf16x4*>(p + n * tile_elems(RB) + k1 * 8);
    f.t[n] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return f;
}

// Transposed fragment: feature 16 mt + (lane & 15), token slots of block kb.  Lane
// 4 e + q of each sixteen addresses token 16 (2 kb + h) + 4 g + e, features 4 q .. + 3.
template <int RB, int N>
__device__ __forceinline__ Frag<N> cols_of(const bf16* tile, int mt, int kb,
                                           int lane = lane_id()) {
  typedef short short4v __attribute__((ext_vector_type(4)));
  constexpr int RS = row_chunks(RB);
  const int r16 = lane & 15, row = 4 * (lane >> 4) + (r16 >> 2);
  const int k = (2 * mt + ((r16 & 3) >> 1)) ^ swz<RS>(row);
  const bf16* p = tile + ((32 * kb + row) * RS + k) * 8 + 4 * (r16 & 1);
  Frag<N> f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    bf16x4 h[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bf16* a = p + n * tile_elems(RB) + i * 16 * RS * 8;
      h[i] = __builtin_bit_cast(
          bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                      (__attribute__((address_space(3))) short4v*)(uintptr_t)(uint32_t)(uintptr_t)a));
    }
    f.t[n] = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return f;
}

// The first sixteen slots of a fragment.
template <int N> struct Half { bf16x4 t[N]; };
__device__ __forceinline__ bf16x4 low_half(const bf16x8& x) {
  return __builtin_shufflevector(x, x, 0, 1, 2, 3);
}
__device__ __forceinline__ f32x4 mma_half(f32x4 c, const bf16x4& a, const bf16x4& b) {
  typedef short short4v __attribute__((ext_vector_type(4)));
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4v, a),
                                                   __builtin_bit_cast(short4v, b), c, 0, 0, 0);
}

// x += T f for a stored lower triangle, two row tiles at a time; OUT: the result
// transposed, x's columns in registers.
template <int NA> struct Two {
  Frag<NA> a[2];
  Half<NA> h;
};
template <bool OUT, int NA, int NB>
__device__ __forceinline__ void triangle(f32x4 (&x)[4], const bf16* tl, const Frag<NB> (&f)[2],
                                         int lane) {
  // row tiles 0, 1 meet one block, 2, 3 two; the first of a pair's last block is half
  constexpr int TS = kLow * kFrag, M = NA > NB ? NA : NB;
  auto mt_of = [](int st) { return st == 0 ? 0 : 2; };
  auto kb_of = [](int st) { return st == 2 ? 1 : 0; };
  pipelined<3, Two<NA>>(
      [&](int st, Two<NA>& b) {
        const int mt = mt_of(st), kb = kb_of(st);
        b.a[1] = load_frag<NA>(tl + tri(mt + 1, kb) * kFrag, TS, lane);
        if (half_tri(mt, kb)) {
#pragma unroll
          for (int n = 0; n < NA; ++n)
            b.h.t[n] = *reinterpret_cast<const bf16x4*>(tl + n * TS + lane * 8 + 4 * kb);
        } else {
          b.a[0] = load_frag<NA>(tl + tri(mt, kb) * kFrag, TS, lane);
        }
      },
      [&](int st, Two<NA>& b) {
        const int mt = mt_of(st), kb = kb_of(st);
        const Frag<NB>& g = f[kb];
#pragma unroll
        for (int o = M - 1; o >= 0; --o)
#pragma unroll
          for (int i = 0; i < NA; ++i)
            if (o - i >= 0 && o - i < NB) {
              const bf16x8 y = g.t[o - i];
              if (half_tri(mt, kb))
                x[mt] = OUT ? mma_half(x[mt], low_half(y), b.h.t[i])
                            : mma_half(x[mt], b.h.t[i], low_half(y));
              else
                x[mt] = OUT ? mma(x[mt], y, b.a[0].t[i]) : mma(x[mt], b.a[0].t[i], y);
              x[mt + 1] = OUT ? mma(x[mt + 1], y, b.a[1].t[i]) : mma(x[mt + 1], b.a[1].t[i], y);
            }
      });
}
// x += T^T f for a stored upper triangle.
template <int NA, int NB>
__device__ __forceinline__ void triangle_t(f32x4 (&x)[4], const bf16* tl, const Frag<NB> (&f)[2],
                                           int lane) {
  // row tiles 2, 3 meet one block, 0, 1 two
  constexpr int TS = kTri * kFrag;
  auto mt_of = [](int st) { return st == 0 ? 2 : 0; };
  auto kb_of = [](int st) { return st == 1 ? 0 : 1; };
  struct Pair {
    Frag<NA> a[2];
  };
  pipelined<3, Pair>(
      [&](int st, Pair& b) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
          b.a[u] = load_frag<NA>(tl + tri_t(mt_of(st) + u, kb_of(st)) * kFrag, TS, lane);
      },
      [&](int st, Pair& b) {
        const int mt = mt_of(st), kb = kb_of(st);
        f32x4 c[2] = {x[mt], x[mt + 1]};
        const Frag<NB> g[2] = {f[kb], f[kb]};
        mul_each(c, b.a, g);
        x[mt] = c[0];
        x[mt + 1] = c[1];
      });
}

// Row tiles a step takes of K S and of K^T U: as many as leave room for the next step's
// operands.
constexpr int row_step(int terms, int RB) { return terms == 1 ? (RB == 4 ? 2 : 4) : terms == 2 ? 2 : 1; }
constexpr int col_step(int terms) { return terms == 1 ? 2 : 1; }
template <int NT, int U> struct Rows {
  Frag<NT> k[U], q[U];
};
template <int NT, int U, bool Q> struct Cols {
  Frag<NT> k[2][U], q[Q ? 2 : 1][U];
};

// S <- aC S + K^T f (+ Q^T h) by feature tiles, and sb its terms.
template <int RB, int NT, bool Q, int NI>
__device__ __forceinline__ void update_state(f32x4 (&S)[2 * RB], Frag<NI> (&sb)[RB], float aC,
                                             const bf16* kt, const Frag<NI> (&f)[2],
                                             const bf16* qt, const Frag<NI> (&h)[2], int lane) {
  constexpr int U = col_step(NT);
  typedef Cols<NT, U, Q> Buf;
  pipelined<2 * RB / U, Buf>(
      [&](int st, Buf& b) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            b.k[kb][u] = cols_of<RB, NT>(kt, st * U + u, kb, lane);
            if constexpr (Q) b.q[kb][u] = cols_of<RB, NT>(qt, st * U + u, kb, lane);
          }
      },
      [&](int st, Buf& b) {
        f32x4 c[U];
        Frag<NI> g[U];
#pragma unroll
        for (int u = 0; u < U; ++u) c[u] = S[st * U + u] * aC;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
          for (int u = 0; u < U; ++u) g[u] = f[kb];
          mul_each(c, b.k[kb], g);
          if constexpr (Q) {
#pragma unroll
            for (int u = 0; u < U; ++u) g[u] = h[kb];
            mul_each(c, b.q[kb], g);
          }
        }
        // the pair of tiles finished a step ago, while this one's products run
        const int done = st * U - 2;
        if (done >= 0 && done % 2 == 0) sb[done / 2] = split<NI>(S[done], S[done + 1]);
#pragma unroll
        for (int u = 0; u < U; ++u) S[st * U + u] = c[u];
      });
  sb[RB - 1] = split<NI>(S[2 * RB - 2], S[2 * RB - 1]);
}

// Four consecutive features of token t: the terms' sum, exactly the input's values.
template <int RB, int N> __device__ __forceinline__ f32x4 tile_values(const bf16* tile, int t, int f0) {
  constexpr int RS = row_chunks(RB);
  const bf16* p = tile + (t * RS + ((f0 >> 3) ^ swz<RS>(t))) * 8 + (f0 & 4);
  f32x4 x = zero4();
#pragma unroll
  for (int n = N - 1; n >= 0; --n) {
    const bf16x4 v = *reinterpret_cast<const bf16x4*>(p + n * tile_elems(RB));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] += to_f32(v[i]);
  }
  return x;
}

// Where a key sequence's tiles come from.
struct TileSrc {
  const bf16* ws;          // tiles (nbk, nch, terms); or null
  const bf16* raw;         // the caller's rows, strides sb, st
  int64_t sb, st;
};

// A result tile's rows of fp32: p is the wave's row 0 (uniform), off the lane's bytes
// to row 4 gq and its column, rows ld floats apart.
__device__ __forceinline__ void put_rows(float* p, uint32_t off, int ld, const f32x4& x) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<float*>(reinterpret_cast<char*>(p + (int64_t)i * ld) + off) = x[i];
}
__device__ __forceinline__ int uniform_wave() {
  return __builtin_amdgcn_readfirstlane(wave_id());
}

// One copy of 16 bytes a lane into LDS, as lds_dma16<true>, from a uniform address
// and a lane's byte offset: no vector address arithmetic.  Five wait states lie before
// the copy, for a base that a vector instruction has just written (a reload from a
// spill); the last three also serve the write of m0.
__device__ __forceinline__ void dma16(const void* base, uint32_t off, const void* dst) {
  const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)dst);
  uint32_t keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 2\n\t"
      "global_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(off), "s"(base), "s"(m0)
      : "memory");
}

// Copies of 1 KB a wave into LDS, spread over W waves (w is this one, uniform); they
// land by the next wait_vmcnt<0>() and barrier.
template <int KB, int W>
__device__ __forceinline__ void stage(void* dst, const void* src, int w) {
#pragma unroll
  for (int u = 0; u < (KB + W - 1) / W; ++u)
    if (KB % W == 0 || u * W + w < KB)
      dma16((const char*)src + (u * W + w) * 1024, lane_id() * 16, (char*)dst + (u * W + w) * 1024);
}

// The lane, new to the compiler wherever this is called: addresses built from it in a
// loop are formed there instead of being kept in registers across it.
__device__ __forceinline__ int fresh_lane() {
  int l = lane_id();
  asm volatile("" : "+v"(l));
  return l;
}

// A key sequence's tile of chunk c.  Wave w's copies are rows 16 W / .. apart, whole
// turns of the swizzle, so one lane offset serves all of a full chunk's.
template <int RB, int N, int W> struct TileStage {
  static constexpr int RS = row_chunks(RB), RPU = 64 / RS;      // rows a copy
  static_assert((RPU * W) % 16 == 0, "");
  uint32_t off;
  bool fast;               // full rows, and offsets within 32 bits

  __device__ __forceinline__ TileStage(const TileSrc& src, int r, int w) {
    const int t = w * RPU + lane_id() / RS, k = (lane_id() % RS) ^ swz<RS>(t);
    fast = N == 1 && r == 8 * RS && src.st >= 0 && src.st < (1 << 24);
    off = fast ? (uint32_t)((t * src.st + 8 * k) * 2) : 0;
  }
  __device__ __forceinline__ void operator()(bf16* dst, const TileSrc& src, int64_t ks,
                                             int64_t nch, int c, int t0, int len, int r,
                                             const float* vec, int w) const {
    if (N > 1 || src.ws) {
      stage<N * RS, W>(dst, src.ws + (ks * nch + c) * (int64_t)N * tile_elems(RB), w);
      return;
    }
    const bf16* base = src.raw + ks * src.sb + (int64_t)t0 * src.st;
    if (fast && len == C) {
#pragma unroll
      for (int u = 0; u < (RS + W - 1) / W; ++u)
        if (RS % W == 0 || u * W + w < RS)
          dma16(base + (int64_t)(u * W * RPU) * src.st, off, dst + (u * W + w) * 512);
      return;
    }
    for (int u = w; u < RS; u += W) {
      const int l = u * 64 + lane_id(), t = l / RS, k = (l % RS) ^ swz<RS>(t);
      const void* p = t < len && 8 * k < r ? (const void*)(base + (int64_t)t * src.st + 8 * k)
                                           : (const void*)(vec + kZero);
      lds_dma16<true>(p, dst + u * 512);
    }
  }
};

// A chunk's 64 values of a column in result-tile order: element j is token
// 16 (j >> 2) + 4 gq + (j & 3), loaded a chunk ahead of their use.  The bits are kept a
// register each: packed in pairs, they would be waited for where they are loaded.
template <typename In> __device__ __forceinline__ uint32_t bits_of(const In* p) {
  if constexpr (sizeof(In) == 4)
    return *reinterpret_cast<const uint32_t*>(p);
  else
    return *reinterpret_cast<const uint16_t*>(p);
}
template <typename In> __device__ __forceinline__ float value_of(uint32_t b) {
  if constexpr (__is_same(In, float))
    return __uint_as_float(b);
  else if constexpr (__is_same(In, bf16))
    return __uint_as_float(b << 16);
  else
    return to_f32(__builtin_bit_cast(f16, (uint16_t)b));
}
// Without a branch: at a join the compiler waits for the loads of either side.  Absent
// tokens and columns (col past the last) read the last one there is; column_values drops
// them.  Rows lie less than 2^23 elements apart, so a chunk's offsets have 32 bits.
template <typename In>
__device__ __forceinline__ void load_column(uint32_t* v, const In* rows, int64_t st, int64_t t0,
                                            int len, int col, int cols) {
  const char* p = reinterpret_cast<const char*>(rows + t0 * st);
  const uint32_t step = (uint32_t)st * sizeof(In), c0 = min(col, cols - 1) * sizeof(In);
  const uint32_t first = 4 * (lane_id() >> 4) * step + c0, last = (len - 1) * step + c0;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    v[j] = bits_of(reinterpret_cast<const In*>(
        p + min(first + (16 * (j >> 2) + (j & 3)) * step, last)));
}
template <typename In>
__device__ __forceinline__ void column_values(f32x4* x, const uint32_t* v, bool live, int len) {
  if (len == C) {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j >> 2][j & 3] = live ? value_of<In>(v[j]) : 0.f;
  } else {
    const int g4 = 4 * (lane_id() >> 4);
#pragma unroll
    for (int j = 0; j < 16; ++j)
      x[j >> 2][j & 3] =
          live && 16 * (j >> 2) + (j & 3) + g4 < len ? value_of<In>(v[j]) : 0.f;
  }
}
inline bool near_rows(int64_t st) { return st >= 0 && st < (1 << 23); }

// x of this lane and of lane ^ D, summed in registers (a shuffle through LDS takes ten
// times as long, and a token is a chain of them).
template <int D> __device__ __forceinline__ float sum_across(float x) {
  static_assert(D == 8 || D == 16 || D == 32, "");
  if constexpr (D == 8) {                          // a rotation within 16 lanes
    return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x128, 0xf, 0xf,
                                                           false));
  } else {
    const uint32_t b = __float_as_uint(x);
    const auto r = D == 16 ? __builtin_amdgcn_permlane16_swap(b, b, false, false)
                           : __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
}
template <int CL> __device__ __forceinline__ float sum_rows(float x) {
  if constexpr (CL <= 8) x = sum_across<8>(x);
  if constexpr (CL <= 16) x = sum_across<16>(x);
  return sum_across<32>(x);
}

// Four consecutive elements; those at and past nv are zero.
template <typename In>
__device__ __forceinline__ f32x4 load4(const In* p, int nv, bool vec) {
  f32x4 x = zero4();
  if (vec && nv >= 4) {
    typedef In In4 __attribute__((ext_vector_type(4)));
    const In4 v = *reinterpret_cast<const In4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f32(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < nv) x[i] = to_f32(p[i]);
  }
  return x;
}
template <typename In>
__device__ __forceinline__ void store4(In* p, const f32x4& x, int nv, bool vec) {
  if (vec && nv >= 4) {
    typedef In In4 __attribute__((ext_vector_type(4)));
    In4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = from_f32<In>(x[i]);
    *reinterpret_cast<In4*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < nv) p[i] = from_f32<In>(x[i]);
  }
}

// Whether groups of four elements of rows at p may be read at once.
inline bool vec4_ok(const void* p, int64_t sb, int64_t st, int eb) {
  return (reinterpret_cast<uintptr_t>(p) % (4 * eb)) == 0 && sb % 4 == 0 && st % 4 == 0;
}

// One call's geometry.  Chunks and runs (consecutive chunks of one segment that one
// wave walks) come from tables when the sequences are segmented, else from
// arithmetic: chunk c is tokens [64 c, 64 c + 64), run g chunks [g K, g K + K).
struct Geo {
  const int32_t* chunks;   // (nch, 2): first token, tokens; or null
  const int32_t* runs;     // (nruns, 4): first chunk, end chunk, segment, turn; or null
  const int32_t* segrun;   // (nseg + 1): first run of each segment; or null
  int nb, nbk, T, nseg, nch, nruns, K, r, p;
  float scale;
  int64_t q_sb, q_st, k_sb, k_st, v_sb, v_st, a_sb, a_st, b_sb, b_st;
};
__device__ __forceinline__ void chunk_of(const Geo& g, int c, int& t0, int& len) {
  if (g.chunks) {
    t0 = g.chunks[2 * c];
    len = g.chunks[2 * c + 1];
  } else {
    t0 = c * C;
    len = min(C, g.T - t0);
  }
}
__device__ __forceinline__ void run_of(const Geo& g, int turn, int& i, int& c0, int& c1, int& seg,
                                       bool& first, bool& last) {
  i = turn;
  if (g.runs) {
    i = g.runs[4 * turn + 3];
    c0 = g.runs[4 * i];
    c1 = g.runs[4 * i + 1];
    seg = g.runs[4 * i + 2];
    first = g.segrun[seg] == i;
    last = g.segrun[seg + 1] == i + 1;
  } else {
    c0 = i * g.K;
    c1 = min(c0 + g.K, g.nch);
    seg = 0;
    first = i == 0;
    last = i + 1 == g.nruns;
  }
}

// The chunks' operands.
struct Ops {
  TileSrc k, q;
  bf16 *kw, *qw;            // the tiles' place in the workspace; or null
  bf16 *tm, *pm;            // T and P by rows
  bf16 *tt, *pt;            // transposed
  float* vec;
};

__device__ __forceinline__ int64_t key_of(const Geo& g, int s) { return s / (g.nb / g.nbk); }

// Hands out 256-byte aligned pieces of a workspace; with no base it only counts.
struct Arena {
  char* base;
  int64_t used = 0;
  template <typename T> T* take(int64_t n) {
    T* p = reinterpret_cast<T*>(base + used);
    used += (n * (int64_t)sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

constexpr int kMaxLds = 160 * 1024;

inline int rblocks(int r) { return (r + 31) / 32; }
inline int p32(int p) { return (p + 31) / 32 * 32; }
inline int in_terms(int dtype) { return dtype == SMAT_BF16 ? 1 : dtype == SMAT_F16 ? 2 : 3; }

// Whether rows can be copied as they are: bf16 in aligned groups of eight.
inline bool raw_ok(int dtype, const void* p, int64_t sb, int64_t st, int r) {
  return dtype == SMAT_BF16 && r % 8 == 0 && rows_vec8_ok(p, sb, st);
}

// raw: no tiles in the workspace.
inline Ops take_ops(Arena& ar, int dtype, int64_t nb, int64_t nbk, int64_t nch, int r, bool bwd,
                    bool raw) {
  const int64_t tiles = nbk * nch * in_terms(dtype) * tile_elems(rblocks(r));
  const int64_t tris = nb * nch * (bwd ? kTri : kLow) * kFrag * kMid;
  Ops o = {};
  if (!raw) {
    o.kw = ar.take<bf16>(tiles);
    o.qw = ar.take<bf16>(tiles);
    o.k.ws = o.kw;
    o.q.ws = o.qw;
  }
  (bwd ? o.tt : o.tm) = ar.take<bf16>(tris);
  (bwd ? o.pt : o.pm) = ar.take<bf16>(tris);
  o.vec = ar.take<float>(nb * nch * kVec);
  return o;
}

inline Ops place_ops(Arena& ar, int dtype, const Geo& g, const void* q, const void* k, bool bwd) {
  const bool raw = raw_ok(dtype, q, g.q_sb, g.q_st, g.r) && raw_ok(dtype, k, g.k_sb, g.k_st, g.r);
  Ops o = take_ops(ar, dtype, g.nb, g.nbk, g.nch, g.r, bwd, raw);
  o.k.raw = (const bf16*)k;
  o.k.sb = g.k_sb;
  o.k.st = g.k_st;
  o.q.raw = (const bf16*)q;
  o.q.sb = g.q_sb;
  o.q.st = g.q_st;
  return o;
}

// What the runs' states take: E, the states entering runs, and M as the carry's operand,
// split into terms where it is formed (in the carry every step would wait for that).  The
// gradient's M is the forward's, kept transposed: `own` = false.
struct Carry {
  float *E, *start;
  const bf16* M;
  bf16* trans;
};
// Fragment (row tile rt, contraction block kb) of the M at index sn.
template <int RB> __device__ __forceinline__ int64_t trans_at(int64_t sn, int rt, int kb) {
  return ((sn * 2 * RB + rt) * RB + kb) * kMid * kFrag;
}
inline Carry take_carry(Arena& ar, int64_t nb, int64_t nruns, int r, int p, bool own) {
  const int64_t R = 32 * rblocks(r);
  Carry c = {};
  c.E = ar.take<float>(nruns * nb * r * p);
  c.start = ar.take<float>(nruns * nb * r * p);
  if (own) c.M = c.trans = ar.take<bf16>(nruns * nb * R * R * kMid);
  return c;
}

// fn(In(), integral_constant of the 32-row blocks of r).
template <typename F>
inline int dispatch(int dtype, int r, F fn) {
  auto rows = [&](auto in) {
    switch (rblocks(r)) {
      case 1: return fn(in, std::integral_constant<int, 1>());
      case 2: return fn(in, std::integral_constant<int, 2>());
      case 3: return fn(in, std::integral_constant<int, 3>());
      default: return fn(in, std::integral_constant<int, 4>());
    }
  };
  if (dtype == SMAT_BF16) return rows(bf16());
  if (dtype == SMAT_F16) return rows(f16());
  return rows(float());
}

// The checks that the forward and the backward share, and those of the chunks' kernels.
int check_geo(const char* who, int dtype, const Geo& g);
constexpr int kMaxGrid = 65535;
int check_grid(const char* who, const Geo& g);
// Up to this many tokens a sequence are taken one after another (delta_step.hip; callers,
// who give such calls no workspace, hold the same number).
constexpr int kFewTokens = 16;
int launch_tokens(const char* who, int dtype, const Geo& g, const void* q, const void* k, const void* v,
                  const float* logA, const float* beta, const float* S_in, float* S_out, void* o,
                  hipStream_t st);
using smat::allow_lds;

// Launches the runs' carry (both directions).
int launch_carry(const Geo& g, const float* init, const Carry& c, bool rev, hipStream_t st);

}  // namespace dl
}  // namespace smat
