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
// The columns of the state do not mix, so a wave takes 16 or 32 of them with all key rows in
// registers (fp32).  A workgroup has all columns of a sequence: its four or eight waves share
// the chunk's rows in LDS and one P = (Q K^T) o D, of which each forms a few tiles.
//
// Operands: every product runs on v_mfma_f32_16x16x32_bf16, values held in fewer than
// their own bits as sums of bf16 terms (delta_common.hpp): bf16 inputs one term, fp16 two,
// fp32 and what is computed in fp32, the state and P, three, 24 bits, whatever the output's
// type: with two, outputs that are small differences of large sums are off by many of their own
// steps.  Results are rounded once, where they are stored.
//
// Per chunk, bf16, r = p = 128: 240 MFMA and some 870 vector instructions a wave (the splits
// most of them), two waves a SIMD; 8 sequences of 131072 take 313 us with outputs (3.4 TB/s;
// every row in L2 takes a fifth less) and 125 in the first pass (4.3); 32 of 8192, 64 x 64, 40
// and 20.  So it is bound by how well two or three waves a SIMD cover a chunk's chain of LDS
// reads, products, splits and barriers, and next by HBM.  fp16 has twice the tiles and products
// and one workgroup of eight waves a CU: 12 of 10007, 96 x 96, 86 and 29.  Widths between the
// blocks (96 of 128) run the larger block's products, and every chunk takes the path with bounds.
// Kernels that spill (registers a lane; none in 16 bits without learned decays): the walk for q
// with learned decays, bf16 96 x 64: 4, fp16 64 x 64, 96 and 128 x 128: 10, fp32 up to 32; those
// for k and v in fp16 at 128: 10 and 2, in fp32 at 128 columns up to 12 and 20; fp32's outputs
// without, 96 and 128 x 128: 4 and 10.
// Tried and slower or no faster: volatile LDS reads, products and splits interleaved by hand,
// two column tiles a wave with LEARN (spills), splits in registers ahead of fp16's products.
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
  float* part;             // LEARN: (nruns, nb, W)
};
// Up to three walks of the same sequences in one launch (their widths in the same blocks).
struct Walks {
  Walk w[3];
  int n;
};

// fp32 values as three bf16 terms, exactly: each term takes the next eight bits, so none is
// rounded up past the type's end.
__device__ __forceinline__ Frag<kMid> cut(const f32x4& a, const f32x4& b) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  u4 t[kMid];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float x = q < 2 ? a[2 * q] : b[2 * q - 4], y = q < 2 ? a[2 * q + 1] : b[2 * q - 3];
#pragma unroll
    for (int n = 0; n < kMid; ++n) {
      const uint32_t u = __float_as_uint(x), v = __float_as_uint(y);
      t[n][q] = __builtin_amdgcn_perm(v, u, 0x07060302);     // the upper halves
      if (n + 1 < kMid) {
        x -= __uint_as_float(u & 0xffff0000u);
        y -= __uint_as_float(v & 0xffff0000u);
      }
    }
  }
  Frag<kMid> f;
#pragma unroll
  for (int n = 0; n < kMid; ++n) f.t[n] = __builtin_bit_cast(bf16x8, t[n]);
  return f;
}
// For products with one-term operands, which keep every term; others drop products of low
// terms, and rounded terms are half as large and of either sign.
template <int NT> __device__ __forceinline__ Frag<kMid> terms(const f32x4& a, const f32x4& b) {
  if constexpr (NT == 1)
    return cut(a, b);
  else
    return dl::split<kMid>(a, b);
}

// A chunk's rows in LDS, 32 B columns of 16 bits: row t at t (64 B + 32) bytes, and 16 more in
// every second eight rows.  That keeps both reads free of bank conflicts (64 banks, 32 lanes
// a phase): rows of 16 bytes from 16 rows, and transposing ones of 32 bytes from 8 rows; and
// every address is one a lane and constants.
constexpr int pitch(int B) { return 32 * B + 16; }
constexpr int tile_elems(int B) { return C * pitch(B); }
__device__ __forceinline__ int row_at(int B, int t) { return t * pitch(B) + ((t >> 3) & 1) * 8; }

// Rows fragment: token 16 mt + (lane & 15), the column slots of block kb (delta_common.hpp).
template <int B, int N, typename T = bf16>
__device__ __forceinline__ Frag<N> rows_of(const T* tile, int mt, int kb) {
  const int m = lane_id() & 15, g = lane_id() >> 4;
  const T* p = tile + row_at(B, m) + 4 * g + 16 * mt * pitch(B) + 32 * kb;
  Frag<N> f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(p + n * tile_elems(B));
    const bf16x4 b = *reinterpret_cast<const bf16x4*>(p + n * tile_elems(B) + 16);
    f.t[n] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return f;
}

// Transposed fragment: column 16 mt + (lane & 15), the token slots of block kb.  Lane 4 e + q
// of each sixteen addresses token 4 (lane >> 4) + e, columns 4 q .. + 3.
template <int B, int N>
__device__ __forceinline__ Frag<N> cols_of(const bf16* tile, int mt, int kb) {
  typedef short short4v __attribute__((ext_vector_type(4)));
  const int r16 = lane_id() & 15, t = 4 * (lane_id() >> 4) + (r16 >> 2);
  const bf16* p = tile + row_at(B, t) + 4 * (r16 & 3) + 16 * mt + 32 * kb * pitch(B);
  Frag<N> f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    bf16x4 h[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      h[i] = __builtin_bit_cast(
          bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                      (__attribute__((address_space(3))) short4v*)(uintptr_t)(uint32_t)(uintptr_t)(
                          p + n * tile_elems(B) + i * 16 * pitch(B))));
    f.t[n] = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return f;
}

// A value that is new to the compiler here: what only a rare path needs of it is formed there,
// and not kept in registers across the walk.
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// One operand's rows of a chunk on their way to LDS: loaded a chunk ahead into registers,
// then written as a tile a term, or (V) as they are.  B: 32-column blocks.  A thread has the
// same eight columns of every STEP-th row.
template <typename In, int B, int W, bool RAW> struct Rows {
  static constexpr int MIN = B == 1 ? 4 : B == 2 ? 8 : 16, LC = MIN < W ? W : MIN;
  static constexpr int STEP = 64 * W / LC, U = C / STEP;
  static_assert(STEP % 16 == 0 && U * STEP == C, "");
  Raw<In> x[U];

  __device__ __forceinline__ static int row(int tid = threadIdx.x) { return tid / LC; }
  __device__ __forceinline__ static int group(int tid = threadIdx.x) { return tid % LC; }
  // The lane's offset in bytes from a chunk's first row, sb bytes to the next one; turned order
  // counts from the last of 64.  Columns past the end are read earlier in the row (cols >= 8).
  __device__ __forceinline__ static uint32_t offset(uint32_t sb, int cols, bool rev) {
    const int t = rev ? STEP - 1 - row() : row();
    return t * sb + min(8 * group(), cols - 8) * (int)sizeof(In);
  }
  __device__ __forceinline__ void load(const char* base, uint32_t off, uint32_t sb, bool rev) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      x[u].load(reinterpret_cast<const In*>(base + (int64_t)((rev ? U - 1 - u : u) * STEP) * sb +
                                            off));
  }
  // Of len < 64 rows: those past the last are the last one's, so every address lies in the
  // operand.
  __device__ __forceinline__ void load_part(const char* base, uint32_t sb, int len, int cols,
                                            bool rev) {
    const int tid = fresh((int)threadIdx.x);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = min(u * STEP + row(tid), len - 1);
      x[u].load(reinterpret_cast<const In*>(base + (int64_t)(rev ? len - 1 - t : t) * sb) +
                min(8 * group(tid), cols - 8));
    }
  }
  __device__ __forceinline__ void put(bf16* tile) {
#pragma unroll
    for (int u = 0; u < U; ++u) put_one(u, tile, threadIdx.x);
  }
  __device__ __forceinline__ void put_part(bf16* tile, int len, int cols) {
    const int tid = fresh((int)threadIdx.x), k = group(tid), over = cols & 7;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (over && 8 * k + 8 > cols && 8 * k < cols) x[u].drop(8 - over);
      if (u * STEP + row(tid) >= len || 8 * k >= cols) x[u].zero();
      put_one(u, tile, tid);
    }
  }
  __device__ __forceinline__ void put_one(int u, bf16* tile, int tid) {
    const int t = row(tid), k = group(tid);
    if (LC > 4 * B && k >= 4 * B) return;
    typedef typename Raw<In>::u4 u4;
    if constexpr (RAW && sizeof(In) == 4) {
      float* at = reinterpret_cast<float*>(tile) + (u * STEP + t) * (32 * B + 4) + 8 * k;
      reinterpret_cast<u4*>(at)[0] = x[u].x[0];
      reinterpret_cast<u4*>(at)[1] = x[u].x[1];
    } else {
      bf16* at = tile + row_at(B, t) + 8 * k + u * STEP * pitch(B);
      if constexpr (RAW || __is_same(In, bf16)) {
        *reinterpret_cast<u4*>(at) = x[u].x[0];
      } else {
        f32x4 a, b;
        x[u].values(a, b);
        const Frag<Terms<In>::in> f = dl::split<Terms<In>::in>(a, b);
#pragma unroll
        for (int n = 0; n < Terms<In>::in; ++n)
          *reinterpret_cast<bf16x8*>(at + n * tile_elems(B)) = f.t[n];
      }
    }
  }
};

// V's tile holds values as they come (fp32: rows of 32 B + 4 floats).  A lane's eight values of
// a column, the token slots of block kb, and of a row (token 16 mt + lane & 15).
template <typename In, int B>
__device__ __forceinline__ void value_cols(const bf16* tile, int ct, int kb, f32x4& a, f32x4& b) {
  if constexpr (sizeof(In) == 4) {
    const float* p = reinterpret_cast<const float*>(tile) +
                     (32 * kb + 4 * (lane_id() >> 4)) * (32 * B + 4) + 16 * ct + (lane_id() & 15);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = p[i * (32 * B + 4)];
      b[i] = p[(16 + i) * (32 * B + 4)];
    }
  } else {
    Raw<In> x;
    x.x[0] = __builtin_bit_cast(typename Raw<In>::u4, cols_of<B, 1>(tile, ct, kb).t[0]);
    x.values(a, b);
  }
}
template <typename In, int B>
__device__ __forceinline__ Frag<Terms<In>::in> value_rows(const bf16* tile, int mt, int kb) {
  if constexpr (__is_same(In, bf16)) {
    return rows_of<B, 1>(tile, mt, kb);
  } else {
    f32x4 a, b;
    if constexpr (sizeof(In) == 4) {
      const float* p = reinterpret_cast<const float*>(tile) +
                       (16 * mt + (lane_id() & 15)) * (32 * B + 4) + 32 * kb + 4 * (lane_id() >> 4);
      a = *reinterpret_cast<const f32x4*>(p);
      b = *reinterpret_cast<const f32x4*>(p + 16);
    } else {
      Raw<In> x;
      x.x[0] = __builtin_bit_cast(typename Raw<In>::u4, rows_of<B, 1>(tile, mt, kb).t[0]);
      x.values(a, b);
    }
    return dl::split<Terms<In>::in>(a, b);
  }
}

// The column tiles of a wave and the waves of a workgroup, by the columns of all (64 or 128):
// two tiles a wave share the reads of K, Q and P (8 sequences of 131072, 128 x 128: with one tile
// 352 us where two took 297).  With LEARN they would not fit the registers,
// inputs of several terms leave LDS for one workgroup a CU, which eight waves fill better, and the
// first pass reads K alone: four waves a SIMD there (125 us, two of two tiles 152).
template <typename In, int P, bool OUT, int LEARN> constexpr int tiles() {
  return P == 64 || !OUT || LEARN || Terms<In>::in > 1 ? 1 : 2;
}
template <typename In, int P, bool OUT, int LEARN> constexpr int waves() {
  return P / 16 / tiles<In, P, OUT, LEARN>();
}
constexpr int kMaxWaves = 8;
template <typename In, int P> constexpr int value_elems() {
  return sizeof(In) == 4 ? 2 * C * (P + 4) : tile_elems(P / 32);
}
template <typename In, int RB, int P, bool OUT> constexpr int set_elems() {
  return Terms<In>::in * (OUT ? 2 : 1) * tile_elems(RB) + value_elems<In, P>();
}
// Floats: a^0 .. a^64; the update's factors, zeros behind; and, where inputs of one term leave
// room and four registers a tile are dear, D by the tiles' distances, lane by lane.
template <typename In> constexpr int tab_floats() {
  return C + 4 + 2 * C + (Terms<In>::in == 1 ? 4 * 256 : 0);
}
template <typename In, int RB, int P, bool OUT> constexpr int walk_lds(int sets) {
  return sets * set_elems<In, RB, P, OUT>() * 2 + (OUT ? kMid * kLow * kFrag * 2 : 0) +
         tab_floats<In>() * 4;
}
// Waves a SIMD: as many as registers and LDS have room for.
template <typename In, int RB, int P, bool OUT, int LEARN> constexpr int walk_occ() {
  const int fit = dl::kMaxLds / walk_lds<In, RB, P, OUT>(1) * waves<In, P, OUT, LEARN>() / 4;
  const bool few = P == 128 && RB * Terms<In>::in > (Terms<In>::in == 3 ? 3 : 6);
  const int most = LEARN ? 2 : !OUT ? (few ? 2 : 4) : P == 64 && RB < 3 ? 3 : 2;
  return fit < most ? fit : most;
}
// Two sets, so that the next chunk's rows are written beside this one's use, where that many
// still fit.
template <typename In, int RB, int P, bool OUT, int LEARN> constexpr int walk_sets() {
  return walk_lds<In, RB, P, OUT>(2) * walk_occ<In, RB, P, OUT, LEARN>() * 4 /
                     waves<In, P, OUT, LEARN>() <= dl::kMaxLds ? 2 : 1;
}

// Four consecutive values of a row as they come, at the element's own alignment: of columns
// col .. col + 3 of `cols` (a multiple of four; those past the last read as zero).
template <typename In> struct Quad {
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  typedef uint32_t u2h __attribute__((ext_vector_type(2), aligned(2)));
  typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
  typename std::conditional<sizeof(In) == 2, u2, f32x4>::type x;
  __device__ __forceinline__ void load(const In* row, int col, int cols) {
    const In* p = row + min(col, cols - 4);
    if constexpr (sizeof(In) == 2)
      x = *reinterpret_cast<const u2h*>(p);
    else
      x = *reinterpret_cast<const f32x4u*>(p);
  }
  __device__ __forceinline__ f32x4 get(bool live) const {
    f32x4 y;
    if constexpr (__is_same(In, bf16)) {
      y = f32x4{__uint_as_float(x[0] << 16), __uint_as_float(x[0] & 0xffff0000u),
                __uint_as_float(x[1] << 16), __uint_as_float(x[1] & 0xffff0000u)};
    } else if constexpr (__is_same(In, f16)) {
      const f16x4 h = __builtin_bit_cast(f16x4, x);
      y = f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
    } else {
      y = x;
    }
    return live ? y : zero4();
  }
};
// The same one by one, for any number of columns.
template <typename In>
__device__ __forceinline__ f32x4 four_of(const In* row, int col, int cols, bool live) {
  f32x4 y;
  col = fresh(col);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = to_f32(row[min(col + i, cols - 1)]);
    y[i] = live && col + i < cols ? x : 0.f;
  }
  return y;
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

// Steps whose operands come from LDS: AHEAD issues the next step's reads before a step's
// products, and keeps them there; else they come as the compiler likes (several terms: registers).
template <int STEPS, bool AHEAD, typename Buf, typename Load, typename Use>
__device__ __forceinline__ void steps(Load load, Use use) {
  if constexpr (AHEAD) {
    dl::pipelined<STEPS, Buf>(load, use);
  } else {
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      Buf b;
      load(st, b);
      use(st, b);
    }
  }
}

template <typename In, int RB, int P, bool OUT, int LEARN>
__global__
__launch_bounds__((64 * waves<In, P, OUT, LEARN>()), (walk_occ<In, RB, P, OUT, LEARN>())) void
decay_walk_kernel(Walks all) {
  // with several, workgroups of one sequence and run lie eight apart: on one XCD, whose L2 they
  // share the rows in
  const int role = all.n == 1 ? 0 : (int)blockIdx.x / 8 % 3;
  const int s = all.n == 1 ? (int)blockIdx.x : (int)blockIdx.x / 24 * 8 + (int)blockIdx.x % 8;
  const Walk& g = all.w[role];
  if (s >= g.nb) return;
  constexpr int W = waves<In, P, OUT, LEARN>(), CT = tiles<In, P, OUT, LEARN>(), VB = P / 32;
  constexpr int NT = Terms<In>::in, NI = kMid;
  constexpr int KT = NT * tile_elems(RB), VT = value_elems<In, P>();
  constexpr int SET = set_elems<In, RB, P, OUT>();
  constexpr int KD = walk_sets<In, RB, P, OUT, LEARN>(), TP = (kTiles + W - 1) / W;
  constexpr bool AHEAD = NT == 1;                  // (two terms: as fast without)
  extern __shared__ __align__(1024) bf16 lds[];
  bf16* pl = lds + KD * SET;
  float* tab = reinterpret_cast<float*>(pl + (OUT ? NI * kLow * kFrag : 0));   // a^0 .. a^64
  float* wt = tab + C + 4;                         // wt[64 - n + j] = w_j of a chunk of n
  const int w = dl::uniform_wave();
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
  const int chunks = c1 - c0, tile0 = w * CT;      // the wave's first column tile
  const int64_t sn = (int64_t)run * g.nb + s, rp = (int64_t)g.r * g.p;
  // a run's chunks lie one behind the other, all but its last whole
  int begin = 0, end = 0;
  if (chunks > 0) {
    begin = g.chunks ? g.chunks[2 * c0] : c0 * C;
    end = g.chunks ? g.chunks[2 * c1 - 2] + g.chunks[2 * c1 - 1] : min(c1 * C, g.T);
  }
  Rows<In, RB, W, false> rq, rk;
  Rows<In, VB, W, true> rv;
  constexpr uint32_t EB = sizeof(In);
  const uint32_t qb = (uint32_t)g.q.st * EB, kb_ = (uint32_t)g.k.st * EB,
                 vb_ = (uint32_t)g.v.st * EB;
  auto rows_at = [&](const Side& x, int t) {
    return (const char*)x.p + (s / x.div * x.sb + (int64_t)t * x.st) * EB;
  };
  const char *qp = rows_at(g.q, begin), *kp = rows_at(g.k, begin), *vp = rows_at(g.v, begin);
  const uint32_t qo = rq.offset(qb, g.r, g.rev), ko = rk.offset(kb_, g.r, g.rev),
                 vo = rv.offset(vb_, g.p, g.rev);
  // chunk i of the walk: its first token from the run's, its tokens
  auto first_of = [&](int i) { return (g.rev ? chunks - 1 - i : i) * C; };
  auto load = [&](int i) {
    const int64_t t = first_of(i);
    const int len = min(C, end - begin - (int)t);
    if (len == C) {
      if (OUT) rq.load(qp + t * qb, qo, qb, g.rev);
      rk.load(kp + t * kb_, ko, kb_, g.rev);
      rv.load(vp + t * vb_, vo, vb_, g.rev);
    } else {
      if (OUT) rq.load_part(qp + t * qb, qb, len, g.r, g.rev);
      rk.load_part(kp + t * kb_, kb_, len, g.r, g.rev);
      rv.load_part(vp + t * vb_, vb_, len, g.p, g.rev);
    }
  };
  const bool full = g.r == 32 * RB && g.p == 32 * VB;
  auto put = [&](int i) {
    bf16* set = lds + (KD == 2 ? (i & 1) * SET : 0);
    const int len = min(C, end - begin - first_of(i));
    if (full && len == C) {
      rk.put(set);
      rv.put(set + KT);
      if (OUT) rq.put(set + KT + VT);
    } else {
      rk.put_part(set, len, g.r);
      rv.put_part(set + KT, len, g.p);
      if (OUT) rq.put_part(set + KT + VT, len, g.r);
    }
  };
  if (chunks > 0) load(0);
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
  // element i of S[ct][mt]: row 16 mt + 4 gq + i of column 16 (tile0 + ct) + m
  f32x4 S[CT][2 * RB];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int mt = 0; mt < 2 * RB; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int a = 16 * mt + 4 * gq + i, col = 16 * (tile0 + ct) + m;
        S[ct][mt][i] = g.start && a < g.r && col < g.p
                           ? g.start[sn * rp + (int64_t)a * g.s_row + (int64_t)col * g.s_col]
                           : 0.f;
      }
  if (chunks > 0) put(0);
  lds_barrier();
  float e[4];
  f32x4* dt = reinterpret_cast<f32x4*>(wt + 2 * C);
  f32x4 D[OUT && NT > 1 ? TP : 1];
  if (OUT) {
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) e[mt] = g.inter * tab[16 * mt + m + (g.rev ? 0 : 1)];
    auto factors = [&](int q) {                    // of tiles 16 q tokens apart
      f32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 16 * q + m - 4 * gq - i;
        x[i] = d >= 0 ? g.intra * tab[d] : 0.f;
      }
      return x;
    };
    if constexpr (NT == 1) {
      for (int q = w; q < 4; q += W) dt[q * 64 + lane_id()] = factors(q);
      lds_barrier();
    } else {
#pragma unroll
      for (int u = 0; u < TP; ++u) {
        int mt, jt;
        tile_of(min(w + u * W, kTiles - 1), mt, jt);
        D[u] = factors(mt - jt);
      }
    }
  }
  float acc = 0.f;                                 // LEARN: this lane's part of the gradient
  const In* xs = LEARN ? (const In*)g.x.p + s / g.x.div * g.x.sb : nullptr;
  const int64_t x_st = g.rev ? -g.x.st : g.x.st;
  const bool quads = g.p % 4 == 0;

  for (int c = 0; c < chunks; ++c) {
    bf16* set = lds + (KD == 2 ? (c & 1) * SET : 0);
    const bf16 *kt = set, *vt = set + KT, *qt = vt + VT;
    const bool more = c + 1 < chunks;
    __builtin_amdgcn_s_setprio(0);
    const int t0 = begin + first_of(c), len = min(C, end - t0);
    if (c > 0) lds_barrier();
    // ---- the chunk's rows are in LDS
    if (more) load(c + 1);
    const float aC = tab[len];
    const In* xrow = LEARN ? xs + (int64_t)(g.rev ? t0 + len - 1 : t0) * g.x.st : nullptr;
    // LEARN: what meets the products below from memory, read here, well before
    constexpr bool EARLY = LEARN && sizeof(In) == 2;
    Quad<In> xq[LEARN && LEARN != kDv ? 4 : 1], xz[EARLY && LEARN == kDq ? TP * VB * 2 : 1];
    f32x4 xS[LEARN == kDv ? 2 * RB : 1];
    auto row_of = [&](int mt) { return xrow + min(16 * mt + m, len - 1) * x_st; };
    if constexpr (LEARN) {
      static_assert(CT == 1, "");
      if constexpr (LEARN == kDv) {
        const f32x4* from = reinterpret_cast<const f32x4*>(g.load_s) +
                            (((int64_t)s * g.nch + c1 - 1 - c) * W + w) * (2 * RB * 64) + lane_id();
#pragma unroll
        for (int mt = 0; mt < 2 * RB; ++mt) xS[mt] = from[mt * 64];
      } else if (quads) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) xq[mt].load(row_of(mt), 16 * tile0 + 4 * gq, g.p);
        if constexpr (EARLY && LEARN == kDq) {
#pragma unroll
          for (int i = 0; i < TP * VB * 2; ++i) {
            int mt, jt;
            tile_of(min(w + i / (VB * 2) * W, kTiles - 1), mt, jt);
            xz[i].load(row_of(mt), 16 * (i % (VB * 2)) + 4 * gq, g.p);
          }
        }
      }
    }
    f32x4 ot[OUT ? CT : 1][OUT ? 4 : 1];
    if constexpr (OUT) {
      if (g.save_s) {
        f32x4* to = reinterpret_cast<f32x4*>(g.save_s) +
                    (((int64_t)s * g.nch + c0 + c) * W + w) * (CT * 2 * RB * 64) + lane_id();
#pragma unroll
        for (int i = 0; i < CT * 2 * RB; ++i) to[i * 64] = S[i / (2 * RB)][i % (2 * RB)];
      }
      // tiles of P, transposed: rows are tokens j, columns i (the last ones twice: no branch)
      struct Pair {
        Frag<NT> k[RB], q[RB];
        f32x4 d;
      };
      steps<TP, AHEAD, Pair>(
          [&](int u, Pair& b) {
            int mt, jt;
            tile_of(min(w + u * W, kTiles - 1), mt, jt);
#pragma unroll
            for (int kb = 0; kb < RB; ++kb) {
              b.k[kb] = rows_of<RB, NT>(kt, jt, kb);
              b.q[kb] = rows_of<RB, NT>(qt, mt, kb);
            }
            b.d = NT == 1 ? dt[(mt - jt) * 64 + lane_id()] : D[NT == 1 ? 0 : u];
          },
          [&](int u, Pair& b) {
            int mt, jt;
            tile_of(min(w + u * W, kTiles - 1), mt, jt);
            f32x4 x = zero4();
#pragma unroll
            for (int kb = 0; kb < RB; ++kb) x = dl::mul_inputs(x, b.k[kb], b.q[kb]);
            x = rounded(x * b.d);
            if constexpr (LEARN == kDq) {
              if (w + u * W < kTiles) {   // here i: dO, j: V; K in V's place
                f32x4 z = zero4();
                const bool live = 16 * mt + m < len;
#pragma unroll
                for (int kb = 0; kb < VB; ++kb) {
                  f32x4 h[2];
#pragma unroll
                  for (int j = 0; j < 2; ++j) {
                    const int col = 32 * kb + 16 * j + 4 * gq;
                    if (EARLY && quads) {
                      h[j] = xz[EARLY ? (u * VB + kb) * 2 + j : 0].get(live && col < g.p);
                    } else if (quads) {
                      Quad<In> q;
                      q.load(row_of(mt), col, g.p);
                      h[j] = q.get(live && col < g.p);
                    } else {
                      h[j] = four_of(row_of(mt), col, g.p, live);
                    }
                  }
                  z = dl::mul_inputs(z, value_rows<In, VB>(vt, jt, kb),
                                     dl::split<NT>(h[0], h[1]));
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  acc += (float)(16 * (mt - jt) + m - 4 * gq - i) * (x[i] * z[i]);
              }
            }
            const Frag<NI> f = terms<NT>(x, zero4());
            const int half = mt == 2 && jt == 2 ? 1 : jt & 1;
            bf16* at = pl + dl::tri(mt, jt >> 1) * kFrag + lane_id() * 8 + 4 * half;
#pragma unroll
            for (int n = 0; n < NI; ++n)
              *reinterpret_cast<bf16x4*>(at + n * kLow * kFrag) = dl::low_half(f.t[n]);
          });
      // (Q S)^T: columns in registers, the token in the lane
#pragma unroll
      for (int i = 0; i < CT * 4; ++i) ot[i / 4][i % 4] = zero4();
      struct Four {
        Frag<NT> q[4];
      };
      steps<RB, AHEAD, Four>(
          [&](int kb, Four& b) {
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) b.q[mt] = rows_of<RB, NT>(qt, mt, kb);
          },
          [&](int kb, Four& b) {
            Frag<NI> sb[CT];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) sb[ct] = terms<NT>(S[ct][2 * kb], S[ct][2 * kb + 1]);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
              Frag<NI> all[4];
#pragma unroll
              for (int mt = 0; mt < 4; ++mt) all[mt] = sb[ct];
              dl::mul_each(ot[ct], all, b.q);
            }
          });
#pragma unroll
      for (int i = 0; i < CT * 4; ++i) ot[i / 4][i % 4] = rounded(ot[i / 4][i % 4] * e[i % 4]);
      if constexpr (LEARN) {
        if constexpr (LEARN == kDv) {              // n a^n <S, Y>
          float dot = 0.f;
#pragma unroll
          for (int mt = 0; mt < 2 * RB; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) dot += xS[mt][i] * S[0][mt][i];
          acc += (float)len * aC * dot;
        } else {                                   // (i + 1) q . dq, and i k . dk in turned order
          const int col = 16 * tile0 + 4 * gq;
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) {
            const int t = 16 * mt + m;
            const f32x4 x = quads ? xq[mt].get(t < len && col < g.p)
                                  : four_of(row_of(mt), col, g.p, t < len);
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) dot += x[i] * ot[0][mt][i];
            acc += (float)(t + (g.rev ? 0 : 1)) * dot;
          }
        }
      }
    }
    // the wave's columns of V by token slots: what P meets
    Frag<NT> vf[OUT || NT == 1 ? CT : 1][2];
    if constexpr (OUT || NT == 1) {
#pragma unroll
      for (int i = 0; i < CT * 2; ++i) {
        if constexpr (NT == 1) {
          vf[i / 2][i % 2] = cols_of<VB, 1>(vt, tile0 + i / 2, i % 2);
        } else {
          f32x4 a, b;
          value_cols<In, VB>(vt, tile0 + i / 2, i % 2, a, b);
          vf[i / 2][i % 2] = dl::split<NT>(a, b);
        }
      }
    }
    if constexpr (OUT) {
      lds_barrier();
      // ---- P is in LDS
      __builtin_amdgcn_s_setprio(1);
      struct One {
        Frag<NI> p;
      };
      steps<6, AHEAD, One>(
          [&](int st, One& b) {
            const int mt = st < 2 ? st : st < 4 ? 2 : 3, kb = st < 2 ? 0 : st & 1;
            const bf16* at = pl + dl::tri(mt, kb) * kFrag + lane_id() * 8;
#pragma unroll
            for (int n = 0; n < NI; ++n) {
              if (dl::half_tri(mt, kb)) {
                const bf16x4 h =
                    *reinterpret_cast<const bf16x4*>(at + n * kLow * kFrag + (mt == 2 ? 4 : 0));
                const bf16x4 no = {(bf16)0.f, (bf16)0.f, (bf16)0.f, (bf16)0.f};
                b.p.t[n] = __builtin_shufflevector(h, no, 0, 1, 2, 3, 4, 5, 6, 7);
              } else {
                b.p.t[n] = *reinterpret_cast<const bf16x8*>(at + n * kLow * kFrag);
              }
            }
          },
          [&](int st, One& b) {
            const int mt = st < 2 ? st : st < 4 ? 2 : 3, kb = st < 2 ? 0 : st & 1;
            f32x4 x[CT];
            Frag<NT> v[CT];
            Frag<NI> all[CT];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
              x[ct] = ot[ct][mt];
              v[ct] = vf[ct][kb];
              all[ct] = b.p;
            }
            dl::mul_each(x, v, all);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) ot[ct][mt] = x[ct];
          });
      auto store = [&](auto* o) {
        typedef typename std::remove_pointer<decltype(o)>::type Out;
        typedef Out out4u __attribute__((ext_vector_type(4), aligned(sizeof(Out))));
        // the chunk's lowest row, the lane's place in a row tile from its lowest
        char* base = reinterpret_cast<char*>(o + ((int64_t)s * g.T + t0 + (g.rev ? len - C : 0)) *
                                                     g.p + 16 * tile0);
        const int lane = fresh(lane_id()), m = lane & 15, gq = lane >> 4;
        const uint32_t at = ((g.rev ? 15 - m : m) * g.p + 4 * gq) * (uint32_t)sizeof(Out);
        const int tile = 16 * g.p * (int)sizeof(Out);
        auto row = [&](int mt) {
          return reinterpret_cast<Out*>(base + (g.rev ? 3 - mt : mt) * tile + at);
        };
        if (full && len == C) {
#pragma unroll
          for (int i = 0; i < CT * 4; ++i) {
            out4u y;
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = from_f32<Out>(ot[i % CT][i / CT][j]);
            *reinterpret_cast<out4u*>(row(i / CT) + 16 * (i % CT)) = y;
          }
        } else {
#pragma unroll
          for (int i = 0; i < CT * 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (16 * (i / CT) + m < len && 16 * (tile0 + i % CT) + 4 * gq + j < g.p)
                row(i / CT)[16 * (i % CT) + j] = from_f32<Out>(ot[i % CT][i / CT][j]);
        }
      };
      if (!__is_same(In, float) && g.wide)
        store((float*)g.o);
      else
        store((In*)g.o);
    }
    // S <- a^n S + K^T (w V), half the tokens at a time
#pragma unroll
    for (int i = 0; i < CT * 2 * RB; ++i) S[i / (2 * RB)][i % (2 * RB)] *= aC;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      f32x4 wa, wb;
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
      Frag<NI> f[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        f32x4 a, b;
        if constexpr (NT == 1) {
          Raw<bf16> x;
          x.x[0] = __builtin_bit_cast(Raw<bf16>::u4, vf[ct][kb].t[0]);
          x.values(a, b);
        } else {
          value_cols<In, VB>(vt, tile0 + ct, kb, a, b);
        }
        f[ct] = terms<NT>(rounded(wa * a), rounded(wb * b));
      }
      constexpr int U = NT == 1 ? 2 : 1;
      struct Some {
        Frag<NT> k[U];
      };
      steps<2 * RB / U, AHEAD, Some>(
          [&](int st, Some& b) {
#pragma unroll
            for (int u = 0; u < U; ++u) b.k[u] = cols_of<RB, NT>(kt, st * U + u, kb);
          },
          [&](int st, Some& b) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
              f32x4 x[U];
              Frag<NI> all[U];
#pragma unroll
              for (int u = 0; u < U; ++u) {
                x[u] = S[ct][st * U + u];
                all[u] = f[ct];
              }
              dl::mul_each(x, b.k, all);
#pragma unroll
              for (int u = 0; u < U; ++u) S[ct][st * U + u] = x[u];
            }
          });
    }
    if (more) {
      if (KD == 1) lds_barrier();                  // the tiles are read
      put(c + 1);
    }
  }
  if (LEARN) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) acc += __shfl_xor(acc, d);
    if (lane_id() == 0) g.part[sn * W + w] = acc;
  }
  if (!g.fin || (OUT && !(g.rev ? head : tail))) return;
  float* out = g.fin + (OUT ? (int64_t)seg * g.nb + s : sn) * rp;
  const int lane = fresh(lane_id());
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int mt = 0; mt < 2 * RB; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int a = 16 * mt + 4 * (lane >> 4) + i, col = 16 * (tile0 + ct) + (lane & 15);
        if (a < g.r && col < g.p)
          out[(int64_t)a * g.s_row + (int64_t)col * g.s_col] = S[ct][mt][i];
      }
}

inline int learn_waves(int p) { return p <= 64 ? 4 : 8; }

template <typename In, int RB, int P, bool OUT, int LEARN>
static void walk(const Walks& a, hipStream_t st) {
  constexpr int lds = walk_lds<In, RB, P, OUT>(walk_sets<In, RB, P, OUT, LEARN>());
  static_assert(lds <= dl::kMaxLds, "");
  auto kern = decay_walk_kernel<In, RB, P, OUT, LEARN>;
  static uint64_t done;
  dl::allow_lds(kern, lds, done);
  const int nb = a.w[0].nb, x = a.n == 1 ? nb : (nb + 7) / 8 * 24;
  hipLaunchKernelGGL(kern, dim3(x, a.w[0].nruns), dim3(64 * waves<In, P, OUT, LEARN>()), lds, st, a);
}

// One file a type instantiates it.
template <typename In> int launch_walk(const Walks& g, bool out, int learn, hipStream_t st) {
  auto go = [&](auto rb, auto cols) {
    constexpr int RB = decltype(rb)::value, P = decltype(cols)::value;
    if (!out)
      walk<In, RB, P, false, kNone>(g, st);
    else if (learn == kDq)
      walk<In, RB, P, true, kDq>(g, st);
    else if (learn == kDk)
      walk<In, RB, P, true, kDk>(g, st);
    else if (learn == kDv)
      walk<In, RB, P, true, kDv>(g, st);
    else
      walk<In, RB, P, true, kNone>(g, st);
    return launch_status("smat_head_decay_scan");
  };
  auto rows = [&](auto cols) {
    switch (dl::rblocks(g.w[0].r)) {
      case 1: return go(std::integral_constant<int, 1>(), cols);
      case 2: return go(std::integral_constant<int, 2>(), cols);
      case 3: return go(std::integral_constant<int, 3>(), cols);
      default: return go(std::integral_constant<int, 4>(), cols);
    }
  };
  return g.w[0].p <= 64 ? rows(std::integral_constant<int, 64>())
                   : rows(std::integral_constant<int, 128>());
}
extern template int launch_walk<bf16>(const Walks&, bool, int, hipStream_t);
extern template int launch_walk<f16>(const Walks&, bool, int, hipStream_t);
extern template int launch_walk<float>(const Walks&, bool, int, hipStream_t);

}  // namespace hd
}  // namespace smat
