// The end of a block (block_join) and its gradient, a row of D columns at a time:
//
//   y  = post f / rms(f)                         the norm after the block
//   u  = m gate(z) y                             its gate, and dropout's m = 0 or 1 / (1 - p)
//   h' = h + s u                                 the residual scale and sum
//   x  = pre h' / rms(h')                        the norm before the next block
//
// with rms(t)^2 = mean t^2 + eps; every part but h and f may be absent.  Backward, from the
// gradients dh' and dx of both results, with r = 1 / rms:
//
//   g   = dh' + r2 t - h' r2^3 mean(t h'),  t = pre dx
//   df  = r1 v - f r1^3 mean(v f),          v = post gate m s g
//   dh  = g,  dz = gate'(z) m s g y,  dpost = sum (gate m s g) f r1,
//   ds  = sum g u,  dpre = sum dx h' r2     (sums over the rows)
//
// Bandwidth kernels: each tensor is read once and written once.  The backward reads f, h and
// z and forms y, u and h' again in fp32 as the forward did, the rows' two factors r1 and r2
// are kept; so no rounded h' enters the gradients.  A row is a group of waves', a lane has eight
// of its columns; rows are walked with the weights, and in the backward the columns' sums, in
// registers.  The sums leave through the workgroups' parts, added in a fixed order.
//
// Measured: without dropout at 131072 x 1024 (bf16, h fp32) the forward takes 351 us, 5.3 TB/s,
// above a copy's rate, and the gradient 526, 5.6.  32768 x 768, all bf16, has half the bytes a
// value and is bound by instructions: forward 71 us (3.5 TB/s; 56 without dropout, 41 without a
// gate too), gradient 124 (3.4; 105 without dropout), sums 4.  The generator is a lane's 36 wide
// multiply-adds a row at a quarter rate and their exclusive ors, the gate eight exponentials and
// reciprocals; a quarter of the lanes have no columns there (as many values at 1024 columns: 46
// us for 55); and one kernel for every gate and absent tensor spills 16 to 18 scalars (gradient
// 24 to 27), read back in the rows' loop.  A row is a wave's at least: at 64 columns, 8 lanes of
// 64, the forward runs at 0.8 TB/s.
// Beyond 4096 columns a row is nine to sixteen waves' and a lane has 128 registers: the gradient's
// sums go to LDS there, and no row is loaded ahead (6144 x 4104, bf16: 188 us, 2.1 TB/s; sums in
// registers 344, and rows ahead 600); 5 to 8 registers are spilt still, in fp32 39 (330 us, 2.4).
//
// Dropout's mask is never stored: place (row, column) is kept where its word of Philox 4x32,
// ten rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, SC 2011),
// is at least p 2^32 (rounded to even, at most 2^32 - 1); key = the seed's halves, counter =
// (column / 4, row, salt, 0), the word column % 4 of the four.
#include "row_groups.hpp"
#include "smat_host.hpp"

namespace smat {
namespace join {

constexpr int kMinD = 8, kMaxD = 8192;   // columns
enum Gate { kAbsent = 0, kLinear = 1, kSigmoid = 2, kSilu = 3 };

struct Args {
  const void *f, *h, *z;
  const void *post, *s, *pre;              // weights (D) of types wt[0..2]; or null
  int wt[3];
  const int64_t* seed;                     // or null: no dropout; the backward's is the kept one
  uint32_t salt, threshold;
  float scale, keep, eps;                  // scale: where s is null; keep: a kept place's factor
  int gate;
  int64_t rows, f_st, h_st, z_st;
  int D, group;                            // threads a row
  // forward
  void *h2, *x;
  float* factors;                          // (rows, 2): r1, r2, and behind them the seed; or null
  // backward
  const void *dh, *dx;                     // or null: zero
  int64_t dh_st, dx_st;
  void *df, *dz, *dh_out;                  // dz: null without a gate
  float* part;                             // (workgroups, 3, D); or null
};

// The four words of a place's block of columns.  Rows are a wave's, so the first two rounds
// cost a lane nothing in the rows' loop: every product in them is of the columns or of the
// row alone.
__device__ __forceinline__ void philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)0xD2511F53u * c[0], b = (uint64_t)0xCD9E8D57u * c[2];
    const uint32_t x = (uint32_t)(b >> 32) ^ c[1] ^ k0, y = (uint32_t)(a >> 32) ^ c[3] ^ k1;
    c[1] = (uint32_t)b;
    c[3] = (uint32_t)a;
    c[0] = x;
    c[2] = y;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// What a lane has of a row: eight columns.
typedef float f8 __attribute__((ext_vector_type(8)));
template <typename In>
__device__ __forceinline__ f8 eight(Raw<In> x, int c, int D) {
  if ((D & 7) && c + 8 > D && c < D) x.drop(8 - (D & 7));
  if (c >= D) x.zero();
  f32x4 a, b;
  x.values(a, b);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <typename Out>
__device__ __forceinline__ void put(Out* row, const f8& y, int c, int D) {
  if (c < D)
    store8(row + c, __builtin_shufflevector(y, y, 0, 1, 2, 3),
           __builtin_shufflevector(y, y, 4, 5, 6, 7), D - c);
}
__device__ __forceinline__ float sum8(const f8& x) {
  return ((x[0] + x[4]) + (x[1] + x[5])) + ((x[2] + x[6]) + (x[3] + x[7]));
}

// Eight weights; `absent` where there are none, and past the last column.
__device__ __forceinline__ f8 weights(const void* w, int type, float absent, int c, int D) {
  f8 y;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = absent;
  if (!w) return y;
  auto read = [&](auto t) {
    typedef decltype(t) T;
    Raw<T> x;
    x.load((const T*)w + min(c, D - 8));
    return eight(x, c, D);
  };
  const f8 x = type == SMAT_F32 ? read(float()) : type == SMAT_BF16 ? read(bf16()) : read(f16());
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = c + i < D ? x[i] : absent;
  return y;
}

// gate(z), and its slope.  The exp is of x = -|z|, and 1 - sigmoid(z) is sigmoid(-z), so nothing
// cancels at either end.  x ends at -200, where exp(x) has long been zero in fp32: beyond 2.3e38
// and at infinity the products below would overflow, and then cancel to no number.  (A comparison,
// not a minimum: what is not a number stays so.)  exp(x) is 2^(x log2 e) with the product's
// rounding error put back, since the hardware's exponential takes it as it is, and as the square
// of 2^(x log2 e / 2), since that instruction gives no subnormal results.
__device__ __forceinline__ void sigmoid(float z, float& s, float& t, float& x) {
  constexpr float high = 0x1.715476p+0f, low = 0x1.4ae0cp-26f;     // log2 e
  x = -fabsf(z);
  x = x < -200.f ? -200.f : x;
  const float y = x * high;
  const float off = fmaf(x, low, fmaf(x, high, -y));
  const float root = __builtin_amdgcn_exp2f(0.5f * y);
  const float e = root * fmaf(off, 0x1.62e43p-1f, 1.f) * root;
  const float d = __builtin_amdgcn_rcpf(1.f + e);
  s = z >= 0.f ? d : e * d;
  t = z >= 0.f ? e * d : d;
}
template <bool SLOPE>
__device__ __forceinline__ void gate_of(int kind, const f8& z, f8& a, f8& slope) {
  if (kind == kLinear) {
    a = z;
#pragma unroll
    for (int i = 0; i < 8; ++i) slope[i] = 1.f;
  } else if (kind == kSigmoid) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float s, t, x;
      sigmoid(z[i], s, t, x);
      a[i] = s;
      if (SLOPE) slope[i] = s * t;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // at an infinite z the factor that is zero meets a finite one
      float s, t, x;
      sigmoid(z[i], s, t, x);
      a[i] = (z[i] >= 0.f ? z[i] : x) * s;
      if (SLOPE) slope[i] = s * (1.f + (z[i] >= 0.f ? -x : x) * t);
    }
  }
}

// The rows' walk.  A workgroup has `per` groups of threads, one row each, and takes `per` rows
// at a time; all its groups make as many turns, since those of several waves share barriers.
// A turn's rows are loaded while the last one's are worked on.
struct Walk {
  int c, in_group, group, of, per, turn = 0;       // `of`: which group this thread is of
  float (*sums)[16];
  __device__ __forceinline__ Walk(int group, float (*sums)[16]) : group(group), sums(sums) {
    in_group = (int)threadIdx.x % group;
    of = __builtin_amdgcn_readfirstlane((int)threadIdx.x / group);
    per = blockDim.x / group;
    c = in_group * 8;
  }
  // A row's sum over its threads: a wave's, or several waves' through LDS (sums alternate
  // between two places, so one barrier a sum).
  __device__ __forceinline__ float sum(float x) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    if (group > 64) {
      float* at = sums[turn];
      turn ^= 1;
      if (lane_id() == 0) at[wave_id()] = x;
      __syncthreads();
      const int waves = group / 64, w0 = of * waves;
      x = at[w0];
      for (int i = 1; i < waves; ++i) x += at[w0 + i];
    }
    return x;
  }
};

template <typename In, typename H> struct RowIn {
  Raw<In> f, z;
  Raw<H> h;
  __device__ __forceinline__ void load(const Args& g, int64_t row, int c) {
    c = min(c, g.D - 8);
    f.load((const In*)g.f + row * g.f_st + c);
    h.load((const H*)g.h + row * g.h_st + c);
    if (g.gate) z.load((const In*)g.z + row * g.z_st + c);
  }
};
template <typename In, typename H> struct RowBack : RowIn<In, H> {
  Raw<In> x;
  Raw<H> d;
  float r1, r2;
  __device__ __forceinline__ void load(const Args& g, int64_t row, int c) {
    RowIn<In, H>::load(g, row, c);
    c = min(c, g.D - 8);
    if (g.dx) x.load((const In*)g.dx + row * g.dx_st + c);
    if (g.dh) d.load((const H*)g.dh + row * g.dh_st + c);
    r1 = g.factors[2 * row];
    r2 = g.factors[2 * row + 1];
  }
};

__device__ __forceinline__ f8 mask_of(const Args& g, int c, uint32_t row, uint32_t k0,
                                      uint32_t k1) {
  f8 m;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    uint32_t w[4] = {(uint32_t)(c / 4 + b), row, g.salt, 0};
    philox(w, k0, k1);
#pragma unroll
    for (int i = 0; i < 4; ++i) m[4 * b + i] = w[i] >= g.threshold ? g.keep : 0.f;
  }
  return m;
}

// What a kernel's lane keeps through its rows.
struct Kept {
  f8 post, s, pre;
  uint32_t k0 = 0, k1 = 0;
  float mean;
  __device__ __forceinline__ Kept(const Args& g, int c) {
    post = weights(g.post, g.wt[0], 1.f, c, g.D);
    s = weights(g.s, g.wt[1], g.scale, c, g.D);
    pre = weights(g.pre, g.wt[2], 0.f, c, g.D);
    if (g.seed) {
      const uint32_t* k = reinterpret_cast<const uint32_t*>(g.seed);
      k0 = k[0];
      k1 = k[1];
    }
    mean = 1.f / (float)g.D;
  }
};

// MOST: threads a workgroup.
template <typename In, typename H, int MOST>
__global__ __launch_bounds__(MOST) void join_kernel(Args g) {
  __shared__ float sums[2][16];
  Walk l(g.group, sums);
  const int D = g.D, c = l.c;
  const Kept k(g, c);
  if (g.factors && g.seed && blockIdx.x == 0 && threadIdx.x == 0) {
    uint32_t* kept = reinterpret_cast<uint32_t*>(g.factors + 2 * g.rows);
    kept[0] = k.k0;
    kept[1] = k.k1;
  }
  const int64_t step = (int64_t)l.per * gridDim.x;
  int64_t r0 = (int64_t)blockIdx.x * l.per;
  RowIn<In, H> next;
  next.load(g, min(r0 + l.of, g.rows - 1), c);
  for (; r0 < g.rows; r0 += step) {
    const int64_t row = r0 + l.of;
    const bool live = row < g.rows;
    const RowIn<In, H> in = next;
    if (r0 + step < g.rows) next.load(g, min(row + step, g.rows - 1), c);
    f8 y = eight(in.f, c, D);
    float r1 = 1.f, r2 = 1.f;
    if (g.post) {
      r1 = rsqrtf(l.sum(sum8(y * y)) * k.mean + g.eps);
      y = y * r1 * k.post;
    }
    if (g.gate) {
      f8 a, slope;
      gate_of<false>(g.gate, eight(in.z, c, D), a, slope);
      y *= a;
    }
    if (g.seed) {
      const f8 m = mask_of(g, c, (uint32_t)row, k.k0, k.k1);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = m[i] != 0.f ? y[i] * m[i] : 0.f;
    }
    y = eight(in.h, c, D) + k.s * y;
    if (live) put((H*)g.h2 + row * D, y, c, D);
    if (g.pre) {
      r2 = rsqrtf(l.sum(sum8(y * y)) * k.mean + g.eps);
      if (live) put((In*)g.x + row * D, y * r2 * k.pre, c, D);
    }
    if (g.factors && live && l.in_group == 0) {
      g.factors[2 * row] = r1;
      g.factors[2 * row + 1] = r2;
    }
  }
}

template <typename In, typename H, int MOST>
__global__ __launch_bounds__(MOST) void join_backward_kernel(Args g) {
  __shared__ float sums[2][16];
  extern __shared__ __align__(16) float part[];    // the columns' sums of the groups: 3 D
  // Nine waves a row and more leave a lane 128 registers: the next row is not loaded ahead, and the
  // sums are in LDS, every lane's own, (3, 8, threads).
  constexpr bool MANY = MOST <= 512;
  Walk l(g.group, sums);
  const int D = g.D, c = l.c;
  Kept k(g, c);
  const f8 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  f8 apost = zero, as = zero, apre = zero;
  const int64_t step = (int64_t)l.per * gridDim.x;
  int64_t r0 = (int64_t)blockIdx.x * l.per;
  if (!MANY && g.part) {
#pragma unroll
    for (int i = 0; i < 24; ++i) part[i * l.group + l.in_group] = 0.f;
  }
  auto add = [&](f8& sum, int j, const f8& x) {
    if (MANY) {
      sum += x;
    } else if (g.part) {
#pragma unroll
      for (int i = 0; i < 8; ++i) part[(j * 8 + i) * l.group + l.in_group] += x[i];
    }
  };
  RowBack<In, H> next;
  if (MANY) next.load(g, min(r0 + l.of, g.rows - 1), c);
  for (; r0 < g.rows; r0 += step) {
    const int64_t row = r0 + l.of;
    const bool live = row < g.rows;
    if (!MANY) next.load(g, min(row, g.rows - 1), c);
    const RowBack<In, H> in = next;
    if (MANY && r0 + step < g.rows) next.load(g, min(row + step, g.rows - 1), c);
    if constexpr (!MANY && sizeof(In) == 4) {      // (rows of twice the registers)
      k.post = weights(g.post, g.wt[0], 1.f, c, D);
      k.s = weights(g.s, g.wt[1], g.scale, c, D);
      k.pre = weights(g.pre, g.wt[2], 0.f, c, D);
    }
    const float r1 = in.r1, r2 = in.r2;            // (r1 is one without a norm after the block)
    const f8 f = eight(in.f, c, D);
    f8 y = f * r1 * k.post;
    f8 a = zero + 1.f, z = zero;                   // gate m, and m gate'
    if (g.gate) gate_of<true>(g.gate, eight(in.z, c, D), a, z);
    // A dropped place counts for nothing, as in the forward, whatever y, gate and dh' hold there.
    // (Where registers are few, y goes by the places' bits and behind the branch, else 120 of them
    // are spilt: 287 us at 6144 x 4104 bf16, 197 so.)
    uint32_t dropped = 0;
    if (g.seed) {
      const f8 m = mask_of(g, c, (uint32_t)row, k.k0, k.k1);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] = m[i] != 0.f ? m[i] * a[i] : 0.f;
        z[i] = m[i] != 0.f ? m[i] * z[i] : 0.f;
        if (MANY) y[i] = m[i] != 0.f ? y[i] : 0.f;
        dropped |= m[i] != 0.f ? 0u : 1u << i;
      }
    }
    if (!MANY) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = dropped >> i & 1 ? 0.f : y[i];
    }
    f8 d = g.dh ? eight(in.d, c, D) : zero;        // dh', then dh
    if (g.dx) {
      const f8 h = eight(in.h, c, D) + k.s * (a * y);
      f8 t = eight(in.x, c, D);
      if (live) add(apre, 2, t * h * r2);
      t *= k.pre;
      const float q = l.sum(sum8(t * h)) * k.mean * r2 * r2 * r2;
      d += r2 * t - h * q;
    }
    if (live) {
      put((H*)g.dh_out + row * D, d, c, D);
      add(as, 1, d * (a * y));
    }
    if (g.seed) {
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = dropped >> i & 1 ? 0.f : d[i];
    }
    d *= k.s;
    if (g.gate && live) put((In*)g.dz + row * D, z * (d * y), c, D);
    d *= a;                                        // dy
    if (g.post) {
      if (live) add(apost, 0, d * f * r1);
      d *= k.post;
      const float q = l.sum(sum8(d * f)) * k.mean * r1 * r1 * r1;
      d = r1 * d - f * q;
    }
    if (live) put((In*)g.df + row * D, d, c, D);
  }
  if (!g.part) return;
  // the groups' sums one after another into LDS, the last into the workgroup's part
  float* out = g.part + (int64_t)blockIdx.x * 3 * D;
  if (!MANY) {
#pragma unroll
    for (int i = 0; i < 24; ++i)
      if (c + i % 8 < D) out[i / 8 * D + c + i % 8] = part[i * l.group + l.in_group];
    return;
  }
  for (int n = 0; n < l.per; ++n) {
    if (n) __syncthreads();
    if (l.of != n) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (c + i >= D) break;
      float x[3] = {apost[i], as[i], apre[i]};
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        if (n) x[j] += part[j * D + c + i];
        (n + 1 < l.per ? part : out)[j * D + c + i] = x[j];
      }
    }
  }
}

// The columns' sums of the workgroups' parts, in the same order every time.
__global__ __launch_bounds__(1024) void join_sums_kernel(const float* __restrict__ part, int parts,
                                                         int D, float* post, float* s,
                                                         float* pre) {
  __shared__ float sums[64][17];
  const int i = threadIdx.x % 16, c = blockIdx.x * 16 + i, k = threadIdx.x / 16, n = 3 * D;
  float x = 0.f;
  if (c < n) {
#pragma unroll 8
    for (int j = k; j < parts; j += 64) x += part[(int64_t)j * n + c];
  }
  sums[k][i] = x;
  __syncthreads();
  if (k == 0 && c < n) {
    for (int j = 1; j < 64; ++j) x += sums[j][i];
    float* to = c < D ? post : c < 2 * D ? s : pre;
    if (to) to[c % D] = x;
  }
}

// Threads a row (whole waves, eight columns a lane), rows a workgroup takes at a time, and
// workgroups: as many as stay on the CUs, each walking its rows (16 waves a CU, 8 in the
// backward).
inline int group_of(int D) { return (D + 511) / 512 * 64; }
inline int rows_of(int D) { return group_of(D) < 512 ? 512 / group_of(D) : 1; }
inline int64_t grid_of(int64_t rows, int D, bool backward) {
  const int waves = group_of(D) * rows_of(D) / 64, on = (backward ? 8 : 16) / waves;
  const int64_t most = 256 * (on > 1 ? on : 1), need = (rows + rows_of(D) - 1) / rows_of(D);
  return need < most ? need : most;
}

template <bool BACKWARD>
static int launch_join(int dtype, int h_dtype, Args& g, hipStream_t st) {
  g.group = group_of(g.D);
  const dim3 grid(grid_of(g.rows, g.D, BACKWARD)), block(g.group * rows_of(g.D));
  auto go = [&](auto in, auto h) {
    typedef decltype(in) In;
    typedef decltype(h) H;
    auto kern = [&](auto most) {
      constexpr int MOST = decltype(most)::value;
      if constexpr (BACKWARD) {
        auto back = join_backward_kernel<In, H, MOST>;
        if (MOST > 512) {
          static uint64_t done;
          allow_lds(back, 96 * MOST, done);
        }
        const int lds = !g.part ? 0 : MOST > 512 ? 96 * g.group : rows_of(g.D) > 1 ? 12 * g.D : 0;
        hipLaunchKernelGGL(back, grid, block, lds, st, g);
      } else {
        hipLaunchKernelGGL((join_kernel<In, H, MOST>), grid, block, 0, st, g);
      }
    };
    if (g.group <= 512)
      kern(std::integral_constant<int, 512>());
    else
      kern(std::integral_constant<int, 1024>());
    return launch_status(BACKWARD ? "smat_block_join_backward" : "smat_block_join");
  };
  if (dtype == SMAT_BF16) return h_dtype == SMAT_F32 ? go(bf16(), float()) : go(bf16(), bf16());
  if (dtype == SMAT_F16) return h_dtype == SMAT_F32 ? go(f16(), float()) : go(f16(), f16());
  return go(float(), float());
}

static int check(const char* who, int dtype, int h_dtype, const Args& g, double p) {
  SMAT_REQUIRE(dtype == SMAT_BF16 || dtype == SMAT_F16 || dtype == SMAT_F32, SMAT_EINVAL,
               "%s: unknown dtype %d", who, dtype);
  SMAT_REQUIRE(h_dtype == dtype || h_dtype == SMAT_F32, SMAT_EINVAL,
               "%s: the residual stream's dtype %d is neither %d nor fp32", who, h_dtype, dtype);
  SMAT_REQUIRE(g.rows >= 0 && g.rows < (1ll << 31), SMAT_EUNSUPPORTED, "%s: %lld rows", who,
               (long long)g.rows);
  SMAT_REQUIRE(g.D >= kMinD && g.D <= kMaxD, SMAT_EUNSUPPORTED, "%s: %d columns, not %d to %d",
               who, g.D, kMinD, kMaxD);
  SMAT_REQUIRE(g.gate >= kAbsent && g.gate <= kSilu, SMAT_EINVAL, "%s: unknown gate %d", who,
               g.gate);
  for (int t : g.wt)
    SMAT_REQUIRE(t == SMAT_BF16 || t == SMAT_F16 || t == SMAT_F32, SMAT_EINVAL,
                 "%s: unknown weight dtype %d", who, t);
  SMAT_REQUIRE(g.eps >= 0.f && p >= 0 && p < 1 && (p == 0 || g.seed), SMAT_EINVAL,
               "%s: eps=%g, dropout=%g (needs a seed)", who, g.eps, p);
  return SMAT_OK;
}

static Args make(const void* f, const void* h, const void* z, const void* post, const void* s,
                 const void* pre, int post_t, int s_t, int pre_t, const int64_t* seed, int64_t rows,
                 int D, int gate, float eps, float scale, double p, uint32_t salt, int64_t f_st,
                 int64_t h_st, int64_t z_st) {
  Args g = {};
  g.f = f;
  g.h = h;
  g.z = z;
  g.post = post;
  g.s = s;
  g.pre = pre;
  g.wt[0] = post_t;
  g.wt[1] = s_t;
  g.wt[2] = pre_t;
  g.seed = p > 0 ? seed : nullptr;
  g.rows = rows;
  g.D = D;
  g.gate = gate;
  g.eps = eps;
  g.scale = scale;
  const double t = rint(p * 4294967296.0);         // ties to even
  g.threshold = t >= 4294967295.0 ? 4294967295u : (uint32_t)t;
  // the inverse of the rate that the threshold keeps, not of 1 - p: near one they differ
  g.keep = (float)(4294967296.0 / (4294967296.0 - g.threshold));
  g.salt = salt;
  g.f_st = f_st;
  g.h_st = h_st;
  g.z_st = z_st;
  return g;
}

}  // namespace join
}  // namespace smat

extern "C" int smat_block_join(int dtype, int h_dtype, const void* f, const void* h, const void* z,
                               const void* post, const void* s, const void* pre, int post_t,
                               int s_t, int pre_t, const int64_t* seed, void* h2, void* x,
                               float* factors, int64_t rows, int D, int gate, float eps,
                               float scale, double p, uint32_t salt, int64_t f_st, int64_t h_st,
                               int64_t z_st, void* stream) {
  using namespace smat;
  using namespace smat::join;
  clear_error();
  const char* who = "smat_block_join";
  Args g = make(f, h, z, post, s, pre, post_t, s_t, pre_t, seed, rows, D, gate, eps, scale, p, salt,
                f_st, h_st, z_st);
  const int rc = check(who, dtype, h_dtype, g, p);
  if (rc) return rc;
  if (rows == 0) return SMAT_OK;
  SMAT_REQUIRE(f && h && h2 && (!gate || z) && (!pre || x), SMAT_EINVAL, "%s: null pointer", who);
  g.h2 = h2;
  g.x = x;
  g.factors = factors;
  return launch_join<false>(dtype, h_dtype, g, (hipStream_t)stream);
}

extern "C" int64_t smat_block_join_workspace_bytes(int64_t rows, int D) {
  using namespace smat::join;
  if (rows <= 0 || D < kMinD || D > kMaxD) return 0;
  return grid_of(rows, D, true) * 12 * D;
}

extern "C" int smat_block_join_backward(
    int dtype, int h_dtype, const void* f, const void* h, const void* z, const void* post,
    const void* s, const void* pre, int post_t, int s_t, int pre_t, const float* factors,
    const void* dh, const void* dx, void* df, void* dh_out, void* dz,
    float* dpost, float* ds, float* dpre, int64_t rows, int D, int gate, float eps, float scale,
    double p, uint32_t salt, int64_t f_st, int64_t h_st, int64_t z_st, int64_t dh_st,
    int64_t dx_st, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace smat;
  using namespace smat::join;
  clear_error();
  const char* who = "smat_block_join_backward";
  const int64_t* seed = (const int64_t*)(factors ? factors + 2 * rows : nullptr);
  Args g = make(f, h, z, post, s, pre, post_t, s_t, pre_t, seed, rows, D, gate, eps, scale, p, salt,
                f_st, h_st, z_st);
  const int rc = check(who, dtype, h_dtype, g, p);
  if (rc) return rc;
  if (rows == 0) return SMAT_OK;
  SMAT_REQUIRE(f && h && factors && ((uintptr_t)factors & 7) == 0 && df && dh_out &&
                   (!gate || (z && dz)) && (!dx || pre),
               SMAT_EINVAL, "%s: null pointer, or factors not 8-byte aligned", who);
  const bool sums = dpost || ds || dpre;
  const int64_t need = sums ? smat_block_join_workspace_bytes(rows, D) : 0;
  SMAT_REQUIRE(workspace_bytes >= need && (workspace || !need) && ((uintptr_t)workspace & 15) == 0,
               SMAT_EINVAL, "%s: workspace of %lld bytes, %lld needed (16-byte aligned)", who,
               (long long)workspace_bytes, (long long)need);
  g.factors = const_cast<float*>(factors);
  g.dh = dh;
  g.dx = dx;
  g.dh_st = dh_st;
  g.dx_st = dx_st;
  g.df = df;
  g.dz = dz;
  g.dh_out = dh_out;
  g.part = sums ? (float*)workspace : nullptr;
  hipStream_t st = (hipStream_t)stream;
  const int rl = launch_join<true>(dtype, h_dtype, g, st);
  if (rl || !sums) return rl;
  const int parts = (int)(need / (12 * D));
  hipLaunchKernelGGL(join_sums_kernel, dim3((3 * D + 15) / 16), dim3(1024), 0, st, g.part, parts, D,
                     dpost, ds, dpre);
  return launch_status(who);
}
