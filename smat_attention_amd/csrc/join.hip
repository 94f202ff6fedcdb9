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
// are kept; so no rounded h' enters the gradients.  A row is one wave's up to 512 columns, else
// a workgroup's of up to eight, each lane with one or two groups of eight columns; rows are
// walked with the weights, and in the backward the columns' sums, in registers.  The sums leave
// through the workgroups' parts, added in a fixed order.
//
// Dropout's mask is never stored: place (row, column) is kept where its word of Philox 4x32,
// ten rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, SC 2011),
// is at least p 2^32; key = the seed's halves, counter = (column / 4, row, salt, 0), the word
// column % 4 of the four.
#include "row_groups.hpp"
#include "smat_host.hpp"

namespace smat {
namespace join {

constexpr int kMinD = 8, kMaxD = 8192, kMost = 512;   // columns, and threads a workgroup
enum Gate { kAbsent = 0, kLinear = 1, kSigmoid = 2, kSilu = 3 };

struct Args {
  const void *f, *h, *z;
  const void *post, *s, *pre;              // weights (D) of types wt[0..2]; or null
  int wt[3];
  const int64_t* seed;                     // or null: no dropout; the backward's is the kept one
  uint32_t salt, threshold;
  float scale, keep, eps;                  // scale: where s is null; keep: 1 / (1 - p)
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
  float* part;                             // (groups, 3, D); or null
};

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

__device__ __forceinline__ float weight(const void* w, int type, int c) {
  return type == SMAT_F32   ? ((const float*)w)[c]
         : type == SMAT_BF16 ? to_f32(((const bf16*)w)[c])
                             : to_f32(((const f16*)w)[c]);
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
  return x;
}
// A row's sum over its threads: a wave's, or a workgroup's through LDS (sums of either
// parity of calls alternate between two places, so one barrier a sum).
__device__ __forceinline__ float row_sum(float x, int group, float (*lds)[16], int& turn) {
  x = wave_sum(x);
  if (group > 64) {
    float* at = lds[turn];
    turn ^= 1;
    if (lane_id() == 0) at[wave_id()] = x;
    __syncthreads();
    x = at[0];
    for (int i = 1; i < group / 64; ++i) x += at[i];
  }
  return x;
}

// What a lane has of a row: NV groups of eight columns.
template <typename In, int NV> struct Cols {
  Raw<In> x[NV];
  __device__ __forceinline__ void load(const In* row, const int (&c)[NV], int D) {
#pragma unroll
    for (int v = 0; v < NV; ++v) x[v].load(row + min(c[v], D - 8));
  }
  // Element i of group v as fp32; columns past the last are zero.
  __device__ __forceinline__ void get(float (&y)[NV][8], const int (&c)[NV], int D) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if ((D & 7) && c[v] + 8 > D && c[v] < D) x[v].drop(8 - (D & 7));
      if (c[v] >= D) x[v].zero();
      f32x4 a, b;
      x[v].values(a, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[v][i] = a[i];
        y[v][i + 4] = b[i];
      }
    }
  }
};
template <typename Out, int NV>
__device__ __forceinline__ void put(Out* row, const float (&y)[NV][8], const int (&c)[NV], int D) {
#pragma unroll
  for (int v = 0; v < NV; ++v)
    if (c[v] < D)
      store8(row + c[v], f32x4{y[v][0], y[v][1], y[v][2], y[v][3]},
             f32x4{y[v][4], y[v][5], y[v][6], y[v][7]}, D - c[v]);
}

// gate(z), and its slope.  The exp is of -|z|, and 1 - sigmoid(z) is sigmoid(-z): neither
// overflows, and nothing cancels at either end.
__device__ __forceinline__ float gate_of(int kind, float z, float& slope) {
  if (kind == kLinear) {
    slope = 1.f;
    return z;
  }
  const float e = expf(-fabsf(z)), d = 1.f / (1.f + e);
  const float s = z >= 0.f ? d : e * d, t = z >= 0.f ? e * d : d;
  slope = kind == kSigmoid ? s * t : s * (1.f + z * t);
  return kind == kSigmoid ? s : z * s;
}

template <int NV> struct Lane {
  int c[NV];
  __device__ __forceinline__ Lane(int group) {
#pragma unroll
    for (int v = 0; v < NV; ++v) c[v] = (v * group + (int)threadIdx.x % group) * 8;
  }
};

// u of the gate's factor a and y, and the mask's factors m.
template <int NV>
__device__ __forceinline__ void masks(const Args& g, float (&m)[NV][8], const int (&c)[NV],
                                      int64_t row, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint32_t w[4] = {(uint32_t)(c[v] / 4 + b), (uint32_t)row, g.salt, 0};
      philox(w, k0, k1);
#pragma unroll
      for (int i = 0; i < 4; ++i) m[v][4 * b + i] = w[i] >= g.threshold ? g.keep : 0.f;
    }
}

template <int NV>
__device__ __forceinline__ void weights(float (&y)[NV][8], const void* w, int type, float absent,
                                        const int (&c)[NV], int D) {
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[v][i] = w && c[v] + i < D ? weight(w, type, c[v] + i) : absent;
}

template <typename In, typename H, int NV>
__global__ __launch_bounds__(kMost) void join_kernel(Args g) {
  __shared__ float sums[2][16];
  int turn = 0;
  const int group = g.group, D = g.D;
  const Lane<NV> l(group);
  const int64_t per = blockDim.x / group, step = per * gridDim.x;
  float post[NV][8], s[NV][8], pre[NV][8];
  weights<NV>(post, g.post, g.wt[0], 1.f, l.c, D);
  weights<NV>(s, g.s, g.wt[1], g.scale, l.c, D);
  weights<NV>(pre, g.pre, g.wt[2], 0.f, l.c, D);
  uint32_t k0 = 0, k1 = 0;
  if (g.seed) {
    const uint32_t* k = reinterpret_cast<const uint32_t*>(g.seed);
    k0 = k[0];
    k1 = k[1];
  }
  if (g.factors && g.seed && blockIdx.x == 0 && threadIdx.x == 0) {
    uint32_t* kept = reinterpret_cast<uint32_t*>(g.factors + 2 * g.rows);
    kept[0] = k0;
    kept[1] = k1;
  }
  const float mean = 1.f / (float)D;
  for (int64_t row = (int64_t)blockIdx.x * per + threadIdx.x / group; row < g.rows; row += step) {
    Cols<In, NV> fc, zc;
    Cols<H, NV> hc;
    fc.load((const In*)g.f + row * g.f_st, l.c, D);
    hc.load((const H*)g.h + row * g.h_st, l.c, D);
    if (g.gate) zc.load((const In*)g.z + row * g.z_st, l.c, D);
    float y[NV][8], h[NV][8];
    fc.get(y, l.c, D);
    float r1 = 1.f, r2 = 1.f;
    if (g.post) {
      float q = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) q += y[v][i] * y[v][i];
      r1 = rsqrtf(row_sum(q, group, sums, turn) * mean + g.eps);
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) y[v][i] = y[v][i] * r1 * post[v][i];
    }
    if (g.gate) {
      float z[NV][8];
      zc.get(z, l.c, D);
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float slope;
          y[v][i] *= gate_of(g.gate, z[v][i], slope);
        }
    }
    if (g.seed) {
      float m[NV][8];
      masks<NV>(g, m, l.c, row, k0, k1);
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) y[v][i] = m[v][i] != 0.f ? y[v][i] * m[v][i] : 0.f;
    }
    hc.get(h, l.c, D);
    float q = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[v][i] += s[v][i] * y[v][i];
        if (l.c[v] + i < D) q += h[v][i] * h[v][i];
      }
    put((H*)g.h2 + row * D, h, l.c, D);
    if (g.pre) {
      r2 = rsqrtf(row_sum(q, group, sums, turn) * mean + g.eps);
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) h[v][i] = h[v][i] * r2 * pre[v][i];
      put((In*)g.x + row * D, h, l.c, D);
    }
    if (g.factors && threadIdx.x % group == 0) {
      g.factors[2 * row] = r1;
      g.factors[2 * row + 1] = r2;
    }
  }
}

template <typename In, typename H, int NV>
__global__ __launch_bounds__(kMost) void join_backward_kernel(Args g) {
  __shared__ float sums[2][16];
  int turn = 0;
  const int group = g.group, D = g.D;
  const Lane<NV> l(group);
  const int64_t per = blockDim.x / group, step = per * gridDim.x;
  float post[NV][8], s[NV][8], pre[NV][8];
  weights<NV>(post, g.post, g.wt[0], 1.f, l.c, D);
  weights<NV>(s, g.s, g.wt[1], g.scale, l.c, D);
  weights<NV>(pre, g.pre, g.wt[2], 0.f, l.c, D);
  uint32_t k0 = 0, k1 = 0;
  if (g.seed) {
    const uint32_t* k = reinterpret_cast<const uint32_t*>(g.seed);
    k0 = k[0];
    k1 = k[1];
  }
  const float mean = 1.f / (float)D;
  float apost[NV][8], as[NV][8], apre[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < 8; ++i) apost[v][i] = as[v][i] = apre[v][i] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * per + threadIdx.x / group; row < g.rows; row += step) {
    Cols<In, NV> fc, zc, xc;
    Cols<H, NV> hc, dc;
    fc.load((const In*)g.f + row * g.f_st, l.c, D);
    hc.load((const H*)g.h + row * g.h_st, l.c, D);
    if (g.gate) zc.load((const In*)g.z + row * g.z_st, l.c, D);
    if (g.dx) xc.load((const In*)g.dx + row * g.dx_st, l.c, D);
    if (g.dh) dc.load((const H*)g.dh + row * g.dh_st, l.c, D);
    const float r1 = g.factors[2 * row], r2 = g.factors[2 * row + 1];
    // a = gate m, y, and z's part of dz
    float f[NV][8], z[NV][8], a[NV][8], d[NV][8];
    fc.get(f, l.c, D);
    if (g.gate) zc.get(z, l.c, D);
    if (g.seed) masks<NV>(g, a, l.c, row, k0, k1);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float m = g.seed ? a[v][i] : 1.f;
        float slope = 0.f;
        const float gate = g.gate ? gate_of(g.gate, z[v][i], slope) : 1.f;
        a[v][i] = m != 0.f ? m * gate : 0.f;
        z[v][i] = m != 0.f ? m * slope : 0.f;
      }
    if (g.dh) {
      dc.get(d, l.c, D);
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) d[v][i] = 0.f;
    }
    if (g.dx) {
      float h[NV][8], t[NV][8];
      hc.get(h, l.c, D);
      xc.get(t, l.c, D);
      float q = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = g.post ? f[v][i] * r1 * post[v][i] : f[v][i];
          h[v][i] += s[v][i] * (a[v][i] * y);
          apre[v][i] += t[v][i] * h[v][i] * r2;
          t[v][i] *= pre[v][i];
          q += t[v][i] * h[v][i];
        }
      q = row_sum(q, group, sums, turn) * mean * r2 * r2 * r2;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) d[v][i] += r2 * t[v][i] - h[v][i] * q;
    }
    put((H*)g.dh_out + row * D, d, l.c, D);
    float q = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = g.post ? f[v][i] * r1 * post[v][i] : f[v][i];
        as[v][i] += d[v][i] * (a[v][i] * y);
        const float du = d[v][i] * s[v][i];
        z[v][i] *= du * y;
        d[v][i] = du * a[v][i];                    // dy
        if (g.post) {
          apost[v][i] += d[v][i] * f[v][i] * r1;
          d[v][i] *= post[v][i];
          q += d[v][i] * f[v][i];
        }
      }
    if (g.gate) put((In*)g.dz + row * D, z, l.c, D);
    if (g.post) {
      q = row_sum(q, group, sums, turn) * mean * r1 * r1 * r1;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) d[v][i] = r1 * d[v][i] - f[v][i] * q;
    }
    put((In*)g.df + row * D, d, l.c, D);
  }
  if (!g.part) return;
  const int64_t at = (int64_t)blockIdx.x * per + threadIdx.x / group;
  float* p = g.part + at * 3 * D;
  put(p, apost, l.c, D);
  put(p + D, as, l.c, D);
  put(p + 2 * D, apre, l.c, D);
}

// The columns' sums of the groups' parts, in the same order every time.
__global__ __launch_bounds__(256) void join_sums_kernel(const float* __restrict__ part, int groups,
                                                        int D, float* post, float* s, float* pre) {
  __shared__ float sums[16][17];
  const int c = blockIdx.x * 16 + threadIdx.x % 16, k = threadIdx.x / 16, n = 3 * D;
  float x = 0.f;
  if (c < n)
    for (int i = k; i < groups; i += 16) x += part[(int64_t)i * n + c];
  sums[k][threadIdx.x % 16] = x;
  __syncthreads();
  if (k == 0 && c < n) {
    for (int i = 1; i < 16; ++i) x += sums[i][threadIdx.x];
    float* to = c < D ? post : c < 2 * D ? s : pre;
    if (to) to[c % D] = x;
  }
}

// Threads a row: whole waves, a lane for eight columns up to 4096, for sixteen beyond.
inline int group_of(int D) {
  const int lanes = (D + 7) / 8;
  return ((lanes <= kMost ? lanes : (lanes + 1) / 2) + 63) / 64 * 64;
}
// Rows a workgroup, and workgroups: up to as many as stay on the CUs, each walking its rows.
inline int rows_of(int D) { return group_of(D) == 64 ? 4 : 1; }
inline int64_t grid_of(int64_t rows, int D, bool backward) {
  const int waves = group_of(D) * rows_of(D) / 64;
  const int64_t most = 256 * ((backward ? 12 : 20) / waves > 1 ? (backward ? 12 : 20) / waves : 1);
  const int64_t need = (rows + rows_of(D) - 1) / rows_of(D);
  return need < most ? need : most;
}

template <bool BACKWARD>
static int launch_join(int dtype, int h_dtype, Args& g, hipStream_t st) {
  g.group = group_of(g.D);
  const dim3 grid(grid_of(g.rows, g.D, BACKWARD)), block(g.group * rows_of(g.D));
  auto go = [&](auto in, auto h) {
    typedef decltype(in) In;
    typedef decltype(h) H;
    auto kern = [&](auto nv) {
      constexpr int NV = decltype(nv)::value;
      if constexpr (BACKWARD)
        hipLaunchKernelGGL((join_backward_kernel<In, H, NV>), grid, block, 0, st, g);
      else
        hipLaunchKernelGGL((join_kernel<In, H, NV>), grid, block, 0, st, g);
    };
    if (g.D <= 8 * kMost)
      kern(std::integral_constant<int, 1>());
    else
      kern(std::integral_constant<int, 2>());
    return launch_status(BACKWARD ? "smat_block_join_backward" : "smat_block_join");
  };
  if (dtype == SMAT_BF16) return h_dtype == SMAT_F32 ? go(bf16(), float()) : go(bf16(), bf16());
  if (dtype == SMAT_F16) return h_dtype == SMAT_F32 ? go(f16(), float()) : go(f16(), f16());
  return go(float(), float());
}

static int check(const char* who, int dtype, int h_dtype, const Args& g, float p) {
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
  SMAT_REQUIRE(g.eps >= 0.f && p >= 0.f && p < 1.f && (p == 0.f || g.seed), SMAT_EINVAL,
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
  g.keep = (float)(1.0 / (1.0 - p));
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
  const int rc = check(who, dtype, h_dtype, g, (float)p);
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
  return grid_of(rows, D, true) * rows_of(D) * 12 * D;
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
  const int rc = check(who, dtype, h_dtype, g, (float)p);
  if (rc) return rc;
  if (rows == 0) return SMAT_OK;
  SMAT_REQUIRE(f && h && factors && ((uintptr_t)factors & 7) == 0 && df && dh_out && (!gate || (z && dz)) && (!dx || pre),
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
  const int groups = (int)(need / (12 * D));
  hipLaunchKernelGGL(join_sums_kernel, dim3((3 * D + 15) / 16), dim3(256), 0, st, g.part, groups, D,
                     dpost, ds, dpre);
  return launch_status(who);
}
