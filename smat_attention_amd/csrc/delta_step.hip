// A token, or a few, of the gated delta rule for a batch of sequences (gated_delta_step;
// gated_delta_scan of up to 16 tokens):
//   S' = a S + k u^T,  u = b (v - a S^T k),  o = scale S'^T q = scale (a S^T q + (q.k) u)
//
// A bandwidth kernel: the state is read once and written once, whatever the tokens.
// Both column sums of a token, S^T k and S^T q, come from one pass over the rows in
// registers, so that one exchange through LDS settles u, o and the update.  A workgroup
// takes 4 CL columns; thread (row group, column lane) holds every RG-th row of four
// columns, all loaded before the first exchange.  Columns do not mix, so S' may be S.
// 2048 sequences of 128 x 128: 43 us a token, 6.3 TB/s (the state partly stays in the
// last-level cache).  Seven tokens of 8 sequences of 64 x 64 take one launch of 9 us
// here; as a chunk they are 18 us of two dependent kernels.
#include "delta_common.hpp"

namespace smat {
namespace dl {

constexpr int kStepThreads = 256;

struct Tokens {
  const void *q, *k, *v;
  const float *logA, *beta, *S_in;   // S_in: null is zero
  float* S_out;                      // or null
  void* o;
  int T, group, r, p;
  float scale;
  int64_t q_sb, q_st, k_sb, k_st, v_sb, v_st, a_sb, a_st, b_sb, b_st, o_sb, o_st;
};

// ONE: a single token (less LDS and fewer registers, so more of the state in flight).
template <typename In, int CL, bool VEC, bool ONE>
__global__ __launch_bounds__(kStepThreads, ONE ? 4 : 2) void delta_tokens_kernel(Tokens g) {
  constexpr int RG = kStepThreads / CL, ROWS = kMaxR / RG, WAVES = kStepThreads / 64;
  constexpr int MOST = ONE ? 1 : kFewTokens, BUFS = ONE ? 1 : 2;
  __shared__ float sq[MOST][kMaxR], sk[MOST][kMaxR], sa[MOST], sb[MOST];
  __shared__ __align__(16) f32x4 sv[ONE ? 1 : MOST][ONE ? 1 : CL];
  __shared__ __align__(16) f32x4 rk[BUFS][WAVES][CL], rq[BUFS][WAVES][CL];
  __shared__ float rqk[BUFS][WAVES];
  const int T = ONE ? 1 : g.T;
  const int64_t s = blockIdx.x, ks = s / g.group;
  const int tid = threadIdx.x, cl = tid % CL, rg = tid / CL, w = wave_id();
  const int c0 = (blockIdx.y * CL + cl) * 4, nv = min(4, g.p - c0);
  const float* Sb = g.S_in ? g.S_in + s * g.r * g.p : nullptr;

  f32x4 S[ROWS];
  if (Sb) {
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int row = rg + j * RG;
      if constexpr (VEC) {
        // a clamped address keeps every load in flight; rows and columns past the
        // end are multiplied by zero features or not stored
        const f32x4 x = *reinterpret_cast<const f32x4*>(Sb + (int64_t)min(row, g.r - 1) * g.p +
                                                        min(c0, g.p - 4));
        S[j] = row < g.r ? x : zero4();
      } else {
        S[j] = row < g.r ? load4(Sb + (int64_t)row * g.p + c0, nv, false) : zero4();
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < ROWS; ++j) S[j] = zero4();
  }
  // four rows of q and k a thread in flight; those past the last token's are not kept
  constexpr int ROUND = ONE ? 1 : 4, STEP = kStepThreads / kMaxR;
  const int a0 = tid % kMaxR, ac = min(a0, g.r - 1);
  const In *qs = (const In*)g.q + ks * g.q_sb + ac, *kk = (const In*)g.k + ks * g.k_sb + ac;
  for (int t0 = tid / kMaxR; t0 < T; t0 += ROUND * STEP) {
    In xq[ROUND], xk[ROUND];
#pragma unroll
    for (int i = 0; i < ROUND; ++i) {
      const int t = min(t0 + i * STEP, T - 1);
      xq[i] = qs[t * g.q_st];
      xk[i] = kk[t * g.k_st];
    }
#pragma unroll
    for (int i = 0; i < ROUND; ++i)
      if (t0 + i * STEP < T) {
        sq[t0 + i * STEP][a0] = a0 < g.r ? to_f32(xq[i]) : 0.f;
        sk[t0 + i * STEP][a0] = a0 < g.r ? to_f32(xk[i]) : 0.f;
      }
  }
  // the tokens' gates and values too: a load inside the loop would be waited for in it
  const In* vs = (const In*)g.v + s * g.v_sb;
  auto values = [&](const In* row, int c) {        // columns past the last: the last one's
    f32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f32(row[min(c + i, g.p - 1)]);
    return x;
  };
  float a = 0.f, b = 0.f;
  f32x4 v = zero4();
  if constexpr (ONE) {
    a = expf(g.logA[s * g.a_sb]);
    b = g.beta[s * g.b_sb];
    v = values(vs, c0);
  } else {
    if (tid < T) {
      sa[tid] = expf(g.logA[s * g.a_sb + tid * g.a_st]);
      sb[tid] = g.beta[s * g.b_sb + tid * g.b_st];
    }
    for (int e = tid; e < T * CL; e += kStepThreads) {
      const int t = e / CL;
      sv[t][e % CL] = values(vs + t * g.v_st, (blockIdx.y * CL + e % CL) * 4);
    }
  }
  __syncthreads();
  for (int t = 0; t < T; ++t) {
    if constexpr (!ONE) {
      a = sa[t];
      b = sb[t];
      v = sv[t][cl];
    }
    f32x4 ks4 = zero4(), qs4 = zero4();
    float qk = 0.f;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const float kr = sk[t][rg + j * RG], qr = sq[t][rg + j * RG];
      ks4 += kr * S[j];
      qs4 += qr * S[j];
      qk += kr * qr;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ks4[i] = sum_rows<CL>(ks4[i]);
      qs4[i] = sum_rows<CL>(qs4[i]);
    }
    qk = sum_rows<CL>(qk);
    const int buf = ONE ? 0 : t & 1;                         // alternating: one barrier a token
    if (lane_id() < CL) {
      rk[buf][w][cl] = ks4;
      rq[buf][w][cl] = qs4;
      if (cl == 0) rqk[buf][w] = qk;
    }
    __syncthreads();
    ks4 = rk[buf][0][cl];
    qs4 = rq[buf][0][cl];
    qk = rqk[buf][0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
      ks4 += rk[buf][i][cl];
      qs4 += rq[buf][i][cl];
      qk += rqk[buf][i];
    }
    const f32x4 u = b * (v - a * ks4);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) S[j] = a * S[j] + sk[t][rg + j * RG] * u;
    if (rg == 0)
      store4((In*)g.o + s * g.o_sb + t * g.o_st + c0, g.scale * (a * qs4 + qk * u), nv, false);
  }
  if (g.S_out) {
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int row = rg + j * RG;
      if (row < g.r) store4(g.S_out + (s * g.r + row) * g.p + c0, S[j], nv, VEC);
    }
  }
}

template <typename In>
static int tokens(const char* who, const Tokens& g, int nb, hipStream_t st) {
  auto go = [&](auto kern, int CL) {
    hipLaunchKernelGGL(kern, dim3(nb, (g.p + 4 * CL - 1) / (4 * CL)), dim3(kStepThreads), 0, st, g);
  };
  // 128 columns a workgroup while that leaves two a CU, else 32
  const bool wide = (int64_t)nb * ((g.p + 127) / 128) >= 512;
  const bool vec = g.p % 4 == 0 && aligned16(g.S_in) && aligned16(g.S_out);
  auto cols = [&](auto one) {
    constexpr bool ONE = decltype(one)::value;
    if (vec)
      wide ? go(delta_tokens_kernel<In, 32, true, ONE>, 32)
           : go(delta_tokens_kernel<In, 8, true, ONE>, 8);
    else
      wide ? go(delta_tokens_kernel<In, 32, false, ONE>, 32)
           : go(delta_tokens_kernel<In, 8, false, ONE>, 8);
  };
  if (g.T == 1)
    cols(std::true_type());
  else
    cols(std::false_type());
  return launch_status(who);
}

int launch_tokens(const char* who, int dtype, const Geo& g, const void* q, const void* k,
                  const void* v, const float* logA, const float* beta, const float* S_in,
                  float* S_out, void* o, hipStream_t st) {
  // a grid has less than 2^32 threads along an axis
  SMAT_REQUIRE(g.nb < (1 << 24), SMAT_EUNSUPPORTED, "%s: nb=%d must stay below 2^24", who, g.nb);
  const Tokens t = {q, k, v, logA, beta, S_in, S_out, o, g.T, g.nb / g.nbk, g.r, g.p, g.scale,
                    g.q_sb, g.q_st, g.k_sb, g.k_st, g.v_sb, g.v_st, g.a_sb, g.a_st, g.b_sb,
                    g.b_st, (int64_t)g.T * g.p, g.p};
  if (dtype == SMAT_BF16) return tokens<bf16>(who, t, g.nb, st);
  if (dtype == SMAT_F16) return tokens<f16>(who, t, g.nb, st);
  return tokens<float>(who, t, g.nb, st);
}

}  // namespace dl
}  // namespace smat

extern "C" int smat_delta_step(int dtype, const void* q, const void* k, const void* v,
                               const float* logA, const float* beta, const float* S_in,
                               float* S_out, void* out, int nb, int nbk, int r, int p, float scale,
                               int64_t q_sb, int64_t k_sb, int64_t v_sb, int64_t a_sb,
                               int64_t b_sb, void* stream) {
  using namespace smat;
  using namespace smat::dl;
  clear_error();
  const char* who = "smat_delta_step";
  SMAT_REQUIRE(nb >= 0 && nbk >= 1 && nb % nbk == 0, SMAT_EINVAL,
               "%s: nbk=%d must divide nb=%d", who, nbk, nb);
  SMAT_REQUIRE(r >= 1 && r <= dl::kMaxR && p >= 1 && p <= dl::kMaxP, SMAT_EUNSUPPORTED,
               "%s: r=%d p=%d beyond r<=%d, p<=%d", who, r, p, dl::kMaxR, dl::kMaxP);
  if (nb == 0) return SMAT_OK;
  SMAT_REQUIRE(q && k && v && logA && beta && S_in && S_out && out, SMAT_EINVAL,
               "%s: null pointer", who);
  SMAT_REQUIRE(dtype == SMAT_BF16 || dtype == SMAT_F16 || dtype == SMAT_F32, SMAT_EINVAL,
               "%s: unknown dtype %d", who, dtype);
  Geo g = {};
  g.nb = nb;
  g.nbk = nbk;
  g.T = 1;
  g.r = r;
  g.p = p;
  g.scale = scale;
  g.q_sb = q_sb;
  g.k_sb = k_sb;
  g.v_sb = v_sb;
  g.a_sb = a_sb;
  g.b_sb = b_sb;
  return launch_tokens(who, dtype, g, q, k, v, logA, beta, S_in, S_out, out, (hipStream_t)stream);
}
