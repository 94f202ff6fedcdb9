// One token of the gated delta rule for a batch of sequences (gated_delta_step):
//   S' = a S + k u^T,  u = b (v - a S^T k),  o = scale S'^T q = scale (a S^T q + (q.k) u)
//
// A bandwidth kernel: S is read once and S' written once.  Both column sums, S^T k
// and S^T q, come from one pass over the rows in registers, so that one exchange
// through LDS settles u, o and the update.  A workgroup takes 4 CL columns; thread
// (row group, column lane) holds every RG-th row of four columns, all loaded before
// the exchange.  Columns do not mix, so S' may be S.
#include "delta_common.hpp"

namespace smat {
namespace dl {

constexpr int kStepThreads = 256;

template <typename In, int CL, bool VEC>
__global__ __launch_bounds__(kStepThreads) void delta_step_kernel(
    const In* __restrict__ q, const In* __restrict__ k, const In* __restrict__ v,
    const float* __restrict__ logA, const float* __restrict__ beta, const float* S_in,
    float* S_out, In* __restrict__ o, int group, int r, int p, float scale, int64_t q_sb,
    int64_t k_sb, int64_t v_sb, int64_t a_sb, int64_t b_sb) {
  constexpr int RG = kStepThreads / CL, ROWS = kMaxR / RG, WAVES = kStepThreads / 64;
  __shared__ float sq[kMaxR], sk[kMaxR];
  __shared__ __align__(16) f32x4 rk[WAVES][CL], rq[WAVES][CL];
  __shared__ float rqk[WAVES];
  const int64_t s = blockIdx.x;
  const int tid = threadIdx.x, cl = tid % CL, rg = tid / CL;
  const int c0 = (blockIdx.y * CL + cl) * 4, nv = min(4, p - c0);
  const float* Sb = S_in + s * r * p;
  float* Ob = S_out + s * r * p;

  f32x4 S[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int row = rg + j * RG;
    if constexpr (VEC) {
      // a clamped address keeps every load in flight; rows and columns past the
      // end are multiplied by zero features or not stored
      const f32x4 x = *reinterpret_cast<const f32x4*>(Sb + (int64_t)min(row, r - 1) * p +
                                                      min(c0, p - 4));
      S[j] = row < r ? x : zero4();
    } else {
      S[j] = row < r ? load4(Sb + (int64_t)row * p + c0, nv, false) : zero4();
    }
  }
  if (tid < kMaxR) {
    const int64_t ks = s / group;
    sq[tid] = tid < r ? to_f32(q[ks * q_sb + tid]) : 0.f;
    sk[tid] = tid < r ? to_f32(k[ks * k_sb + tid]) : 0.f;
  }
  const float a = expf(logA[s * a_sb]), b = beta[s * b_sb];
  const f32x4 vv = load4(v + s * v_sb + c0, nv, false);
  __syncthreads();
  f32x4 ks4 = zero4(), qs4 = zero4();
  float qk = 0.f;
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const float kr = sk[rg + j * RG], qr = sq[rg + j * RG];
    ks4 += kr * S[j];
    qs4 += qr * S[j];
    qk += kr * qr;
  }
#pragma unroll
  for (int d = CL; d < 64; d <<= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ks4[i] += __shfl_xor(ks4[i], d);
      qs4[i] += __shfl_xor(qs4[i], d);
    }
    qk += __shfl_xor(qk, d);
  }
  const int w = wave_id();
  if (lane_id() < CL) {
    rk[w][cl] = ks4;
    rq[w][cl] = qs4;
    if (cl == 0) rqk[w] = qk;
  }
  __syncthreads();
  ks4 = rk[0][cl];
  qs4 = rq[0][cl];
  qk = rqk[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) {
    ks4 += rk[i][cl];
    qs4 += rq[i][cl];
    qk += rqk[i];
  }
  const f32x4 u = b * (vv - a * ks4);
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int row = rg + j * RG;
    if (row < r) store4(Ob + (int64_t)row * p + c0, a * S[j] + sk[row] * u, nv, VEC);
  }
  if (rg == 0) store4(o + s * p + c0, scale * (a * qs4 + qk * u), nv, false);
}

template <typename In>
static int step(const void* q, const void* k, const void* v, const float* logA, const float* beta,
                const float* S_in, float* S_out, void* o, int nb, int group, int r, int p,
                float scale, int64_t q_sb, int64_t k_sb, int64_t v_sb, int64_t a_sb, int64_t b_sb,
                hipStream_t st) {
  auto go = [&](auto kern, int CL) {
    hipLaunchKernelGGL(kern, dim3(nb, (p + 4 * CL - 1) / (4 * CL)), dim3(kStepThreads), 0, st,
                       (const In*)q, (const In*)k, (const In*)v, logA, beta, S_in, S_out, (In*)o,
                       group, r, p, scale, q_sb, k_sb, v_sb, a_sb, b_sb);
  };
  // 128 columns a workgroup while that leaves two a CU, else 32
  const bool wide = (int64_t)nb * ((p + 127) / 128) >= 512;
  const bool vec = p % 4 == 0 && aligned16(S_in) && aligned16(S_out);
  if (vec)
    wide ? go(delta_step_kernel<In, 32, true>, 32) : go(delta_step_kernel<In, 8, true>, 8);
  else
    wide ? go(delta_step_kernel<In, 32, false>, 32) : go(delta_step_kernel<In, 8, false>, 8);
  return launch_status("smat_delta_step");
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
  hipStream_t st = (hipStream_t)stream;
  const int group = nb / nbk;
  if (dtype == SMAT_BF16)
    return step<bf16>(q, k, v, logA, beta, S_in, S_out, out, nb, group, r, p, scale, q_sb, k_sb,
                      v_sb, a_sb, b_sb, st);
  if (dtype == SMAT_F16)
    return step<f16>(q, k, v, logA, beta, S_in, S_out, out, nb, group, r, p, scale, q_sb, k_sb,
                     v_sb, a_sb, b_sb, st);
  if (dtype == SMAT_F32)
    return step<float>(q, k, v, logA, beta, S_in, S_out, out, nb, group, r, p, scale, q_sb, k_sb,
                       v_sb, a_sb, b_sb, st);
  set_error("%s: unknown dtype %d", who, dtype);
  return SMAT_EINVAL;
}
