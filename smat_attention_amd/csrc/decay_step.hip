// A token of linear attention with a decay for each head, for a batch of sequences
// (head_decay_step):  S' = a S + k v^T,  o = scale S'^T q.
//
// A bandwidth kernel: the state is read once and written once.  A workgroup takes 4 CL
// columns; thread (row group, column lane) holds every RG-th row of four columns, all
// loaded before the first use.  Only o waits for the other rows, in one exchange through
// LDS.  Columns do not mix, so S' may be S.  2048 sequences of 128 x 128: 43 us, 6.2 TB/s (the
// state partly stays in the last cache); 8 of 64 x 64: 3.6, a launch and two trips to memory.
#include "decay_walk.hpp"

namespace smat {
namespace hd {

constexpr int kStepThreads = 256;

struct Token {
  const void *q, *k, *v;
  const float *logA, *S_in;
  float* S_out;
  void* o;
  int group, heads, r, p;
  float scale;
  int64_t q_sb, k_sb, v_sb;
};

template <typename In, int CL, bool VEC>
__global__ __launch_bounds__(kStepThreads, 4) void decay_token_kernel(Token g) {
  constexpr int RG = kStepThreads / CL, ROWS = kMaxD / RG, WAVES = kStepThreads / 64;
  __shared__ float sq[kMaxD], sk[kMaxD];
  __shared__ __align__(16) f32x4 so[WAVES][CL];
  const int64_t s = blockIdx.x, ks = s / g.group;
  const int tid = threadIdx.x, cl = tid % CL, rg = tid / CL;
  const int c0 = (blockIdx.y * CL + cl) * 4, nv = min(4, g.p - c0);
  const float* Sb = g.S_in + s * g.r * g.p;
  f32x4 S[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int row = rg + j * RG;
    if constexpr (VEC) {
      // clamped addresses keep every load in flight; what is past the end is not stored
      S[j] = *reinterpret_cast<const f32x4*>(Sb + (int64_t)min(row, g.r - 1) * g.p +
                                             min(c0, g.p - 4));
    } else {
      S[j] = row < g.r ? dl::load4(Sb + (int64_t)row * g.p + c0, nv, false) : zero4();
    }
  }
  if (tid < kMaxD) {
    const int a = min(tid, g.r - 1);
    const float x = to_f32(((const In*)g.q)[ks * g.q_sb + a]);
    const float y = to_f32(((const In*)g.k)[ks * g.k_sb + a]);
    sq[tid] = tid < g.r ? x : 0.f;
    sk[tid] = tid < g.r ? y : 0.f;
  }
  const In* vs = (const In*)g.v + s * g.v_sb;
  f32x4 v, o = zero4();
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_f32(vs[min(c0 + i, g.p - 1)]);
  const float a = expf(g.logA[s % g.heads]);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int row = rg + j * RG;
    if (row < g.r) {
      S[j] = a * S[j] + sk[row] * v;
      o += sq[row] * S[j];
      dl::store4(g.S_out + (s * g.r + row) * g.p + c0, S[j], nv, VEC);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = dl::sum_rows<CL>(o[i]);
  if (lane_id() < CL) so[wave_id()][cl] = o;
  __syncthreads();
  if (rg == 0) {
    o = so[0][cl];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) o += so[i][cl];
    dl::store4((In*)g.o + s * g.p + c0, g.scale * o, nv, false);
  }
}

template <typename In> static int token(const Token& g, int nb, hipStream_t st) {
  auto go = [&](auto kern, int CL) {
    hipLaunchKernelGGL(kern, dim3(nb, (g.p + 4 * CL - 1) / (4 * CL)), dim3(kStepThreads), 0, st, g);
  };
  // 128 columns a workgroup while that leaves two a CU, else 32: few sequences give more
  // workgroups so, many read whole rows
  const bool wide = nb >= 512;
  const bool vec = g.p % 4 == 0 && aligned16(g.S_in) && aligned16(g.S_out);
  if (vec)
    wide ? go(decay_token_kernel<In, 32, true>, 32) : go(decay_token_kernel<In, 8, true>, 8);
  else
    wide ? go(decay_token_kernel<In, 32, false>, 32) : go(decay_token_kernel<In, 8, false>, 8);
  return launch_status("smat_head_decay_step");
}

}  // namespace hd
}  // namespace smat

extern "C" int smat_head_decay_step(int dtype, const void* q, const void* k, const void* v,
                                    const float* logA, const float* S_in, float* S_out, void* out,
                                    int nb, int nbk, int heads, int r, int p, float scale,
                                    int64_t q_sb, int64_t k_sb, int64_t v_sb, void* stream) {
  using namespace smat;
  using namespace smat::hd;
  clear_error();
  const char* who = "smat_head_decay_step";
  SMAT_REQUIRE(nb >= 0 && nbk >= 1 && heads >= 1 && nb % nbk == 0 && nb % heads == 0, SMAT_EINVAL,
               "%s: nbk=%d and heads=%d must divide nb=%d", who, nbk, heads, nb);
  SMAT_REQUIRE(r >= 1 && r <= kMaxD && p >= 1 && p <= kMaxD, SMAT_EUNSUPPORTED,
               "%s: r=%d p=%d must lie in 1..%d", who, r, p, kMaxD);
  SMAT_REQUIRE(dtype == SMAT_BF16 || dtype == SMAT_F16 || dtype == SMAT_F32, SMAT_EINVAL,
               "%s: unknown dtype %d", who, dtype);
  // a grid has less than 2^32 threads along an axis
  SMAT_REQUIRE(nb < (1 << 24), SMAT_EUNSUPPORTED, "%s: nb=%d must stay below 2^24", who, nb);
  if (nb == 0) return SMAT_OK;
  SMAT_REQUIRE(q && k && v && logA && S_in && S_out && out, SMAT_EINVAL, "%s: null pointer", who);
  const Token t = {q, k, v, logA, S_in, S_out, out, nb / nbk, heads, r, p, scale, q_sb, k_sb, v_sb};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SMAT_BF16) return token<bf16>(t, nb, st);
  if (dtype == SMAT_F16) return token<f16>(t, nb, st);
  return token<float>(t, nb, st);
}
