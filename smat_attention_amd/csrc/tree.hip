// Drafted trees over the decoder's cache (SmatDecoder.tree_step / tree_state): the
// tokens of a tree are read against the cache of one prefix, each node seeing the
// prefix, its ancestors and itself.  For node j at level l (a root is at level 0)
//
//   N_j = phi_j (S + U[(i + l) mod B]) + sum_a (phi_j . psi_a) vb_a,  out_j = N_j[:-1] / N_j[-1]
//
// over the ancestors a of j and j itself: what step-by-step decoding of j's path
// gives, with S read once and each level's type row U_h once.
//
// Bound by reading the tables (r p fp32 a level and sequence).  A wave owns 15 value
// columns and the normaliser's, so its division needs no other wave; it adds S and
// U_h in registers, the next level's U_h in flight meanwhile, and multiplies the
// level's nodes by the sum on bf16 MFMA in three terms (fp32's 24 bits; two for the
// features in fp16, three in fp32).  What every level needs of the nodes, their Phi
// rows and all scores phi_j . psi_a, is formed once a workgroup, in LDS.  The masked
// scores meet vb on MFMA too; a vb that is not finite is left out there, where it would
// meet other branches' zeros, and added to its descendants alone.  16 trees of 64 nodes
// and 8 heads of 128: 35 us, 2.2 TB/s (a chain of levels: sum, split, products, store),
// the accepted paths' states 9.
#include "delta_common.hpp"

namespace smat {
namespace tr {

using dl::Frag;
using dl::load4;
using dl::mul;
using dl::split;

constexpr int kMaxNodes = 64;
constexpr int kMaxWaves = 5;       // half of the ceil(143 / 15) column tiles

struct Args {
  const int64_t* anc;      // (trees, M): bit a of word j: a is j or an ancestor of j
  const int32_t* order;    // (trees, M): nodes by level, unused ones last
  const int32_t* lstart;   // (trees, M + 1): first of each level in order
  const int32_t* ahead;    // (requests): tokens past `step`; or null
  int nb, trees, requests, M, levels, B, r, p;
  int64_t step;
  int64_t q_sb, q_st, k_sb, k_st, v_sb, v_st;
};

constexpr int kScLd = kMaxNodes + 4;
// LDS: Phi's fragments by place in the order, Psi's, the scores, and each wave's vb
// columns.
template <typename In, int RB> constexpr int tree_lds(int W) {
  return 2 * dl::Terms<In>::in * 4 * RB * dl::kFrag * 2 + kMaxNodes * kScLd * 4 +
         W * kMaxNodes * 16 * 4;
}

template <typename In, int RB>
__global__ __launch_bounds__(64 * kMaxWaves) void tree_step_kernel(
    const In* __restrict__ phi, const In* __restrict__ psi, const In* __restrict__ vb,
    const float* __restrict__ S, const float* __restrict__ U, float* __restrict__ out, Args g,
    bool qvec, bool kvec) {
  constexpr int NT = dl::Terms<In>::in, FP = 4 * RB * dl::kFrag;
  extern __shared__ __align__(16) bf16 lds[];
  bf16 *ph = lds, *ps = ph + NT * FP;
  float* sc = reinterpret_cast<float*>(ps + NT * FP);          // [place j][node a]
  const int s = blockIdx.x, w = dl::uniform_wave(), W = blockDim.x >> 6;
  float* vl = sc + kMaxNodes * kScLd + w * kMaxNodes * 16;     // [node a][lane's column]
  const int lane = lane_id(), m = lane & 15, gq = lane >> 4;
  const int tree = g.trees == 1 ? 0 : s / (g.nb / g.trees);
  const int64_t* anc = g.anc + (int64_t)tree * g.M;
  const int32_t* order = g.order + (int64_t)tree * g.M;
  const int32_t* lstart = g.lstart + (int64_t)tree * (g.M + 1);
  const int nval = g.p - 1, used = lstart[g.levels];
  // value columns v0 .. v0 + 14, then p - 1 (a wave past the last tile: p - 1 alone)
  const int v0 = (blockIdx.y * W + w) * 15;
  const bool mine = m < 15 && v0 + m < nval;
  const int col = mine ? v0 + m : nval;
  const int64_t at = g.step + (g.ahead ? max(0, g.ahead[s / (g.nb / g.requests)]) : 0);
  const uint32_t M1 = g.M - 1;

  // In issue order: vb's columns, Phi and Psi rows, then the tables, which arrive while
  // the scores are formed.
  // lane = node: its word; lane = place: the node there and its word; lane = level: its start
  const uint64_t word = (uint64_t)anc[min((uint32_t)lane, M1)];
  const int ord = order[min((uint32_t)lane, M1)], begin = lstart[min(lane, g.levels)];
  const uint64_t path = (uint64_t)anc[ord];
  float vr[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    vr[i] = to_f32(vb[(int64_t)s * g.v_sb + (int64_t)min((uint32_t)(4 * i + gq), M1) * g.v_st + col]);
  // tile u < 4: Phi's places 16 u .., else Psi's nodes 16 (u - 4) ..
  const int tiles = (g.M + 15) / 16;
  for (int u = w; u < 8; u += W) {
    const int t = u & 3;
    if (t >= tiles) continue;
    const uint32_t place = min((uint32_t)(16 * t + m), M1);
    const bool q = u < 4;
    const In* row = q ? phi + (int64_t)s * g.q_sb + (int64_t)__shfl(ord, (int)place) * g.q_st
                      : psi + (int64_t)s * g.k_sb + (int64_t)place * g.k_st;
    f32x4 x[RB][2];
#pragma unroll
    for (int kb = 0; kb < RB; ++kb)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = 32 * kb + 16 * h + 4 * gq;
        x[kb][h] = load4(row + c, g.r - c, q ? qvec : kvec);
      }
#pragma unroll
    for (int kb = 0; kb < RB; ++kb)
      dl::store_frag<NT>((q ? ph : ps) + (t * RB + kb) * dl::kFrag, FP, split<NT>(x[kb][0], x[kb][1]));
  }
  // rows past r read the last one; their features are zero
  uint32_t off[2 * RB];
#pragma unroll
  for (int mt = 0; mt < 2 * RB; ++mt) off[mt] = (uint32_t)(16 * mt + 4 * gq) * g.p + col;
  const uint32_t last = (uint32_t)(g.r - 1) * g.p + col;
  auto load_table = [&](f32x4* x, const float* p) {
#pragma unroll
    for (int mt = 0; mt < 2 * RB; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[mt][i] = p[min(off[mt] + i * (uint32_t)g.p, last)];
  };
  auto table = [&](int l) {
    return U + ((int64_t)s * g.B + (at + l) % g.B) * g.r * g.p;
  };
  f32x4 St[2 * RB], Ut[2 * RB];
  load_table(St, S + (int64_t)s * g.r * g.p);
  load_table(Ut, table(min((int)blockIdx.z, max(g.levels - 1, 0))));

  // this wave's columns of vb; an unused node's are zero
  const uint64_t in_use = __ballot(word != 0 && lane < g.M);
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int a = 4 * i + gq;
    const float y = (in_use >> a) & 1 ? vr[i] : 0.f;
    vl[a * 16 + m] = y;
    odd |= !(fabsf(y) < INFINITY);
  }
  odd = __any(odd);
  lds_barrier();                                   // Phi and Psi; the tables stay in flight
  for (int t = w; t < tiles * tiles; t += W) {
    const int jt = t / tiles, ta = t % tiles;
    f32x4 x = zero4();
#pragma unroll
    for (int kb = 0; kb < RB; ++kb)                // place in the lane, a in registers
      x = dl::mul_inputs(x, dl::load_frag<NT>(ps + (ta * RB + kb) * dl::kFrag, FP),
                         dl::load_frag<NT>(ph + (jt * RB + kb) * dl::kFrag, FP));
    *reinterpret_cast<f32x4*>(sc + (16 * jt + m) * kScLd + 16 * ta + 4 * gq) = x;
  }
  lds_barrier();
  Frag<NT> vf[2];
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    f32x4 x[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int a = 32 * kb + 16 * h + 4 * gq + i;
        const float y = a < g.M ? vl[a * 16 + m] : 0.f;
        x[h][i] = fabsf(y) < INFINITY ? y : 0.f;
      }
    vf[kb] = split<NT>(x[0], x[1]);
  }

  for (int l = blockIdx.z; l < g.levels; l += gridDim.z) {
    const int n0 = __builtin_amdgcn_readlane(begin, l);
    const int n1 = l + 1 < g.levels ? __builtin_amdgcn_readlane(begin, l + 1) : used;
    if (n0 >= n1) break;                           // this tree has fewer levels
    Frag<3> tb[RB];
#pragma unroll
    for (int kb = 0; kb < RB; ++kb)
      tb[kb] = split<3>(St[2 * kb] + Ut[2 * kb], St[2 * kb + 1] + Ut[2 * kb + 1]);
    load_table(Ut, table(min(l + (int)gridDim.z, g.levels - 1)));   // (no branch: the last again)
    for (int n = n0; n < n1; n += 16) {
      const int j = min(n + m, n1 - 1);
      const uint64_t mask = __shfl((unsigned long long)path, j);
      f32x4 acc = zero4();
#pragma unroll
      for (int kb = 0; kb < RB; ++kb)              // column in the lane, places 4 gq + i
        acc = mul(acc,
                  dl::load_frag<NT>(ph + ((j >> 4) * RB + kb) * dl::kFrag, FP, gq * 16 + (j & 15)),
                  tb[kb]);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        if (32 * kb < g.M) {
          f32x4 x[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int a = 32 * kb + 16 * h + 4 * gq;
            const f32x4 y = *reinterpret_cast<const f32x4*>(sc + j * kScLd + a);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[h][i] = (mask >> (a + i)) & 1 ? y[i] : 0.f;
          }
          acc = mul(acc, split<3>(x[0], x[1]), vf[kb]);
        }
      if (odd) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ji = min(n + 4 * gq + i, n1 - 1);
          for (uint64_t left = __shfl((unsigned long long)path, ji); left; left &= left - 1) {
            const int a = __ffsll((unsigned long long)left) - 1;
            const float y = vl[a * 16 + m];
            if (!(fabsf(y) < INFINITY)) acc[i] += sc[ji * kScLd + a] * y;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float den = __shfl(acc[i], gq * 16 + 15);
        const int ji = n + 4 * gq + i, node = __shfl(ord, min(ji, n1 - 1));
        if (mine && ji < n1) out[((int64_t)s * g.M + node) * nval + col] = acc[i] / den;
      }
    }
  }
  if (blockIdx.z == 0)                             // unused nodes read nothing and give zeros
    for (int j0 = used; j0 < g.M; j0 += 4) {
      const int node = __shfl(ord, min(j0 + gq, (int)M1));
      if (mine && j0 + gq < g.M) out[((int64_t)s * g.M + node) * nval + col] = 0.f;
    }
}

// S' = S + sum of psi_a vb_a^T over the accepted path of each request, ancestors in
// order, eight at a time through LDS (their rows loaded together); `ahead` moves by the
// path's length.
constexpr int kElems = 8;          // elements of S a thread
constexpr int kBatch = 8;          // ancestors a round

template <typename In>
__global__ __launch_bounds__(256) void tree_state_kernel(
    const In* __restrict__ psi, const In* __restrict__ vb, const float* __restrict__ S,
    float* __restrict__ So, const int32_t* __restrict__ nodes, int32_t* ahead, Args g) {
  __shared__ float sp[kBatch][128], sv[kBatch][144];
  const int s = blockIdx.x, tid = threadIdx.x;
  const int per = g.nb / g.requests, req = s / per;
  const int tree = g.trees == 1 ? 0 : s / (g.nb / g.trees);
  const int node = nodes[req];
  const uint64_t path =
      node >= 0 && node < g.M ? (uint64_t)g.anc[(int64_t)tree * g.M + node] : 0;
  const int rp = g.r * g.p;
  const int64_t base = (int64_t)s * rp;
  float x[kElems];
  int row[kElems], col[kElems];
#pragma unroll
  for (int j = 0; j < kElems; ++j) {
    const int e = (blockIdx.y * kElems + j) * 256 + tid;
    row[j] = min(e, rp - 1) / g.p;
    col[j] = min(e, rp - 1) - row[j] * g.p;
    x[j] = S[base + min(e, rp - 1)];
  }
  const In* pr = psi + (int64_t)s * g.k_sb + min(tid, g.r - 1);
  const In* vr = vb + (int64_t)s * g.v_sb + min(tid, g.p - 1);
  uint64_t left = path;
  while (left) {
    int n = 0, at = 0;
    float a[kBatch], b[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {             // past the path's end: the last one again
      if (left) {
        at = __ffsll((unsigned long long)left) - 1;
        left &= left - 1;
        ++n;
      }
      a[i] = to_f32(pr[(int64_t)at * g.k_st]);
      b[i] = to_f32(vr[(int64_t)at * g.v_st]);
    }
    __syncthreads();                               // the last round's are read
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (tid < g.r) sp[i][tid] = a[i];
      if (tid < g.p) sv[i][tid] = b[i];
    }
    __syncthreads();
    for (int i = 0; i < n; ++i)
#pragma unroll
      for (int j = 0; j < kElems; ++j) x[j] += sp[i][row[j]] * sv[i][col[j]];
  }
#pragma unroll
  for (int j = 0; j < kElems; ++j) {
    const int e = (blockIdx.y * kElems + j) * 256 + tid;
    if (e < rp) So[base + e] = x[j];
  }
  if (ahead && blockIdx.y == 0 && tid == 0 && s % per == 0)
    ahead[req] += __popcll((unsigned long long)path);
}

static int check(const char* who, int dtype, const Args& g) {
  SMAT_REQUIRE(dtype == SMAT_BF16 || dtype == SMAT_F16 || dtype == SMAT_F32, SMAT_EINVAL,
               "%s: unknown dtype %d", who, dtype);
  SMAT_REQUIRE(g.nb >= 0 && g.trees >= 1 && g.requests >= 1 && g.nb % g.trees == 0 &&
                   g.nb % g.requests == 0,
               SMAT_EINVAL, "%s: %d trees and %d requests must divide nb=%d", who, g.trees,
               g.requests, g.nb);
  SMAT_REQUIRE(g.M >= 1 && g.M <= kMaxNodes, SMAT_EUNSUPPORTED, "%s: %d nodes, at most %d", who,
               g.M, kMaxNodes);
  SMAT_REQUIRE(g.r >= 1 && g.r <= kMaxR && g.p >= 2 && g.p <= kMaxP, SMAT_EUNSUPPORTED,
               "%s: r=%d p=%d beyond r<=%d, 2<=p<=%d", who, g.r, g.p, kMaxR, kMaxP);
  // a grid has less than 2^32 threads along an axis
  SMAT_REQUIRE(g.nb < (1 << 23), SMAT_EUNSUPPORTED, "%s: nb=%d must stay below 2^23", who, g.nb);
  return SMAT_OK;
}

}  // namespace tr
}  // namespace smat

extern "C" int smat_tree_step(int dtype, const void* phi, const void* psi, const void* vb,
                              const float* S, const float* U, float* out, const int64_t* anc,
                              const int32_t* order, const int32_t* lstart, const int32_t* ahead,
                              int nb, int trees, int requests, int M, int levels, int B, int r,
                              int p, int64_t step, int64_t q_sb, int64_t q_st, int64_t k_sb,
                              int64_t k_st, int64_t v_sb, int64_t v_st, void* stream) {
  using namespace smat;
  using namespace smat::tr;
  clear_error();
  const char* who = "smat_tree_step";
  const Args g = {anc, order, lstart, ahead, nb, trees, requests, M, levels, B, r, p, step,
                  q_sb, q_st, k_sb, k_st, v_sb, v_st};
  const int rc = check(who, dtype, g);
  if (rc) return rc;
  SMAT_REQUIRE(levels >= 0 && levels <= M && B >= 1 && step >= 0, SMAT_EINVAL,
               "%s: bad sizes (levels=%d B=%d step=%lld)", who, levels, B, (long long)step);
  if (nb == 0) return SMAT_OK;
  SMAT_REQUIRE(phi && psi && vb && S && U && out && anc && order && lstart, SMAT_EINVAL,
               "%s: null pointer", who);
  // a workgroup takes half of the column tiles (a third while sequences are few); its waves
  // walk every z-th level, z as large as leaves the GPU full
  const int tiles = (p - 1 + 14) / 15;
  const int W = nb < 64 ? (tiles + 2) / 3 : (tiles + 1) / 2;
  int z = (int)(2048 / ((int64_t)nb * tiles));
  z = z < 1 ? 1 : z > levels ? (levels > 0 ? levels : 1) : z;
  return dl::dispatch(dtype, r, [&](auto in, auto rb) {
    typedef decltype(in) In;
    constexpr int eb = sizeof(In), RB = decltype(rb)::value;
    const int lds = tree_lds<In, RB>(W);
    auto kern = tree_step_kernel<In, RB>;
    static uint64_t done;
    dl::allow_lds(kern, tree_lds<In, RB>(kMaxWaves), done);
    hipLaunchKernelGGL(kern, dim3(nb, (tiles + W - 1) / W, z), dim3(64 * W), lds,
                       (hipStream_t)stream, (const In*)phi, (const In*)psi, (const In*)vb, S, U,
                       out, g, dl::vec4_ok(phi, q_sb, q_st, eb), dl::vec4_ok(psi, k_sb, k_st, eb));
    return launch_status(who);
  });
}

extern "C" int smat_tree_state(int dtype, const void* psi, const void* vb, const float* S,
                               float* S_out, const int64_t* anc, const int32_t* nodes,
                               int32_t* ahead, int nb, int trees, int requests, int M, int r,
                               int p, int64_t k_sb, int64_t k_st, int64_t v_sb, int64_t v_st,
                               void* stream) {
  using namespace smat;
  using namespace smat::tr;
  clear_error();
  const char* who = "smat_tree_state";
  Args g = {};
  g.anc = anc;
  g.nb = nb;
  g.trees = trees;
  g.requests = requests;
  g.M = M;
  g.r = r;
  g.p = p;
  g.k_sb = k_sb;
  g.k_st = k_st;
  g.v_sb = v_sb;
  g.v_st = v_st;
  const int rc = check(who, dtype, g);
  if (rc) return rc;
  if (nb == 0) return SMAT_OK;
  SMAT_REQUIRE(psi && vb && S && S_out && anc && nodes, SMAT_EINVAL, "%s: null pointer", who);
  SMAT_REQUIRE(S != S_out, SMAT_EINVAL, "%s: S and S_out must differ", who);
  const dim3 grid(nb, (r * p + 256 * kElems - 1) / (256 * kElems));
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto in) {
    typedef decltype(in) In;
    hipLaunchKernelGGL(tree_state_kernel<In>, grid, dim3(256), 0, st, (const In*)psi,
                       (const In*)vb, S, S_out, nodes, ahead, g);
    return launch_status(who);
  };
  if (dtype == SMAT_BF16) return go(bf16());
  if (dtype == SMAT_F16) return go(f16());
  return go(float());
}
