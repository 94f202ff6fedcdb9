// Linear attention with a decay for each head: the entry points over whole sequences
// (head_decay_scan and its gradient).  The mathematics and the walk are in decay_walk.hpp.
//
// A workgroup walks a whole segment where sequences give enough workgroups.  Where they do
// not, segments are cut into runs: a first pass takes every run but the last from the zero
// state for its end E, the carry adds them up, S <- a^(tokens of the run) S + E, and the
// second pass takes every run from its own state.
#include <initializer_list>

#include "decay_walk.hpp"

namespace smat {
namespace hd {

// The states entering the runs of a segment, from init or from zero; `rev`: the runs in
// turned order.  Every element on its own, sixteen runs' E in flight; bound by E in and the
// states out: 16 sequences of 32 runs of 128 x 128 in 6 segments 11.6 us, 5.5 TB/s (one element a
// thread 20), and where runs are many and elements few by a batch's latency: 8 of 64 runs 16.
// T: one element, or four (a wave then reads 1 KB of a run).
template <typename T, int BLOCK>
__global__ __launch_bounds__(BLOCK) void decay_carry_kernel(Walk g, const T* __restrict__ init,
                                                            const T* __restrict__ E,
                                                            T* __restrict__ start) {
  constexpr int U = 16;
  __shared__ float decay[BLOCK];                   // of the tokens of a block of runs
  const int s = blockIdx.x, seg = blockIdx.z;
  const int64_t rp = (int64_t)g.r * g.p / (sizeof(T) / 4);
  const int64_t e = (int64_t)blockIdx.y * BLOCK + threadIdx.x;
  const int r0 = g.segrun ? g.segrun[seg] : 0, r1 = g.segrun ? g.segrun[seg + 1] : g.nruns;
  auto run_at = [&](int n) { return g.rev ? r0 + r1 - 1 - n : n; };
  const int64_t step = g.nb * rp;                  // between a sequence's runs
  const T* E0 = E + s * rp + min(e, rp - 1);
  T* start0 = start + s * rp + e;
  T S = {};
  if (init && e < rp) S = init[((int64_t)seg * g.nb + s) * rp + e];
  for (int b = r0; b < r1; b += BLOCK) {
    __syncthreads();
    if (b + (int)threadIdx.x < r1) {
      const int i = run_at(b + threadIdx.x);
      int tokens;
      if (g.runs) {
        const int first = g.runs[4 * i], last = g.runs[4 * i + 1];
        tokens = 0;
        if (last > first)
          tokens = g.chunks[2 * last - 2] + g.chunks[2 * last - 1] - g.chunks[2 * first];
      } else {
        tokens = (int)min((int64_t)(i + 1) * g.K * C, (int64_t)g.T) - i * g.K * C;
      }
      decay[threadIdx.x] = tokens ? (float)exp((double)g.logA[s % g.heads] * tokens) : 1.f;
    }
    __syncthreads();
    for (int n = b; n < min(b + BLOCK, r1); n += U) {
      T x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {                // a segment's last run has no E: another's
        x[u] = T{};
        if (r1 - r0 > 1) x[u] = E0[run_at(min(n + u, r1 - 2)) * step];
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (n + u < r1) {
          if (e < rp) start0[run_at(n + u) * step] = S;
          S = decay[n + u - b] * S + x[u];
        }
    }
  }
}

// out = the sum over a key head's value heads of fp32 rows, rounded once.  Bound by HBM: 16
// value heads of 8192 x 128 to 8 of bf16: 14 us, 6.0 TB/s (the rows partly lie in the last cache).
template <typename In>
__global__ __launch_bounds__(256) void decay_heads_kernel(const float* __restrict__ part,
                                                          In* __restrict__ out, int group,
                                                          int64_t n) {
  const int64_t ks = blockIdx.y;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n;
       i += (int64_t)gridDim.x * 1024) {
    const int nv = (int)(n - i < 4 ? n - i : 4);
    f32x4 x = zero4();
    for (int j = 0; j < group; ++j) x += dl::load4(part + (ks * group + j) * n + i, nv, n % 4 == 0);
    dl::store4(out + ks * n + i, x, nv, n % 4 == 0);
  }
}

// dlogA of a head: its parts of the three walks, in the same order every time.
__global__ __launch_bounds__(256) void decay_grad_kernel(const float* p0, const float* p1,
                                                         const float* p2, int W0, int W1, int W2,
                                                         int nruns, int nb, int heads,
                                                         float* __restrict__ dlogA) {
  const int h = blockIdx.x;
  const float* ps[3] = {p0, p1, p2};
  const int Ws[3] = {W0, W1, W2};
  const int64_t batch = nb / heads;
  double x = 0;
  for (int k = 0; k < 3; ++k)
    for (int64_t i = threadIdx.x; i < nruns * batch * Ws[k]; i += 256) {
      const int64_t rb = i / Ws[k];                // run, batch
      x += ps[k][(rb / batch * nb + rb % batch * heads + h) * Ws[k] + i % Ws[k]];
    }
  __shared__ double sum[256];
  sum[threadIdx.x] = x;
  __syncthreads();
  for (int d = 128; d > 0; d >>= 1) {
    if (threadIdx.x < d) sum[threadIdx.x] += sum[threadIdx.x + d];
    __syncthreads();
  }
  if (threadIdx.x == 0) dlogA[h] = (float)sum[0];
}

static int walk_all(int dtype, const Walks& g, bool out, int learn, hipStream_t st) {
  if (dtype == SMAT_BF16) return launch_walk<bf16>(g, out, learn, st);
  if (dtype == SMAT_F16) return launch_walk<f16>(g, out, learn, st);
  return launch_walk<float>(g, out, learn, st);
}

static int walk_any(int dtype, const Walk& g, bool out, int learn, hipStream_t st) {
  return walk_all(dtype, {{g}, 1}, out, learn, st);
}

// First pass and carry of a walk (k, v, rev and upd set): start from init.
static int carry(int dtype, const Walk& base, const float* init, float* E, float* start,
                 hipStream_t st) {
  Walk g = base;
  g.start = nullptr;
  g.fin = E;
  int rc = walk_any(dtype, g, false, kNone, st);
  if (rc) return rc;
  const int64_t rp = (int64_t)g.r * g.p;
  if (rp % 4 == 0 && aligned16(init) && aligned16(E) && aligned16(start))
    hipLaunchKernelGGL((decay_carry_kernel<f32x4, 64>), dim3(g.nb, (rp + 255) / 256, g.nseg),
                       dim3(64), 0, st, g, (const f32x4*)init, (const f32x4*)E, (f32x4*)start);
  else
    hipLaunchKernelGGL((decay_carry_kernel<float, 256>), dim3(g.nb, (rp + 255) / 256, g.nseg),
                       dim3(256), 0, st, g, init, E, start);
  return launch_status("smat_head_decay_scan: carry");
}

static int check(const char* who, int dtype, const Walk& g, int nbk, int r, int p,
                 std::initializer_list<int64_t> rows) {
  SMAT_REQUIRE(dtype == SMAT_BF16 || dtype == SMAT_F16 || dtype == SMAT_F32, SMAT_EINVAL,
               "%s: unknown dtype %d", who, dtype);
  SMAT_REQUIRE(g.nb >= 0 && nbk >= 1 && g.heads >= 1 && g.T >= 0 && g.T <= 0x7fffffff - C + 1 &&
                   g.nseg >= 1 && g.nch >= 0,
               SMAT_EINVAL, "%s: bad sizes (nb=%d nbk=%d heads=%d T=%d nseg=%d nch=%d)", who, g.nb,
               nbk, g.heads, g.T, g.nseg, g.nch);
  SMAT_REQUIRE(g.nb % nbk == 0 && g.nb % g.heads == 0, SMAT_EINVAL,
               "%s: nbk=%d and heads=%d must divide nb=%d", who, nbk, g.heads, g.nb);
  for (int64_t st : rows)
    SMAT_REQUIRE(g.T <= 1 || dl::near_rows(st), SMAT_EUNSUPPORTED,
                 "%s: rows %lld elements apart, not 0 to 2^23", who, (long long)st);
  SMAT_REQUIRE(r >= kMinD && r <= kMaxD && p >= kMinD && p <= kMaxD, SMAT_EUNSUPPORTED,
               "%s: r=%d p=%d must lie in %d..%d", who, r, p, kMinD, kMaxD);
  if (g.chunks || g.runs || g.segrun) {
    SMAT_REQUIRE(g.chunks && g.runs && g.segrun && g.nruns >= g.nseg, SMAT_EINVAL,
                 "%s: segments need the chunk, run and segment tables", who);
  } else {
    SMAT_REQUIRE(g.nseg == 1 && g.nch == (g.T + C - 1) / C, SMAT_EINVAL,
                 "%s: %d chunks for T=%d", who, g.nch, g.T);
    SMAT_REQUIRE(g.K >= 1 && g.nruns == (g.nch > 0 ? (g.nch + g.K - 1) / g.K : 1), SMAT_EINVAL,
                 "%s: %d runs of %d chunks for %d chunks", who, g.nruns, g.K, g.nch);
  }
  // a grid has less than 2^32 threads along its first axis and 65535 workgroups along others
  SMAT_REQUIRE(g.nb < (1 << 23) && g.nruns <= dl::kMaxGrid && g.nseg <= dl::kMaxGrid,
               SMAT_EUNSUPPORTED,
               "%s: nb=%d must stay below 2^23, %d segments and %d runs within %d", who, g.nb,
               g.nseg, g.nruns, dl::kMaxGrid);
  return SMAT_OK;
}

static int check_workspace(const char* who, const void* ws, int64_t got, int64_t need) {
  SMAT_REQUIRE(got >= need && (ws || need == 0) && ((uintptr_t)ws & 255) == 0, SMAT_EINVAL,
               "%s: workspace of %lld bytes, %lld needed (256-byte aligned)", who, (long long)got,
               (long long)need);
  return SMAT_OK;
}

struct Scratch {
  float *E, *start;        // the runs' ends and starts
  float *dq, *dk;          // rows of every value head, where they share key heads
  float* part[3];          // the parts of dlogA
};
static Scratch take(dl::Arena& ar, int64_t nb, int64_t nbk, int64_t T, int nseg, int64_t nruns,
                    int r, int p, bool backward, bool learn) {
  Scratch c = {};
  if (nruns > nseg) {
    c.E = ar.take<float>(nruns * nb * r * p);
    c.start = ar.take<float>(nruns * nb * r * p);
  }
  if (backward && nb > nbk) {
    c.dq = ar.take<float>(nb * T * r);
    c.dk = ar.take<float>(nb * T * r);
  }
  if (backward && learn)
    for (float*& x : c.part) x = ar.take<float>(nruns * nb * kMaxWaves);
  return c;
}

}  // namespace hd
}  // namespace smat

// Run length: of the lengths that cut the longest segment into 1 to 256 runs, the one whose
// passes take least by what their steps measure, in microseconds a chunk of a workgroup with
// its CU to itself: 1.6 + 0.7 RB with outputs, half as much again at 128 columns, 1.35 and 1.7
// times that where inputs have two and three terms, and 0.42 of it in the first pass.  Two
// workgroups on a CU take 1.45 times as long each, three (bf16, 64 columns) 1.9; more than fit
// follow one another.  The carry moves its states at 4 TB/s, and two launches more
// take 9.  (bf16, 8 sequences of 2048 chunks, r = p = 128: 7823 in two runs, 575 in 32, 466 in
// 64, 506 in 128; 32 of 128 chunks, 64 x 64: 350 whole, 84 in 8, 66 in 16, 67 in 22; 96 of 64
// chunks with gradients: 415 whole, 275 in 4, 244 in 8, 279 in 16; fp16, 12 of 157 chunks,
// 96 x 96: 141 in 16, 120 in 20, 120 in 40; fp32, 8 of 64 chunks, 128 x 128: 140 in 8, 88 in 16,
// 66 in 32; 4 of 16, 64 x 64: 90 whole, 46 in 4, 31 in 8.)
extern "C" int smat_head_decay_run_chunks(int dtype, int nb, int nch, const int32_t* lengths,
                                          const int32_t* times, int n, int r, int p) {
  using namespace smat;
  const bool packed = lengths && times && n > 0;
  int longest = packed ? 0 : nch;
  for (int i = 0; packed && i < n; ++i) longest = lengths[i] > longest ? lengths[i] : longest;
  if (longest < 1 || nb < 1 || r < 1 || p < 1 || r > hd::kMaxD || p > hd::kMaxD ||
      dtype < SMAT_BF16 || dtype > SMAT_F32)
    return 1;
  int on = 1;                                      // workgroups a CU
  dl::dispatch(dtype, r, [&](auto in, auto rb) {
    typedef decltype(in) In;
    constexpr int RB = decltype(rb)::value;
    on = p <= 64 ? hd::walk_occ<In, RB, 64, true, 0>() * 4 / hd::waves<In, 64, true, 0>()
                 : hd::walk_occ<In, RB, 128, true, 0>() * 4 / hd::waves<In, 128, true, 0>();
    return 0;
  });
  static const double terms[] = {1.0, 1.35, 1.7}, share[] = {0.0, 1.0, 1.45, 1.9};
  const double step = (1.6 + 0.7 * dl::rblocks(r)) * (p <= 64 ? 1.0 : 1.5) *
                      terms[dl::in_terms(dtype) - 1];
  // wgs workgroups of up to K chunks, `steps` chunks in all
  auto pass = [&](double wgs, double steps, int K) {
    const double rounds = (double)(int64_t)(wgs / (256 * on)), left = wgs - rounds * 256 * on;
    const int most = left <= 0 ? 0 : left <= 256 ? 1 : left <= 512 ? 2 : 3;
    const double even = steps / (wgs * K);         // runs shorter than K end earlier
    return K * (rounds * share[on] * even + share[most < on ? most : on]);
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
    if (G > 1 && runs > dl::kMaxGrid) continue;    // more than a grid holds
    double us = step * pass(runs * nb, chunks * nb, K);
    if (ends > 0)
      us += 0.42 * step * pass(ends * nb, ends * K * nb, K) + 9 + runs * nb * r * p * 16 / 4e6;
    if (G == 1 || us < least) {
      least = us;
      best = K;
    }
  }
  return best;
}

extern "C" int64_t smat_head_decay_workspace_bytes(int nb, int nbk, int T, int nseg, int nruns,
                                                   int r, int p, int backward, int learn) {
  using namespace smat;
  dl::Arena ar{nullptr};
  hd::take(ar, nb, nbk, T, nseg, nruns, r, p, backward != 0, learn != 0);
  return ar.used;
}

extern "C" int smat_head_decay_scan(int dtype, const void* q, const void* k, const void* v,
                                    const float* logA, const float* state, void* out,
                                    float* state_out, float* save_start, float* save_s,
                                    const int32_t* chunks, const int32_t* runs,
                                    const int32_t* segrun, int nb, int nbk, int heads, int T,
                                    int nseg, int nch, int nruns, int K, int r, int p, float scale,
                                    int64_t q_sb, int64_t q_st, int64_t k_sb, int64_t k_st,
                                    int64_t v_sb, int64_t v_st, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  using namespace smat;
  using namespace smat::hd;
  clear_error();
  const char* who = "smat_head_decay_scan";
  Walk g = {chunks, runs, segrun, nb, T, nseg, nch, nruns, K, r, p};
  g.heads = heads;
  int rc = check(who, dtype, g, nbk, r, p, {q_st, k_st, v_st});
  if (rc) return rc;
  if (nb == 0) return SMAT_OK;
  SMAT_REQUIRE(logA && (nch == 0 || (q && k && v && out)), SMAT_EINVAL, "%s: null pointer", who);
  SMAT_REQUIRE(state_out != state || !state, SMAT_EINVAL, "%s: state_out must not be state", who);
  SMAT_REQUIRE(aligned16(save_s), SMAT_EINVAL, "%s: save_s is not 16-byte aligned", who);
  rc = check_workspace(who, workspace, workspace_bytes,
                       smat_head_decay_workspace_bytes(nb, nbk, T, nseg, nruns, r, p, 0, 0));
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  dl::Arena ar{(char*)workspace};
  const Scratch sc = take(ar, nb, nbk, T, nseg, nruns, r, p, false, false);
  const int group = nb / nbk;
  g.q = {q, q_sb, q_st, group};
  g.k = {k, k_sb, k_st, group};
  g.v = {v, v_sb, v_st, 1};
  g.logA = logA;
  g.upd = 1.f;
  g.inter = g.intra = scale;
  g.start = state;
  g.s_row = p;
  g.s_col = 1;
  if (nruns > nseg) {
    float* start = save_start ? save_start : sc.start;
    rc = carry(dtype, g, state, sc.E, start, st);
    if (rc) return rc;
    g.start = start;
  }
  g.fin = state_out;
  g.o = out;
  g.save_s = save_s;
  return walk_any(dtype, g, true, kNone, st);
}

extern "C" int smat_head_decay_scan_backward(
    int dtype, const void* q, const void* k, const void* v, const float* logA, const void* dout,
    const float* dstate_out, const float* start, const float* save_s, void* dq, void* dk, void* dv,
    float* dstate, float* dlogA, const int32_t* chunks, const int32_t* runs, const int32_t* segrun,
    int nb, int nbk, int heads, int T, int nseg, int nch, int nruns, int K, int r, int p,
    float scale, int64_t q_sb, int64_t q_st, int64_t k_sb, int64_t k_st, int64_t v_sb, int64_t v_st,
    int64_t d_sb, int64_t d_st, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace smat;
  using namespace smat::hd;
  clear_error();
  const char* who = "smat_head_decay_scan_backward";
  Walk base = {chunks, runs, segrun, nb, T, nseg, nch, nruns, K, r, p};
  base.heads = heads;
  int rc = check(who, dtype, base, nbk, r, p, {q_st, k_st, v_st, d_st});
  if (rc) return rc;
  const bool learn = dlogA != nullptr;
  if (nb == 0) return SMAT_OK;
  SMAT_REQUIRE(logA && (nch == 0 || (q && k && v && dout && dq && dk && dv)), SMAT_EINVAL,
               "%s: null pointer", who);
  SMAT_REQUIRE((nruns == nseg || start) && (!learn || save_s || nch == 0), SMAT_EINVAL,
               "%s: the states that the forward kept are missing", who);
  SMAT_REQUIRE(aligned16(save_s), SMAT_EINVAL, "%s: save_s is not 16-byte aligned", who);
  rc = check_workspace(
      who, workspace, workspace_bytes,
      smat_head_decay_workspace_bytes(nb, nbk, T, nseg, nruns, r, p, 1, learn));
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  dl::Arena ar{(char*)workspace};
  const Scratch sc = take(ar, nb, nbk, T, nseg, nruns, r, p, true, learn);
  const int group = nb / nbk;
  base.logA = logA;
  base.intra = scale;
  const Side Q = {q, q_sb, q_st, group}, Kk = {k, k_sb, k_st, group}, V = {v, v_sb, v_st, 1},
             dO = {dout, d_sb, d_st, 1};
  // backwards: the gradients of v and k
  Walk g = base;
  g.rev = true;
  g.q = Kk;
  g.k = Q;
  g.v = dO;
  g.upd = scale;
  g.inter = 1.f;
  g.start = dstate_out;
  g.s_row = p;
  g.s_col = 1;
  if (nruns > nseg) {
    rc = carry(dtype, g, dstate_out, sc.E, sc.start, st);
    if (rc) return rc;
    g.start = sc.start;
  }
  g.fin = dstate;
  g.o = dv;
  g.load_s = save_s;
  g.part = sc.part[0];
  Walks all = {{g}, 3};
  g.q = V;
  g.k = dO;
  g.v = Q;
  g.r = p;
  g.p = r;
  g.s_row = 1;
  g.s_col = p;
  g.fin = nullptr;
  g.o = group > 1 ? (void*)sc.dk : dk;
  g.wide = group > 1;
  g.x = Kk;
  g.part = sc.part[1];
  all.w[1] = g;
  // forward: that of q
  g.rev = false;
  g.q = dO;
  g.k = V;
  g.v = Kk;
  g.upd = 1.f;
  g.inter = scale;
  g.start = start;
  g.o = group > 1 ? (void*)sc.dq : dq;
  g.x = Q;
  g.part = sc.part[2];
  all.w[2] = g;
  // in one launch where one kernel serves all three (96 sequences of 4096, 64 x 64:
  // 149 us, one after the other 174; now 140), and its grid has less than
  // 2^32 threads along the axis
  if (!learn && dl::rblocks(r) == dl::rblocks(p) && (r <= 64) == (p <= 64) && nb < (1 << 21)) {
    rc = walk_all(dtype, all, true, kNone, st);
    if (rc) return rc;
  } else {
    const int roles[] = {kDv, kDk, kDq};
    for (int i = 0; i < 3; ++i) {
      rc = walk_any(dtype, all.w[i], true, learn ? roles[i] : kNone, st);
      if (rc) return rc;
    }
  }
  if (group > 1 && nch > 0) {
    const int64_t n = (int64_t)T * r;
    const int blocks = (int)((n + 1023) / 1024 < 4096 ? (n + 1023) / 1024 : 4096);
    auto sum = [&](auto in) {
      typedef decltype(in) In;
      for (int ks = 0; ks < nbk; ks += dl::kMaxGrid) {   // (a grid's second axis)
        const int many = nbk - ks < dl::kMaxGrid ? nbk - ks : dl::kMaxGrid;
        const int64_t in0 = (int64_t)ks * group * n, out0 = (int64_t)ks * n;
        hipLaunchKernelGGL(decay_heads_kernel<In>, dim3(blocks, many), dim3(256), 0, st,
                           sc.dq + in0, (In*)dq + out0, group, n);
        hipLaunchKernelGGL(decay_heads_kernel<In>, dim3(blocks, many), dim3(256), 0, st,
                           sc.dk + in0, (In*)dk + out0, group, n);
      }
    };
    if (dtype == SMAT_BF16) sum(bf16());
    else if (dtype == SMAT_F16) sum(f16());
    else sum(float());
  }
  if (learn)
    hipLaunchKernelGGL(decay_grad_kernel, dim3(heads), dim3(256), 0, st, sc.part[0], sc.part[1],
                       sc.part[2], learn_waves(p), learn_waves(r),
                       learn_waves(r), nruns, nb, heads, dlogA);
  return launch_status(who);
}
