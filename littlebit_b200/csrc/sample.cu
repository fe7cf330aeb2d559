// Verification of sampled drafts from given random numbers
// (speculative_decoding.py:331-363): p = softmax(target / T), q =
// softmax(draft / T); draft i is accepted while u_i < min(1, p_i(d_i) /
// max(q_i(d_i), 1e-10)); then argmax_v r_v / e_v with r the positive part of
// p_a - q_a, or p_k.
#include "common.cuh"

namespace lbx {

struct AcceptParams {
  int k, vocab, dtype;
  float temperature;
  const float *temps;
  const int64_t *tokens; int64_t tokens_ld;
  const int32_t *n_draft;
  const void *target; int64_t target_seq, target_row;
  const void *draft; int64_t draft_seq, draft_row;
  const float *u; int64_t u_ld;
  const float *e; int64_t e_ld;
  int64_t *accepted;
  int64_t *next;
};

// (NaN counts as -inf)
LBX_DEV float logit_at(const void *p, int dtype, int64_t i) {
  const float x = load_act(p, dtype, i);
  return x == x ? x : -INFINITY;
}
// weight of a logit against its row's maximum m: exp((x - m) / T), 1 at the
// maximum (an infinite one too), 0 for -inf
LBX_DEV float logit_weight(float x, float m, float T) {
  return x == m ? 1.f : expf((x - m) / T);
}

constexpr int AC_THREADS = 512;

__global__ void __launch_bounds__(AC_THREADS) accept_simple_kernel(const __grid_constant__ AcceptParams p) {
  __shared__ float rf[AC_THREADS / 32];
  __shared__ unsigned long long ru[AC_THREADS / 32];
  const int s = blockIdx.x, tid = threadIdx.x, V = p.vocab;
  const float T = p.temps ? p.temps[s] : p.temperature;
  const bool greedy = !(T > 0.f);
  auto bmax = [&](float v) {
    v = warp_max(v);
    __syncthreads();
    if ((tid & 31) == 0) rf[tid >> 5] = v;
    __syncthreads();
    float m = rf[0];
    for (int i = 1; i < AC_THREADS / 32; ++i) m = fmaxf(m, rf[i]);
    return m;
  };
  auto bsum = [&](float v) {
    v = warp_sum(v);
    __syncthreads();
    if ((tid & 31) == 0) rf[tid >> 5] = v;
    __syncthreads();
    float m = rf[0];
    for (int i = 1; i < AC_THREADS / 32; ++i) m += rf[i];
    return m;
  };
  // largest value first, then the lowest index; values >= 0
  auto bbest = [&](unsigned long long v) {
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((tid & 31) == 0) ru[tid >> 5] = v;
    __syncthreads();
    unsigned long long m = ru[0];
    for (int i = 1; i < AC_THREADS / 32; ++i) m = max(m, ru[i]);
    return m;
  };
  auto first_max = [&](const void *row, int64_t off, float m) {
    unsigned long long b = 0;
    for (int v = tid; v < V; v += AC_THREADS)
      if (m > -INFINITY && logit_at(row, p.dtype, off + v) == m) b = max(b, (unsigned long long)(0xffffffffu - v));
    return bbest(b);
  };
  // (max, sum of weights, first maximum's index) of a row; sum 0: no probability
  auto stats = [&](const void *row, int64_t off, float &m, float &l, int &at) {
    float x = -INFINITY;
    for (int v = tid; v < V; v += AC_THREADS) x = fmaxf(x, logit_at(row, p.dtype, off + v));
    m = bmax(x);
    at = -1;
    if (m == -INFINITY) {
      l = 0.f;
      return;
    }
    if (greedy) {
      l = 1.f;
      at = (int)(0xffffffffu - (unsigned)first_max(row, off, m));
      return;
    }
    float t = 0.f;
    for (int v = tid; v < V; v += AC_THREADS) t += logit_weight(logit_at(row, p.dtype, off + v), m, T);
    l = bsum(t);
  };
  auto prob = [&](const void *row, int64_t off, int v, float m, float l, int at) {
    if (!(l > 0.f)) return 0.f;
    if (greedy) return v == at ? 1.f : 0.f;
    return logit_weight(logit_at(row, p.dtype, off + v), m, T) / l;
  };
  int nd = p.k;
  if (p.n_draft) {
    nd = p.n_draft[s];
    if (nd < 0 || nd > p.k) {
      if (tid == 0) atomicCAS(&g_lbx_device_error, 0, 0x812);
      nd = min(max(nd, 0), p.k);
    }
  }
  int a = 0;
  float pm = 0.f, pl = 0.f, qm = 0.f, ql = 0.f;
  int pa = -1, qa = -1;
  int64_t po = 0, qo = 0;
  int64_t d = -1;
  for (;; ++a) {
    po = s * p.target_seq + a * p.target_row;
    stats(p.target, po, pm, pl, pa);
    if (a >= nd) break;
    d = p.tokens[s * p.tokens_ld + a];
    const bool in = d >= 0 && d < V;
    if (!in && tid == 0) atomicCAS(&g_lbx_device_error, 0, 0x811);
    const float pd = in ? prob(p.target, po, (int)d, pm, pl, pa) : 0.f;
    float qd = 1.f;
    if (p.draft) {
      qo = s * p.draft_seq + a * p.draft_row;
      stats(p.draft, qo, qm, ql, qa);
      qd = in ? prob(p.draft, qo, (int)d, qm, ql, qa) : 0.f;
    }
    if (!(p.u[s * p.u_ld + a] < fminf(pd / fmaxf(qd, 1e-10f), 1.f))) break;
  }
  unsigned long long best = 0;
  for (int pass = a < nd ? 0 : 1; pass < 2 && best == 0; ++pass) {
    unsigned long long b = 0;
    for (int v = tid; v < V; v += AC_THREADS) {
      float r = prob(p.target, po, v, pm, pl, pa);
      if (pass == 0) r -= p.draft ? prob(p.draft, qo, v, qm, ql, qa) : (v == d ? 1.f : 0.f);
      if (!(r > 0.f)) continue;
      const float sc = r / p.e[s * p.e_ld + v];
      b = max(b, (unsigned long long)__float_as_uint(sc) << 32 | (0xffffffffu - v));
    }
    best = bbest(b);
  }
  if (tid == 0) {
    p.accepted[s] = a;
    p.next[s] = best ? (int64_t)(0xffffffffu - (unsigned)best) : -1;
  }
}

}  // namespace lbx

extern "C" int lbx_accept_sampled(const lbx_accept_args *a, cudaStream_t stream) {
  using namespace lbx;
  LBX_CHECK_ARG(a, "args is NULL");
  LBX_CHECK_ARG(a->n_seq >= 0 && a->k >= 0 && a->vocab >= 1, "bad shape");
  LBX_CHECK_SUP(a->k <= LBX_ACCEPT_MAX_K, "k must be <= %d", LBX_ACCEPT_MAX_K);
  LBX_CHECK_ARG(a->dtype == LBX_F32 || a->dtype == LBX_BF16, "bad dtype");
  LBX_CHECK_ARG(a->temps || (a->temperature >= 0.f && a->temperature < INFINITY), "temperature must be >= 0");
  if (a->n_seq == 0) return LBX_OK;
  LBX_CHECK_ARG(a->target && a->e && a->accepted && a->next, "NULL pointer");
  LBX_CHECK_ARG(a->k == 0 || (a->tokens && a->u), "NULL pointer");
  LBX_CHECK_ARG(a->target_seq >= 0 && a->target_row >= 0 && a->draft_seq >= 0 && a->draft_row >= 0 && a->e_ld >= 0 &&
                    a->u_ld >= 0 && a->tokens_ld >= 0,
                "negative stride");
  AcceptParams p = {};
  p.k = a->k;
  p.vocab = a->vocab;
  p.dtype = a->dtype;
  p.temperature = a->temperature;
  p.temps = a->temps;
  p.tokens = a->tokens;
  p.tokens_ld = a->tokens_ld;
  p.n_draft = a->n_draft;
  p.target = a->target;
  p.target_seq = a->target_seq;
  p.target_row = a->target_row;
  p.draft = a->draft;
  p.draft_seq = a->draft_seq;
  p.draft_row = a->draft_row;
  p.u = a->u;
  p.u_ld = a->u_ld;
  p.e = a->e;
  p.e_ld = a->e_ld;
  p.accepted = a->accepted;
  p.next = a->next;
  accept_simple_kernel<<<a->n_seq, AC_THREADS, 0, stream>>>(p);
  return cuda_status(cudaGetLastError(), "accept_sampled launch");
}
