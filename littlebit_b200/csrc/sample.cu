// Verification of sampled drafts from given random numbers
// (speculative_decoding.py:331-363): p = softmax(target / T), q =
// softmax(draft / T); draft i is accepted while u_i < min(1, p_i(d_i) /
// max(q_i(d_i), 1e-10)); then argmax_v r_v / e_v with r the positive part of
// p_a - q_a, or p_k.
#include <cooperative_groups.h>
#include <type_traits>

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

// One cluster of AC_C blocks a sequence, each with a slice of the vocabulary, in one
// launch: the statistics of all rows at once (a warp takes 512 logits of one
// row at a time, four 16-byte loads a lane in flight), joined by shuffles and sent to every
// block's shared memory; every block then makes the same decisions and takes its slice of the
// drawing.  All rows are read before the first decision is known: deciding row
// by row would read fewer of them and wait for the cluster once a draft.
// Bound by memory for many sequences, by three round trips to it and two cluster barriers
// for one: 64 sequences of up to 8 drafts, 32000 logits, 82 MB: 32 us; 1 of 4: 10.3 from the
// kernel's first instruction to its last (13 with parts joined by one thread a row and
// read from the blocks that hold them).
// As many threads as let all blocks be on the GPU at once: 1024 up to AC_ONE sequences, 512 (two
// blocks an SM) up to AC_TWO, 256 (four) past it.  us with 1024, 512, 256 threads, 4 drafts,
// behind a flush of L2: 8 sequences of 32000 logits 18, 18, 21, of 128256 29, 35, 47; 12 of 128256
// 33, 37, 50; 16: 31, 21, 23 and 55, 43, 53; 32: 45, 25, 25 and 82, 54, 66; 64: 70, 41, 33
// and 129, 96, 84.
constexpr int AC_ONE = 12, AC_TWO = 32;
constexpr int AC_C = 8;      // blocks a sequence
constexpr int AC_Q = 4;      // quads of logits a lane loads together
constexpr int AC_ROWS = 2 * LBX_ACCEPT_MAX_K + 1;
// Logits are kept within [-inf, AC_TOP], NaN as -inf, and a row's top starts at -AC_TOP:
// weights 2^((x - top) log2(e) / T) then need no case of their own for infinities, and 36
// instructions a logit (selects turned into branches) became 7.  -inf has the weight 0 against
// any top; a mask of the type's lowest number is a number, and a row of nothing else has
// equal probabilities.  (Scaled before the subtraction, such numbers overflowed.)
constexpr float AC_TOP = 3.402823466e38f;  // the largest float
constexpr int AC_MAXV = 1 << 30;   // logits a row: indexes past the end stay 32-bit numbers
constexpr float AC_COLD = 1e-30f;  // temperatures up to here take the maximum

// does a row start on 16 (fp32) or 8 (bf16) bytes
template <int DT>
LBX_DEV bool ac_aligned(const void *row) { return (reinterpret_cast<uintptr_t>(row) & (DT == LBX_F32 ? 15u : 7u)) == 0; }
// four logits (what is past V: -inf)
template <int DT>
LBX_DEV float4 ac_quad_full(const void *row, int q) {
  if constexpr (DT == LBX_F32) {
    return __ldg(reinterpret_cast<const float4 *>(row) + q);
  } else {
    const uint2 x = __ldg(reinterpret_cast<const uint2 *>(row) + q);
    return make_float4(__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xFFFF0000u), __uint_as_float(x.y << 16),
                       __uint_as_float(x.y & 0xFFFF0000u));
  }
}
template <int DT>
LBX_DEV float4 ac_quad(const void *row, bool vec, int q, int V) {
  if (vec && 4 * q + 3 < V) return ac_quad_full<DT>(row, q);
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = 4 * q + i < V ? load_act(row, DT, 4 * (int64_t)q + i) : -INFINITY;
  return make_float4(v[0], v[1], v[2], v[3]);
}
LBX_DEV float ac_held(float x) { return fminf(fmaxf(x, -INFINITY), AC_TOP); }
LBX_DEV float ac_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// the larger value first, then the lower index; 0 for -inf and NaN
LBX_DEV uint64_t ac_key(float x, uint32_t i) {
  const uint32_t b = __float_as_uint(__fadd_rn(x, 0.f));  // (-0 becomes 0: the two are equal)
  return x > -INFINITY ? (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - i) : 0ull;
}
LBX_DEV uint64_t warp_max64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor_sync(0xffffffffu, (unsigned long long)v, o);
    v = w > v ? w : v;
  }
  return v;
}
// the weight of x against a top, c = log2(e) / T
LBX_DEV float ac_weight(float x, float top, float c) { return ac_ex2((x - top) * c); }
// (top, sum of weights against it) of two parts of a row; a part of nothing: (-AC_TOP, 0)
LBX_DEV float2 ac_join(float2 a, float2 b, float c) {
  const float m = fmaxf(a.x, b.x);
  return make_float2(m, a.y * ac_weight(a.x, m, c) + b.y * ac_weight(b.x, m, c));
}
LBX_DEV uint64_t ac_pack(float2 v) { return (uint64_t)__float_as_uint(v.x) << 32 | __float_as_uint(v.y); }
LBX_DEV float2 ac_pair(uint64_t v) { return make_float2(__uint_as_float((uint32_t)(v >> 32)), __uint_as_float((uint32_t)v)); }

template <int DT, int AC_T>
__global__ void __launch_bounds__(AC_T, 1024 / AC_T) accept_kernel(const __grid_constant__ AcceptParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  constexpr int ES = DT == LBX_F32 ? 4 : 2;
  constexpr int NWARP = AC_T / 32;
  __shared__ uint64_t part[AC_ROWS][NWARP];  // each warp's share of a row: (top, sum) pairs, or keys (greedy)
  __shared__ uint64_t all[AC_C][AC_ROWS], tot[AC_ROWS];  // every block's share of a row, and the row
  __shared__ uint64_t best[2][AC_C];          // every block's
  __shared__ uint64_t wbest[AC_T / 32];
  __shared__ int rejected;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int s = blockIdx.x / AC_C, rank = (int)cl.block_rank(), V = p.vocab;
  cl.barrier_arrive();  // (waited for before the first store to another block's shared memory)
  pdl_trigger();
  pdl_wait();
  const float T = p.temps ? __ldg(p.temps + s) : p.temperature;
  const bool greedy = !(T > AC_COLD);
  const float c = fmaxf(1.4426950408889634f / T, 1e-30f);  // (an infinite T: -inf times 0 would be no number)
  const uint64_t none = greedy ? 0ull : ac_pack(make_float2(-AC_TOP, 0.f));
  int nd = p.k;
  if (p.n_draft) {
    nd = __ldg(p.n_draft + s);
    if (nd < 0 || nd > p.k) {
      if (rank == 0 && tid == 0) atomicCAS(&g_lbx_device_error, 0, 0x812);
      nd = min(max(nd, 0), p.k);
    }
  }
  const bool has_q = p.draft != nullptr && !greedy;
  // rows 0 .. nd: the target's; nd + 1 ..: the drafts'
  const int nrow = nd + 1 + (has_q ? nd : 0);
  auto row_at = [&](int r) {
    return r <= nd ? reinterpret_cast<const uint8_t *>(p.target) + (s * p.target_seq + r * p.target_row) * ES
                   : reinterpret_cast<const uint8_t *>(p.draft) + (s * p.draft_seq + (r - nd - 1) * p.draft_row) * ES;
  };
  // this block's quads, in batches of 32 lanes x AC_Q
  constexpr int BQ = 32 * AC_Q;
  const int nq = (V + 3) / 4, per = (nq + AC_C - 1) / AC_C;
  const int q0 = min(nq, rank * per), q1 = min(nq, q0 + per), nb = (per + BQ - 1) / BQ;

  // the random numbers of the drawing, to L2 meanwhile (8 sequences of 128256 logits: 31
  // to 29 us; many sequences leave memory no idle time, 41 to 43)
  if (AC_T > 256 && !greedy)
    for (int v = 4 * q0 + 32 * tid; v < min(4 * q1, V); v += 32 * AC_T)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.e + s * p.e_ld + v));

  // ---- statistics of every row's slice: the (row, batch) items dealt evenly to the
  // warps, the next item's loads under way while one is worked on
  int64_t tok = -1;
  float tl = -INFINITY, dl = -INFINITY, uu = 2.f;
  for (int i = tid; i < nrow * NWARP; i += AC_T) (&part[0][0])[i] = none;
  {
    const int items = nrow * nb;
    int it = (int)((int64_t)items * warp / NWARP);
    const int end = (int)((int64_t)items * (warp + 1) / NWARP);
    int r = it / nb, b = it - r * nb;
    float m = -AC_TOP, l = 0.f;
    uint64_t key = 0;
    auto load = [&](float4 (&x)[AC_Q], int r, int b) {
      const uint8_t *row = row_at(r);
      const bool vec = ac_aligned<DT>(row);
      const int q = q0 + b * BQ;
      if (vec && q + BQ <= q1 && 4 * (q + BQ) <= V) {
#pragma unroll
        for (int i = 0; i < AC_Q; ++i) x[i] = ac_quad_full<DT>(row, q + 32 * i + lane);
      } else {
#pragma unroll
        for (int i = 0; i < AC_Q; ++i) {
          x[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
          if (q + 32 * i + lane < q1) x[i] = ac_quad<DT>(row, vec, q + 32 * i + lane, V);
        }
      }
    };
    // works on x, item (r, b), with item it + 1 on its way into y
    auto work = [&](float4 (&x)[AC_Q], float4 (&y)[AC_Q]) {
      const int b2 = b + 1 < nb ? b + 1 : 0, r2 = b2 ? r : r + 1;
      if (it + 1 < end) load(y, r2, b2);
      if (greedy) {
#pragma unroll
        for (int i = 0; i < AC_Q; ++i) {
          const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint64_t k = ac_key(v[e], (uint32_t)(4 * (q0 + b * BQ + 32 * i + lane) + e));
            key = k > key ? k : key;
          }
        }
      } else {
        float mn = m;
#pragma unroll
        for (int i = 0; i < AC_Q; ++i) {
          x[i] = make_float4(ac_held(x[i].x), ac_held(x[i].y), ac_held(x[i].z), ac_held(x[i].w));
          mn = fmaxf(mn, fmaxf(fmaxf(x[i].x, x[i].y), fmaxf(x[i].z, x[i].w)));
        }
        l *= ac_weight(m, mn, c);
        m = mn;
#pragma unroll
        for (int i = 0; i < AC_Q; ++i)
          l += (ac_weight(x[i].x, m, c) + ac_weight(x[i].y, m, c)) + (ac_weight(x[i].z, m, c) + ac_weight(x[i].w, m, c));
      }
      if (r2 != r || it + 1 >= end) {
        if (greedy) {
          key = warp_max64(key);
        } else {
          float2 ml = make_float2(m, l);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1)
            ml = ac_join(ml, make_float2(__shfl_xor_sync(0xffffffffu, ml.x, o), __shfl_xor_sync(0xffffffffu, ml.y, o)), c);
          key = ac_pack(ml);
        }
        if (lane == 0) part[r][warp] = key;
        key = 0;
        m = -AC_TOP;
        l = 0.f;
      }
      r = r2;
      b = b2;
      ++it;
    };
    float4 x[AC_Q], y[AC_Q];
    if (it < end) load(x, r, b);
    __syncthreads();
    // what a decision needs besides the rows' statistics, on its way meanwhile
    if (tid < nd) {
      tok = __ldg(p.tokens + s * p.tokens_ld + tid);
      uu = __ldg(p.u + s * p.u_ld + tid);
      if (tok >= 0 && tok < V) {
        tl = load_act(row_at(tid), DT, tok);
        if (has_q) dl = load_act(row_at(nd + 1 + tid), DT, tok);
      } else if (rank == 0) {
        atomicCAS(&g_lbx_device_error, 0, 0x811);
      }
    }
    while (it < end) {
      work(x, y);
      if (it < end) work(y, x);
    }
  }
  auto join = [&](uint64_t a, uint64_t b) {
    if (greedy) return a > b ? a : b;
    return ac_pack(ac_join(ac_pair(a), ac_pair(b), c));
  };
  // lanes xor o, 2 o, ... joined; every block goes the same way
  auto reduce = [&](uint64_t v, int o) {
    for (; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, (unsigned long long)v, o));
    return v;
  };
  __syncthreads();
  cl.barrier_wait();
  for (int r = warp; r < nrow; r += NWARP) {
    uint64_t v = reduce(lane < NWARP ? part[r][lane] : none, 16);
    v = __shfl_sync(0xffffffffu, (unsigned long long)v, 0);
    if (lane < AC_C) *cl.map_shared_rank(&all[rank][r], lane) = v;
  }
  cl.sync();
  for (int r0 = 4 * warp; r0 < nrow; r0 += 4 * NWARP) {  // eight lanes a row
    const int r = r0 + lane / AC_C;
    const uint64_t v = reduce(r < nrow ? all[lane % AC_C][r] : none, AC_C / 2);
    if (r < nrow && lane % AC_C == 0) tot[r] = v;
  }
  if (tid == 0) rejected = nd;
  __syncthreads();

  // ---- decisions (the same in every block)
  auto first_of = [](uint64_t k) { return k ? (int64_t)(0xFFFFFFFFu - (uint32_t)k) : -1; };
  auto prob = [&](float x, int r) {
    const float2 ml = ac_pair(tot[r]);
    return ml.y > 0.f ? ac_weight(ac_held(x), ml.x, c) / ml.y : 0.f;
  };
  if (tid < nd) {
    bool ok;
    if (greedy) {
      ok = first_of(tot[tid]) == tok && tok >= 0 && uu < 1.f;
    } else {
      const float qd = !has_q ? 1.f : prob(dl, nd + 1 + tid);
      ok = uu < fminf(prob(tl, tid) / fmaxf(qd, 1e-10f), 1.f);
    }
    if (!ok) atomicMin(&rejected, tid);
  }
  __syncthreads();
  const int a = rejected;
  int64_t next = -1;
  if (greedy) {
    next = first_of(tot[a]);
  } else {
    // ---- the token after them: the largest r_v / e_v of this block's slice
    const float2 pm = ac_pair(tot[a]);
    const bool cut = a < nd, q = cut && has_q;
    const float2 qm = q ? ac_pair(tot[nd + 1 + a]) : make_float2(0.f, 0.f);
    const float pi = pm.y > 0.f ? 1.f / pm.y : 0.f, qi = qm.y > 0.f ? 1.f / qm.y : 0.f;
    const uint8_t *prow = row_at(a), *qrow = q ? row_at(nd + 1 + a) : prow;
    const bool pv = ac_aligned<DT>(prow), qv = ac_aligned<DT>(qrow);
    const float *er = p.e + s * p.e_ld;
    const bool ev = ac_aligned<LBX_F32>(er);
    int64_t dtok = -1;
    if (cut && !p.draft) dtok = __ldg(p.tokens + s * p.tokens_ld + a);
    uint64_t got = 0;
    for (int pass = cut ? 0 : 1; pass < 2; ++pass) {
      uint64_t key = 0;
      const bool less = pass == 0;
      constexpr int NB = AC_T == 256 ? 2 : 1;
      for (int b = q0 + tid; b < q1; b += NB * AC_T) {
        float4 x[NB], y[NB], z[NB];
        const int last = b + (NB - 1) * AC_T;
        if (pv && qv && ev && last < q1 && 4 * last + 3 < V) {  // (no branch between the loads)
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            x[i] = ac_quad_full<DT>(prow, b + i * AC_T);
            y[i] = ac_quad_full<DT>(qrow, b + i * AC_T);
            z[i] = ac_quad_full<LBX_F32>(er, b + i * AC_T);
          }
        } else {
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const int k = b + i * AC_T;
            x[i] = y[i] = z[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (k < q1) {
              x[i] = ac_quad<DT>(prow, pv, k, V);
              y[i] = ac_quad<DT>(qrow, qv, k, V);
              z[i] = ac_quad<LBX_F32>(er, ev, k, V);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const float xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w}, ys[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
          const float zs[4] = {z[i].x, z[i].y, z[i].z, z[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int v = 4 * (b + i * AC_T) + e;
            // (products rounded on their own: equal rows leave exactly nothing)
            float r = __fmul_rn(ac_weight(ac_held(xs[e]), pm.x, c), pi);
            if (less) {
              if (q) r = __fsub_rn(r, __fmul_rn(ac_weight(ac_held(ys[e]), qm.x, c), qi));
              else if (v == dtok) r -= 1.f;
            }
            if (r > 0.f) {
              const uint64_t k = (uint64_t)__float_as_uint(r / zs[e]) << 32 | (0xFFFFFFFFu - (uint32_t)v);
              key = k > key ? k : key;
            }
          }
        }
      }
      key = warp_max64(key);
      if (lane == 0) wbest[warp] = key;
      __syncthreads();
      if (warp == 0) {
        key = warp_max64(lane < NWARP ? wbest[lane] : 0ull);
        if (lane < AC_C) *cl.map_shared_rank(&best[pass][rank], lane) = key;
      }
      cl.sync();
#pragma unroll
      for (int i = 0; i < AC_C; ++i) got = best[pass][i] > got ? best[pass][i] : got;
      if (got) break;  // (else p and q are equal, nothing is left over, and the token comes from p)
    }
    next = first_of(got);
  }
  // (no store to another block's shared memory is later than the last cluster barrier: blocks may leave)
  if (rank == 0 && tid == 0) {
    p.accepted[s] = a;
    p.next[s] = next;
  }
}

}  // namespace lbx

extern "C" int lbx_accept_sampled(const lbx_accept_args *a, cudaStream_t stream) {
  using namespace lbx;
  LBX_CHECK_ARG(a, "args is NULL");
  LBX_CHECK_ARG(a->n_seq >= 0 && a->k >= 0 && a->vocab >= 1, "bad shape");
  LBX_CHECK_SUP(a->k <= LBX_ACCEPT_MAX_K, "k must be <= %d", LBX_ACCEPT_MAX_K);
  LBX_CHECK_SUP(a->vocab <= AC_MAXV, "vocab must be <= %d", AC_MAXV);
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
  LBX_CHECK_SUP((int64_t)a->n_seq * AC_C <= 0x7fffffff, "too many sequences");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a->n_seq * AC_C);
  const int threads = a->n_seq <= AC_ONE ? 1024 : a->n_seq <= AC_TWO ? 512 : 256;
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = AC_C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a->use_pdl ? 2 : 1;
  auto go = [&](auto kern) { return cudaLaunchKernelEx(&cfg, kern, p); };
  auto pick = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return threads == 1024 ? go(accept_kernel<DT, 1024>) : threads == 512 ? go(accept_kernel<DT, 512>) : go(accept_kernel<DT, 256>);
  };
  return cuda_status(a->dtype == LBX_F32 ? pick(std::integral_constant<int, LBX_F32>{}) : pick(std::integral_constant<int, LBX_BF16>{}),
                     "accept_sampled launch");
}
