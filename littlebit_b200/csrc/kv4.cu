// KV cache held in 4 bits: append, read-back, attention.
//
// Each head and slot holds head_dim codes and, for each group of 64
// dimensions, (step, least) in bf16; a value is least + step * code.
// See include/lbx.h for the layout.
#include "common.cuh"

namespace lbx {

constexpr int KV4_G = 64;       // dimensions a group
constexpr uint16_t KV4_NAN = 0x7FC0u;

// word index, in its row, of block b (dimensions 8b .. 8b+7)
template <int D, bool VALUE>
__host__ __device__ constexpr int kv4_word(int b) {
  return VALUE ? (b & 7) * (D / 64) + (b >> 3) : ((b & 7) & 3) * (D / 32) + 2 * (b >> 3) + ((b & 7) >> 2);
}
LBX_DEV float kv4_step(uint32_t par) { return __uint_as_float(par << 16); }
LBX_DEV float kv4_least(uint32_t par) { return __uint_as_float(par & 0xFFFF0000u); }

struct Kv4View {
  uint8_t *kc; uint32_t *kp;
  uint8_t *vc; uint32_t *vp;
  int n_seq, kvh, max_seq;
};

struct Kv4AppendParams {
  Kv4View c;
  int n, max_start, dtype;
  const int32_t *start;
  const void *k; const void *v; int64_t ld;
  const float2 *rope;
};

// One warp a (token, head, key or value).  Lane l holds dimensions 2l, 2l+1 of
// each group of 64 after the rotation.
template <int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(const __grid_constant__ Kv4AppendParams p) {
  constexpr int NG = D / KV4_G;
  __shared__ __align__(16) float sx[8][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 8 + warp;
  const int64_t per = (int64_t)p.c.n_seq * p.n * p.c.kvh;
  pdl_trigger();
  pdl_wait();
  if (item >= 2 * per) return;
  const bool value = item >= per;
  const int64_t it = value ? item - per : item;
  const int h = (int)(it % p.c.kvh);
  const int64_t row = it / p.c.kvh;  // token row
  const int s = (int)(row / p.n), i = (int)(row - (int64_t)s * p.n);
  const int st = p.start ? p.start[s] : p.max_start;
  if (st < 0 || st > p.max_start) {
    if (lane == 0) atomicCAS(&g_lbx_device_error, 0, 0x801);
    return;
  }
  const void *src = value ? p.v : p.k;
  const int64_t off = row * p.ld + (int64_t)h * D;
  float *x = sx[warp];
#pragma unroll
  for (int e = lane; e < D; e += 32) x[e] = load_act(src, p.dtype, off + e);
  __syncwarp();
  if (!value && p.rope) {
    float y1[D / 64], y2[D / 64];
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
      const int j = lane + 32 * u;
      const float2 cs = p.rope[row * (D / 2) + j];
      const float x1 = x[j], x2 = x[j + D / 2];
      y1[u] = __fsub_rn(__fmul_rn(x1, cs.x), __fmul_rn(x2, cs.y));
      y2[u] = __fadd_rn(__fmul_rn(x2, cs.x), __fmul_rn(x1, cs.y));
    }
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
      const int j = lane + 32 * u;
      x[j] = y1[u];
      x[j + D / 2] = y2[u];
    }
    __syncwarp();
  }
  const int64_t slot = ((int64_t)s * p.c.kvh + h) * p.c.max_seq + st + i;
  uint32_t *words = reinterpret_cast<uint32_t *>((value ? p.c.vc : p.c.kc) + slot * (D / 2));
  uint32_t *par = (value ? p.c.vp : p.c.kp) + slot * NG;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float a = x[64 * g + 2 * lane], b = x[64 * g + 2 * lane + 1];
    const bool fin = __all_sync(0xffffffffu, fabsf(a) < INFINITY && fabsf(b) < INFINITY);
    const float lo = -warp_max(fmaxf(-a, -b)), hi = warp_max(fmaxf(a, b));
    uint16_t sb = f32_to_bf16(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
    uint16_t lb = f32_to_bf16(lo);
    float step = bf16_to_f32(sb);
    if (step < 1.1754943508222875e-38f) {
      step = 0.f;
      sb = 0;
    }
    const float least = bf16_to_f32(lb);
    if (!fin || !(step < INFINITY) || !(fabsf(least) < INFINITY)) {
      sb = lb = KV4_NAN;
      step = 0.f;
    }
    const float inv = step > 0.f ? __fdiv_rn(1.0f, step) : 0.f;
    auto code = [&](float y) {
      if (!(step > 0.f)) return 0u;
      return (uint32_t)__float2int_rn(fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(y, least), inv)), 0.f), 15.f));
    };
    // 8 codes of a block: lanes 4r .. 4r+3
    uint32_t w = (code(a) | code(b) << 4) << (8 * (lane & 3));
    w |= __shfl_xor_sync(0xffffffffu, w, 1);
    w |= __shfl_xor_sync(0xffffffffu, w, 2);
    if ((lane & 3) == 0) {
      const int blk = 8 * g + (lane >> 2);
      words[value ? kv4_word<D, true>(blk) : kv4_word<D, false>(blk)] = w;
    }
    if (lane == 0) par[g] = (uint32_t)sb | (uint32_t)lb << 16;
  }
}

struct Kv4ReadParams {
  Kv4View c;
  int n, max_start;
  const int32_t *start;
  float *out[2];
};

// one thread a block of eight dimensions of one (sequence, head, token), keys then values
template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4ReadParams p) {
  constexpr int NB = D / 8;
  const bool value = blockIdx.y == 1;
  float *out = p.out[blockIdx.y];
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (!out || e >= (int64_t)p.c.n_seq * p.c.kvh * p.n * NB) return;
  const int b = (int)(e % NB);
  const int64_t r = e / NB;  // (sequence, head, token)
  const int64_t sh = r / p.n;
  const int i = (int)(r - sh * p.n), s = (int)(sh / p.c.kvh);
  const int st = p.start ? p.start[s] : p.max_start;
  const bool ok = st >= 0 && st <= p.max_start;
  if (!ok) atomicCAS(&g_lbx_device_error, 0, 0x802);
  float v[8];
  if (ok) {
    const int64_t slot = sh * p.c.max_seq + st + i;
    const uint32_t *words = reinterpret_cast<const uint32_t *>((value ? p.c.vc : p.c.kc) + slot * (D / 2));
    const uint32_t w = words[value ? kv4_word<D, true>(b) : kv4_word<D, false>(b)];
    const uint32_t par = (value ? p.c.vp : p.c.kp)[slot * (D / KV4_G) + (b >> 3)];
#pragma unroll
    for (int t = 0; t < 8; ++t)
      v[t] = __fadd_rn(kv4_least(par), __fmul_rn(kv4_step(par), (float)((w >> (4 * t)) & 15u)));
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] = __uint_as_float(0x7FC00000u);
  }
  float4 *o = reinterpret_cast<float4 *>(out + r * D + 8 * b);
  o[0] = make_float4(v[0], v[1], v[2], v[3]);
  o[1] = make_float4(v[4], v[5], v[6], v[7]);
}

struct Kv4AttnParams {
  Kv4View c;
  int n, heads, rep, max_prefix, dtype;
  float scale;
  const int32_t *prefix;
  const void *q; int64_t q_ld;
  const float2 *rope;
  const uint64_t *tree;
  void *out;
};

// does query i of its sequence see slot j
LBX_DEV bool kv4_sees(int j, int prefix, int n, int i, const uint64_t *mask) {
  if (j < prefix) return true;
  const int t = j - prefix;
  return t < n && (mask ? (t < 64 && ((*mask >> t) & 1ull)) : t <= i);
}

// One CTA a (query head, token row): 128 slots at a time, a thread each for the
// scores, a thread a dimension for the sums; one pass with the running maximum.
template <int D>
__global__ void __launch_bounds__(128) kv4_attn_simple_kernel(const __grid_constant__ Kv4AttnParams p) {
  __shared__ float qs[D], ps[128], red[4];
  const int tid = threadIdx.x, hq = blockIdx.x, h = hq / p.rep;
  const int64_t row = blockIdx.y;
  const int s = (int)(row / p.n), i = (int)(row - (int64_t)s * p.n);
  const int prefix = p.prefix ? p.prefix[s] : p.max_prefix;
  const int64_t o = row * (int64_t)p.heads * D + (int64_t)hq * D;
  auto store = [&](int t, float v) {
    if (p.dtype == LBX_F32) reinterpret_cast<float *>(p.out)[o + t] = v;
    else reinterpret_cast<uint16_t *>(p.out)[o + t] = f32_to_bf16(v);
  };
  if (prefix < 0 || prefix > p.max_prefix) {
    if (tid == 0) atomicCAS(&g_lbx_device_error, 0, 0x803);
    if (tid < D) store(tid, __uint_as_float(0x7FC00000u));
    return;
  }
  for (int j = tid; j < D / 2; j += 128) {
    const int64_t qo = row * p.q_ld + (int64_t)hq * D;
    const float x1 = load_act(p.q, p.dtype, qo + j), x2 = load_act(p.q, p.dtype, qo + j + D / 2);
    const float2 cs = p.rope ? p.rope[row * (D / 2) + j] : make_float2(1.f, 0.f);
    qs[j] = (x1 * cs.x - x2 * cs.y) * p.scale;
    qs[j + D / 2] = (x2 * cs.x + x1 * cs.y) * p.scale;
  }
  __syncthreads();
  const uint64_t *mask = p.tree ? p.tree + row : nullptr;
  const int top = prefix + p.n;
  const int64_t base = ((int64_t)s * p.c.kvh + h) * p.c.max_seq;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int j0 = 0; j0 < top; j0 += 128) {
    const int j = j0 + tid;
    float sc = -INFINITY;
    if (j < top && kv4_sees(j, prefix, p.n, i, mask)) {
      const uint32_t *w = reinterpret_cast<const uint32_t *>(p.c.kc + (base + j) * (D / 2));
      sc = 0.f;
      for (int b = 0; b < D / 8; ++b) {
        const uint32_t x = w[kv4_word<D, false>(b)];
        const uint32_t par = p.c.kp[(base + j) * (D / KV4_G) + (b >> 3)];
#pragma unroll
        for (int t = 0; t < 8; ++t)
          sc = fmaf(qs[8 * b + t], fmaf(kv4_step(par), (float)((x >> (4 * t)) & 15u), kv4_least(par)), sc);
      }
    }
    const float wm = warp_max(sc);
    if ((tid & 31) == 0) red[tid >> 5] = wm;
    __syncthreads();
    const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    ps[tid] = sc == -INFINITY ? 0.f : expf(sc - mn);
    __syncthreads();
    const float f = m == -INFINITY ? 0.f : expf(m - mn);
    l *= f;
    acc *= f;
    m = mn;
    const int jn = min(128, top - j0);
    for (int jj = 0; jj < jn; ++jj) {
      const float pr = ps[jj];
      if (!(pr > 0.f) && pr == pr) continue;
      l += pr;
      if (tid < D) {
        const int b = tid >> 3;
        const uint32_t *w = reinterpret_cast<const uint32_t *>(p.c.vc + (base + j0 + jj) * (D / 2));
        const uint32_t x = w[kv4_word<D, true>(b)];
        const uint32_t par = p.c.vp[(base + j0 + jj) * (D / KV4_G) + (b >> 3)];
        acc = fmaf(pr, fmaf(kv4_step(par), (float)((x >> (4 * (tid & 7))) & 15u), kv4_least(par)), acc);
      }
    }
    __syncthreads();
  }
  if (tid < D) store(tid, l == 0.f ? 0.f : acc / l);
}

// the cache's checks, shared by the three calls
static int kv4_view(const lbx_kv4_cache &c, Kv4View &v) {
  LBX_CHECK_ARG(c.n_seq >= 1 && c.kv_heads >= 1 && c.max_seq >= 1, "bad cache shape");
  LBX_CHECK_SUP(c.head_dim == 64 || c.head_dim == 128, "head_dim must be 64 or 128");
  LBX_CHECK_ARG(c.max_seq % 64 == 0, "max_seq must be a multiple of 64");
  LBX_CHECK_ARG(c.k_codes && c.k_params && c.v_codes && c.v_params, "NULL pointer");
  LBX_CHECK_ARG(aligned16(c.k_codes) && aligned16(c.k_params) && aligned16(c.v_codes) && aligned16(c.v_params),
                "cache arrays must be 16-byte aligned");
  v.kc = c.k_codes;
  v.kp = reinterpret_cast<uint32_t *>(c.k_params);
  v.vc = c.v_codes;
  v.vp = reinterpret_cast<uint32_t *>(c.v_params);
  v.n_seq = c.n_seq;
  v.kvh = c.kv_heads;
  v.max_seq = c.max_seq;
  return LBX_OK;
}

static int kv4_attn_prep(const lbx_kv4_attn_args *a, Kv4AttnParams &p) {
  LBX_CHECK_ARG(a, "args is NULL");
  const int rc = kv4_view(a->cache, p.c);
  if (rc) return rc;
  LBX_CHECK_ARG(a->n >= 1 && a->heads >= a->cache.kv_heads && a->heads % a->cache.kv_heads == 0,
                "heads must be a multiple of kv_heads, n >= 1");
  LBX_CHECK_ARG(a->max_prefix >= 0 && (int64_t)a->max_prefix + a->n <= a->cache.max_seq,
                "max_prefix + n exceeds max_seq");
  LBX_CHECK_ARG(a->dtype == LBX_F32 || a->dtype == LBX_BF16, "bad dtype");
  LBX_CHECK_SUP(!a->tree_mask || a->n <= 64, "a tree has at most 64 tokens");
  LBX_CHECK_ARG(a->q_ld >= (int64_t)a->heads * a->cache.head_dim, "q rows overlap");
  p.n = a->n;
  p.heads = a->heads;
  p.rep = a->heads / a->cache.kv_heads;
  p.max_prefix = a->max_prefix;
  p.dtype = a->dtype;
  p.scale = a->scale;
  p.prefix = a->prefix;
  p.q = a->q;
  p.q_ld = a->q_ld;
  p.rope = reinterpret_cast<const float2 *>(a->rope_cs);
  p.tree = a->tree_mask;
  p.out = a->out;
  return LBX_OK;
}

}  // namespace lbx

extern "C" int lbx_kv4_append(const lbx_kv4_append_args *a, cudaStream_t stream) {
  using namespace lbx;
  LBX_CHECK_ARG(a, "args is NULL");
  Kv4AppendParams p = {};
  const int rc = kv4_view(a->cache, p.c);
  if (rc) return rc;
  LBX_CHECK_ARG(a->n >= 0 && a->max_start >= 0 && (int64_t)a->max_start + a->n <= a->cache.max_seq,
                "max_start + n exceeds max_seq");
  LBX_CHECK_ARG(a->dtype == LBX_F32 || a->dtype == LBX_BF16, "bad dtype");
  if (a->n == 0) return LBX_OK;
  LBX_CHECK_ARG(a->k_new && a->v_new, "NULL pointer");
  LBX_CHECK_ARG(a->kv_ld >= (int64_t)a->cache.kv_heads * a->cache.head_dim, "rows overlap");
  p.n = a->n;
  p.max_start = a->max_start;
  p.dtype = a->dtype;
  p.start = a->start;
  p.k = a->k_new;
  p.v = a->v_new;
  p.ld = a->kv_ld;
  p.rope = reinterpret_cast<const float2 *>(a->rope_cs);
  const int64_t items = 2ll * a->cache.n_seq * a->n * a->cache.kv_heads;
  LBX_CHECK_SUP((items + 7) / 8 <= 0x7fffffff, "too many rows");
  const dim3 grid((unsigned)((items + 7) / 8));
  const cudaError_t e = a->cache.head_dim == 128
                            ? launch(kv4_append_kernel<128>, grid, dim3(256), 0, stream, a->use_pdl != 0, p)
                            : launch(kv4_append_kernel<64>, grid, dim3(256), 0, stream, a->use_pdl != 0, p);
  return cuda_status(e, "kv4_append launch");
}

extern "C" int lbx_kv4_read(const lbx_kv4_cache *c, const int32_t *start, int32_t max_start, int32_t n, float *k,
                            float *v, cudaStream_t stream) {
  using namespace lbx;
  LBX_CHECK_ARG(c, "cache is NULL");
  Kv4ReadParams p = {};
  const int rc = kv4_view(*c, p.c);
  if (rc) return rc;
  LBX_CHECK_ARG(n >= 0 && max_start >= 0 && (int64_t)max_start + n <= c->max_seq, "max_start + n exceeds max_seq");
  if (n == 0 || (!k && !v)) return LBX_OK;
  LBX_CHECK_ARG(aligned16(k) && aligned16(v), "outputs must be 16-byte aligned");
  p.n = n;
  p.max_start = max_start;
  p.start = start;
  p.out[0] = k;
  p.out[1] = v;
  const int64_t items = (int64_t)c->n_seq * c->kv_heads * n * (c->head_dim / 8);
  LBX_CHECK_SUP((items + 255) / 256 <= 0x7fffffff, "too many rows");
  const dim3 grid((unsigned)((items + 255) / 256), 2);
  if (c->head_dim == 128)
    kv4_read_kernel<128><<<grid, 256, 0, stream>>>(p);
  else
    kv4_read_kernel<64><<<grid, 256, 0, stream>>>(p);
  return cuda_status(cudaGetLastError(), "kv4_read launch");
}

extern "C" size_t lbx_kv4_attn_workspace_size(const lbx_kv4_attn_args *a) {
  lbx::Kv4AttnParams p = {};
  if (lbx::kv4_attn_prep(a, p)) return 0;
  return 256;
}

extern "C" int lbx_kv4_attn(const lbx_kv4_attn_args *a, void *ws, size_t ws_bytes, cudaStream_t stream) {
  using namespace lbx;
  Kv4AttnParams p = {};
  const int rc = kv4_attn_prep(a, p);
  if (rc) return rc;
  LBX_CHECK_ARG(a->q && a->out, "NULL pointer");
  LBX_CHECK_ARG(ws && ws_bytes >= 256, "workspace too small");
  const int64_t rows = (int64_t)a->cache.n_seq * a->n;
  LBX_CHECK_SUP(rows <= 65535, "too many query rows");
  const dim3 grid(a->heads, (unsigned)rows);
  if (a->cache.head_dim == 128)
    kv4_attn_simple_kernel<128><<<grid, 128, 0, stream>>>(p);
  else
    kv4_attn_simple_kernel<64><<<grid, 128, 0, stream>>>(p);
  return cuda_status(cudaGetLastError(), "kv4_attn launch");
}
