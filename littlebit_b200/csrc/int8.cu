// Matrix product in 8-bit integers, a scale for each token and each channel:
//
//   y_tn = s_t * w_n * sum_k c_tk W_nk (+ b_n),   c_tk = rint(x_tk * 127 / a_t),
//   a_t = max_k |x_tk|,  s_t = a_t / 127
//
// The sums are exact int32 (127 * 128 * 131072 < 2^31), so every split of the
// work gives the same bits.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "tcgen05.cuh"

namespace lbx {

constexpr int Q8_THREADS = 256;
constexpr int Q8_MAXK = 131072;

// one CTA per row: the absolute maximum, then the codes
__global__ void __launch_bounds__(Q8_THREADS) quant_tokens_kernel(const void *__restrict__ x, int xdt, int64_t x_ld,
                                                                  int k, int8_t *__restrict__ q, int64_t q_ld,
                                                                  float *__restrict__ scale) {
  __shared__ uint32_t red[Q8_THREADS / 32];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  pdl_wait();
  pdl_trigger();  // (a kernel that starts early may count on all that came before this one)
  // |x| as an integer: the order of the non-negative floats, infinities and
  // NaNs (0x7f800000 and up) above every number
  uint32_t m = 0;
  for (int i = tid; i < k; i += Q8_THREADS) {
    const uint32_t b = __float_as_uint(load_act(x, xdt, row * x_ld + i)) & 0x7FFFFFFFu;
    m = max(m, b);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((tid & 31) == 0) red[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Q8_THREADS / 32; ++i) m = max(m, red[i]);
  const bool fin = m < 0x7F800000u;
  const float a = __uint_as_float(m);
  const float inv = fin && a > 0.f ? __fdiv_rn(127.0f, a) : 0.f;
  if (tid == 0) scale[row] = fin ? __fmul_rn(a, 1.0f / 127.0f) : __uint_as_float(0x7FC00000u);
  for (int i = tid; i < k; i += Q8_THREADS) {
    const float v = load_act(x, xdt, row * x_ld + i);
    q[row * q_ld + i] = (int8_t)(fin ? __float2int_rn(__fmul_rn(v, inv)) : 0);
  }
}

// ---------------------------------------------------------------------------
// Product on the tensor cores (tcgen05.mma kind::i8, int32 sums in TMEM).
//
// A CTA's tile is 128 channels (operand A: the weights) x BN tokens (operand
// B, BN = 16, or a multiple of 32 up to 256), K in blocks of 128 bytes that TMA
// lands in 128-byte swizzle; out-of-range rows and bytes arrive as zeros, so odd
// sizes need no other care.  A lane of the accumulator is a channel, a column a
// token: each column's store is 128 consecutive results.
//
// Tiles are dealt to one persistent CTA an SM: whole rounds of tiles first
// ("full"), and what does not fill a round (everything, for few tiles) is cut
// into equal runs of K blocks over the CTAs ("rest"), so that a single token's
// 250 tiles keep all SMs streaming.  A tile that is cut leaves its parts as
// int32 in the workspace and the CTA that completes it adds them: the
// sums are exact, so neither the cut nor the order shows in the result.
// ---------------------------------------------------------------------------
constexpr int I8_THREADS = 192;   // warp 0: copies, warp 1: MMA, warps 2-5: results
constexpr int I8_KB = 128;        // K bytes a block
constexpr int I8_MAXST = 12;      // stages at most
constexpr int I8_MAXCTA = 1024;   // ticket words
constexpr int I8_MINBLK = 4;      // K blocks a CTA takes of the rest, at least

struct I8Params {
  int m, n, KB;
  int TN, TM, BN;      // channel tiles, token tiles, tokens a tile
  int full, T;         // tiles of whole rounds, all tiles
  int G, Gr;           // CTAs, CTAs that share the rest
  int64_t rb;          // K blocks of the rest
  int ST;              // stages
  uint32_t idesc, tcols;
  const float *s, *ws, *bias;
  void *y; int64_t y_ld; int ydt;
  int32_t *part;       // [CTA][2][BN][128] parts of cut tiles
  unsigned *ticket;    // [T - full] K blocks arrived, zero between calls
};

// a CTA's pieces: its run of the rest, then its whole tiles
struct I8Pieces {
  int64_t r0, r1;
  int t, G, full, KB;
  LBX_DEV I8Pieces(const I8Params &p, int c) : r0(0), r1(0), t(c), G(p.G), full(p.full), KB(p.KB) {
    if (c < p.Gr) {
      r0 = p.rb * c / p.Gr;
      r1 = p.rb * (c + 1) / p.Gr;
    }
  }
  LBX_DEV bool next(int &tile, int &k0, int &k1) {
    if (r0 < r1) {
      const int64_t q = r0 / KB;
      tile = full + (int)q;
      k0 = (int)(r0 - q * KB);
      k1 = (int)min((int64_t)KB, k0 + (r1 - r0));
      r0 += k1 - k0;
      return true;
    }
    if (t < full) {
      tile = t;
      k0 = 0;
      k1 = KB;
      t += G;
      return true;
    }
    return false;
  }
};

// tile -> (channel tile, token tile): groups of 16 token tiles, so that the
// tiles of a round share few weight and few token rows (both stay in L2)
constexpr int I8_GT = 16;
LBX_DEV void i8_tile(const I8Params &p, int tile, int &tn, int &tm) {
  const int g = tile / (p.TN * I8_GT), gs = min(I8_GT, p.TM - g * I8_GT), r = tile - g * p.TN * I8_GT;
  tn = r / gs;
  tm = g * I8_GT + (r - tn * gs);
}

LBX_DEV void tma_2d(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

LBX_DEV void i8_store(const I8Params &p, int64_t t, int ch, int acc, float wsc, float b, bool has_b) {
  float v = __int2float_rn(acc) * __ldcg(p.s + t) * wsc;
  if (has_b) v += b;
  if (p.ydt == LBX_F32) reinterpret_cast<float *>(p.y)[t * p.y_ld + ch] = v;
  else reinterpret_cast<uint16_t *>(p.y)[t * p.y_ld + ch] = f32_to_bf16(v);
}

__global__ void __launch_bounds__(I8_THREADS, 1)
    linear_int8_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
                       const __grid_constant__ I8Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *sm = align1024(smem_raw);
  __shared__ __align__(8) uint64_t full[I8_MAXST], empty[I8_MAXST], tfull[2], tempty[2], drain;
  __shared__ uint32_t tbase;
  __shared__ int abort_flag, s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
  const int abytes = 128 * I8_KB, bbytes = p.BN * I8_KB, stage = abytes + bbytes;
  volatile int *abrt = &abort_flag;
  if (tid == 0) {
    for (int i = 0; i < p.ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 4);
    }
    mbar_init(&drain, 1);
    fence_mbar_init();
    abort_flag = 0;
  }
  if (warp == 1) tmem_alloc(&tbase, p.tcols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tbase, tbuf = p.tcols / 2;

  if (warp == 0 && lane == 0) {
    // ---- copies.  The weights do not come from the kernel before this one:
    // the first stages' are on their way before its codes are waited for.
    auto load_w = [&](int j, int tile, int kb) {
      int tn, tm;
      i8_tile(p, tile, tn, tm);
      uint8_t *d = sm + (j % p.ST) * stage;
      mbar_arrive_expect_tx(&full[j % p.ST], (uint32_t)stage);
      tma_2d(d, &tw, kb * I8_KB, tn * 128, &full[j % p.ST]);
    };
    auto load_x = [&](int j, int tile, int kb) {
      int tn, tm;
      i8_tile(p, tile, tn, tm);
      tma_2d(sm + (j % p.ST) * stage + abytes, &tx, kb * I8_KB, tm * p.BN, &full[j % p.ST]);
    };
    int tile, k0, k1, j = 0;
    {
      I8Pieces pre(p, cta);
      while (j < p.ST && pre.next(tile, k0, k1))
        for (int kb = k0; kb < k1 && j < p.ST; ++kb) load_w(j++, tile, kb);
    }
    const int npre = j;
    pdl_wait();
    I8Pieces it(p, cta);
    j = 0;
    bool ok = true;
    while (ok && it.next(tile, k0, k1)) {
      for (int kb = k0; kb < k1; ++kb, ++j) {
        if (j >= npre) {
          if (!wd_wait(&empty[j % p.ST], (uint32_t)(j / p.ST - 1) & 1u, 0x821, abrt)) {
            ok = false;
            break;
          }
          load_w(j, tile, kb);
        }
        load_x(j, tile, kb);
      }
    }
    if (*abrt) {  // copies in flight land before shared memory is given up
      int none = 0;
      for (int i = max(0, j - p.ST); i < j; ++i) wd_wait(&full[i % p.ST], (uint32_t)(i / p.ST) & 1u, 0x822, &none);
    }
  } else if (warp == 1 && lane == 0) {
    // ---- MMA
    I8Pieces it(p, cta);
    int tile, k0, k1, j = 0, n = 0;
    bool ok = true;
    while (ok && it.next(tile, k0, k1)) {
      const uint32_t d = tmem + (uint32_t)(n & 1) * tbuf;
      if (n >= 2 && !wd_wait(&tempty[n & 1], (uint32_t)(n / 2 - 1) & 1u, 0x823, abrt)) break;
      tc_fence_after();
      for (int kb = k0; kb < k1; ++kb, ++j) {
        if (!wd_wait(&full[j % p.ST], (uint32_t)(j / p.ST) & 1u, 0x824, abrt)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a = smem_u32(sm + (j % p.ST) * stage), b = a + (uint32_t)abytes;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          umma_i8(d, sw128_desc(a + 32 * q), sw128_desc(b + 32 * q), p.idesc, kb > k0 || q > 0 ? 1u : 0u);
        umma_commit(&empty[j % p.ST]);
      }
      if (ok) umma_commit(&tfull[n & 1]);
      ++n;
    }
    if (*abrt) {  // products in flight end before TMEM is given up
      int none = 0;
      umma_commit(&drain);
      wd_wait(&drain, 0, 0x825, &none);
    }
  } else if (warp >= 2) {
    // ---- results: this warp's lane quarter is warp % 4
    pdl_wait();
    const int row = 32 * (warp & 3) + lane;
    const uint32_t lq = (uint32_t)(32 * (warp & 3)) << 16;
    I8Pieces it(p, cta);
    int tile, k0, k1, n = 0;
    while (it.next(tile, k0, k1)) {
      // (after a wait that gave up all four warps still go through the same
      // barriers: the pieces left then pass at once, and the call has failed)
      wd_wait(&tfull[n & 1], (uint32_t)(n / 2) & 1u, 0x826, abrt);
      __syncwarp();
      tc_fence_after();
      int tn, tm;
      i8_tile(p, tile, tn, tm);
      const int ch = tn * 128 + row, t0 = tm * p.BN, nc = min(p.BN, p.m - t0);
      const bool cok = ch < p.n, whole = k0 == 0 && k1 == p.KB, hb = p.bias != nullptr;
      const float wsc = cok ? p.ws[ch] : 0.f, bs = cok && hb ? p.bias[ch] : 0.f;
      int32_t *slot = p.part + ((int64_t)cta * 2 + (k0 > 0 ? 0 : 1)) * 128 * p.BN;
      const uint32_t ta = tmem + (uint32_t)(n & 1) * tbuf + lq;
      for (int c0 = 0; c0 < nc; c0 += 16) {
        uint32_t r[16];
        tmem_ld<16>(ta + c0, r);
        tmem_ld_wait();
        if (whole) {
          if (cok) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (c0 + j < nc) i8_store(p, t0 + c0 + j, ch, (int)r[j], wsc, bs, hb);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < nc) __stcg(slot + (c0 + j) * 128 + row, (int)r[j]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive1(&tempty[n & 1]);
      ++n;
      if (whole) continue;
      // the part is out; the CTA whose part completes the tile adds them all
      __threadfence();
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (tid == 64) {
        const unsigned old = atomicAdd(p.ticket + (tile - p.full), (unsigned)(k1 - k0));
        s_last = old + (unsigned)(k1 - k0) == (unsigned)p.KB;
        if (s_last) p.ticket[tile - p.full] = 0u;  // ready for the next call
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (!s_last) continue;
      __threadfence();
      const int64_t base = (int64_t)(tile - p.full) * p.KB;
      int cl = (int)(base * p.Gr / p.rb);  // the first CTA with K blocks of this tile
      while (cl > 0 && p.rb * cl / p.Gr > base) --cl;
      while (p.rb * (cl + 1) / p.Gr <= base) ++cl;
      for (int c0 = 0; c0 < nc; c0 += 16) {
        int acc[16] = {};
        for (int c = cl; c < p.Gr; ++c) {
          const int64_t b0 = p.rb * c / p.Gr;
          if (b0 >= base + p.KB) break;
          const int32_t *ps = p.part + ((int64_t)c * 2 + (b0 > base ? 0 : 1)) * 128 * p.BN;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < nc) acc[j] += __ldcg(ps + (c0 + j) * 128 + row);
        }
        if (cok) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < nc) i8_store(p, t0 + c0 + j, ch, acc[j], wsc, bs, hb);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, p.tcols);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// the split of a call, and its workspace: [tickets, at a fixed place][parts][scales][codes]
struct I8Plan {
  I8Params p;
  size_t part, s, q, total;
  int64_t q_ld;
};
static I8Plan i8_plan(int m, int n, int k) {
  auto al = [](size_t v) { return (v + 255) & ~(size_t)255; };
  I8Plan w = {};
  I8Params &p = w.p;
  p.m = m;
  p.n = n;
  p.KB = (k + I8_KB - 1) / I8_KB;
  p.TN = (n + 127) / 128;
  p.TM = (m + 255) / 256;
  const int per = (m + p.TM - 1) / p.TM;
  p.BN = per <= 16 ? 16 : (per + 31) / 32 * 32;
  p.idesc = idesc_i8(p.BN);
  p.tcols = 32;
  while (p.tcols < 2u * p.BN) p.tcols *= 2;
  p.G = std::min(device_sm_count(), I8_MAXCTA);
  p.T = p.TN * p.TM;
  p.full = p.T / p.G * p.G;
  p.rb = (int64_t)(p.T - p.full) * p.KB;
  p.Gr = (int)std::min<int64_t>(p.G, std::max<int64_t>(1, p.rb / I8_MINBLK));
  if (p.full == 0) p.G = p.Gr;
  w.part = al((size_t)I8_MAXCTA * 4);
  w.s = w.part + al((size_t)p.Gr * 2 * 128 * p.BN * 4);
  w.q = w.s + al((size_t)m * 4);
  w.q_ld = (k + 15) & ~15;
  w.total = w.q + al((size_t)m * w.q_ld);
  return w;
}

// a [rows, k] int8 matrix in boxes of `box` rows x 128 bytes, 128-byte swizzle
static int i8_map(CUtensorMap *map, const void *base, int64_t rows, int k, int64_t ld, int box) {
  static DevCache<PFN_cuTensorMapEncodeTiled_v12000> fn;
  PFN_cuTensorMapEncodeTiled_v12000 enc = nullptr;
  const int rc = fn.get(enc, [](PFN_cuTensorMapEncodeTiled_v12000 &f) {
    void *v = nullptr;
    cudaDriverEntryPointQueryResult st;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &v, 12000, cudaEnableDefault, &st);
    if (e != cudaSuccess) return cuda_status(e, "cuTensorMapEncodeTiled lookup");
    if (!v) {
      set_error("the driver has no cuTensorMapEncodeTiled");
      return (int)LBX_EUNSUPPORTED;
    }
    f = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(v);
    return (int)LBX_OK;
  });
  if (rc) return rc;
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
  const cuuint32_t bx[2] = {(cuuint32_t)I8_KB, (cuuint32_t)box}, es[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, bx, es,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
    return LBX_ECUDA;
  }
  return LBX_OK;
}

static int quant_tokens_launch(const void *x, int xdt, int64_t x_ld, int m, int k, int8_t *q, int64_t q_ld,
                               float *scale, bool pdl, cudaStream_t stream) {
  return cuda_status(launch(quant_tokens_kernel, dim3(m), dim3(Q8_THREADS), 0, stream, pdl, x, xdt, x_ld, k, q, q_ld, scale),
                     "quant_tokens launch");
}

}  // namespace lbx

extern "C" int lbx_quant_tokens(const void *x, int32_t x_dtype, int64_t x_ld, int32_t m, int32_t k, int8_t *q,
                                int64_t q_ld, float *scale, cudaStream_t stream) {
  using namespace lbx;
  LBX_CHECK_ARG(m >= 0 && k >= 1, "bad shape");
  LBX_CHECK_ARG(x_dtype == LBX_F32 || x_dtype == LBX_BF16, "bad dtype");
  LBX_CHECK_ARG(x_ld >= k && q_ld >= k, "row strides must be at least k");
  if (m == 0) return LBX_OK;
  LBX_CHECK_ARG(x && q && scale, "NULL pointer");
  return quant_tokens_launch(x, x_dtype, x_ld, m, k, q, q_ld, scale, false, stream);
}

extern "C" size_t lbx_linear_int8_workspace_size(int32_t m, int32_t n, int32_t k) {
  if (m < 1 || n < 1 || k < 1) return 0;
  return lbx::i8_plan(m, n, k).total;
}

extern "C" int lbx_linear_int8(const lbx_int8_args *a, void *ws, size_t ws_bytes, cudaStream_t stream) {
  using namespace lbx;
  LBX_CHECK_ARG(a, "args is NULL");
  LBX_CHECK_ARG(a->m >= 0 && a->n >= 1 && a->k >= 1, "bad shape");
  LBX_CHECK_SUP(a->k <= Q8_MAXK, "k must be <= %d", Q8_MAXK);
  LBX_CHECK_ARG((a->x_dtype == LBX_F32 || a->x_dtype == LBX_BF16) && (a->y_dtype == LBX_F32 || a->y_dtype == LBX_BF16),
                "bad dtype");
  if (a->m == 0) return LBX_OK;
  LBX_CHECK_ARG(a->x && a->w && a->w_scale && a->y, "NULL pointer");
  LBX_CHECK_ARG(a->x_ld >= a->k && a->w_ld >= a->k && a->y_ld >= a->n, "row strides smaller than the rows");
  LBX_CHECK_ARG(aligned16(a->w) && a->w_ld % 16 == 0, "weight rows must start on 16 bytes");
  I8Plan W = i8_plan(a->m, a->n, a->k);
  LBX_CHECK_ARG(ws && ws_bytes >= W.total, "workspace too small (%zu < %zu)", ws_bytes, W.total);
  LBX_CHECK_ARG(aligned16(ws), "the workspace must be 16-byte aligned");
  uint8_t *b = reinterpret_cast<uint8_t *>(ws);
  int8_t *q = reinterpret_cast<int8_t *>(b + W.q);
  float *s = reinterpret_cast<float *>(b + W.s);
  I8Params &p = W.p;
  static DevCache<size_t> smax_cache;
  size_t smax = 0;
  int rc = smax_cache.get(smax, [](size_t &out) {
    return cuda_status(allow_max_smem(linear_int8_kernel, &out), "linear_int8 smem attribute");
  });
  if (rc) return rc;
  const int stage = (128 + p.BN) * I8_KB;
  p.ST = std::min(I8_MAXST, (int)((smax - 1024) / stage));
  p.s = s;
  p.ws = a->w_scale;
  p.bias = a->bias;
  p.y = a->y;
  p.y_ld = a->y_ld;
  p.ydt = a->y_dtype;
  p.part = reinterpret_cast<int32_t *>(b + W.part);
  p.ticket = reinterpret_cast<unsigned *>(b);
  CUtensorMap tw, tx;
  rc = i8_map(&tw, a->w, a->n, a->k, a->w_ld, 128);
  if (rc) return rc;
  rc = i8_map(&tx, q, a->m, a->k, W.q_ld, p.BN);
  if (rc) return rc;
  rc = quant_tokens_launch(a->x, a->x_dtype, a->x_ld, a->m, a->k, q, W.q_ld, s, a->use_pdl != 0, stream);
  if (rc) return rc;
  return cuda_status(launch(linear_int8_kernel, dim3(p.G), dim3(I8_THREADS), (size_t)p.ST * stage + 1024, stream, true, tw,
                            tx, p),
                     "linear_int8 launch");
}
