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
constexpr int Q8_MAXDIM = 1 << 30;  // tokens, channels, features of a row: indexes past the end stay 32-bit numbers

// One CTA a row: the absolute maximum, then the codes.  VEC: 16-byte loads, up to
// Q8_NR of them held in registers from the first pass to the second (rows of up
// to 8192 float / 16384 bf16 values are read once; what is longer is read again,
// from L2).  The kernel is one round trip to memory and two block barriers long (one
// row of 4096: 5.5 us by itself, 320 rows of 8192 6.7); 4096 bf16 rows of 8192, 101 MB, 24 us,
// are bound by instructions.
constexpr int Q8_NR = 8;
LBX_DEV uint32_t q8_abs(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
LBX_DEV uint32_t q8_code(float v, float inv, bool fin) {
  return fin ? (uint32_t)(__float2int_rn(__fmul_rn(v, inv)) & 255) : 0u;
}
template <int XDT>
LBX_DEV void q8_unpack(const uint4 &r, float *v) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (XDT == LBX_F32) {
      v[i] = __uint_as_float(w[i]);
    } else {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
}

template <int XDT, bool VEC>
__global__ void __launch_bounds__(Q8_THREADS) quant_tokens_kernel(const void *__restrict__ x, int64_t x_ld, int k,
                                                                  int8_t *__restrict__ q, int64_t q_ld,
                                                                  float *__restrict__ scale) {
  constexpr int E = XDT == LBX_F32 ? 4 : 8, ES = 16 / E;
  __shared__ uint32_t red[Q8_THREADS / 32];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  pdl_wait();
  pdl_trigger();  // (a kernel that starts early may count on all that came before this one)
  const uint8_t *xr = reinterpret_cast<const uint8_t *>(x) + row * x_ld * ES;
  const uint4 *xv = reinterpret_cast<const uint4 *>(xr);
  int8_t *qr = q + row * q_ld;
  const int nv = VEC ? k / E : 0;
  uint4 r[Q8_NR];
  // |x| as an integer: the order of the non-negative floats, infinities and
  // NaNs (0x7f800000 and up) above every number
  uint32_t m = 0;
  float v[E];
#pragma unroll
  for (int i = 0; i < Q8_NR; ++i) {
    const int e = tid + i * Q8_THREADS;
    r[i] = make_uint4(0u, 0u, 0u, 0u);
    if (e < nv) r[i] = __ldg(xv + e);
  }
#pragma unroll
  for (int i = 0; i < Q8_NR; ++i) {
    q8_unpack<XDT>(r[i], v);
#pragma unroll
    for (int j = 0; j < E; ++j) m = max(m, q8_abs(v[j]));
  }
  for (int e = tid + Q8_NR * Q8_THREADS; e < nv; e += Q8_THREADS) {
    q8_unpack<XDT>(__ldg(xv + e), v);
#pragma unroll
    for (int j = 0; j < E; ++j) m = max(m, q8_abs(v[j]));
  }
  for (int i = nv * E + tid; i < k; i += Q8_THREADS) m = max(m, q8_abs(load_act(xr, XDT, i)));
  m = __reduce_max_sync(0xffffffffu, m);
  if ((tid & 31) == 0) red[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Q8_THREADS / 32; ++i) m = max(m, red[i]);
  const bool fin = m < 0x7F800000u;
  const float a = __uint_as_float(m);
  float inv = fin && a > 0.f ? __fdiv_rn(127.0f, a) : 0.f;
  if (!(inv < INFINITY)) inv = 0.f;  // (a below 127 / FLT_MAX: the row is 0, as a 4-bit group with so small a step)
  if (tid == 0) scale[row] = fin ? __fmul_rn(a, 1.0f / 127.0f) : __uint_as_float(0x7FC00000u);
  auto put = [&](int e, const uint4 &w) {
    q8_unpack<XDT>(w, v);
    uint32_t c[E / 4];
#pragma unroll
    for (int j = 0; j < E / 4; ++j)
      c[j] = q8_code(v[4 * j], inv, fin) | q8_code(v[4 * j + 1], inv, fin) << 8 | q8_code(v[4 * j + 2], inv, fin) << 16 |
             q8_code(v[4 * j + 3], inv, fin) << 24;
    if constexpr (E == 4) reinterpret_cast<uint32_t *>(qr)[e] = c[0];
    else reinterpret_cast<uint2 *>(qr)[e] = make_uint2(c[0], c[1]);
  };
#pragma unroll
  for (int i = 0; i < Q8_NR; ++i)
    if (tid + i * Q8_THREADS < nv) put(tid + i * Q8_THREADS, r[i]);
  for (int e = tid + Q8_NR * Q8_THREADS; e < nv; e += Q8_THREADS) put(e, __ldg(xv + e));
  for (int i = nv * E + tid; i < k; i += Q8_THREADS) qr[i] = (int8_t)q8_code(load_act(xr, XDT, i), inv, fin);
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
// The work is dealt to one persistent CTA an SM in one of three ways, whichever
// i8_plan() reckons the cheapest:
//   rounds  whole tiles, round after round
//   cut     whole rounds, and the tiles that do not fill a round cut into equal
//           runs of K blocks over the CTAs.  A cut tile leaves its parts as int32
//           in the workspace and the CTA that completes it adds them: the sums
//           are exact, so neither the cut nor the order shows in the result.
//   even    one token tile: the channels dealt evenly in units of 32, a CTA's
//           share in tiles of up to 128 (rows past it are multiplied and not
//           stored).  For few tokens, where the weights' stream is the time:
//           32000 channels are 7 units for each of 148 CTAs, nothing is joined.  Joining
//           cost 10 us there: under a saturated memory a fence, an atomic or a
//           load takes as long as the queue of loads ahead of it.
//
// Bound for few tokens by the weights' stream and what comes before it: 1 x 32000 x 4096, 131 MB,
// 28.4 us with the quantiser; twice and four times the bytes (8 x 32000 x 8192, x 16384) 50.7 and
// 94.3: 6.0 TB/s for what is added, and 6.6 us for the quantiser, the first loads and the last results.
// For many by the copies from L2 and the clock that the power leaves: a block of 128 x 256 brings
// 48 KB for 512 cycles of MMA and takes 730 (4096 x 28672 x 8192: 701 us by itself, 793 to 833 in a row of
// calls, 2.74 POP/s, tensor pipes busy 70 % of cycles).
// Two channel tiles at once from one CTA, a token tile loaded once for both, was slower
// (1020 us for 897 then: half the stages).
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
  int units;           // "even": units of 32 channels; else 0
  int64_t rb;          // K blocks of the rest
  int ST, KS;          // stages, K blocks a stage
  uint32_t idesc, tcols;
  const float *s, *ws, *bias;
  void *y; int64_t y_ld; int ydt;
  int32_t *part;       // [CTA][2][BN][128] parts of cut tiles
  unsigned *ticket;    // [T - full] K blocks arrived, zero between calls
};

// a CTA's pieces: its run of the rest, then its whole tiles; or its even share
// tile -> (channel tile, token tile): groups of 16 token tiles, so that the
// tiles of a round share few weight and few token rows (both stay in L2)
constexpr int I8_GT = 16;
struct I8Piece {
  int tile, k0, k1;
  int ch0, rows, t0;  // first channel, channels, first token
};
struct I8Pieces {
  const I8Params &p;
  int64_t r0, r1;
  int t, u, u1;
  LBX_DEV I8Pieces(const I8Params &p, int c) : p(p), r0(0), r1(0), t(c), u(0), u1(0) {
    if (p.units) {
      u = (int)((int64_t)p.units * c / p.G);
      u1 = (int)((int64_t)p.units * (c + 1) / p.G);
    } else if (c < p.Gr) {
      r0 = p.rb * c / p.Gr;
      r1 = p.rb * (c + 1) / p.Gr;
    }
  }
  LBX_DEV bool next(I8Piece &e) {
    e.k0 = 0;
    e.k1 = p.KB;
    if (p.units) {
      if (u >= u1) return false;
      e.tile = 0;
      e.t0 = 0;
      e.ch0 = 32 * u;
      const int nu = min(4, u1 - u);
      e.rows = 32 * nu;
      u += nu;
      return true;
    }
    if (r0 < r1) {
      const int64_t q = r0 / p.KB;
      e.tile = p.full + (int)q;
      e.k0 = (int)(r0 - q * p.KB);
      e.k1 = (int)min((int64_t)p.KB, e.k0 + (r1 - r0));
      r0 += e.k1 - e.k0;
    } else if (t < p.full) {
      e.tile = t;
      t += p.G;
    } else {
      return false;
    }
    const int g = e.tile / (p.TN * I8_GT), gs = min(I8_GT, p.TM - g * I8_GT), r = e.tile - g * p.TN * I8_GT;
    const int tn = r / gs;
    e.ch0 = 128 * tn;
    e.rows = 128;
    e.t0 = p.BN * (g * I8_GT + (r - tn * gs));
    return true;
  }
};

LBX_DEV void tma_2d(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

// Results of 16 tokens from t on (nc of them in range) at channel ch; ts: the
// tokens' scales, in shared memory since the piece began.  (A load from L2 behind a store
// to memory that may be the same waits for its turn: one a token, 256 x 700 cycles a
// tile, held the whole kernel at a quarter of its rate.)
LBX_DEV void i8_store16(const I8Params &p, const float *ts, int64_t t, int nc, int ch, const int *acc, float wsc, float b,
                        bool has_b) {
  float v[16];
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    const float4 s = *reinterpret_cast<const float4 *>(ts + j);
    v[j] = s.x;
    v[j + 1] = s.y;
    v[j + 2] = s.z;
    v[j + 3] = s.w;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    v[j] = __int2float_rn(acc[j]) * v[j] * wsc;
    if (has_b) v[j] += b;
  }
  if (p.ydt == LBX_F32) {
    float *y = reinterpret_cast<float *>(p.y) + t * p.y_ld + ch;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < nc) y[j * p.y_ld] = v[j];
  } else {
    uint16_t *y = reinterpret_cast<uint16_t *>(p.y) + t * p.y_ld + ch;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < nc) y[j * p.y_ld] = f32_to_bf16(v[j]);
  }
}

// ONE: one K block a stage (known, the copying and issuing threads have no inner
// loops: each is one thread with some 500 cycles a block)
template <bool ONE>
__global__ void __launch_bounds__(I8_THREADS, 1)
    linear_int8_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tw32,
                       const __grid_constant__ CUtensorMap tx, const __grid_constant__ I8Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *sm = align1024(smem_raw);
  __shared__ __align__(8) uint64_t full[I8_MAXST], empty[I8_MAXST], tfull[2], tempty[2], drain;
  __shared__ uint32_t tbase;
  __shared__ int abort_flag, s_last;
  __shared__ __align__(16) float tsc[2][256];  // the piece's token scales, and the next one's
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
  // a stage: KS tiles of weights, then KS of tokens
  const int KS = ONE ? 1 : p.KS;
  const int abytes = 128 * I8_KB, bbytes = p.BN * I8_KB, stage = KS * (abytes + bbytes), boff = KS * abytes;
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
    auto load_w = [&](int st, const I8Piece &e, int kb) {
      const int nk = min(KS, e.k1 - kb);
      mbar_arrive_expect_tx(&full[st], (uint32_t)(nk * (e.rows * I8_KB + bbytes)));
      for (int i = 0; i < nk; ++i) {
        uint8_t *d = sm + st * stage + i * abytes;
        if (e.rows == 128) {
          tma_2d(d, &tw, (kb + i) * I8_KB, e.ch0, &full[st]);
        } else {
          for (int r = 0; r < e.rows; r += 32) tma_2d(d + r * I8_KB, &tw32, (kb + i) * I8_KB, e.ch0 + r, &full[st]);
        }
      }
    };
    I8Piece e;
    int j = 0;
    {
      I8Pieces pre(p, cta);
      while (j < p.ST && pre.next(e))
        for (int kb = e.k0; kb < e.k1 && j < p.ST; kb += KS) load_w(j++, e, kb);
    }
    const int npre = j;
    pdl_wait();
    I8Pieces it(p, cta);
    int st = 0;
    uint32_t ph = 1;  // parity of the stage's last release
    j = 0;
    bool ok = true;
    while (ok && it.next(e)) {
      for (int kb = e.k0; kb < e.k1; kb += KS, ++j) {
        if (j >= npre) {
          if (!wd_wait(&empty[st], ph, 0x821, abrt)) {
            ok = false;
            break;
          }
          load_w(st, e, kb);
        }
        for (int i = 0; i < KS && kb + i < e.k1; ++i)
          tma_2d(sm + st * stage + boff + i * bbytes, &tx, (kb + i) * I8_KB, e.t0, &full[st]);
        if (++st == p.ST) {
          st = 0;
          ph ^= 1u;
        }
      }
    }
    if (*abrt) {  // copies in flight land before shared memory is given up
      int none = 0;
      for (int i = max(0, j - p.ST); i < j; ++i) wd_wait(&full[i % p.ST], (uint32_t)(i / p.ST) & 1u, 0x822, &none);
    }
  } else if (warp == 1 && lane == 0) {
    // ---- MMA
    I8Pieces it(p, cta);
    I8Piece e;
    int n = 0, st = 0;
    uint32_t ph = 0;
    bool ok = true;
    while (ok && it.next(e)) {
      const uint32_t d = tmem + (uint32_t)(n & 1) * tbuf;
      if (n >= 2 && !wd_wait(&tempty[n & 1], (uint32_t)(n / 2 - 1) & 1u, 0x823, abrt)) break;
      tc_fence_after();
      for (int kb = e.k0; kb < e.k1; kb += KS) {
        if (!wd_wait(&full[st], ph, 0x824, abrt)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint64_t a = sw128_desc(smem_u32(sm + st * stage)), b = sw128_desc(smem_u32(sm + st * stage + boff));
        for (int i = 0; i < KS && kb + i < e.k1; ++i, a += abytes >> 4, b += bbytes >> 4) {
#pragma unroll
          for (int q = 0; q < 4; ++q)  // (32 bytes on: 2 in the descriptors' address units)
            umma_i8(d, a + 2 * q, b + 2 * q, p.idesc, kb + i > e.k0 || q > 0 ? 1u : 0u);
        }
        umma_commit(&empty[st]);
        if (++st == p.ST) {
          st = 0;
          ph ^= 1u;
        }
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
    I8Piece e;
    int n = 0;
    while (it.next(e)) {
      float *ts = tsc[n & 1];
      for (int c = tid - 64; c < min(p.BN, p.m - e.t0); c += 128) ts[c] = __ldcg(p.s + e.t0 + c);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      // (after a wait that gave up all four warps still go through the same
      // barriers: the pieces left then pass at once, and the call has failed)
      wd_wait(&tfull[n & 1], (uint32_t)(n / 2) & 1u, 0x826, abrt);
      __syncwarp();
      tc_fence_after();
      const int tile = e.tile, k0 = e.k0, k1 = e.k1;
      const int ch = e.ch0 + row, t0 = e.t0, nc = min(p.BN, p.m - t0);
      const bool cok = row < e.rows && ch < p.n, whole = k0 == 0 && k1 == p.KB, hb = p.bias != nullptr;
      const float wsc = cok ? p.ws[ch] : 0.f, bs = cok && hb ? p.bias[ch] : 0.f;
      int32_t *slot = p.part + ((int64_t)cta * 2 + (k0 > 0 ? 0 : 1)) * 128 * p.BN;
      const uint32_t ta = tmem + (uint32_t)(n & 1) * tbuf + lq;
      for (int c0 = 0; c0 < nc; c0 += 16) {
        uint32_t r[16];
        tmem_ld<16>(ta + c0, r);
        tmem_ld_wait();
        if (whole) {
          if (cok) i8_store16(p, ts + c0, t0 + c0, nc - c0, ch, reinterpret_cast<const int *>(r), wsc, bs, hb);
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
      // the parts: those of CTAs cl .. ch_, four at a time so that their loads
      // are in flight together
      const int base = (tile - p.full) * p.KB;
      int cl = (int)((int64_t)base * p.Gr / p.rb);  // the first CTA with K blocks of this tile
      while (cl > 0 && p.rb * cl / p.Gr > base) --cl;
      while (p.rb * (cl + 1) / p.Gr <= base) ++cl;
      int ce = (int)((int64_t)(base + p.KB) * p.Gr / p.rb);  // and the first without any more
      while (ce > cl && p.rb * ce / p.Gr >= base + p.KB) --ce;
      while (ce < p.Gr && p.rb * ce / p.Gr < base + p.KB) ++ce;
      const int32_t *p0 = p.part + ((int64_t)cl * 2 + (p.rb * cl / p.Gr > base ? 0 : 1)) * 128 * p.BN + row;
      const int32_t *pn = p.part + (int64_t)(cl + 1) * 2 * 128 * p.BN + row;  // (the others start inside the tile)
      const int64_t ps = (int64_t)2 * 128 * p.BN;
      const int np = ce - cl;
      for (int c0 = 0; c0 < nc; c0 += 16) {
        int acc[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[j] = c0 + j < nc ? __ldcg(p0 + (c0 + j) * 128) : 0;
        for (int c = 1; c < np; c += 4) {
          int v[4][16];
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < 16; ++j)
              v[u][j] = c + u < np && c0 + j < nc ? __ldcg(pn + (c - 1 + u) * ps + (c0 + j) * 128) : 0;
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[j] += v[u][j];
        }
        if (cok) i8_store16(p, ts + c0, t0 + c0, nc - c0, ch, acc, wsc, bs, hb);
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
  const int sms = std::min(device_sm_count(), I8_MAXCTA);
  // The cheapest of tokens a tile and of the ways to deal, by the cycles of the
  // busiest SM.  A K block costs the longest of: its MMAs (2 BN cycles, 81 an MMA
  // at least), its bytes from L2 (37 a cycle and SM, measured with every SM
  // loading), its weights' share of memory (23.7 a cycle and SM, once for all token tiles).
  // A tile's results cost 20 cycles a token and 1000; a cut tile's parts go to
  // L2 and back (40 bytes a cycle, 12000 cycles of fences, tickets and latency), and
  // CTAs that begin their rounds at different times share less in L2 (5 %).
  // Both sides measured: 320 tokens x 32000 x 8192 103 us cut, 112 in rounds; 4096 x 28672
  // x 8192 726 and 691; 128 x 4096 x 4096 30 and 24; 5 x 4096 x 28672 48 cut, 71 even; 16 x
  // 4096 x 4096 24 and 19; 1 x 32000 x 4096 46 cut, 40 even.
  auto block = [&](int bn, int tm, int rows) {
    return std::max({324.0, 2.0 * bn, (rows + bn) * 128.0 / 37, rows * 128.0 / 23.7 / tm});
  };
  double best = 0;
  auto take = [&](double c) {
    if (best != 0 && c >= best) return false;
    best = c;
    return true;
  };
  for (int bn = 16; bn <= 256; bn += bn < 32 ? 16 : 32) {
    const int tm = (m + bn - 1) / bn;
    const int64_t T = (int64_t)p.TN * tm;
    if (T > 0x3fffffff) continue;
    const double out = 20.0 * std::min(bn, m) + 1000, tile = p.KB * block(bn, tm, 128) + out;
    const int64_t full = T / sms * sms, rb = (T - full) * p.KB;
    const int gr = (int)std::min<int64_t>(sms, std::max<int64_t>(1, rb / I8_MINBLK));
    auto set = [&](int64_t nfull, int64_t nrb, int ngr, int units) {
      p.BN = bn;
      p.TM = tm;
      p.T = (int)T;
      p.full = (int)nfull;
      p.rb = nrb;
      p.Gr = ngr;
      p.units = units;
      p.G = (int)std::min<int64_t>(sms, units ? units : nfull ? T : ngr);
    };
    if (take((double)((T + sms - 1) / sms) * tile)) set(T, 0, 1, 0);
    if (rb) {
      const double parts = 2 + (double)gr / (T - full);
      if (take((double)(T / sms) * tile * (tm > 1 ? 1.05 : 1) + (double)rb / gr * block(bn, tm, 128) + out + 12000 +
               parts * std::min(bn, m) * 512 / 40))
        set(full, rb, gr, 0);
    }
    if (tm == 1) {
      const int units = (n + 31) / 32, per = (units + sms - 1) / sms, tail = per % 4;
      if (take((per / 4) * tile + (tail ? p.KB * block(bn, 1, 32 * tail) + out : 0))) set(0, 0, 1, units);
    }
  }
  p.idesc = idesc_i8(p.BN);
  p.tcols = 32;
  while (p.tcols < 2u * p.BN) p.tcols *= 2;
  static_assert(I8_MAXCTA * 4 == LBX_INT8_TICKET_BYTES, "tickets");
  w.part = LBX_INT8_TICKET_BYTES;
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
  const int es = xdt == LBX_F32 ? 4 : 2, e = 16 / es;
  const bool vec = aligned16(x) && x_ld * es % 16 == 0 && reinterpret_cast<uintptr_t>(q) % e == 0 && q_ld % e == 0;
  auto go = [&](auto kern) { return launch(kern, dim3(m), dim3(Q8_THREADS), 0, stream, pdl, x, x_ld, k, q, q_ld, scale); };
  const cudaError_t r = xdt == LBX_F32 ? (vec ? go(quant_tokens_kernel<LBX_F32, true>) : go(quant_tokens_kernel<LBX_F32, false>))
                                       : (vec ? go(quant_tokens_kernel<LBX_BF16, true>) : go(quant_tokens_kernel<LBX_BF16, false>));
  return cuda_status(r, "quant_tokens launch");
}

}  // namespace lbx

extern "C" int lbx_quant_tokens(const void *x, int32_t x_dtype, int64_t x_ld, int32_t m, int32_t k, int8_t *q,
                                int64_t q_ld, float *scale, cudaStream_t stream) {
  using namespace lbx;
  LBX_CHECK_ARG(m >= 0 && k >= 1, "bad shape");
  LBX_CHECK_ARG(x_dtype == LBX_F32 || x_dtype == LBX_BF16, "bad dtype");
  LBX_CHECK_SUP(k <= Q8_MAXDIM, "k must be <= %d", Q8_MAXDIM);
  LBX_CHECK_ARG(x_ld >= k && q_ld >= k, "row strides must be at least k");
  if (m == 0) return LBX_OK;
  LBX_CHECK_ARG(x && q && scale, "NULL pointer");
  return quant_tokens_launch(x, x_dtype, x_ld, m, k, q, q_ld, scale, false, stream);
}

extern "C" size_t lbx_linear_int8_workspace_size(int32_t m, int32_t n, int32_t k) {
  if (m < 1 || n < 1 || k < 1 || m > lbx::Q8_MAXDIM || n > lbx::Q8_MAXDIM || k > lbx::Q8_MAXK) return 0;
  const lbx::I8Plan w = lbx::i8_plan(m, n, k);
  return w.p.BN > 0 ? w.total : 0;
}

extern "C" int lbx_linear_int8(const lbx_int8_args *a, void *ws, size_t ws_bytes, cudaStream_t stream) {
  using namespace lbx;
  LBX_CHECK_ARG(a, "args is NULL");
  LBX_CHECK_ARG(a->m >= 0 && a->n >= 1 && a->k >= 1, "bad shape");
  LBX_CHECK_SUP(a->k <= Q8_MAXK, "k must be <= %d", Q8_MAXK);
  LBX_CHECK_SUP(a->m <= Q8_MAXDIM && a->n <= Q8_MAXDIM, "m and n must be <= %d", Q8_MAXDIM);
  LBX_CHECK_ARG((a->x_dtype == LBX_F32 || a->x_dtype == LBX_BF16) && (a->y_dtype == LBX_F32 || a->y_dtype == LBX_BF16),
                "bad dtype");
  if (a->m == 0) return LBX_OK;
  LBX_CHECK_ARG(a->x && a->w && a->w_scale && a->y, "NULL pointer");
  LBX_CHECK_ARG(a->x_ld >= a->k && a->w_ld >= a->k && a->y_ld >= a->n, "row strides smaller than the rows");
  LBX_CHECK_ARG(aligned16(a->w) && a->w_ld % 16 == 0, "weight rows must start on 16 bytes");
  I8Plan W = i8_plan(a->m, a->n, a->k);
  LBX_CHECK_SUP(W.p.BN > 0, "too many tiles");
  LBX_CHECK_ARG(ws && ws_bytes >= W.total, "workspace too small (%zu < %zu)", ws_bytes, W.total);
  LBX_CHECK_ARG(aligned16(ws), "the workspace must be 16-byte aligned");
  uint8_t *b = reinterpret_cast<uint8_t *>(ws);
  int8_t *q = reinterpret_cast<int8_t *>(b + W.q);
  float *s = reinterpret_cast<float *>(b + W.s);
  I8Params &p = W.p;
  static DevCache<size_t> smax_cache;
  size_t smax = 0;
  int rc = smax_cache.get(smax, [](size_t &out) {
    size_t o2 = 0;
    cudaError_t e = allow_max_smem(linear_int8_kernel<true>, &out);
    if (e == cudaSuccess) e = allow_max_smem(linear_int8_kernel<false>, &o2);
    out = std::min(out, o2);
    return cuda_status(e, "linear_int8 smem attribute");
  });
  if (rc) return rc;
  const int blk = (128 + p.BN) * I8_KB;
  // The even deal is a stream from memory: up to 4 K blocks a stage, so that 512
  // consecutive bytes of a row are asked for together (262 MB for 8 tokens, behind a flush
  // whose lines L2 has yet to write back: 72.7 us with one block a stage, 66.6 with two,
  // 64.5 with four), with three stages at least.
  const int st_max = (int)((smax - 1024) / blk);
  p.KS = !p.units ? 1 : st_max >= 12 ? 4 : st_max >= 6 ? 2 : 1;
  p.ST = std::min(I8_MAXST, st_max / p.KS);
  const int stage = p.KS * blk;
  p.s = s;
  p.ws = a->w_scale;
  p.bias = a->bias;
  p.y = a->y;
  p.y_ld = a->y_ld;
  p.ydt = a->y_dtype;
  p.part = reinterpret_cast<int32_t *>(b + W.part);
  p.ticket = reinterpret_cast<unsigned *>(b);
  CUtensorMap tw, tw32 = {}, tx;  // (only the even deal copies 32 rows at a time)
  rc = i8_map(&tw, a->w, a->n, a->k, a->w_ld, 128);
  if (rc) return rc;
  if (p.units) rc = i8_map(&tw32, a->w, a->n, a->k, a->w_ld, 32);
  if (rc) return rc;
  rc = i8_map(&tx, q, a->m, a->k, W.q_ld, p.BN);
  if (rc) return rc;
  rc = quant_tokens_launch(a->x, a->x_dtype, a->x_ld, a->m, a->k, q, W.q_ld, s, a->use_pdl != 0, stream);
  if (rc) return rc;
  auto go = [&](auto kern) {
    return launch(kern, dim3(p.G), dim3(I8_THREADS), (size_t)p.ST * stage + 1024, stream, true, tw, tw32, tx, p);
  };
  return cuda_status(p.KS == 1 ? go(linear_int8_kernel<true>) : go(linear_int8_kernel<false>), "linear_int8 launch");
}
