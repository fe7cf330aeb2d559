// KV cache held in 4 bits: append, read-back, attention.
//
// Each head and slot holds head_dim codes and, for each group of 64
// dimensions, (step, least) in bf16; a value is least + step * code.
// See include/lbx.h for the layout.
#include <cuda_fp16.h>
#include <type_traits>

#include "tcgen05.cuh"

namespace lbx {

constexpr int KV4_G = 64;       // dimensions a group
constexpr uint16_t KV4_NAN = 0x7FC0u;
constexpr int KV4_MAXSEQ = 1 << 30;  // slots of a sequence: those past the end stay 32-bit numbers

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
  int n, max_start, rows;  // tokens of a sequence, their starts' bound, tokens in all
  int vec;                 // inputs on 16 (fp32) or 8 (bf16) bytes
  const int32_t *start;
  const void *k; const void *v; int64_t ld;
  const float2 *rope;
};

// A row (one token's key or value of one head) is D / 4 lanes of four dimensions:
// both members of a rotation pair are D / 8 lanes apart, a group of 64 is 16
// lanes, two lanes make a word of codes.  Bound by one round trip to memory (6.2 us for 64
// rows) and, for a prompt, by instructions: 2048 tokens x 8 heads, 37 MB, 16.4 us.  (Several
// rows a warp, their loads in flight together, 18.5 us, and 9.1 for the 64 rows.)
template <int D, int DT>
__global__ void __launch_bounds__(256) kv4_append_kernel(const __grid_constant__ Kv4AppendParams p) {
  constexpr int LPR = D / 4, NG = D / KV4_G, RPW = 32 / LPR;  // lanes a row, rows a warp
  const int lane = threadIdx.x & 31, l = lane % LPR, g = l / 16;
  const uint32_t heads = (uint32_t)p.c.kvh, per = (uint32_t)p.rows * heads;  // (token, head) rows
  const bool value = blockIdx.y == 1;
  const uint32_t it = (blockIdx.x * 8 + (threadIdx.x >> 5)) * RPW + lane / LPR;
  const bool ok = it < per;
  const uint32_t row = ok ? it / heads : 0, h = ok ? it - row * heads : 0;
  const int s = (int)(row / (uint32_t)p.n), i = (int)(row - (uint32_t)s * (uint32_t)p.n);
  pdl_trigger();
  pdl_wait();
  const int st = p.start ? __ldg(p.start + s) : p.max_start;
  float x[4];
  const void *src = value ? p.v : p.k;
  const int64_t off = (int64_t)row * p.ld + (int64_t)h * D + 4 * l;
  if (p.vec) {
    if constexpr (DT == LBX_F32) {
      const float4 v = __ldg(reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(src) + off));
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
      const uint2 v = __ldg(reinterpret_cast<const uint2 *>(reinterpret_cast<const uint16_t *>(src) + off));
      x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xFFFF0000u);
      x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = load_act(src, DT, off + e);
  }
  if (!value && p.rope) {
    const float4 *t = reinterpret_cast<const float4 *>(p.rope + (int64_t)row * (D / 2) + 4 * (l % (LPR / 2)));
    const float4 c0 = __ldg(t), c1 = __ldg(t + 1);
    const float c[4] = {c0.x, c0.z, c1.x, c1.z}, sn[4] = {c0.y, c0.w, c1.y, c1.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = __shfl_xor_sync(0xffffffffu, x[e], LPR / 2);
      x[e] = l < LPR / 2 ? __fsub_rn(__fmul_rn(x[e], c[e]), __fmul_rn(y, sn[e]))
                         : __fadd_rn(__fmul_rn(x[e], c[e]), __fmul_rn(y, sn[e]));
    }
  }
  float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
  float hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  bool fin = fabsf(x[0]) < INFINITY && fabsf(x[1]) < INFINITY && fabsf(x[2]) < INFINITY && fabsf(x[3]) < INFINITY;
  fin = (__ballot_sync(0xffffffffu, !fin) & (0xFFFFu << (lane & 16))) == 0u;
#pragma unroll
  for (int o = 1; o < 16; o *= 2) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
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
  uint32_t w = 0;
  if (step > 0.f) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w |= (uint32_t)__float2int_rn(fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[e], least), inv)), 0.f), 15.f)) << (4 * e);
  }
  w |= __shfl_xor_sync(0xffffffffu, w, 1) << 16;  // (the even lane's: its codes below, its neighbour's above)
  if (!ok) return;
  if (st < 0 || st > p.max_start) {
    if (l == 0) atomicCAS(&g_lbx_device_error, 0, 0x801);
    return;
  }
  const int64_t slot = ((int64_t)s * p.c.kvh + h) * p.c.max_seq + st + i;
  const int b = l / 2;
  if (!(l & 1))
    reinterpret_cast<uint32_t *>((value ? p.c.vc : p.c.kc) + slot * (D / 2))[value ? kv4_word<D, true>(b) : kv4_word<D, false>(b)] = w;
  if (l % 16 == 0) (value ? p.c.vp : p.c.kp)[slot * NG + g] = (uint32_t)sb | (uint32_t)lb << 16;
}

struct Kv4ReadParams {
  Kv4View c;
  int n, max_start;
  const int32_t *start;
  float *out[2];
};

// one thread a block of eight dimensions: (slot, block) along x, head, (sequence, keys or values)
template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4ReadParams p) {
  constexpr uint32_t NB = D / 8;
  const bool value = blockIdx.z & 1;
  pdl_wait();
  float *out = p.out[value];
  const uint32_t e = blockIdx.x * 256 + threadIdx.x, i = e / NB, b = e % NB;
  if (!out || i >= (uint32_t)p.n) return;
  const int s = blockIdx.z >> 1;
  const int64_t sh = (int64_t)s * p.c.kvh + blockIdx.y;
  const int st = p.start ? __ldg(p.start + s) : p.max_start;
  float v[8];
  if (st >= 0 && st <= p.max_start) {
    const int64_t slot = sh * p.c.max_seq + st + i;
    const uint32_t *words = reinterpret_cast<const uint32_t *>((value ? p.c.vc : p.c.kc) + slot * (D / 2));
    const uint32_t w = words[value ? kv4_word<D, true>(b) : kv4_word<D, false>(b)];
    const uint32_t par = (value ? p.c.vp : p.c.kp)[slot * (D / KV4_G) + (b >> 3)];
#pragma unroll
    for (int t = 0; t < 8; ++t)
      v[t] = __fadd_rn(kv4_least(par), __fmul_rn(kv4_step(par), (float)((w >> (4 * t)) & 15u)));
  } else {
    atomicCAS(&g_lbx_device_error, 0, 0x802);
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] = __uint_as_float(0x7FC00000u);
  }
  float4 *o = reinterpret_cast<float4 *>(out + (sh * p.n + i) * D + 8 * b);
  o[0] = make_float4(v[0], v[1], v[2], v[3]);
  o[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// ---------------------------------------------------------------------------
// Attention: o_i = sum_j p_ij v_j / sum_j p_ij, p_ij = 2^(s_ij - m_i),
// s_ij = q_i . k_j (q scaled by scale * log2 e), one pass with the running maximum.
//
// Both products run on the tensor cores (mma.m16n8k16, fp16 in, fp32 sums)
// straight from the packed codes.  With step and least value of a group of
// dimensions outside the sum,
//
//   q . k = sum_g [ step_g (sum_{d in g} q_d (c_d - 8)) + (least_g + 8 step_g) (sum_{d in g} q_d) ]
//   o_d   = sum_j (p_j step_jg) (c_jd - 8) + sum_j p_j (least_jg + 8 step_jg)
//
// only the queries and p * step are rounded to fp16; they are brought up by a power of
// two first (a query by its row's largest, p * step by the largest step the row has seen).
// The tensor cores round their sums towards zero, and over thousands of slots
// that showed (4e-5 of the result at 4000 slots, 6e-4 at 130 000), so a sum on them
// never runs longer than 64 dimensions or 32 slots, small terms first, and the rest is
// ordinary additions.  float32 calls centre their codes (a pair of codes is two logic
// operations at most and one exact subtraction): 3e-7 and 1.2e-6.  bfloat16 calls keep c: in
// the low bits of a 16-bit lane it IS the fp16 subnormal c * 2^-24, which the tensor cores
// multiply exactly.  Nibbles 1 and 3 are left at 16 times their value.  Their sums are centred
// all the same: they begin at 8 times what rounding took from the queries' sum, and at -8
// times the sum of the rounded weights, so that what a rounding leaves is multiplied by
// c - 8 and not by c (left out, errors of a head over 2046 slots were 3.1e-3 where the result's
// own rounding makes 1.7e-3).
// Codes are the A operand (16 slots x 16 dimensions of the keys, 16 dimensions x 16
// slots of the values) and query rows the columns of B, eight to a column tile, so that
// a decode step's few rows waste half a tile at most and the running sums take 4
// registers for 16 dimensions.  The weights reach B's layout by one 8 x 8 transposition
// (movmatrix) a tile.  (Rows as A measured 500 instructions per 16 slots, half of them moves
// and masks, and 1.28 times this form's time when it was taken; two column tiles a warp share the
// unpacked codes but halve the warps: 1.2 times, for five tiles.)
//
// What bounds it is issue: 340 (bf16) to 450 (float32) instructions per 16 slots and warp at
// half an instruction a cycle, where 6.5 TB/s would be 400 cycles per 16 slots of
// 128-wide keys and values: 64 sequences of up to 8100 slots, 64 heads over 8, one token each
// 126 to 133 us in bf16 and 172 in float32, five tokens 613 and 825.  Neither more warps
// (queries' fragments in shared memory, 16 a multiprocessor: 1.2 times) nor longer steps
// (64 slots, 255 registers: equal) changed that.
//
// float32 calls (SPLIT) take each query and weight in two fp16 terms, 22 bits;
// bfloat16 ones in one, 11 bits against the result's 8.
//
// Work: a warp takes a run of sub-chunks of ck slots for one tile of query rows, 32
// slots a step, and leaves each sub-chunk's (m, l, o) to be merged in order; the
// row tiles of a block share the ring of bulk copies.  Sub-chunks and steps lie at
// fixed slots and a row's arithmetic involves no other row, so its bits do not
// depend on what else the call holds.
// ---------------------------------------------------------------------------
constexpr int KA_STEP = 32;     // slots a step of the softmax
constexpr int KA_SLOTS = 64;    // slots a stage of the ring
constexpr int KA_ST = 2;        // stages
constexpr float KA_LAZY = 8.f;  // a row's reference moves when its maximum is 2^8 above it: o is rescaled once or twice a sub-chunk
constexpr int KA_WARPS = 4;     // warps a block at most

struct Kv4AttnParams {
  Kv4View c;
  int n, heads, rep, max_prefix, dtype;
  int i0, R;           // first token of this launch's rows, query rows of a kv head
  int ck, nsub;        // slots a sub-chunk, sub-chunks of the longest sequence
  int kw, rw, ntile;   // warps' runs and row tiles a block, row tiles in all
  int cpw;             // sub-chunks a warp's run
  int qvec;            // queries on 16 bytes
  float scale;         // times log2 e
  const int32_t *prefix;
  const void *q; int64_t q_ld;
  const float2 *rope;
  const uint64_t *tree;
  void *out;
  float *part_o;       // [n_seq][kvh][nsub][R][D]
  float2 *part_ml;     // [n_seq][kvh][nsub][R]
};

// d[16 x 8] (+)= a[16 x 16] b[16 x 8]
LBX_DEV void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// (from sums of its own, not d's)
LBX_DEV void mma_f16_from(float (&d)[4], const float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
LBX_DEV void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
LBX_DEV uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
LBX_DEV uint32_t f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// what the fp16 rounding of (lo, hi) in r left over; as fp16; its sum
LBX_DEV float2 f16x2_left(uint32_t r, float lo, float hi) {
  const __half2 h = *reinterpret_cast<const __half2 *>(&r);
  return make_float2(lo - __low2float(h), hi - __high2float(h));
}
LBX_DEV uint32_t f16x2_rest(uint32_t r, float lo, float hi) {
  const float2 v = f16x2_left(r, lo, hi);
  return f16x2(v.x, v.y);
}
LBX_DEV float f16x2_lost(uint32_t r, float lo, float hi) {
  const float2 v = f16x2_left(r, lo, hi);
  return v.x + v.y;
}
// exponent of |x| <- its bits, within what the power-of-two factors reach: steps up to 2^100
// (past it the sums of the weighted values overflow anyway), queries up to top
LBX_DEV int kv4_exp(uint32_t bits, int top = 100) { return min(max((int)(bits >> 23) - 127, -112), top); }
LBX_DEV float kv4_pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// The masks of the unpacking, in registers: with both a mask and bits to set,
// immediates would make two instructions of each.
struct Kv4Masks {
  uint32_t m0, m1, one;
  LBX_DEV Kv4Masks() {
    asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(m0));
    asm volatile("mov.b32 %0, 0x00F000F0;" : "=r"(m1));
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(one));
  }
};
// codes in bits 4 N .. 4 N + 3 of both halves -> 16^N (code - 8) as fp16: 1024 + 16^N code by
// its bits, less 1024 + 8 * 16^N, both exact
template <int N>
LBX_DEV uint32_t kv4_mid(const Kv4Masks &k, uint32_t x) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(x), "r"(N ? k.m1 : k.m0), "r"(k.one));  // (x & mask) | one
  const uint32_t off = N ? 0x64806480u : 0x64086408u;
  const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&v), *reinterpret_cast<const __half2 *>(&off));
  return *reinterpret_cast<const uint32_t *>(&d);
}
// a pair of the keys' codes: centred, or as the subnormals 2^-24 code
template <bool MID, int N>
LBX_DEV uint32_t kv4_kcode(const Kv4Masks &k, uint32_t x) {
  if constexpr (MID) return kv4_mid<N>(k, x);
  return x & (N ? 0x00F000F0u : 0x000F000Fu);
}
LBX_DEV float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
LBX_DEV float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// over the eight lanes of one j
LBX_DEV float col_max(float v) {
#pragma unroll
  for (int o = 4; o < 32; o *= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
LBX_DEV float col_sum(float v) {
#pragma unroll
  for (int o = 4; o < 32; o *= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
LBX_DEV float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Is a group's step or least value an infinity or a NaN?  Either may be alone; least + 8 step
// is then one too.
LBX_DEV bool kv4_no_number(float least8) { return !(fabsf(least8) < INFINITY); }

// does query i of its sequence see slot j
LBX_DEV bool kv4_sees(int j, int prefix, int n, int i, bool tree, uint64_t mask) {
  if (j < prefix) return true;
  const int t = j - prefix;
  return t < n && (tree ? (t < 64 && ((mask >> t) & 1ull)) : t <= i);
}

// slot, among the eight of an MMA's column tile, of column rho: neighbours keep
// opposite parity (two rows of keys per shared-memory wavefront), and so do
// columns 0, 2, 4, 6 in turn (the value rows a warp reads together)
LBX_DEV int kv4_key(int rho) { return rho ^ ((rho >> 1) & 1); }

template <int NG>
LBX_DEV void kv4_params(const uint32_t *a, uint32_t (&pp)[NG]) {
  if constexpr (NG == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(a);
    pp[0] = v.x;
    pp[1] = v.y;
  } else {
    pp[0] = *a;
  }
}

template <int D>
struct Kv4Stage {
  static constexpr int CB = KA_SLOTS * D / 2, PB = KA_SLOTS * (D / KV4_G) * 4;  // bytes of codes, of params
  static constexpr int BYTES = 2 * (CB + PB);
};

// One query row's fragment values: the 8-dimension blocks of lane j (block
// b(t) = (t >> 1) * 8 + (t & 1) * 4 + j for head_dim 128, t * 4 + j for 64),
// rotated and scaled; both members of every rotation pair are the lane's own.
template <int D>
LBX_DEV void kv4_load_q(const Kv4AttnParams &p, int64_t row, int hq, int j, bool ok, float (&x)[D / 4]) {
  constexpr int NW = D / 32;  // blocks a lane
#pragma unroll
  for (int t = 0; t < NW; ++t) {
    const int b = D == 128 ? (t >> 1) * 8 + (t & 1) * 4 + j : t * 4 + j;
    const int64_t o = row * p.q_ld + (int64_t)hq * D + 8 * b;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[8 * t + i] = 0.f;
    if (!ok) continue;
    if (!p.qvec) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[8 * t + i] = load_act(p.q, p.dtype, o + i);
    } else if (p.dtype == LBX_F32) {
      const float4 *v = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p.q) + o);
      const float4 a = __ldg(v), c = __ldg(v + 1);
      x[8 * t] = a.x; x[8 * t + 1] = a.y; x[8 * t + 2] = a.z; x[8 * t + 3] = a.w;
      x[8 * t + 4] = c.x; x[8 * t + 5] = c.y; x[8 * t + 6] = c.z; x[8 * t + 7] = c.w;
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(p.q) + o));
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[8 * t + 2 * i] = __uint_as_float(w[i] << 16);
        x[8 * t + 2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
  }
  if (p.rope && ok) {
#pragma unroll
    for (int t = 0; t < NW / 2; ++t) {
      const int b = t * 4 + j;  // (first half of the dimensions)
      const float4 *cs = reinterpret_cast<const float4 *>(p.rope + row * (D / 2) + 8 * b);
      float4 cv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) cv[i] = __ldg(cs + i);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 c = (i & 1) ? make_float2(cv[i / 2].z, cv[i / 2].w) : make_float2(cv[i / 2].x, cv[i / 2].y);
        const float x1 = x[8 * t + i], x2 = x[8 * (t + NW / 2) + i];
        x[8 * t + i] = x1 * c.x - x2 * c.y;
        x[8 * (t + NW / 2) + i] = x2 * c.x + x1 * c.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < D / 4; ++i) x[i] *= p.scale;
}

template <int D, bool SPLIT>
__global__ void __launch_bounds__(KA_WARPS * 32, 3) kv4_attn_kernel(const __grid_constant__ Kv4AttnParams p) {
  constexpr int NG = D / KV4_G, NW = D / 32, NS = SPLIT ? 2 : 1;
  constexpr int RT = 8;              // query rows a tile
  constexpr int NK = KA_STEP / 8;    // slots of a step that a lane holds the weights of
  using Stage = Kv4Stage<D>;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[KA_WARPS][KA_ST], empty[KA_WARPS][KA_ST];
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, j = lane & 3;
  const int kg = warp / p.rw, rt = warp - kg * p.rw;  // this warp's sub-chunk and row tile in the block
  const int rgroups = (p.ntile + p.rw - 1) / p.rw;
  const int cblk = blockIdx.x / rgroups, rg = blockIdx.x - cblk * rgroups;
  const int c0 = (cblk * p.kw + kg) * p.cpw, h = blockIdx.y, s = blockIdx.z;  // (first sub-chunk)
  volatile int *abrt = &abort_flag;
  if (tid == 0) {
    for (int g = 0; g < p.kw; ++g)
      for (int i = 0; i < KA_ST; ++i) {
        mbar_init(&full[g][i], 1);
        mbar_init(&empty[g][i], p.rw);
      }
    fence_mbar_init();
    abort_flag = 0;
  }
  __syncthreads();
  pdl_trigger();
  pdl_wait();
  const int prefix = p.prefix ? __ldg(p.prefix + s) : p.max_prefix;
  if (prefix < 0 || prefix > p.max_prefix) {
    if (tid == 0) atomicCAS(&g_lbx_device_error, 0, 0x803);
    if (p.nsub > 1 || kg > 0) return;  // (the merge tells the rows)
    for (int R = (rg * p.rw + rt) * RT; R < min(p.R, (rg * p.rw + rt + 1) * RT); ++R) {
      const int i = p.i0 + R / p.rep;
      const int64_t d0 = (((int64_t)s * p.n + i) * p.heads + h * p.rep + R % p.rep) * D;
      for (int d = lane; d < D; d += 32) {
        if (p.dtype == LBX_F32) reinterpret_cast<float *>(p.out)[d0 + d] = __uint_as_float(0x7FC00000u);
        else reinterpret_cast<uint16_t *>(p.out)[d0 + d] = KV4_NAN;
      }
    }
    return;
  }
  // slots this block's row tiles see, and this warp's
  const int t0 = rg * p.rw, tl = min(t0 + p.rw, p.ntile) - 1;  // first and last tile of the block
  const int tile = t0 + rt;
  auto seen_end = [&](int tl_) {
    return prefix + (p.tree ? p.n : p.i0 + (min(p.R, (tl_ + 1) * RT) - 1) / p.rep + 1);
  };
  const int lo = c0 * p.ck;
  const int run = min(p.cpw, p.nsub - c0) * p.ck;
  const int hi_blk = run > 0 ? min(lo + run, seen_end(tl)) : 0;
  const int nst = hi_blk > lo ? (hi_blk - lo + KA_SLOTS - 1) / KA_SLOTS : 0;
  if (nst == 0) return;  // (every warp of this ring)
  const bool live_tile = tile < p.ntile;
  const int my_end = live_tile ? min(lo + run, seen_end(tile)) : 0;

  uint8_t *ring = smem_raw + kg * KA_ST * Stage::BYTES;
  const int64_t base = ((int64_t)s * p.c.kvh + h) * p.c.max_seq + lo;
  auto issue = [&](int i) {  // (one lane)
    const int st = i % KA_ST;
    uint8_t *d = ring + st * Stage::BYTES;
    const int64_t slot = base + (int64_t)i * KA_SLOTS;
    mbar_arrive_expect_tx(&full[kg][st], Stage::BYTES);
    bulk_g2s(d, p.c.kc + slot * (D / 2), Stage::CB, &full[kg][st]);
    bulk_g2s(d + Stage::CB, p.c.kp + slot * NG, Stage::PB, &full[kg][st]);
    bulk_g2s(d + Stage::CB + Stage::PB, p.c.vc + slot * (D / 2), Stage::CB, &full[kg][st]);
    bulk_g2s(d + 2 * Stage::CB + Stage::PB, p.c.vp + slot * NG, Stage::PB, &full[kg][st]);
  };
  int issued = 0;
  if (rt == 0 && lane == 0)
    for (; issued < KA_ST && issued < nst; ++issued) issue(issued);

  // ---- the queries' fragments: lane (r, j) makes its dimensions of row r; as
  // accumulator columns it owns rows 2 j and 2 j + 1
  uint32_t qb[NS][2 * NW][2];
  float fq[2], qs[2][NG];  // the queries' unit, and their sums in it
  float ql[NG][4];         // bfloat16 calls: 8 times what the rounding took from the sums, as accumulators
  int qi[2];               // token index of the rows
  bool rok[2];
  const bool tree = p.tree != nullptr;
  uint64_t mask[2];
  const int64_t qrow0 = (int64_t)s * p.n + p.i0;
  {
    float x[D / 4];
    const int Rr = tile * RT + r;
    const bool ok = live_tile && Rr < p.R;
    kv4_load_q<D>(p, qrow0 + (ok ? Rr / p.rep : 0), h * p.rep + (ok ? Rr % p.rep : 0), j, ok, x);
    float mq = 0.f;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) mq = fmaxf(mq, fabsf(x[i]));
    const int e = kv4_exp(__float_as_uint(quad_max(mq)), SPLIT ? 127 : 117);  // (unit stays a float)
    const float up = kv4_pow2(14 - e), unit = kv4_pow2(e - 14) * (SPLIT ? 1.f : 16777216.f);
    float sum[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      constexpr int PER = D / 4 / NG;
      float a = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) a += x[g * PER + i];
      sum[g] = quad_sum(a) * (SPLIT ? up : up * 5.9604644775390625e-8f);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {  // (from the lanes that made rows 2 j + b)
      const int src = 4 * (2 * j + b);
      fq[b] = __shfl_sync(0xffffffffu, unit, src);
#pragma unroll
      for (int g = 0; g < NG; ++g) qs[b][g] = __shfl_sync(0xffffffffu, sum[g], src);
      const int R = tile * RT + 2 * j + b;
      rok[b] = live_tile && R < p.R;
      qi[b] = p.i0 + (rok[b] ? R / p.rep : 0);
      mask[b] = tree && rok[b] ? __ldg(p.tree + (int64_t)s * p.n + qi[b]) : 0ull;
    }
    float lost[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) lost[g] = 0.f;
#pragma unroll
    for (int t = 0; t < NW; ++t) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[8 * t + i] * ((i & 1) ? up * 0.0625f : up);
#pragma unroll
      for (int k = 0; k < 2; ++k) {  // (k step 2t + k: dimensions 2k, 2k+4 and 2k+1, 2k+5 of the block)
        const uint32_t b0 = f16x2(y[2 * k], y[2 * k + 4]), b1 = f16x2(y[2 * k + 1], y[2 * k + 5]);
        qb[0][2 * t + k][0] = b0;
        qb[0][2 * t + k][1] = b1;
        if constexpr (SPLIT) {
          qb[1][2 * t + k][0] = f16x2_rest(b0, y[2 * k], y[2 * k + 4]);
          qb[1][2 * t + k][1] = f16x2_rest(b1, y[2 * k + 1], y[2 * k + 5]);
        } else {
          lost[t * NG / NW] += f16x2_lost(b0, y[2 * k], y[2 * k + 4]) + 16.f * f16x2_lost(b1, y[2 * k + 1], y[2 * k + 5]);
        }
      }
    }
    if constexpr (!SPLIT) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float a = quad_sum(lost[g]) * (8.f * 5.9604644775390625e-8f);
        ql[g][0] = ql[g][2] = __shfl_sync(0xffffffffu, a, 8 * j);
        ql[g][1] = ql[g][3] = __shfl_sync(0xffffffffu, a, 8 * j + 4);
      }
    }
  }

  const Kv4Masks km;
  float o[D / 16][4];  // row tile 4 g + q: dimensions 64 g + 8 r + 2 q (+ 1: the second half), rows 2 j, 2 j + 1
  float m[2], l[2], om[2][NG];  // reference of the weights, their sum, sum of weight * (least + 8 step)
  int eo[2];                    // exponent of the largest step seen
  float lim[2];                 // 2^(eo + 1)
  auto reset = [&]() {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      m[b] = -INFINITY;
      l[b] = 0.f;
      eo[b] = -112;
      lim[b] = kv4_pow2(-111);
#pragma unroll
      for (int g = 0; g < NG; ++g) om[b][g] = 0.f;
    }
  };
  reset();

  for (int i = 0; i < nst; ++i) {
    const int st = i % KA_ST;
    // the stage read before is free once all row tiles have read it
    if (rt == 0 && lane == 0 && i > 0 && issued < nst &&
        wd_wait(&empty[kg][(i - 1) % KA_ST], (uint32_t)((i - 1) / KA_ST) & 1u, 0x805, abrt))
      issue(issued++);
    __syncwarp();
    if (!__all_sync(0xffffffffu, wd_wait(&full[kg][st], (uint32_t)(i / KA_ST) & 1u, 0x804, abrt))) break;
#pragma unroll 1  // (two steps of code do not fit the instruction cache as well as one: 285 us a pass became 311)
    for (int hs = 0; hs < KA_SLOTS; hs += KA_STEP) {
      const int j0 = lo + i * KA_SLOTS + hs;
      if (j0 >= my_end) break;
      const uint8_t *sk = ring + st * Stage::BYTES + hs * (D / 2);
      const uint32_t *skp = reinterpret_cast<const uint32_t *>(ring + st * Stage::BYTES + Stage::CB) + hs * NG;
      const uint8_t *sv = sk + Stage::CB + Stage::PB;
      const uint32_t *svp = skp + (Stage::CB + Stage::PB) / 4;
      // ---- scores in the queries' unit: sc[2 a + k][b], slot 16 a + 8 k + kv4_key(r), row 2 j + b
      float sc[NK][2];
#pragma unroll
      for (int a = 0; a < NK / 2; ++a) {
        uint32_t w[2][NW];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint8_t *kr = sk + (16 * a + 8 * k + kv4_key(r)) * (D / 2) + j * (D / 8);
          if constexpr (D == 128) {
            const uint4 v = *reinterpret_cast<const uint4 *>(kr);
            w[k][0] = v.x; w[k][1] = v.y; w[k][2] = v.z; w[k][3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2 *>(kr);
            w[k][0] = v.x; w[k][1] = v.y;
          }
        }
        float acc[NG][4];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          constexpr int KS = 2 * NW / NG;  // k steps of a group
          uint32_t f[KS][4];
#pragma unroll
          for (int q = 0; q < KS; ++q) {
            const int wi = (g * KS + q) / 2;
            const uint32_t w0 = (q & 1) ? w[0][wi] >> 8 : w[0][wi], w1 = (q & 1) ? w[1][wi] >> 8 : w[1][wi];
            f[q][0] = kv4_kcode<SPLIT, 0>(km, w0);
            f[q][1] = kv4_kcode<SPLIT, 0>(km, w1);
            f[q][2] = kv4_kcode<SPLIT, 1>(km, w0);
            f[q][3] = kv4_kcode<SPLIT, 1>(km, w1);
          }
#pragma unroll
          for (int e = NS - 1; e >= 0; --e)  // (the small terms first)
#pragma unroll
            for (int q = 0; q < KS; ++q) {
              const uint32_t(&b)[2] = qb[e][g * KS + q];
              if (!SPLIT && q == 0) mma_f16_from(acc[g], ql[g], f[q][0], f[q][1], f[q][2], f[q][3], b[0], b[1]);
              else if (e == NS - 1 && q == 0) mma_f16_first(acc[g], f[q][0], f[q][1], f[q][2], f[q][3], b[0], b[1]);
              else mma_f16(acc[g], f[q][0], f[q][1], f[q][2], f[q][3], b[0], b[1]);
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t pp[NG];
          kv4_params<NG>(skp + (16 * a + 8 * k + kv4_key(r)) * NG, pp);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const float sg = kv4_step(pp[g]), lg = SPLIT ? fmaf(8.f, sg, kv4_least(pp[g])) : kv4_least(pp[g]);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              float &x = sc[2 * a + k][b];
              x = fmaf(acc[g][2 * k + b], sg, g == 0 ? lg * qs[b][g] : fmaf(lg, qs[b][g], x));
            }
          }
        }
      }
      // ---- the values' params of this lane's slots; what each row sees of the step
      const bool whole = j0 + KA_STEP <= prefix;
      float sg[NK][NG], lg[NK][NG];
      float sx[2] = {0.f, 0.f};
#pragma unroll
      for (int t = 0; t < NK; ++t) {
        uint32_t pp[NG];
        kv4_params<NG>(svp + (8 * t + kv4_key(r)) * NG, pp);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          sg[t][g] = kv4_step(pp[g]);
          lg[t][g] = fmaf(8.f, sg[t][g], kv4_least(pp[g]));
          sx[0] = fmaxf(sx[0], fabsf(sg[t][g]));  // (a NaN is passed over)
        }
      }
      sx[1] = sx[0];
      if (!whole) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          float a = 0.f;
#pragma unroll
          for (int t = 0; t < NK; ++t) {
            if (rok[b] && kv4_sees(j0 + 8 * t + kv4_key(r), prefix, p.n, qi[b], tree, mask[b])) {
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                a = fmaxf(a, fabsf(sg[t][g]));
                // what is not a number reaches the rows that see it, and (below) no other
                if (kv4_no_number(lg[t][g])) om[b][g] += __uint_as_float(0x7FC00000u);
              }
            } else {
              sc[t][b] = -INFINITY;
            }
          }
          sx[b] = a;
        }
#pragma unroll
        for (int t = 0; t < NK; ++t)
#pragma unroll
          for (int g = 0; g < NG; ++g)
            if (kv4_no_number(lg[t][g])) sg[t][g] = lg[t][g] = 0.f;
      }
      // ---- references: a row's moves when its maximum is 2^8 above it (or a step is above all before)
      float mx[2];
      bool change = false;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        mx[b] = sc[0][b];
#pragma unroll
        for (int t = 1; t < NK; ++t) mx[b] = fmaxf(mx[b], sc[t][b]);
        change |= mx[b] * fq[b] > m[b] + KA_LAZY || sx[b] >= lim[b];
      }
      if (__any_sync(0xffffffffu, change)) {
        float al[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const float top = col_max(mx[b]) * fq[b];
          const int e = max(kv4_exp(__float_as_uint(col_max(sx[b]))), eo[b]);
          const float mn = top > m[b] + KA_LAZY ? top : m[b];
          al[b] = mn == m[b] ? 1.f : ex2(m[b] - mn);  // (from -inf: 0)
          l[b] *= al[b];
#pragma unroll
          for (int g = 0; g < NG; ++g) om[b][g] *= al[b];
          al[b] *= kv4_pow2(max(eo[b] - e, -126));
          m[b] = mn;
          eo[b] = e;
          lim[b] = kv4_pow2(e + 1);
        }
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
          o[t][0] *= al[0];
          o[t][1] *= al[1];
          o[t][2] *= al[0];
          o[t][3] *= al[1];
        }
      }
      // ---- weights (at most 2^8; with a step below 2^(eo + 1), times f, below 2^15)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float ref = m[b] == -INFINITY ? 0.f : m[b];  // (nothing seen so far: weights 0)
        const float f = kv4_pow2(6 - eo[b]);
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < NK; ++t) {
          const float w = ex2(fmaf(sc[t][b], fq[b], -ref));
          sum += w;
#pragma unroll
          for (int g = 0; g < NG; ++g) om[b][g] = fmaf(w, lg[t][g], om[b][g]);
          sc[t][b] = w * f;
        }
        l[b] += sum;
      }
      // ---- values: 16 slots an MMA, the step's 32 in one sum, which joins the running one by ordinary additions
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint32_t pb[NK / 2][NS][2], vw[NK / 2][4];
#pragma unroll
        for (int a = 0; a < NK / 2; ++a) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float x0 = sc[2 * a + k][0] * sg[2 * a + k][g], x1 = sc[2 * a + k][1] * sg[2 * a + k][g];
            const uint32_t hi = f16x2(x0, x1);
            pb[a][0][k] = transpose8(hi);
            if constexpr (SPLIT) pb[a][1][k] = transpose8(f16x2_rest(hi, x0, x1));
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
            vw[a][k] = *reinterpret_cast<const uint32_t *>(
                sv + (16 * a + 8 * (k >> 1) + kv4_key(2 * j + (k & 1))) * (D / 2) + r * (D / 16) + 4 * g);
        }
        float c8[4];  // bfloat16 calls: -8 times the sum of the rounded weights, where their sums of codes begin
        if constexpr (!SPLIT) {
          mma_f16_first(c8, 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, pb[0][0][0], pb[0][0][1]);
#pragma unroll
          for (int a = 1; a < NK / 2; ++a)
            mma_f16(c8, 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, pb[a][0][0], pb[a][0][1]);
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {  // nibbles 0-3, 4-7 of the word
          uint32_t v[NK / 2][2];
#pragma unroll
          for (int a = 0; a < NK / 2; ++a)
#pragma unroll
            for (int k = 0; k < 2; ++k) v[a][k] = __byte_perm(vw[a][2 * k], vw[a][2 * k + 1], hf ? 0x7632 : 0x5410);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float t[4];
            uint32_t f[NK / 2][4];
#pragma unroll
            for (int a = 0; a < NK / 2; ++a) {
              f[a][0] = kv4_kcode<SPLIT, 0>(km, v[a][0]);
              f[a][1] = kv4_kcode<SPLIT, 1>(km, v[a][0]);
              f[a][2] = kv4_kcode<SPLIT, 0>(km, v[a][1]);
              f[a][3] = kv4_kcode<SPLIT, 1>(km, v[a][1]);
              v[a][0] >>= 8;
              v[a][1] >>= 8;
            }
#pragma unroll
            for (int e = NS - 1; e >= 0; --e)
#pragma unroll
              for (int a = 0; a < NK / 2; ++a) {
                if (!SPLIT && a == 0) mma_f16_from(t, c8, f[a][0], f[a][1], f[a][2], f[a][3], pb[a][e][0], pb[a][e][1]);
                else if (e == NS - 1 && a == 0) mma_f16_first(t, f[a][0], f[a][1], f[a][2], f[a][3], pb[a][e][0], pb[a][e][1]);
                else mma_f16(t, f[a][0], f[a][1], f[a][2], f[a][3], pb[a][e][0], pb[a][e][1]);
              }
#pragma unroll
            for (int i = 0; i < 4; ++i) o[4 * g + 2 * hf + q][i] += t[i];
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive1(&empty[kg][st]);
    const int j1 = lo + (i + 1) * KA_SLOTS;
    if (j1 % p.ck != 0 && i + 1 < nst) continue;
    const int c = (j1 - 1) / p.ck;
    if (c * p.ck >= my_end) continue;

    // ---- the sub-chunk's (m, l, o): lane (r, j) holds dimensions 64 g + 8 r .. + 7 of rows 2 j, 2 j + 1
    const bool single = p.nsub == 1;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float lsum = col_sum(l[b]);
      float oms[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) oms[g] = col_sum(om[b][g]);
      if (!rok[b]) continue;
      const int R = tile * RT + 2 * j + b;
      const float dn = kv4_pow2(eo[b] - 6) * (SPLIT ? 1.f : 16777216.f);
      const int64_t pr = (((int64_t)s * p.c.kvh + h) * p.nsub + c) * p.R + R;
      const int64_t od = (((int64_t)s * p.n + qi[b]) * p.heads + h * p.rep + R % p.rep) * D;
      if (!single && r == 0) p.part_ml[pr] = make_float2(m[b], lsum);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          v[q] = fmaf(o[4 * g + q / 2][2 * (q & 1) + b], (q & 1) ? dn * 0.0625f : dn, oms[g]);
          if (single) v[q] = lsum == 0.f ? 0.f : v[q] / lsum;  // (as the merge of one sub-chunk)
        }
        const int d = 64 * g + 8 * r;
        if (!single || p.dtype == LBX_F32) {
          float *dst = single ? reinterpret_cast<float *>(p.out) + od + d : p.part_o + pr * D + d;
          reinterpret_cast<float4 *>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
          reinterpret_cast<float4 *>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
          uint32_t w[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) w[q] = (uint32_t)f32_to_bf16(v[2 * q]) | (uint32_t)f32_to_bf16(v[2 * q + 1]) << 16;
          *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(p.out) + od + d) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    reset();
  }
  if (rt == 0 && lane == 0 && *abrt) {  // copies in flight land before shared memory is given up
    int none = 0;
    for (int i = max(0, issued - KA_ST); i < issued; ++i)
      wd_wait(&full[kg][i % KA_ST], (uint32_t)(i / KA_ST) & 1u, 0x806, &none);
  }
}

// Merge of the sub-chunks' (m, l, o), one block a query row: warp w adds sub-chunks
// w, w + 8, ... in order, a lane D / 32 dimensions, then the warps in order.  Bound by the
// round trips: prefix, then everything of 32 sub-chunks at once (their maxima with
// them), 16 bytes a lane.  (4096 rows of 32 sub-chunks, 67 MB: 17.0 us by itself, 36.2
// with the maxima fetched first and values four bytes at a time.)
constexpr int KM_WARPS = 8, KM_BATCH = 4;  // warps, and partial results a lane loads together
template <int D>
__global__ void __launch_bounds__(KM_WARPS * 32) kv4_merge_kernel(const __grid_constant__ Kv4AttnParams p) {
  constexpr int V = D / 32;
  __shared__ float red[KM_WARPS], wo[KM_WARPS][D], wl[KM_WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int R = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
  const int i = p.i0 + R / p.rep, hq = h * p.rep + R % p.rep;
  pdl_wait();
  const int prefix = p.prefix ? __ldg(p.prefix + s) : p.max_prefix;
  const bool bad = prefix < 0 || prefix > p.max_prefix;
  const int end = prefix + (p.tree ? p.n : i + 1), ns = bad ? 0 : (end + p.ck - 1) / p.ck;
  const int64_t base = ((int64_t)s * p.c.kvh + h) * p.nsub * p.R + R;
  using Vec = std::conditional_t<V == 4, float4, float2>;
  float2 ml[KM_BATCH];
  alignas(16) float x[KM_BATCH][V];
  auto load = [&](int c0) {
#pragma unroll
    for (int b = 0; b < KM_BATCH; ++b) {
      const int c = c0 + KM_WARPS * b;
      ml[b] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int v = 0; v < V; ++v) x[b][v] = 0.f;
      if (c < ns) {
        const int64_t pr = base + (int64_t)c * p.R;
        ml[b] = __ldcg(p.part_ml + pr);
        *reinterpret_cast<Vec *>(x[b]) = __ldcg(reinterpret_cast<const Vec *>(p.part_o + pr * D) + lane);
      }
    }
  };
  load(warp);
  float mx = -INFINITY;
#pragma unroll
  for (int b = 0; b < KM_BATCH; ++b) mx = fmaxf(mx, ml[b].x);
  for (int c = KM_WARPS * KM_BATCH + tid; c < ns; c += KM_WARPS * 32)
    mx = fmaxf(mx, __ldcg(p.part_ml + base + (int64_t)c * p.R).x);
  mx = warp_max(mx);
  if (lane == 0) red[warp] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < KM_WARPS; ++w) mx = fmaxf(mx, red[w]);
  float o[V], l = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) o[v] = 0.f;
  for (int c0 = warp; c0 < ns;) {
#pragma unroll
    for (int b = 0; b < KM_BATCH; ++b) {
      // (no sub-chunk, or nothing of it seen: nothing to add; a sum that is not a number stays one)
      const float w = ml[b].x == -INFINITY ? 0.f : exp2f(ml[b].x - mx);
      l = fmaf(w, ml[b].y, l);
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = fmaf(w, x[b][v], o[v]);
    }
    c0 += KM_WARPS * KM_BATCH;
    if (c0 < ns) load(c0);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) wo[warp][lane * V + v] = o[v];
  if (lane == 0) wl[warp] = l;
  __syncthreads();
  if (tid < D) {
    float lt = 0.f, ot = 0.f;
#pragma unroll
    for (int w = 0; w < KM_WARPS; ++w) {
      lt += wl[w];
      ot += wo[w][tid];
    }
    const float y = bad ? __uint_as_float(0x7FC00000u) : lt == 0.f ? 0.f : ot / lt;
    const int64_t d = (((int64_t)s * p.n + i) * p.heads + hq) * D + tid;
    if (p.dtype == LBX_F32) reinterpret_cast<float *>(p.out)[d] = y;
    else reinterpret_cast<uint16_t *>(p.out)[d] = f32_to_bf16(y);
  }
}

// slots a sub-chunk: by the cache's size alone (a row's bits then do not depend
// on the lengths a call is given)
static int kv4_sub_chunk(int max_seq) {
  int ck = 128;
  while (ck < 1024 && ck * 32 < max_seq) ck *= 2;
  return ck;
}

// the cache's checks, shared by the three calls
static int kv4_view(const lbx_kv4_cache &c, Kv4View &v) {
  LBX_CHECK_ARG(c.n_seq >= 1 && c.kv_heads >= 1 && c.max_seq >= 1, "bad cache shape");
  LBX_CHECK_SUP(c.head_dim == 64 || c.head_dim == 128, "head_dim must be 64 or 128");
  LBX_CHECK_ARG(c.max_seq % 64 == 0, "max_seq must be a multiple of 64");
  LBX_CHECK_SUP(c.max_seq <= KV4_MAXSEQ, "max_seq must be <= %d", KV4_MAXSEQ);
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
  p.scale = a->scale * 1.4426950408889634f;
  p.prefix = a->prefix;
  p.q = a->q;
  p.q_ld = a->q_ld;
  p.rope = reinterpret_cast<const float2 *>(a->rope_cs);
  LBX_CHECK_ARG(aligned16(a->rope_cs), "rope_cs must be 16-byte aligned");
  p.qvec = aligned16(a->q) && a->q_ld % (a->dtype == LBX_F32 ? 4 : 8) == 0;
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
  p.start = a->start;
  p.k = a->k_new;
  p.v = a->v_new;
  p.ld = a->kv_ld;
  p.rope = reinterpret_cast<const float2 *>(a->rope_cs);
  LBX_CHECK_ARG(aligned16(a->rope_cs), "rope_cs must be 16-byte aligned");
  const int64_t rows = (int64_t)a->cache.n_seq * a->n, items = rows * a->cache.kv_heads;
  LBX_CHECK_SUP(items <= 0x3fffffff, "too many rows");
  p.rows = (int)rows;
  const int es = a->dtype == LBX_F32 ? 4 : 2;
  p.vec = ((reinterpret_cast<uintptr_t>(a->k_new) | reinterpret_cast<uintptr_t>(a->v_new)) & (uintptr_t)(4 * es - 1)) == 0 &&
          a->kv_ld % 4 == 0;
  const int d = a->cache.head_dim, blk = 8 * (128 / d);  // (rows a block)
  const dim3 grid((unsigned)((items + blk - 1) / blk), 2);
  auto go = [&](auto kern) { return launch(kern, grid, dim3(256), 0, stream, a->use_pdl != 0, p); };
  auto pick = [&](auto dd, auto dt) {
    constexpr int D = decltype(dd)::value, DT = decltype(dt)::value;
    return go(kv4_append_kernel<D, DT>);
  };
  using F = std::integral_constant<int, LBX_F32>;
  using B = std::integral_constant<int, LBX_BF16>;
  const cudaError_t e = d == 128 ? (es == 4 ? pick(std::integral_constant<int, 128>{}, F{}) : pick(std::integral_constant<int, 128>{}, B{}))
                                 : (es == 4 ? pick(std::integral_constant<int, 64>{}, F{}) : pick(std::integral_constant<int, 64>{}, B{}));
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
  const int64_t items = (int64_t)n * (c->head_dim / 8);
  LBX_CHECK_SUP(items <= 0x7fffffff && c->kv_heads <= 65535 && c->n_seq <= 32767, "too many rows");
  const dim3 grid((unsigned)((items + 255) / 256), c->kv_heads, 2 * c->n_seq);
  // (the kernel waits for the one before it, so it may be launched while that runs)
  return cuda_status(c->head_dim == 128 ? launch(kv4_read_kernel<128>, grid, dim3(256), 0, stream, true, p)
                                        : launch(kv4_read_kernel<64>, grid, dim3(256), 0, stream, true, p),
                     "kv4_read launch");
}

namespace lbx {
// how a launch of nt tokens is cut
static void kv4_cut(Kv4AttnParams &p, int i0, int nt) {
  const int end = p.max_prefix + (p.tree ? p.n : i0 + nt);
  p.ck = kv4_sub_chunk(p.c.max_seq);
  p.i0 = i0;
  p.R = nt * p.rep;
  p.ntile = (p.R + 7) / 8;
  p.nsub = (end + p.ck - 1) / p.ck;
  // sub-chunks a warp takes on end: a few rounds of warps are enough, and the
  // queries' fragments are made once for all of them (bf16, 5 tokens of 64
  // sequences over up to 4000 slots, 64 heads over 8: 370 us, one sub-chunk each 417)
  const int64_t units = (int64_t)p.c.n_seq * p.c.kvh * p.ntile * p.nsub;
  p.cpw = (int)std::min<int64_t>(8, std::max<int64_t>(1, units / (48 * device_sm_count())));
  // Row tiles a block, evenly (the same 5 tiles: 370 us sharing the
  // ring, 398 each with its own); with one sub-chunk a warp a tile has its own ring (5 tiles
  // over 130 000 slots: 245 us, shared 280).  The warps left take further runs.
  const int groups = (p.ntile + KA_WARPS - 1) / KA_WARPS;
  p.rw = p.cpw == 1 ? 1 : (p.ntile + groups - 1) / groups;
  p.kw = std::min(KA_WARPS / p.rw, (p.nsub + p.cpw - 1) / p.cpw);
}

// Tokens a launch (its partial results stay within a gigabyte), and what the call wants
// of scratch: never less for a longer prefix or for more tokens, so that scratch sized for
// the longest serves every call (whole tokens times their bytes would not: a shorter
// prefix may fit one token more into the gigabyte).
static int kv4_slice(const Kv4AttnParams &p, int D, int64_t &bytes) {
  constexpr int64_t cap = 1ll << 30;
  const int ck = kv4_sub_chunk(p.c.max_seq), nsub = (p.max_prefix + p.n + ck - 1) / ck;
  if (nsub <= 1) {
    bytes = 0;
    return p.n;
  }
  const int64_t per = (int64_t)p.c.n_seq * p.c.kvh * nsub * p.rep * (D * 4 + 8);
  const int sl = (int)std::min<int64_t>(p.n, std::max<int64_t>(1, cap / per));
  bytes = sl == p.n ? per * sl : std::max(cap, per);
  return sl;
}

template <int D>
static int kv4_attn_launch(Kv4AttnParams p, void *ws, bool pdl, cudaStream_t stream) {
  const bool split = p.dtype == LBX_F32;
  int64_t bytes = 0;
  const int sl = kv4_slice(p, D, bytes);
  static DevCache<int> attr;
  int unused = 0;
  int rc = attr.get(unused, [](int &) {
    cudaError_t e = allow_max_smem(kv4_attn_kernel<D, true>);
    if (e == cudaSuccess) e = allow_max_smem(kv4_attn_kernel<D, false>);
    return cuda_status(e, "kv4_attn smem attribute");
  });
  if (rc) return rc;
  for (int i0 = 0; i0 < p.n; i0 += sl) {
    kv4_cut(p, i0, std::min(sl, p.n - i0));
    p.part_ml = reinterpret_cast<float2 *>(ws);
    const int64_t rows = (int64_t)p.c.n_seq * p.c.kvh * p.nsub * p.R;
    p.part_o = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(ws) + ((rows * 8 + 255) & ~(int64_t)255));
    const int runs = (p.nsub + p.cpw - 1) / p.cpw;
    const int64_t gx = (int64_t)((runs + p.kw - 1) / p.kw) * ((p.ntile + p.rw - 1) / p.rw);
    LBX_CHECK_SUP(gx <= 0x7fffffff && p.c.kvh <= 65535 && p.c.n_seq <= 65535, "too many heads, sequences or rows");
    const dim3 grid((unsigned)gx, p.c.kvh, p.c.n_seq), block(32 * p.kw * p.rw);
    const size_t smem = (size_t)p.kw * KA_ST * Kv4Stage<D>::BYTES;
    const bool dep = pdl || i0 > 0;  // (every kernel here waits for the one before it)
    rc = cuda_status(split ? launch(kv4_attn_kernel<D, true>, grid, block, smem, stream, dep, p)
                           : launch(kv4_attn_kernel<D, false>, grid, block, smem, stream, dep, p),
                     "kv4_attn launch");
    if (rc) return rc;
    if (p.nsub > 1) {
      rc = cuda_status(launch(kv4_merge_kernel<D>, dim3(p.R, p.c.kvh, p.c.n_seq), dim3(KM_WARPS * 32), 0, stream, true, p),
                       "kv4_merge launch");
      if (rc) return rc;
    }
  }
  return LBX_OK;
}
}  // namespace lbx

extern "C" size_t lbx_kv4_attn_workspace_size(const lbx_kv4_attn_args *a) {
  lbx::Kv4AttnParams p = {};
  if (lbx::kv4_attn_prep(a, p)) return 0;
  int64_t bytes = 0;
  lbx::kv4_slice(p, a->cache.head_dim, bytes);
  return (size_t)bytes + 512;
}

extern "C" int lbx_kv4_attn(const lbx_kv4_attn_args *a, void *ws, size_t ws_bytes, cudaStream_t stream) {
  using namespace lbx;
  Kv4AttnParams p = {};
  int rc = kv4_attn_prep(a, p);
  if (rc) return rc;
  LBX_CHECK_ARG(a->q && a->out, "NULL pointer");
  LBX_CHECK_ARG(aligned16(a->out), "out must be 16-byte aligned");
  const size_t need = lbx_kv4_attn_workspace_size(a);
  LBX_CHECK_ARG(ws && ws_bytes >= need, "workspace too small (%zu < %zu)", ws_bytes, need);
  LBX_CHECK_ARG(aligned16(ws), "the workspace must be 16-byte aligned");
  return a->cache.head_dim == 128 ? kv4_attn_launch<128>(p, ws, a->use_pdl != 0, stream)
                                  : kv4_attn_launch<64>(p, ws, a->use_pdl != 0, stream);
}
