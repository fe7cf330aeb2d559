// Matrix product in 8-bit integers, a scale for each token and each channel:
//
//   y_tn = s_t * w_n * sum_k c_tk W_nk (+ b_n),   c_tk = rint(x_tk * 127 / a_t),
//   a_t = max_k |x_tk|,  s_t = a_t / 127
//
// The sums are exact int32 (127 * 128 * 131072 < 2^31), so every split of the
// work gives the same bits.
#include "common.cuh"

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

// 64 tokens x 64 channels a CTA, four products at a time (dp4a)
constexpr int I8_T = 64;
__global__ void __launch_bounds__(256) linear_int8_kernel(const int8_t *__restrict__ q, int64_t q_ld,
                                                          const float *__restrict__ s, const int8_t *__restrict__ w,
                                                          int64_t w_ld, const float *__restrict__ ws,
                                                          const float *__restrict__ bias, int m, int n, int k,
                                                          void *__restrict__ y, int64_t y_ld, int ydt) {
  __shared__ int sx[16][I8_T + 1], sw[16][I8_T + 1];
  const int n0 = blockIdx.x * I8_T, m0 = blockIdx.y * I8_T;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < k; k0 += 64) {
    for (int e = tid; e < 16 * I8_T; e += 256) {
      const int c = e & 15, r = e >> 4, kk = k0 + 4 * c;
      int a = 0, b = 0;
      for (int i = 0; i < 4; ++i) {
        if (kk + i >= k) break;
        if (m0 + r < m) a |= (int)(uint8_t)q[(int64_t)(m0 + r) * q_ld + kk + i] << (8 * i);
        if (n0 + r < n) b |= (int)(uint8_t)w[(int64_t)(n0 + r) * w_ld + kk + i] << (8 * i);
      }
      sx[c][r] = a;
      sw[c][r] = b;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 16; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sx[c][ty + 16 * i], sw[c][tx + 16 * j], acc[i][j]);
    }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int t = m0 + ty + 16 * i, c = n0 + tx + 16 * j;
      if (t >= m || c >= n) continue;
      float v = __int2float_rn(acc[i][j]) * s[t] * ws[c];
      if (bias) v += bias[c];
      if (ydt == LBX_F32) reinterpret_cast<float *>(y)[(int64_t)t * y_ld + c] = v;
      else reinterpret_cast<uint16_t *>(y)[(int64_t)t * y_ld + c] = f32_to_bf16(v);
    }
}

struct Int8Ws {
  size_t q, s, total;
  int64_t q_ld;
};
static Int8Ws int8_ws(int m, int k) {
  auto al = [](size_t v) { return (v + 255) & ~(size_t)255; };
  Int8Ws w;
  w.q_ld = (k + 15) & ~15;
  w.s = 0;
  w.q = al((size_t)m * 4);
  w.total = w.q + al((size_t)m * w.q_ld);
  return w;
}

static int quant_tokens_launch(const void *x, int xdt, int64_t x_ld, int m, int k, int8_t *q, int64_t q_ld,
                               float *scale, cudaStream_t stream) {
  quant_tokens_kernel<<<m, Q8_THREADS, 0, stream>>>(x, xdt, x_ld, k, q, q_ld, scale);
  return cuda_status(cudaGetLastError(), "quant_tokens launch");
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
  return quant_tokens_launch(x, x_dtype, x_ld, m, k, q, q_ld, scale, stream);
}

extern "C" size_t lbx_linear_int8_workspace_size(int32_t m, int32_t n, int32_t k) {
  if (m < 1 || n < 1 || k < 1) return 0;
  return lbx::int8_ws(m, k).total;
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
  const Int8Ws W = int8_ws(a->m, a->k);
  LBX_CHECK_ARG(ws && ws_bytes >= W.total, "workspace too small (%zu < %zu)", ws_bytes, W.total);
  uint8_t *b = reinterpret_cast<uint8_t *>(ws);
  int8_t *q = reinterpret_cast<int8_t *>(b + W.q);
  float *s = reinterpret_cast<float *>(b + W.s);
  int rc = quant_tokens_launch(a->x, a->x_dtype, a->x_ld, a->m, a->k, q, W.q_ld, s, stream);
  if (rc) return rc;
  const dim3 grid((a->n + I8_T - 1) / I8_T, (a->m + I8_T - 1) / I8_T);
  linear_int8_kernel<<<grid, 256, 0, stream>>>(q, W.q_ld, s, a->w, a->w_ld, a->w_scale, a->bias, a->m, a->n, a->k,
                                               a->y, a->y_ld, a->y_dtype);
  return cuda_status(cudaGetLastError(), "linear_int8 launch");
}
