// A linear layer in 8-bit integers: y[m,n] = act(x_scale[m] w_scale[n] sum_k x[m,k] w[n,k] + bias[n])
// with one scale per token and one per output channel, and the operator that makes x: rows divided
// by their largest magnitude / 127 and rounded to the nearest whole number, ties to even.
//
// The sums are exact (32-bit integers, K <= 131071 keeps |sum| below 2^31); scales, bias and the
// activation are 32-bit floats, rounded once at the store.
#include "common.cuh"

namespace b200 {
namespace int8 {

constexpr int64_t kMaxK = 131071;  // 128 * 128 * K < 2^31

// ------------------------------------------------------------------------- rows to 8 bits
// One CTA per row.  The magnitudes are compared as integers, which order like the floats and put
// a NaN above infinity: a row that holds either gets a scale that is not finite and zero codes.
struct QuantParams {
  const void *x;
  int8_t *out;
  float *scale;
  int64_t x_row, o_row;
  int M, K;
};

__device__ __forceinline__ int round_code(float x, float scale, float inv) {
  const float y = x * inv;  // |y| <= 127: within 3e-5 of the quotient while 1 / scale is normal
  float r = rintf(y);
  if (!(fabsf(fabsf(y - r) - 0.5f) > 1e-4f) || scale < 1e-30f)
    r = (float)rint((double)x / (double)scale);
  return (int)fminf(fmaxf(r, -127.f), 127.f);
}

constexpr int QTHREADS = 256;

template <typename T>
__global__ void __launch_bounds__(QTHREADS) quantize_rows_kernel(const QuantParams p) {
  __shared__ unsigned int tops[QTHREADS / 32];
  const int64_t m = blockIdx.x;
  const T *x = (const T *)p.x + m * p.x_row;
  unsigned int top = 0;
  for (int i = threadIdx.x; i < p.K; i += QTHREADS)
    top = max(top, __float_as_uint(io<T>::load(x[i])) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int w = 0; w < QTHREADS / 32; ++w) top = max(top, tops[w]);
  const float scale = __fdiv_rn(__uint_as_float(top), 127.f);
  const bool usable = scale > 0.f && scale < INFINITY;
  const float inv = 1.f / scale;
  int8_t *out = p.out + m * p.o_row;
  for (int i = threadIdx.x; i < p.K; i += QTHREADS)
    out[i] = usable ? (int8_t)round_code(io<T>::load(x[i]), scale, inv) : (int8_t)0;
  if (threadIdx.x == 0) p.scale[m] = scale;
}

// ------------------------------------------------------------------------- the product
struct Params {
  const int8_t *x, *w;
  const float *x_scale, *w_scale;
  const void *bias;
  void *y;
  int64_t x_row, w_row, y_row;
  int M, N, K;
  int act, bias_kind;
};

__device__ __forceinline__ float load_bias(const void *bias, int kind, int col) {
  if (kind == 0) return 0.f;
  if (kind == B200_DTYPE_FLOAT32) return ((const float *)bias)[col];
  if (kind == B200_DTYPE_BFLOAT16) return __bfloat162float(((const __nv_bfloat16 *)bias)[col]);
  return __half2float(((const __half *)bias)[col]);
}

// 16-bit results take the short tanh (its error is below half their rounding)
template <typename T> __device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case B200_ACT_GELU_ERF: return 0.5f * z * (1.0f + erff(z * 0.7071067811865476f));
    case B200_ACT_GELU_TANH: return 0.5f * z * (1.0f + tanhf(0.79788456f * (z + 0.044715f * z * z * z)));
    case B200_ACT_LEAKY_RELU: return z >= 0.f ? z : 0.01f * z;
    default: return z;
  }
}

// Any sizes and alignment: 32 x 32 outputs per CTA, operands staged in shared memory.
constexpr int TILE = 32;

template <typename T>
__global__ void __launch_bounds__(256) linear_int8_tile_kernel(const Params p) {
  __shared__ int8_t xs[TILE][TILE + 4], ws[TILE][TILE + 4];
  const int m0 = (int)blockIdx.y * TILE, n0 = (int)blockIdx.x * TILE;
  const int col = threadIdx.x & 31, group = threadIdx.x >> 5;  // 8 groups of 4 rows
  int acc[4] = {0, 0, 0, 0};
  for (int k0 = 0; k0 < p.K; k0 += TILE) {
    for (int i = group; i < TILE; i += 8) {
      const int k = k0 + col;
      xs[i][col] = (m0 + i < p.M && k < p.K) ? p.x[(int64_t)(m0 + i) * p.x_row + k] : (int8_t)0;
      ws[i][col] = (n0 + i < p.N && k < p.K) ? p.w[(int64_t)(n0 + i) * p.w_row + k] : (int8_t)0;
    }
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < TILE; ++k) {
      const int b = ws[col][k];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += b * (int)xs[group * 4 + i][k];
    }
    __syncthreads();
  }
  const int n = n0 + col;
  if (n >= p.N) return;
  const float sw = p.w_scale[n], b = load_bias(p.bias, p.bias_kind, n);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + group * 4 + i;
    if (m < p.M)
      ((T *)p.y)[(int64_t)m * p.y_row + n] =
          io<T>::store(activate<T>(fmaf((float)acc[i], p.x_scale[m] * sw, b), p.act));
  }
}

template <typename T> static int launch(const Params &p, cudaStream_t stream) {
  const dim3 grid((unsigned)((p.N + TILE - 1) / TILE), (unsigned)((p.M + TILE - 1) / TILE));
  if (grid.y > 65535u) return fail(B200_REJECTED, "%d rows exceed the limit of the unaligned path", p.M);
  linear_int8_tile_kernel<T><<<grid, 256, 0, stream>>>(p);
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}

}  // namespace int8
}  // namespace b200

extern "C" int b200_quantize_rows(const b200_tensor *x, b200_tensor *out, b200_tensor *scale, void *stream) {
  using namespace b200;
  int st;
  if ((st = check_tensor(x, "x", 2)) || (st = check_tensor(out, "out", 2)) || (st = check_tensor(scale, "scale", 1)))
    return st;
  const int64_t M = x->shape[0], K = x->shape[1];
  B200_REQUIRE(is_float_io(x->dtype), "x: dtype %u is not f16/bf16/f32", x->dtype);
  B200_REQUIRE(out->dtype == B200_DTYPE_INT8 && out->shape[0] == M && out->shape[1] == K, "out must be int8 [M, K]");
  B200_REQUIRE(scale->dtype == B200_DTYPE_FLOAT32 && scale->shape[0] == M && scale->stride[0] == 1,
               "scale must be contiguous f32 [M]");
  B200_REQUIRE(x->stride[1] == 1 && out->stride[1] == 1, "x and out need a unit column stride");
  B200_REQUIRE(M < (1ll << 31) && K < (1ll << 31), "rows or columns out of range");
  if (M == 0) return B200_OK;
  if ((st = check_reachable(x->data, "x")) || (st = check_reachable(out->data, "out")) ||
      (st = check_reachable(scale->data, "scale")))
    return st;
  int8::QuantParams p;
  p.x = x->data; p.out = (int8_t *)out->data; p.scale = (float *)scale->data;
  p.x_row = x->stride[0]; p.o_row = out->stride[0]; p.M = (int)M; p.K = (int)K;
  cudaStream_t s = (cudaStream_t)stream;
  if (x->dtype == B200_DTYPE_FLOAT32) int8::quantize_rows_kernel<float><<<(unsigned)M, int8::QTHREADS, 0, s>>>(p);
  else if (x->dtype == B200_DTYPE_FLOAT16) int8::quantize_rows_kernel<__half><<<(unsigned)M, int8::QTHREADS, 0, s>>>(p);
  else int8::quantize_rows_kernel<__nv_bfloat16><<<(unsigned)M, int8::QTHREADS, 0, s>>>(p);
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}

extern "C" int b200_linear_int8(const b200_tensor *x, const b200_tensor *x_scale, const b200_tensor *w,
                                const b200_tensor *w_scale, const b200_tensor *bias, b200_tensor *y, int act,
                                void *stream) {
  using namespace b200;
  int st;
  if ((st = check_tensor(x, "x", 2)) || (st = check_tensor(x_scale, "x_scale", 1)) || (st = check_tensor(w, "w", 2)) ||
      (st = check_tensor(w_scale, "w_scale", 1)) || (st = check_tensor(y, "y", 2)))
    return st;
  const int64_t M = x->shape[0], K = x->shape[1], N = w->shape[0];
  B200_REQUIRE(x->dtype == B200_DTYPE_INT8 && w->dtype == B200_DTYPE_INT8, "x and w must be int8");
  B200_REQUIRE(w->shape[1] == K, "x has %lld columns, w has %lld", (long long)K, (long long)w->shape[1]);
  B200_REQUIRE(K >= 1 && K <= int8::kMaxK, "K %lld out of range 1..%lld (32-bit sums)", (long long)K,
               (long long)int8::kMaxK);
  B200_REQUIRE(is_float_io(y->dtype) && y->shape[0] == M && y->shape[1] == N, "y must be f16/bf16/f32 [M, N]");
  B200_REQUIRE(x_scale->dtype == B200_DTYPE_FLOAT32 && x_scale->shape[0] == M && x_scale->stride[0] == 1,
               "x_scale must be contiguous f32 [M]");
  B200_REQUIRE(w_scale->dtype == B200_DTYPE_FLOAT32 && w_scale->shape[0] == N && w_scale->stride[0] == 1,
               "w_scale must be contiguous f32 [N]");
  B200_REQUIRE(x->stride[1] == 1 && w->stride[1] == 1 && y->stride[1] == 1, "x, w and y need a unit column stride");
  if (bias != nullptr) {
    if ((st = check_tensor(bias, "bias", 1))) return st;
    B200_REQUIRE(bias->shape[0] == N && bias->stride[0] == 1 && is_float_io(bias->dtype),
                 "bias must be contiguous f16/bf16/f32 [N]");
  }
  if (act != B200_ACT_NONE && act != B200_ACT_GELU_ERF && act != B200_ACT_GELU_TANH && act != B200_ACT_LEAKY_RELU)
    return fail(B200_USAGE, "activation %d is not available here", act);
  B200_REQUIRE(M < (1ll << 31) && N < (1ll << 31), "rows or columns out of range");
  if (M == 0 || N == 0) return B200_OK;
  if ((st = check_reachable(x->data, "x")) || (st = check_reachable(x_scale->data, "x_scale")) ||
      (st = check_reachable(w->data, "w")) || (st = check_reachable(w_scale->data, "w_scale")) ||
      (st = check_reachable(bias ? bias->data : nullptr, "bias")) || (st = check_reachable(y->data, "y")))
    return st;
  int8::Params p;
  p.x = (const int8_t *)x->data; p.w = (const int8_t *)w->data;
  p.x_scale = (const float *)x_scale->data; p.w_scale = (const float *)w_scale->data;
  p.bias = bias ? bias->data : nullptr;
  p.bias_kind = bias ? (int)bias->dtype : 0;
  p.y = y->data;
  p.x_row = x->stride[0]; p.w_row = w->stride[0]; p.y_row = y->stride[0];
  p.M = (int)M; p.N = (int)N; p.K = (int)K; p.act = act;
  cudaStream_t s = (cudaStream_t)stream;
  if (y->dtype == B200_DTYPE_FLOAT32) return int8::launch<float>(p, s);
  if (y->dtype == B200_DTYPE_FLOAT16) return int8::launch<__half>(p, s);
  return int8::launch<__nv_bfloat16>(p, s);
}
