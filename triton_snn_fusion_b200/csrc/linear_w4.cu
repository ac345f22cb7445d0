// Linear layer over a few tokens with 4-bit weights:
//
//   y[m][n] = sum_k x[m][k] (q[n][k] - zero[n][k / G]) scale[n][k / G] + b[n]
//
// q holds two weights per byte along K (even k in the low half), zero defaults to 8.
#include "common.cuh"

namespace snnb {
namespace {

struct W4Args {
  const void *x, *scales, *bias;
  const uint8_t *q, *zeros;
  void *y;
  int64_t xs, ys, M;
  int K, N, G, groups;
};

// One warp per output value.
template <typename T>
__global__ void __launch_bounds__(256) linear_w4_kernel(W4Args a) {
  const int lane = threadIdx.x % 32;
  const int n = blockIdx.x * 8 + threadIdx.x / 32;
  const int64_t m = blockIdx.y + (int64_t)blockIdx.z * 65535;
  if (n >= a.N || m >= a.M) return;
  const T *x = static_cast<const T *>(a.x) + m * a.xs;
  const uint8_t *w = a.q + (int64_t)n * (a.K / 2);
  float acc = 0.f;
  for (int k = 2 * lane; k < a.K; k += 64) {
    const int64_t g = (int64_t)n * a.groups + k / a.G;
    const float s = DT<T>::to_f(static_cast<const T *>(a.scales)[g]), z = a.zeros ? (float)a.zeros[g] : 8.f;
    const int b = w[k / 2];
    acc += s * (DT<T>::to_f(x[k]) * ((float)(b & 15) - z) + DT<T>::to_f(x[k + 1]) * ((float)(b >> 4) - z));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane == 0) {
    if (a.bias) acc += DT<T>::to_f(static_cast<const T *>(a.bias)[n]);
    static_cast<T *>(a.y)[m * a.ys + n] = DT<T>::from_f(acc);
  }
}

}  // namespace
}  // namespace snnb

extern "C" int snnb_linear_w4(const void *x, int64_t x_stride, const void *q_weight, const void *scales,
                              const void *zeros, const void *bias, void *y, int64_t y_stride,
                              int64_t M, int K, int N, int group_size, int dtype, void *stream) {
  using namespace snnb;
  SNNB_CHECK_ARG(M >= 0 && M <= 0x7fffffffLL && K >= 1 && N >= 1, "linear_w4: sizes must be positive");
  SNNB_CHECK_ARG(is_act_dtype(dtype), "linear_w4: unsupported dtype %d", dtype);
  SNNB_CHECK_ARG(group_size == 32 || group_size == 64 || group_size == 128, "linear_w4: groups of 32, 64 or 128 values, got %d",
                 group_size);
  if (K % 32 != 0) return fail(SNNB_ERR_UNSUPPORTED, "linear_w4: K must be a multiple of 32, got %d", K);
  SNNB_CHECK_ARG((int64_t)N * K < (1LL << 40), "linear_w4: problem too large");
  if (M == 0) return SNNB_OK;
  SNNB_CHECK_ARG(x && q_weight && scales && y, "linear_w4: null pointer");
  SNNB_CHECK_ARG(x_stride >= 0 && (M <= 1 || y_stride >= N), "linear_w4: bad row stride");
  SNNB_CHECK_ARG(aligned16(q_weight), "linear_w4: q_weight must be 16-byte aligned");
  W4Args a;
  a.x = x; a.scales = scales; a.bias = bias; a.q = static_cast<const uint8_t *>(q_weight);
  a.zeros = static_cast<const uint8_t *>(zeros); a.y = y; a.xs = x_stride; a.ys = y_stride; a.M = M;
  a.K = K; a.N = N; a.G = group_size; a.groups = (K + group_size - 1) / group_size;
  const dim3 grid((unsigned)((N + 7) / 8), (unsigned)(M < 65535 ? M : 65535), (unsigned)((M + 65534) / 65535));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SNNB_F32: linear_w4_kernel<float><<<grid, 256, 0, s>>>(a); break;
    case SNNB_BF16: linear_w4_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a); break;
    default: linear_w4_kernel<__half><<<grid, 256, 0, s>>>(a); break;
  }
  SNNB_CHECK_LAUNCH("linear_w4");
  return SNNB_OK;
}
