// The norm behind a block, its gate and residual scale, and the norm in front of the next block, on rows of D values:
//
//   n      = y * rstd(y) * w_post              (or y, without the norm behind the block)
//   res'   = res + alpha * res_scale * act(gate) * n
//   z      = res' * rstd(res') * w_pre
//   rstd(v) = 1 / sqrt(mean(v^2) + eps)
//
// Backward, with G the whole gradient of res' and nh = y * rstd(y):
//
//   u  = w_pre dz                    G = dres' + rstd(res') u - res' rstd(res')^3 mean(res' u)
//   c  = alpha res_scale w_post      e = G c act(gate)         dy = rstd(y) e - y rstd(y)^3 mean(y e)
//   dgate = G c nh act'(gate)        dres = G                  dw_pre = sum_m dz res' rstd(res')
//   Q  = alpha sum_m G act(gate) nh  dw_post = Q res_scale     dres_scale = Q w_post
//
// so that both parameters of the block's end share one column sum.
#include "common.cuh"

namespace snnb {
namespace {

constexpr int kThreads = 256;

struct NormArgs {
  const void *y, *gate, *res, *w_post, *scale, *w_pre, *dres_out, *dz;
  int64_t ys, gs, rs, dos, dzs;      // row strides
  void *res_out, *z;                 // forward outputs
  void *dy, *dgate, *dres;           // backward outputs
  float *partial;                    // [blocks][2][D]: column sums Q and dw_pre
  float *dw_post, *dscale, *dw_pre;
  int64_t M;
  int D, w_f32, act, post_norm;
  float alpha, eps;
};

template <typename T> __device__ __forceinline__ float param(const void *p, int f32, int i) {
  if (p == nullptr) return 1.f;
  return f32 ? static_cast<const float *>(p)[i] : DT<T>::to_f(static_cast<const T *>(p)[i]);
}

__device__ __forceinline__ float sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

// act(g) and its derivative
__device__ __forceinline__ void act_of(int act, float g, float &v, float &dv) {
  if (act == SNNB_ACT_NONE) { v = 1.f; dv = 0.f; return; }
  const float p = sigmoid(g);
  if (act == SNNB_ACT_SIGMOID) { v = p; dv = p * sigmoid(-g); }
  else { v = g * p; dv = p * (1.f + g * sigmoid(-g)); }
}

__device__ __forceinline__ float block_sum(float v, float *sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) s += sh[i];
  return s;
}

template <typename T> struct Row {
  const NormArgs &q;
  const T *y, *gate, *res;
  __device__ Row(const NormArgs &a, int64_t m)
      : q(a), y(static_cast<const T *>(a.y) + (a.y ? m * a.ys : 0)),
        gate(static_cast<const T *>(a.gate) + (a.gate ? m * a.gs : 0)),
        res(static_cast<const T *>(a.res) + (a.res ? m * a.rs : 0)) {}
  __device__ float out(int i, float rstd_y) const {
    float r = q.res ? DT<T>::to_f(res[i]) : 0.f;
    if (q.y) {
      float av, dv;
      act_of(q.act, q.gate ? DT<T>::to_f(gate[i]) : 0.f, av, dv);
      const float c = q.alpha * param<T>(q.scale, q.w_f32, i) * (q.post_norm ? param<T>(q.w_post, q.w_f32, i) : 1.f);
      r += c * av * (DT<T>::to_f(y[i]) * rstd_y);
    }
    return r;
  }
  __device__ float rstd_y(float *sh) const {
    if (!q.y || !q.post_norm) return 1.f;
    float s = 0.f;
    for (int i = threadIdx.x; i < q.D; i += kThreads) { const float v = DT<T>::to_f(y[i]); s += v * v; }
    return rsqrtf(block_sum(s, sh) / q.D + q.eps);
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) block_norm_kernel(NormArgs q) {
  __shared__ float sh[kThreads / 32];
  for (int64_t m = blockIdx.x; m < q.M; m += gridDim.x) {
    const Row<T> row(q, m);
    const float ry = row.rstd_y(sh);
    float s = 0.f;
    if (q.z) {
      for (int i = threadIdx.x; i < q.D; i += kThreads) { const float v = row.out(i, ry); s += v * v; }
      s = rsqrtf(block_sum(s, sh) / q.D + q.eps);
    }
    for (int i = threadIdx.x; i < q.D; i += kThreads) {
      const float v = row.out(i, ry);
      if (q.z) static_cast<T *>(q.z)[m * q.D + i] = DT<T>::from_f(v * s * param<T>(q.w_pre, q.w_f32, i));
      if (q.res_out) static_cast<T *>(q.res_out)[m * q.D + i] = DT<T>::from_f(v);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) block_norm_backward_kernel(NormArgs q) {
  __shared__ float sh[kThreads / 32];
  float *pq = q.partial + (int64_t)blockIdx.x * 2 * q.D, *pw = pq + q.D;
  for (int i = threadIdx.x; i < q.D; i += kThreads) pq[i] = pw[i] = 0.f;
  for (int64_t m = blockIdx.x; m < q.M; m += gridDim.x) {
    const Row<T> row(q, m);
    const T *dz = static_cast<const T *>(q.dz) + (q.dz ? m * q.dzs : 0);
    const T *dro = static_cast<const T *>(q.dres_out) + (q.dres_out ? m * q.dos : 0);
    const float ry = row.rstd_y(sh);
    float so = 0.f, sd = 0.f, ro = 0.f, mo = 0.f;
    if (q.dz) {
      for (int i = threadIdx.x; i < q.D; i += kThreads) {
        const float v = row.out(i, ry);
        so += v * v;
        sd += v * DT<T>::to_f(dz[i]) * param<T>(q.w_pre, q.w_f32, i);
      }
      ro = rsqrtf(block_sum(so, sh) / q.D + q.eps);
      mo = block_sum(sd, sh) / q.D * ro * ro * ro;
    }
    float se = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      const float me = pass ? block_sum(se, sh) / q.D * ry * ry * ry : 0.f;
      for (int i = threadIdx.x; i < q.D; i += kThreads) {
        float G = q.dres_out ? DT<T>::to_f(dro[i]) : 0.f;
        if (q.dz) {
          const float v = row.out(i, ry), d = DT<T>::to_f(dz[i]);
          G += ro * d * param<T>(q.w_pre, q.w_f32, i) - v * mo;
          if (pass) pw[i] += d * v * ro;
        }
        if (q.y) {
          float av, dv;
          act_of(q.act, q.gate ? DT<T>::to_f(row.gate[i]) : 0.f, av, dv);
          const float c = q.alpha * param<T>(q.scale, q.w_f32, i) * (q.post_norm ? param<T>(q.w_post, q.w_f32, i) : 1.f);
          const float yv = DT<T>::to_f(row.y[i]), e = G * c * av;
          if (!pass) {
            se += yv * e;
          } else {
            static_cast<T *>(q.dy)[m * q.D + i] = DT<T>::from_f(q.post_norm ? ry * e - yv * me : e);
            if (q.dgate) static_cast<T *>(q.dgate)[m * q.D + i] = DT<T>::from_f(G * c * yv * ry * dv);
            pq[i] += q.alpha * G * av * yv * ry;
          }
        }
        if (pass && q.dres) static_cast<T *>(q.dres)[m * q.D + i] = DT<T>::from_f(G);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) block_norm_sums_kernel(NormArgs q, int blocks) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= q.D) return;
  float sq = 0.f, sw = 0.f;
  for (int b = 0; b < blocks; ++b) {
    sq += q.partial[(int64_t)b * 2 * q.D + i];
    sw += q.partial[(int64_t)b * 2 * q.D + q.D + i];
  }
  if (q.dw_post) q.dw_post[i] = sq * param<T>(q.scale, q.w_f32, i);
  if (q.dscale) q.dscale[i] = sq * (q.post_norm ? param<T>(q.w_post, q.w_f32, i) : 1.f);
  if (q.dw_pre) q.dw_pre[i] = sw;
}

// Blocks of the backward pass, each of which leaves one row of column sums.
int backward_blocks(int64_t M) { return (int)(M < 592 ? (M < 1 ? 1 : M) : 592); }

int check_common(const NormArgs &q, int dtype, int w_dtype, const char *what) {
  SNNB_CHECK_ARG(q.M >= 0 && q.M <= 0x7fffffffLL, "%s: bad number of rows", what);
  SNNB_CHECK_ARG(q.D >= 1, "%s: D must be positive", what);
  if (q.D > SNNB_BLOCK_NORM_MAX_D)
    return fail(SNNB_ERR_UNSUPPORTED, "%s: rows of more than %d values are not implemented", what, SNNB_BLOCK_NORM_MAX_D);
  SNNB_CHECK_ARG(is_act_dtype(dtype), "%s: unsupported dtype %d", what, dtype);
  SNNB_CHECK_ARG(w_dtype == dtype || w_dtype == SNNB_F32, "%s: parameter dtype must be the y dtype or f32", what);
  SNNB_CHECK_ARG(q.act >= SNNB_ACT_NONE && q.act <= SNNB_ACT_SILU, "%s: bad gate activation %d", what, q.act);
  SNNB_CHECK_ARG(q.M == 0 || (q.act == SNNB_ACT_NONE) == (q.gate == nullptr), "%s: a gate needs an activation and the reverse", what);
  SNNB_CHECK_ARG(q.eps >= 0.f, "%s: eps must not be negative", what);
  SNNB_CHECK_ARG(q.ys >= 0 && q.gs >= 0 && q.rs >= 0 && q.dos >= 0 && q.dzs >= 0, "%s: negative stride", what);
  if (!q.y) {
    SNNB_CHECK_ARG(!q.gate && !q.w_post && !q.scale && !q.post_norm, "%s: gate, w_post and res_scale belong to y", what);
    SNNB_CHECK_ARG(q.res || q.M == 0, "%s: neither y nor res", what);
  }
  SNNB_CHECK_ARG(q.post_norm || !q.w_post, "%s: w_post without the norm it belongs to", what);
  return SNNB_OK;
}

}  // namespace
}  // namespace snnb

extern "C" int snnb_block_norm(const void *y, int64_t y_stride, const void *gate, int64_t gate_stride,
                               const void *res, int64_t res_stride, const void *w_post, const void *res_scale,
                               const void *w_pre, void *res_out, void *z, int64_t M, int D, float alpha, float eps,
                               int gate_act, int post_norm, int dtype, int w_dtype, void *stream) {
  using namespace snnb;
  NormArgs q = {};
  q.y = y; q.ys = y_stride; q.gate = gate; q.gs = gate_stride; q.res = res; q.rs = res_stride;
  q.w_post = w_post; q.scale = res_scale; q.w_pre = w_pre; q.res_out = res_out; q.z = z;
  q.M = M; q.D = D; q.alpha = alpha; q.eps = eps; q.act = gate_act; q.post_norm = post_norm != 0;
  q.w_f32 = w_dtype == SNNB_F32;
  if (const int st = check_common(q, dtype, w_dtype, "block_norm")) return st;
  SNNB_CHECK_ARG(res_out || z || M == 0, "block_norm: neither res_out nor z");
  SNNB_CHECK_ARG(z || !w_pre, "block_norm: w_pre without z");
  SNNB_CHECK_ARG(!res || res_out != res || M <= 1 || res_stride == D,
                 "block_norm: res can be updated in place only if its rows are dense");
  if (M == 0) return SNNB_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned blocks = (unsigned)M;
  switch (dtype) {
    case SNNB_F32: block_norm_kernel<float><<<blocks, kThreads, 0, s>>>(q); break;
    case SNNB_BF16: block_norm_kernel<__nv_bfloat16><<<blocks, kThreads, 0, s>>>(q); break;
    default: block_norm_kernel<__half><<<blocks, kThreads, 0, s>>>(q); break;
  }
  SNNB_CHECK_LAUNCH("block_norm");
  return SNNB_OK;
}

extern "C" int64_t snnb_block_norm_backward_workspace_bytes(int64_t M, int D) {
  return (int64_t)snnb::backward_blocks(M) * 2 * (D > 0 ? D : 0) * (int64_t)sizeof(float);
}

namespace snnb {
namespace {
template <typename T> void launch_backward(const NormArgs &q, cudaStream_t s) {
  const int blocks = backward_blocks(q.M);
  block_norm_backward_kernel<T><<<blocks, kThreads, 0, s>>>(q);
  if (q.dw_post || q.dscale || q.dw_pre)
    block_norm_sums_kernel<T><<<(q.D + kThreads - 1) / kThreads, kThreads, 0, s>>>(q, blocks);
}
}  // namespace
}  // namespace snnb

extern "C" int snnb_block_norm_backward(const void *dres_out, int64_t dres_out_stride, const void *dz, int64_t dz_stride,
                                        const void *y, int64_t y_stride, const void *gate, int64_t gate_stride,
                                        const void *res, int64_t res_stride, const void *w_post, const void *res_scale,
                                        const void *w_pre, void *dy, void *dgate, void *dres,
                                        float *dw_post, float *dres_scale, float *dw_pre,
                                        void *workspace, int64_t workspace_bytes, int64_t M, int D,
                                        float alpha, float eps, int gate_act, int post_norm, int dtype, int w_dtype,
                                        void *stream) {
  using namespace snnb;
  NormArgs q = {};
  q.y = y; q.ys = y_stride; q.gate = gate; q.gs = gate_stride; q.res = res; q.rs = res_stride;
  q.dres_out = dres_out; q.dos = dres_out_stride; q.dz = dz; q.dzs = dz_stride;
  q.w_post = w_post; q.scale = res_scale; q.w_pre = w_pre;
  q.dy = dy; q.dgate = dgate; q.dres = dres; q.dw_post = dw_post; q.dscale = dres_scale; q.dw_pre = dw_pre;
  q.partial = static_cast<float *>(workspace);
  q.M = M; q.D = D; q.alpha = alpha; q.eps = eps; q.act = gate_act; q.post_norm = post_norm != 0;
  q.w_f32 = w_dtype == SNNB_F32;
  if (const int st = check_common(q, dtype, w_dtype, "block_norm_backward")) return st;
  SNNB_CHECK_ARG(dres_out || dz || M == 0, "block_norm_backward: neither dres_out nor dz");
  SNNB_CHECK_ARG(dz || !w_pre, "block_norm_backward: w_pre without dz");
  SNNB_CHECK_ARG(!dy == !y || M == 0, "block_norm_backward: dy belongs to y and the reverse");
  SNNB_CHECK_ARG(!dgate == !gate || M == 0, "block_norm_backward: dgate belongs to the gate and the reverse");
  SNNB_CHECK_ARG(!dw_post || post_norm, "block_norm_backward: dw_post without the norm it belongs to");
  SNNB_CHECK_ARG(!dres_scale || y || M == 0, "block_norm_backward: dres_scale without y");
  SNNB_CHECK_ARG(!dw_pre || dz || M == 0, "block_norm_backward: dw_pre without dz");
  SNNB_CHECK_ARG(workspace && workspace_bytes >= snnb_block_norm_backward_workspace_bytes(M, D),
                 "block_norm_backward: workspace too small");
  SNNB_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "block_norm_backward: workspace must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SNNB_F32: launch_backward<float>(q, s); break;
    case SNNB_BF16: launch_backward<__nv_bfloat16>(q, s); break;
    default: launch_backward<__half>(q, s); break;
  }
  SNNB_CHECK_LAUNCH("block_norm_backward");
  return SNNB_OK;
}
