// Gated linear recurrence over time: the leaky charge step of a LIF neuron without the spike and with its leak given
// per step and channel.
//
//   a_t = gate_t  or  1 / (1 + exp(-gate_t))
//   h_t = a_t h_{t-1} + (1 - a_t) x_t   (leaky)      h_t = a_t h_{t-1} + x_t   (plain)
//
// Backward, with lam_t the whole gradient of h_t:
//
//   lam_t = dh_t + a_{t+1} lam_{t+1}        (lam_{T-1} = dh_{T-1} + dh_last)
//   dx_t  = (1 - a_t) lam_t   or lam_t      da_t = lam_t (h_{t-1} - x_t)   or lam_t h_{t-1}
//   dgate = da_t a_t (1 - a_t) or da_t      dh_init = a_0 lam_0
//
// The backward pass needs h_{t-1} in 32 bits; it recomputes the states of 128 steps at a time from the fp32
// checkpoints that the forward pass leaves, which is less traffic than reading the 16-bit h and more exact.
#include "common.cuh"

namespace snnb {
namespace {

constexpr int kCkptSteps = SNNB_GATED_SCAN_CKPT_STEPS;

struct Seq {          // rows of D values; element (t, b, d) at t * ts + b * bs + d
  const void *p;
  int64_t ts, bs;
};

struct ScanArgs {
  Seq x, g, h;        // h: the output of the forward pass, the gradient dh of the backward pass
  Seq dx, dg;
  const void *h_init;
  const void *dh_last;
  void *h_last;       // forward: last state; backward: dh_init
  float *ckpt;
  const int *lengths;
  int64_t T, B, D;
  int state_f32;
};

template <typename T> __device__ __forceinline__ float at(const Seq &s, int64_t t, int64_t b, int64_t d) {
  return DT<T>::to_f(static_cast<const T *>(s.p)[t * s.ts + b * s.bs + d]);
}
template <typename T> __device__ __forceinline__ void put(const Seq &s, int64_t t, int64_t b, int64_t d, float v) {
  static_cast<T *>(const_cast<void *>(s.p))[t * s.ts + b * s.bs + d] = DT<T>::from_f(v);
}
template <typename T> __device__ __forceinline__ float state_at(const void *p, int f32, int64_t i) {
  if (p == nullptr) return 0.f;
  return f32 ? static_cast<const float *>(p)[i] : DT<T>::to_f(static_cast<const T *>(p)[i]);
}
template <typename T> __device__ __forceinline__ void state_put(void *p, int f32, int64_t i, float v) {
  if (p == nullptr) return;
  if (f32) static_cast<float *>(p)[i] = v;
  else static_cast<T *>(p)[i] = DT<T>::from_f(v);
}

// Both a and 1 - a keep their relative accuracy: neither is the difference of the other from one.
template <bool SIG> __device__ __forceinline__ void gate_of(float g, float &a, float &b) {
  if constexpr (SIG) {
    const float e = __expf(-fabsf(g));
    const float big = __fdividef(1.f, 1.f + e), small = e * big;
    a = g >= 0.f ? big : small;
    b = g >= 0.f ? small : big;
  } else {
    a = g;
    b = 1.f - g;
  }
}

template <typename T, bool SIG, bool LEAKY>
__global__ void gated_scan_kernel(ScanArgs q) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= q.B * q.D) return;
  const int64_t b = i / q.D, d = i % q.D;
  int64_t len = q.T;
  if (q.lengths) len = min(max((int64_t)q.lengths[b], (int64_t)0), q.T);
  float h = state_at<T>(q.h_init, q.state_f32, i);
  for (int64_t t = 0; t < q.T; ++t) {
    if (t > 0 && t % kCkptSteps == 0 && q.ckpt) q.ckpt[(t / kCkptSteps - 1) * q.B * q.D + i] = h;
    if (t < len) {
      float a, bb;
      gate_of<SIG>(at<T>(q.g, t, b, d), a, bb);
      const float x = at<T>(q.x, t, b, d);
      h = fmaf(a, h, LEAKY ? bb * x : x);
      put<T>(q.h, t, b, d, h);
    } else {
      put<T>(q.h, t, b, d, 0.f);
    }
  }
  state_put<T>(q.h_last, q.state_f32, i, h);
}

template <typename T, bool SIG, bool LEAKY>
__global__ void gated_scan_backward_kernel(ScanArgs q) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= q.B * q.D) return;
  const int64_t b = i / q.D, d = i % q.D;
  int64_t len = q.T;
  if (q.lengths) len = min(max((int64_t)q.lengths[b], (int64_t)0), q.T);
  float lam = state_at<T>(q.dh_last, q.state_f32, i);
  for (int64_t t = len; t < q.T; ++t) {
    put<T>(q.dx, t, b, d, 0.f);
    put<T>(q.dg, t, b, d, 0.f);
  }
  float before[kCkptSteps];
  for (int64_t t0 = (len - 1) / kCkptSteps * kCkptSteps; len > 0 && t0 >= 0; t0 -= kCkptSteps) {
    const int n = (int)min((int64_t)kCkptSteps, len - t0);
    float h = t0 == 0 ? state_at<T>(q.h_init, q.state_f32, i) : q.ckpt[(t0 / kCkptSteps - 1) * q.B * q.D + i];
    for (int k = 0; k < n; ++k) {
      float a, bb;
      gate_of<SIG>(at<T>(q.g, t0 + k, b, d), a, bb);
      const float x = at<T>(q.x, t0 + k, b, d);
      before[k] = h;
      h = fmaf(a, h, LEAKY ? bb * x : x);
    }
    for (int k = n - 1; k >= 0; --k) {
      float a, bb;
      gate_of<SIG>(at<T>(q.g, t0 + k, b, d), a, bb);
      const float x = at<T>(q.x, t0 + k, b, d);
      lam += at<T>(q.h, t0 + k, b, d);
      float dg = lam * (LEAKY ? before[k] - x : before[k]);
      if (SIG) dg *= a * bb;
      put<T>(q.dx, t0 + k, b, d, LEAKY ? bb * lam : lam);
      put<T>(q.dg, t0 + k, b, d, dg);
      lam *= a;
    }
  }
  state_put<T>(q.h_last, q.state_f32, i, lam);
}

template <typename T, bool BWD>
void launch(const ScanArgs &q, int gate_kind, int leaky, cudaStream_t s) {
  const unsigned blocks = (unsigned)((q.B * q.D + 127) / 128);
  auto go = [&](auto kern) { kern<<<blocks, 128, 0, s>>>(q); };
  const bool sig = gate_kind == SNNB_GATE_SIGMOID;
  if constexpr (BWD) {
    if (sig && leaky) go(gated_scan_backward_kernel<T, true, true>);
    else if (sig) go(gated_scan_backward_kernel<T, true, false>);
    else if (leaky) go(gated_scan_backward_kernel<T, false, true>);
    else go(gated_scan_backward_kernel<T, false, false>);
  } else {
    if (sig && leaky) go(gated_scan_kernel<T, true, true>);
    else if (sig) go(gated_scan_kernel<T, true, false>);
    else if (leaky) go(gated_scan_kernel<T, false, true>);
    else go(gated_scan_kernel<T, false, false>);
  }
}

// Whether the T * B rows of an output lie apart from one another.
bool rows_apart(int64_t ts, int64_t bs, int64_t T, int64_t B, int64_t D) {
  if (T <= 1 && B <= 1) return true;
  if (T <= 1) return bs >= D;
  if (B <= 1) return ts >= D;
  return ts >= bs ? (bs >= D && ts >= bs * (B - 1) + D) : (ts >= D && bs >= ts * (T - 1) + D);
}

bool partly_same(const void *a, const void *b, int64_t bytes) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
  return p && q && p != q && p < q + (uintptr_t)bytes && q < p + (uintptr_t)bytes;
}

int check_common(const ScanArgs &q, int gate_kind, int dtype, int state_dtype, const char *what) {
  SNNB_CHECK_ARG(q.T >= 0 && q.B >= 0 && q.D >= 0, "%s: sizes must not be negative", what);
  SNNB_CHECK_ARG(q.T <= 0x7fffffffLL && q.B <= 0x7fffffffLL && q.D <= 0x7fffffffLL && q.B * q.D <= (1LL << 36),
                 "%s: problem too large", what);
  SNNB_CHECK_ARG(gate_kind == SNNB_GATE_VALUE || gate_kind == SNNB_GATE_SIGMOID, "%s: bad gate kind %d", what, gate_kind);
  SNNB_CHECK_ARG(is_act_dtype(dtype), "%s: unsupported dtype %d", what, dtype);
  SNNB_CHECK_ARG(state_dtype == dtype || state_dtype == SNNB_F32, "%s: state dtype must be the x dtype or f32", what);
  SNNB_CHECK_ARG(q.x.ts >= 0 && q.x.bs >= 0 && q.g.ts >= 0 && q.g.bs >= 0 && q.h.ts >= 0 && q.h.bs >= 0,
                 "%s: negative stride", what);
  if (q.T * q.B * q.D > 0) SNNB_CHECK_ARG(q.x.p && q.g.p && q.h.p, "%s: null pointer", what);
  return SNNB_OK;
}

}  // namespace
}  // namespace snnb

extern "C" int64_t snnb_gated_scan_ckpt_rows(int64_t T) {
  return T <= snnb::kCkptSteps ? 0 : (T - 1) / snnb::kCkptSteps;
}

extern "C" int snnb_gated_scan(const void *x, int64_t x_t_stride, int64_t x_b_stride,
                               const void *gate, int64_t g_t_stride, int64_t g_b_stride,
                               const void *h_init, const int *lengths,
                               void *h_seq, int64_t h_t_stride, int64_t h_b_stride, void *h_last, float *ckpt,
                               int64_t T, int64_t B, int64_t D, int gate_kind, int leaky, int dtype, int state_dtype,
                               void *stream) {
  using namespace snnb;
  ScanArgs q = {};
  q.x = {x, x_t_stride, x_b_stride};
  q.g = {gate, g_t_stride, g_b_stride};
  q.h = {h_seq, h_t_stride, h_b_stride};
  q.h_init = h_init; q.h_last = h_last; q.ckpt = ckpt; q.lengths = lengths;
  q.T = T; q.B = B; q.D = D; q.state_f32 = state_dtype == SNNB_F32;
  if (const int st = check_common(q, gate_kind, dtype, state_dtype, "gated_scan")) return st;
  SNNB_CHECK_ARG(rows_apart(h_t_stride, h_b_stride, T, B, D), "gated_scan: rows of h_seq overlap");
  SNNB_CHECK_ARG(!partly_same(h_init, h_last, B * D * dtype_size(state_dtype)),
                 "gated_scan: h_init and h_last overlap without being the same buffer");
  if (B * D == 0) return SNNB_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SNNB_F32: launch<float, false>(q, gate_kind, leaky, s); break;
    case SNNB_BF16: launch<__nv_bfloat16, false>(q, gate_kind, leaky, s); break;
    default: launch<__half, false>(q, gate_kind, leaky, s); break;
  }
  SNNB_CHECK_LAUNCH("gated_scan");
  return SNNB_OK;
}

extern "C" int snnb_gated_scan_backward(const void *dh, int64_t dh_t_stride, int64_t dh_b_stride, const void *dh_last,
                                        const void *x, int64_t x_t_stride, int64_t x_b_stride,
                                        const void *gate, int64_t g_t_stride, int64_t g_b_stride,
                                        const void *h_init, const float *ckpt, const int *lengths,
                                        void *dx, int64_t dx_t_stride, int64_t dx_b_stride,
                                        void *dgate, int64_t dg_t_stride, int64_t dg_b_stride, void *dh_init,
                                        int64_t T, int64_t B, int64_t D, int gate_kind, int leaky, int dtype,
                                        int state_dtype, void *stream) {
  using namespace snnb;
  ScanArgs q = {};
  q.x = {x, x_t_stride, x_b_stride};
  q.g = {gate, g_t_stride, g_b_stride};
  q.h = {dh, dh_t_stride, dh_b_stride};
  q.dx = {dx, dx_t_stride, dx_b_stride};
  q.dg = {dgate, dg_t_stride, dg_b_stride};
  q.h_init = h_init; q.dh_last = dh_last; q.h_last = dh_init; q.ckpt = const_cast<float *>(ckpt); q.lengths = lengths;
  q.T = T; q.B = B; q.D = D; q.state_f32 = state_dtype == SNNB_F32;
  if (const int st = check_common(q, gate_kind, dtype, state_dtype, "gated_scan_backward")) return st;
  SNNB_CHECK_ARG(T * B * D == 0 || (dx && dgate), "gated_scan_backward: null pointer");
  SNNB_CHECK_ARG(T * B * D == 0 || T <= kCkptSteps || ckpt,
                 "gated_scan_backward: more than %d steps need the checkpoints of the forward pass", kCkptSteps);
  SNNB_CHECK_ARG(rows_apart(dx_t_stride, dx_b_stride, T, B, D) && rows_apart(dg_t_stride, dg_b_stride, T, B, D),
                 "gated_scan_backward: rows of dx or dgate overlap");
  SNNB_CHECK_ARG(!partly_same(dh_last, dh_init, B * D * dtype_size(state_dtype)),
                 "gated_scan_backward: dh_last and dh_init overlap without being the same buffer");
  if (B * D == 0) return SNNB_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SNNB_F32: launch<float, true>(q, gate_kind, leaky, s); break;
    case SNNB_BF16: launch<__nv_bfloat16, true>(q, gate_kind, leaky, s); break;
    default: launch<__half, true>(q, gate_kind, leaky, s); break;
  }
  SNNB_CHECK_LAUNCH("gated_scan_backward");
  return SNNB_OK;
}
