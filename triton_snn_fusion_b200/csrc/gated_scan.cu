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
//
// The kernels are in gated_scan_impl.cuh; this file checks the arguments.
#include "gated_scan.cuh"

namespace snnb {
namespace {

constexpr int kCkptSteps = SNNB_GATED_SCAN_CKPT_STEPS;

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

bool some(int64_t T, int64_t B, int64_t D) { return T > 0 && B > 0 && D > 0; }

int check_common(const ScanArgs &q, int gate_kind, int dtype, int state_dtype, const char *what) {
  SNNB_CHECK_ARG(q.T >= 0 && q.B >= 0 && q.D >= 0, "%s: sizes must not be negative", what);
  SNNB_CHECK_ARG(q.T <= (1LL << 30) && q.B <= 0x7fffffffLL && q.D <= 0x7fffffffLL && q.B * q.D <= (1LL << 36),
                 "%s: problem too large", what);
  SNNB_CHECK_ARG(gate_kind == SNNB_GATE_VALUE || gate_kind == SNNB_GATE_SIGMOID, "%s: bad gate kind %d", what, gate_kind);
  SNNB_CHECK_ARG(is_act_dtype(dtype), "%s: unsupported dtype %d", what, dtype);
  SNNB_CHECK_ARG(state_dtype == dtype || state_dtype == SNNB_F32, "%s: state dtype must be the x dtype or f32", what);
  SNNB_CHECK_ARG(q.x.ts >= 0 && q.x.bs >= 0 && q.g.ts >= 0 && q.g.bs >= 0 && q.h.ts >= 0 && q.h.bs >= 0,
                 "%s: negative stride", what);
  if (some(q.T, q.B, q.D)) SNNB_CHECK_ARG(q.x.p && q.g.p && q.h.p, "%s: null pointer", what);
  return SNNB_OK;
}

bool rows16(const ScanSeq &s, int size) {
  const int n = 16 / size;
  return s.p == nullptr || (aligned16(s.p) && s.ts % n == 0 && s.bs % n == 0 && s.ts < (1 << 22));      // 128 rows lie within 2^32 bytes
}

int dispatch(ScanArgs q, bool backward, int gate_kind, int dtype, cudaStream_t s) {
  // Time outermost and the batch dense inside it: one row of B * D channels.
  if (q.T <= 1) q.x.ts = q.g.ts = q.h.ts = q.dx.ts = q.dg.ts = 0;      // one step has no use for its time stride
  auto dense = [&](const ScanSeq &t) { return t.p == nullptr || t.bs == q.D; };
  if (!q.lengths && q.B > 1 && dense(q.x) && dense(q.g) && dense(q.h) && dense(q.dx) && dense(q.dg)) {
    q.D *= q.B;
    q.B = 1;
  }
  if (q.B == 1) q.x.bs = q.g.bs = q.h.bs = q.dx.bs = q.dg.bs = 0;
  const int sz = dtype_size(dtype);
  const bool aligned = q.D % (16 / sz) == 0 && aligned16(q.h_init) && aligned16(q.dh_last) && aligned16(q.h_last) &&
                       rows16(q.x, sz) && rows16(q.g, sz) && rows16(q.h, sz) && rows16(q.dx, sz) && rows16(q.dg, sz);
  for (const ScanSeq *t : {&q.x, &q.g, &q.h, &q.dx, &q.dg})
    if (t->ts >= (1LL << 29))
      return fail(SNNB_ERR_UNSUPPORTED, "gated_scan: time strides of 2^29 values or more are not implemented");
  switch (dtype) {
    case SNNB_F32: return gated_scan_launch<float>(q, backward, gate_kind, aligned, s);
    case SNNB_BF16: return gated_scan_launch<__nv_bfloat16>(q, backward, gate_kind, aligned, s);
    default: return gated_scan_launch<__half>(q, backward, gate_kind, aligned, s);
  }
}

}  // namespace
}  // namespace snnb

int snnb::gated_scan_device_status(int *out) {
  int a = 0, b = 0, c = 0;
  if (const int rc = gated_scan_status_f32(&a)) return rc;
  if (const int rc = gated_scan_status_bf16(&b)) return rc;
  if (const int rc = gated_scan_status_f16(&c)) return rc;
  *out = a | b | c;
  return SNNB_OK;
}

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
  q.T = T; q.B = B; q.D = D; q.state_f32 = state_dtype == SNNB_F32; q.leaky = leaky != 0;
  if (const int st = check_common(q, gate_kind, dtype, state_dtype, "gated_scan")) return st;
  SNNB_CHECK_ARG(!h_seq || (h_seq != x && h_seq != gate), "gated_scan: h_seq is one of the inputs");
  SNNB_CHECK_ARG(rows_apart(h_t_stride, h_b_stride, T, B, D), "gated_scan: rows of h_seq overlap");
  SNNB_CHECK_ARG(!partly_same(h_init, h_last, B * D * dtype_size(state_dtype)),
                 "gated_scan: h_init and h_last overlap without being the same buffer");
  if (B * D == 0) return SNNB_OK;
  return dispatch(q, false, gate_kind, dtype, static_cast<cudaStream_t>(stream));
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
  q.T = T; q.B = B; q.D = D; q.state_f32 = state_dtype == SNNB_F32; q.leaky = leaky != 0;
  if (const int st = check_common(q, gate_kind, dtype, state_dtype, "gated_scan_backward")) return st;
  SNNB_CHECK_ARG(!some(T, B, D) || (dx && dgate), "gated_scan_backward: null pointer");
  for (const void *out : {(const void *)dx, (const void *)dgate})
    SNNB_CHECK_ARG(!out || (out != dh && out != x && out != gate), "gated_scan_backward: an output is one of the inputs");
  SNNB_CHECK_ARG(!dx || dx != dgate, "gated_scan_backward: dx and dgate are one buffer");
  SNNB_CHECK_ARG(!some(T, B, D) || T <= kCkptSteps || ckpt,
                 "gated_scan_backward: more than %d steps need the checkpoints of the forward pass", kCkptSteps);
  SNNB_CHECK_ARG(rows_apart(dx_t_stride, dx_b_stride, T, B, D) && rows_apart(dg_t_stride, dg_b_stride, T, B, D),
                 "gated_scan_backward: rows of dx or dgate overlap");
  SNNB_CHECK_ARG(!partly_same(dh_last, dh_init, B * D * dtype_size(state_dtype)),
                 "gated_scan_backward: dh_last and dh_init overlap without being the same buffer");
  if (B * D == 0) return SNNB_OK;
  return dispatch(q, true, gate_kind, dtype, static_cast<cudaStream_t>(stream));
}
