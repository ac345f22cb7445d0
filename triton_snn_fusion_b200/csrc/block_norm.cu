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
//
// What bounds it, on B200: forward 5 values an element (read y, gate, res; write res', z), backward 8. A block takes whole
// rows, 8 (16-bit) or 4 columns a thread, one after the other; the next rows are copied into shared memory meanwhile. 16384
// rows of 2048 bf16 values, device time in us: forward 55 = 6.1 TB/s (93 % of the measured copy rate; a call alone with cold
// caches 60, three rows in shared memory instead of two 68, the next row in registers 90), backward 104 with its sums = 5.1
// TB/s (78 %; alone 113); 1024 fp32 columns 57 and 104. The backward pass: 60 instructions an element, a third of them the
// four sums over a row, at two blocks an SM for its 123 registers (three blocks of 80 with spills 160, rows in registers
// instead of shared memory 181). Gradients of the parameters leave as one row per block and are joined in a fixed order by a
// second kernel, which costs 4 us; nothing is summed by atomics.
#include "packed.cuh"
#include "umma.cuh"

namespace snnb {
namespace {

struct NormArgs {
  const void *y, *gate, *res, *w_post, *scale, *w_pre, *dres_out, *dz;
  int64_t ys, gs, rs, dos, dzs;      // row strides
  void *res_out, *z;                 // forward outputs
  void *dy, *dgate, *dres;           // backward outputs
  float *partial;                    // [blocks][2][D]: column sums Q and dw_pre
  float *dw_post, *dscale, *dw_pre;
  int64_t M;
  int D, w_f32, act, post_norm;
  int tpr;                           // threads of a row: a power of two
  int w_vec;                         // parameters may be read 16 bytes at a time
  float alpha, eps;
};

template <typename T> __device__ __forceinline__ float param(const void *p, int f32, int i) {
  if (p == nullptr) return 1.f;
  return f32 ? static_cast<const float *>(p)[i] : DT<T>::to_f(static_cast<const T *>(p)[i]);
}

// act(g) and its derivative, element by element; the kind is the same for the whole launch.
template <int N, bool ALL = false> __device__ __forceinline__ void act_of(int act, const float (&g)[N], float (&v)[N], float (&dv)[N]) {
  float p[N], m[N];
  if (!ALL && act == SNNB_ACT_NONE) {
    v_set(v, 1.f);
    v_set(dv, 0.f);
    return;
  }
  v_sigmoid(g, p, m);
  if (act == SNNB_ACT_SIGMOID) {
    v_mul(p, m, dv);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = p[k];
  } else {      // g p, with the derivative p (1 + g (1 - p))
    float one[N];
    v_set(one, 1.f);
    v_mul(g, p, v);
    v_fma(g, m, one, dv);
    v_mul(p, dv, dv);
  }
}

// Sums over the threads of a row: a part of a warp (TPR 0: tpr <= 32 threads), or all TPR / 32 warps of the block. sh: 2 x 32
// floats; two calls in a row take different ones.
template <int TPR, int N> __device__ __forceinline__ void row_sums(float (&v)[N], int tpr, float (*sh)[32]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (TPR > 0 || o < tpr)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (TPR > 0) {
    constexpr int WARPS = TPR / 32, W = WARPS < 4 ? WARPS : 4;
    if (threadIdx.x % 32 == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) sh[i][threadIdx.x / 32] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t[W];
      v_set(t, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; w += W) {
        float f[W];
        sh_load<W>(&sh[i][w], f);
#pragma unroll
        for (int k = 0; k < W; ++k) t[k] += f[k];
      }
      v[i] = W == 4 ? (t[0] + t[1]) + (t[W - 2] + t[W - 1]) : t[0] + t[W - 1];
    }
  }
}

// A thread's columns of a row: NV pieces of VEC neighbouring ones, tpr * VEC columns apart; zeros where there is nothing.
template <typename T, int VEC, int NV> struct Piece {
  Pack<T, VEC> p[NV];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int v = 0; v < NV; ++v) p[v] = Pack<T, VEC>{};
  }
  // the thread's columns of a row, which then steps on by inc; in: those that exist
  template <bool ALL> __device__ __forceinline__ void load(const T *&row, int64_t inc, int step, const bool (&in)[NV]) {
    if (!ALL && row == nullptr) return;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (!in[v]) continue;
      if constexpr (sizeof(T) * VEC == 16) *reinterpret_cast<int4 *>(&p[v]) = __ldcs(reinterpret_cast<const int4 *>(row + v * step));
      else p[v].v[0] = __ldcs(row + v * step);
    }
    row += inc;
  }
  __device__ __forceinline__ void get(int v, float (&f)[VEC]) const { widen<T, VEC>(p[v].v, f); }
};
// The same in shared memory, for the rows that are worked on and on their way: one slot of a thread's own per stage.
template <typename T, int VEC, int NV, int THREADS> struct StagedPiece {
  Pack<T, VEC> *p;      // [NV][THREADS], from the thread's first
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int v = 0; v < NV; ++v) p[v * THREADS] = Pack<T, VEC>{};
  }
  template <bool ALL> __device__ __forceinline__ void load(const T *&row, int64_t inc, int step, const bool (&in)[NV]) {
    if (!ALL && row == nullptr) return;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (in[v]) copy_async16(p + v * THREADS, row + v * step);
    row += inc;
  }
  __device__ __forceinline__ void get(int v, float (&f)[VEC]) const { widen<T, VEC>(p[v * THREADS].v, f); }
};
template <typename T, int VEC> __device__ __forceinline__ void put(T *p, const float (&f)[VEC]) { store_pack<T, VEC, false>(p, f); }
template <typename T> __device__ __forceinline__ const T *row_of(const void *p, int64_t off) {
  return p == nullptr ? nullptr : static_cast<const T *>(p) + off;
}
// The sum of a thread's partial sums, added up in lanes of their own until the end of a row.
template <int N> __device__ __forceinline__ float sum_of(const float (&f)[N]) {
  float t[N];
#pragma unroll
  for (int k = 0; k < N; ++k) t[k] = f[k];
#pragma unroll
  for (int n = N / 2; n > 0; n /= 2)
#pragma unroll
    for (int k = 0; k < n; ++k) t[k] += t[k + n];
  return t[0];
}

// VEC parameters from column i on (i + VEC <= D); ones where there are none.
template <typename T, int VEC> __device__ __forceinline__ void params_at(const NormArgs &q, const void *p, int i, float (&v)[VEC]) {
  if (VEC == 1 || !q.w_vec || p == nullptr) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = param<T>(p, q.w_f32, i + k);
  } else if (q.w_f32) {
    load_pack<float, VEC>(static_cast<const float *>(p) + i, v);
  } else {
    load_pack<T, VEC>(static_cast<const T *>(p) + i, v);
  }
}
// alpha * res_scale * w_post, and w_pre, of a thread's columns; zeros behind the last one
template <typename T, int VEC, int NV>
__device__ __forceinline__ void params_of(const NormArgs &q, int col, int step, float (&c)[NV][VEC], float (&wp)[NV][VEC]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int i = col + v * step;
    v_set(c[v], 0.f);
    v_set(wp[v], 0.f);
    if (i >= q.D) continue;
    params_at<T, VEC>(q, q.w_pre, i, wp[v]);
    if (!q.y) continue;
    float a[VEC], b[VEC], al[VEC];
    params_at<T, VEC>(q, q.scale, i, a);
    params_at<T, VEC>(q, q.w_post, i, b);
    v_set(al, q.alpha);
    v_mul(a, al, a);
    v_mul(a, b, c[v]);
  }
}

// One row after the other, the next row's values on their way while one is worked on. The parameters of a thread's
// columns stay in registers.
// ST: rows in shared memory, all but one of them on their way; 0: one row ahead in registers.
template <typename T, int VEC, int NV, int TPR, int ST>
__global__ void __launch_bounds__(TPR > 0 ? TPR : 128) block_norm_kernel(const __grid_constant__ NormArgs q) {
  __shared__ __align__(16) float sh[2][2][32];
  const int tpr = TPR > 0 ? TPR : q.tpr, groups = TPR > 0 ? 1 : blockDim.x / tpr, tid = threadIdx.x % tpr, step = tpr * VEC;
  const int col = tid * VEC;
  const int64_t stride = (int64_t)gridDim.x * groups;
  float c[NV][VEC], wp[NV][VEC];
  params_of<T, VEC, NV>(q, col, step, c, wp);
  bool in[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) in[v] = col + v * step < q.D;
  int64_t m = (int64_t)blockIdx.x * groups + threadIdx.x / tpr;
  const T *yp = row_of<T>(q.y, m * q.ys + col), *gp = row_of<T>(q.gate, m * q.gs + col), *rp = row_of<T>(q.res, m * q.rs + col);
  int64_t at = m * q.D + col;
  constexpr int THREADS = TPR > 0 ? TPR : 128, SLOT = NV * THREADS;
  using P = std::conditional_t<(ST > 0), StagedPiece<T, VEC, NV, THREADS>, Piece<T, VEC, NV>>;
  extern __shared__ __align__(16) unsigned char dyn[];
  Pack<T, VEC> *const slots = reinterpret_cast<Pack<T, VEC> *>(dyn) + threadIdx.x;      // [ST][3][NV][THREADS]
  P y, g, r;
  auto to_stage = [&](int st) {
    if constexpr (ST > 0) { y.p = slots + st * 3 * SLOT; g.p = y.p + SLOT; r.p = g.p + SLOT; }
  };
  auto fetch = [&]() {
    y.template load<false>(yp, stride * q.ys, step, in);
    g.template load<false>(gp, stride * q.gs, step, in);
    r.template load<false>(rp, stride * q.rs, step, in);
  };
#pragma unroll
  for (int st = 0; st < (ST > 0 ? ST : 1); ++st) {
    to_stage(st);
    y.clear(); g.clear(); r.clear();
  }
#pragma unroll
  for (int st = 0; st < (ST > 0 ? ST - 1 : 1); ++st) {
    to_stage(st);
    if (m + st * stride < q.M) fetch();
    if (ST > 0) copy_commit();
  }
  int st = 0;
  const float inv_d = 1.f / (float)q.D;
  // every group of a block goes round as often as the first, whose row comes first
  for (int64_t first = (int64_t)blockIdx.x * groups; first < q.M; first += stride, m += stride, at += stride * q.D) {
    const bool live = TPR > 0 || m < q.M;
    if constexpr (ST > 0) {
      to_stage(st == 0 ? ST - 1 : st - 1);
      if (m + (ST - 1) * stride < q.M) fetch();
      copy_commit();
      copy_wait<ST - 1>();
      to_stage(st);
      st = st == ST - 1 ? 0 : st + 1;
    }
    float out[NV][VEC], s[1], acc[VEC], f[VEC], gv[VEC], a[VEC], da[VEC], ry[VEC];
    v_set(ry, 1.f);
    if (q.post_norm) {
      v_set(acc, 0.f);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        y.get(v, f);
        v_fma(f, f, acc, acc);
      }
      s[0] = sum_of(acc);
      row_sums<TPR>(s, tpr, sh[0]);
      v_set(ry, rsqrtf(s[0] * inv_d + q.eps));
    } else if (TPR > 0) {
      __syncthreads();      // the sums of the row before have been read
    }
    v_set(acc, 0.f);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      r.get(v, out[v]);
      if (q.y) {
        y.get(v, f);
        g.get(v, gv);
        act_of<VEC, false>(q.act, gv, a, da);
        v_mul(f, ry, f);
        v_mul(c[v], a, a);
        v_fma(a, f, out[v], out[v]);
      }
      v_fma(out[v], out[v], acc, acc);
    }
    if (ST == 0 && m + stride < q.M) fetch();
    if (q.res_out && live) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (in[v]) put<T, VEC>(static_cast<T *>(q.res_out) + at + v * step, out[v]);
    }
    if (!q.z) {
      if (TPR > 0) __syncthreads();
      continue;
    }
    s[0] = sum_of(acc);
    row_sums<TPR>(s, tpr, sh[1]);
    float ro[VEC];
    v_set(ro, rsqrtf(s[0] * inv_d + q.eps));
    if (!live) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      v_mul(out[v], ro, out[v]);
      v_mul(out[v], wp[v], out[v]);
      if (in[v]) put<T, VEC>(static_cast<T *>(q.z) + at + v * step, out[v]);
    }
  }
}

// The same for the gradients. The column sums and parameters of a thread's columns stay in registers over all rows of the
// block, or, with two pieces a thread, in shared memory (each value is only touched by its thread).
// ALL: every operand is there (y with its norm, gate, res, both gradients), so nothing is asked: 116 us instead of 128 for
// 16384 rows of 2048 bf16 values. (The forward pass gains nothing from it.)
template <typename T, int VEC, int NV, int ST, bool ACC_SH, int TPR, int MINB, bool ALL>
__global__ void __launch_bounds__(TPR > 0 ? TPR : 128, MINB) block_norm_backward_kernel(const __grid_constant__ NormArgs q) {
  __shared__ __align__(16) float sh[3][2][32];
  umma::pdl_trigger();      // the sums' kernel may take its place; it waits for this one to end
  constexpr int THREADS = TPR > 0 ? TPR : 128, SLOT = NV * THREADS;
  extern __shared__ __align__(16) unsigned char dyn[];
  Pack<T, VEC> *const slots = reinterpret_cast<Pack<T, VEC> *>(dyn) + threadIdx.x;      // [ST][5][NV][THREADS]
  float *const acc_sh = reinterpret_cast<float *>(dyn + ST * 5 * SLOT * sizeof(Pack<T, VEC>));      // [4][D] with ACC_SH: the sums and the parameters; [groups][2][D] to join the rows of a block with tpr <= 32
  const int tpr = TPR > 0 ? TPR : q.tpr, groups = TPR > 0 ? 1 : blockDim.x / tpr, tid = threadIdx.x % tpr, step = tpr * VEC;
  const int col = tid * VEC;
  const int64_t stride = (int64_t)gridDim.x * groups;
  bool in[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) in[v] = col + v * step < q.D;
  constexpr int NR = ACC_SH ? 1 : NV;
  float cr[NR][VEC], wr[NR][VEC], aq[NR][VEC], aw[NR][VEC];
  if constexpr (ACC_SH) {
    float c2[NV][VEC], w2[NV][VEC], zero[VEC];
    params_of<T, VEC, NV>(q, col, step, c2, w2);
    v_set(zero, 0.f);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = col + v * step;
      if (i >= q.D) continue;
      sh_store<VEC>(acc_sh + i, zero);
      sh_store<VEC>(acc_sh + q.D + i, zero);
      sh_store<VEC>(acc_sh + 2 * q.D + i, c2[v]);
      sh_store<VEC>(acc_sh + 3 * q.D + i, w2[v]);
    }
  } else {
    params_of<T, VEC, NV>(q, col, step, cr, wr);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      v_set(aq[v], 0.f);
      v_set(aw[v], 0.f);
    }
  }
  auto param_at = [&](int which, int v, float (&t)[VEC]) {      // 0: alpha res_scale w_post, 1: w_pre
    if constexpr (ACC_SH) {
      if (col + v * step < q.D) sh_load<VEC>(acc_sh + (2 + which) * q.D + col + v * step, t);
      else v_set(t, 0.f);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) t[k] = which ? wr[v][k] : cr[v][k];
    }
  };
  // adds to a column sum
  auto add = [&](float *sum, int v, const float (&x)[VEC], const float (&w)[VEC]) {
    if (col + v * step >= q.D) return;
    float t[VEC];
    sh_load<VEC>(sum + col + v * step, t);
    v_fma(x, w, t, t);
    sh_store<VEC>(sum + col + v * step, t);
  };
  int64_t m = (int64_t)blockIdx.x * groups + threadIdx.x / tpr;
  const T *yp = row_of<T>(q.y, m * q.ys + col), *gp = row_of<T>(q.gate, m * q.gs + col), *rp = row_of<T>(q.res, m * q.rs + col);
  const T *op = row_of<T>(q.dres_out, m * q.dos + col), *zp = row_of<T>(q.dz, m * q.dzs + col);
  int64_t at = m * q.D + col;
  using P = std::conditional_t<(ST > 0), StagedPiece<T, VEC, NV, THREADS>, Piece<T, VEC, NV>>;
  P y, g, r, o, z;
  auto to_stage = [&](int st) {
    if constexpr (ST > 0) { y.p = slots + st * 5 * SLOT; g.p = y.p + SLOT; r.p = g.p + SLOT; o.p = r.p + SLOT; z.p = o.p + SLOT; }
  };
  auto fetch = [&](int64_t row) {
    if (row >= q.M) return;
    y.template load<ALL>(yp, stride * q.ys, step, in);
    g.template load<ALL>(gp, stride * q.gs, step, in);
    r.template load<ALL>(rp, stride * q.rs, step, in);
    o.template load<ALL>(op, stride * q.dos, step, in);
    z.template load<ALL>(zp, stride * q.dzs, step, in);
  };
#pragma unroll
  for (int st = 0; st < (ST > 0 ? ST : 1); ++st) {
    to_stage(st);
    y.clear(); g.clear(); r.clear(); o.clear(); z.clear();
  }
#pragma unroll
  for (int st = 0; st < ST - 1; ++st) {
    to_stage(st);
    fetch(m + st * stride);
    copy_commit();
  }
  int st = 0;
  const float inv_d = 1.f / (float)q.D;
  for (int64_t first = (int64_t)blockIdx.x * groups; first < q.M; first += stride, m += stride, at += stride * q.D) {
    // A group that has no row left works on whatever is in its place, and neither stores nor adds any of it: even a row of
    // zeros would add 0 * rstd(0) to the column sums, which is not a number where eps is zero.
    const bool live = TPR > 0 || m < q.M;
    if constexpr (ST > 0) {
      to_stage(st == 0 ? ST - 1 : st - 1);
      fetch(m + (ST - 1) * stride);
      copy_commit();
      copy_wait<ST - 1>();
      to_stage(st);
      st = st == ST - 1 ? 0 : st + 1;
    } else {
      fetch(m);
    }
    float G[NV][VEC], a[NV][VEC], da[ACC_SH ? 1 : NV][VEC], f[VEC], t[VEC], p[VEC], acc[VEC], acc2[VEC], s[2], ry1 = 1.f, ry[VEC];
    if (ALL || q.post_norm) {
      float s1[1];
      v_set(acc, 0.f);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        y.get(v, f);
        v_fma(f, f, acc, acc);
      }
      s1[0] = sum_of(acc);
      row_sums<TPR>(s1, tpr, sh[0]);
      ry1 = rsqrtf(s1[0] * inv_d + q.eps);
    }
    v_set(ry, ry1);
    // out, kept in G until it is the gradient
    v_set(acc, 0.f);
    v_set(acc2, 0.f);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      r.get(v, G[v]);
      if (ALL || q.y) {
        y.get(v, f);
        g.get(v, t);
        act_of<VEC, ALL>(q.act, t, a[v], da[ACC_SH ? 0 : v]);
        v_mul(f, ry, f);
        param_at(0, v, p);
        v_mul(p, a[v], t);
        v_fma(t, f, G[v], G[v]);
      }
      if (ALL || q.dz) {
        z.get(v, f);
        param_at(1, v, p);
        v_mul(f, p, f);
        v_fma(G[v], G[v], acc, acc);
        v_fma(G[v], f, acc2, acc2);
      }
    }
    float ro[VEC], mo[VEC];
    v_set(ro, 0.f);
    v_set(mo, 0.f);
    if (ALL || q.dz) {
      s[0] = sum_of(acc);
      s[1] = sum_of(acc2);
      row_sums<TPR>(s, tpr, sh[1]);
      const float r1 = rsqrtf(s[0] * inv_d + q.eps);
      v_set(ro, r1);
      v_set(mo, -s[1] * inv_d * r1 * r1 * r1);
    }
    v_set(acc, 0.f);
    float al[VEC];
    v_set(al, q.alpha * ry1);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (ALL || q.dz) {
        z.get(v, f);
        v_mul(f, ro, f);
        if constexpr (ACC_SH) add(acc_sh + q.D, v, f, G[v]);
        else if (live) v_fma(f, G[v], aw[v], aw[v]);
        o.get(v, t);
        v_fma(mo, G[v], t, G[v]);
        param_at(1, v, p);
        v_fma(f, p, G[v], G[v]);
      } else {
        o.get(v, G[v]);
      }
      if ((ALL || q.dres) && live && in[v]) put<T, VEC>(static_cast<T *>(q.dres) + at + v * step, G[v]);
      if (ALL || q.y) {
        y.get(v, f);
        v_mul(f, a[v], t);
        v_mul(G[v], t, t);
        param_at(0, v, p);
        v_fma(t, p, acc, acc);
        if constexpr (ACC_SH) add(acc_sh, v, t, al);
        else if (live) v_fma(t, al, aq[v], aq[v]);
      }
    }
    float me[VEC];
    v_set(me, 0.f);
    if (ALL || q.post_norm) {
      float s1[1] = {sum_of(acc)};
      row_sums<TPR>(s1, tpr, sh[2]);
      v_set(me, -s1[0] * inv_d * ry1 * ry1 * ry1);
    } else if (TPR > 0) {
      __syncthreads();      // the sums have been read
    }
    if (ALL || q.y) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        y.get(v, f);
        param_at(0, v, p);
        v_mul(G[v], p, G[v]);
        v_mul(G[v], ry, G[v]);
        v_mul(f, me, t);
        v_fma(G[v], a[v], t, t);
        if (live && in[v]) put<T, VEC>(static_cast<T *>(q.dy) + at + v * step, t);
        if (ALL || q.dgate) {
          if constexpr (ACC_SH) {      // again, rather than kept: the registers are full
            g.get(v, t);
            act_of<VEC, ALL>(q.act, t, p, da[0]);
          }
          v_mul(G[v], f, t);
          v_mul(t, da[ACC_SH ? 0 : v], t);
          if (live && in[v]) put<T, VEC>(static_cast<T *>(q.dgate) + at + v * step, t);
        }
      }
    }
  }
  // one row of partial sums per block
  float *pq = q.partial + (int64_t)blockIdx.x * 2 * q.D;
  if constexpr (ACC_SH) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * q.D; i += blockDim.x) pq[i] = acc_sh[i];
  } else {
    float *mine = groups > 1 ? acc_sh + (threadIdx.x / tpr) * 2 * q.D : pq;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const int i = col + v * step + k;
        if (i < q.D) {
          mine[i] = aq[v][k];
          mine[q.D + i] = aw[v][k];
        }
      }
    if (groups > 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * q.D; i += blockDim.x) {
        float t = 0.f;
        for (int gr = 0; gr < groups; ++gr) t += acc_sh[gr * 2 * q.D + i];
        pq[i] = t;
      }
    }
  }
}

// Rows too long for the registers of a block: every pass reads the row again, from L1 or L2.
constexpr int kLongThreads = 1024;

template <typename T, int VEC> struct LongRow {
  const NormArgs &q;
  const T *y, *gate, *res;
  __device__ __forceinline__ LongRow(const NormArgs &a, int64_t m)
      : q(a), y(row_of<T>(a.y, m * a.ys)), gate(row_of<T>(a.gate, m * a.gs)), res(row_of<T>(a.res, m * a.rs)) {}
  static __device__ __forceinline__ void at(const T *row, int i, float (&v)[VEC]) {
    if (row == nullptr) { v_set(v, 0.f); return; }
    widen<T, VEC>(reinterpret_cast<const Pack<T, VEC> *>(row + i)->v, v);
  }
  // what res_out is at VEC columns, and what of it the gradients need: y, act, act' and the coefficient
  struct Out { float out[VEC], y[VEC], a[VEC], da[VEC], c[VEC]; };
  __device__ __forceinline__ void out(int i, float rstd_y, Out &o) const {
    at(res, i, o.out);
    if (!q.y) return;
    float g[VEC], t[VEC], f[VEC];
    at(y, i, o.y);
    at(gate, i, g);
    act_of(q.act, g, o.a, o.da);
    params_at<T, VEC>(q, q.scale, i, o.c);
    params_at<T, VEC>(q, q.w_post, i, t);
    v_mul(o.c, t, o.c);
    v_set(t, q.alpha);
    v_mul(o.c, t, o.c);
    v_set(t, rstd_y);
    v_mul(o.y, t, t);
    v_mul(o.c, o.a, f);
    v_fma(f, t, o.out, o.out);
  }
  __device__ __forceinline__ float rstd_y(float (*sh)[32]) const {
    if (!q.post_norm) return 1.f;
    float s[1] = {0.f}, acc[VEC], f[VEC];
    v_set(acc, 0.f);
    for (int i = threadIdx.x * VEC; i < q.D; i += kLongThreads * VEC) {
      at(y, i, f);
      v_fma(f, f, acc, acc);
    }
    s[0] = sum_of(acc);
    row_sums<kLongThreads>(s, 0, sh);
    return rsqrtf(s[0] / q.D + q.eps);
  }
};

template <typename T, int VEC>
__global__ void __launch_bounds__(kLongThreads) block_norm_long_kernel(const __grid_constant__ NormArgs q) {
  __shared__ __align__(16) float sh[2][2][32];
  for (int64_t m = blockIdx.x; m < q.M; m += gridDim.x) {
    const LongRow<T, VEC> row(q, m);
    const float ry = row.rstd_y(sh[0]);
    float s[1] = {0.f}, acc[VEC], w[VEC], ro[VEC];
    typename LongRow<T, VEC>::Out o;
    if (q.z) {
      v_set(acc, 0.f);
      for (int i = threadIdx.x * VEC; i < q.D; i += kLongThreads * VEC) {
        row.out(i, ry, o);
        v_fma(o.out, o.out, acc, acc);
      }
      s[0] = sum_of(acc);
      row_sums<kLongThreads>(s, 0, sh[1]);
      s[0] = rsqrtf(s[0] / q.D + q.eps);
    }
    v_set(ro, s[0]);
    for (int i = threadIdx.x * VEC; i < q.D; i += kLongThreads * VEC) {
      row.out(i, ry, o);      // before res_out, which may be res
      if (q.res_out) put<T, VEC>(static_cast<T *>(q.res_out) + m * q.D + i, o.out);
      if (q.z) {
        params_at<T, VEC>(q, q.w_pre, i, w);
        v_mul(o.out, ro, o.out);
        v_mul(o.out, w, o.out);
        put<T, VEC>(static_cast<T *>(q.z) + m * q.D + i, o.out);
      }
    }
    __syncthreads();      // the sums have been read
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kLongThreads) block_norm_backward_long_kernel(const __grid_constant__ NormArgs q) {
  using Row = LongRow<T, VEC>;
  __shared__ __align__(16) float sh[3][2][32];
  umma::pdl_trigger();
  float *pq = q.partial + (int64_t)blockIdx.x * 2 * q.D, *pw = pq + q.D;
  for (int i = threadIdx.x; i < 2 * q.D; i += kLongThreads) pq[i] = 0.f;
  __syncthreads();
  for (int64_t m = blockIdx.x; m < q.M; m += gridDim.x) {
    const Row row(q, m);
    const T *dz = row_of<T>(q.dz, m * q.dzs), *dro = row_of<T>(q.dres_out, m * q.dos);
    const float ry = row.rstd_y(sh[0]);
    float s[2] = {0.f, 0.f}, ro = 0.f, mo = 0.f, acc[VEC], acc2[VEC], w[VEC], d[VEC], t[VEC], G[VEC];
    typename Row::Out o;
    if (q.dz) {
      v_set(acc, 0.f);
      v_set(acc2, 0.f);
      for (int i = threadIdx.x * VEC; i < q.D; i += kLongThreads * VEC) {
        row.out(i, ry, o);
        Row::at(dz, i, d);
        params_at<T, VEC>(q, q.w_pre, i, w);
        v_mul(d, w, d);
        v_fma(o.out, o.out, acc, acc);
        v_fma(o.out, d, acc2, acc2);
      }
      s[0] = sum_of(acc);
      s[1] = sum_of(acc2);
      row_sums<kLongThreads>(s, 0, sh[1]);
      ro = rsqrtf(s[0] / q.D + q.eps);
      mo = s[1] / q.D * ro * ro * ro;
    }
    float me = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      if (pass) {
        float se[1] = {sum_of(acc)};
        row_sums<kLongThreads>(se, 0, sh[2]);
        me = -se[0] / q.D * ry * ry * ry;
      }
      v_set(acc, 0.f);
      for (int i = threadIdx.x * VEC; i < q.D; i += kLongThreads * VEC) {
        Row::at(dro, i, G);
        row.out(i, ry, o);
        if (q.dz) {
          Row::at(dz, i, d);
          params_at<T, VEC>(q, q.w_pre, i, w);
          v_set(t, ro);
          v_mul(d, t, d);
          if (pass) {
            sh_load<VEC>(pw + i, t);
            v_fma(d, o.out, t, t);
            sh_store<VEC>(pw + i, t);
          }
          v_fma(d, w, G, G);
          v_set(t, -mo);
          v_fma(t, o.out, G, G);
        }
        if (q.y) {
          float e[VEC];
          v_mul(G, o.c, e);
          v_mul(e, o.a, t);
          if (!pass) {
            v_fma(t, o.y, acc, acc);
          } else {
            float r[VEC];
            v_set(r, ry);
            v_mul(t, r, t);
            v_set(w, q.post_norm ? me : 0.f);
            v_fma(o.y, w, t, t);
            put<T, VEC>(static_cast<T *>(q.dy) + m * q.D + i, t);
            v_mul(o.y, r, o.y);
            if (q.dgate) {
              v_mul(e, o.y, t);
              v_mul(t, o.da, t);
              put<T, VEC>(static_cast<T *>(q.dgate) + m * q.D + i, t);
            }
            v_set(w, q.alpha);
            v_mul(o.a, w, o.a);
            v_mul(o.a, o.y, o.a);
            sh_load<VEC>(pq + i, t);
            v_fma(G, o.a, t, t);
            sh_store<VEC>(pq + i, t);
          }
        }
        if (pass && q.dres) put<T, VEC>(static_cast<T *>(q.dres) + m * q.D + i, G);
      }
    }
    __syncthreads();      // the sums have been read
  }
}

// Joins the blocks' column sums in a fixed order: 32 columns of one of the two sums a block, each by 32 threads.
template <typename T>
__global__ void __launch_bounds__(1024) block_norm_sums_kernel(const __grid_constant__ NormArgs q, int blocks) {
  __shared__ float sh[32][33];
  const int x = threadIdx.x % 32, part = threadIdx.x / 32, i = blockIdx.x * 32 + x, which = blockIdx.y;
  umma::pdl_wait();
  float t = 0.f;
  if (i < q.D) {
#pragma unroll 4
    for (int b = part; b < blocks; b += 32) t += q.partial[((int64_t)b * 2 + which) * q.D + i];
  }
  sh[part][x] = t;
  __syncthreads();
  // the thread takes column `part` over, its lane one of the 32 parts
  t = sh[x][part];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const int c = blockIdx.x * 32 + part;
  if (x != 0 || c >= q.D) return;
  if (which == 0) {
    if (q.dw_post) q.dw_post[c] = t * param<T>(q.scale, q.w_f32, c);
    if (q.dscale) q.dscale[c] = t * param<T>(q.w_post, q.w_f32, c);
  } else if (q.dw_pre) {
    q.dw_pre[c] = t;
  }
}

// How the rows are laid over threads. One piece of 16 bytes a thread: with two and half the threads the forward pass took
// 70 us instead of 61 (16384 rows of 2048 bf16 values), and the backward pass has no registers for them. Two pieces only
// where 512 threads with one do not reach (up to 8192 16-bit or 4096 fp32 columns), single columns where rows do not start
// on 16-byte boundaries (4096 rows of 2047 bf16 values: forward 29 us = 2.9 TB/s, backward 79 us = 1.7), and the long-row
// kernel (1.1 TB/s backward at 16384 columns, rows being read five times) behind that.
// A plan: `vec` columns in `nv` pieces for each of tpr threads; nv = 0: the long-row kernel.
struct Plan { int vec, nv, tpr, threads; };
Plan plan_of(int D, int dtype, bool aligned) {
  Plan p;
  p.vec = aligned && D % (16 / dtype_size(dtype)) == 0 ? 16 / dtype_size(dtype) : 1;
  p.nv = p.vec > 1 ? 1 : 4;
  p.tpr = 8;
  while (p.tpr < 512 && p.tpr * p.vec * p.nv < D) p.tpr *= 2;
  if (p.tpr * p.vec * p.nv < D) p.nv *= 2;
  if (p.tpr * p.vec * p.nv < D) { p.nv = 0; p.tpr = kLongThreads; }
  p.threads = p.tpr <= 32 ? 128 : p.tpr;
  return p;
}

// Blocks of the backward pass, each of which leaves one row of column sums: the same for every type and alignment, so that
// the workspace depends on the sizes alone, and chosen for 16-bit rows on 16-byte boundaries. Device time in us for 1, 2, 3,
// 4, 6, 8 blocks an SM (the choice in brackets):
//   bf16    65536 x 128    45 32 [29] 28 34 33      fp32    32768 x 256   136 74 [59] 50 50 55
//           32768 x 512    171 92 75 61 [54] 54             16384 x 512   79 52 48 52 [57] 54
//           16384 x 1024   95 63 [56] 54 64 61              16384 x 1024  106 95 [106] 93 94 96
//           16384 x 2048   136 [104] 118 113 120 131        8192 x 2048   95 [99] 103 111 121 125
//           8192 x 4096    [125] 135 142 151 167 182        1023 x 1001   18.5 15.6 [17.5] 17.8 20.2 21.5
//           1024 x 16384   241 [252] 262 268 284 290
//   ragged bf16  65536 x 63  103 58 [44] 37 48 41   16384 x 333  185 99 71 58 [75] 60   8192 x 1001  109 65 [84] 68 73 74
//                4096 x 2047  75 [78] 82 83 89 95
int backward_blocks(int64_t M, int D) {
  const int most = 148 * (D <= 256 ? 3 : D <= 512 ? 6 : D <= 1024 ? 3 : D <= 2048 ? 2 : D <= 8192 ? 1 : 2);
  return (int)(M < most ? (M < 1 ? 1 : M) : most);
}

bool rows16(const void *p, int64_t stride, int size) {
  return p == nullptr || (aligned16(p) && stride % (16 / size) == 0);
}

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

// The kernel for a plan's threads of a row.
#define SNNB_NORM_BY_TPR(CALL)         \
  switch (p.tpr) {                     \
    case 64: CALL(64); break;          \
    case 128: CALL(128); break;        \
    case 256: CALL(256); break;        \
    case 512: CALL(512); break;        \
    default: CALL(0); break;           \
  }

template <auto Kern> void launch_kernel(const NormArgs &q, int blocks, int threads, int smem, cudaStream_t s) {
  raise_smem_limit_once<Kern>(227 * 1024 - 2048);      // a failure shows at the launch
  Kern<<<(unsigned)blocks, threads, smem, s>>>(q);
}

template <typename T> void launch_forward(NormArgs q, int dtype, cudaStream_t s) {
  const int sz = (int)sizeof(T);
  const bool aligned = rows16(q.y, q.ys, sz) && rows16(q.gate, q.gs, sz) && rows16(q.res, q.rs, sz) &&
                       rows16(q.res_out, q.D, sz) && rows16(q.z, q.D, sz);
  const Plan p = plan_of(q.D, dtype, aligned);
  const int smem = 2 * 3 * 16 * p.threads;
  q.tpr = p.tpr;
  q.w_vec = aligned16(q.w_post) && aligned16(q.scale) && aligned16(q.w_pre);
  const int64_t rows = (q.M + p.threads / p.tpr - 1) / (p.threads / p.tpr);
  const int most = 148 * (p.threads <= 512 ? 1024 / p.threads : 2);
  const int blocks = (int)(rows < most ? rows : most);
  constexpr int V = 16 / (int)sizeof(T);
#define SNNB_CALL_V(TPR) launch_kernel<block_norm_kernel<T, V, 1, TPR, 2>>(q, blocks, p.threads, smem, s)
#define SNNB_CALL_1(TPR) block_norm_kernel<T, 1, 4, TPR, 0><<<blocks, p.threads, 0, s>>>(q)
  if (p.nv == 0 && p.vec == V) block_norm_long_kernel<T, V><<<blocks, p.threads, 0, s>>>(q);
  else if (p.nv == 0) block_norm_long_kernel<T, 1><<<blocks, p.threads, 0, s>>>(q);
  else if (p.vec == V && p.nv == 1) { SNNB_NORM_BY_TPR(SNNB_CALL_V) }
  else if (p.vec == V) launch_kernel<block_norm_kernel<T, V, 2, 512, 2>>(q, blocks, p.threads, 2 * smem, s);
  else if (p.nv == 4) { SNNB_NORM_BY_TPR(SNNB_CALL_1) }
  else block_norm_kernel<T, 1, 8, 512, 0><<<blocks, p.threads, 0, s>>>(q);
#undef SNNB_CALL_V
#undef SNNB_CALL_1
}

template <typename T> void launch_backward(NormArgs q, int dtype, cudaStream_t s) {
  const int sz = (int)sizeof(T);
  const bool aligned = rows16(q.y, q.ys, sz) && rows16(q.gate, q.gs, sz) && rows16(q.res, q.rs, sz) && rows16(q.dy, q.D, sz) &&
                       rows16(q.dgate, q.D, sz) && rows16(q.dres, q.D, sz) && rows16(q.dres_out, q.dos, sz) && rows16(q.dz, q.dzs, sz);
  const Plan p = plan_of(q.D, dtype, aligned);
  q.tpr = p.tpr;
  q.w_vec = aligned16(q.w_post) && aligned16(q.scale) && aligned16(q.w_pre);
  const int blocks = backward_blocks(q.M, q.D), groups = p.threads / p.tpr;
  constexpr int V = 16 / (int)sizeof(T);
  const bool all = q.y && q.post_norm && q.gate && q.res && q.dres_out && q.dz && q.dres;
  const int join = groups > 1 ? groups * 2 * q.D * (int)sizeof(float) : 0;      // at most 4 rows of 256 columns: 8 KB
#define SNNB_CALL_V(TPR) \
  launch_kernel<block_norm_backward_kernel<T, V, 1, (TPR == 512 ? 2 : 3), false, TPR, (TPR == 256 ? 2 : 1), false>>(q, blocks, p.threads, (TPR == 512 ? 2 : 3) * 5 * 16 * p.threads + join, s)
#define SNNB_CALL_A(TPR) \
  launch_kernel<block_norm_backward_kernel<T, V, 1, (TPR == 512 ? 2 : 3), false, TPR, (TPR == 256 ? 2 : 1), true>>(q, blocks, p.threads, (TPR == 512 ? 2 : 3) * 5 * 16 * p.threads + join, s)
#define SNNB_CALL_1(TPR) block_norm_backward_kernel<T, 1, 4, 0, false, TPR, 1, false><<<blocks, p.threads, join, s>>>(q)
  if (p.nv == 0 && p.vec == V) {
    block_norm_backward_long_kernel<T, V><<<blocks, p.threads, 0, s>>>(q);
  } else if (p.nv == 0) {
    block_norm_backward_long_kernel<T, 1><<<blocks, p.threads, 0, s>>>(q);
  } else if (p.vec == V && p.nv == 1 && all) {
    SNNB_NORM_BY_TPR(SNNB_CALL_A)
  } else if (p.vec == V && p.nv == 1) {
    SNNB_NORM_BY_TPR(SNNB_CALL_V)
  } else if (p.vec == V) {
    launch_kernel<block_norm_backward_kernel<T, V, 2, 0, true, 512, 1, false>>(q, blocks, p.threads, 4 * q.D * (int)sizeof(float), s);
  } else if (p.nv == 4) {
    SNNB_NORM_BY_TPR(SNNB_CALL_1)
  } else {
    block_norm_backward_kernel<T, 1, 8, 0, false, 512, 1, false><<<blocks, p.threads, join, s>>>(q);
  }
#undef SNNB_CALL_V
#undef SNNB_CALL_A
#undef SNNB_CALL_1
  if (q.dw_post || q.dscale || q.dw_pre) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((q.D + 31) / 32), 2);
    cfg.blockDim = dim3(1024);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    cudaLaunchKernelEx(&cfg, block_norm_sums_kernel<T>, q, blocks);
  }
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
  for (const void *in : {y, gate, (const void *)res_out})
    SNNB_CHECK_ARG(!z || z != in, "block_norm: z shares its buffer with another argument");
  SNNB_CHECK_ARG(!z || z != res, "block_norm: z shares its buffer with another argument");
  SNNB_CHECK_ARG(!res_out || (res_out != y && res_out != gate), "block_norm: res_out shares its buffer with y or the gate");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SNNB_F32: launch_forward<float>(q, dtype, s); break;
    case SNNB_BF16: launch_forward<__nv_bfloat16>(q, dtype, s); break;
    default: launch_forward<__half>(q, dtype, s); break;
  }
  SNNB_CHECK_LAUNCH("block_norm");
  return SNNB_OK;
}

extern "C" int64_t snnb_block_norm_backward_workspace_bytes(int64_t M, int D) {
  return (int64_t)snnb::backward_blocks(M, D) * 2 * (D > 0 ? D : 0) * (int64_t)sizeof(float);
}

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
  const void *outs[] = {dy, dgate, dres}, *ins[] = {dres_out, dz, y, gate, res};
  for (int i = 0; i < 3; ++i) {
    for (const void *in : ins)
      SNNB_CHECK_ARG(!outs[i] || outs[i] != in, "block_norm_backward: an output is one of the inputs");
    SNNB_CHECK_ARG(!outs[i] || outs[i] != outs[(i + 1) % 3], "block_norm_backward: two outputs are one buffer");
  }
  SNNB_CHECK_ARG(workspace && workspace_bytes >= snnb_block_norm_backward_workspace_bytes(M, D),
                 "block_norm_backward: workspace too small");
  SNNB_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "block_norm_backward: workspace must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SNNB_F32: launch_backward<float>(q, dtype, s); break;
    case SNNB_BF16: launch_backward<__nv_bfloat16>(q, dtype, s); break;
    default: launch_backward<__half>(q, dtype, s); break;
  }
  SNNB_CHECK_LAUNCH("block_norm_backward");
  return SNNB_OK;
}
