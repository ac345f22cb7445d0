// Kernels of the gated scan. The formulas are in gated_scan.cu.
//
// A step is the affine map h -> a h + u, and maps compose: (A, H) followed by (a, u) is (a A, a H + u). So a block takes
// a tile of CH channels x SEG * L steps; a thread owns VEC channels x L consecutive steps (a segment) in registers and
//   1. composes its L steps and leaves (A, H) in shared memory;
//   2. one thread per channel, a joiner, walks the SEG maps from the state in front of the tile;
//   3. every thread walks its L steps from the state that the joiner left for its segment.
// Long sequences with few channels are split over a cluster of blocks as well: the blocks of a cluster take consecutive
// tiles, their joiners exchange the tiles' maps through distributed shared memory, and all step on by S tiles. Every input
// is read once, the loads of the next tile are in flight while the current one is worked on, and nothing is summed by
// atomics, so a result depends on the split (which depends on the sizes and the number of SMs alone) but not on the run.
//
// What bounds it, on B200: forward 6, backward 10 bytes an element (bf16) at the floor. B8 T2048 D2048 bf16, 33.5 M
// elements, device time: forward 39 us = 5.1 TB/s (78 % of the measured copy rate), backward 70 us = 4.8 TB/s (73 %); the
// same in fp32 with D1024 39 and 69, padded batches of half as many steps 33 and 57. An element costs 19 instructions
// forward, two of them on the special-function pipe, and the 512 blocks leave every seventh place of the GPU's 592 empty:
// issue slots and that imbalance are what is left (issue 51 % of the active cycles). The packed fp32 instructions, the
// joiners (instead of every thread folding the maps in front of it: 128 registers and spills, 71 us) and the copies past L1
// are what brought it there from 195 us.
#pragma once

#include <cooperative_groups.h>

#include <type_traits>

#include "gated_scan.cuh"
#include "packed.cuh"
#include "umma.cuh"

namespace snnb {
namespace {

namespace cg = cooperative_groups;

constexpr int kCkpt = SNNB_GATED_SCAN_CKPT_STEPS;
constexpr int kMaxCluster = 8;      // blocks of a cluster: the portable limit

template <typename T, int N> __device__ __forceinline__ Pack<T, N> ld_raw(const T *p) {
  constexpr int BYTES = sizeof(T) * N;
  Pack<T, N> r;
  if constexpr (BYTES == 16) *reinterpret_cast<int4 *>(&r) = __ldcs(reinterpret_cast<const int4 *>(p));
  else if constexpr (BYTES == 8) *reinterpret_cast<int2 *>(&r) = __ldcs(reinterpret_cast<const int2 *>(p));
  else if constexpr (BYTES == 4) *reinterpret_cast<int *>(&r) = __ldcs(reinterpret_cast<const int *>(p));
  else *reinterpret_cast<unsigned short *>(&r) = __ldcs(reinterpret_cast<const unsigned short *>(p));
  return r;
}

template <typename T, int N> __device__ __forceinline__ void st_raw(T *p, const float (&v)[N]) {
  constexpr int BYTES = sizeof(T) * N;
  Pack<T, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = DT<T>::from_f(v[i]);
  if constexpr (BYTES == 16) *reinterpret_cast<int4 *>(p) = *reinterpret_cast<const int4 *>(&r);
  else if constexpr (BYTES == 8) *reinterpret_cast<int2 *>(p) = *reinterpret_cast<const int2 *>(&r);
  else if constexpr (BYTES == 4) *reinterpret_cast<int *>(p) = *reinterpret_cast<const int *>(&r);
  else *p = r.v[0];
}

template <typename T, int N>
__device__ __forceinline__ void state_load(const void *p, int f32, int64_t i, bool ok, float (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = 0.f;
  if (p == nullptr || !ok) return;
  if (f32) {
    const Pack<float, N> r = ld_raw<float, N>(static_cast<const float *>(p) + i);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = r.v[k];
  } else {
    const Pack<T, N> r = ld_raw<T, N>(static_cast<const T *>(p) + i);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = DT<T>::to_f(r.v[k]);
  }
}

template <typename T, int N>
__device__ __forceinline__ void state_store(void *p, int f32, int64_t i, bool ok, const float (&v)[N]) {
  if (p == nullptr || !ok) return;
  if (f32) st_raw<float, N>(static_cast<float *>(p) + i, v);
  else st_raw<T, N>(static_cast<T *>(p) + i, v);
}

// The decay a and 1 - a of each channel.
template <bool SIG, int N> __device__ __forceinline__ void gates_of(const float (&g)[N], float (&a)[N], float (&b)[N]) {
  if constexpr (SIG) {
    v_sigmoid(g, a, b);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) { a[k] = g[k]; b[k] = 1.f - g[k]; }
  }
}

// One channel's walk over the maps (pA, pX) of a tile's segments, stride floats apart, from the first (DIR 1) or the last
// (DIR -1): each pX becomes the value in front of its segment, and the value behind the tile is returned. The maps are
// read eight at a time before the walk over them, so that their loads overlap.
template <int SEG, int DIR> __device__ __forceinline__ float join(const float *pA, float *pX, int stride, float v) {
  constexpr int N = SEG < 8 ? SEG : 8;
#pragma unroll
  for (int s0 = 0; s0 < SEG; s0 += N) {
    float fA[N], fX[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int s = DIR > 0 ? s0 + i : SEG - 1 - s0 - i;
      fA[i] = pA[s * stride];
      fX[i] = pX[s * stride];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int s = DIR > 0 ? s0 + i : SEG - 1 - s0 - i;
      pX[s * stride] = v;
      v = fmaf(fA[i], v, fX[i]);
    }
  }
  return v;
}

static __device__ int g_scan_status = 0;      // set when a bounded wait gave up

// The maps of the tiles that the blocks of a cluster work on at the same time. Each joiner stores its channel's map in the
// shared memory of every block with an asynchronous store that counts on a barrier there, and waits for its own block's
// barrier. (A cluster barrier instead would order all stores of h before it as well: with it, two blocks that shared a
// sequence took longer than one alone.) Two slots: a block sends for step i + 2 after it has received everybody's map of
// step i + 1, which they sent after they had read those of step i.
// A block of which a joiner's wait gives up (the maps of a step did not come within about two seconds) sends, re-arms and
// reads nothing from its next step on, so the others' waits run out as well, and the call's results are worthless. No block
// leaves before all of its cluster have stopped sending, for a map may still be on its way to one that has given up.
template <int CH> struct Exchange {
  float2 *map;            // [2][S][CH]
  uint32_t bar, bytes;    // two barriers, 8 bytes apart
  int S, rank;
  volatile int *abort;    // a wait of the block gave up; in shared memory, for the backward pass has no register for it

  __device__ __forceinline__ void init(float2 *m, uint64_t *bars, int *abort_flag, int s, int r, const ScanArgs &q) {
    map = m; bar = umma::smem_u32(bars); S = s; rank = r; abort = abort_flag;
    bytes = (uint32_t)(S * CH * sizeof(float2));
    if (S == 1) return;
    if (threadIdx.x == 0) {
      *abort = 0;
      umma::mbar_init(bar, 1);
      umma::mbar_init(bar + 8, 1);
      umma::fence_mbar_init();
      umma::mbar_expect_tx(bar, bytes + (q.miss_map && (int)blockIdx.x == S - 1 ? 8 : 0));
      umma::mbar_expect_tx(bar + 8, bytes);
    }
    cg::this_cluster().sync();
  }
  // threads 0 .. CH - 1, one channel each; false: there are no maps
  __device__ __forceinline__ bool swap(const ScanArgs &q, int it, float A, float X) {
    if (*abort) return false;
    const int slot = it & 1;
    const uint32_t at = umma::smem_u32(map + (slot * S + rank) * CH + threadIdx.x), b = bar + 8 * slot;
    for (int r = 0; r < S; ++r) {
      uint32_t ra, rb;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(at), "r"(r));
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rb) : "r"(b), "r"(r));
      asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];"
                   ::"r"(ra), "f"(A), "f"(X), "r"(rb) : "memory");
    }
    if (!umma::mbar_wait(b, (it >> 1) & 1, abort, q.wait_limit)) {
      atomicExch(&g_scan_status, 1);
      return false;
    }
    if (threadIdx.x == 0) umma::mbar_expect_tx(b, bytes);      // for step it + 2
    return true;
  }
  // all threads, at the end of the kernel; nothing has to be ordered, so the barrier does not wait for the stores of h
  __device__ __forceinline__ void leave() const {
    if (S == 1) return;
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    asm volatile("barrier.cluster.wait;" ::: "memory");
    if (*abort)      // the last maps of the others land meanwhile
      for (int i = 0; i < 32; ++i) __nanosleep(1000);
  }
  __device__ __forceinline__ float2 of(int it, int r) const { return map[((it & 1) * S + r) * CH + threadIdx.x]; }
};

// How a row of a tile is accessed.
enum class Rows {
  copied,   // through shared memory, VEC neighbouring channels a thread; rows start on 16-byte boundaries
  direct,   // straight to registers, VEC neighbouring channels a thread, as above
  ragged    // straight to registers, VEC channels LANES apart a thread; rows start anywhere
};

// Where a thread stands, and how it reaches the values of its steps. NA: arrays that are read. A warp copies the rows of
// its own segments into shared memory, 16 bytes a lane, and only the warp waits for them.
template <typename T, Rows R, int VEC, int LANES, int SEG, int L, int STAGES, int NA> struct Tile {
  static constexpr int CH = LANES * VEC, TC = SEG * L, SZ = (int)sizeof(T);
  static constexpr int ROW = CH * SZ, ARRAY = TC * ROW, STAGE = NA * ARRAY;
  // Offsets from the first row and channel of the tile: 32 bits where the launch has checked that they fit, so that an
  // address is a base that all threads share and a 32-bit offset; else the 64-bit product of two 32-bit numbers.
  using Off = std::conditional_t<R == Rows::copied, uint32_t, int64_t>;

  const ScanArgs &q;
  unsigned char *dyn;
  int lane, seg, S, rank, len;
  int64_t b, d0;

  __device__ __forceinline__ Tile(const ScanArgs &args, unsigned char *smem) : q(args), dyn(smem) {
    lane = threadIdx.x % LANES;
    seg = threadIdx.x / LANES;
    S = SEG > 1 ? (int)cg::this_cluster().num_blocks() : 1;
    rank = SEG > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const int tile = blockIdx.x / S;
    b = tile / q.tiles_d;
    d0 = (int64_t)(tile % q.tiles_d) * CH;
    len = (int)q.T;
    if (q.lengths) len = min(max(q.lengths[b], 0), (int)q.T);
  }
  __device__ __forceinline__ int channel(int k) const { return R == Rows::ragged ? lane + k * LANES : lane * VEC + k; }
  // whether the thread has channels at all, and whether all of the tile's exist
  __device__ __forceinline__ bool any() const { return d0 + channel(0) < q.D; }
  __device__ __forceinline__ bool all() const { return d0 + CH <= q.D; }
  // the channel that thread j of the first CH joins
  __device__ __forceinline__ int64_t joined(int j) const { return d0 + (R == Rows::ragged ? j % VEC * LANES + j / VEC : j); }

  __device__ __forceinline__ char *rows(const ScanSeq &s, int tile0) const {
    return const_cast<char *>(static_cast<const char *>(s.p)) + (b * s.bs + (int64_t)tile0 * s.ts + d0) * SZ;
  }
  __device__ __forceinline__ Off row_off(const ScanSeq &s, int row) const { return (Off)row * (Off)(int)(s.ts * SZ); }
  __device__ __forceinline__ void copy(int array, int st, const ScanSeq &s, int tile0) const {
    constexpr int WSEG = 32 / LANES, CHUNKS = ROW / 16;
    const char *from = rows(s, tile0);
    const int chunk = threadIdx.x % CHUNKS;
    const bool cok = d0 + chunk * (16 / SZ) < q.D;
    unsigned char *to = dyn + st * STAGE + array * ARRAY + chunk * 16;
#pragma unroll
    for (int i = 0; i < WSEG * L * CHUNKS / 32; ++i) {
      const int r = i * (32 / CHUNKS) + threadIdx.x % 32 / CHUNKS;
      const int l = r / WSEG, sg = (int)(threadIdx.x / 32) * WSEG + r % WSEG;
      if (cok && tile0 + sg * L + l < len)
        copy_async16(to + (l * SEG + sg) * ROW, from + (row_off(s, sg * L + l) + (Off)(chunk * 16)));
    }
  }
  // the thread's values of its step l, in shared memory
  __device__ __forceinline__ Pack<T, VEC> *slot(int array, int st, int l) const {
    return reinterpret_cast<Pack<T, VEC> *>(dyn + st * STAGE + array * ARRAY) + l * LANES * SEG + threadIdx.x;
  }
  __device__ __forceinline__ void zero(const ScanSeq &s, int tile0) const {
    float z[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) z[k] = 0.f;
    for (int l = 0; l < L; ++l)
      if (any() && tile0 + seg * L + l < (int)q.T) store<false>(s, tile0, l, z);
  }
  template <bool FULL> __device__ __forceinline__ Pack<T, VEC> load(const ScanSeq &s, int tile0, int l) const {
    const T *p = reinterpret_cast<const T *>(rows(s, tile0) + (row_off(s, seg * L + l) + (Off)(channel(0) * SZ)));
    if constexpr (R == Rows::ragged) {
      Pack<T, VEC> r = {};
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (FULL || d0 + channel(k) < q.D) r.v[k] = __ldcs(p + k * LANES);
      return r;
    } else {
      return ld_raw<T, VEC>(p);
    }
  }
  template <bool FULL> __device__ __forceinline__ void store(const ScanSeq &s, int tile0, int l, const float (&v)[VEC]) const {
    char *p = rows(s, tile0) + (row_off(s, seg * L + l) + (Off)(channel(0) * SZ));
    if constexpr (R == Rows::ragged) {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (FULL || d0 + channel(k) < q.D) *reinterpret_cast<T *>(p + k * LANES * SZ) = DT<T>::from_f(v[k]);
    } else {
      st_raw<T, VEC>(reinterpret_cast<T *>(p), v);
    }
  }
};

// LK: 0 plain, 1 leaky, 2 as q.leaky says (the forms that are not worth a kernel each).
// STAGES: tiles in shared memory, all but one of them on their way while one is worked on.
template <typename T, Rows R, bool SIG, int LK, int VEC, int LANES, int SEG, int L, int STAGES, int MINB>
__global__ void __launch_bounds__(LANES *SEG, MINB) gated_scan_kernel(const __grid_constant__ ScanArgs q) {
  using G = Tile<T, R, VEC, LANES, SEG, L, STAGES, 2>;
  constexpr int CH = G::CH, TC = G::TC;
  constexpr bool STAGED = R == Rows::copied;
  static_assert(SEG == 1 || (kCkpt % TC == 0 && CH <= LANES * SEG), "checkpoints lie in front of tiles; a thread per channel");
  __shared__ __align__(16) float sA[SEG > 1 ? SEG * CH : 4], sH[SEG > 1 ? SEG * CH : 4];
  __shared__ uint64_t bars[2];
  __shared__ int abort_flag;
  extern __shared__ __align__(16) unsigned char dyn[];      // the tiles on their way, then the exchange of the cluster
  const G g(q, dyn);
  const int T_ = (int)q.T, S = g.S;
  const bool leaky = LK == 1 || (LK == 2 && q.leaky);

  // The state in front of the cluster's current tiles: with one segment each thread has its channels', otherwise the
  // first CH threads, the joiners, have one channel each.
  constexpr int CV = SEG == 1 ? VEC : 1;
  const int64_t jd = SEG == 1 ? g.d0 + g.channel(0) : g.joined(threadIdx.x);
  const bool joiner = SEG == 1 || threadIdx.x < CH, jok = joiner && jd < q.D;
  const int64_t ji = g.b * q.D + jd;
  float carry[CV];
  state_load<T, CV>(q.h_init, q.state_f32, ji, jok, carry);

  auto fetch = [&](int tile0, int st) {
    if constexpr (STAGED) {
      g.copy(0, st, q.g, tile0);
      g.copy(1, st, q.x, tile0);
      copy_commit();
    }
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch((i * S + g.rank) * TC, i);
  Exchange<CH> cluster_maps;
  if constexpr (SEG > 1)      // behind every block's read of h_init: the first block may write h_last to the same buffer
    cluster_maps.init(reinterpret_cast<float2 *>(dyn + (STAGED ? STAGES * G::STAGE : 0)), bars, &abort_flag, S, g.rank, q);
  int st = 0, base = 0, it = 0;
  // One tile. FULL: every step of it counts and all channels exist, so nothing is asked.
  auto work = [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
    const int tile0 = base + g.rank * TC, t0 = tile0 + g.seg * L;
    const int n = FULL ? L : (g.any() ? min(g.len - t0, L) : 0);
    float a[L][VEC], u[L][VEC];
    Pack<T, VEC> in[STAGED ? 1 : L][2];
    if constexpr (STAGED) {
      __syncwarp();      // the warp has read what it overwrites
      fetch(tile0 + (STAGES - 1) * S * TC, st == 0 ? STAGES - 1 : st - 1);
      copy_wait<STAGES - 1>();
      __syncwarp();
    } else {
#pragma unroll
      for (int l = 0; l < L; ++l)
        if (FULL || l < n) {
          in[l][0] = g.template load<FULL>(q.g, tile0, l);
          in[l][1] = g.template load<FULL>(q.x, tile0, l);
        }
    }
#pragma unroll
    for (int l = 0; l < L; ++l) {
      if (FULL || l < n) {
        float gv[VEC], bb[VEC];
        if constexpr (STAGED) {
          widen<T, VEC>(g.slot(0, st, l)->v, gv);
          widen<T, VEC>(g.slot(1, st, l)->v, u[l]);
        } else {
          // (ragged rows one by one: 96 us instead of 139 for B8 T2048 D2047 bf16; the backward pass, which keeps them
          // longer, is faster with words: 104 instead of 117 for B64 T64 D2047)
          widen<T, VEC, R != Rows::ragged>(in[l][0].v, gv);
          widen<T, VEC, R != Rows::ragged>(in[l][1].v, u[l]);
        }
        gates_of<SIG, VEC>(gv, a[l], bb);
        if (leaky) v_mul(bb, u[l], u[l]);
      } else {
        v_set(a[l], 1.f);
        v_set(u[l], 0.f);
      }
    }
    if constexpr (STAGED) st = st == STAGES - 1 ? 0 : st + 1;
    float h[VEC];
    if constexpr (SEG == 1) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) h[k] = carry[k];
    } else {
      float A[VEC], H[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) { A[k] = a[0][k]; H[k] = u[0][k]; }
#pragma unroll
      for (int l = 1; l < L; ++l) {
        v_fma(a[l], H, u[l], H);
        v_mul(A, a[l], A);
      }
      sh_store<VEC>(sA + g.seg * CH + g.lane * VEC, A);
      sh_store<VEC>(sH + g.seg * CH + g.lane * VEC, H);
      __syncthreads();
      if (joiner) {
        float h1 = carry[0];
        if (S > 1) {
          float tA = 1.f, tH = 0.f;      // the tile's map
#pragma unroll
          for (int s = 0; s < SEG; ++s) {
            const float fA = sA[s * CH + threadIdx.x];
            tH = fmaf(fA, tH, sH[s * CH + threadIdx.x]);
            tA *= fA;
          }
          if (cluster_maps.swap(q, it, tA, tH)) {
            float c = carry[0];
            for (int r = 0; r < S; ++r) {
              if (r == g.rank) h1 = c;
              const float2 m = cluster_maps.of(it, r);
              c = fmaf(m.x, c, m.y);
            }
            carry[0] = c;
          }
        }
        if (jok && q.ckpt && tile0 > 0 && tile0 % kCkpt == 0 && tile0 < T_)
          q.ckpt[(int64_t)(tile0 / kCkpt - 1) * q.B * q.D + ji] = h1;
        h1 = join<SEG, 1>(sA + threadIdx.x, sH + threadIdx.x, CH, h1);
        if (S == 1) carry[0] = h1;
      }
      __syncthreads();
      sh_load<VEC>(sH + g.seg * CH + g.lane * VEC, h);      // written by this thread alone from here to the next barrier
    }
    const int m = g.any() ? min(T_ - t0, L) : 0;
#pragma unroll
    for (int l = 0; l < L; ++l) {
      float out[VEC];
      v_fma(a[l], h, u[l], h);
#pragma unroll
      for (int k = 0; k < VEC; ++k) out[k] = FULL || l < n ? h[k] : 0.f;
      if (FULL || l < m) g.template store<FULL>(q.h, tile0, l, out);
    }
    if constexpr (SEG == 1) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) carry[k] = h[k];
    }
  };
  for (; base < T_ && (base < g.len || SEG == 1); base += S * TC, ++it) {
    if (g.all() && base + (g.rank + 1) * TC <= g.len) work(std::true_type{});
    else work(std::false_type{});
  }
  if (g.rank == 0) state_store<T, CV>(q.h_last, q.state_f32, ji, jok, carry);
  if constexpr (SEG > 1) {
    for (; base < T_; base += S * TC) g.zero(q.h, base + g.rank * TC);      // tiles behind the sequence
    cluster_maps.leave();
  }
}

// The same split from the end. With c the gradient that reaches a step from the one behind it (c = a_{t+1} lam_{t+1}):
// lam = dh + c, and the step hands a dh + a c on to the one before, again an affine map, with the same factor a. The
// states in front of the steps are rebuilt from the checkpoint in front of the tile.
template <typename T, Rows R, bool SIG, int LK, int VEC, int LANES, int SEG, int L, int STAGES, int MINB>
__global__ void __launch_bounds__(LANES *SEG, MINB) gated_scan_backward_kernel(const __grid_constant__ ScanArgs q) {
  using G = Tile<T, R, VEC, LANES, SEG, L, STAGES, 3>;
  constexpr int CH = G::CH, TC = G::TC, SZ = G::SZ;
  constexpr bool STAGED = R == Rows::copied;
  static_assert(SEG == 1 || 2 * CH <= LANES * SEG, "two threads per channel");
  static_assert(SEG == 1 || TC == kCkpt || TC <= 64, "a tile starts from a checkpoint, or is the only one");
  __shared__ __align__(16) float sA[SEG > 1 ? SEG * CH : 4], sH[SEG > 1 ? SEG * CH : 4], sC[SEG > 1 ? SEG * CH : 4];
  __shared__ uint64_t bars[2];
  __shared__ int abort_flag;
  extern __shared__ __align__(16) unsigned char dyn[];
  const G g(q, dyn);
  const int T_ = (int)q.T, S = g.S;
  const bool leaky = LK == 1 || (LK == 2 && q.leaky);

  // The first CH threads join the gradients of a channel each, the next CH threads the states. carry: the gradient that
  // reaches the cluster's current tiles from behind.
  constexpr int CV = SEG == 1 ? VEC : 1;
  const bool join_c = SEG == 1 || threadIdx.x < CH, join_h = SEG == 1 || (threadIdx.x >= CH && threadIdx.x < 2 * CH);
  const int jc = threadIdx.x % CH;
  const int64_t jd = SEG == 1 ? g.d0 + g.channel(0) : g.joined(jc);
  const bool jok = (join_c || join_h) && jd < q.D;
  const int64_t ji = g.b * q.D + jd;
  float carry[CV];
  state_load<T, CV>(q.dh_last, q.state_f32, ji, jok && join_c, carry);

  auto fetch = [&](int tile0, int st) {
    if constexpr (STAGED) {
      if (tile0 >= 0) {
        g.copy(0, st, q.g, tile0);
        g.copy(1, st, q.x, tile0);
        g.copy(2, st, q.h, tile0);
      }
      copy_commit();
    }
  };
  // the state in front of the block's tile, if any of its steps count
  auto front_of = [&](int tile0, float (&v)[CV]) {
    if (tile0 == 0) state_load<T, CV>(q.h_init, q.state_f32, ji, jok && join_h, v);
    else if (tile0 > 0 && tile0 < g.len) state_load<float, CV>(q.ckpt, 1, (int64_t)(tile0 / kCkpt - 1) * q.B * q.D + ji, jok && join_h, v);
  };
  const int last = T_ > 0 ? (T_ - 1) / (S * TC) * (S * TC) : -1;
  int base = SEG == 1 ? last : g.len > 0 ? (g.len - 1) / (S * TC) * (S * TC) : -1;
  float front[CV] = {};
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(base - i * S * TC < 0 ? -1 : base + g.rank * TC - i * S * TC, i);
  front_of(base < 0 ? -1 : base + g.rank * TC, front);
  Exchange<CH> cluster_maps;
  if constexpr (SEG > 1) {
    // behind every block's read of dh_last: the first block may write dh_init to the same buffer
    cluster_maps.init(reinterpret_cast<float2 *>(dyn + (STAGED ? STAGES * G::STAGE : 0)), bars, &abort_flag, S, g.rank, q);
    for (int t = last; t > base && t >= 0; t -= S * TC) {      // tiles behind the sequence
      g.zero(q.dx, t + g.rank * TC);
      g.zero(q.dg, t + g.rank * TC);
    }
  }
  int st = 0, it = 0;
  auto work = [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
    const int tile0 = base + g.rank * TC, t0 = tile0 + g.seg * L;
    const int n = FULL ? L : (g.any() ? min(g.len - t0, L) : 0), m = g.any() ? min(T_ - t0, L) : 0;
    float a[L][VEC], bb[L][VEC], h[VEC];
    Pack<T, VEC> in[STAGED ? 1 : L][3];
    if constexpr (STAGED) {
      __syncwarp();      // the warp has read what it overwrites
      fetch(base - (STAGES - 1) * S * TC < 0 ? -1 : tile0 - (STAGES - 1) * S * TC, st == 0 ? STAGES - 1 : st - 1);
      copy_wait<STAGES - 1>();
      __syncwarp();
    } else {
#pragma unroll
      for (int l = 0; l < L; ++l)
        if (FULL || l < n) {
          in[l][0] = g.template load<FULL>(q.g, tile0, l);
          in[l][1] = g.template load<FULL>(q.x, tile0, l);
          in[l][2] = g.template load<FULL>(q.h, tile0, l);
        }
    }
    // gate (0), input (1), gradient of h (2) of a step; zeros for one that does not count
    auto value_of = [&](int l, int which, float (&v)[VEC]) {
      if (!FULL && l >= n) {
        v_set(v, 0.f);
      } else if constexpr (STAGED) {
        widen<T, VEC>(g.slot(which, st, l)->v, v);
      } else {
        widen<T, VEC>(in[l][which].v, v);
      }
    };
    auto input_of = [&](int l, float (&v)[VEC]) {
      value_of(l, 1, v);
      if (leaky) v_mul(bb[l], v, v);
    };
#pragma unroll
    for (int l = 0; l < L; ++l) {
      if (FULL || l < n) {
        float gv[VEC];
        value_of(l, 0, gv);
        gates_of<SIG, VEC>(gv, a[l], bb[l]);
      } else {
        v_set(a[l], 1.f);
        v_set(bb[l], 0.f);
      }
    }
    float now[CV];      // a tile behind the sequence has none, and no step that asks for it
#pragma unroll
    for (int k = 0; k < CV; ++k) now[k] = front[k];
    if (base > 0) front_of(tile0 - S * TC, front);
    float c[VEC];
    if constexpr (SEG == 1) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) { c[k] = carry[k]; h[k] = now[k]; }
    } else {
      float A[VEC], H[VEC], C[VEC];
      v_set(A, 1.f);
      v_set(H, 0.f);
      v_set(C, 0.f);
#pragma unroll
      for (int l = 0; l < L; ++l) {
        float u[VEC], dh[VEC];
        input_of(l, u);
        value_of(L - 1 - l, 2, dh);
        v_fma(a[l], H, u, H);
        v_mul(A, a[l], A);
        v_add(dh, C, C);
        v_mul(a[L - 1 - l], C, C);
      }
      sh_store<VEC>(sA + g.seg * CH + g.lane * VEC, A);
      sh_store<VEC>(sH + g.seg * CH + g.lane * VEC, H);
      sh_store<VEC>(sC + g.seg * CH + g.lane * VEC, C);
      __syncthreads();
      if (join_c) {
        float c1 = carry[0];
        if (S > 1) {
          float tA = 1.f, tC = 0.f;      // the tile's map
#pragma unroll
          for (int s = SEG - 1; s >= 0; --s) {
            const float fA = sA[s * CH + jc];
            tC = fmaf(fA, tC, sC[s * CH + jc]);
            tA *= fA;
          }
          if (cluster_maps.swap(q, it, tA, tC)) {
            float v = carry[0];
            for (int r = S - 1; r >= 0; --r) {
              if (r == g.rank) c1 = v;
              const float2 mp = cluster_maps.of(it, r);
              v = fmaf(mp.x, v, mp.y);
            }
            carry[0] = v;
          }
        }
        c1 = join<SEG, -1>(sA + jc, sC + jc, CH, c1);
        if (S == 1) carry[0] = c1;
      } else if (join_h) {
        join<SEG, 1>(sA + jc, sH + jc, CH, now[0]);
      }
      __syncthreads();
      sh_load<VEC>(sH + g.seg * CH + g.lane * VEC, h);
      sh_load<VEC>(sC + g.seg * CH + g.lane * VEC, c);
    }
    // What the gate's gradient needs of each step, the state in front of it (less its input): kept in fp32, in shared
    // memory in the place of the gate and, for 16-bit types, the input that are not needed any more.
    float hb[STAGED ? 1 : L][VEC];
    auto keep = [&](int l, float (&w)[VEC], auto write) {
      constexpr bool W = decltype(write)::value;
      if constexpr (!STAGED) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          if (W) hb[l][k] = w[k];
          else w[k] = hb[l][k];
        }
      } else {
        constexpr int PARTS = SZ == 2 ? 2 : 1, N = VEC / PARTS;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          Pack<float, N> *f = reinterpret_cast<Pack<float, N> *>(g.slot(i, st, l));
#pragma unroll
          for (int k = 0; k < N; ++k) {
            if (W) f->v[k] = w[i * N + k];
            else w[i * N + k] = f->v[k];
          }
        }
      }
    };
#pragma unroll
    for (int l = 0; l < L; ++l) {
      float u[VEC], w[VEC];
      value_of(l, 1, w);
#pragma unroll
      for (int k = 0; k < VEC; ++k) u[k] = leaky ? bb[l][k] * w[k] : w[k];
#pragma unroll
      for (int k = 0; k < VEC; ++k) w[k] = leaky ? h[k] - w[k] : h[k];
      v_fma(a[l], h, u, h);
      if (FULL || l < n) keep(l, w, std::true_type{});
    }
    // the gradients, from the last step to the first
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
      float gx[VEC], gg[VEC], dh[VEC], w[VEC], lam[VEC];
      value_of(l, 2, dh);
      v_set(w, 0.f);
      if (FULL || l < n) keep(l, w, std::false_type{});
      v_add(dh, c, lam);
      v_mul(a[l], lam, c);
      v_mul(lam, w, gg);
      if constexpr (SIG) {
        float ab[VEC];
        v_mul(a[l], bb[l], ab);
        v_mul(gg, ab, gg);
      }
      if (leaky) {
        v_mul(bb[l], lam, gx);
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) gx[k] = lam[k];
      }
      if (!FULL && l >= n) {
        v_set(gx, 0.f);
        v_set(gg, 0.f);
      }
      if (FULL || l < m) {
        g.template store<FULL>(q.dx, tile0, l, gx);
        g.template store<FULL>(q.dg, tile0, l, gg);
      }
    }
    if constexpr (STAGED) st = st == STAGES - 1 ? 0 : st + 1;
    if constexpr (SEG == 1) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) carry[k] = c[k];
    }
  };
  for (; base >= 0; base -= S * TC, ++it) {
    if (g.all() && base + (g.rank + 1) * TC <= g.len) work(std::true_type{});
    else work(std::false_type{});
  }
  if (g.rank == 0) state_store<T, CV>(q.h_last, q.state_f32, ji, jok && join_c, carry);
  if constexpr (SEG > 1) cluster_maps.leave();
}

// smem: of the stages; the exchange of a cluster of S comes on top.
template <auto Kern>
int launch_tiles(ScanArgs q, int threads, int CH, int S, int smem, cudaStream_t s) {
  const int64_t tiles_d = (q.D + CH - 1) / CH, blocks = tiles_d * q.B * S;
  if (blocks > 0x7fffffffLL) return fail(SNNB_ERR_INVALID, "gated_scan: problem too large");
  q.tiles_d = (int)tiles_d;
  q.wait_limit = 4000000000ll;
  q.miss_map = 0;
  if (S > 1) consume_wait_selftest(&q.wait_limit, &q.miss_map);
  cudaError_t e = smem > 0 ? raise_smem_limit_once<Kern>(smem + 2 * kMaxCluster * CH * 8) : cudaSuccess;
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)(smem + 2 * S * CH * 8);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)S;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = S > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, Kern, q);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(SNNB_ERR_CUDA, "gated_scan: launch failed: %s", cudaGetErrorString(e));
  }
  return SNNB_OK;
}

// Blocks of a cluster for `tiles` channel tiles of `steps` tiles of time: doubled while each block has a tile of time and
// all blocks run at once, `most` of them to an SM, or fewer where shared memory (`smem` bytes a block, and the exchange of
// the cluster's CH channels) holds fewer: the backward pass of 16-bit rows, with 55 KB, has room for four blocks in clusters
// of one or two and for three in larger ones. Device time (bf16, us, forward / backward) with 1, 2, 4, 8 blocks:
//   B1 T4096 D2048 (64 tiles)       33 23 16 14 / 61 39 26 31       B1 T16384 D2048   126 85 56 45 / 238 148 95 106
//   B2 T4096 D2048 (128)            34 29 24 27 / 62 49 52 51       B1 T1024 D4096    10.3 10.1 8.9 11.2 / 17 15 17 18
//   B4 T2048 D2048 (256)            24 23 25 29 / 42 40 48 55       B16 T1024 D1024 (512)   21 25 28 37 / 37 40 49 64
//   B2 T16384 D512 (32)             126 85 44 31 / 238 147 75 50
// The ragged backward kernel (512 threads, two blocks an SM) is given as many blocks as two waves take, its loads being
// what it waits for: B2 T4096 D2047 (128 tiles) 188 131 110 105, B1 T8192 D2047 (64) 361 203 131 116, B4 T2048 D2047 (256)
// 120 105 100 107; at short sequences one wave is a little better: B1 T1024 D2047 38 23 17 18, B6 T1031 D1001 fp32 (192)
// 51 53 55 75.
int scan_cluster(int64_t tiles, int64_t steps, int CH, int most, int smem) {
  const int sms = sm_count() > 0 ? sm_count() : 148;
  auto at_once = [&](int S) {
    const int room = 228 * 1024 / (smem + 2 * S * CH * 8 + 64 + 1024);      // the barriers, and what the system takes of each block
    return (int64_t)sms * (room < most ? room : most);
  };
  int S = 1;
  while (S < kMaxCluster && 2 * S <= steps && 2 * S * tiles <= at_once(2 * S)) S *= 2;
  return S;
}

// Up to 8 steps a thread walks alone. Beyond that:
// (The figures below are single calls, timed in steps of about 2 us.)
// - rows on 16-byte boundaries, up to 64 steps: one tile, no longer than needed, through shared memory. Measured against
//   the tile of 32 steps straight to registers and, from 33 steps on, the tile of 128 (bf16, D2048, us, forward and
//   backward): T16 B256 23 43 instead of 41 64, T24 B160 25 41 instead of 31 45, T33 B128 33 49 instead of 51 80, T64 B64
//   21 29 instead of 31 47. At T100 and T128 a single stage is no faster than the two of the long form (27 37 to 25 38).
// - the same, longer: tiles of 64 bytes of channels x 128 steps, two of them in shared memory, 128 threads with 8
//   steps of 8 bytes each and four blocks to an SM. Wider tiles leave too few blocks (64 channels, 256 threads: 71 us
//   instead of 47 for B8 T2048 D2048 bf16), 4 steps a thread double the joining (61 us); the backward pass with three
//   blocks and three tiles in shared memory took 86 us instead of 77, its 512 blocks then being more than run at once.
// - ragged rows: nothing wider than a value can be loaded, so the loads of many warps hide each other instead (64
//   registers, 32 warps to an SM): 96 us forward and 199 backward for B8 T2048 D2047 bf16. Copying the 16-byte blocks or
//   the words that a row lies in took 106 and 152 us: the addresses cost more than the loads; loading a tile ahead into
//   registers took as long. Up to 32 steps, backward 64, one tile no longer than needed, 4 steps a thread: 25 and 39 us for
//   T16 B256 D2047, 27 and 41 for T64 B64; with 8 steps of one channel a thread in 128 threads 139 and 152, in the long
//   form 104 backward for T64 B64.
template <typename T, bool SIG, int SEG, int L> int forward_tile(const ScanArgs &q, cudaStream_t s) {
  constexpr int VEC = 8 / (int)sizeof(T);
  using G = Tile<T, Rows::copied, VEC, 8, SEG, L, 1, 2>;
  return launch_tiles<gated_scan_kernel<T, Rows::copied, SIG, 2, VEC, 8, SEG, L, 1, 64 / SEG>>(q, 8 * SEG, G::CH, 1, G::STAGE, s);
}
template <typename T, bool SIG, int SEG, int L> int backward_tile(const ScanArgs &q, cudaStream_t s) {
  constexpr int VEC = 8 / (int)sizeof(T);
  using G = Tile<T, Rows::copied, VEC, 8, SEG, L, 1, 3>;
  return launch_tiles<gated_scan_backward_kernel<T, Rows::copied, SIG, 2, VEC, 8, SEG, L, 1, 64 / SEG>>(q, 8 * SEG, G::CH, 1, G::STAGE, s);
}

template <typename T, bool SIG, Rows R> int forward(const ScanArgs &q, cudaStream_t s) {
  constexpr int VEC = R == Rows::ragged ? 1 : 8 / (int)sizeof(T);
  if (q.T <= 1) return launch_tiles<gated_scan_kernel<T, R == Rows::ragged ? Rows::ragged : Rows::direct, SIG, 2, VEC, 64, 1, 1, 1, 1>>(q, 64, 64 * VEC, 1, 0, s);
  if (q.T <= 8) return launch_tiles<gated_scan_kernel<T, R == Rows::ragged ? Rows::ragged : Rows::direct, SIG, 2, VEC, 64, 1, 8, 1, 1>>(q, 64, 64 * VEC, 1, 0, s);
  if constexpr (R == Rows::copied) {
    if (q.T <= 16) return forward_tile<T, SIG, 4, 4>(q, s);
    if (q.T <= 32) return forward_tile<T, SIG, 4, 8>(q, s);
    if (q.T <= 64) return forward_tile<T, SIG, 8, 8>(q, s);
  } else {
    if (q.T <= 16) return launch_tiles<gated_scan_kernel<T, R, SIG, 2, 2, 16, 4, 4, 0, 16>>(q, 64, 32, 1, 0, s);
    if (q.T <= 32) return launch_tiles<gated_scan_kernel<T, R, SIG, 2, 2, 16, 8, 4, 0, 8>>(q, 128, 32, 1, 0, s);
  }
  constexpr bool RAG = R == Rows::ragged;
  constexpr int V = RAG ? 2 : VEC, LANES = RAG ? 16 : 8, SEG = 16, L = RAG ? 4 : 8, ST = RAG ? 0 : 2, MINB = 4;
  using G = Tile<T, R, V, LANES, SEG, L, ST, 2>;
  const int S = scan_cluster((q.D + G::CH - 1) / G::CH * q.B, (q.T + G::TC - 1) / G::TC, G::CH, 4,
                             ST * G::STAGE + 2 * SEG * G::CH * 4);
  if (q.leaky)
    return launch_tiles<gated_scan_kernel<T, R, SIG, 1, V, LANES, SEG, L, ST, MINB>>(q, LANES * SEG, G::CH, S, ST * G::STAGE, s);
  return launch_tiles<gated_scan_kernel<T, R, SIG, 0, V, LANES, SEG, L, ST, MINB>>(q, LANES * SEG, G::CH, S, ST * G::STAGE, s);
}

template <typename T, bool SIG, Rows R> int backward(const ScanArgs &q, cudaStream_t s) {
  constexpr int VEC = R == Rows::ragged ? 1 : 8 / (int)sizeof(T);
  if (q.T <= 8) return launch_tiles<gated_scan_backward_kernel<T, R == Rows::ragged ? Rows::ragged : Rows::direct, SIG, 2, VEC, 64, 1, 8, 1, 1>>(q, 64, 64 * VEC, 1, 0, s);
  if constexpr (R == Rows::copied) {
    if (q.T <= 16) return backward_tile<T, SIG, 8, 2>(q, s);
    if (q.T <= 32) return backward_tile<T, SIG, 8, 4>(q, s);
    if (q.T <= 64) return backward_tile<T, SIG, 8, 8>(q, s);
  } else {
    if (q.T <= 16) return launch_tiles<gated_scan_backward_kernel<T, R, SIG, 2, 2, 16, 4, 4, 0, 16>>(q, 64, 32, 1, 0, s);
    if (q.T <= 32) return launch_tiles<gated_scan_backward_kernel<T, R, SIG, 2, 2, 16, 8, 4, 0, 8>>(q, 128, 32, 1, 0, s);
    if (q.T <= 64) return launch_tiles<gated_scan_backward_kernel<T, R, SIG, 2, 2, 16, 16, 4, 0, 4>>(q, 256, 32, 1, 0, s);
  }
  constexpr bool RAG = R == Rows::ragged;
  constexpr int V = RAG ? 2 : VEC, LANES = RAG ? 16 : 8, SEG = RAG ? 32 : 16, L = RAG ? 4 : 8, ST = RAG ? 0 : 2, MINB = RAG ? 2 : 4;
  using G = Tile<T, R, V, LANES, SEG, L, ST, 3>;
  const int S = scan_cluster((q.D + G::CH - 1) / G::CH * q.B, (q.T + G::TC - 1) / G::TC, G::CH, 4,
                             ST * G::STAGE + 3 * SEG * G::CH * 4);
  if (q.leaky)
    return launch_tiles<gated_scan_backward_kernel<T, R, SIG, 1, V, LANES, SEG, L, ST, MINB>>(q, LANES * SEG, G::CH, S, ST * G::STAGE, s);
  return launch_tiles<gated_scan_backward_kernel<T, R, SIG, 0, V, LANES, SEG, L, ST, MINB>>(q, LANES * SEG, G::CH, S, ST * G::STAGE, s);
}

}  // namespace

template <typename T> int gated_scan_launch(ScanArgs q, bool bwd, int gate_kind, bool aligned, cudaStream_t s) {
  const bool sig = gate_kind == SNNB_GATE_SIGMOID;
  if (bwd) {
    if (aligned) return sig ? backward<T, true, Rows::copied>(q, s) : backward<T, false, Rows::copied>(q, s);
    return sig ? backward<T, true, Rows::ragged>(q, s) : backward<T, false, Rows::ragged>(q, s);
  }
  if (aligned) return sig ? forward<T, true, Rows::copied>(q, s) : forward<T, false, Rows::copied>(q, s);
  return sig ? forward<T, true, Rows::ragged>(q, s) : forward<T, false, Rows::ragged>(q, s);
}

// Reads and clears this translation unit's status word.
static int scan_unit_status(int *out) {
  int h = 0;
  const cudaError_t e = cudaMemcpyFromSymbol(&h, g_scan_status, sizeof(int));
  if (e != cudaSuccess) return fail(SNNB_ERR_CUDA, "device_status: %s", cudaGetErrorString(e));
  if (h != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_scan_status, &zero, sizeof(int));
  }
  *out = h;
  return SNNB_OK;
}

}  // namespace snnb
