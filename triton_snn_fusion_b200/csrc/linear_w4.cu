// Linear layer over a few tokens with 4-bit weights:
//
//   y[m][n] = sum_k x[m][k] (q[n][k] - zero[n][k / G]) scale[n][k / G] + b[n]
//
// q holds two weights per byte along K (even k in the low half), zero defaults to 8.
//
// The layer is bound by the bytes of its weights (N K / 2), as long as a weight costs about two instructions: so the
// products go to the tensor cores, with 16 weight rows as M and 8 tokens as N of a warp-level 16 x 8 x 16 product (the
// 128-row tensor-memory instructions would leave most of their columns empty and want the weights widened in shared
// memory first). q - zero is a small whole number and exact in either 16-bit type, so only the fp32 sums round; the scale
// is applied to the fp32 sum of its group. A sum over k may run in any order: a lane takes G / 4 neighbouring weights of
// its row, so that the four lanes of a row cover one group and its loads are 16, 8 or 4 bytes wide, and the matching x
// values, eight neighbours at a time.
//
// What bounds it, on B200: not the bytes. Device time, bf16: 1 token 4096 -> 4096 5.6 us (8.4 MB, 1.3 us at the copy rate),
// 8192 -> 16384 21 us = 3.3 TB/s (50 % of the copy rate); 16 tokens 38 us with zero points, 36 without. A warp spends 160
// to 230 instructions on the 2048 weights of a step and tile where 88 unpack them, at 0.5 instructions a cycle. Three blocks
// an SM in place of two (80 registers) took 55 us for 16 tokens of 8192 -> 16384 and 35 for one.
#include "common.cuh"

#include <type_traits>

namespace snnb {
namespace {

struct W4Args {
  const void *x, *scales, *bias;
  const uint8_t *q, *zeros;
  void *y;
  int64_t xs, ys, M;
  int K, N, groups;
  int x16;      // x may be read 16 bytes at a time
};

template <typename T> struct Half16 { using type = T; };
template <> struct Half16<float> { using type = __nv_bfloat16; };      // fp32 tokens: three bf16 pieces, see pieces_of

// Two weights as two 16-bit floats, the well-known way by the bits of a larger number: magic + q has q in its lowest bits
// (1024 + q in fp16, 128 + q in bf16), and subtracting magic + zero is exact.
template <typename H> __device__ __forceinline__ uint32_t magic() { return std::is_same_v<H, __half> ? 0x64006400u : 0x43004300u; }
template <typename H> __device__ __forceinline__ uint32_t minus(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same_v<H, __half>) asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// (a & b) | c in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// Weights (0, 4), (1, 5), (2, 6), (3, 7) of the eight in w, less their zero point; zero: magic + zero, and for fp16, where
// the nibbles at bits 4 .. 7 stay there (1024 + 16 q, times 1/16), 64 + zero.
template <typename H> __device__ __forceinline__ void unpack8(uint32_t w, const uint32_t (&zero)[2], uint32_t (&p)[4]) {
  if constexpr (std::is_same_v<H, __half>) {
    const uint32_t w8 = w >> 8;
    p[0] = minus<H>(and_or(w, 0x000f000fu, magic<H>()), zero[0]);
    p[2] = minus<H>(and_or(w8, 0x000f000fu, magic<H>()), zero[0]);
    const uint32_t a = and_or(w, 0x00f000f0u, magic<H>()), b = and_or(w8, 0x00f000f0u, magic<H>());
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(p[1]) : "r"(a), "r"(0x2c002c00u), "r"(zero[1]));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(p[3]) : "r"(b), "r"(0x2c002c00u), "r"(zero[1]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = minus<H>(and_or(w >> (4 * i), 0x000f000fu, magic<H>()), zero[0]);
  }
}
// The two constants of unpack8 for a zero point (ZERO: any may come, else it is 8). Beyond 127, magic + zero is no bf16 number
// any more: the byte's sign, copied beside it, then makes it infinite or NaN, and with it the products, rather than wrong.
template <typename H, bool ZERO> __device__ __forceinline__ void zeros_of(uint32_t z, uint32_t (&zero)[2]) {
  if constexpr (ZERO && !std::is_same_v<H, __half>) {
    asm("prmt.b32 %0, %1, 0, 0x8080;" : "=r"(zero[0]) : "r"(z));
    zero[0] |= magic<H>();
  } else {
    zero[0] = magic<H>() + 0x00010001u * z;
  }
  if constexpr (std::is_same_v<H, __half>) {      // -(64 + z): 64 .. 127 have steps of 1/16 in fp16, beyond that of 1/8
    const __half2 v = __half2half2(__int2half_rn(-64 - (int)z));
    zero[1] = *reinterpret_cast<const uint32_t *>(&v);
  } else {
    zero[1] = 0;
  }
}

template <typename H>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<H, __half>)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int BYTES> __device__ __forceinline__ void load_words(const uint8_t *p, uint32_t *w) {
  if constexpr (BYTES == 16)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
  else if constexpr (BYTES == 8)
    asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  else
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
}

constexpr int kXPad = 32;              // bytes between the columns of x in shared memory

// Columns of x: a 16-bit token each, or for an fp32 token three, the bf16 pieces that it is the sum of (eight bits each, cut
// off, not rounded, so that none overflows).
template <typename T> constexpr int kPieces = sizeof(T) == 4 ? 3 : 1;

// Copies the columns' values k0 .. k0 + len - 1 (a multiple of 1024; zeros from K on) into shared memory, `pitch` bytes
// apart. 128 threads take a token, each 16 bytes of every 1024 values.
template <typename T, int THREADS>
__device__ __forceinline__ void fill_x(const W4Args &a, int64_t m0, int tokens, int k0, int len, unsigned char *to, int pitch) {
  constexpr int PARTS = THREADS / 128;
  const int u = threadIdx.x % 128, first = threadIdx.x / 128;
  if (first >= tokens) {
    asm volatile("cp.async.commit_group;" ::: "memory");
    return;
  }
  for (int at = u * 8; at < len; at += 1024) {
    const int k = k0 + at;
    const bool in = k < a.K;
    unsigned char *dst = to + at * 2 + first * kPieces<T> * pitch;
    const T *src = static_cast<const T *>(a.x) + (m0 + first) * a.xs + k;
    for (int tok = first; tok < tokens; tok += PARTS, dst += PARTS * kPieces<T> * pitch, src += PARTS * a.xs) {
      if constexpr (sizeof(T) == 2) {
        if (a.x16 && in) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
        } else {
          uint4 v = {};
          if (in) {
            const unsigned short *h = reinterpret_cast<const unsigned short *>(src);
            v = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
          }
          *reinterpret_cast<uint4 *>(dst) = v;
        }
      } else {
        uint32_t b[3][4];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = in ? src[e] : 0.f;
          const float hi = __uint_as_float(__float_as_uint(f) & 0xffff0000u), r1 = f == hi ? 0.f : f - hi;      // also of infinities
          const float mid = __uint_as_float(__float_as_uint(r1) & 0xffff0000u);
          const float part[3] = {hi, mid, r1 - mid};
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            const uint32_t v = __float_as_uint(part[p]) >> 16;
            b[p][e / 2] = e % 2 ? b[p][e / 2] | v << 16 : v;
          }
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4 *>(dst + p * pitch) = make_uint4(b[p][0], b[p][1], b[p][2], b[p][3]);
      }
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

// Scale and zero point (ZERO: there are any, else it is 8) of a group. With several groups in a step each is loaded by one
// of the four lanes of a row and handed to all of them when it is used.
template <typename T, bool ZERO, bool SHARED> struct Scales {
  static constexpr bool WIDE = sizeof(T) == 4;
  using Raw = std::conditional_t<WIDE, float, unsigned short>;
  Raw s;
  uint8_t z;
  __device__ __forceinline__ void load(const T *scales, const uint8_t *zeros, uint32_t at) {
    s = __ldg(reinterpret_cast<const Raw *>(scales) + at);
    if constexpr (ZERO) z = __ldg(zeros + at);
  }
  __device__ __forceinline__ void get(int src, float &scale, uint32_t &zero) const {
    uint32_t v = (uint32_t)(ZERO ? z : 8), r = 0;
    if constexpr (WIDE) {
      scale = SHARED ? __shfl_sync(0xffffffffu, s, src) : s;
      zero = SHARED && ZERO ? __shfl_sync(0xffffffffu, v, src) : v;
    } else {
      if constexpr (SHARED && ZERO) {      // both in one word
        r = __shfl_sync(0xffffffffu, (uint32_t)s << 16 | v, src);
        v = r & 0xffffu;
        r >>= 16;
      } else {
        r = SHARED ? __shfl_sync(0xffffffffu, (uint32_t)s, src) : s;
      }
      if constexpr (std::is_same_v<T, __half>) scale = __half2float(__ushort_as_half((unsigned short)r));
      else scale = __uint_as_float(r << 16);
      zero = v;
    }
  }
};

// The kWarps warps of a block share its rows and take the steps of 128 values along K in turn. RT tiles of 16 rows and NT
// tiles of 8 columns a warp; DEPTH steps of weights on their way in registers. x passes through shared memory in chunks of
// `spc` steps a warp, the next chunk copied while one is worked on.
constexpr int kWarps = 8;

template <typename T, bool ZERO, int G, int NT, int RT, int DEPTH>
__global__ void __launch_bounds__(kWarps * 32) linear_w4_kernel(const __grid_constant__ W4Args a, int spc) {
  using H = typename Half16<T>::type;
  constexpr int PIECES = kPieces<T>, TOKENS = 8 * NT / PIECES, SUB = 128 / G, WORDS = G / 32;
  constexpr int ROWS = 16 * RT, COLS = 8 * NT, RPITCH = COLS + 2;
  extern __shared__ __align__(16) unsigned char dyn[];
  const int lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x / 32), 0);      // the same for all lanes, and known to be
  const int n0 = blockIdx.x * ROWS;
  const int64_t m0 = (int64_t)blockIdx.y * TOKENS;
  const int tokens = (int)min((int64_t)TOKENS, a.M - m0), cols = tokens * PIECES;
  const int iters = (a.K + kWarps * 128 - 1) / (kWarps * 128);
  const int len = spc * kWarps * 128, pitch = len * 2 + kXPad, buffer = cols * pitch;

  // Offsets of the lane's rows in the weights and in the scales; where a step lies within a row is the same for all lanes.
  uint32_t wrow[RT][2], srow[RT][2];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t n = min(n0 + t * 16 + g + 8 * r, a.N - 1);      // rows behind the last one are computed and dropped
      wrow[t][r] = n * (uint32_t)(a.K / 2) + c * (G / 8);
      srow[t][r] = n * (uint32_t)a.groups + c % SUB;
    }
  uint32_t w[DEPTH][RT][2][4];
  Scales<T, ZERO, (SUB > 1)> sc[DEPTH][RT][2];
  int ahead = warp;      // the step that is fetched next
  auto fetch = [&](int slot) {
    const int k = ahead * 128;
    const uint8_t *wp = a.q + k / 2, *zp = a.zeros + ahead * SUB;
    const T *sp = static_cast<const T *>(a.scales) + ahead * SUB;
    if (k + 128 <= a.K) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int h = 0; h < SUB; ++h) load_words<G / 8>(wp + h * (G / 2) + wrow[t][r], &w[slot][t][r][h * WORDS]);
          sc[slot][t][r].load(sp, zp, srow[t][r]);
        }
    } else if (k < a.K) {      // the last step of a row, part of it behind the end: any weight will do, x is zero there
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int h = 0; h < SUB; ++h) {
            if (k + h * G + c * (G / 4) < a.K) load_words<G / 8>(wp + h * (G / 2) + wrow[t][r], &w[slot][t][r][h * WORDS]);
            else
#pragma unroll
              for (int i = 0; i < WORDS; ++i) w[slot][t][r][h * WORDS + i] = 0;
          }
          sc[slot][t][r] = {};
          if (k + c % SUB * G < a.K) sc[slot][t][r].load(sp, zp, srow[t][r]);
        }
    }
    ahead += kWarps;
  };
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) fetch(i);
  fill_x<T, kWarps * 32>(a, m0, tokens, 0, len, dyn, pitch);

  const unsigned char *xcol[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j)      // a column that does not exist repeats the last one and is dropped
    xcol[j] = dyn + min(j * 8 + g, cols - 1) * pitch + warp * 256 + c * WORDS * 16;
  float acc[RT][NT][4] = {};
  int in_chunk = 0, chunk = 0, it = 0, off = 0;
  while (it < iters) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i, ++it) {
      if (it >= iters) break;
      if (in_chunk == 0) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();      // the chunk is there, and nobody reads the one before it any more
        off = (chunk & 1) * buffer;
        ++chunk;
        if (chunk * spc < iters) fill_x<T, kWarps * 32>(a, m0, tokens, chunk * len, len, dyn + (chunk & 1) * buffer, pitch);
        in_chunk = spc;
      }
      --in_chunk;
      if ((it * kWarps + warp) * 128 < a.K) {
#pragma unroll
        for (int h = 0; h < SUB; ++h) {
          float scale[RT][2], part[RT][NT][4] = {};
          uint32_t zero[RT][2][2];
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              uint32_t z;
              sc[i][t][r].get((lane & ~3) | h, scale[t][r], z);
              zeros_of<H, ZERO>(z, zero[t][r]);
            }
#pragma unroll
          for (int v = 0; v < WORDS; ++v) {
            uint32_t b[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const uint4 x = *reinterpret_cast<const uint4 *>(xcol[j] + off + h * (G * 2) + v * 16);
              b[j][0] = __byte_perm(x.x, x.z, 0x5410);
              b[j][1] = __byte_perm(x.x, x.z, 0x7632);
              b[j][2] = __byte_perm(x.y, x.w, 0x5410);
              b[j][3] = __byte_perm(x.y, x.w, 0x7632);
            }
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              uint32_t lo[4], hi[4];
              unpack8<H>(w[i][t][0][h * WORDS + v], zero[t][0], lo);
              unpack8<H>(w[i][t][1][h * WORDS + v], zero[t][1], hi);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                mma16816<H>(part[t][j], lo[0], hi[0], lo[1], hi[1], b[j][0], b[j][1]);
                mma16816<H>(part[t][j], lo[2], hi[2], lo[3], hi[3], b[j][2], b[j][3]);
              }
            }
          }
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int k = 0; k < 4; ++k) acc[t][j][k] = fmaf(scale[t][k / 2], part[t][j][k], acc[t][j][k]);
        }
        fetch(i);
      }
      off += kWarps * 256;
    }
  }
  __syncthreads();      // x is not needed any more: its place takes the warps' sums
  float *red = reinterpret_cast<float *>(dyn);      // [kWarps][ROWS][RPITCH]
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        *reinterpret_cast<float2 *>(&red[(warp * ROWS + t * 16 + g + 8 * r) * RPITCH + j * 8 + 2 * c]) =
            make_float2(acc[t][j][2 * r], acc[t][j][2 * r + 1]);
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * tokens; i += kWarps * 32) {
    const int row = i % ROWS, tok = i / ROWS, n = n0 + row;
    if (n >= a.N) continue;
    float s = 0.f;
#pragma unroll
    for (int p = PIECES - 1; p >= 0; --p)      // the small pieces first
#pragma unroll
      for (int k = 0; k < kWarps; ++k) s += red[(k * ROWS + row) * RPITCH + tok * PIECES + p];
    if (a.bias) s += DT<T>::to_f(static_cast<const T *>(a.bias)[n]);
    static_cast<T *>(a.y)[(m0 + tok) * a.ys + n] = DT<T>::from_f(s);
  }
}

template <typename T, bool ZERO, int G, int NT, int RT, int DEPTH> int go(const W4Args &a, cudaStream_t s) {
  constexpr int TOKENS = 8 * NT / kPieces<T>;
  const dim3 grid((unsigned)((a.N + 16 * RT - 1) / (16 * RT)), (unsigned)((a.M + TOKENS - 1) / TOKENS));
  // all of x at once if that is at most 64 KB, else two chunks of one step a warp
  const int cols = (int)(a.M < TOKENS ? a.M : TOKENS) * kPieces<T>, iters = (a.K + kWarps * 128 - 1) / (kWarps * 128);
  int spc = iters, buffers = 1;
  auto bytes = [&](int n) { return cols * (n * kWarps * 256 + kXPad); };
  if (iters > 64 || bytes(iters) > 64 * 1024) { spc = 1; buffers = 2; }
  const int red = kWarps * 16 * RT * (8 * NT + 2) * (int)sizeof(float);
  const int smem = buffers * bytes(spc) > red ? buffers * bytes(spc) : red;
  constexpr auto kern = linear_w4_kernel<T, ZERO, G, NT, RT, DEPTH>;
  cudaError_t e = raise_smem_limit_once<kern>(160 * 1024);
  if (e == cudaSuccess) {
    kern<<<grid, kWarps * 32, smem, s>>>(a, spc);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return fail(SNNB_ERR_CUDA, "linear_w4: launch failed: %s", cudaGetErrorString(e));
  return SNNB_OK;
}

// Rows a warp and steps ahead: device time on B200 in us for (RT, DEPTH) = (1, 4) (2, 2) (2, 1) (4, 1), groups of 128, bf16;
// in brackets the tiles of 16 rows.
//   1 token    4096 -> 2368 (148)   4.2  5.9  6.2  8.2      4096 -> 12288 (768)   12.4 12.7 10.2 11.6
//              4096 -> 4096 (256)   5.6  6.3  6.4  8.5      4096 -> 13312 (832)   12.7 12.8 10.3 11.7
//              4096 -> 4736 (296)   5.7  6.5  6.6  8.6      4096 -> 14336 (896)   14.6 14.2 13.7 11.8
//              4096 -> 5120 (320)   7.2  7.4  7.3  8.7      4096 -> 16384 (1024)  14.9 14.7 14.1 11.9
//              4096 -> 8192 (512)   9.8  8.3  8.1  9.6      8192 -> 16384 (1024)  28.7 24.8 24.5 21.0
//   fp32       4096 -> 4096 (256)   7.6  8.0  8.1 10.1      4096 -> 16384 (1024)  23.8 17.5 17.6 14.0
//   8 tokens   8192 -> 8192 (512)  21.5 15.2 15.3 16.7      4096 -> 12288 (768)   16.3 14.2 12.6 13.7
//   16 tokens  4096 -> 4096 (256)   9.2  7.9  8.3 10.8      8192 -> 16384 (1024)  50.3 35.7 35.7 36.8
// and with (RT, DEPTH) = (2, 2) (2, 1) (4, 1), 32 tokens 8192 -> 8192 37 38 27, 64 tokens 4096 -> 8192 40 41 29.
// More rows a warp share what a step costs beside the weights; fewer blocks than twice the SMs cost more than that. With two
// tiles a block three blocks run on an SM (65 registers; 111 and two blocks with two steps ahead), so that up to six tiles an
// SM are one wave.
template <typename T, bool ZERO, int G> int by_tokens(const W4Args &a, cudaStream_t s) {
  const int cols = (int)(a.M < 64 ? a.M : 64) * kPieces<T>, tiles = (a.N + 15) / 16, sms = sm_count() > 0 ? sm_count() : 148;
  if (cols > 16) return go<T, ZERO, G, 4, 4, 1>(a, s);
  if (cols > 8) return go<T, ZERO, G, 2, 2, 1>(a, s);
  if (tiles <= 2 * sms) return go<T, ZERO, G, 1, 1, 4>(a, s);
  if (tiles < 6 * sms) return go<T, ZERO, G, 1, 2, 1>(a, s);
  return go<T, ZERO, G, 1, 4, 1>(a, s);
}

template <typename T, bool ZERO> int by_group(const W4Args &a, int G, cudaStream_t s) {
  if (G == 128) return by_tokens<T, ZERO, 128>(a, s);
  if (G == 64) return by_tokens<T, ZERO, 64>(a, s);
  return by_tokens<T, ZERO, 32>(a, s);
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
  SNNB_CHECK_ARG(K <= (1 << 30) && (int64_t)N * K < (1LL << 33) && M <= 65535 * 2, "linear_w4: problem too large");
  if (M == 0) return SNNB_OK;
  SNNB_CHECK_ARG(x && q_weight && scales && y, "linear_w4: null pointer");
  SNNB_CHECK_ARG(x_stride >= 0 && (M <= 1 || y_stride >= N), "linear_w4: bad row stride");
  SNNB_CHECK_ARG(y != x, "linear_w4: y is x");
  SNNB_CHECK_ARG(aligned16(q_weight), "linear_w4: q_weight must be 16-byte aligned");
  W4Args a;
  a.x = x; a.scales = scales; a.bias = bias; a.q = static_cast<const uint8_t *>(q_weight);
  a.zeros = static_cast<const uint8_t *>(zeros); a.y = y; a.xs = x_stride; a.ys = y_stride; a.M = M;
  a.K = K; a.N = N; a.groups = (K + group_size - 1) / group_size;
  a.x16 = aligned16(x) && x_stride % (16 / dtype_size(dtype)) == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SNNB_F32: return zeros ? by_group<float, true>(a, group_size, s) : by_group<float, false>(a, group_size, s);
    case SNNB_BF16: return zeros ? by_group<__nv_bfloat16, true>(a, group_size, s) : by_group<__nv_bfloat16, false>(a, group_size, s);
    default: return zeros ? by_group<__half, true>(a, group_size, s) : by_group<__half, false>(a, group_size, s);
  }
}
