// What the host part of the gated scan (gated_scan.cu) and its kernels (gated_scan_impl.cuh) share.
#pragma once

#include "common.cuh"

namespace snnb {

struct ScanSeq {      // rows of D dense values; element (t, b, d) at t * ts + b * bs + d
  const void *p;
  int64_t ts, bs;
};

struct ScanArgs {
  ScanSeq x, g, h;    // h: the output of the forward pass, the gradient dh of the backward pass
  ScanSeq dx, dg;
  const void *h_init;
  const void *dh_last;
  void *h_last;       // forward: the last state; backward: dh_init
  float *ckpt;
  const int *lengths;
  int64_t T, B, D;
  int state_f32, leaky;
  // filled in by the launch
  int tiles_d;            // channel tiles of a row
  long long wait_limit;   // bound of every wait of a cluster's exchange, in SM cycles (about two seconds unless a self-test shortens it)
  int miss_map;           // self-test: the last block of the first cluster waits for a map that nobody sends
};

void consume_wait_selftest(long long *limit_cycles, int *drop_load);      // conv_pair.cu

// One translation unit per activation type. gate_kind as in the C ABI; aligned: every row starts on a 16-byte boundary
// and ends on one, and so do the states.
template <typename T> int gated_scan_launch(ScanArgs q, bool backward, int gate_kind, bool aligned, cudaStream_t s);
int gated_scan_status_f32(int *out);
int gated_scan_status_bf16(int *out);
int gated_scan_status_f16(int *out);
int gated_scan_device_status(int *out);

extern template int gated_scan_launch<float>(ScanArgs, bool, int, bool, cudaStream_t);
extern template int gated_scan_launch<__nv_bfloat16>(ScanArgs, bool, int, bool, cudaStream_t);
extern template int gated_scan_launch<__half>(ScanArgs, bool, int, bool, cudaStream_t);

}  // namespace snnb
