// Gated scan kernels for one activation type (see gated_scan_impl.cuh).
#include "gated_scan_impl.cuh"

namespace snnb {
template int gated_scan_launch<float>(ScanArgs, bool, int, bool, cudaStream_t);
int gated_scan_status_f32(int *out) { return scan_unit_status(out); }
}  // namespace snnb
