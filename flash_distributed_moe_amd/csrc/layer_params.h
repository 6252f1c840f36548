// What the host code and the kernels of the operators around a layer's blocks share: the router's choice with its
// losses, the norms before and after a block, the adapters beside a projection.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>

namespace fmoe {

// ------------------------------------------------------------------ the router's choice
struct RouteArgs {
  const void* logits;         // [T, E], rows ld elements apart
  const unsigned char* mask;  // [T], 0: padding; NULL: none is
  long long ld;
  int T, E, k, renormalize;
  float* weights;   // [T, k]
  int* experts;     // [T, k]
  int* counts;      // [E]
  int* totals;      // [2]: rows with a candidate, slots filled
  float* balance;   // [1]
  float* zed;       // [1]
  float* partial;   // of more than one workgroup: [blocks, kRouteColumns] sums of probabilities, then as many counts
  // backward
  const float* dweights;  // [T, k] or NULL
  const float* dbalance;  // [1] or NULL
  const float* dzed;      // [1] or NULL
  void* dlogits;          // [T, E], rows ldd elements apart
  long long ldd;
};
constexpr int kRouteExperts = 256, kRouteTopK = 32;
constexpr int kRouteColumns = kRouteExperts + 1;  // a last one for the squared logsumexps, and of the counts for the rows
// Workgroups of a forward pass. One alone finishes by itself, which saves the second launch. At most one a CU, so that
// the one workgroup that joins their sums reads no more than half a MiB.
struct RouteGrid {
  int blocks, threads;
};
inline RouteGrid route_grid(int T) {
  const int threads = T <= 64 || T > 4096 ? 1024 : 256, rows = threads / 16;
  const long long blocks = (T + rows - 1LL) / rows;
  return {static_cast<int>(blocks < 1 ? 1 : blocks < 256 ? blocks : 256), threads};
}
hipError_t launch_route(const RouteArgs& a, int dtype, hipStream_t stream);
hipError_t launch_route_backward(const RouteArgs& a, int dtype, hipStream_t stream);

}  // namespace fmoe
