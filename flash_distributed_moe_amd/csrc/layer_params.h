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
  float* weights;   // [T, k]; read by the backward pass
  int* experts;     // [T, k]
  int* counts;      // [E]
  int* kept;        // [2 + E], for the backward pass: rows with a candidate, slots filled, the counts once more; NULL: not wanted
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
// Workgroups of a forward pass. One alone finishes by itself, which saves the second launch (64 tokens 7.3 us, in four workgroups 8.2).
// At most one a CU, so that the one workgroup that joins their sums reads no more than 514 KiB. With 256 and 1024 threads each, us with the
// joining in a replayed graph: float32 E=128, k=8 4099 tokens 13.8 and 12.1, 8192 16.0 and 13.2, 16384 21.3 and 15.9; bfloat16 E=60, k=4 4099
// tokens 11.2 and 8.7, 8192 11.8 and 9.6, 12000 13.1 and 14.0, 16384 14.4 and 11.9. More threads leave fewer sums to join, fewer
// deal the tokens out more evenly. The border was set by the tokens' kernels alone (E=60, 4099 tokens 4.9 and 5.7 without joining);
// of whole calls 1024 threads are ahead below it as well (E=128, 1000 tokens 13.5 and 11.8).
struct RouteGrid {
  int blocks, threads;
};
inline RouteGrid route_grid(int T) {
  // one workgroup has a wave for four tokens, and a thread for every expert
  const int threads = T <= 16 ? 256 : T <= 64 ? (T + 3) / 4 * 64 : T > 6000 ? 1024 : 256, rows = threads / 16;
  const long long blocks = (T + rows - 1LL) / rows;
  return {static_cast<int>(blocks < 1 ? 1 : blocks < 256 ? blocks : 256), threads};
}
hipError_t launch_route(const RouteArgs& a, int dtype, hipStream_t stream);
hipError_t launch_route_backward(const RouteArgs& a, int dtype, hipStream_t stream);

// ------------------------------------------------------------------ the norms around a block
enum GateKind { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_GROUP = 2, GATE_TOKEN = 3, GATE_FULL = 4 };

struct NormArgs {
  const void* x;       // [T, H]
  const void* branch;  // [T, H], or NULL: the norm in front of a block alone, y = x
  const void* post;    // [H] or NULL
  const void* gate;    // by kind: [H], [T / shared, H], [T] or [T, H]
  const void* next;    // [H] or NULL
  void* y;             // [T, H] or NULL
  void* h;             // [T, H] if next
  float* branch_rms;   // [T]: one over the root mean square of the branch's rows and of y's; NULL: not kept
  float* y_rms;        // [T]
  long long ldx, ldb;
  int T, H, gate_kind;
  int shared;  // rows that share a gate row (GATE_GROUP)
  float alpha, beta, eps;
  // backward
  const void* dy;  // [T, H] or NULL
  const void* dh;  // [T, H] or NULL
  long long lddy, lddh;
  void *dx, *dbranch, *dpost, *dgate, *dnext;  // without gaps, or NULL
  float* partial;                              // [arrays, blocks, H]
  // GATE_GROUP: `parts` workgroups take a group's rows each, or one takes `groups` groups
  int blocks, parts, groups;
};
constexpr int kNormWidth = 8192;
constexpr int kNormLane = 16;  // backward: values a lane has of a row
// Waves that have a row together in the backward pass.
__host__ __device__ inline int norm_waves(int H) { return H <= 1024 ? 1 : H <= 2048 ? 2 : H <= 4096 ? 4 : 8; }
__host__ __device__ inline int norm_threads(int H) { return norm_waves(H) == 8 ? 512 : 256; }
// Workgroups of the backward pass, and which rows they take: two a CU, since each leaves column sums that are read again (8192 x 4096 in
// bfloat16 with 384, 512, 768 and 1024 of them 84, 81, 86 and 89 us).
inline void plan_norm_backward(NormArgs& a) {
  const int at_once = norm_threads(a.H) / 64 / norm_waves(a.H);
  const long long most = 512, steps = (a.T + at_once - 1LL) / at_once;
  a.blocks = static_cast<int>(steps < 1 ? 1 : steps < most ? steps : most);
  a.parts = 0, a.groups = 1;
  if (a.gate_kind != GATE_GROUP || a.T == 0) return;
  const int count = a.T / a.shared;
  const long long rows = (a.T + a.blocks - 1LL) / a.blocks;  // a workgroup's
  if (a.shared > rows) {
    a.parts = static_cast<int>((a.shared + rows - 1) / rows);
    a.blocks = count * a.parts;
  } else {
    a.groups = static_cast<int>((rows + a.shared - 1) / a.shared);
    a.blocks = (count + a.groups - 1) / a.groups;
  }
}
// Column sums that the workgroups leave: of the next norm's weight, of the post norm's (with a gate a channel: of both), of a group's gate.
inline int norm_arrays(const NormArgs& a) { return a.gate_kind == GATE_GROUP ? 3 : 2; }
hipError_t launch_norm(const NormArgs& a, int dtype, hipStream_t stream);
hipError_t launch_norm_backward(const NormArgs& a, int dtype, hipStream_t stream);

// ------------------------------------------------------------------ adapters beside a projection
struct AdapterArgs {
  const void* x;        // [T, K], rows ldx values apart
  const void* y;        // [T, N]
  void* out;            // [T, N]; may be y
  const int* ids;       // [T]: a row's adapter, negative: none
  const void* down;     // [adapters, r, K]
  const void* up;       // [adapters, N, r]
  const float* scales;  // [adapters]
  long long ldx, ldy, ldo;
  int T, K, N, r, adapters;
  float* u;    // x A^T: [splits, T, r]; of few rows scaled, of many by place in `order`
  int* order;  // [T]: rows by adapter
  int* tiles;  // [tiles + 1, 4]: adapter, first place, rows; the last one's first value is their number
  int most_tiles, tile_rows, splits;
};
constexpr int kAdapterRank = 128, kAdapters = 1000;
// Few rows: every row reads its adapter by itself, which costs as much for each of them; tiles cost three kernels, the more the higher
// the rank, before the number of rows is felt. us by rows and in tiles, K=N=4096: rank 8, 768 rows 15 and 19, 1024 17 and 21; rank 16, 512 rows
// 17 and 18, 768 22 and 20; rank 64, 256 rows 26 and 28, 384 38 and 28; rank 128, 256 rows 50 and 63, 384 72 and 55. How many adapters
// the rows have between them is not asked: it is on the device, and the number of adapters that are kept says little of it.
__host__ __device__ inline bool adapter_rows_alone(const AdapterArgs& a) {
  return a.T <= 4096 && static_cast<long long>(a.T) * a.r * (static_cast<long long>(a.K) + a.N) <= 56000000ll + 1400000ll * a.r;
}
// Many: tiles of 16 or 64 rows of one adapter, whose k several workgroups share while there are few of them.
inline void plan_adapters(AdapterArgs& a) {
  if (adapter_rows_alone(a)) {
    a.splits = 1;
    return;
  }
  // Tiles of 64 read B and A less often and fill slower: with 16 and 64 rows, K=N=4096, rank 16, 1024 rows 22 and 23 us, 2048 30 and 27; rank
  // 64, 512 rows 24 and 30, 1024 35 and 31; of 200 adapters (N=12288) 1024 rows 125 and 137, 4096 197 and 165.
  a.tile_rows = a.T >= 768 && static_cast<long long>(a.T) * (a.r + 8) >= 28672 && a.T >= 12 * a.adapters ? 64 : 16;
  const long long full = (a.T + a.tile_rows - 1LL) / a.tile_rows;
  // a last tile each, of every adapter, of the rows without one and of those of an adapter that is not there
  a.most_tiles = static_cast<int>(full + (a.adapters + 2 < a.T ? a.adapters + 2 : a.T));
  // (8192 rows, K=4096, rank 64 with 1, 2 and 4 workgroups a tile of 64: 36, 23 and 23 to 28 us, and their sums are read again for every
  // few columns)
  const long long some = a.tile_rows == 64 ? 256 : 128, wanted = (some + full - 1) / full, most = (a.K + 511) / 512;
  a.splits = static_cast<int>(wanted < most ? wanted : most);
}
struct AdapterBytes {
  size_t u, order, tiles;
  size_t all() const { return u + order + tiles; }
};
inline AdapterBytes adapter_bytes(const AdapterArgs& a) {
  const auto whole = [](size_t v) { return (v + 255) / 256 * 256; };
  AdapterBytes b{whole(size_t(a.splits) * a.T * a.r * 4), 0, 0};
  if (!adapter_rows_alone(a)) b.order = whole(size_t(a.T) * 4), b.tiles = whole((size_t(a.most_tiles) + 1) * 16);
  return b;
}
hipError_t launch_adapters(const AdapterArgs& a, hipStream_t stream);

}  // namespace fmoe
