// C ABI of the operators around a layer's blocks (include/flash_moe.h): checks of the arguments and workspace sizes.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "../../include/flash_moe.h"
#include "layer_params.h"

#define FMOE_FILENAME (strrchr(__FILE__, '/') ? strrchr(__FILE__, '/') + 1 : __FILE__)

// As the launcher's: print to stdout, return the first failing code.
#define FMOE_HIP_CHECK(expr)                                               \
  do {                                                                     \
    const hipError_t fmoe_err_ = (expr);                                   \
    if (fmoe_err_ != hipSuccess) {                                         \
      printf("[MOE HIP ERROR: %s:%i]: %s\n", FMOE_FILENAME, __LINE__,      \
             hipGetErrorString(fmoe_err_));                                \
      fflush(stdout);                                                      \
      return fmoe_err_;                                                    \
    }                                                                      \
  } while (0)

#define FMOE_FAIL(code, fmt, ...)                                                      \
  do {                                                                                 \
    printf("[MOE ERROR: %s:%i]: " fmt "\n", FMOE_FILENAME, __LINE__, ##__VA_ARGS__);   \
    fflush(stdout);                                                                    \
    return (code);                                                                     \
  } while (0)

namespace {

constexpr long long kMaxStride = 1ll << 20;
bool on(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
size_t size_of(int dtype) { return dtype == FLASH_MOE_F32 ? 4 : 2; }

hipError_t check_dtype(int dtype) {
  if (dtype != FLASH_MOE_F32 && dtype != FLASH_MOE_BF16)
    FMOE_FAIL(hipErrorInvalidValue, "dtype %i is neither float32 (0) nor bfloat16 (1)", dtype);
  return hipSuccess;
}

hipError_t validate(const FlashMoeRouteDesc* d, int tokens) {
  if (d == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null description");
  FMOE_HIP_CHECK(check_dtype(d->dtype));
  if (d->experts < 1 || d->experts > fmoe::kRouteExperts || d->top_k < 1 || d->top_k > fmoe::kRouteTopK || d->top_k > d->experts)
    FMOE_FAIL(hipErrorInvalidValue, "E=%i, top_k=%i: E up to %i, top_k up to min(E, %i)", d->experts, d->top_k,
              fmoe::kRouteExperts, fmoe::kRouteTopK);
  // the slots are counted in 32 bits
  if (tokens < 0 || tokens > (1 << 30) / d->top_k)
    FMOE_FAIL(hipErrorInvalidValue, "%i tokens of %i slots (at most 2^30 slots)", tokens, d->top_k);
  return hipSuccess;
}
hipError_t check_logits(const char* name, const void* p, long long ld, const FlashMoeRouteDesc* d) {
  if (p == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null %s pointer", name);
  if (!on(p, size_of(d->dtype))) FMOE_FAIL(hipErrorInvalidValue, "%s does not begin on a value", name);
  if (ld < d->experts || ld > kMaxStride)
    FMOE_FAIL(hipErrorInvalidValue, "%s: %lld values from row to row (at least %i, at most %lld)", name, ld, d->experts, kMaxStride);
  return hipSuccess;
}
hipError_t check_word(const char* name, const void* p) {
  if (p == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null %s pointer", name);
  if (!on(p, 4)) FMOE_FAIL(hipErrorInvalidValue, "%s does not begin on 4 bytes", name);
  return hipSuccess;
}

fmoe::RouteArgs route_args(const FlashMoeRouteDesc* d, const void* logits, long long ld, const unsigned char* mask, int tokens) {
  fmoe::RouteArgs a{};
  a.logits = logits, a.ld = ld, a.mask = mask;
  a.T = tokens, a.E = d->experts, a.k = d->top_k, a.renormalize = d->renormalize;
  return a;
}

hipError_t validate(const FlashMoeNormDesc* d, int tokens, bool branch) {
  if (d == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null description");
  FMOE_HIP_CHECK(check_dtype(d->dtype));
  if (d->hidden < 8 || d->hidden > fmoe::kNormWidth || d->hidden % 8 != 0)
    FMOE_FAIL(hipErrorInvalidValue, "H=%i: a multiple of 8, at most %i", d->hidden, fmoe::kNormWidth);
  if (tokens < 0 || tokens > 1 << 30) FMOE_FAIL(hipErrorInvalidValue, "%i tokens (at most 2^30)", tokens);
  if (d->gate < FLASH_MOE_GATE_NONE || d->gate > FLASH_MOE_GATE_FULL)
    FMOE_FAIL(hipErrorInvalidValue, "gate %i is none of FLASH_MOE_GATE_*", d->gate);
  if (d->gate == FLASH_MOE_GATE_GROUP && (d->shared < 1 || tokens % d->shared != 0))
    FMOE_FAIL(hipErrorInvalidValue, "%i tokens in groups of %i", tokens, d->shared);
  if (!(d->eps >= 0)) FMOE_FAIL(hipErrorInvalidValue, "eps is negative or NaN");
  if ((d->gate != FLASH_MOE_GATE_NONE) != (d->gate_values != nullptr))
    FMOE_FAIL(hipErrorInvalidValue, "gate %i %s values", d->gate, d->gate_values != nullptr ? "with" : "without");
  if (!branch && (d->post_weight != nullptr || d->gate != FLASH_MOE_GATE_NONE))
    FMOE_FAIL(hipErrorInvalidValue, "a post norm or a gate without a branch");
  if (!branch && d->next_weight == nullptr) FMOE_FAIL(hipErrorInvalidValue, "neither a branch nor a norm");
  for (const void* p : {d->post_weight, d->next_weight, d->gate == FLASH_MOE_GATE_TOKEN ? nullptr : d->gate_values})
    if (!on(p, 16)) FMOE_FAIL(hipErrorInvalidValue, "a weight or the gate does not begin on 16 bytes");
  if (!on(d->gate_values, size_of(d->dtype))) FMOE_FAIL(hipErrorInvalidValue, "the gate does not begin on a value");
  return hipSuccess;
}
// Rows of H values: where they begin and how far apart they lie.
hipError_t check_rows(const char* name, const void* p, long long ld, const FlashMoeNormDesc* d) {
  if (p == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null %s pointer", name);
  if (!on(p, 16)) FMOE_FAIL(hipErrorInvalidValue, "%s does not begin on 16 bytes", name);
  if (ld < d->hidden || ld > kMaxStride || ld * static_cast<long long>(size_of(d->dtype)) % 16 != 0)
    FMOE_FAIL(hipErrorInvalidValue, "%s: %lld values from row to row (at least %i, at most %lld, whole 16 bytes)", name, ld,
              d->hidden, kMaxStride);
  return hipSuccess;
}

fmoe::NormArgs norm_args(const FlashMoeNormDesc* d, int tokens, bool branch) {
  fmoe::NormArgs a{};
  a.T = tokens, a.H = d->hidden, a.gate_kind = d->gate, a.shared = d->shared;
  // without a branch y = x, whatever the scales are
  a.alpha = branch ? static_cast<float>(d->residual_scale) : 1.0f, a.beta = static_cast<float>(d->branch_scale);
  a.eps = static_cast<float>(d->eps);
  a.post = d->post_weight, a.gate = d->gate_values, a.next = d->next_weight;
  return a;
}
size_t partial_bytes(const fmoe::NormArgs& a) { return size_t(fmoe::norm_arrays(a)) * a.blocks * a.H * 4; }

hipError_t validate(const FlashMoeAdapterDesc* d, int rows) {
  if (d == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null description");
  if (d->adapters < 1 || d->adapters > fmoe::kAdapters || d->rank < 8 || d->rank > fmoe::kAdapterRank || d->rank % 8 != 0)
    FMOE_FAIL(hipErrorInvalidValue, "%i adapters of rank %i: up to %i, ranks multiples of 8 up to %i", d->adapters, d->rank,
              fmoe::kAdapters, fmoe::kAdapterRank);
  for (const int width : {d->n, d->k})
    if (width < 8 || width % 8 != 0 || width > kMaxStride)
      FMOE_FAIL(hipErrorInvalidValue, "n=%i, k=%i: multiples of 8, at most %lld", d->n, d->k, kMaxStride);
  // eight workgroups for each of their tiles are still one launch
  if (rows < 0 || rows > 1 << 26) FMOE_FAIL(hipErrorInvalidValue, "%i rows (at most 2^26)", rows);
  return hipSuccess;
}
hipError_t check_bf16_rows(const char* name, const void* p, long long ld, int width) {
  if (p == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null %s pointer", name);
  if (!on(p, 16)) FMOE_FAIL(hipErrorInvalidValue, "%s does not begin on 16 bytes", name);
  if (ld < width || ld > kMaxStride || ld % 8 != 0)
    FMOE_FAIL(hipErrorInvalidValue, "%s: %lld values from row to row (at least %i, at most %lld, whole 16 bytes)", name, ld, width,
              kMaxStride);
  return hipSuccess;
}
fmoe::AdapterArgs adapter_args(const FlashMoeAdapterDesc* d, int rows) {
  fmoe::AdapterArgs a{};
  a.T = rows, a.K = d->k, a.N = d->n, a.r = d->rank, a.adapters = d->adapters;
  a.down = d->down, a.up = d->up, a.scales = d->scales;
  fmoe::plan_adapters(a);
  return a;
}

}  // namespace

extern "C" {

int flashMoeRouteBytes(const FlashMoeRouteDesc* desc, int tokens, size_t* bytes) {
  FMOE_HIP_CHECK(validate(desc, tokens));
  if (bytes == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null result");
  const int blocks = fmoe::route_grid(tokens).blocks;
  *bytes = blocks > 1 ? size_t(blocks) * 2 * fmoe::kRouteColumns * 4 : 0;
  return hipSuccess;
}

int flashMoeRoute(const FlashMoeRouteDesc* desc, const void* logits, long long ld, const unsigned char* mask, int tokens,
                  float* weights, int* experts, int* counts, float* balance, float* zed, int* kept, void* workspace,
                  void* stream) {
  FMOE_HIP_CHECK(validate(desc, tokens));
  FMOE_HIP_CHECK(check_word("counts", counts));
  if (!on(kept, 4)) FMOE_FAIL(hipErrorInvalidValue, "kept does not begin on 4 bytes");
  FMOE_HIP_CHECK(check_word("balance", balance));
  FMOE_HIP_CHECK(check_word("zed", zed));
  if (tokens > 0) {
    FMOE_HIP_CHECK(check_logits("logits", logits, ld, desc));
    FMOE_HIP_CHECK(check_word("weights", weights));
    FMOE_HIP_CHECK(check_word("experts", experts));
    if (fmoe::route_grid(tokens).blocks > 1) FMOE_HIP_CHECK(check_word("workspace", workspace));
  }
  fmoe::RouteArgs a = route_args(desc, logits, ld, mask, tokens);
  a.weights = weights, a.experts = experts, a.counts = counts, a.kept = kept, a.balance = balance, a.zed = zed;
  a.partial = static_cast<float*>(workspace);
  FMOE_HIP_CHECK(fmoe::launch_route(a, desc->dtype, static_cast<hipStream_t>(stream)));
  return hipSuccess;
}

int flashMoeRouteBackward(const FlashMoeRouteDesc* desc, const void* logits, long long ld, const unsigned char* mask, int tokens,
                          const float* weights, const int* experts, const int* kept, const float* dweights,
                          const float* dbalance, const float* dzed, void* dlogits, long long ldd,
                          void* stream) {
  FMOE_HIP_CHECK(validate(desc, tokens));
  if (tokens == 0) return hipSuccess;
  FMOE_HIP_CHECK(check_logits("logits", logits, ld, desc));
  FMOE_HIP_CHECK(check_logits("dlogits", dlogits, ldd, desc));
  FMOE_HIP_CHECK(check_word("weights", weights));
  FMOE_HIP_CHECK(check_word("experts", experts));
  FMOE_HIP_CHECK(check_word("kept", kept));
  for (const void* p : {static_cast<const void*>(dweights), static_cast<const void*>(dbalance), static_cast<const void*>(dzed)})
    if (!on(p, 4)) FMOE_FAIL(hipErrorInvalidValue, "a gradient does not begin on 4 bytes");
  fmoe::RouteArgs a = route_args(desc, logits, ld, mask, tokens);
  a.weights = const_cast<float*>(weights), a.experts = const_cast<int*>(experts), a.kept = const_cast<int*>(kept);
  a.dweights = dweights, a.dbalance = dbalance, a.dzed = dzed, a.dlogits = dlogits, a.ldd = ldd;
  FMOE_HIP_CHECK(fmoe::launch_route_backward(a, desc->dtype, static_cast<hipStream_t>(stream)));
  return hipSuccess;
}

int flashMoeBlockNormBytes(const FlashMoeNormDesc* desc, int tokens, size_t* bytes) {
  if (bytes == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null result");
  // whether there is a branch is not known here, and of no consequence
  FMOE_HIP_CHECK(validate(desc, tokens, true));
  fmoe::NormArgs a = norm_args(desc, tokens, true);
  fmoe::plan_norm_backward(a);
  *bytes = partial_bytes(a);
  return hipSuccess;
}

int flashMoeBlockNorm(const FlashMoeNormDesc* desc, const void* x, long long ldx, const void* branch, long long ldb, int tokens,
                      void* y, void* h, float* kept, void* stream) {
  FMOE_HIP_CHECK(validate(desc, tokens, branch != nullptr || tokens == 0));
  if (tokens == 0) return hipSuccess;
  FMOE_HIP_CHECK(check_rows("x", x, ldx, desc));
  if (branch != nullptr) {
    FMOE_HIP_CHECK(check_rows("branch", branch, ldb, desc));
    FMOE_HIP_CHECK(check_rows("y", y, desc->hidden, desc));
  } else if (y != nullptr) {
    FMOE_FAIL(hipErrorInvalidValue, "y without a branch");
  }
  if (desc->next_weight != nullptr) FMOE_HIP_CHECK(check_rows("h", h, desc->hidden, desc));
  if (!on(kept, 4)) FMOE_FAIL(hipErrorInvalidValue, "kept does not begin on 4 bytes");
  fmoe::NormArgs a = norm_args(desc, tokens, branch != nullptr);
  a.x = x, a.ldx = ldx, a.branch = branch, a.ldb = ldb, a.y = y, a.h = h;
  if (kept != nullptr) a.branch_rms = kept, a.y_rms = kept + tokens;
  FMOE_HIP_CHECK(fmoe::launch_norm(a, desc->dtype, static_cast<hipStream_t>(stream)));
  return hipSuccess;
}

int flashMoeBlockNormBackward(const FlashMoeNormDesc* desc, const void* x, long long ldx, const void* branch, long long ldb,
                              const void* dy, long long lddy, const void* dh, long long lddh, int tokens, const float* kept,
                              void* workspace, void* dx, void* dbranch, void* dpost, void* dgate, void* dnext, void* stream) {
  FMOE_HIP_CHECK(validate(desc, tokens, branch != nullptr || tokens == 0));
  if (tokens > 0) {
    FMOE_HIP_CHECK(check_rows("x", x, ldx, desc));
    if (branch != nullptr) FMOE_HIP_CHECK(check_rows("branch", branch, ldb, desc));
    if (dy != nullptr) FMOE_HIP_CHECK(check_rows("dy", dy, lddy, desc));
    if (dh != nullptr) FMOE_HIP_CHECK(check_rows("dh", dh, lddh, desc));
    FMOE_HIP_CHECK(check_word("kept", kept));
  }
  if ((dbranch != nullptr && branch == nullptr && tokens > 0) || (dpost != nullptr && desc->post_weight == nullptr) ||
      (dgate != nullptr && desc->gate == FLASH_MOE_GATE_NONE) || (dnext != nullptr && desc->next_weight == nullptr))
    FMOE_FAIL(hipErrorInvalidValue, "a gradient of an input that is not there");
  for (const void* p : {dx, dbranch, desc->gate == FLASH_MOE_GATE_FULL ? dgate : nullptr})
    if (!on(p, 16)) FMOE_FAIL(hipErrorInvalidValue, "a gradient does not begin on 16 bytes");
  for (const void* p : {dpost, dgate, dnext})
    if (!on(p, size_of(desc->dtype))) FMOE_FAIL(hipErrorInvalidValue, "a gradient does not begin on a value");
  const bool columns = dpost != nullptr || dnext != nullptr ||
                       (dgate != nullptr && (desc->gate == FLASH_MOE_GATE_CHANNEL || desc->gate == FLASH_MOE_GATE_GROUP));
  if (columns) FMOE_HIP_CHECK(check_word("workspace", workspace));
  if (!columns && tokens == 0) return hipSuccess;
  fmoe::NormArgs a = norm_args(desc, tokens, branch != nullptr);
  a.x = x, a.ldx = ldx, a.branch = branch, a.ldb = ldb, a.dy = dy, a.lddy = lddy, a.dh = dh, a.lddh = lddh;
  if (tokens > 0) a.branch_rms = const_cast<float*>(kept), a.y_rms = a.branch_rms + tokens;
  a.dx = dx, a.dbranch = dbranch, a.dpost = dpost, a.dgate = dgate, a.dnext = dnext;
  a.partial = static_cast<float*>(workspace);
  fmoe::plan_norm_backward(a);
  FMOE_HIP_CHECK(fmoe::launch_norm_backward(a, desc->dtype, static_cast<hipStream_t>(stream)));
  return hipSuccess;
}

int flashMoeAdapterBytes(const FlashMoeAdapterDesc* desc, int rows, size_t* bytes) {
  FMOE_HIP_CHECK(validate(desc, rows));
  if (bytes == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null result");
  *bytes = rows > 0 ? fmoe::adapter_bytes(adapter_args(desc, rows)).all() : 0;
  return hipSuccess;
}

int flashMoeAdapterAdd(const FlashMoeAdapterDesc* desc, const void* x, long long ldx, const void* y, long long ldy, const int* ids,
                       int rows, void* out, long long ldo, void* workspace, void* stream) {
  FMOE_HIP_CHECK(validate(desc, rows));
  if (rows == 0) return hipSuccess;
  FMOE_HIP_CHECK(check_bf16_rows("x", x, ldx, desc->k));
  FMOE_HIP_CHECK(check_bf16_rows("y", y, ldy, desc->n));
  FMOE_HIP_CHECK(check_bf16_rows("out", out, ldo, desc->n));
  if (out == y && ldo != ldy) FMOE_FAIL(hipErrorInvalidValue, "out is y, but its rows lie otherwise");
  FMOE_HIP_CHECK(check_word("ids", ids));
  FMOE_HIP_CHECK(check_word("scales", desc->scales));
  if (desc->down == nullptr || desc->up == nullptr || !on(desc->down, 16) || !on(desc->up, 16))
    FMOE_FAIL(hipErrorInvalidValue, "adapters are missing or do not begin on 16 bytes");
  if (workspace == nullptr || !on(workspace, 16)) FMOE_FAIL(hipErrorInvalidValue, "the workspace is missing or does not begin on 16 bytes");
  fmoe::AdapterArgs a = adapter_args(desc, rows);
  a.x = x, a.ldx = ldx, a.y = y, a.ldy = ldy, a.ids = ids, a.out = out, a.ldo = ldo;
  const fmoe::AdapterBytes b = fmoe::adapter_bytes(a);
  char* p = static_cast<char*>(workspace);
  a.u = reinterpret_cast<float*>(p);
  a.order = reinterpret_cast<int*>(p + b.u);
  a.tiles = reinterpret_cast<int*>(p + b.u + b.order);
  FMOE_HIP_CHECK(fmoe::launch_adapters(a, static_cast<hipStream_t>(stream)));
  return hipSuccess;
}

}  // extern "C"
