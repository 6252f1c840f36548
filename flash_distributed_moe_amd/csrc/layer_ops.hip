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
                  float* weights, int* experts, int* counts, int* totals, float* balance, float* zed, void* workspace,
                  void* stream) {
  FMOE_HIP_CHECK(validate(desc, tokens));
  FMOE_HIP_CHECK(check_word("counts", counts));
  FMOE_HIP_CHECK(check_word("totals", totals));
  FMOE_HIP_CHECK(check_word("balance", balance));
  FMOE_HIP_CHECK(check_word("zed", zed));
  if (tokens > 0) {
    FMOE_HIP_CHECK(check_logits("logits", logits, ld, desc));
    FMOE_HIP_CHECK(check_word("weights", weights));
    FMOE_HIP_CHECK(check_word("experts", experts));
    if (fmoe::route_grid(tokens).blocks > 1) FMOE_HIP_CHECK(check_word("workspace", workspace));
  }
  fmoe::RouteArgs a = route_args(desc, logits, ld, mask, tokens);
  a.weights = weights, a.experts = experts, a.counts = counts, a.totals = totals, a.balance = balance, a.zed = zed;
  a.partial = static_cast<float*>(workspace);
  FMOE_HIP_CHECK(fmoe::launch_route(a, desc->dtype, static_cast<hipStream_t>(stream)));
  return hipSuccess;
}

int flashMoeRouteBackward(const FlashMoeRouteDesc* desc, const void* logits, long long ld, const unsigned char* mask, int tokens,
                          const int* experts, const int* counts, const int* totals, const float* dweights,
                          const float* dbalance, const float* dzed, void* dlogits, long long ldd, void* stream) {
  FMOE_HIP_CHECK(validate(desc, tokens));
  if (tokens == 0) return hipSuccess;
  FMOE_HIP_CHECK(check_logits("logits", logits, ld, desc));
  FMOE_HIP_CHECK(check_logits("dlogits", dlogits, ldd, desc));
  FMOE_HIP_CHECK(check_word("experts", experts));
  FMOE_HIP_CHECK(check_word("counts", counts));
  FMOE_HIP_CHECK(check_word("totals", totals));
  for (const void* p : {static_cast<const void*>(dweights), static_cast<const void*>(dbalance), static_cast<const void*>(dzed)})
    if (!on(p, 4)) FMOE_FAIL(hipErrorInvalidValue, "a gradient does not begin on 4 bytes");
  fmoe::RouteArgs a = route_args(desc, logits, ld, mask, tokens);
  a.experts = const_cast<int*>(experts), a.counts = const_cast<int*>(counts), a.totals = const_cast<int*>(totals);
  a.dweights = dweights, a.dbalance = dbalance, a.dzed = dzed, a.dlogits = dlogits, a.ldd = ldd;
  FMOE_HIP_CHECK(fmoe::launch_route_backward(a, desc->dtype, static_cast<hipStream_t>(stream)));
  return hipSuccess;
}

}  // extern "C"
