// C ABI of the dense gated feed-forward block and of MXFP4 (include/flash_moe.h): checks of the
// arguments, workspace layouts, and which kernels a call takes.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "../../include/flash_moe.h"
#include "ffn_params.h"

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

using fmoe::GemmArgs;

// A tile's rows are addressed with 32 bits from its first one: 256 rows of up to this many values.
constexpr long long kMaxStride = 1ll << 20;
// Rows of a product, or columns: with tiles' worth more they still count in 32 bits, and no launch takes more.
constexpr int kMaxRows = 1 << 30;

size_t align_up(size_t v) { return (v + 255) / 256 * 256; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
size_t size_of(int dtype) { return dtype == FLASH_MOE_F32 ? 4 : 2; }

// Rows of `width` values in memory: where they begin and how far apart they lie.
hipError_t check_rows(const char* name, const void* p, long long ld, long long width, int dtype) {
  if (p == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null %s pointer", name);
  if (!aligned16(p)) FMOE_FAIL(hipErrorInvalidValue, "%s does not begin on 16 bytes", name);
  if (ld < width || ld > kMaxStride || ld * static_cast<long long>(size_of(dtype)) % 16 != 0)
    FMOE_FAIL(hipErrorInvalidValue, "%s: %lld values from row to row (at least %lld, at most %lld, whole 16 bytes)", name,
              ld, width, kMaxStride);
  return hipSuccess;
}

hipError_t validate(const FlashMoeFfnDesc* d, int tokens) {
  if (d == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null description");
  if (d->dtype != FLASH_MOE_F32 && d->dtype != FLASH_MOE_BF16)
    FMOE_FAIL(hipErrorInvalidValue, "dtype %i is neither float32 (0) nor bfloat16 (1)", d->dtype);
  if (d->activation != FLASH_MOE_ACT_SILU && d->activation != FLASH_MOE_ACT_GELU_TANH)
    FMOE_FAIL(hipErrorInvalidValue, "activation %i is neither SiLU (0) nor GELU's tanh form (1)", d->activation);
  if (d->weights != FLASH_MOE_FFN_ROW_MAJOR && d->weights != FLASH_MOE_FFN_MXFP4)
    FMOE_FAIL(hipErrorInvalidValue, "weights %i are neither row-major (0) nor MXFP4 (1)", d->weights);
  const bool mx = d->weights == FLASH_MOE_FFN_MXFP4;
  const int of = mx ? 32 : 8;
  if (d->hidden < of || d->hidden % of != 0 || d->intermediate < of || d->intermediate % of != 0 ||
      d->hidden > kMaxStride || d->intermediate >= kMaxStride / 2)
    FMOE_FAIL(hipErrorInvalidValue, "H=%i, I=%i: multiples of %i, H up to %lld, I below half of that", d->hidden,
              d->intermediate, of, kMaxStride);
  if (mx && d->dtype != FLASH_MOE_BF16) FMOE_FAIL(hipErrorInvalidValue, "MXFP4 weights take bfloat16 tokens");
  if (tokens < 0 || tokens > kMaxRows) FMOE_FAIL(hipErrorInvalidValue, "%i tokens (at most %i)", tokens, kMaxRows);
  return hipSuccess;
}

hipError_t validate_weights(const FlashMoeFfnDesc* d) {
  if (d->w13 == nullptr || d->w2 == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null weight pointer");
  if (!aligned16(d->w13) || !aligned16(d->w2)) FMOE_FAIL(hipErrorInvalidValue, "weights do not begin on 16 bytes");
  if (d->weights == FLASH_MOE_FFN_MXFP4 && (d->w13_scales == nullptr || d->w2_scales == nullptr))
    FMOE_FAIL(hipErrorInvalidValue, "MXFP4 weights without scales");
  return hipSuccess;
}

// Rows of the library's own buffers do not lie a multiple of 4 KiB apart: a tile's rows would begin in the same few
// channels of the L2 (8192 x 4096 x 4096, rows of A and B 8 KiB apart 208 to 228 us, 64 values more 194).
long long apart(long long width, int dtype) { return width * static_cast<long long>(size_of(dtype)) % 4096 == 0 ? width + 64 : width; }

// What a forward pass leaves for the backward pass: the two projections before the activation in
// float32 and h in the layer's dtype; the gradients of the projections, the backward pass's own.
// h and those gradients are rounded to the layer's dtype between two products, which in bfloat16 is one rounding more than the
// results' own: they are off by 0.0023 of their norm instead of 0.0017 (by up to 0.0026 for a single token, where few values
// count). In 32 bits they would be operands of two bfloat16 parts, and the products that take them, a third of a forward
// pass's multiplications and five sixths of a backward pass's, would be twice as many.
size_t gu_bytes(const FlashMoeFfnDesc& d, int tokens) { return align_up(size_t(tokens) * 2 * d.intermediate * 4); }
size_t h_bytes(const FlashMoeFfnDesc& d, int tokens) {
  return align_up(size_t(tokens) * apart(d.intermediate, d.dtype) * size_of(d.dtype));
}
size_t dgu_bytes(const FlashMoeFfnDesc& d, int tokens) {
  return align_up(size_t(tokens) * apart(2LL * d.intermediate, d.dtype) * size_of(d.dtype));
}

// The products of a call, without their matrices; a workspace holds the partial sums of one whose k is split
// (one product at a time has some) behind what the passes lay there.
GemmArgs up_sizes(const FlashMoeFfnDesc& d, int tokens) {
  GemmArgs p{};
  p.M = tokens, p.N = d.intermediate, p.K = d.hidden, p.act = d.activation;
  return p;
}
GemmArgs down_sizes(const FlashMoeFfnDesc& d, int tokens) {
  GemmArgs p{};
  p.M = tokens, p.N = d.hidden, p.K = d.intermediate;
  return p;
}
fmoe::FfnGrads grads_sizes(const FlashMoeFfnDesc& d, int tokens, bool dx, bool dw13, bool dw2) {
  const int H = d.hidden, I = d.intermediate;
  fmoe::FfnGrads g{};
  if (tokens > 0 && dx) g.dx.M = tokens, g.dx.N = H, g.dx.K = 2 * I;
  if (dw13) g.dw13.M = 2 * I, g.dw13.N = H, g.dw13.K = tokens;
  if (dw2) g.dw2.M = H, g.dw2.N = I, g.dw2.K = tokens;
  return g;
}
size_t product_bytes(const FlashMoeFfnDesc& d, int epi, const GemmArgs& p) {
  return d.weights == FLASH_MOE_FFN_MXFP4 ? fmoe::mxfp4_gemm_bytes(false, epi, p)
                                          : fmoe::ffn_gemm_bytes(d.dtype, epi == fmoe::EPI_SLOPE, epi, p);
}
size_t forward_partial_bytes(const FlashMoeFfnDesc& d, int tokens) {
  const size_t up = product_bytes(d, fmoe::EPI_GATED, up_sizes(d, tokens));
  const size_t down = product_bytes(d, fmoe::EPI_STORE, down_sizes(d, tokens));
  return align_up(up > down ? up : down);
}
// (fewer gradients than three are split into what room these leave)
size_t backward_partial_bytes(const FlashMoeFfnDesc& d, int tokens) {
  const size_t dh = product_bytes(d, fmoe::EPI_SLOPE, up_sizes(d, tokens));
  const size_t grads = fmoe::ffn_grads_bytes(d.dtype, grads_sizes(d, tokens, true, true, true));
  return align_up(dh > grads ? dh : grads);
}
float* as_partial(void* workspace, size_t behind, size_t bytes) {
  return workspace == nullptr || bytes == 0 ? nullptr : reinterpret_cast<float*>(static_cast<char*>(workspace) + behind);
}

}  // namespace

extern "C" {

int flashMoeFfnBytes(const FlashMoeFfnDesc* desc, int tokens, size_t* saved, size_t* forward, size_t* backward) {
  const hipError_t v = validate(desc, tokens);
  if (v != hipSuccess) return v;
  if (saved != nullptr) *saved = gu_bytes(*desc, tokens) + h_bytes(*desc, tokens);
  if (forward != nullptr) *forward = h_bytes(*desc, tokens) + forward_partial_bytes(*desc, tokens);
  if (backward != nullptr) {
    const bool mx = desc->weights == FLASH_MOE_FFN_MXFP4;  // no backward pass
    *backward = dgu_bytes(*desc, tokens) + (mx ? 0 : backward_partial_bytes(*desc, tokens));
  }
  return hipSuccess;
}

int flashMoeFfnSavingBytes(const FlashMoeFfnDesc* desc, int tokens, size_t* forward) {
  const hipError_t v = validate(desc, tokens);
  if (v != hipSuccess) return v;
  if (forward == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null result pointer");
  *forward = forward_partial_bytes(*desc, tokens);
  return hipSuccess;
}

int flashMoeFfnForward(const FlashMoeFfnDesc* desc, const void* x, long long ldx, void* y, long long ldy, int tokens,
                       void* saved, void* workspace, void* stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  hipError_t v = validate(desc, tokens);
  if (v != hipSuccess) return v;
  if (tokens == 0) return hipSuccess;
  const FlashMoeFfnDesc& d = *desc;
  const int H = d.hidden, I = d.intermediate;
  if ((v = validate_weights(desc)) != hipSuccess) return v;
  if ((v = check_rows("x", x, ldx, H, d.dtype)) != hipSuccess) return v;
  if ((v = check_rows("y", y, ldy, H, d.dtype)) != hipSuccess) return v;
  const bool mx = d.weights == FLASH_MOE_FFN_MXFP4;
  if (mx && saved != nullptr) FMOE_FAIL(hipErrorInvalidValue, "a block of MXFP4 weights has no backward pass");
  if (workspace == nullptr && saved == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null workspace");
  if (!aligned16(workspace) || !aligned16(saved)) FMOE_FAIL(hipErrorInvalidValue, "workspace does not begin on 16 bytes");
  char* keep = static_cast<char*>(saved);
  void* h = keep != nullptr ? keep + gu_bytes(d, tokens) : workspace;

  GemmArgs up = up_sizes(d, tokens), down = down_sizes(d, tokens);
  // Plans that flashMoeFfnBytes made too fit what it asked for. With MXFP4 weights the scales' addresses, which it does not
  // see, count for which kernel runs: a product may then want more, and gets what there is.
  const size_t room = mx ? forward_partial_bytes(d, tokens) : ~size_t{0};
  up.partial = down.partial = as_partial(workspace, keep != nullptr ? 0 : h_bytes(d, tokens), room);
  up.a = x, up.b = d.w13, up.b_scales = static_cast<const unsigned char*>(d.w13_scales);
  up.c = h, up.gu = reinterpret_cast<float*>(keep);
  up.lda = ldx, up.ldb = H, up.ldc = apart(I, d.dtype);
  down.a = h, down.b = d.w2, down.b_scales = static_cast<const unsigned char*>(d.w2_scales);
  down.c = y;
  down.lda = up.ldc, down.ldb = I, down.ldc = ldy;
  if (mx) {
    FMOE_HIP_CHECK(fmoe::launch_mxfp4_gemm(false, fmoe::EPI_GATED, up, room, stream));
    FMOE_HIP_CHECK(fmoe::launch_mxfp4_gemm(false, fmoe::EPI_STORE, down, room, stream));
  } else {
    FMOE_HIP_CHECK(fmoe::launch_ffn_gemm(d.dtype, false, fmoe::EPI_GATED, up, room, stream));
    FMOE_HIP_CHECK(fmoe::launch_ffn_gemm(d.dtype, false, fmoe::EPI_STORE, down, room, stream));
  }
  return hipSuccess;
}

int flashMoeFfnBackward(const FlashMoeFfnDesc* desc, const void* x, long long ldx, const void* dy, long long lddy,
                        int tokens, const void* saved, void* workspace, void* dx, long long lddx, void* dw13, void* dw2,
                        void* stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  hipError_t v = validate(desc, tokens);
  if (v != hipSuccess) return v;
  const FlashMoeFfnDesc& d = *desc;
  const int H = d.hidden, I = d.intermediate;
  if (d.weights != FLASH_MOE_FFN_ROW_MAJOR) FMOE_FAIL(hipErrorInvalidValue, "a block of MXFP4 weights has no backward pass");
  if (!aligned16(dw13) || !aligned16(dw2)) FMOE_FAIL(hipErrorInvalidValue, "gradients do not begin on 16 bytes");
  if (tokens > 0) {
    if ((v = validate_weights(desc)) != hipSuccess) return v;
    if ((v = check_rows("x", x, ldx, H, d.dtype)) != hipSuccess) return v;
    if ((v = check_rows("dy", dy, lddy, H, d.dtype)) != hipSuccess) return v;
    if (dx != nullptr && (v = check_rows("dx", dx, lddx, H, d.dtype)) != hipSuccess) return v;
    if (saved == nullptr || !aligned16(saved)) FMOE_FAIL(hipErrorInvalidValue, "null or unaligned saved results");
    if (((dx != nullptr || dw13 != nullptr) && workspace == nullptr) || !aligned16(workspace))
      FMOE_FAIL(hipErrorInvalidValue, "null or unaligned workspace");
  }
  const char* keep = static_cast<const char*>(saved);
  const long long ld_h = apart(I, d.dtype), ld_dgu = apart(2LL * I, d.dtype);
  const bool all = dx != nullptr && dw13 != nullptr && dw2 != nullptr;  // which is what the workspace was made for
  const size_t room = all ? ~size_t{0} : backward_partial_bytes(d, tokens);
  float* partial = as_partial(workspace, dgu_bytes(d, tokens), room);
  if (tokens > 0 && (dx != nullptr || dw13 != nullptr)) {
    // dh = dy W2, and with it the gradients of both projections
    GemmArgs p = up_sizes(d, tokens);
    p.partial = partial;
    p.a = dy, p.b = d.w2, p.c = workspace, p.gu = reinterpret_cast<float*>(const_cast<char*>(keep));
    p.lda = lddy, p.ldb = I, p.ldc = ld_dgu;
    FMOE_HIP_CHECK(fmoe::launch_ffn_gemm(d.dtype, true, fmoe::EPI_SLOPE, p, room, stream));
  }
  // the weights' gradients sum over the tokens; of no tokens they are zeros
  fmoe::FfnGrads grads = grads_sizes(d, tokens, dx != nullptr, dw13 != nullptr, dw2 != nullptr);
  if (tokens > 0 && dx != nullptr) {
    GemmArgs& p = grads.dx;
    p.a = workspace, p.b = d.w13, p.c = dx;
    p.lda = ld_dgu, p.ldb = H, p.ldc = lddx;
  }
  if (dw13 != nullptr) {
    GemmArgs& p = grads.dw13;
    p.a = workspace, p.b = x, p.c = dw13;
    p.lda = ld_dgu, p.ldb = ldx, p.ldc = H;
  }
  if (dw2 != nullptr) {
    GemmArgs& p = grads.dw2;
    p.a = dy, p.b = keep + (tokens > 0 ? gu_bytes(d, tokens) : 0), p.c = dw2;
    p.lda = lddy, p.ldb = ld_h, p.ldc = I;
  }
  FMOE_HIP_CHECK(fmoe::launch_ffn_grads(d.dtype, grads, partial, room, stream));
  return hipSuccess;
}

int flashMoeMxfp4Quantize(int dtype, const void* x, long long ldx, int rows, int k, void* codes, void* scales, void* stream) {
  if (dtype != FLASH_MOE_F32 && dtype != FLASH_MOE_BF16)
    FMOE_FAIL(hipErrorInvalidValue, "dtype %i is neither float32 (0) nor bfloat16 (1)", dtype);
  if (rows < 0 || k < 32 || k % 32 != 0) FMOE_FAIL(hipErrorInvalidValue, "%i rows of %i values (a multiple of 32)", rows, k);
  if (rows == 0) return hipSuccess;
  if (codes == nullptr || scales == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null codes or scales pointer");
  if (!aligned16(codes)) FMOE_FAIL(hipErrorInvalidValue, "codes do not begin on 16 bytes");
  if (x == nullptr || !aligned16(x) || ldx < k || ldx * static_cast<long long>(size_of(dtype)) % 16 != 0)
    FMOE_FAIL(hipErrorInvalidValue, "x: null, not on 16 bytes, or rows %lld values apart", ldx);
  FMOE_HIP_CHECK(fmoe::launch_mxfp4_quantize(dtype, x, ldx, rows, k, codes, scales, static_cast<hipStream_t>(stream)));
  return hipSuccess;
}

int flashMoeMxfp4Dequantize(int dtype, const void* codes, const void* scales, int rows, int k, void* out, long long ldo,
                            void* stream) {
  if (dtype != FLASH_MOE_F32 && dtype != FLASH_MOE_BF16)
    FMOE_FAIL(hipErrorInvalidValue, "dtype %i is neither float32 (0) nor bfloat16 (1)", dtype);
  if (rows < 0 || k < 32 || k % 32 != 0) FMOE_FAIL(hipErrorInvalidValue, "%i rows of %i values (a multiple of 32)", rows, k);
  if (rows == 0) return hipSuccess;
  if (codes == nullptr || scales == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null codes or scales pointer");
  if (!aligned16(codes)) FMOE_FAIL(hipErrorInvalidValue, "codes do not begin on 16 bytes");
  if (out == nullptr || !aligned16(out) || ldo < k || ldo * static_cast<long long>(size_of(dtype)) % 16 != 0)
    FMOE_FAIL(hipErrorInvalidValue, "out: null, not on 16 bytes, or rows %lld values apart", ldo);
  FMOE_HIP_CHECK(fmoe::launch_mxfp4_dequantize(dtype, codes, scales, rows, k, out, ldo, static_cast<hipStream_t>(stream)));
  return hipSuccess;
}

int flashMoeMxfp4LinearBytes(int x_format, int rows, int n, int k, size_t* bytes) {
  if (x_format != FLASH_MOE_BF16 && x_format != FLASH_MOE_MXFP4)
    FMOE_FAIL(hipErrorInvalidValue, "x_format %i is neither bfloat16 (1) nor MXFP4 (2)", x_format);
  if (rows < 0 || rows > kMaxRows || n < 0 || n > kMaxRows || k < 32 || k % 32 != 0 || k > kMaxStride)
    FMOE_FAIL(hipErrorInvalidValue, "%i x %i x %i (up to %i twice, the last a multiple of 32 up to %lld)", rows, n, k, kMaxRows, kMaxStride);
  if (bytes == nullptr) FMOE_FAIL(hipErrorInvalidValue, "null result pointer");
  GemmArgs p{};
  p.M = rows, p.N = n, p.K = k;
  *bytes = rows == 0 || n == 0 ? 0 : fmoe::mxfp4_gemm_bytes(x_format == FLASH_MOE_MXFP4, fmoe::EPI_STORE, p);
  return hipSuccess;
}

int flashMoeMxfp4Linear(int x_format, const void* x, const void* x_scales, long long ldx, int rows, const void* codes,
                        const void* scales, int n, int k, void* y, long long ldy, void* workspace, void* stream) {
  size_t bytes = 0;
  hipError_t v = static_cast<hipError_t>(flashMoeMxfp4LinearBytes(x_format, rows, n, k, &bytes));
  if (v != hipSuccess) return v;
  if (rows == 0 || n == 0) return hipSuccess;
  if (bytes > 0 && (workspace == nullptr || !aligned16(workspace)))
    FMOE_FAIL(hipErrorInvalidValue, "null or unaligned workspace");
  const bool mx = x_format == FLASH_MOE_MXFP4;
  if (mx) {
    if (x == nullptr || x_scales == nullptr || !aligned16(x)) FMOE_FAIL(hipErrorInvalidValue, "x: null or unaligned pointer");
    if (ldx != k) FMOE_FAIL(hipErrorInvalidValue, "MXFP4 rows lie one behind the other");
  } else if ((v = check_rows("x", x, ldx, k, FLASH_MOE_BF16)) != hipSuccess) {
    return v;
  }
  if (codes == nullptr || scales == nullptr || !aligned16(codes))
    FMOE_FAIL(hipErrorInvalidValue, "null codes or scales pointer, or codes that do not begin on 16 bytes");
  if (y == nullptr || ldy < n || (reinterpret_cast<uintptr_t>(y) & 1) != 0)
    FMOE_FAIL(hipErrorInvalidValue, "y: null, at an odd address, or rows %lld values apart", ldy);
  if (n % 8 == 0 && (!aligned16(y) || ldy % 8 != 0))
    FMOE_FAIL(hipErrorInvalidValue, "y: rows of a multiple of 8 values begin on 16 bytes");
  GemmArgs p{};
  p.a = x, p.a_scales = static_cast<const unsigned char*>(x_scales), p.lda = ldx;
  p.b = codes, p.b_scales = static_cast<const unsigned char*>(scales), p.ldb = k;
  p.c = y, p.ldc = ldy;
  p.M = rows, p.N = n, p.K = k;
  p.partial = as_partial(workspace, 0, bytes);
  FMOE_HIP_CHECK(fmoe::launch_mxfp4_gemm(mx, fmoe::EPI_STORE, p, bytes, static_cast<hipStream_t>(stream)));
  return hipSuccess;
}

}  // extern "C"
