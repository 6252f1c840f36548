// Whether the dense block's and MXFP4's calls keep to the workspaces they ask for. This program stands in for the
// runtime's launches, so nothing runs and no GPU is needed: of every kernel that the library would enqueue
// the arguments are looked at, which say where its partial sums begin and how many there are.
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "flash_distributed_moe_amd/csrc/ffn_params.h"
#include "include/flash_moe.h"
#include "tests/cpp/mini_test.h"

namespace {

using fmoe::FfnGrads;
using fmoe::GemmArgs;

struct Launch {
  FfnGrads grads;  // as many bytes as the kernel's argument may have; a product's are the first of them
  GemmArgs product() const {
    GemmArgs p;
    std::memcpy(&p, &grads, sizeof(p));
    return p;
  }
};
std::vector<Launch> launches;
size_t argument_bytes = 0;  // of the kernels from here on: of those that take three products, sizeof(FfnGrads)

struct Configuration {
  dim3 grid, block;
  size_t lds;
  hipStream_t stream;
} configuration;

}  // namespace

extern "C" hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t stream) {
  configuration = {grid, block, lds, stream};
  return hipSuccess;
}
extern "C" hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* stream) {
  *grid = configuration.grid, *block = configuration.block, *lds = configuration.lds, *stream = configuration.stream;
  return hipSuccess;
}
extern "C" hipError_t hipLaunchKernel(const void*, dim3, dim3, void** args, size_t, hipStream_t) {
  Launch l{};
  // a backward pass: one product, its finishing kernel if it has splits, and then kernels of three products
  if (argument_bytes == 0) {
    GemmArgs p;
    std::memcpy(&p, args[0], sizeof(p));
    const bool one = launches.empty() || (launches.size() == 1 && launches[0].product().splits > 1);
    std::memcpy(&l.grads, args[0], one ? sizeof(GemmArgs) : sizeof(FfnGrads));
  } else {
    std::memcpy(&l.grads, args[0], argument_bytes);
  }
  launches.push_back(l);
  return hipSuccess;
}
extern "C" hipError_t hipGetLastError() { return hipSuccess; }

namespace {

// Addresses that nothing is read from or written to: each buffer has 2^44 bytes to itself.
char* at(int buffer, int offset = 0) { return reinterpret_cast<char*>((static_cast<uintptr_t>(buffer) << 44) + offset); }
enum { X = 1, Y, W13, W2, S13, S2, SAVED, WORK, DX, DW13, DW2 };

// the last byte behind the workspace's first that a product's partial sums take, or 0
long long end_of_sums(const GemmArgs& p, int columns) {
  if (p.M == 0 || p.splits <= 1) return 0;
  const char* end = reinterpret_cast<const char*>(p.partial) + static_cast<long long>(p.splits) * p.M * fmoe::partial_ld(columns) * 4;
  return end - at(WORK);
}
bool keeps_to(const GemmArgs& p, int columns, size_t bytes, const char* what, int T, int H, int I) {
  const long long end = end_of_sums(p, columns);
  const bool ok = end == 0 || (reinterpret_cast<const char*>(p.partial) >= at(WORK) && end <= static_cast<long long>(bytes));
  if (!ok) printf("%s, T=%d H=%d I=%d: partial sums end at byte %lld of %zu\n", what, T, H, I, end, bytes);
  return ok;
}

FlashMoeFfnDesc describe(int H, int I, int dtype, bool mx, int off13 = 0, int off2 = 0) {
  FlashMoeFfnDesc d{};
  d.hidden = H, d.intermediate = I, d.dtype = dtype;
  d.weights = mx ? FLASH_MOE_FFN_MXFP4 : FLASH_MOE_FFN_ROW_MAJOR;
  d.w13 = at(W13), d.w2 = at(W2), d.w13_scales = at(S13, off13), d.w2_scales = at(S2, off2);
  return d;
}

bool forward_keeps_to(int T, const FlashMoeFfnDesc& d, bool save) {
  size_t bytes = 0;
  if (save ? flashMoeFfnSavingBytes(&d, T, &bytes) : flashMoeFfnBytes(&d, T, nullptr, &bytes, nullptr)) return false;
  launches.clear(), argument_bytes = sizeof(GemmArgs);
  if (flashMoeFfnForward(&d, at(X), d.hidden, at(Y), d.hidden, T, save ? at(SAVED) : nullptr, at(WORK), nullptr)) return false;
  bool ok = launches.size() >= 2;
  for (const Launch& l : launches) {
    const GemmArgs p = l.product();
    ok &= keeps_to(p, p.c == at(Y) ? p.N : 2 * p.N, bytes, p.c == at(Y) ? "output" : "projections", T, d.hidden, d.intermediate);
  }
  return ok;
}

bool backward_keeps_to(int T, const FlashMoeFfnDesc& d, bool dx, bool dw13, bool dw2) {
  size_t bytes = 0;
  if (flashMoeFfnBytes(&d, T, nullptr, nullptr, &bytes)) return false;
  launches.clear(), argument_bytes = dx || dw13 ? 0 : sizeof(FfnGrads);
  if (flashMoeFfnBackward(&d, at(X), d.hidden, at(Y), d.hidden, T, at(SAVED), at(WORK), dx ? at(DX) : nullptr, d.hidden,
                          dw13 ? at(DW13) : nullptr, dw2 ? at(DW2) : nullptr, nullptr))
    return false;
  bool ok = true;
  size_t i = 0;
  if (dx || dw13) {
    const GemmArgs p = launches[0].product();
    ok &= keeps_to(p, p.N, bytes, "slope", T, d.hidden, d.intermediate);
    i = p.splits > 1 ? 2 : 1;
  }
  for (; i < launches.size(); ++i) {
    const FfnGrads& g = launches[i].grads;
    for (const GemmArgs* p : {&g.dx, &g.dw13, &g.dw2}) ok &= keeps_to(*p, p->N, bytes, "gradient", T, d.hidden, d.intermediate);
  }
  return ok;
}

const int kTokens[] = {1, 3, 8, 16, 32, 33, 40, 65, 130, 700, 4097};
const int kWidths[] = {32, 96, 416, 1280, 2048, 4096, 5024, 7168, 9984, 12288, 16384, 16416, 17408, 18432, 22880, 36768, 53248};

TEST(FfnWorkspace, forwardOnMxfp4WeightsWithScalesAnywhere) {
  bool ok = true, shared = false;
  for (int T : kTokens)
    for (int H : kWidths)
      for (int I : kWidths)
        for (int off = 0; off < 16; ++off) {  // scales of w13 / of w2 begin off % 4 / off / 4 bytes behind a multiple of 4
          ok &= forward_keeps_to(T, describe(H, I, FLASH_MOE_BF16, true, off % 4, off / 4), false);
          for (const Launch& l : launches) shared |= l.product().splits > 1;
        }
  ASSERT_TRUE(ok);
  ASSERT_TRUE(shared);
}

TEST(FfnWorkspace, forwardOnRowMajorWeights) {
  bool ok = true, shared = false;
  for (int dtype : {FLASH_MOE_F32, FLASH_MOE_BF16})
    for (int T : kTokens)
      for (int H : kWidths)
        for (int I : kWidths)
          for (bool save : {false, true}) {
            ok &= forward_keeps_to(T, describe(H + 8, I + 8, dtype, false), save);
            for (const Launch& l : launches) shared |= l.product().splits > 1;
          }
  ASSERT_TRUE(ok);
  ASSERT_TRUE(shared);
}

TEST(FfnWorkspace, backwardForEveryChoiceOfGradients) {
  bool ok = true, shared = false;
  for (int dtype : {FLASH_MOE_F32, FLASH_MOE_BF16})
    for (int T : kTokens)
      for (int H : kWidths)
        for (int I : kWidths)
          for (int want = 1; want < 8; ++want) {
            ok &= backward_keeps_to(T, describe(H + 8, I, dtype, false), want & 1, want & 2, want & 4);
            for (const Launch& l : launches) shared |= l.grads.dw13.splits > 1;
          }
  ASSERT_TRUE(ok);
  ASSERT_TRUE(shared);
}

TEST(FfnWorkspace, productsWithScalesAnywhere) {
  bool ok = true, shared = false;
  for (int format : {int(FLASH_MOE_BF16), int(FLASH_MOE_MXFP4)})
    for (int M : kTokens)
      for (int N : {1, 37, 200, 4096, 16385})
        for (int K : kWidths)
          for (int off = 0; off < 16; ++off) {
            size_t bytes = 0;
            launches.clear(), argument_bytes = sizeof(GemmArgs);
            ok &= flashMoeMxfp4LinearBytes(format, M, N, K, &bytes) == hipSuccess;
            ok &= flashMoeMxfp4Linear(format, at(X), at(S13, off % 4), K, M, at(W2), at(S2, off / 4), N, K, at(Y), N,
                                      bytes > 0 ? at(WORK) : nullptr, nullptr) == hipSuccess;
            for (const Launch& l : launches) {
              ok &= keeps_to(l.product(), N, bytes, "product", M, N, K);
              shared |= l.product().splits > 1;
            }
          }
  ASSERT_TRUE(ok);
  ASSERT_TRUE(shared);
}

}  // namespace

int main() { return mini::run_all(); }
