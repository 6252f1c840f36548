// What becomes of a product whose k was split between workgroups: its partial sums [splits, M, columns] in float32 are
// added in the splits' order, and what the unsplit kernels do with their sums is done with these. A read of every
// partial sum (mostly from the last-level cache, they were just written) is what it takes.
#include "ffn_device.h"

namespace fmoe {

constexpr int EIGHT = 8;       // splits a thread asks for at a time
constexpr int THREADS = 64;    // few results are on many CUs

// four neighbours of a row, `at` values from its beginning
__device__ __forceinline__ f32x4 sum_splits(const GemmArgs& p, long long ld, long long row, int at) {
  const float* from = p.partial + row * ld + at;
  const long long apart = p.M * ld;
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  int s = 0;
  for (; s + EIGHT <= p.splits; s += EIGHT) {
    f32x4 v[EIGHT];
#pragma unroll
    for (int i = 0; i < EIGHT; ++i) v[i] = *reinterpret_cast<const f32x4*>(from + (s + i) * apart);
#pragma unroll
    for (int i = 0; i < EIGHT; ++i) sum += v[i];
  }
  f32x4 v[EIGHT];
#pragma unroll
  for (int i = 0; i < EIGHT; ++i) v[i] = s + i < p.splits ? *reinterpret_cast<const f32x4*>(from + (s + i) * apart) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < EIGHT; ++i) sum += v[i];
  return sum;
}

// columns n .. n + 3 of a row; rows of bfloat16 whose width is no multiple of 8 begin anywhere
template <bool F32>
__device__ __forceinline__ void store_four(void* row, int n, int columns, const f32x4& v) {
  if constexpr (F32) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(row) + n) = v;
  } else {
    unsigned short* to = static_cast<unsigned short*>(row) + n;
    const unsigned lo = pack_bf16(v[0], v[1]), hi = pack_bf16(v[2], v[3]);
    if ((columns & 7) == 0) {
      *reinterpret_cast<u32x2*>(to) = u32x2{lo, hi};
    } else {
      const unsigned short each[4] = {static_cast<unsigned short>(lo), static_cast<unsigned short>(lo >> 16),
                                      static_cast<unsigned short>(hi), static_cast<unsigned short>(hi >> 16)};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < columns) to[j] = each[j];
    }
  }
}

template <bool F32, int EPI>
__device__ __forceinline__ void finish_four(const GemmArgs& p, long long at) {
  constexpr int SIZE = F32 ? 4 : 2;
  const int fours = (p.N + 3) / 4;
  const long long m = at / fours;
  if (m >= p.M) return;
  const int n = static_cast<int>(at - m * fours) * 4;
  const long long ld = partial_ld(EPI == EPI_GATED ? 2 * p.N : p.N);
  const f32x4 sum = sum_splits(p, ld, m, n);
  char* row = static_cast<char*>(p.c) + m * p.ldc * SIZE;
  if constexpr (EPI == EPI_STORE) {
    store_four<F32>(row, n, p.N, sum);
  } else if constexpr (EPI == EPI_GATED) {
    const f32x4 up = sum_splits(p, ld, m, p.N + n);
    f32x4 h;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = act_of<F32>(p.act, sum[i]) * up[i];
    store_four<F32>(row, n, p.N, h);
    if (p.gu != nullptr) {
      store_four<true>(p.gu + m * (2LL * p.N), n, p.N, sum);
      store_four<true>(p.gu + m * (2LL * p.N) + p.N, n, p.N, up);
    }
  } else {
    const float* gu = p.gu + m * (2LL * p.N) + n;
    const f32x4 gate = *reinterpret_cast<const f32x4*>(gu), up = *reinterpret_cast<const f32x4*>(gu + p.N);
    f32x4 dg, du;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, slope;
      act_and_slope<F32>(p.act, gate[i], a, slope);
      dg[i] = sum[i] * up[i] * slope;
      du[i] = sum[i] * a;
    }
    store_four<F32>(row, n, p.N, dg);
    store_four<F32>(row + static_cast<long long>(p.N) * SIZE, n, p.N, du);
  }
}

template <bool F32, int EPI>
__global__ __launch_bounds__(THREADS) void ffn_finish_kernel(GemmArgs p) {
  finish_four<F32, EPI>(p, blockIdx.x * static_cast<long long>(THREADS) + threadIdx.x);
}

// begin: the first workgroup of each gradient's
template <bool F32>
__global__ __launch_bounds__(THREADS) void ffn_finish_grads_kernel(FfnGrads p) {
  const int id = blockIdx.x, which = id >= p.begin[2] ? 2 : id >= p.begin[1] ? 1 : 0;
  finish_four<F32, EPI_STORE>(which == 0 ? p.dx : which == 1 ? p.dw13 : p.dw2, (id - p.begin[which]) * static_cast<long long>(THREADS) + threadIdx.x);
}

static long long blocks_for(const GemmArgs& p) { return (static_cast<long long>(p.M) * ((p.N + 3) / 4) + THREADS - 1) / THREADS; }

hipError_t launch_ffn_finish(int dtype, int epi, const GemmArgs& p, hipStream_t stream) {
  const long long blocks = blocks_for(p);
  if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
  auto kernel = dtype == 1 ? (epi == EPI_STORE ? ffn_finish_kernel<false, EPI_STORE> : epi == EPI_GATED ? ffn_finish_kernel<false, EPI_GATED>
                                                                                                        : ffn_finish_kernel<false, EPI_SLOPE>)
                           : (epi == EPI_STORE ? ffn_finish_kernel<true, EPI_STORE> : epi == EPI_GATED ? ffn_finish_kernel<true, EPI_GATED>
                                                                                                       : ffn_finish_kernel<true, EPI_SLOPE>);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(THREADS), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_ffn_finish_grads(int dtype, const FfnGrads& grads, hipStream_t stream) {
  FfnGrads p = grads;
  GemmArgs* of[] = {&p.dx, &p.dw13, &p.dw2};
  long long at = 0;
  for (int i = 0; i < 3; ++i) {
    p.begin[i] = static_cast<int>(at < 0x7FFFFFFF ? at : 0x7FFFFFFF);
    if (of[i]->M > 0 && of[i]->splits > 1) at += blocks_for(*of[i]);
  }
  if (at == 0) return hipSuccess;
  if (at > 0x7FFFFFFF) return hipErrorInvalidValue;
  auto kernel = dtype == 1 ? ffn_finish_grads_kernel<false> : ffn_finish_grads_kernel<true>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(at)), dim3(THREADS), 0, stream, p);
  return hipGetLastError();
}

}  // namespace fmoe
