// Matrix products of few rows (the tokens of a decode batch) with row-major weights. The weights are read once,
// and reading them is what such a product's time is. A workgroup takes HB groups of 8 weight rows over the whole
// of k; its waves take the steps of k in turn, 128 bytes of a row a step, so that the workgroup reads its
// rows front to back; the waves' sums meet in LDS and are added in the waves' order.
//
// A load instruction takes 8 rows x 128 bytes, whole cache lines: the 16 rows x 64 bytes that a 16 x 16 matrix
// instruction's operand has are twice as many line lookups, and a CU manages about 16 bytes a clock that way
// (measured, 128 workgroups on 16 rows x 8 KiB each: 5.3 us, in whole lines 3.9). So of an
// operand's 16 "rows" r the first eight are 8 real rows with the first half of the line and the
// other eight are the same rows with its second half; the rows of x likewise, 8 at a time. Of the product's four
// quadrants the two on the diagonal, whose halves agree, are sums over half of the k each, and
// the other two mean nothing. They are as many instructions as with 16 rows an operand while there are 8 rows of x.
#include "ffn_device.h"

namespace fmoe {

enum SkinnyKind { SKINNY_BF16 = 0, SKINNY_F32 = 1, SKINNY_MXFP4_WEIGHTS = 2, SKINNY_MXFP4_BOTH = 3 };

__host__ __device__ constexpr int skinny_step_k(int kind) {
  return kind == SKINNY_BF16 ? 64 : kind == SKINNY_F32 ? 32 : 256;
}

__device__ __forceinline__ i32x4 load16(__amdgpu_buffer_rsrc_t r, unsigned offset) {
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(offset), 0, 0));
}

// `bytes` to LDS by the whole workgroup, 16 at a time and the last few one at a time. Whole rounds are
// written: up to copied_bytes(bytes).
template <int THREADS>
__device__ __forceinline__ void copy_to_lds(char* lds, const unsigned char* from, int bytes) {
  const int whole = bytes & ~15;
  const __amdgpu_buffer_rsrc_t r = make_rsrc(from, 0x7FFFFFFFu);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int at = 0; at < whole; at += THREADS * 16) {
    const int mine = at + threadIdx.x * 16;
    load_to_lds16(r, lds + at + wave * 1024, mine < whole ? static_cast<unsigned>(mine) : kOutside);
  }
  // (behind the rounds' own zeros, which a wave writes where it has nothing to load)
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < bytes - whole) lds[whole + threadIdx.x] = static_cast<char>(from[whole + threadIdx.x]);
}
template <int THREADS>
__host__ __device__ constexpr int copied_bytes(int bytes) {
  return (bytes + THREADS * 16) / (THREADS * 16) * (THREADS * 16);
}

// LDS: rows of x on their way (two rounds a wave) and, afterwards, the waves' sums; then the scales.
__host__ __device__ constexpr int skinny_fixed_bytes(int kind, int hb, int xb, int waves, int depth) {
  const int x = kind == SKINNY_MXFP4_WEIGHTS ? waves * 2 * depth * xb * 4 * 1024 : 0, part = waves * hb * xb * 256;
  return x > part ? x : part;
}
template <int KIND, bool GATED, int HB, int XB, int WAVES, int DEPTH>
static int skinny_lds_bytes(int blocks) {
  constexpr int SIDE = GATED ? HB / 2 : HB, THREADS = WAVES * 64;
  int bytes = skinny_fixed_bytes(KIND, HB, XB, WAVES, DEPTH);
  if (KIND >= SKINNY_MXFP4_WEIGHTS) bytes += (GATED ? 2 : 1) * copied_bytes<THREADS>(SIDE * 8 * blocks);
  if (KIND == SKINNY_MXFP4_BOTH) bytes += copied_bytes<THREADS>(XB * 8 * blocks);
  return bytes;
}

template <int KIND, bool GATED, int HB, int XB, int WAVES, int DEPTH>
__global__ __launch_bounds__(WAVES * 64) void ffn_skinny_kernel(GemmArgs p) {
  constexpr bool MX = KIND >= SKINNY_MXFP4_WEIGHTS, X_IN_LDS = KIND == SKINNY_MXFP4_WEIGHTS, F32 = KIND == SKINNY_F32;
  constexpr int SIDE = GATED ? HB / 2 : HB;  // groups of 8 columns
  constexpr int THREADS = WAVES * 64, STEP = skinny_step_k(KIND);
  constexpr int X_PIECES = XB * 4;            // X_IN_LDS: 1 KiB pieces of a step's rows of x, 2 rows each
  extern __shared__ __attribute__((aligned(128))) char lds[];  // skinny_lds_bytes

  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int row8 = r & 7, piece = (r >> 3) * 4 + g;  // of a group of 8 rows, of a line
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * SIDE * 8, m0 = blockIdx.y * XB * 8;

  const long long w_row = MX ? p.ldb / 2 : p.ldb * (F32 ? 4 : 2);  // bytes from row to row
  const long long x_row = KIND == SKINNY_MXFP4_BOTH ? p.lda / 2 : p.lda * (F32 ? 4 : 2);
  const char* wp = static_cast<const char*>(p.b) + n0 * w_row;
  const __amdgpu_buffer_rsrc_t wr[2] = {make_rsrc(wp, 0x7FFFFFFFu), make_rsrc(wp + (GATED ? p.N * w_row : 0), 0x7FFFFFFFu)};
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(static_cast<const char*>(p.a) + m0 * x_row, 0x7FFFFFFFu);

  // this lane's piece of the first line of each of its rows
  unsigned w_at[SIDE], x_at[XB];
#pragma unroll
  for (int b = 0; b < SIDE; ++b)
    w_at[b] = n0 + b * 8 + row8 < p.N ? static_cast<unsigned>((b * 8 + row8) * w_row) + piece * 16 : kOutside;
#pragma unroll
  for (int b = 0; b < XB; ++b)
    x_at[b] = m0 + b * 8 + row8 < p.M ? static_cast<unsigned>((b * 8 + row8) * x_row) + piece * 16 : kOutside;

  const int blocks = p.K / 32;
  char* scales = lds + skinny_fixed_bytes(KIND, HB, XB, WAVES, DEPTH);
  const int side_bytes = copied_bytes<THREADS>(SIDE * 8 * blocks);
  char* x_scales = scales + (GATED ? 2 : 1) * side_bytes;
  if constexpr (MX) {
    const int rows = p.N - n0 < SIDE * 8 ? p.N - n0 : SIDE * 8;
    const unsigned char* from = p.b_scales + static_cast<long long>(n0) * blocks;
    copy_to_lds<THREADS>(scales, from, rows * blocks);
    if constexpr (GATED) copy_to_lds<THREADS>(scales + side_bytes, from + static_cast<long long>(p.N) * blocks, rows * blocks);
    if constexpr (KIND == SKINNY_MXFP4_BOTH) {
      const int x_rows = p.M - m0 < XB * 8 ? p.M - m0 : XB * 8;
      copy_to_lds<THREADS>(x_scales, p.a_scales + static_cast<long long>(m0) * blocks, x_rows * blocks);
    }
  }

  struct Round {
    i32x4 w[DEPTH][HB];
    i32x4 x[DEPTH][X_IN_LDS ? 1 : XB];
  };
  constexpr int LOADS = DEPTH * (HB + (X_IN_LDS ? X_PIECES : 0));  // X_IN_LDS: of a round
  char* x_lds = lds + wave * (2 * DEPTH * X_PIECES * 1024);

  auto load = [&](Round& o, int round) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int step = (round * DEPTH + d) * WAVES + wave;
      // (a step behind the end, and a piece behind the end of k, arrive as zeros)
      const bool in = step * STEP + piece * (STEP / 8) < p.K;
      if constexpr (X_IN_LDS) {
        // 512 bytes of each row of x, two rows a load, their 16-byte pieces swapped about by the row
#pragma unroll
        for (int i = 0; i < X_PIECES; ++i) {
          const int row = i * 2 + (lane >> 5), at = (lane & 31) ^ (row & 7);
          const bool ok = m0 + row < p.M && step * STEP + at * 8 < p.K;
          load_to_lds16(xr, x_lds + (((round & 1) * DEPTH + d) * X_PIECES + i) * 1024,
                        ok ? static_cast<unsigned>(row * x_row) + step * (STEP * 2) + at * 16 : kOutside);
        }
      } else {
#pragma unroll
        for (int b = 0; b < XB; ++b) o.x[d][b] = load16(xr, in ? x_at[b] + step * 128 : kOutside);
      }
#pragma unroll
      for (int b = 0; b < HB; ++b) o.w[d][b] = load16(wr[b / SIDE], in ? w_at[b % SIDE] + step * 128 : kOutside);
    }
  };

  f32x4 acc[HB][XB];
#pragma unroll
  for (int b = 0; b < HB; ++b)
#pragma unroll
    for (int c = 0; c < XB; ++c) acc[b][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  auto scale_of = [&](const char* side, int row, int step) -> unsigned {
    const int kb = step * 8 + piece;
    return kb < blocks ? *(const FFN_LDS unsigned char*)(side + row * blocks + kb) : 127u;
  };

  auto multiply = [&](const Round& o, int round) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      [[maybe_unused]] const int step = (round * DEPTH + d) * WAVES + wave;
      if constexpr (KIND == SKINNY_BF16) {
#pragma unroll
        for (int b = 0; b < HB; ++b)
#pragma unroll
          for (int c = 0; c < XB; ++c)
            acc[b][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, o.w[d][b]),
                                                                __builtin_bit_cast(bf16x8, o.x[d][c]), acc[b][c], 0, 0, 0);
      } else if constexpr (KIND == SKINNY_F32) {
#pragma unroll
        for (int b = 0; b < HB; ++b)
#pragma unroll
          for (int c = 0; c < XB; ++c) {
            const f32x4 wf = __builtin_bit_cast(f32x4, o.w[d][b]), xf = __builtin_bit_cast(f32x4, o.x[d][c]);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[b][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[j], xf[j], acc[b][c], 0, 0, 0);
          }
      } else if constexpr (KIND == SKINNY_MXFP4_BOTH) {
        unsigned xs[XB];
#pragma unroll
        for (int c = 0; c < XB; ++c) xs[c] = scale_of(x_scales, c * 8 + row8, step);
#pragma unroll
        for (int b = 0; b < HB; ++b) {
          const unsigned ws = scale_of(scales + (b / SIDE) * side_bytes, b % SIDE * 8 + row8, step);
          const i32x4& q = o.w[d][b];
          const i32x8 w = {q[0], q[1], q[2], q[3], 0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < XB; ++c) {
            const i32x4& y = o.x[d][c];
            const i32x8 x = {y[0], y[1], y[2], y[3], 0, 0, 0, 0};
            acc[b][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, acc[b][c], 4, 4, 0, ws, 0, xs[c]);
          }
        }
      } else {
        float ws[HB];
#pragma unroll
        for (int b = 0; b < HB; ++b)
          ws[b] = __uint_as_float(scale_of(scales + (b / SIDE) * side_bytes, b % SIDE * 8 + row8, step) << 23);
        const char* xl = x_lds + ((round & 1) * DEPTH + d) * X_PIECES * 1024;
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // eight of the lane's 32 weights
          bf16x8 x[XB];
#pragma unroll
          for (int c = 0; c < XB; ++c) x[c] = *(const FFN_LDS bf16x8*)(xl + (c * 8 + row8) * 512 + (((piece * 4 + j) ^ row8) << 4));
#pragma unroll
          for (int b = 0; b < HB; ++b) {
            const unsigned codes = static_cast<unsigned>(o.w[d][b][j]);
            const bf16x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, ws[b], 0);
            const bf16x2 v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, ws[b], 1);
            const bf16x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, ws[b], 2);
            const bf16x2 v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, ws[b], 3);
            const bf16x8 w = {v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
#pragma unroll
            for (int c = 0; c < XB; ++c) acc[b][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x[c], acc[b][c], 0, 0, 0);
          }
        }
      }
    }
  };

  // Rows of x that go through LDS are this wave's alone: it waits until no more loads are in flight than the
  // next round's, which were issued behind its own.
  auto arrived = [&](bool next) {
    if constexpr (X_IN_LDS) {
      __builtin_amdgcn_sched_barrier(0);
      if (next) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LOADS) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto done = [&] {  // the reads of a round's LDS are over before it is loaded into again
    if constexpr (X_IN_LDS) asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
  };

  const int steps = (p.K + STEP - 1) / STEP;
  const int rounds = (steps + WAVES * DEPTH - 1) / (WAVES * DEPTH);
  Round even, odd;
  load(even, 0);
  if constexpr (MX) __syncthreads();  // the scales' last bytes
  for (int i = 0; i < rounds; i += 2) {
    if (i + 1 < rounds) load(odd, i + 1);
    arrived(i + 1 < rounds);
    multiply(even, i);
    done();
    if (i + 1 < rounds) {
      if (i + 2 < rounds) load(even, i + 2);
      arrived(i + 2 < rounds);
      multiply(odd, i + 1);
      done();
    }
  }

  // the two quadrants: (rows 0-7, x 0-7) of lanes r < 8, g < 2 and what lies 8 rows of x and 2 quarters on
  f32x4(*part)[HB * XB][16] = reinterpret_cast<f32x4(*)[HB * XB][16]>(lds);
  if constexpr (X_IN_LDS) __syncthreads();
#pragma unroll
  for (int b = 0; b < HB; ++b)
#pragma unroll
    for (int c = 0; c < XB; ++c) {
      f32x4 v = acc[b][c];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += __shfl(v[j], (lane + 40) & 63, 64);
      if (r < 8 && g < 2) part[wave][b * XB + c][g * 8 + r] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < SIDE * XB * 16; i += THREADS) {
    const int block = i >> 4, l = i & 15;
    f32x4 sum = part[0][block][l], up = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += part[w][block][l];
    if constexpr (GATED) {
#pragma unroll
      for (int w = 0; w < WAVES; ++w) up += part[w][SIDE * XB + block][l];
    }
    const int m = m0 + block % XB * 8 + (l & 7), n = n0 + block / XB * 8 + (l >> 3) * 4;
    if (m >= p.M || n >= p.N) continue;
    f32x4 out = sum;
    if constexpr (GATED) {
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = act_of<F32>(p.act, sum[j]) * up[j];
      if (p.gu != nullptr) {
        float* row = p.gu + m * (2LL * p.N);
        *reinterpret_cast<f32x4*>(row + n) = sum;
        *reinterpret_cast<f32x4*>(row + p.N + n) = up;
      }
    }
    if constexpr (F32) {
      *reinterpret_cast<f32x4*>(static_cast<float*>(p.c) + m * p.ldc + n) = out;
    } else {
      unsigned short* to = static_cast<unsigned short*>(p.c) + m * p.ldc + n;
      const unsigned lo = pack_bf16(out[0], out[1]), hi = pack_bf16(out[2], out[3]);
      if ((p.N & 7) == 0) {
        *reinterpret_cast<u32x2*>(to) = u32x2{lo, hi};
      } else {  // rows of any width begin anywhere
        const unsigned short v[4] = {static_cast<unsigned short>(lo), static_cast<unsigned short>(lo >> 16),
                                     static_cast<unsigned short>(hi), static_cast<unsigned short>(hi >> 16)};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) to[j] = v[j];
      }
    }
  }
}

template <int KIND, bool GATED, int HB, int XB, int WAVES, int DEPTH>
static hipError_t go(const GemmArgs& p, hipStream_t stream) {
  constexpr int COLUMNS = (GATED ? HB / 2 : HB) * 8;
  const dim3 grid((p.N + COLUMNS - 1) / COLUMNS, (p.M + XB * 8 - 1) / (XB * 8));
  const int lds = skinny_lds_bytes<KIND, GATED, HB, XB, WAVES, DEPTH>(p.K / 32);
  hipLaunchKernelGGL((ffn_skinny_kernel<KIND, GATED, HB, XB, WAVES, DEPTH>), grid, dim3(WAVES * 64), lds, stream, p);
  return hipGetLastError();
}
// How many groups of 8 weight rows a workgroup takes. Reading is bound by the CUs: one gets about 16 bytes a clock
// however many waves ask (128 workgroups on rows of 8 / 16 KiB: 3.9 / 8.5 us, 256 with the same rows each
// 6.9 / 14.0), so what counts is what the fullest of the 256 CUs has to read: its workgroups' weight rows, and
// x once for each of them, which comes out of the L2 (or through LDS) at twice the rate.
// Measured, bf16: N=6144 gated, K=2048, T=1, 2 / 4 / 8 groups 9.3 / 11.4 / 11.2 us; N=2048, K=6144, T=1,
// 1 / 2 / 4 groups 5.7 / 8.1 / 13.4, T=16 10.3 / 12.8 / 18.7; MXFP4 weights N=4096, K=12288, T=16 15.6 / 10.4 / 13.5.
static int pick_groups(const GemmArgs& p, int least, int most, bool gated, double w_bytes, double x_bytes) {
  int best = least;
  double least_cost = 0;
  for (int hb = least; hb <= most; hb = hb == 4 && most == 6 ? 6 : hb * 2) {
    const long long columns = (gated ? hb / 2 : hb) * 8, groups = (p.N + columns - 1) / columns;
    const double cost = static_cast<double>((groups + 255) / 256) * (hb * 8 * w_bytes + 0.5 * p.M * x_bytes);
    if (hb == least || cost < least_cost) best = hb, least_cost = cost;
  }
  return best;
}

template <int KIND, int XB>
static hipError_t go_plain(const GemmArgs& p, hipStream_t stream) {
  constexpr double W = KIND == SKINNY_F32 ? 4 : KIND == SKINNY_BF16 ? 2 : 0.53, X = KIND == SKINNY_F32 ? 4 : KIND == SKINNY_MXFP4_BOTH ? 0.53 : 2;
  if constexpr (KIND == SKINNY_MXFP4_WEIGHTS) {
    // The waves' rows of x take LDS: with long rows eight waves a workgroup pay, with short ones there are few steps
    // for each. Measured over 8 K, 5 N and M = 1, 5, 12 (graphs of 24 calls), us, 4 / 8 waves: M=5, N=2048, K=1024 3.1 / 3.7,
    // 4096 5.4 / 5.4, 8192 7.5 / 6.9, 16384 12.0 / 9.6; N=8192 4.4 / 5.1, 7.0 / 7.6, 13.0 / 12.2, 21.0 / 19.9; M=12, N=512
    // 3.6 / 4.4, 5.7 / 5.5, 9.2 / 7.8, 15.4 / 11.4. Behind, of what this rule chooses, are M=12, N=16384, K=8192 with
    // 22.0 / 26.3 to K=12288 with 32.7 / 35.8, and by up to 10 % M=1 and 5 there with K=16384.
    const int hb = pick_groups(p, 2, 4, false, W, X);
    if (p.K >= 8192 && XB <= 2)
      return hb == 2 ? go<KIND, false, 2, XB, XB <= 2 ? 8 : 4, 1>(p, stream) : go<KIND, false, 4, XB, XB <= 2 ? 8 : 4, 1>(p, stream);
    return hb == 2 ? go<KIND, false, 2, XB, 4, 1>(p, stream) : go<KIND, false, 4, XB, 4, 1>(p, stream);
  } else {
    const int hb = pick_groups(p, 1, 4, false, W, X);
    if (hb == 1) return go<KIND, false, 1, XB, 8, 2>(p, stream);
    return hb == 2 ? go<KIND, false, 2, XB, 8, 2>(p, stream) : go<KIND, false, 4, XB, 8, 1>(p, stream);
  }
}

template <int KIND, int XB>
static hipError_t go_gated(const GemmArgs& p, hipStream_t stream) {
  constexpr double W = KIND == SKINNY_F32 ? 4 : KIND == SKINNY_BF16 ? 2 : 0.53, X = KIND == SKINNY_F32 ? 4 : 2;
  const int hb = pick_groups(p, 2, KIND == SKINNY_MXFP4_WEIGHTS ? 6 : 8, true, W, X);
  if constexpr (KIND == SKINNY_MXFP4_WEIGHTS) {
    if (hb == 6) return go<KIND, true, 6, XB, 4, 1>(p, stream);
    return hb == 2 ? go<KIND, true, 2, XB, 4, 1>(p, stream) : go<KIND, true, 4, XB, 4, 1>(p, stream);
  } else {
    if (hb == 2) return go<KIND, true, 2, XB, 8, 2>(p, stream);
    return hb == 4 ? go<KIND, true, 4, XB, 8, 1>(p, stream) : go<KIND, true, 8, XB, 8, 1>(p, stream);
  }
}

template <int KIND>
static hipError_t pick(bool gated, const GemmArgs& p, hipStream_t stream) {
  if constexpr (KIND != SKINNY_MXFP4_BOTH) {
    if (gated) return p.M <= 8 ? go_gated<KIND, 1>(p, stream) : p.M <= 16 ? go_gated<KIND, 2>(p, stream) : go_gated<KIND, 4>(p, stream);
  }
  return p.M <= 8 ? go_plain<KIND, 1>(p, stream) : p.M <= 16 ? go_plain<KIND, 2>(p, stream) : go_plain<KIND, 4>(p, stream);
}

bool ffn_skinny_takes(const GemmArgs& p) { return p.M <= 32; }

// (the scales of a workgroup's rows have to fit LDS beside the rest, and are read 4 bytes and more at a time)
bool mxfp4_skinny_takes(bool x_mxfp4, const GemmArgs& p) {
  const auto fours = [](const void* a) { return (reinterpret_cast<unsigned long long>(a) & 3) == 0; };
  return p.M <= 32 && p.K <= 16384 && fours(p.b_scales) && (!x_mxfp4 || fours(p.a_scales));
}

hipError_t launch_ffn_skinny(int dtype, bool gated, const GemmArgs& p, hipStream_t stream) {
  return dtype == 1 ? pick<SKINNY_BF16>(gated, p, stream) : pick<SKINNY_F32>(gated, p, stream);
}

hipError_t launch_mxfp4_skinny(bool x_mxfp4, bool gated, const GemmArgs& p, hipStream_t stream) {
  return x_mxfp4 ? pick<SKINNY_MXFP4_BOTH>(false, p, stream) : pick<SKINNY_MXFP4_WEIGHTS>(gated, p, stream);
}

}  // namespace fmoe
