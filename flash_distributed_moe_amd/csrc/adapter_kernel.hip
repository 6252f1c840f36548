// Low-rank adapters of many requests beside a shared projection: out_t = y_t + s (x_t A^T) B^T in bfloat16, with A [r, K], B [N, r]
// and s of the adapter that row t names; rows without one keep y_t.
//
// u = x A^T is summed in float32 and stays so between the two products (as two bfloat16 parts where the matrix
// instructions take it: what is left out is below 2^-16 of it); out is rounded once.
//
// Few rows are bound by the start of two kernels and by reading every row's adapter: a wave takes one row and two ranks of
// A, then a lane takes two columns of B, with vector instructions. Many rows are bound by reading x and reading and writing y.
// They are put in the order of their adapters (one workgroup counts and places them, so that rows in any order make whole
// tiles), then a tile's rows share their adapter's A and B on the matrix cores.
#include "ffn_device.h"
#include "lane_device.h"
#include "layer_params.h"

namespace fmoe {
namespace {

__device__ __forceinline__ float low(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high(unsigned u) { return __uint_as_float(u & 0xFFFF0000u); }
__device__ __forceinline__ const u32x4* piece(const void* p, size_t value) {
  return reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(p) + value * 2);
}

// ------------------------------------------------------------------ few rows
constexpr int kRanks = 2;  // of a wave

__global__ __launch_bounds__(256) void few_shrink_kernel(AdapterArgs a) {
  const int row = blockIdx.y, lane = threadIdx.x & 63, j = (blockIdx.x * 4 + (threadIdx.x >> 6)) * kRanks;
  const int id = a.ids[row];
  if (id < 0 || j >= a.r) return;
  if (id >= a.adapters) {
    if (lane < kRanks) a.u[static_cast<size_t>(row) * a.r + j + lane] = __uint_as_float(0x7FC00000u);
    return;
  }
  const size_t from = (static_cast<size_t>(id) * a.r + j) * a.K;
  float s[kRanks] = {};
#pragma unroll 4
  for (int k = lane * 8; k < a.K; k += 512) {
    const u32x4 x = *piece(a.x, static_cast<size_t>(row) * a.ldx + k);
    u32x4 w[kRanks];
#pragma unroll
    for (int i = 0; i < kRanks; ++i) w[i] = *piece(a.down, from + static_cast<size_t>(i) * a.K + k);
#pragma unroll
    for (int i = 0; i < kRanks; ++i) {
#pragma unroll
      for (int q = 0; q < 4; ++q) s[i] = fmaf(high(x[q]), high(w[i][q]), fmaf(low(x[q]), low(w[i][q]), s[i]));
    }
  }
#pragma unroll
  for (int i = 0; i < kRanks; ++i) {
    const float u = wave_sum(s[i]);
    if (lane == 0) a.u[static_cast<size_t>(row) * a.r + j + i] = u * a.scales[id];
  }
}

__global__ __launch_bounds__(256) void few_expand_kernel(AdapterArgs a) {
  const int row = blockIdx.y, n = (blockIdx.x * 256 + threadIdx.x) * 2;
  if (n >= a.N) return;
  const int id = a.ids[row];
  const unsigned y = *reinterpret_cast<const unsigned*>(reinterpret_cast<const unsigned short*>(a.y) + static_cast<size_t>(row) * a.ldy + n);
  float s0 = 0.0f, s1 = 0.0f;
  if (id >= 0) {
    const float* u = a.u + static_cast<size_t>(row) * a.r;
    // an adapter that is not there: its u is NaN, and any B will do
    const size_t from = (static_cast<size_t>(id < a.adapters ? id : 0) * a.N + n) * a.r;
#pragma unroll 4
    for (int j = 0; j < a.r; j += 8) {
      const u32x4 w0 = *piece(a.up, from + j), w1 = *piece(a.up, from + a.r + j);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        s0 = fmaf(u[j + 2 * q + 1], high(w0[q]), fmaf(u[j + 2 * q], low(w0[q]), s0));
        s1 = fmaf(u[j + 2 * q + 1], high(w1[q]), fmaf(u[j + 2 * q], low(w1[q]), s1));
      }
    }
  } else if (a.out == a.y) {
    return;
  }
  const unsigned sum = id < 0 ? y : pack_bf16(low(y) + s0, high(y) + s1);
  *reinterpret_cast<unsigned*>(reinterpret_cast<unsigned short*>(a.out) + static_cast<size_t>(row) * a.ldo + n) = sum;
}

// ------------------------------------------------------------------ many rows
constexpr int kPlaceThreads = 1024, kPlaceEach = 8;

// Adds one for every lane to its bucket and returns what was there before; lanes that agree with the wave's first one, as those
// of a run do, add together.
__device__ __forceinline__ int join_bucket(int* counts, int bucket, bool real) {
  const unsigned long long all = __ballot(real);
  if (all == 0) return 0;
  const int leader = __ffsll(static_cast<long long>(all)) - 1;
  const unsigned long long same = __ballot(real && bucket == __builtin_amdgcn_readlane(bucket, leader));
  const int lane = threadIdx.x & 63;
  int at = 0;
  if (lane == leader) at = atomicAdd(&counts[bucket], __popcll(same));
  at = __builtin_amdgcn_readlane(at, leader);
  if (same >> lane & 1) return at + __popcll(same & ((1ull << lane) - 1));
  return real ? atomicAdd(&counts[bucket], 1) : 0;
}

// Rows by adapter, then those without one, then those of an adapter that is not there; and the tiles they make. Which place a
// row of an adapter has among its others may differ from call to call; no result depends on it.
__global__ __launch_bounds__(kPlaceThreads) void place_kernel(AdapterArgs a) {
  __shared__ int counts[kPlaceThreads], begins[kPlaceThreads];
  __shared__ int wave_rows[16], wave_tiles[16];
  const int me = threadIdx.x;
  counts[me] = 0;
  __syncthreads();
  const auto bucket_of = [&](int id) { return id < 0 ? a.adapters : min(id, a.adapters + 1) + (id == a.adapters); };
  int kept[kPlaceEach];
  const long long chunk = kPlaceThreads * kPlaceEach;
  for (long long first = 0; first < a.T; first += chunk) {
#pragma unroll
    for (int i = 0; i < kPlaceEach; ++i) {
      const long long t = first + i * kPlaceThreads + me;
      kept[i] = t < a.T ? a.ids[t] : 0;
    }
#pragma unroll
    for (int i = 0; i < kPlaceEach; ++i) join_bucket(counts, bucket_of(kept[i]), first + i * kPlaceThreads + me < a.T);
  }
  __syncthreads();
  const int rows = counts[me], tiles = (rows + a.tile_rows - 1) / a.tile_rows;
  int rows_to = rows, tiles_to = tiles;
  for (int off = 1; off < 64; off <<= 1) {
    const int r = __shfl_up(rows_to, off, 64), t = __shfl_up(tiles_to, off, 64);
    if ((me & 63) >= off) rows_to += r, tiles_to += t;
  }
  if ((me & 63) == 63) wave_rows[me >> 6] = rows_to, wave_tiles[me >> 6] = tiles_to;
  __syncthreads();
  for (int w = 0; w < me >> 6; ++w) rows_to += wave_rows[w], tiles_to += wave_tiles[w];
  begins[me] = rows_to - rows;
  counts[me] = 0;
  for (int i = 0; i < tiles; ++i) {
    int* tile = a.tiles + (static_cast<size_t>(tiles_to) - tiles + i + 1) * 4;
    tile[0] = me, tile[1] = rows_to - rows + i * a.tile_rows, tile[2] = min(a.tile_rows, rows - i * a.tile_rows);
  }
  if (me == kPlaceThreads - 1) a.tiles[0] = tiles_to;
  __syncthreads();
  for (long long first = 0; first < a.T; first += chunk) {
    if (a.T > chunk) {
#pragma unroll
      for (int i = 0; i < kPlaceEach; ++i) {
        const long long t = first + i * kPlaceThreads + me;
        kept[i] = t < a.T ? a.ids[t] : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < kPlaceEach; ++i) {
      const long long t = first + i * kPlaceThreads + me;
      const int bucket = bucket_of(kept[i]), at = join_bucket(counts, bucket, t < a.T);
      if (t < a.T) a.order[begins[bucket] + at] = static_cast<int>(t);
    }
  }
}

__device__ __forceinline__ bf16x8 as_bf16(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }

// u of a tile: ranks are the rows of the matrix instruction's result and tokens its columns, so that a lane has four neighbouring
// ranks of one token. The waves of a workgroup deal its k among them and add their sums in LDS, in one order: (0 + 2) + (1 + 3).
// TB blocks of 16 tokens, RB of 16 ranks.
template <int TB, int RB>
__global__ __launch_bounds__(256) void shrink_kernel(AdapterArgs a) {
  __shared__ __align__(16) float sums[2][TB * 16][RB * 16 + 4];
  if (static_cast<int>(blockIdx.x) >= a.tiles[0]) return;
  const int* tile = a.tiles + (static_cast<size_t>(blockIdx.x) + 1) * 4;
  const int id = tile[0], first = tile[1], rows = tile[2];
  if (id >= a.adapters) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, of = lane & 15, group = lane >> 4;
  size_t token[TB];
#pragma unroll
  for (int b = 0; b < TB; ++b) token[b] = static_cast<size_t>(a.order[first + min(b * 16 + of, rows - 1)]) * a.ldx;
  const size_t from = static_cast<size_t>(id) * a.r * a.K;
  f32x4 acc[TB][RB] = {};
  // 64 k at a time, dealt to the waves of all the workgroups that share the tile
  for (int k0 = (blockIdx.y * 4 + wave) * 64; k0 < a.K; k0 += a.splits * 256) {
    u32x4 x[TB][2], w[RB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + h * 32 + group * 8;
#pragma unroll
      for (int b = 0; b < TB; ++b) x[b][h] = k < a.K ? *piece(a.x, token[b] + k) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int b = 0; b < RB; ++b)
        w[b][h] = k < a.K && b * 16 + of < a.r ? *piece(a.down, from + static_cast<size_t>(b * 16 + of) * a.K + k) : u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int b = 0; b < TB; ++b)
#pragma unroll
        for (int c = 0; c < RB; ++c)
          acc[b][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(w[c][h]), as_bf16(x[b][h]), acc[b][c], 0, 0, 0);
  }
  const auto place = [&](int b, int c) { return reinterpret_cast<f32x4*>(&sums[wave & 1][b * 16 + of][c * 16 + group * 4]); };
#pragma unroll
  for (int turn = 2; turn >= 0; turn -= 2) {
    if (turn == (wave & 2)) {
#pragma unroll
      for (int b = 0; b < TB; ++b)
#pragma unroll
        for (int c = 0; c < RB; ++c) *place(b, c) = turn == 0 ? acc[b][c] + *place(b, c) : acc[b][c];
    }
    __syncthreads();
  }
  float* u = a.u + (static_cast<size_t>(blockIdx.y) * a.T + first) * a.r;
  const int fours = a.r / 4;
  for (int i = threadIdx.x; i < rows * fours; i += 256) {
    const int t = i / fours, j = i % fours * 4;
    *reinterpret_cast<f32x4*>(u + static_cast<size_t>(t) * a.r + j) =
        *reinterpret_cast<const f32x4*>(&sums[0][t][j]) + *reinterpret_cast<const f32x4*>(&sums[1][t][j]);
  }
}

// Columns of B are the rows of the matrix instruction's result, dealt four at a time to four blocks, so that a lane has sixteen
// neighbouring columns of one token: row i of block f is column 16 (i / 4) + 4 f + i % 4. KS steps of 32 ranks.
constexpr int kUnit = 64;  // columns at a time
template <int KS>
__global__ __launch_bounds__(256) void expand_kernel(AdapterArgs a, int units) {
  if (static_cast<int>(blockIdx.x) >= a.tiles[0]) return;
  const int* tile = a.tiles + (static_cast<size_t>(blockIdx.x) + 1) * 4;
  const int id = tile[0], first = tile[1], rows = tile[2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, of = lane & 15, group = lane >> 4;
  // tiles of 64 rows: 16 a wave, the same columns; tiles of 16 rows: the waves deal the columns
  const bool tall = a.tile_rows == 64;
  const int mine = tall ? wave * 16 : 0;
  if (mine >= rows || (id == a.adapters && a.out == a.y)) return;
  const bool real = mine + of < rows;
  const int place = first + min(mine + of, rows - 1), row = a.order[place];
  const unsigned short* y = reinterpret_cast<const unsigned short*>(a.y) + static_cast<size_t>(row) * a.ldy;
  unsigned short* out = reinterpret_cast<unsigned short*>(a.out) + static_cast<size_t>(row) * a.ldo;
  const int begin = blockIdx.y * units * kUnit + (tall ? 0 : wave * kUnit), step = tall ? kUnit : 4 * kUnit;
  const int end = min(a.N, static_cast<int>(blockIdx.y + 1) * units * kUnit);
  if (id >= a.adapters) {
    const unsigned nan = 0x7FC07FC0u;
    for (int n = begin + group * 16; n < end; n += step) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (real && n + h * 8 < a.N)
          *reinterpret_cast<u32x4*>(out + n + h * 8) =
              id == a.adapters ? *reinterpret_cast<const u32x4*>(y + n + h * 8) : u32x4{nan, nan, nan, nan};
    }
    return;
  }
  // a token's u in two parts
  bf16x8 big[KS], rest[KS];
  const float scale = a.scales[id];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int j = s * 32 + group * 8;
    f32x4 v[2] = {};
    if (j < a.r) {
      for (int p = 0; p < a.splits; ++p) {
        const f32x4* u = reinterpret_cast<const f32x4*>(a.u + (static_cast<size_t>(p) * a.T + place) * a.r + j);
        v[0] += u[0], v[1] += u[1];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = v[i >> 2][i & 3] * scale;
      big[s][i] = static_cast<__bf16>(f);
      const float left = f - static_cast<float>(big[s][i]);
      rest[s][i] = static_cast<__bf16>(fabsf(left) < INFINITY ? left : 0.0f);  // of infinities nothing is left
    }
  }
  const size_t from = static_cast<size_t>(id) * a.N;
  for (int n = begin; n < end; n += step) {
    u32x4 have[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = n + group * 16 + h * 8;
      have[h] = c < a.N ? *reinterpret_cast<const u32x4*>(y + c) : u32x4{0, 0, 0, 0};
    }
    f32x4 acc[4] = {};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int j = s * 32 + group * 8;
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int c = n + 16 * (of >> 2) + 4 * f + (of & 3);
        const u32x4 w = j < a.r && c < a.N ? *piece(a.up, (from + c) * a.r + j) : u32x4{0, 0, 0, 0};
        acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(w), big[s], acc[f], 0, 0, 0);
        acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(w), rest[s], acc[f], 0, 0, 0);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = n + group * 16 + h * 8;
      u32x4 sum;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4& s = acc[2 * h + (q >> 1)];
        sum[q] = pack_bf16(low(have[h][q]) + s[(q & 1) * 2], high(have[h][q]) + s[(q & 1) * 2 + 1]);
      }
      if (real && c < a.N) *reinterpret_cast<u32x4*>(out + c) = sum;
    }
  }
}

template <int TB>
void enqueue_shrink(const AdapterArgs& a, hipStream_t stream) {
  const dim3 grid(a.most_tiles, a.splits), block(256);
  if (a.r <= 16) shrink_kernel<TB, 1><<<grid, block, 0, stream>>>(a);
  else if (a.r <= 32) shrink_kernel<TB, 2><<<grid, block, 0, stream>>>(a);
  else if (a.r <= 64) shrink_kernel<TB, 4><<<grid, block, 0, stream>>>(a);
  else shrink_kernel<TB, 8><<<grid, block, 0, stream>>>(a);
}

}  // namespace

hipError_t launch_adapters(const AdapterArgs& a, hipStream_t stream) {
  if (adapter_rows_alone(a.T)) {
    few_shrink_kernel<<<dim3((a.r + 4 * kRanks - 1) / (4 * kRanks), a.T), dim3(256), 0, stream>>>(a);
    few_expand_kernel<<<dim3((a.N + 511) / 512, a.T), dim3(256), 0, stream>>>(a);
    return hipGetLastError();
  }
  place_kernel<<<dim3(1), dim3(kPlaceThreads), 0, stream>>>(a);
  a.tile_rows == 64 ? enqueue_shrink<4>(a, stream) : enqueue_shrink<1>(a, stream);
  // columns of a workgroup: enough workgroups to fill the CUs, and no more than that so that u is read seldom
  const int all = (a.N + kUnit - 1) / kUnit;
  const long long parts = (1024 + a.most_tiles - 1LL) / a.most_tiles;
  int units = static_cast<int>((all + parts - 1) / parts);
  if (a.tile_rows == 16) units = (units + 3) / 4 * 4;
  const dim3 grid(a.most_tiles, (all + units - 1) / units), block(256);
  if (a.r <= 32) expand_kernel<1><<<grid, block, 0, stream>>>(a, units);
  else if (a.r <= 64) expand_kernel<2><<<grid, block, 0, stream>>>(a, units);
  else expand_kernel<4><<<grid, block, 0, stream>>>(a, units);
  return hipGetLastError();
}

}  // namespace fmoe
