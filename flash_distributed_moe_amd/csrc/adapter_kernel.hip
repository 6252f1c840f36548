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
  __shared__ int counts[kPlaceThreads], begins[kPlaceThreads], ends[kPlaceThreads], tile_ends[kPlaceThreads];
  __shared__ int wave_rows[16], wave_tiles[16];
  const int me = threadIdx.x;
  counts[me] = 0;
  __syncthreads();
  const auto bucket_of = [&](int id) { return id < 0 ? a.adapters : min(id, a.adapters + 1) + (id == a.adapters); };
  int kept[kPlaceEach], rank[kPlaceEach];
  const long long chunk = kPlaceThreads * kPlaceEach;
  for (long long first = 0; first < a.T; first += chunk) {
#pragma unroll
    for (int i = 0; i < kPlaceEach; ++i) {
      const long long t = first + i * kPlaceThreads + me;
      kept[i] = t < a.T ? a.ids[t] : 0;
    }
#pragma unroll
    for (int i = 0; i < kPlaceEach; ++i)
      rank[i] = join_bucket(counts, bucket_of(kept[i]), first + i * kPlaceThreads + me < a.T);
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
  begins[me] = rows_to - rows, ends[me] = rows_to, tile_ends[me] = tiles_to;
  counts[me] = 0;
  __syncthreads();
  const int total = tile_ends[kPlaceThreads - 1];
  if (me == 0) a.tiles[0] = total;
  for (int i = me; i < total; i += kPlaceThreads) {
    // the first bucket that ends behind tile i has it
    int low = 0, high = kPlaceThreads - 1;
    while (low < high) {
      const int mid = (low + high) / 2;
      if (tile_ends[mid] > i) high = mid;
      else low = mid + 1;
    }
    const int all = ends[low] - begins[low], mine = i - (tile_ends[low] - (all + a.tile_rows - 1) / a.tile_rows);
    int* tile = a.tiles + (static_cast<size_t>(i) + 1) * 4;
    tile[0] = low, tile[1] = begins[low] + mine * a.tile_rows, tile[2] = min(a.tile_rows, all - mine * a.tile_rows);
  }
  for (long long first = 0; first < a.T; first += chunk) {
    // more rows than the threads hold: counted a second time
    if (a.T > chunk) {
#pragma unroll
      for (int i = 0; i < kPlaceEach; ++i) {
        const long long t = first + i * kPlaceThreads + me;
        kept[i] = t < a.T ? a.ids[t] : 0;
      }
#pragma unroll
      for (int i = 0; i < kPlaceEach; ++i) rank[i] = join_bucket(counts, bucket_of(kept[i]), first + i * kPlaceThreads + me < a.T);
    }
#pragma unroll
    for (int i = 0; i < kPlaceEach; ++i) {
      const long long t = first + i * kPlaceThreads + me;
      if (t < a.T) a.order[begins[bucket_of(kept[i])] + rank[i]] = static_cast<int>(t);
    }
  }
}

// The matrix instructions give a lane pieces of one token of sixteen, so that a load of one piece a lane would be 64 bytes of
// each of sixteen rows; memory is read and written at half again that rate where it is 128 bytes of eight rows (an array of 8192
// x 12288 there and back 81 us instead of 102). So two loads of four lanes' pieces of sixteen rows are made as one of eight lanes' of the
// first eight and one of the last eight, and the lanes eight apart exchange what is the other's. Takes either form to the other.
__device__ __forceinline__ void exchange(u32x4& p, u32x4& q) {
  const bool lower = (threadIdx.x & 8) == 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned got = static_cast<unsigned>(dpp<kRotate8>(static_cast<int>(lower ? q[i] : p[i])));
    p[i] = lower ? p[i] : got;
    q[i] = lower ? got : q[i];
  }
}

__device__ __forceinline__ bf16x8 as_bf16(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }

// u of a tile: ranks are the rows of the matrix instruction's result and tokens its columns, so that a lane has four neighbouring
// ranks of one token. The waves of a workgroup deal its k among them and add their sums in LDS, in one order.
// TB blocks of 16 tokens, RB of 16 ranks.
constexpr int kShrinkWaves = 4;
template <int TB, int RB>
__global__ __launch_bounds__(kShrinkWaves * 64, TB * RB < 32 ? 2 : 1) void shrink_kernel(AdapterArgs a) {
  __shared__ __align__(16) float sums[kShrinkWaves / 2][TB * 16][RB * 16 + 4];
  if (static_cast<int>(blockIdx.x) >= a.tiles[0]) return;
  const int* tile = a.tiles + (static_cast<size_t>(blockIdx.x) + 1) * 4;
  const int id = tile[0], first = tile[1], rows = tile[2];
  if (id >= a.adapters) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, of = lane & 15, group = lane >> 4;
  // what a lane loads: of tokens 0 to 7 of a block and of 8 to 15, 16 of 128 bytes
  const int eighth = (of >> 3) * 32 + group * 8;
  size_t token[TB][2];
#pragma unroll
  for (int b = 0; b < TB; ++b)
#pragma unroll
    for (int h = 0; h < 2; ++h) token[b][h] = static_cast<size_t>(a.order[first + min(b * 16 + h * 8 + (of & 7), rows - 1)]) * a.ldx + eighth;
  size_t rank[RB][2];  // ranks behind the last one are read as the last one, and nobody reads their sums
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      rank[b][h] = (static_cast<size_t>(id) * a.r + min(b * 16 + h * 8 + (of & 7), a.r - 1)) * a.K + eighth;
  f32x4 acc[TB][RB] = {};
  const auto step = [&](int k0, auto load) {
    u32x4 x[TB][2], w[RB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int b = 0; b < TB; ++b) x[b][h] = load(a.x, token[b][h], k0, eighth);
#pragma unroll
      for (int b = 0; b < RB; ++b) w[b][h] = load(a.down, rank[b][h], k0, eighth);
    }
#pragma unroll
    for (int b = 0; b < TB; ++b) exchange(x[b][0], x[b][1]);
#pragma unroll
    for (int b = 0; b < RB; ++b) exchange(w[b][0], w[b][1]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int b = 0; b < TB; ++b)
#pragma unroll
        for (int c = 0; c < RB; ++c)
          acc[b][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(w[c][h]), as_bf16(x[b][h]), acc[b][c], 0, 0, 0);
  };
  // 64 k at a time, dealt to the waves of all the workgroups that share the tile
  int k0 = (blockIdx.y * kShrinkWaves + wave) * 64;
  for (; k0 + 64 <= a.K; k0 += a.splits * kShrinkWaves * 64)
    step(k0, [](const void* p, size_t at, int k, int) { return *piece(p, at + k); });
  if (k0 < a.K)
    step(k0, [&](const void* p, size_t at, int k, int in) { return k + in < a.K ? *piece(p, at + k) : u32x4{0, 0, 0, 0}; });
  // the upper half of the waves leave their sums, the lower half add theirs
  constexpr int kHalf = kShrinkWaves / 2;
  const auto place = [&](int b, int c) { return reinterpret_cast<f32x4*>(&sums[wave % kHalf][b * 16 + of][c * 16 + group * 4]); };
#pragma unroll
  for (int upper = 1; upper >= 0; --upper) {
    if (upper == wave / kHalf) {
#pragma unroll
      for (int b = 0; b < TB; ++b)
#pragma unroll
        for (int c = 0; c < RB; ++c) *place(b, c) = upper ? acc[b][c] : acc[b][c] + *place(b, c);
    }
    __syncthreads();
  }
  float* u = a.u + (static_cast<size_t>(blockIdx.y) * a.T + first) * a.r;
  const int fours = a.r / 4;
  for (int i = threadIdx.x; i < rows * fours; i += kShrinkWaves * 64) {
    const int t = i / fours, j = i % fours * 4;
    f32x4 s = *reinterpret_cast<const f32x4*>(&sums[0][t][j]);
#pragma unroll
    for (int w = 1; w < kHalf; ++w) s += *reinterpret_cast<const f32x4*>(&sums[w][t][j]);
    *reinterpret_cast<f32x4*>(u + static_cast<size_t>(t) * a.r + j) = s;
  }
}

// Columns of B are the rows of the matrix instruction's result, dealt four at a time to two blocks, so that a lane has eight
// neighbouring columns of one token: row i of block f is column 32 (f / 2) + 8 (i / 4) + 4 (f % 2) + i % 4 of a unit of 64. A wave has 16
// tokens. KS steps of 32 ranks.
constexpr int kUnit = 64;
constexpr float kMostBf16 = 0x1.FEp127f;
template <int KS>
struct Tokens {
  const unsigned short* y[2];  // what a lane loads and stores: of tokens 0 to 7 and of 8 to 15, 16 of 128 bytes
  unsigned short* out[2];
  bool real[2];
  int eighth;
  bf16x8 big[KS], rest[KS];  // u in two parts
};
// The tokens from place `part` of a tile of `rows` on; places behind the last one stand for it, and are not stored.
template <int KS>
__device__ __forceinline__ void find_tokens(const AdapterArgs& a, Tokens<KS>& t, int first, int rows, int part) {
  const int of = threadIdx.x & 15, group = threadIdx.x >> 4 & 3;
  t.eighth = (of >> 3) * 32 + group * 8;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = part + h * 8 + (of & 7);
    const size_t row = a.order[first + min(at, rows - 1)];
    t.y[h] = reinterpret_cast<const unsigned short*>(a.y) + row * a.ldy;
    t.out[h] = reinterpret_cast<unsigned short*>(a.out) + row * a.ldo + t.eighth;
    t.real[h] = at < rows;
  }
}
// Columns behind the last ones are read as the last ones, and not stored: no load has a branch of its own.
template <int KS>
__device__ __forceinline__ void load_y(const AdapterArgs& a, const Tokens<KS>& t, int n, u32x4 (&have)[2]) {
  const int c = min(n + t.eighth, a.N - 8);
#pragma unroll
  for (int h = 0; h < 2; ++h) have[h] = *reinterpret_cast<const u32x4*>(t.y[h] + c);
}
template <int KS>
__device__ __forceinline__ void store_y(const AdapterArgs& a, const Tokens<KS>& t, int n, const u32x4 (&v)[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (t.real[h] && n + t.eighth < a.N) *reinterpret_cast<u32x4*>(t.out[h] + n) = v[h];
}
template <int KS>
__device__ __forceinline__ void load_u(const AdapterArgs& a, Tokens<KS>& t, int id, int first, int rows, int part) {
  const int of = threadIdx.x & 15, group = threadIdx.x >> 4 & 3;
  const size_t place = first + min(part + of, rows - 1);
  const float scale = a.scales[id];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int j = s * 32 + group * 8;
    f32x4 v[2] = {};
    if (j < a.r) {
      for (int p = 0; p < a.splits; p += 4) {  // four at a time in flight; behind the last one it is read again, for nothing
        f32x4 u[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float* from = a.u + (static_cast<size_t>(min(p + i, a.splits - 1)) * a.T + place) * a.r + j;
          u[i][0] = *reinterpret_cast<const f32x4*>(from), u[i][1] = *reinterpret_cast<const f32x4*>(from + 4);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (p + i < a.splits) v[0] += u[i][0], v[1] += u[i][1];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = v[i >> 2][i & 3] * scale;
      // a number beyond the greatest of bfloat16 would be rounded to infinity: what it is more than that is the rest's
      const float held = fabsf(f) < INFINITY ? __builtin_amdgcn_fmed3f(f, -kMostBf16, kMostBf16) : f;
      t.big[s][i] = static_cast<__bf16>(held);
      const float left = f - static_cast<float>(t.big[s][i]);
      t.rest[s][i] = static_cast<__bf16>(fabsf(left) < INFINITY ? left : 0.0f);  // of infinities nothing is left
    }
  }
}
// have: y on the way in, the results on the way out. w(s, f): B's fragment of step s, block f.
template <int KS, typename W>
__device__ __forceinline__ void add_unit(const Tokens<KS>& t, u32x4 (&have)[2], W w) {
  f32x4 acc[4] = {};
#pragma unroll
  for (int s = 0; s < KS; ++s) {
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const bf16x8 b = as_bf16(w(s, f));
      acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, t.big[s], acc[f], 0, 0, 0);
      acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, t.rest[s], acc[f], 0, 0, 0);
    }
  }
  exchange(have[0], have[1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4& s = acc[2 * h + (q >> 1)];
      have[h][q] = pack_bf16(low(have[h][q]) + s[(q & 1) * 2], high(have[h][q]) + s[(q & 1) * 2 + 1]);
    }
  }
  exchange(have[0], have[1]);
}
// Rows without an adapter, and rows whose adapter is not there.
template <int KS>
__device__ __forceinline__ void pass_on(const AdapterArgs& a, const Tokens<KS>& t, int id, int begin, int end, int step) {
  if (id == a.adapters && a.out == a.y) return;
  const u32x4 nan = {0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
  for (int n = begin; n < end; n += step) {
    u32x4 have[2];
    load_y(a, t, n, have);
    if (id != a.adapters) have[0] = have[1] = nan;
    store_y(a, t, n, have);
  }
}

// Tiles of 16 rows: the waves deal the columns, and each asks for its B itself. (Two sets of registers in turn: copied from one to the
// other they would be waited for.)
template <int KS>
__global__ __launch_bounds__(256) void expand_kernel(AdapterArgs a, int units) {
  if (static_cast<int>(blockIdx.x) >= a.tiles[0]) return;
  const int* tile = a.tiles + (static_cast<size_t>(blockIdx.x) + 1) * 4;
  const int id = tile[0], first = tile[1], rows = tile[2];
  const int wave = threadIdx.x >> 6, of = threadIdx.x & 15, group = threadIdx.x >> 4 & 3;
  const int begin = (blockIdx.y * units * 4 + wave) * kUnit, step = 4 * kUnit;
  const int end = min(a.N, static_cast<int>(blockIdx.y + 1) * units * 4 * kUnit);
  if (begin >= end) return;
  Tokens<KS> t;
  find_tokens(a, t, first, rows, 0);
  if (id >= a.adapters) return pass_on(a, t, id, begin, end, step);
  const size_t from = static_cast<size_t>(id) * a.N;
  const auto load_w = [&](int n, u32x4 (&w)[KS][4]) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int j = min(s * 32 + group * 8, a.r - 8);
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int c = min(n + 32 * (f >> 1) + 8 * (of >> 2) + 4 * (f & 1) + (of & 3), a.N - 1);
        w[s][f] = *piece(a.up, (from + c) * a.r + j);
      }
    }
  };
  const auto unit = [&](int n, const u32x4 (&w)[KS][4], u32x4 (&have)[2], u32x4 (&next_w)[KS][4], u32x4 (&next)[2]) {
    if (n + step < end) load_w(n + step, next_w), load_y(a, t, n + step, next);
    add_unit(t, have, [&](int s, int f) { return s * 32 + group * 8 < a.r ? w[s][f] : u32x4{0, 0, 0, 0}; });
    store_y(a, t, n, have);
  };
  u32x4 have0[2], have1[2], w0[KS][4], w1[KS][4];
  load_y(a, t, begin, have0);
  load_w(begin, w0);
  load_u(a, t, id, first, rows, 0);
  for (int n = begin;;) {
    unit(n, w0, have0, w1, have1);
    if ((n += step) >= end) break;
    unit(n, w1, have1, w0, have0);
    if ((n += step) >= end) break;
  }
}

// Tiles of 64 rows: 16 a wave, which share B's columns through LDS, two units in turn. There a unit lies as the matrix
// instruction takes it, a fragment's 64 pieces side by side, and in memory it is one run. (Each wave asking for its own B, for 32 rows
// of its own, took 120 us where this takes 89: 8192 rows, N=12288, rank 64. Without any B that one took 91.)
template <int KS>
__global__ __launch_bounds__(256) void expand_tall_kernel(AdapterArgs a, int units, int chunks) {
  __shared__ __align__(16) u32x4 shared[2][KS * 4 * 64];
  const int which = blockIdx.x / chunks, chunk = blockIdx.x % chunks;  // neighbours have a tile's rows, and an XCD has columns of its own
  if (which >= a.tiles[0]) return;
  const int* tile = a.tiles + (static_cast<size_t>(which) + 1) * 4;
  const int id = tile[0], first = tile[1], rows = tile[2];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int begin = chunk * units * kUnit, end = min(a.N, (chunk + 1) * units * kUnit);
  if (begin >= end) return;
  Tokens<KS> t;
  find_tokens(a, t, first, rows, wave * 16);
  if (id >= a.adapters) return pass_on(a, t, id, begin, end, kUnit);
  const int pieces = a.r / 8;                       // of a column
  const unsigned all = static_cast<unsigned>(a.N) * pieces;
  const char* from = reinterpret_cast<const char*>(a.up) + static_cast<size_t>(id) * all * 16;
  // where in a unit's fragments the pieces that this thread fetches lie
  int place[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    const int q = threadIdx.x + i * 256, c = q / pieces, p = q % pieces;
    place[i] = c < kUnit ? ((p >> 2) * 4 + 2 * (c >> 5) + (c >> 2 & 1)) * 64 + (p & 3) * 16 + (c >> 3 & 3) * 4 + (c & 3) : -1;
  }
  const auto fetch = [&](int n, u32x4 (&w)[KS]) {
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const unsigned q = static_cast<unsigned>(n) * pieces + threadIdx.x + i * 256;
      w[i] = *reinterpret_cast<const u32x4*>(from + static_cast<size_t>(min(q, all - 1)) * 16);
    }
  };
  const auto keep = [&](int turn, const u32x4 (&w)[KS]) {
#pragma unroll
    for (int i = 0; i < KS; ++i)
      if (place[i] >= 0) shared[turn][place[i]] = w[i];
  };
  const auto meet = [] {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // ranks that are none are zeros
  for (int i = threadIdx.x; i < 2 * KS * 4 * 64; i += 256)
    if ((i >> 8) % KS * 32 + (i >> 4 & 3) * 8 >= a.r) shared[0][i] = u32x4{0, 0, 0, 0};
  u32x4 have0[2], have1[2], w0[KS], w1[KS];
  fetch(begin, w0);
  load_y(a, t, begin, have0);
  if (begin + kUnit < end) fetch(begin + kUnit, w1);
  load_u(a, t, id, first, rows, wave * 16);
  keep(0, w0);
  meet();
  // a unit's B arrives two units ahead, its y one
  const auto unit = [&](int n, int turn, u32x4 (&have)[2], u32x4 (&next)[2], u32x4 (&coming)[KS], u32x4 (&free)[KS]) {
    if (n + 2 * kUnit < end) fetch(n + 2 * kUnit, free);
    if (n + kUnit < end) load_y(a, t, n + kUnit, next), keep(turn ^ 1, coming);
    add_unit(t, have, [&](int s, int f) { return shared[turn][(s * 4 + f) * 64 + lane]; });
    store_y(a, t, n, have);
    meet();
  };
  for (int n = begin;;) {
    unit(n, 0, have0, have1, w1, w0);
    if ((n += kUnit) >= end) break;
    unit(n, 1, have1, have0, w0, w1);
    if ((n += kUnit) >= end) break;
  }
}

template <int TB>
void enqueue_shrink(const AdapterArgs& a, hipStream_t stream) {
  const dim3 grid(a.most_tiles, a.splits), block(kShrinkWaves * 64);
  if (a.r <= 16) return shrink_kernel<TB, 1><<<grid, block, 0, stream>>>(a);
  if (a.r <= 32) return shrink_kernel<TB, 2><<<grid, block, 0, stream>>>(a);
  if (a.r <= 64) return shrink_kernel<TB, 4><<<grid, block, 0, stream>>>(a);
  shrink_kernel<TB, 8><<<grid, block, 0, stream>>>(a);
}

template <int KS>
void enqueue_expand(const AdapterArgs& a, hipStream_t stream) {
  // Columns of a workgroup. The last ones to start leave CUs idle (8192 rows, N=12288, rank 64 with about 1000, 2000, 3300 and 5000
  // workgroups 99, 91, 89 and 96 us), but every one reads its tokens' u again, all parts of it: at least as many units as keep that
  // to a fifth of what y takes (1024 rows, K=N=4096, rank 128 113 us without that, 45 with it), but for the eight that an XCD each
  // has. Of 16 rows the waves have four units at a time, and no such eight: there that rule leaves few workgroups where k is split most (256
  // rows, K=N=4096, rank 128, 8 parts: one for each of 16 to 24 tiles, 45 us of the call's 60).
  const bool tall = a.tile_rows == 64;
  const int across = (tall ? 1 : 4) * kUnit, all = (a.N + across - 1) / across;
  const long long wanted = ((tall ? 3300 : 1024) + a.most_tiles - 1LL) / a.most_tiles;
  const int least = (a.r * a.splits + (tall ? 16 : 64) - 1) / (tall ? 16 : 64);
  int units = static_cast<int>(max((all + wanted - 1) / wanted, static_cast<long long>(least)));
  int chunks = (all + units - 1) / units;
  if (tall) {
    chunks = (chunks + 7) / 8 * 8, units = (all + chunks - 1) / chunks;  // columns of an XCD's own
    return expand_tall_kernel<KS><<<dim3(a.most_tiles * chunks), dim3(256), 0, stream>>>(a, units, chunks);
  }
  expand_kernel<KS><<<dim3(a.most_tiles, chunks), dim3(256), 0, stream>>>(a, units);
}

}  // namespace

hipError_t launch_adapters(const AdapterArgs& a, hipStream_t stream) {
  if (adapter_rows_alone(a)) {
    few_shrink_kernel<<<dim3((a.r + 4 * kRanks - 1) / (4 * kRanks), a.T), dim3(256), 0, stream>>>(a);
    few_expand_kernel<<<dim3((a.N + 511) / 512, a.T), dim3(256), 0, stream>>>(a);
    return hipGetLastError();
  }
  place_kernel<<<dim3(1), dim3(kPlaceThreads), 0, stream>>>(a);
  a.tile_rows == 64 ? enqueue_shrink<4>(a, stream) : enqueue_shrink<1>(a, stream);
  a.r <= 32 ? enqueue_expand<1>(a, stream) : a.r <= 64 ? enqueue_expand<2>(a, stream) : enqueue_expand<4>(a, stream);
  return hipGetLastError();
}

}  // namespace fmoe
