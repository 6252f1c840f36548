// The norms around a block, fused with what joins it to the residual stream:
//   z = post * branch / rms(branch)  (or the branch as it is),  y = alpha x + beta gate z,  h = next * y / rms(y)
// with rms(v) = sqrt(mean v^2 + eps), and the gradients. Without a branch y = x: the norm in front of a block alone.
//
// Backward, with u = branch / rms and v = y / rms(y), both rebuilt from the inputs (what was rounded into y is not used again):
//   t = dy + (next dh - v mean(next dh v)) / rms(y),  dx = alpha t,  dgate = beta t z,  dpost = beta sum gate t u,
//   dbranch = (q - u mean(q u)) / rms(branch) with q = beta gate post t,  dnext = sum dh v
// A gate a channel and the post norm's weight have one sum between them: with S = sum t u, dgate = beta post S and dpost = beta gate S.
// With a gate a token sum q u = gate dgate, so its gradient needs no sum of its own.
//
// Bound by memory: every array is read or written once, rows stay in registers between the two norms (8192 x 4096 in bfloat16 with both
// norms and a gate a channel 50 us forward, 5.4 TB/s, and 81 backward, 5.0; a copy of 256 MB reaches 5.35). A row belongs to one
// wave or to several, which exchange their sums through LDS; the backward pass's column sums stay in registers over all rows of a
// workgroup and are joined by a second kernel, in one order.
#include "ffn_device.h"
#include "lane_device.h"
#include "layer_params.h"

namespace fmoe {
namespace {

template <bool BF>
constexpr int kPiece = BF ? 8 : 4;  // values in 16 bytes

// A row, or a vector, of `count` pieces of 16 bytes. Through a descriptor of its own: what is asked for behind its end arrives as zeros,
// and what is stored there is dropped, so no access has a branch. A row that is not `real` has no pieces: it counts as zeros.
struct Row {
  __amdgpu_buffer_rsrc_t rsrc;
};
template <bool BF>
__device__ __forceinline__ Row row_at(const void* p, size_t at, int count, bool real = true) {
  return {make_rsrc(reinterpret_cast<const char*>(p) + at * (BF ? 2 : 4), real ? count * 16u : 0u)};
}
// V pieces of a row: piece i of a lane is number i * lanes + its own.
template <int V>
struct Pieces {
  u32x4 u[V];
};
template <int V>
__device__ __forceinline__ Pieces<V> load_pieces(const Row& row, int first, int lanes) {
  Pieces<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i)
    r.u[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(row.rsrc, (first + i * lanes) * 16, 0, 0));
  return r;
}
template <bool BF>
__device__ __forceinline__ float piece_value(const u32x4& u, int j) {
  if constexpr (BF) return __uint_as_float(j & 1 ? u[j >> 1] & 0xFFFF0000u : u[j >> 1] << 16);
  return __uint_as_float(u[j]);
}
template <bool BF>
__device__ __forceinline__ u32x4 pack_piece(const float* v) {
  if constexpr (BF) return u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
  return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
template <bool BF, int V>
__device__ __forceinline__ void store_pieces(const Row& row, int first, int lanes, const float* v) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    __builtin_amdgcn_raw_buffer_store_b128(pack_piece<BF>(v + i * kPiece<BF>), row.rsrc, (first + i * lanes) * 16, 0, 0);
}
template <bool BF>
__device__ __forceinline__ float one_value(const void* p, size_t at) {
  if constexpr (BF) return __uint_as_float(unsigned(reinterpret_cast<const unsigned short*>(p)[at]) << 16);
  return reinterpret_cast<const float*>(p)[at];
}
template <bool BF>
__device__ __forceinline__ void put_value(void* p, size_t at, float v) {
  if constexpr (BF) reinterpret_cast<unsigned short*>(p)[at] = static_cast<unsigned short>(pack_bf16(v, v));
  else reinterpret_cast<float*>(p)[at] = v;
}

// The sum over a row's waves; `room` has a place for each wave of the workgroup. Every wave comes by.
__device__ __forceinline__ float row_sum(float v, int waves, float* room) {
  v = wave_sum(v);
  if (waves == 1) return v;
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) room[wave] = v;
  __syncthreads();
  const int first = wave & ~(waves - 1);
  float sum = 0.0f;
  for (int i = 0; i < waves; ++i) sum += room[first + i];
  return sum;
}

__device__ __forceinline__ size_t gate_row(const NormArgs& a, long long row) {
  return a.gate_kind == GATE_CHANNEL ? 0 : a.gate_kind == GATE_GROUP ? row / a.shared : row;
}

template <bool BF, int V>
__global__ void norm_kernel(NormArgs a, int waves) {
  constexpr int P = kPiece<BF>, N = V * P;
  __shared__ float room[2][16];
  const int lanes = waves * 64, first = threadIdx.x & (lanes - 1), count = a.H / P;
  const int at_once = blockDim.x / lanes, mine = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / waves;
  // the weights are on their way before a row's sums are waited for
  const Pieces<V> wp = load_pieces<V>(row_at<BF>(a.post != nullptr ? a.post : a.x, 0, count, a.post != nullptr), first, lanes);
  const Pieces<V> wn = load_pieces<V>(row_at<BF>(a.next != nullptr ? a.next : a.x, 0, count, a.next != nullptr), first, lanes);
  for (long long start = static_cast<long long>(blockIdx.x) * at_once; start < a.T; start += static_cast<long long>(gridDim.x) * at_once) {
    const bool real = start + mine < a.T;
    const long long row = real ? start + mine : a.T - 1;
    const Pieces<V> x = load_pieces<V>(row_at<BF>(a.x, row * a.ldx, count, real), first, lanes);
    float y[N];
    if (a.branch != nullptr) {
      const Pieces<V> b = load_pieces<V>(row_at<BF>(a.branch, row * a.ldb, count, real), first, lanes);
      Pieces<V> g{};
      float scale = a.beta;
      if (a.gate_kind == GATE_TOKEN) scale *= one_value<BF>(a.gate, row);
      else if (a.gate_kind != GATE_NONE) g = load_pieces<V>(row_at<BF>(a.gate, gate_row(a, row) * a.H, count), first, lanes);
      if (a.post != nullptr) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(piece_value<BF>(b.u[i / P], i % P), piece_value<BF>(b.u[i / P], i % P), s);
        const float rms = rsqrtf(row_sum(s, waves, room[0]) / a.H + a.eps);
        if (first == 0 && real && a.branch_rms != nullptr) a.branch_rms[row] = rms;
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = piece_value<BF>(b.u[i / P], i % P) * rms * piece_value<BF>(wp.u[i / P], i % P);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = piece_value<BF>(b.u[i / P], i % P);
      }
      if (a.gate_kind != GATE_NONE && a.gate_kind != GATE_TOKEN) {
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] *= piece_value<BF>(g.u[i / P], i % P);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = fmaf(scale, y[i], a.alpha * piece_value<BF>(x.u[i / P], i % P));
      store_pieces<BF, V>(row_at<BF>(a.y, row * a.H, count, real), first, lanes, y);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = piece_value<BF>(x.u[i / P], i % P);
    }
    if (a.next != nullptr) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) s = fmaf(y[i], y[i], s);
      const float rms = rsqrtf(row_sum(s, waves, room[1]) / a.H + a.eps);
      if (first == 0 && real && a.y_rms != nullptr) a.y_rms[row] = rms;
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = y[i] * rms * piece_value<BF>(wn.u[i / P], i % P);
      store_pieces<BF, V>(row_at<BF>(a.h, row * a.H, count, real), first, lanes, y);
    }
    // a wave that is ahead writes its next sums where another may still read these
    if (waves > 1 && (a.post == nullptr || a.next == nullptr)) __syncthreads();
  }
}

// The workgroup's column sums: each row's waves have one, and they are added in one order. To `to`, or times `scale` and `by`
// rounded to `rounded`.
template <bool BF, int THREADS>
__device__ __forceinline__ void join_rows(const float* acc, float* room, int lanes, int first, int count, float* to, void* rounded = nullptr,
                                          float scale = 1.0f, const void* by = nullptr) {
  constexpr int P = kPiece<BF>, V = kNormLane / P;
  const int mine = threadIdx.x / lanes, rows = THREADS / lanes;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int n = first + i * lanes;
    if (n < count) {
#pragma unroll
      for (int j = 0; j < P; ++j) room[mine * count * P + n * P + j] = acc[i * P + j];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < count * P; c += THREADS) {
    float s = 0.0f;
    for (int r = 0; r < rows; ++r) s += room[r * count * P + c];
    if (rounded != nullptr) put_value<BF>(rounded, c, by != nullptr ? s * scale * one_value<BF>(by, c) : s * scale);
    else to[c] = s;
  }
}

// With c = beta gate post for a column (of a gate a token or a full one beta post, the gate comes to it row by row) y = alpha x + c u and
// q = c t, so that a row needs little of the weights, and sums over rows of t u give the gradients of both.
template <bool BF, int GATE, int THREADS>
__global__ __launch_bounds__(THREADS, 2) void norm_backward_kernel(NormArgs a) {
  constexpr int P = kPiece<BF>, V = kNormLane / P, N = kNormLane;
  constexpr bool kGroup = GATE == GATE_GROUP;
  __shared__ float room[2][16];
  extern __shared__ __align__(16) float columns[];
  const int waves = norm_waves(a.H), lanes = waves * 64, first = threadIdx.x & (lanes - 1), count = a.H / P;
  const int at_once = THREADS / lanes, mine = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / waves;
  const bool next = a.next != nullptr && a.dh != nullptr, post = a.post != nullptr, branch = a.branch != nullptr;
  float sum_next[N], sum[N], sum_post[kGroup ? N : 1];  // of dh v, of t u (gate t u with a gate a token or a full one); of groups' gate t u
#pragma unroll
  for (int i = 0; i < N; ++i) {
    sum_next[i] = 0.0f, sum[i] = 0.0f;
    if constexpr (kGroup) sum_post[i] = 0.0f;
  }
  float wn[N], c[N];
  {
    const Pieces<V> w = load_pieces<V>(row_at<BF>(next ? a.next : a.x, 0, count, next), first, lanes);
    const Pieces<V> p = load_pieces<V>(row_at<BF>(post ? a.post : a.x, 0, count, post), first, lanes);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      wn[i] = piece_value<BF>(w.u[i / P], i % P);
      c[i] = post ? a.beta * piece_value<BF>(p.u[i / P], i % P) : a.beta;
    }
    if constexpr (GATE == GATE_CHANNEL) {
      const Pieces<V> g = load_pieces<V>(row_at<BF>(a.gate, 0, count), first, lanes);
#pragma unroll
      for (int i = 0; i < N; ++i) c[i] *= piece_value<BF>(g.u[i / P], i % P);
    }
  }

  // the rows of this workgroup: of all, or of one group after the other
  long long group = 0, groups = 1;
  if constexpr (kGroup) {
    if (a.parts > 0) group = blockIdx.x / a.parts;
    else group = static_cast<long long>(blockIdx.x) * a.groups, groups = min(static_cast<long long>(a.groups), a.T / a.shared - group);
  }
  for (const long long last = group + groups; group < last; ++group) {
    long long start = static_cast<long long>(blockIdx.x) * at_once, end = a.T, step = static_cast<long long>(gridDim.x) * at_once;
    float cg[N];  // c of this group
    Pieces<V> gate{};
    if constexpr (kGroup) {
      start = group * a.shared, end = start + a.shared, step = at_once;
      if (a.parts > 0) {
        const long long part = (a.shared + a.parts - 1LL) / a.parts;
        start = min(start + blockIdx.x % a.parts * part, end);
        end = min(start + part, end);
      }
      gate = load_pieces<V>(row_at<BF>(a.gate, group * a.H, count), first, lanes);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) cg[i] = kGroup ? c[i] * piece_value<BF>(gate.u[i / P], i % P) : c[i];
    for (; start < end; start += step) {
      const bool real = start + mine < end;  // rows behind the last one are zeros
      const long long row = real ? start + mine : end - 1;
      const Pieces<V> xs = load_pieces<V>(row_at<BF>(a.x, row * a.ldx, count, real && next), first, lanes);
      const Pieces<V> bs = load_pieces<V>(row_at<BF>(branch ? a.branch : a.x, row * a.ldb, count, real && branch), first, lanes);
      const Pieces<V> dhs = load_pieces<V>(row_at<BF>(next ? a.dh : a.x, row * a.lddh, count, real && next), first, lanes);
      const Pieces<V> dys = load_pieces<V>(row_at<BF>(a.dy != nullptr ? a.dy : a.x, row * a.lddy, count, real && a.dy != nullptr), first, lanes);
      if constexpr (GATE == GATE_FULL) gate = load_pieces<V>(row_at<BF>(a.gate, row * a.H, count), first, lanes);
      const float scalar = GATE == GATE_TOKEN ? one_value<BF>(a.gate, row) : 1.0f;
      const float rb = post && real ? a.branch_rms[row] : 1.0f, ry = next && real ? a.y_rms[row] : 0.0f;
      // what c lacks of the gate
      const auto gate_of = [&](int i) { return GATE == GATE_TOKEN ? scalar : GATE == GATE_FULL ? piece_value<BF>(gate.u[i / P], i % P) : 1.0f; };
      constexpr bool kLacks = GATE == GATE_TOKEN || GATE == GATE_FULL;
      float u[N], t[N], s = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = piece_value<BF>(bs.u[i / P], i % P) * rb;
      if (next) {
        float q[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float x = piece_value<BF>(xs.u[i / P], i % P), dh = piece_value<BF>(dhs.u[i / P], i % P);
          const float y = branch ? fmaf(kLacks ? cg[i] * gate_of(i) : cg[i], u[i], a.alpha * x) : x;
          t[i] = y * ry;
          sum_next[i] = fmaf(dh, t[i], sum_next[i]);
          q[i] = dh * wn[i];
          s = fmaf(q[i], t[i], s);
        }
        const float mean = row_sum(s, waves, room[0]) / a.H;
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = fmaf(ry, fmaf(-t[i], mean, q[i]), piece_value<BF>(dys.u[i / P], i % P));
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = piece_value<BF>(dys.u[i / P], i % P);
      }
      float out[N];
      if (a.dx != nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = a.alpha * t[i];
        store_pieces<BF, V>(row_at<BF>(a.dx, row * a.H, count, real), first, lanes, out);
      }
      if (!branch) {
        if (waves > 1) __syncthreads();
        continue;
      }
      s = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        sum[i] = fmaf(kLacks ? t[i] * gate_of(i) : t[i], u[i], sum[i]);
        t[i] *= cg[i];
        if constexpr (GATE == GATE_FULL) out[i] = t[i] * u[i], t[i] *= gate_of(i);
        s = fmaf(t[i], u[i], s);
      }
      if constexpr (GATE == GATE_FULL) {
        if (a.dgate != nullptr) store_pieces<BF, V>(row_at<BF>(a.dgate, row * a.H, count, real), first, lanes, out);
      }
      if (post || GATE == GATE_TOKEN) {
        s = row_sum(s, waves, room[1]);
        if constexpr (GATE == GATE_TOKEN) {
          if (a.dgate != nullptr && real && first == 0) put_value<BF>(a.dgate, row, s);
        }
      }
      const float mean = post ? s / a.H : 0.0f, scale = GATE == GATE_TOKEN ? scalar * rb : rb;
      if (a.dbranch != nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = scale * fmaf(-u[i], mean, t[i]);
        store_pieces<BF, V>(row_at<BF>(a.dbranch, row * a.H, count, real), first, lanes, t);
      }
      if (waves > 1 && !(next && (post || GATE == GATE_TOKEN))) __syncthreads();
    }
    if constexpr (kGroup) {
#pragma unroll
      for (int i = 0; i < N; ++i) sum_post[i] = fmaf(piece_value<BF>(gate.u[i / P], i % P), sum[i], sum_post[i]);
      if (a.dgate != nullptr) {
        float* to = a.partial + (static_cast<size_t>(2) * a.blocks + blockIdx.x) * a.H;
        void* whole = a.parts > 0 ? nullptr : static_cast<char*>(a.dgate) + group * a.H * (BF ? 2 : 4);
        join_rows<BF, THREADS>(sum, columns, lanes, first, count, to, whole, a.beta, a.post);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) sum[i] = 0.0f;
    }
  }
  float* to = a.partial + static_cast<size_t>(blockIdx.x) * a.H;
  if (next && a.dnext != nullptr) join_rows<BF, THREADS>(sum_next, columns, lanes, first, count, to);
  to += static_cast<size_t>(a.blocks) * a.H;
  if (a.dpost != nullptr || (GATE == GATE_CHANNEL && a.dgate != nullptr))
    join_rows<BF, THREADS>(kGroup ? sum_post : sum, columns, lanes, first, count, to);
}

// Column sums of the workgroups: 64 columns by sixteen threads each. y: 0 the next norm's weight, 1 the post norm's (and the
// gate's of a channel), 2 + g group g's gate.
template <bool BF>
__global__ __launch_bounds__(1024) void norm_finish_kernel(NormArgs a) {
  __shared__ float room[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6;
  const int which = blockIdx.y < 2 ? blockIdx.y : 2;
  const int rows = which < 2 ? a.blocks : a.parts;
  const float* from = a.partial + static_cast<size_t>(which) * a.blocks * a.H;
  if (which == 2) from += static_cast<size_t>(blockIdx.y - 2) * a.parts * a.H;
  float s = 0.0f;
  if (c < a.H) {
#pragma unroll 4
    for (int r = part; r < rows; r += 16) s += from[static_cast<size_t>(r) * a.H + c];
  }
  room[part][threadIdx.x & 63] = s;
  __syncthreads();
  if (part != 0 || c >= a.H) return;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += room[i][threadIdx.x & 63];
  const float post = a.post != nullptr ? one_value<BF>(a.post, c) : 1.0f;
  if (which == 0) {
    // without a gradient of h nothing reaches its norm's weight
    if (a.dnext != nullptr) put_value<BF>(a.dnext, c, a.dh != nullptr ? s : 0.0f);
  } else if (which == 2) {
    put_value<BF>(a.dgate, static_cast<size_t>(blockIdx.y - 2) * a.H + c, a.beta * post * s);
  } else {
    if (a.dpost != nullptr) put_value<BF>(a.dpost, c, a.gate_kind == GATE_CHANNEL ? a.beta * s * one_value<BF>(a.gate, c) : a.beta * s);
    if (a.gate_kind == GATE_CHANNEL && a.dgate != nullptr) put_value<BF>(a.dgate, c, a.beta * post * s);
  }
}

template <bool BF>
void enqueue_forward(const NormArgs& a, hipStream_t stream) {
  constexpr int P = kPiece<BF>, M = 16 / P;  // pieces of up to 16 values a lane
  const int pieces = a.H / P;
  // few rows are spread over as many lanes as they have pieces, many over as few waves as hold them in 16 values a lane (5003 rows of 2048
  // float32 values with 32, 16 and 8 a lane 29, 17 and 16 us, 8192 of 4096 in bfloat16 51, 50 and 57; 1001 of 1344 as few 8.7, as many 7.5)
  const bool few = a.T < 256;
  int waves = 1;
  while (waves < 16 && waves * 64 * (few ? 1 : M) < pieces) waves *= 2;
  const int threads = waves > 4 ? waves * 64 : 256, at_once = threads / (waves * 64);
  const long long blocks = (a.T + at_once - 1LL) / at_once;
  const dim3 grid(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), block(threads);
  const int each = (pieces + waves * 64 - 1) / (waves * 64);
  if (each <= 1) norm_kernel<BF, 1><<<grid, block, 0, stream>>>(a, waves);
  else if (each <= 2) norm_kernel<BF, 2><<<grid, block, 0, stream>>>(a, waves);
  else if constexpr (!BF) norm_kernel<BF, 4><<<grid, block, 0, stream>>>(a, waves);
}

template <bool BF, int THREADS>
void enqueue_rows(const NormArgs& a, hipStream_t stream) {
  const size_t room = static_cast<size_t>(THREADS / 64 / norm_waves(a.H)) * a.H * 4;
  const dim3 grid(a.blocks), block(THREADS);
  switch (a.gate_kind) {
    case GATE_NONE: norm_backward_kernel<BF, GATE_NONE, THREADS><<<grid, block, room, stream>>>(a); break;
    case GATE_CHANNEL: norm_backward_kernel<BF, GATE_CHANNEL, THREADS><<<grid, block, room, stream>>>(a); break;
    case GATE_GROUP: norm_backward_kernel<BF, GATE_GROUP, THREADS><<<grid, block, room, stream>>>(a); break;
    case GATE_TOKEN: norm_backward_kernel<BF, GATE_TOKEN, THREADS><<<grid, block, room, stream>>>(a); break;
    default: norm_backward_kernel<BF, GATE_FULL, THREADS><<<grid, block, room, stream>>>(a); break;
  }
}
template <bool BF>
void enqueue_backward(const NormArgs& a, hipStream_t stream) {
  norm_threads(a.H) == 256 ? enqueue_rows<BF, 256>(a, stream) : enqueue_rows<BF, 512>(a, stream);
  const bool parts = a.gate_kind == GATE_GROUP && a.parts > 0 && a.dgate != nullptr;
  if (a.dnext != nullptr || a.dpost != nullptr || parts || (a.gate_kind == GATE_CHANNEL && a.dgate != nullptr))
    norm_finish_kernel<BF><<<dim3((a.H + 63) / 64, 2 + (parts ? a.T / a.shared : 0)), dim3(1024), 0, stream>>>(a);
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, int dtype, hipStream_t stream) {
  dtype == 0 ? enqueue_forward<false>(a, stream) : enqueue_forward<true>(a, stream);
  return hipGetLastError();
}
hipError_t launch_norm_backward(const NormArgs& a, int dtype, hipStream_t stream) {
  dtype == 0 ? enqueue_backward<false>(a, stream) : enqueue_backward<true>(a, stream);
  return hipGetLastError();
}

}  // namespace fmoe
