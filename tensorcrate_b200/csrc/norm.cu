// norm.cu — layer norm over the rows of a matrix, and its gradients.
//
//   mean = sum(x) / n,  rstd = 1 / sqrt(sum((x - mean)^2) / n + eps)
//   h = (x - mean) rstd,  y = h w + b
//   grad_x = rstd (g w - sum(g w) / n - h sum(g w h) / n)
//   grad_w = sum over rows of g h,  grad_b = sum over rows of g
//
// Everything is computed in f32 and rounded once, where it is stored.  The
// reference states layer norm as a fused program over row statistics and has
// no gradient of it.
#include <algorithm>

#include "rows.cuh"

namespace tc {
namespace {

// A row's elements stay in the registers of the threads that share it (a
// warp's up to 1024 columns, else a block's), so x is read once for both of
// the variance's passes.  Access k of thread t covers the E elements from (t
// + k * threads) * E: neighbours read neighbouring addresses.  A warp a row
// against a block: 59 us for 74 at 131072x256 f32, 115 for 148 at 65536x1001
// bf16, 48 for 47 at 32768x1024 f32.  f32 rows are bound by HBM: 32768x1024 in
// 48 us, 5.6 TB/s (43 us of it the kernel's).  Rows off the 16-byte grid (E =
// 1) are bound by their single accesses: 67041x1001 bf16 in 117 us, 35% of the
// floor; past 1024 columns their 16 elements a thread spill as well (12 to 32
// bytes): 13419x5001 bf16 in 165 us, 25%.
template <class T, class P, int E, int K, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 1024) norm_rows(const typename T::S *x, size_t x_stride,
                                                  const typename P::S *__restrict__ w,
                                                  const typename P::S *__restrict__ b, float eps,
                                                  typename T::S *y, size_t y_stride,
                                                  float2 *__restrict__ statistics, size_t rows, unsigned cols) {
  using S = typename T::S;
  __shared__ float room[2][32];
  const unsigned threads = WARP ? 32 : blockDim.x;
  const unsigned t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const size_t step = WARP ? size_t(gridDim.x) * (blockDim.x >> 5) : gridDim.x;
  const float share = 1.0f / float(cols);
  for (size_t r = WARP ? size_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x; r < rows; r += step) {
    const S *from = x + r * x_stride;
    Run<S, E> raw[K];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const unsigned c = (t + k * threads) * E;
      if (c < cols) raw[k] = load_run<S, E>(from + c);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if ((t + k * threads) * E < cols)
#pragma unroll
        for (int j = 0; j < E; ++j) sum += T::load(raw[k].e[j]);
    const float mean = (WARP ? warp_sum(sum) : block_sum(sum, room[0])) * share;
    float square = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if ((t + k * threads) * E < cols)
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float d = T::load(raw[k].e[j]) - mean;
          square += d * d;
        }
    const float var = (WARP ? warp_sum(square) : block_sum(square, room[1])) * share;
    const float rstd = __frsqrt_rn(var + eps);
    if (t == 0 && statistics) statistics[r] = make_float2(mean, rstd);
    S *to = y + r * y_stride;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const unsigned c = (t + k * threads) * E;
      if (c >= cols) break;
      float wv[E], bv[E];
      if (w) load_wide<P, E>(w + c, wv);
      if (b) load_wide<P, E>(b + c, bv);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        float v = (T::load(raw[k].e[j]) - mean) * rstd;
        if (w) v *= wv[j];
        if (b) v += bv[j];
        raw[k].e[j] = T::store(v);
      }
      store_run<S, E>(to + c, raw[k]);
    }
  }
}

// The same for 16-bit rows on the 16-byte grid, where the weights (often f32)
// would be read again for each row at several times its bytes: blocks that
// stay, of groups of `threads` threads.  A group takes a turn of R
// neighbouring rows at a time and its threads own the same K * E columns of
// every row, whose weights and biases they keep in registers; the next
// turn's rows are loaded before this one's are used.  16384x8192 bf16 with f32
// weights in 109 us, 4.9 TB/s (169 us by blocks of a row each that read the
// weights again); 32768x4096 103, 5.2 TB/s (156); 65536x1024 54 (60).  Rows of
// 8192 to 16384 columns, at 32 a thread, spill 80 bytes: 8192x16384 in 153 us,
// 54% of the floor.  Single elements of rows off the grid gain nothing by it (65536x1001: 152 us for
// 108), they stay with norm_rows.
struct NormTurns {
  const void *x, *w, *b;
  void *y;
  size_t x_stride, y_stride, rows;
  float2 *statistics;
  float eps;
  unsigned cols, threads;
};
template <class T, class P, int K, int R, int MOST, int BLOCKS>
__global__ void __launch_bounds__(MOST, BLOCKS) norm_turns(const NormTurns a) {
  using S = typename T::S;
  using PS = typename P::S;
  constexpr int E = 8, N = K * 4;  // elements of an access, pairs of a row
  __shared__ float room[2][2][32];
  const unsigned threads = a.threads, groups = blockDim.x / threads, cols = a.cols;
  const unsigned group = threadIdx.x / threads, t = threadIdx.x - group * threads;
  const unsigned lane = threadIdx.x & 31, warps = threads >> 5, warp0 = group * warps;
  const size_t every = size_t(gridDim.x) * groups * R;
  size_t row = (size_t(blockIdx.x) * groups + group) * R;
  auto column = [&](int k) { return (t + k * threads) * E; };
  uint4 next[R][K];
  auto fetch = [&](size_t at) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        next[r][k] = make_uint4(0, 0, 0, 0);
        if (at + r < a.rows && column(k) < cols)
          next[r][k] = *reinterpret_cast<const uint4 *>(static_cast<const S *>(a.x) + (at + r) * a.x_stride + column(k));
      }
  };
  fetch(row);
  F2 w[N], b[N];
  auto keep = [&](const void *from, float none, F2 *into) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float v[E];
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = none;
      if (from && column(k) < cols) load_wide<P, E>(static_cast<const PS *>(from) + column(k), v);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) into[k * 4 + j] = pair(v[2 * j], v[2 * j + 1]);
    }
  };
  keep(a.w, 1.0f, w);
  keep(a.b, 0.0f, b);
  const float share = 1.0f / float(cols);
  // A value of each of the R rows, added over the group's threads.
  auto add_up = [&](float (&v)[R], int which) {
    float s;
    if constexpr (R == 2) {  // lanes 0 to 15 add up the first row's, 16 to 31 the second's
      s = lane < 16 ? v[0] : v[1];
      s += __shfl_xor_sync(0xffffffffu, lane < 16 ? v[1] : v[0], 16);
    } else {
      s = v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
    }
#pragma unroll
    for (int o = 8; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (warps > 1) {
      float *at = room[which][R == 2 ? lane >> 4 : 0];
      if ((lane & 15) == 0) at[threadIdx.x >> 5] = s;
      __barrier_sync_count(group + 1, threads);
      s = 0.0f;
      for (unsigned i = lane & 15; i < warps; i += 16) s += at[warp0 + i];
#pragma unroll
      for (int o = 8; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = __shfl_sync(0xffffffffu, s, 16 * r);
  };
  for (; row < a.rows; row += every) {
    uint4 raw[R][K];
    float mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < K; ++k) raw[r][k] = next[r][k];
    fetch(row + every);
    auto pair_at = [&](int r, int i) {
      const uint4 q = raw[r][i / 4];
      return widen2<T>(i % 4 == 0 ? q.x : i % 4 == 1 ? q.y : i % 4 == 2 ? q.z : q.w);
    };
#pragma unroll
    for (int r = 0; r < R; ++r) {
      F2 s = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) s = add2(s, pair_at(r, i));
      const float2 p = split(s);
      mean[r] = p.x + p.y;
    }
    add_up(mean, 0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] *= share;
      const F2 less = pair(-mean[r], -mean[r]);
      F2 s = 0;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (column(k) < cols)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const F2 d = add2(pair_at(r, k * 4 + j), less);
            s = fma2(d, d, s);
          }
      const float2 p = split(s);
      rstd[r] = p.x + p.y;
    }
    add_up(rstd, 1);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      rstd[r] = __frsqrt_rn(rstd[r] * share + a.eps);
      if (row + r >= a.rows) break;
      if (t == 0 && a.statistics) a.statistics[row + r] = make_float2(mean[r], rstd[r]);
      const F2 less = pair(-mean[r], -mean[r]), scale = pair(rstd[r], rstd[r]);
      S *to = static_cast<S *>(a.y) + (row + r) * a.y_stride;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (column(k) < cols) {
          F2 out[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            out[j] = fma2(mul2(add2(pair_at(r, k * 4 + j), less), scale), w[k * 4 + j], b[k * 4 + j]);
          store_pairs<T>(to + column(k), out);
        }
    }
  }
}

// Rows of more than 16384 columns: a block reads its row three times, the
// second and third from L2, by single elements: 8192x20000 bf16 in 538 us (19%
// of the floor), 4096x20000 f32 in 306 (33%).
template <class T, class P>
__global__ void __launch_bounds__(1024) norm_rows_wide(const typename T::S *x, size_t x_stride,
                                                       const typename P::S *__restrict__ w,
                                                       const typename P::S *__restrict__ b, float eps,
                                                       typename T::S *y, size_t y_stride,
                                                       float2 *__restrict__ statistics, size_t rows, size_t cols) {
  using S = typename T::S;
  __shared__ float room[2][32];
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const S *from = x + r * x_stride;
    float sum = 0.0f;
#pragma unroll 8
    for (size_t c = threadIdx.x; c < cols; c += blockDim.x) sum += T::load(from[c]);
    const float mean = block_sum(sum, room[0]) / float(cols);
    float square = 0.0f;
#pragma unroll 8
    for (size_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const float d = T::load(from[c]) - mean;
      square += d * d;
    }
    const float rstd = __frsqrt_rn(block_sum(square, room[1]) / float(cols) + eps);
    if (threadIdx.x == 0 && statistics) statistics[r] = make_float2(mean, rstd);
    S *to = y + r * y_stride;
#pragma unroll 8
    for (size_t c = threadIdx.x; c < cols; c += blockDim.x) {
      float v = (T::load(from[c]) - mean) * rstd;
      if (w) v *= P::load(w[c]);
      if (b) v += P::load(b[c]);
      to[c] = T::store(v);
    }
  }
}

// grad_x, and this block's share of grad_w and grad_b.  A block is `groups`
// groups of `threads` threads; a group takes a turn of R neighbouring rows at
// a time and its threads own the same columns of every row, so the columns'
// sums stay in registers until the block adds its groups' and writes them to
// its row of `partial` (w's sums, then b's).
//
// WIDE: rows too wide for one block's registers are shared by the blocks of a
// cluster, each with `width` columns (and one group): the barrier is then the
// cluster's, and each warp's sums go to every block.
//
// The rows come through a ring of DEPTH turns in shared memory, filled
// asynchronously: HBM is not waited for once the ring runs, whatever few
// threads the columns' sums leave room for.  A row is copied as the aligned
// 16-byte granules that it touches (so rows that start anywhere are read at
// full width; a granule that holds one valid byte can be read whole); E
// elements at a time are taken from there, E > 1 only for rows on the grid.
// One barrier a turn publishes the rows' sums, the next turn's data and the
// stage to be filled again.  A turn's elements are read from the ring twice
// (kept in registers across the barrier, with the sums, they spill).  Two rows
// a turn share its barrier, its waits and its shuffles: one row leaves a block
// of 16 warps, all in step, with too little between them.
//
// What bounds it: the one block that an SM's registers hold, 16 warps that
// issue half of the time (of the HBM floor: f32 rows 92% up to 4096 columns,
// 16-bit rows 90% up to 1024, 77% at 4096 and 72% at 8192); past 8192 columns
// the clusters' barriers too (60% at 16384, where 32 columns a thread spilled
// and reached 28%).  16384x8192 bf16, 805 MB: 168 us for this kernel and 171 to
// 181 a call, 4.6 TB/s (one row a turn: 186 us a call; 1024 threads of 8
// columns each spill: 289 us; rows through registers without the ring: 263
// us); 2048x4096 bf16 24.6 us a call.  Off the 16-byte grid it is the single
// accesses to shared memory and of the stores, 46% at 67041x1001 bf16 (8
// columns a thread: 75 us at 33520x1001 where 16 take 91, 83 for 98 at
// 8386x4001); past 4096 columns a thread's 16 spill 28 to 68 bytes as well, 25%
// at 13419x5001 bf16.
struct NormGrad {
  const void *g, *x, *w;
  size_t g_stride, x_stride, dx_stride, rows;
  const float2 *statistics;
  void *dx;
  float *partial;
  unsigned cols, width, threads, slot;  // slot: bytes of a block's part of one row in the ring
};
constexpr unsigned RING = 200 * 1024, DEPTH = 3, MAX_GROUPS = 15;  // named barriers 1 to 15

// A thread's elements of one row as they are stored: WORDS registers.
template <class T, int E, int K> struct Held {
  static constexpr int N = K * E / 2;                       // pairs of elements
  static constexpr int STEP = E == 1 ? 1 : E / 2;           // pairs of one access
  static constexpr int WORDS = T::code == TC_F32 ? 2 * N : N;
  uint32_t raw[WORDS];
  __device__ __forceinline__ F2 pair_at(int i) const {
    if constexpr (T::code == TC_F32) return pair(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1]));
    else return widen2<T>(raw[i]);
  }
  // The elements of `row` (in shared memory) at the columns of thread t; past
  // the row's end zeros, or (LAST) the row's last elements.
  template <bool LAST> __device__ __forceinline__ void load(const typename T::S *row, unsigned t, unsigned threads, unsigned cols) {
    using S = typename T::S;
    if constexpr (E == 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const unsigned lo = t + 2 * i * threads, hi = lo + threads;
        const S a = LAST ? row[min(lo, cols - 1)] : lo < cols ? row[lo] : S(0);
        const S b = LAST ? row[min(hi, cols - 1)] : hi < cols ? row[hi] : S(0);
        if constexpr (T::code == TC_F32) {
          raw[2 * i] = __float_as_uint(a);
          raw[2 * i + 1] = __float_as_uint(b);
        } else {
          raw[i] = uint32_t(a) | uint32_t(b) << 16;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const unsigned c = (t + k * threads) * E;
        const uint4 v = LAST || c < cols ? *reinterpret_cast<const uint4 *>(row + (LAST ? min(c, cols - E) : c))
                                         : make_uint4(0, 0, 0, 0);
        raw[4 * k] = v.x;
        raw[4 * k + 1] = v.y;
        raw[4 * k + 2] = v.z;
        raw[4 * k + 3] = v.w;
      }
    }
  }
};

template <class T, class P, int E, int K, int R, bool WIDE>
__global__ void __launch_bounds__(512) norm_grad_rows(const NormGrad a) {
  using S = typename T::S;
  using PS = typename P::S;
  using Row = Held<T, E, K>;
  constexpr int N = Row::N, STEP = Row::STEP;
  constexpr int GRANULES = K * E * int(sizeof(S)) / 16 + (E == 1);  // a thread's, of a row
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float room[2][4 * 64];  // four sums of up to 64 warps
  const unsigned part = WIDE ? cluster_part() : 0, parts = WIDE ? cluster_parts() : 1, base = part * a.width;
  const unsigned threads = a.threads, groups = blockDim.x / threads, cols = WIDE ? min(a.width, a.cols - base) : a.cols;
  const unsigned group = threadIdx.x / threads, t = threadIdx.x - group * threads;
  const unsigned lane = threadIdx.x & 31, warps = parts * (threads >> 5), warp0 = group * warps;
  // turn n of this group: rows R (begin + n every), and the next
  const size_t begin = size_t(blockIdx.x / parts) * groups + group, every = size_t(gridDim.x / parts) * groups;
  const size_t turns = (a.rows + R - 1) / R, count = begin < turns ? (turns - begin + every - 1) / every : 0;
  unsigned char *mine = ring + size_t(group) * DEPTH * 2 * R * a.slot;
  const uint32_t mine32 = uint32_t(__cvta_generic_to_shared(mine));
  auto column = [&](int k) { return (t + k * threads) * E; };
  auto sync = [&] {
    if (WIDE) cluster_sync();
    else __barrier_sync_count(group + 1, threads);
  };
  auto row_at = [&](const void *p, size_t stride, size_t row) {
    return reinterpret_cast<uintptr_t>(static_cast<const S *>(p) + row * stride + base);
  };

  // the next turn to be copied
  size_t row_next = begin * R;
  uintptr_t x_next = row_at(a.x, a.x_stride, row_next), g_next = row_at(a.g, a.g_stride, row_next);
  const size_t x_step = a.x_stride * sizeof(S), g_step = a.g_stride * sizeof(S);
  auto fetch = [&](uintptr_t from, uint32_t to) {
    const unsigned off = E == 1 ? unsigned(from) & 15 : 0, bytes = off + cols * unsigned(sizeof(S));
    const char *p = reinterpret_cast<const char *>(from - off) + t * 16;
    to += t * 16;
#pragma unroll
    for (int j = 0; j < GRANULES; ++j)
      if ((t + j * threads) * 16 < bytes) copy_async(to + j * threads * 16, p + j * threads * 16);
  };
  auto fill = [&](unsigned stage) {
    const uint32_t to = mine32 + stage * 2 * R * a.slot;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (row_next + r < a.rows) {
        fetch(x_next + r * x_step, to + 2 * r * a.slot);
        fetch(g_next + r * g_step, to + (2 * r + 1) * a.slot);
      }
    row_next += every * R;
    x_next += every * R * x_step;
    g_next += every * R * g_step;
    copy_commit();
  };
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr unsigned AHEAD = DEPTH - 1;  // turns in the ring at a turn's start
#pragma unroll
  for (unsigned d = 0; d < AHEAD; ++d) fill(d);

  auto load_weight = [&](int i) -> F2 {  // pair i
    if (!a.w) return pair(1.0f, 1.0f);
    const PS *at = static_cast<const PS *>(a.w) + base;
    if constexpr (E == 1) {
      const unsigned lo = column(2 * i), hi = column(2 * i + 1);
      return pair(lo < cols ? P::load(at[lo]) : 1.0f, hi < cols ? P::load(at[hi]) : 1.0f);
    } else {
      const unsigned c = column(i / STEP) + i % STEP * 2;
      if (c >= cols) return pair(1.0f, 1.0f);
      const Run<PS, 2> r = load_run<PS, 2>(at + c);
      return pair(P::load(r.e[0]), P::load(r.e[1]));
    }
  };
  F2 w[N], sum_w[N], sum_b[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = load_weight(i);
    sum_w[i] = sum_b[i] = 0;
  }

  const float share = 1.0f / float(a.cols);
  size_t row = begin * R;
  uintptr_t x_here = x_next - AHEAD * every * R * x_step, g_here = g_next - AHEAD * every * R * g_step;
  S *dx = static_cast<S *>(a.dx) + (a.dx ? row * a.dx_stride + base : 0);
  float2 next[R];
#pragma unroll
  for (int r = 0; r < R; ++r) next[r] = row + r < a.rows ? a.statistics[row + r] : make_float2(0.0f, 0.0f);
  copy_wait<AHEAD - 1>();
  sync();
  unsigned stage = 0, turn = 0;
  for (size_t n = 0; n < count; ++n, turn ^= 1) {
    const unsigned char *here = mine + stage * 2 * R * a.slot;
    auto held_at = [&](int which, uintptr_t from) {
      return reinterpret_cast<const S *>(here + which * a.slot + (E == 1 ? from & 15 : 0));
    };
    Row xr[R], gr[R];
    float2 st[R];
    float value[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // sum(g w), sum(g w h) of each row
#pragma unroll
    for (int r = 0; r < R; ++r) {
      st[r] = next[r];
      // A row past the last has no data: its gradient is zero, and its x the
      // turn's first row's.  An element past the row's end has a zero gradient
      // too, and the x of a real one: an h that is infinite for no other reason
      // than that (0 - mean) rstd is would make the zeros' products NaN.
      const bool real = R == 1 || row + r < a.rows;
      xr[r].template load<true>(held_at(real ? 2 * r : 0, x_here + r * x_step), t, threads, cols);
      gr[r].template load<false>(held_at(2 * r + 1, g_here + r * g_step), t, threads, real ? cols : 0);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const F2 mean = pair(-st[r].x, -st[r].x), rstd = pair(st[r].y, st[r].y);
      F2 s1 = 0, s2 = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const F2 h = mul2(add2(xr[r].pair_at(i), mean), rstd), gv = gr[r].pair_at(i), gw = mul2(gv, w[i]);
        s1 = add2(s1, gw);
        s2 = fma2(gw, h, s2);
        sum_w[i] = fma2(gv, h, sum_w[i]);
        sum_b[i] = add2(sum_b[i], gv);
      }
      const float2 p = split(s1), q = split(s2);
      value[2 * r] = p.x + p.y;
      value[2 * r + 1] = q.x + q.y;
    }
    // the warp's sums: each eighth of a warp's lanes ends with one of the four
    const bool high = lane & 16, odd = lane & 8;
    float v0 = high ? value[2] : value[0], v1 = high ? value[3] : value[1];
    v0 += __shfl_xor_sync(0xffffffffu, high ? value[0] : value[2], 16);
    v1 += __shfl_xor_sync(0xffffffffu, high ? value[1] : value[3], 16);
    float v = odd ? v1 : v0;
    v += __shfl_xor_sync(0xffffffffu, odd ? v0 : v1, 8);
#pragma unroll
    for (int o = 4; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    float *at = room[turn] + (lane >> 3) * 64;
    if ((lane & 7) == 0) {
      if (!WIDE) at[threadIdx.x >> 5] = v;
      else
        for (unsigned p = 0; p < parts; ++p) store_at(at + part * (threads >> 5) + (threadIdx.x >> 5), p, v);
    }
    row += every * R;
#pragma unroll
    for (int r = 0; r < R; ++r) next[r] = row + r < a.rows ? a.statistics[row + r] : make_float2(0.0f, 0.0f);
    copy_wait<AHEAD - 2>();  // this thread's part of the next turn
    sync();
    // every thread is past the last turn, whose stage comes before this one
    fill(stage == 0 ? DEPTH - 1 : stage - 1);
    v = ((lane & 7) < warps ? at[warp0 + (lane & 7)] : 0.0f) + ((lane & 7) + 8 < warps ? at[warp0 + (lane & 7) + 8] : 0.0f);
    if (WIDE)
      for (unsigned i = (lane & 7) + 16; i < warps; i += 8) v += at[i];
#pragma unroll
    for (int o = 4; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    v *= -share;
    if (a.dx) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float c1 = __shfl_sync(0xffffffffu, v, 16 * r) * st[r].y, c2 = __shfl_sync(0xffffffffu, v, 16 * r + 8) * st[r].y;
        if (R > 1 && row - every * R + r >= a.rows) break;
        const F2 mean = pair(-st[r].x, -st[r].x), rstd = pair(st[r].y, st[r].y), k1 = pair(c1, c1), k2 = pair(c2, c2);
        xr[r].template load<false>(held_at(2 * r, x_here + r * x_step), t, threads, cols);
        gr[r].template load<false>(held_at(2 * r + 1, g_here + r * g_step), t, threads, cols);
#pragma unroll
        for (int i = 0; i < N; i += STEP) {
          F2 out[STEP];
#pragma unroll
          for (int j = 0; j < STEP; ++j) {
            const F2 h = mul2(add2(xr[r].pair_at(i + j), mean), rstd), gw = mul2(gr[r].pair_at(i + j), w[i + j]);
            out[j] = fma2(gw, rstd, fma2(h, k2, k1));
          }
          S *to = dx + r * a.dx_stride;
          if constexpr (E == 1) {
            const float2 o = split(out[0]);
            const unsigned lo = column(2 * i), hi = column(2 * i + 1);
            if (lo < cols) to[lo] = T::store(o.x);
            if (hi < cols) to[hi] = T::store(o.y);
          } else if (column(i / STEP) < cols) {
            store_pairs<T>(to + column(i / STEP), out);
          }
        }
      }
      dx += every * R * a.dx_stride;
    }
    x_here += every * R * x_step;
    g_here += every * R * g_step;
    stage = stage + 1 == DEPTH ? 0 : stage + 1;
  }
  copy_wait<0>();
  if (!a.partial) return;
  // the groups' sums: each group's to the ring's memory, then added up in the
  // groups' order by all threads
  float *out = a.partial + size_t(blockIdx.x / parts) * 2 * a.cols + base;
  float *hold = groups > 1 ? reinterpret_cast<float *>(ring) + size_t(group) * 2 * a.cols : out;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 vw = split(sum_w[i]), vb = split(sum_b[i]);
    const unsigned lo = E == 1 ? column(2 * i) : column(i / STEP) + i % STEP * 2, hi = E == 1 ? column(2 * i + 1) : lo + 1;
    if (lo < cols) {
      hold[lo] = vw.x;
      hold[a.cols + lo] = vb.x;
    }
    if (hi < cols) {
      hold[hi] = vw.y;
      hold[a.cols + hi] = vb.y;
    }
  }
  if (groups == 1) return;
  __syncthreads();
  hold = reinterpret_cast<float *>(ring);
  for (unsigned c = threadIdx.x; c < 2 * cols; c += blockDim.x) {
    float sum = hold[c];
    for (unsigned g = 1; g < groups; ++g) sum += hold[size_t(g) * 2 * cols + c];
    out[c] = sum;
  }
}

// Rows of more than 32768 columns, by single elements (2048x40000 bf16 in 470
// us, 16% of the floor; 1024x65536 f32 in 517, 24%): grad_x by blocks that read
// their row twice ...
template <class T, class P>
__global__ void __launch_bounds__(1024) norm_grad_wide(const typename T::S *g, size_t g_stride,
                                                       const typename T::S *x, size_t x_stride,
                                                       const float2 *__restrict__ statistics,
                                                       const typename P::S *__restrict__ w,
                                                       typename T::S *dx, size_t dx_stride, size_t rows,
                                                       size_t cols) {
  using S = typename T::S;
  __shared__ float room[2][2][32];
  int turn = 0;
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x, turn ^= 1) {
    const S *xf = x + r * x_stride, *gf = g + r * g_stride;
    S *to = dx + r * dx_stride;
    const float2 st = statistics[r];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll 4
    for (size_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const float gw = T::load(gf[c]) * (w ? P::load(w[c]) : 1.0f);
      s1 += gw;
      s2 += gw * ((T::load(xf[c]) - st.x) * st.y);
    }
    const float c1 = block_sum(s1, room[turn][0]) / float(cols), c2 = block_sum(s2, room[turn][1]) / float(cols);
#pragma unroll 4
    for (size_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const float gw = T::load(gf[c]) * (w ? P::load(w[c]) : 1.0f);
      to[c] = T::store(st.y * (gw - c1 - ((T::load(xf[c]) - st.x) * st.y) * c2));
    }
  }
}

// ... and the columns' sums by blocks that each own 128 columns of a band of
// rows.
template <class T>
__global__ void __launch_bounds__(128) norm_grad_columns(const typename T::S *g, size_t g_stride,
                                                         const typename T::S *x, size_t x_stride,
                                                         const float2 *__restrict__ statistics,
                                                         float *__restrict__ partial, size_t rows, size_t cols) {
  const size_t c = size_t(blockIdx.x) * 128 + threadIdx.x;
  if (c >= cols) return;
  float sw = 0.0f, sb = 0.0f;
#pragma unroll 4
  for (size_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float2 st = statistics[r];
    const float gv = T::load(g[r * g_stride + c]);
    sw += gv * ((T::load(x[r * x_stride + c]) - st.x) * st.y);
    sb += gv;
  }
  partial[size_t(blockIdx.y) * 2 * cols + c] = sw;
  partial[size_t(blockIdx.y) * 2 * cols + cols + c] = sb;
}

// grad_w and grad_b from the blocks' partial sums, in an order that their
// number gives: 32 columns a block, each of its 32 warps a part of the partials.  The
// block may be resident before the partials are written; it waits for them
// where it says so.
template <class P>
__global__ void __launch_bounds__(1024) norm_grad_join(const float *partial, unsigned parts, size_t cols,
                                                       typename P::S *__restrict__ dw, typename P::S *__restrict__ db) {
  __shared__ float room[32][33];
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t i = size_t(blockIdx.x) * 32 + lane;  // column of [w's sums | b's sums]
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float v = 0.0f;
  if (i < 2 * cols) {
#pragma unroll 5
    for (unsigned p = warp; p < parts; p += 32) v += __ldcg(partial + size_t(p) * 2 * cols + i);
  }
  room[warp][lane] = v;
  __syncthreads();
  // warp w adds up column w of the block
  const float sum = warp_sum(room[lane][warp]);
  const size_t c = size_t(blockIdx.x) * 32 + warp;
  if (lane || c >= 2 * cols) return;
  if (c < cols) {
    if (dw) dw[c] = P::store(sum);
  } else if (db) {
    db[c - cols] = P::store(sum);
  }
}

// Dispatch on the parameters' type: the rows' own, or f32.
template <class F> int with_types(int dtype, int param_dtype, const char *what, F &&f) {
  if (param_dtype != dtype && param_dtype != TC_F32)
    return fail(TC_EINVAL, "%s: parameters of type %d beside rows of type %d (the same, or f32)", what, param_dtype, dtype);
  return with_real(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (param_dtype == T::code) return f(t, t);
    return f(t, F32T{});
  });
}

int check_matrix(const char *what, const char *name, size_t rows, size_t cols, size_t stride) {
  if (rows > 1 && stride < cols)
    return fail(TC_EINVAL, "%s: rows of %s are %zu elements apart, fewer than its %zu columns", what, name, stride, cols);
  size_t end;
  if (__builtin_mul_overflow(rows, stride, &end) || __builtin_add_overflow(end, cols, &end) || end > (size_t(1) << 60))
    return fail(TC_ERANGE, "%s: layout arithmetic of %s overflows", what, name);
  return TC_OK;
}

}  // namespace
}  // namespace tc

using namespace tc;

extern "C" {

int tc_layer_norm(int dtype, int param_dtype, size_t rows, size_t cols, const void *x, size_t x_stride,
                  const void *weight, const void *bias, double eps, void *y, size_t y_stride, float *statistics,
                  void *stream) {
  return with_types(dtype, param_dtype, "layer norm", [&](auto t, auto p) -> int {
    using T = decltype(t);
    using P = decltype(p);
    using S = typename T::S;
    using PS = typename P::S;
    constexpr int V = 16 / sizeof(S);
    if (cols == 0) return fail(TC_EINVAL, "layer norm: rows of no elements");
    if (!(eps >= 0.0)) return fail(TC_EINVAL, "layer norm: eps %g", eps);
    if (int st = check_matrix("layer norm", "x", rows, cols, x_stride)) return st;
    if (int st = check_matrix("layer norm", "y", rows, cols, y_stride)) return st;
    if (rows == 0) return TC_OK;
    if (!x || !y) return fail(TC_EINVAL, "layer norm: null pointer");
    if (reinterpret_cast<uintptr_t>(statistics) % 8) return fail(TC_EINVAL, "layer norm: statistics are not on an 8-byte boundary");
    const S *xs = static_cast<const S *>(x);
    S *ys = static_cast<S *>(y);
    const PS *ws = static_cast<const PS *>(weight), *bs = static_cast<const PS *>(bias);
    float2 *stats = reinterpret_cast<float2 *>(statistics);
    cudaStream_t on = as_stream(stream);
    const bool whole = cols % V == 0 && runs_fit(x, x_stride, rows, sizeof(S), V) &&
                       runs_fit(y, y_stride, rows, sizeof(S), V) && (!weight || reinterpret_cast<uintptr_t>(weight) % 16 == 0) &&
                       (!bias || reinterpret_cast<uintptr_t>(bias) % 16 == 0);
    const unsigned most = unsigned(std::min<size_t>(rows, 1u << 30));
    // 32 elements a lane where a warp holds the row, else 16 a thread
    auto launch = [&](auto e) -> int {
      constexpr int E = decltype(e)::value, KW = 32 / E, KB = 16 / E;
      const unsigned n = unsigned((cols + E - 1) / E);
      if (n <= 32 * KW) {
        norm_rows<T, P, E, KW, true><<<(most + 3) / 4, 128, 0, on>>>(xs, x_stride, ws, bs, float(eps), ys, y_stride, stats,
                                                                     rows, unsigned(cols));
      } else {
        const unsigned threads = ((n + KB - 1) / KB + 31) / 32 * 32;
        norm_rows<T, P, E, KB, false><<<most, threads, 0, on>>>(xs, x_stride, ws, bs, float(eps), ys, y_stride, stats, rows,
                                                                unsigned(cols));
      }
      return check_launch("layer norm");
    };
    if constexpr (sizeof(S) == 2) {
      if (whole && cols <= 16 * 1024) {
        // 16 columns a thread where 512 of them hold a row, else 32
        auto turns = [&](auto kernel, unsigned most_threads, unsigned of_thread, unsigned r) -> int {
          const unsigned threads = unsigned((cols + of_thread - 1) / of_thread + 31) / 32 * 32;
          const NormTurns a{x, weight, bias, y, x_stride, y_stride, rows, stats, float(eps), unsigned(cols), threads};
          const unsigned groups = std::max(1u, most_threads / threads);
          int blocks = 0;
          cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kernel, int(groups * threads), 0);
          const size_t all = (rows + r - 1) / r;
          const unsigned grid = unsigned(std::min<size_t>((all + groups - 1) / groups, size_t(std::max(1, blocks)) * size_t(sm_count())));
          kernel<<<grid, groups * threads, 0, on>>>(a);
          return check_launch("layer norm");
        };
        if (cols <= 16 * 256) return turns(norm_turns<T, P, 2, 2, 256, 2>, 256, 16, 2);
        if (cols <= 16 * 512) return turns(norm_turns<T, P, 2, 2, 512, 1>, 512, 16, 2);
        return turns(norm_turns<T, P, 4, 1, 512, 1>, 512, 32, 1);
      }
    }
    if (cols <= 16 * 1024) {
      if constexpr (sizeof(S) == 4)
        if (whole) return launch(std::integral_constant<int, V>{});
      return launch(std::integral_constant<int, 1>{});
    }
    norm_rows_wide<T, P><<<most, 1024, 0, on>>>(xs, x_stride, ws, bs, float(eps), ys, y_stride, stats, rows, cols);
    return check_launch("layer norm");
  });
}

int tc_layer_norm_backward(int dtype, int param_dtype, size_t rows, size_t cols, const void *grad, size_t grad_stride,
                           const void *x, size_t x_stride, const float *statistics, const void *weight, void *grad_x,
                           size_t grad_x_stride, void *grad_weight, void *grad_bias, void *stream) {
  return with_types(dtype, param_dtype, "layer norm backward", [&](auto t, auto p) -> int {
    using T = decltype(t);
    using P = decltype(p);
    using S = typename T::S;
    using PS = typename P::S;
    constexpr int V = 16 / sizeof(S);
    if (cols == 0) return fail(TC_EINVAL, "layer norm backward: rows of no elements");
    if (int st = check_matrix("layer norm backward", "grad", rows, cols, grad_stride)) return st;
    if (int st = check_matrix("layer norm backward", "x", rows, cols, x_stride)) return st;
    if (int st = check_matrix("layer norm backward", "grad_x", rows, cols, grad_x_stride)) return st;
    cudaStream_t on = as_stream(stream);
    PS *dw = static_cast<PS *>(grad_weight), *db = static_cast<PS *>(grad_bias);
    if (rows == 0) {  // sums over nothing
      if (dw)
        if (int st = check_cuda(cudaMemsetAsync(dw, 0, cols * sizeof(PS), on), "layer norm backward")) return st;
      if (db) return check_cuda(cudaMemsetAsync(db, 0, cols * sizeof(PS), on), "layer norm backward");
      return TC_OK;
    }
    if (!grad || !x || !statistics) return fail(TC_EINVAL, "layer norm backward: null pointer");
    if (reinterpret_cast<uintptr_t>(statistics) % 8)
      return fail(TC_EINVAL, "layer norm backward: statistics are not on an 8-byte boundary");
    if (!grad_x && !dw && !db) return TC_OK;
    const S *gs = static_cast<const S *>(grad), *xs = static_cast<const S *>(x);
    S *dx = static_cast<S *>(grad_x);
    const PS *ws = static_cast<const PS *>(weight);
    const float2 *stats = reinterpret_cast<const float2 *>(statistics);
    const bool sums = dw || db;
    float *partial = nullptr;
    unsigned parts = 0;
    auto room = [&](unsigned n) -> int {
      parts = n;
      void *s = nullptr;
      if (int st = scratch(size_t(n) * 2 * cols * sizeof(float), &s, on)) return st;
      partial = static_cast<float *>(s);
      return TC_OK;
    };
    const bool whole = cols % V == 0 && runs_fit(grad, grad_stride, rows, sizeof(S), V) &&
                       runs_fit(x, x_stride, rows, sizeof(S), V) &&
                       (!grad_x || runs_fit(grad_x, grad_x_stride, rows, sizeof(S), V)) &&
                       (!weight || reinterpret_cast<uintptr_t>(weight) % 16 == 0);
    // A thread owns 16 columns (8 of up to 4096 off the grid), a block those of
    // 512 threads, a cluster those of at most four blocks.  Two rows a turn
    // where their registers and the ring hold them.
    unsigned across = 1;
    while (across < 4 && cols > 16 * 512 * across) across *= 2;
    if (cols <= 16 * 512 * across) {
      auto run = [&](auto e, auto k, auto two, auto wide) -> int {
        constexpr int E = decltype(e)::value, K = decltype(k)::value, R = decltype(two)::value;
        auto kernel = norm_grad_rows<T, P, E, K, R, decltype(wide)::value>;
        static std::atomic<uint64_t> allowed{0};
        if (int st = allow_shared("layer norm backward", reinterpret_cast<const void *>(kernel), RING, allowed)) return st;
        const size_t width = ((cols + across - 1) / across + V - 1) / V * V, slot = (width * sizeof(S) + 15) / 16 * 16 + 16;
        NormGrad a{grad, x, weight, grad_stride, x_stride, grad_x_stride, rows, stats, grad_x, nullptr, unsigned(cols), unsigned(width), 0, unsigned(slot)};
        a.threads = unsigned((width + K * E - 1) / (K * E) + 31) / 32 * 32;
        // as many groups as the block's threads, its named barriers and the ring
        // hold, but no more than give every SM a turn
        const size_t sms = size_t(sm_count()), turns = (rows + R - 1) / R, each = DEPTH * 2 * R * slot;
        const unsigned groups = across > 1 ? 1 : unsigned(std::min<size_t>({MAX_GROUPS, 512 / a.threads, RING / each, (turns + sms - 1) / sms}));
        const unsigned grid = unsigned(std::min<size_t>((turns + groups - 1) / groups, sms / across));
        if (sums) {
          if (int st = room(grid)) return st;
          a.partial = partial;
        }
        return tc::launch("layer norm backward", kernel, grid, across, groups * a.threads,
                          std::max(groups * each, groups > 1 ? groups * cols * 8 : 0), on, a);
      };
      constexpr int R = sizeof(S) == 2 ? 2 : 1;
      const std::integral_constant<int, 1> one;
      const std::integral_constant<int, V> access;
      const std::integral_constant<int, 16 / V> accesses;
      const std::integral_constant<int, 8> eight;
      const std::integral_constant<int, 16> sixteen;
      const std::integral_constant<int, R> two;
      int st;
      if (whole && across == 1) st = run(access, accesses, two, std::false_type{});
      else if (whole) st = run(access, accesses, two, std::true_type{});
      else if (cols <= 8 * 512) st = run(one, eight, one, std::false_type{});
      else if (across == 1) st = run(one, sixteen, one, std::false_type{});
      else st = run(one, sixteen, one, std::true_type{});
      if (st) return st;
    } else {
      if (sums) {  // first: grad_x may replace what they read
        const size_t tiles = (cols + 127) / 128;
        if (tiles > 0x7fffffffu) return fail(TC_ERANGE, "layer norm backward: %zu columns", cols);
        const unsigned bands = unsigned(std::min<size_t>(std::max<size_t>(1, rows / 32), std::max<size_t>(1, size_t(sm_count()) * 16 / tiles)));
        if (int st = room(bands)) return st;
        norm_grad_columns<T><<<dim3(unsigned(tiles), bands), 128, 0, on>>>(gs, grad_stride, xs, x_stride, stats, partial, rows, cols);
        if (int st = check_launch("layer norm backward")) return st;
      }
      if (dx) {
        const unsigned grid = unsigned(std::min<size_t>(rows, 1u << 30));
        norm_grad_wide<T, P><<<grid, 1024, 0, on>>>(gs, grad_stride, xs, x_stride, stats, ws, dx, grad_x_stride, rows, cols);
        if (int st = check_launch("layer norm backward")) return st;
      }
    }
    if (!sums) return TC_OK;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(unsigned((2 * cols + 31) / 32));
    config.blockDim = dim3(1024);
    config.stream = on;
    config.attrs = &early;
    config.numAttrs = 1;
    if (int st = check_cuda(cudaLaunchKernelEx(&config, norm_grad_join<P>, static_cast<const float *>(partial), parts, cols, dw, db),
                            "layer norm backward"))
      return st;
    return check_launch("layer norm backward");
  });
}

}  // extern "C"
