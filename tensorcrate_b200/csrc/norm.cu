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

// A row's elements stay in the registers of the threads that share it, so x
// is read once for both of the variance's passes.  Access k of thread t
// covers the E elements from (t + k * threads) * E: neighbours read
// neighbouring addresses.
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

// Rows too wide for the registers of one block: a block reads its row three
// times, the second and third from L2.
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

// grad_x, and this block's share of grad_w and grad_b: a block walks its
// rows and keeps the sums of the columns that its threads own in registers,
// then writes them to its row of `partial` (w's sums, then b's).
template <class T, class P, int E, int K>
__global__ void __launch_bounds__(512) norm_grad_rows(const typename T::S *g, size_t g_stride,
                                                      const typename T::S *x, size_t x_stride,
                                                      const float2 *__restrict__ statistics,
                                                      const typename P::S *__restrict__ w,
                                                      typename T::S *dx, size_t dx_stride,
                                                      float *__restrict__ partial, size_t rows, unsigned cols) {
  using S = typename T::S;
  __shared__ float room[2][2][32];
  const unsigned t = threadIdx.x, threads = blockDim.x;
  const float share = 1.0f / float(cols);
  float sum_w[K * E], sum_b[K * E];
#pragma unroll
  for (int i = 0; i < K * E; ++i) sum_w[i] = sum_b[i] = 0.0f;
  int turn = 0;
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x, turn ^= 1) {
    Run<S, E> xr[K], gr[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const unsigned c = (t + k * threads) * E;
      if (c < cols) {
        xr[k] = load_run<S, E>(x + r * x_stride + c);
        gr[k] = load_run<S, E>(g + r * g_stride + c);
      }
    }
    const float2 st = statistics[r];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const unsigned c = (t + k * threads) * E;
      if (c >= cols) break;
      float wv[E];
      if (w) load_wide<P, E>(w + c, wv);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float h = (T::load(xr[k].e[j]) - st.x) * st.y, gv = T::load(gr[k].e[j]);
        const float gw = w ? gv * wv[j] : gv;
        s1 += gw;
        s2 += gw * h;
        sum_w[k * E + j] += gv * h;
        sum_b[k * E + j] += gv;
      }
    }
    if (!dx) continue;
    const float c1 = block_sum(s1, room[turn][0]) * share, c2 = block_sum(s2, room[turn][1]) * share;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const unsigned c = (t + k * threads) * E;
      if (c >= cols) break;
      float wv[E];
      if (w) load_wide<P, E>(w + c, wv);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float h = (T::load(xr[k].e[j]) - st.x) * st.y, gv = T::load(gr[k].e[j]);
        xr[k].e[j] = T::store(st.y * ((w ? gv * wv[j] : gv) - c1 - h * c2));
      }
      store_run<S, E>(dx + r * dx_stride + c, xr[k]);
    }
  }
  if (!partial) return;
  float *pw = partial + size_t(blockIdx.x) * 2 * cols, *pb = pw + cols;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const unsigned c = (t + k * threads) * E;
    if (c >= cols) break;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      pw[c + j] = sum_w[k * E + j];
      pb[c + j] = sum_b[k * E + j];
    }
  }
}

// Rows too wide for that: grad_x by blocks that read their row twice ...
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

// grad_w and grad_b from the blocks' partial sums, added in the blocks'
// order: 32 columns a block, its 8 warps each an eighth of the partials.
template <class P>
__global__ void __launch_bounds__(256) norm_grad_join(const float *__restrict__ partial, unsigned parts, size_t cols,
                                                      typename P::S *__restrict__ dw, typename P::S *__restrict__ db) {
  __shared__ float room[8][33];
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t i = size_t(blockIdx.x) * 32 + lane;  // column of [w's sums | b's sums]
  float v = 0.0f;
  if (i < 2 * cols) {
#pragma unroll 8
    for (unsigned p = warp; p < parts; p += 8) v += partial[size_t(p) * 2 * cols + i];
  }
  room[warp][lane] = v;
  __syncthreads();
  if (warp || i >= 2 * cols) return;
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) sum += room[k][lane];
  if (i < cols) {
    if (dw) dw[i] = P::store(sum);
  } else if (db) {
    db[i - cols] = P::store(sum);
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
    if (cols <= 16 * 1024) return whole ? launch(std::integral_constant<int, V>{}) : launch(std::integral_constant<int, 1>{});
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
    auto launch = [&](auto e, auto k) -> int {
      constexpr int E = decltype(e)::value, K = decltype(k)::value;
      const unsigned n = unsigned((cols + E - 1) / E);
      const unsigned threads = ((n + K - 1) / K + 31) / 32 * 32;
      int resident = 0;
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, norm_grad_rows<T, P, E, K>, int(threads), 0);
      const unsigned grid = unsigned(std::min<size_t>(rows, size_t(sm_count()) * size_t(std::max(1, resident))));
      if (sums)
        if (int st = room(grid)) return st;
      norm_grad_rows<T, P, E, K><<<grid, threads, 0, on>>>(gs, grad_stride, xs, x_stride, stats, ws, dx, grad_x_stride,
                                                           partial, rows, unsigned(cols));
      return check_launch("layer norm backward");
    };
    if (cols <= 16 * 512) {
      if (int st = whole ? launch(std::integral_constant<int, V>{}, std::integral_constant<int, 16 / V>{})
                         : launch(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{}))
        return st;
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
    const size_t blocks = (2 * cols + 31) / 32;
    norm_grad_join<P><<<unsigned(blocks), 256, 0, on>>>(partial, parts, cols, dw, db);
    return check_launch("layer norm backward");
  });
}

}  // extern "C"
