// gradnorm.cu — the global norm of many gradients, and clipping by it.
//
//   norm = sqrt(sum over all tensors of sum(g^2))
//   g <- g min(1, limit / norm)
//
// Squares and sums are f64, so that no f32 gradient's square overflows or
// vanishes, and are added in an order that does not change from run to run.
// The reference has no counterpart (its optimizers take gradients as they
// are).
#include <algorithm>

#include "rows.cuh"

namespace tc {
namespace {

// The tensors of one launch travel in the kernel's parameters.  A tensor is
// cut into chunks of CHUNK bytes, which the launch's blocks take in turn;
// first[i] is the number of chunks before tensor i.
constexpr unsigned CHUNK = 32768, MAX_SET = 512;
struct GradSet {
  unsigned count, chunks;
  unsigned first[MAX_SET];
  tc_gradient of[MAX_SET];
};

__device__ __forceinline__ unsigned find(const GradSet &set, unsigned chunk) {
  unsigned low = 0, high = set.count - 1;
  while (low < high) {
    const unsigned mid = (low + high + 1) / 2;
    if (set.first[mid] <= chunk) low = mid;
    else high = mid - 1;
  }
  return low;
}

// Elements [begin, end) of a tensor's chunk: single ones up to the first
// 16-byte boundary, runs of 16 bytes, single ones after them.
template <class S, class One, class Many>
__device__ __forceinline__ void walk_chunk(const S *p, size_t n, unsigned chunk, One &&one, Many &&many) {
  constexpr unsigned V = 16 / sizeof(S), PER = CHUNK / sizeof(S);
  const size_t begin = size_t(chunk) * PER;
  const unsigned len = unsigned(min(size_t(PER), n - begin));
  const S *at = p + begin;
  const unsigned off = unsigned(reinterpret_cast<uintptr_t>(at) & 15) / unsigned(sizeof(S));
  const unsigned head = min(len, (V - off) % V), runs = (len - head) / V, after = head + runs * V;
  const unsigned t = threadIdx.x;
  if (t < head) one(begin + t, at[t]);
  unsigned i = t;
  for (; i + 3 * blockDim.x < runs; i += 4 * blockDim.x) {
    Run<S, V> r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = load_run<S, V>(at + head + size_t(i + u * blockDim.x) * V);
#pragma unroll
    for (int u = 0; u < 4; ++u) many(begin + head + size_t(i + u * blockDim.x) * V, r[u]);
  }
  for (; i < runs; i += blockDim.x) many(begin + head + size_t(i) * V, load_run<S, V>(at + head + size_t(i) * V));
  if (t < len - after) one(begin + after + t, at[after + t]);
}

template <class F> __device__ __forceinline__ void with_kind(int dtype, F &&f) {
  if (dtype == TC_F32) f(F32T{});
  else if (dtype == TC_F16) f(F16T{});
  else f(BF16T{});
}

__device__ __forceinline__ double block_sum(double v, double *room) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) room[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? room[lane] : 0.0;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Each block's sum of squares, at partial[slot + block].
__global__ void __launch_bounds__(256) square_sums(const __grid_constant__ GradSet set, double *partial, unsigned slot) {
  __shared__ double room[8];
  double sum = 0.0;
  for (unsigned c = blockIdx.x; c < set.chunks; c += gridDim.x) {
    const unsigned i = find(set, c);
    with_kind(set.of[i].dtype, [&](auto t) {
      using T = decltype(t);
      using S = typename T::S;
      constexpr unsigned V = 16 / sizeof(S);
      walk_chunk(
          static_cast<const S *>(set.of[i].g), set.of[i].n, c - set.first[i],
          [&](size_t, S e) {
            const double v = T::load(e);
            sum += v * v;
          },
          [&](size_t, const Run<S, V> &r) {
            double part = 0.0;
#pragma unroll
            for (unsigned j = 0; j < V; ++j) {
              const double v = T::load(r.e[j]);
              part += v * v;
            }
            sum += part;
          });
    });
  }
  sum = block_sum(sum, room);
  if (threadIdx.x == 0) partial[slot + blockIdx.x] = sum;
}

__global__ void __launch_bounds__(256) norm_of(const double *partial, unsigned n, float *norm) {
  __shared__ double room[8];
  double sum = 0.0;
  for (unsigned i = threadIdx.x; i < n; i += blockDim.x) sum += partial[i];
  sum = block_sum(sum, room);
  if (threadIdx.x == 0) *norm = float(sqrt(sum));
}

__global__ void __launch_bounds__(256) clip_set(const __grid_constant__ GradSet set, const float *norm, float limit) {
  const float n = *norm;
  // a norm of zero clips nothing; a NaN carries on
  const float by = n <= limit ? 1.0f : limit / n;
  for (unsigned k = blockIdx.x; k < set.chunks; k += gridDim.x) {
    const unsigned c = set.chunks - 1 - k, i = find(set, c);
    const tc_gradient &x = set.of[i];
    if (by == 1.0f && x.out == x.g) continue;  // nothing to change
    with_kind(x.dtype, [&](auto t) {
      using T = decltype(t);
      using S = typename T::S;
      constexpr unsigned V = 16 / sizeof(S);
      S *out = static_cast<S *>(x.out);
      const bool whole = ((reinterpret_cast<uintptr_t>(x.out) ^ reinterpret_cast<uintptr_t>(x.g)) & 15) == 0;
      walk_chunk(
          static_cast<const S *>(x.g), x.n, c - set.first[i], [&](size_t at, S e) { out[at] = T::store(T::load(e) * by); },
          [&](size_t at, Run<S, V> r) {
#pragma unroll
            for (unsigned j = 0; j < V; ++j) r.e[j] = T::store(T::load(r.e[j]) * by);
            if (whole) store_run<S, V>(out + at, r);
            else
#pragma unroll
              for (unsigned j = 0; j < V; ++j) out[at + j] = r.e[j];
          });
    });
  }
}

int check_list(const char *what, const tc_gradient *grads, size_t count, bool outs) {
  if (count && !grads) return fail(TC_EINVAL, "%s: null tensor list", what);
  for (size_t i = 0; i < count; ++i) {
    const tc_gradient &x = grads[i];
    if (x.dtype != TC_F32 && x.dtype != TC_F16 && x.dtype != TC_BF16)
      return fail(TC_EINVAL, "%s: tensor %zu has element type %d", what, i, x.dtype);
    if (x.n && (!x.g || (outs && !x.out))) return fail(TC_EINVAL, "%s: null pointer in tensor %zu", what, i);
    if (x.n > size_t(1) << 40) return fail(TC_ERANGE, "%s: tensor %zu has %zu elements", what, i, x.n);
  }
  return TC_OK;
}

// The list in sets of one launch each: f(set).
template <class F> int in_sets(const tc_gradient *grads, size_t count, F &&f) {
  GradSet set;
  set.count = set.chunks = 0;
  for (size_t i = 0; i < count; ++i) {
    if (grads[i].n == 0) continue;
    const size_t per = CHUNK / dtype_bytes(grads[i].dtype), chunks = (grads[i].n + per - 1) / per;
    if (set.count == MAX_SET || set.chunks + chunks > 0x7fffffffu) {
      if (set.count)
        if (int st = f(set)) return st;
      set.count = set.chunks = 0;
    }
    set.first[set.count] = set.chunks;
    set.of[set.count++] = grads[i];
    set.chunks += unsigned(chunks);
  }
  return set.count ? f(set) : TC_OK;
}

}  // namespace
}  // namespace tc

using namespace tc;

extern "C" {

int tc_grad_norm(const tc_gradient *grads, size_t count, float *norm, void *stream) {
  if (int st = check_list("grad norm", grads, count, false)) return st;
  if (!norm) return fail(TC_EINVAL, "grad norm: null pointer");
  cudaStream_t on = as_stream(stream);
  const unsigned blocks = unsigned(sm_count()) * 8;
  size_t sets = 0;
  if (int st = in_sets(grads, count, [&](const GradSet &) { return ++sets, int(TC_OK); })) return st;
  void *room = nullptr;
  if (int st = scratch(std::max<size_t>(1, sets) * blocks * sizeof(double), &room, on)) return st;
  double *partial = static_cast<double *>(room);
  unsigned filled = 0;
  if (int st = in_sets(grads, count, [&](const GradSet &set) -> int {
        const unsigned grid = std::min(blocks, set.chunks);
        square_sums<<<grid, 256, 0, on>>>(set, partial, filled);
        filled += grid;
        return check_launch("grad norm");
      }))
    return st;
  norm_of<<<1, 256, 0, on>>>(partial, filled, norm);
  return check_launch("grad norm");
}

int tc_clip_grads(const tc_gradient *grads, size_t count, const float *norm, double limit, void *stream) {
  if (int st = check_list("clip grads", grads, count, true)) return st;
  if (!norm) return fail(TC_EINVAL, "clip grads: null pointer");
  if (!(limit >= 0.0)) return fail(TC_EINVAL, "clip grads: limit %g", limit);
  return in_sets(grads, count, [&](const GradSet &set) -> int {
    const unsigned grid = std::min(unsigned(sm_count()) * 8, set.chunks);
    clip_set<<<grid, 256, 0, as_stream(stream)>>>(set, norm, float(limit));
    return check_launch("clip grads");
  });
}

}  // extern "C"
