// gradnorm.cu — the global norm of many gradients, and clipping by it.
//
//   norm = sqrt(sum over all tensors of sum(g^2))
//   g <- g min(1, limit / norm)
//
// Squares and sums are f64, so that no f32 gradient's square overflows or
// vanishes, and are added in an order that does not change from run to run on
// the same buffers.
// The reference has no counterpart (its optimizers take gradients as they
// are).
#include <algorithm>

#include "rows.cuh"

namespace tc {
namespace {

// The tensors of one launch travel in the kernel's parameters: up to MAX of
// them, 16 (0.6 KB of parameters) or 512 (18 KB).  A tensor is cut into
// chunks of CHUNK bytes, which the launch's blocks take in turn; first[i] is
// the number of chunks before tensor i.
constexpr unsigned CHUNK = 32768, FEW = 16, MANY = 512;
template <unsigned MAX> struct GradSet {
  unsigned count, chunks;
  unsigned first[MAX];
  tc_gradient of[MAX];
};

template <unsigned MAX> __device__ __forceinline__ unsigned find(const GradSet<MAX> &set, unsigned chunk) {
  unsigned low = 0, high = set.count - 1;
  while (low < high) {
    const unsigned mid = (low + high + 1) / 2;
    if (set.first[mid] <= chunk) low = mid;
    else high = mid - 1;
  }
  return low;
}

// The elements of a tensor before its first 128-byte line (at most n): the
// first chunk has them beside its own, so that every chunk's runs of 16 bytes
// fill whole lines, wherever the tensor starts.
__host__ __device__ __forceinline__ size_t before_line(const void *p, size_t n, size_t bytes) {
  const size_t k = (128 - reinterpret_cast<uintptr_t>(p) % 128) % 128 / bytes;
  return k < n ? k : n;
}
// one(index, element) and many(index, run) for this thread's share of a chunk.
template <class S, class One, class Many>
__device__ __forceinline__ void walk_chunk(const S *p, size_t n, unsigned chunk, One &&one, Many &&many) {
  constexpr unsigned V = 16 / sizeof(S), PER = CHUNK / sizeof(S);
  const size_t lead = before_line(p, n, sizeof(S)), begin = lead + size_t(chunk) * PER;
  const unsigned t = threadIdx.x;
  if (chunk == 0 && t < lead) one(t, p[t]);
  const unsigned len = unsigned(min(size_t(PER), n - begin)), runs = len / V, after = runs * V;
  const S *at = p + begin;
  unsigned i = t;
  for (; i + 3 * blockDim.x < runs; i += 4 * blockDim.x) {
    Run<S, V> r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = load_run<S, V>(at + size_t(i + u * blockDim.x) * V);
#pragma unroll
    for (int u = 0; u < 4; ++u) many(begin + size_t(i + u * blockDim.x) * V, r[u]);
  }
  for (; i < runs; i += blockDim.x) many(begin + size_t(i) * V, load_run<S, V>(at + size_t(i) * V));
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

// Each block's sum of squares, at partial[slot + block].  Of the blocks of the
// call's last launch (the one with a ticket; the others are done before it
// begins) the last to finish adds up the blocks' sums of all launches, in their
// order, and sets the ticket back to zero.  A launch that fails leaves no ticket
// taken.  Bound by HBM: 769M bf16 in 250 us, 6.2 TB/s, the widening to f64 (16
// lanes a clock) 70% busy.  Of gradients that L2 holds (67 MB), 1 to 20 MB come
// from HBM in a loop of steps, and the 19 us are not HBM's: 7.5 of them are the
// widening's, the rest ramps up, down and through the last block's sum.
template <unsigned MAX>
__global__ void __launch_bounds__(256) square_sums(const __grid_constant__ GradSet<MAX> set, double *partial, unsigned slot,
                                                   int *ticket, float *norm) {
  __shared__ double room[2][8];
  __shared__ bool last;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // clip_set, which waits for the norm
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
  sum = block_sum(sum, room[0]);
  if (threadIdx.x == 0) {
    partial[slot + blockIdx.x] = sum;
    __threadfence();
    last = ticket && unsigned(atomicAdd(ticket, 1)) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  sum = 0.0;
  for (unsigned i = threadIdx.x; i < slot + gridDim.x; i += blockDim.x) sum += __ldcg(partial + i);
  sum = block_sum(sum, room[1]);
  if (threadIdx.x == 0) {
    *norm = float(sqrt(sum));
    *ticket = 0;
  }
}

// The norm of no gradients.
__global__ void zero_norm(float *norm) { *norm = 0.0f; }

// The chunks from the last to the first: the last ones read for the norm are
// still in L2 (of 67 MB, 12 to 21 MB are read from HBM and 47 to 62 written).
// Bound by HBM: 769M bf16 in 550 us, 5.6 TB/s.
template <unsigned MAX>
__global__ void __launch_bounds__(256) clip_set(const __grid_constant__ GradSet<MAX> set, const float *norm, float limit) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
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
            if (whole) {
              union {
                uint4 w;
                Run<S, V> r;
              } u;
              u.r = r;
              __stcs(reinterpret_cast<uint4 *>(out + at), u.w);
            }
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
template <unsigned MAX, class F> int in_sets(const tc_gradient *grads, size_t count, F &&f) {
  GradSet<MAX> set;
  set.count = set.chunks = 0;
  for (size_t i = 0; i < count; ++i) {
    if (grads[i].n == 0) continue;
    const size_t bytes = dtype_bytes(grads[i].dtype), per = CHUNK / bytes;
    const size_t chunks = std::max<size_t>(1, (grads[i].n - before_line(grads[i].g, grads[i].n, bytes) + per - 1) / per);
    if (set.count == MAX || set.chunks + chunks > 0x7fffffffu) {
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

template <unsigned MAX> int norm_run(const tc_gradient *grads, size_t count, float *norm, cudaStream_t on) {
  const unsigned blocks = unsigned(sm_count()) * 8;
  unsigned total = 0;
  in_sets<MAX>(grads, count, [&](const GradSet<MAX> &set) {
    total += std::min(blocks, set.chunks);
    return int(TC_OK);
  });
  if (total == 0) {
    zero_norm<<<1, 1, 0, on>>>(norm);
    return check_launch("grad norm");
  }
  void *room = nullptr;
  if (int st = scratch(size_t(total) * sizeof(double), &room, on)) return st;
  int *ticket = nullptr;
  if (int st = counters(1, &ticket, on)) return st;
  unsigned slot = 0;
  return in_sets<MAX>(grads, count, [&](const GradSet<MAX> &set) -> int {
    const unsigned grid = std::min(blocks, set.chunks);
    int *last = slot + grid == total ? ticket : nullptr;
    square_sums<MAX><<<grid, 256, 0, on>>>(set, static_cast<double *>(room), slot, last, norm);
    slot += grid;
    return check_launch("grad norm");
  });
}

template <unsigned MAX> int clip_run(const tc_gradient *grads, size_t count, const float *norm, float limit, cudaStream_t on) {
  return in_sets<MAX>(grads, count, [&](const GradSet<MAX> &set) -> int {
    cudaLaunchAttribute early{};  // beside the norm's last blocks
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(std::min(unsigned(sm_count()) * 8, set.chunks));
    config.blockDim = dim3(256);
    config.stream = on;
    config.attrs = &early;
    config.numAttrs = 1;
    return check_cuda(cudaLaunchKernelEx(&config, clip_set<MAX>, set, norm, limit), "clip grads");
  });
}

}  // namespace
}  // namespace tc

using namespace tc;

extern "C" {

int tc_grad_norm(const tc_gradient *grads, size_t count, float *norm, void *stream) {
  if (int st = check_list("grad norm", grads, count, false)) return st;
  if (!norm) return fail(TC_EINVAL, "grad norm: null pointer");
  return count <= FEW ? norm_run<FEW>(grads, count, norm, as_stream(stream)) : norm_run<MANY>(grads, count, norm, as_stream(stream));
}

int tc_clip_grads(const tc_gradient *grads, size_t count, const float *norm, double limit, void *stream) {
  if (int st = check_list("clip grads", grads, count, true)) return st;
  if (!norm) return fail(TC_EINVAL, "clip grads: null pointer");
  if (!(limit >= 0.0)) return fail(TC_EINVAL, "clip grads: limit %g", limit);
  return count <= FEW ? clip_run<FEW>(grads, count, norm, float(limit), as_stream(stream))
                      : clip_run<MANY>(grads, count, norm, float(limit), as_stream(stream));
}

}  // extern "C"
