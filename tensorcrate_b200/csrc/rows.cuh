// rows.cuh — what the row kernels of the training operators share (layer
// norm, token log probabilities): runs of elements loaded and stored in one
// access, and sums over a warp and over a block.
#pragma once

#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace tc {

// E consecutive elements of storage type S, moved in one access of E *
// sizeof(S) bytes (2, 4, 8 or 16).
template <class S, int E> struct alignas(E * sizeof(S)) Run {
  S e[E];
};
template <int BYTES> struct Word;
template <> struct Word<2> { using type = unsigned short; };
template <> struct Word<4> { using type = unsigned int; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };

template <class S, int E> __device__ __forceinline__ Run<S, E> load_run(const S *p) {
  using W = typename Word<E * sizeof(S)>::type;
  union {
    W w;
    Run<S, E> r;
  } u;
  u.w = *reinterpret_cast<const W *>(p);
  return u.r;
}
template <class S, int E> __device__ __forceinline__ void store_run(S *p, const Run<S, E> &r) {
  using W = typename Word<E * sizeof(S)>::type;
  union {
    W w;
    Run<S, E> r;
  } u;
  u.r = r;
  *reinterpret_cast<W *>(p) = u.w;
}

// Two f32 in one register pair.  sm_100a adds, multiplies and fuses both in
// one instruction, each half rounded as the scalar operation rounds it.
using F2 = unsigned long long;
__device__ __forceinline__ F2 pair(float lo, float hi) {
  F2 p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ float2 split(F2 p) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// A word of two elements of a 16-bit type, low first, widened and rounded as
// the single ones are.
template <class T> __device__ __forceinline__ F2 widen2(uint32_t w) {
  if constexpr (T::code == TC_BF16) {
    return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return pair(v.x, v.y);
  }
}
template <class T> __device__ __forceinline__ uint32_t narrow2(F2 p) {
  const float2 v = split(p);
  if constexpr (T::code == TC_BF16) return pack2_bf16(v.x, v.y);
  else return pack2_f16(v.x, v.y);
}

// E consecutive elements (16 bytes of them) as pairs of f32, and back.
template <class T> __device__ __forceinline__ void load_pairs(const typename T::S *p, F2 *v) {
  if constexpr (T::code == TC_F32) {
    const ulonglong2 r = *reinterpret_cast<const ulonglong2 *>(p);
    v[0] = r.x;
    v[1] = r.y;
  } else {
    const uint4 r = *reinterpret_cast<const uint4 *>(p);
    v[0] = widen2<T>(r.x);
    v[1] = widen2<T>(r.y);
    v[2] = widen2<T>(r.z);
    v[3] = widen2<T>(r.w);
  }
}
template <class T> __device__ __forceinline__ void store_pairs(typename T::S *p, const F2 *v) {
  if constexpr (T::code == TC_F32) {
    *reinterpret_cast<ulonglong2 *>(p) = make_ulonglong2(v[0], v[1]);
  } else {
    *reinterpret_cast<uint4 *>(p) = make_uint4(narrow2<T>(v[0]), narrow2<T>(v[1]), narrow2<T>(v[2]), narrow2<T>(v[3]));
  }
}

// E consecutive elements of type T as f32, in accesses of at most 16 bytes.
template <class T, int E> __device__ __forceinline__ void load_wide(const typename T::S *p, float (&v)[E]) {
  using S = typename T::S;
  constexpr int A = E * sizeof(S) > 16 ? int(16 / sizeof(S)) : E;
#pragma unroll
  for (int i = 0; i < E; i += A) {
    const Run<S, A> r = load_run<S, A>(p + i);
#pragma unroll
    for (int j = 0; j < A; ++j) v[i + j] = T::load(r.e[j]);
  }
}

// Copies 16 bytes from global to shared memory; a thread's copies complete in
// the order of its commits.
__device__ __forceinline__ void copy_async(uint32_t to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until at most LEFT of this thread's last commits are under way.
template <int LEFT> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The sum of `v` over the block, for every thread of it.  `room` holds one
// float per warp; a caller that sums again before a barrier of its own
// passes another room.
__device__ __forceinline__ float block_sum(float v, float *room) {
  v = warp_sum(v);
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) room[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < warps ? room[lane] : 0.0f);
}

// The blocks of a cluster share a row: this block's part, and how many there
// are (1 without a cluster).
__device__ __forceinline__ unsigned cluster_part() {
  unsigned v;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(v));
  return v;
}
__device__ __forceinline__ unsigned cluster_parts() {
  unsigned v;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(v));
  return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
// Store to the same variable of block `part`, which has to have started: a
// kernel's first such store comes after a barrier of the cluster.
template <class V> __device__ __forceinline__ void store_at(V *own, unsigned part, V v) {
  uint32_t to;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(uint32_t(__cvta_generic_to_shared(own))), "r"(part));
  if constexpr (sizeof(V) == 4) asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to), "r"(__float_as_uint(v)) : "memory");
  else asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(to), "l"(v) : "memory");
}
// Launch `kernel` in clusters of `parts` blocks.
template <class... A>
inline int launch(const char *what, void (*kernel)(A...), size_t clusters, unsigned parts, unsigned threads, size_t shared,
           cudaStream_t stream, std::common_type_t<A>... args) {
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = parts;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(unsigned(clusters * parts));
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  config.attrs = &cluster;
  config.numAttrs = parts > 1 ? 1 : 0;
  return check_cuda(cudaLaunchKernelEx(&config, kernel, args...), what);
}

// Let `kernel` have up to `bytes` of dynamic shared memory on the current
// device; `done` remembers the devices that were told.
inline int allow_shared(const char *what, const void *kernel, size_t bytes, std::atomic<uint64_t> &done) {
  int dev = 0;
  if (int st = check_cuda(cudaGetDevice(&dev), what)) return st;
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return TC_OK;
  if (int st = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)), what)) return st;
  done.fetch_or(bit, std::memory_order_relaxed);
  return TC_OK;
}

// Whether runs of E elements of `bytes` each can be moved whole from rows
// that start at `p`, `stride` elements apart.
inline bool runs_fit(const void *p, size_t stride, size_t rows, size_t bytes, int e) {
  const size_t run = bytes * size_t(e);
  return reinterpret_cast<uintptr_t>(p) % run == 0 && (rows <= 1 || (stride * bytes) % run == 0);
}

}  // namespace tc
