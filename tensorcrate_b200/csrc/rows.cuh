// rows.cuh — what the row kernels of the training operators share (layer
// norm, token log probabilities): runs of elements loaded and stored in one
// access, and sums over a warp and over a block.
#pragma once

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

// Whether runs of E elements of `bytes` each can be moved whole from rows
// that start at `p`, `stride` elements apart.
inline bool runs_fit(const void *p, size_t stride, size_t rows, size_t bytes, int e) {
  const size_t run = bytes * size_t(e);
  return reinterpret_cast<uintptr_t>(p) % run == 0 && (rows <= 1 || (stride * bytes) % run == 0);
}

}  // namespace tc
