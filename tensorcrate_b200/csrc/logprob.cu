// logprob.cu — log probabilities of given tokens under rows of logits, with
// the rows' entropy, their likeliest tokens, and the logits' gradient.
//
//   m = max(x),  S = sum(exp(x - m)),  log p_j = (x_j - m) - log S
//   logprob = log p_token
//   entropy H = -sum(p log p) = log S - sum(exp(x - m) (x - m)) / S
//   gradient of sum(u logprob + v H):  u ([j = token] - p_j) - v p_j (log p_j + H)
//
// Everything is computed in f32.  A row's maximum and log S are kept apart:
// their sum would lose the low bits of log p where the logits are large.
// Elements of minus infinity have probability zero and add nothing; a row of
// nothing else has the statistics (-inf, 0), the logprob -inf, the entropy 0
// and the gradient 0.  A NaN or an infinity among a row's logits makes the
// row's results NaN, as the formulas do.  The reference has no counterpart.
#include <algorithm>
#include <type_traits>

#include "rows.cuh"

namespace tc {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp_of(float x) { return exp2_of(x * LOG2E); }

// The statistics of some elements of a row: their maximum (NaNs passed
// over), the sum of exp(x - m) and, for the entropy, the sum of exp(x - m)
// (x - m).  While m is -inf the sums are those of exp(x).
struct Sums {
  float m = -INFINITY, s = 0.0f, t = 0.0f;
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }

// Restate the sums for the larger maximum `m`.
template <bool ENT> __device__ __forceinline__ void raise(Sums &a, float m) {
  if (a.m != -INFINITY) {  // else s and t are 0, or NaN
    // the bound keeps up s finite where a.m is as low as the type goes (f is 0)
    const float up = fminf(m - a.m, 1e20f), f = exp_of(-up);
    if (ENT) a.t = f * (a.t - up * a.s);
    a.s *= f;
  }
  a.m = m;
}
template <bool ENT> __device__ __forceinline__ void join(Sums &a, Sums b) {
  if (b.m > a.m) raise<ENT>(a, b.m);
  else if (a.m > b.m) raise<ENT>(b, a.m);
  a.s += b.s;
  if (ENT) a.t += b.t;
}
// Over a warp: the maximum first, so that each lane restates its sums once.
template <bool ENT> __device__ __forceinline__ Sums warp_join(Sums a) {
  float m = a.m;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (m > a.m) raise<ENT>(a, m);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    if (ENT) a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
  }
  return a;
}
template <bool ENT> __device__ __forceinline__ Sums block_join(Sums a, Sums *room) {
  a = warp_join<ENT>(a);
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) room[threadIdx.x >> 5] = a;
  __syncthreads();
  return warp_join<ENT>(lane < warps ? room[lane] : Sums{});
}

// 16 bytes of a row: V elements, as they are stored.
template <class T> struct Bits {
  static constexpr unsigned V = 16 / sizeof(typename T::S), PAIRS = V / 2;
  uint4 w;
  __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
  __device__ __forceinline__ F2 pair_at(int i) const {
    if constexpr (T::code == TC_F32) return pair(__uint_as_float(word(2 * i)), __uint_as_float(word(2 * i + 1)));
    else return widen2<T>(word(i));
  }
  // The element, widened, with an index known at run time.
  __device__ __forceinline__ float at(unsigned i) const {
    if constexpr (T::code == TC_F32) return __uint_as_float(word(i));
    else return T::load(uint16_t(word(i / 2) >> (i % 2 * 16)));
  }
};
// The largest of the elements of U of them, NaNs passed over.
template <class T, int U> __device__ __forceinline__ float largest(const Bits<T> (&r)[U]) {
  if constexpr (T::code == TC_F32) {
    float m = r[0].at(0);
#pragma unroll
    for (int i = 1; i < 4 * U; ++i) m = fmaxf(m, __uint_as_float(r[i / 4].word(i % 4)));
    return m;
  } else {
    using H2 = std::conditional_t<T::code == TC_BF16, __nv_bfloat162, __half2>;
    auto as = [](uint32_t w) { return *reinterpret_cast<const H2 *>(&w); };
    H2 m = as(r[0].word(0));
#pragma unroll
    for (int i = 1; i < 4 * U; ++i) m = __hmax2(m, as(r[i / 4].word(i % 4)));
    const float2 v = split(widen2<T>(*reinterpret_cast<const uint32_t *>(&m)));
    return fmaxf(v.x, v.y);
  }
}

// A thread's statistics while it walks, the sums in two halves.
template <class T, bool ENT> struct Running {
  float m = -INFINITY, base = 0.0f;
  F2 s = 0, t = 0;
  __device__ __forceinline__ void lift(float to) {
    if (m != -INFINITY) {
      const float up = fminf(to - m, 1e20f), f = exp_of(-up);
      if (ENT) t = mul2(pair(f, f), fma2(pair(-up, -up), s, t));
      s = mul2(pair(f, f), s);
    }
    m = base = to;
  }
  // Add a pair whose elements m is not below.
  __device__ __forceinline__ void add(F2 v) {
    const F2 d = add2(v, pair(-base, -base));
    const float2 x = split(mul2(d, pair(LOG2E, LOG2E)));
    const F2 e = pair(exp2_of(x.x), exp2_of(x.y));
    s = add2(s, e);
    if (ENT) {
      // 0 for an element of -inf, NaN for a NaN (e is one)
      const float2 y = split(d);
      t = fma2(e, pair(fmaxf(y.x, -1e30f), fmaxf(y.y, -1e30f)), t);
    }
  }
  __device__ __forceinline__ Sums sums() const {
    const float2 a = split(s), b = split(t);
    return Sums{m, a.x + a.y, b.x + b.y};
  }
};

// A row's elements, or the part of them that one of `of` blocks has, as runs
// of 16 aligned bytes with the few single elements before and after them.
template <class T> struct Cut {
  using S = typename T::S;
  static constexpr unsigned V = 16 / sizeof(S);
  unsigned head, body, runs, after, tail;  // [0, head), runs from body, `tail` from after
  __device__ __forceinline__ Cut(const S *row, unsigned n, unsigned part = 0, unsigned of = 1) {
    const unsigned off = unsigned(reinterpret_cast<uintptr_t>(row) & 15) / unsigned(sizeof(S));
    head = min(n, (V - off) % V);
    const unsigned all = (n - head) / V, from = unsigned((unsigned long long)all * part / of);
    body = head + from * V;
    runs = unsigned((unsigned long long)all * (part + 1) / of) - from;
    after = head + all * V;
    tail = part + 1 == of ? n - after : 0;
    if (part) head = 0;
  }
};

// one(index, value) for the single elements that thread t of `threads` takes,
// many(index, bits, runs apart) for its runs, up to four at once, in ascending order.
template <class T, class Load, class One, class Many>
__device__ __forceinline__ void walk(const typename T::S *row, const Cut<T> &c, unsigned t, unsigned threads, Load &&load,
                                     One &&one, Many &&many) {
  if (t < c.head) one(t, row[t]);
  unsigned i = t;
  for (; c.runs > 3 * threads && i < c.runs - 3 * threads; i += 4 * threads) {
    Bits<T> r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = load(i + u * threads);
    many(i, r);
  }
  for (; i < c.runs; i += threads) {
    Bits<T> r[1] = {load(i)};
    many(i, r);
  }
  if (t < c.tail) one(c.after + t, row[c.after + t]);
}
template <class T> __device__ __forceinline__ auto from_row(const typename T::S *row, const Cut<T> &c) {
  const uint4 *p = reinterpret_cast<const uint4 *>(row + c.body);
  return [p](unsigned i) { return Bits<T>{p[i]}; };
}

// ---------------------------------------------------------------------------
// The likeliest tokens.  An element's key orders the row: the larger value
// first, of equal ones the lower index, NaNs last; 0 is no element.
// ---------------------------------------------------------------------------
using Key = unsigned long long;
__device__ __forceinline__ uint32_t ordered(float v) {
  if (isnan(v)) return 0;
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 is 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(Key k) {
  const uint32_t o = uint32_t(k >> 32);
  if (o == 0) return __int_as_float(0x7fc00000);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ Key key_of(float v, unsigned index) { return Key(ordered(v)) << 32 | uint32_t(~index); }

constexpr int MAX_TOP = 32, GROUPS = 64, ROOM = 2048;
struct TopRoom {
  Key group[GROUPS], kept[ROOM], best[MAX_TOP], least;
  unsigned holder[512], holders, count;
};

// The `k` largest keys of a row, in order, into room.best.  `mine` is the
// key of the thread's largest element and `m` a value that none of its
// elements passes.  The k-th largest of the largest keys of 64 groups of
// threads is a bound that k elements at least reach; in rows without
// structure few more do, and only threads with a maximum that large hold
// them.  Those threads' elements are read again, the ones that reach the
// bound are kept and ranked by counting.
template <class T>
__device__ __forceinline__ void top_of_row(const typename T::S *row, const Cut<T> &c, Key mine, float m, unsigned k,
                                           TopRoom &room) {
  using S = typename T::S;
  constexpr unsigned V = Cut<T>::V;
  const auto load = from_row<T>(row, c);
  const unsigned t = threadIdx.x, threads = blockDim.x, lanes = threads / GROUPS;
  Key g = mine;
  for (unsigned o = 1; o < lanes; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
  if (t % lanes == 0) room.group[t / lanes] = g;
  if (t == 0) room.holders = room.count = 0;
  __syncthreads();
  if (t < GROUPS) {
    unsigned rank = 0;
    const Key own = room.group[t];
    for (unsigned i = 0; i < GROUPS; ++i) rank += room.group[i] > own || (room.group[i] == own && i < t);
    if (rank == k - 1) room.least = own;
  }
  __syncthreads();
  const Key least = room.least;
  if ((Key(ordered(m)) << 32 | 0xffffffffu) >= least) room.holder[atomicAdd(&room.holders, 1u)] = t;
  auto keep = [&](unsigned at, float v) {
    const Key key = key_of(v, at);
    if (key < least) return;
    const unsigned slot = atomicAdd(&room.count, 1u);
    if (slot < ROOM) room.kept[slot] = key;
  };
  if (t < c.head) keep(t, T::load(row[t]));
  if (t < c.tail) keep(c.after + t, T::load(row[c.after + t]));
  __syncthreads();
  for (unsigned h = t >> 5; h < room.holders; h += threads >> 5)
    for (size_t i = room.holder[h] + size_t(t & 31) * threads; i < c.runs; i += size_t(threads) * 32) {
      const Bits<T> r = load(unsigned(i));
#pragma unroll
      for (unsigned j = 0; j < V; ++j) keep(c.body + unsigned(i) * V + j, r.at(j));
    }
  __syncthreads();
  const unsigned count = room.count;
  if (count <= ROOM) {
    for (unsigned i = t; i < count; i += threads) {
      const Key own = room.kept[i];
      unsigned rank = 0;
      for (unsigned j = 0; j < count; ++j) rank += room.kept[j] > own;
      if (rank < k) room.best[rank] = own;
    }
    __syncthreads();
    return;
  }
  // More than there is room for (a row with many NaNs, or whose large values
  // lie with few threads): the row is read once for each token.
  Key last = ~Key(0);
  for (unsigned n = 0; n < k; ++n) {
    Key best = 0;
    auto each = [&](unsigned at, float v) {
      const Key key = key_of(v, at);
      if (key < last && key > best) best = key;
    };
    auto many = [&](unsigned i, const auto &r) {
      constexpr int U = sizeof(r) / sizeof(r[0]);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (unsigned j = 0; j < V; ++j) each(c.body + (i + u * threads) * V + j, r[u].at(j));
    };
    walk<T>(row, c, t, threads, load, [&](unsigned at, S e) { each(at, T::load(e)); }, many);
#pragma unroll
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if ((t & 31) == 0) room.group[t >> 5] = best;
    __syncthreads();
    for (unsigned w = 0; w < threads >> 5; ++w) best = max(best, room.group[w]);
    __syncthreads();
    if (t == 0) room.best[n] = best;
    last = best;
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------
// The gradient of one row, given its statistics.
// ---------------------------------------------------------------------------
struct Slope {
  float base, log_sum, entropy, u, v;  // u, v: the gradients of the logprob and of the entropy
  unsigned token;
};
template <bool ENT> __device__ __forceinline__ float slope_at(const Slope &g, float x, unsigned at) {
  const float a = (x - g.base) - g.log_sum, p = exp_of(a);
  // 1 - p without its cancellation, where p is near one
  float d = at == g.token ? -g.u * expm1f(a) : -g.u * p;
  if (ENT) d -= g.v * p * (fmaxf(a, -1e30f) + g.entropy);
  return d;
}
template <bool ENT> __device__ __forceinline__ F2 slope_of_pair(const Slope &g, F2 x) {
  const F2 a = add2(add2(x, pair(-g.base, -g.base)), pair(-g.log_sum, -g.log_sum));
  const float2 y = split(mul2(a, pair(LOG2E, LOG2E)));
  const F2 p = pair(exp2_of(y.x), exp2_of(y.y));
  if (!ENT) return mul2(p, pair(-g.u, -g.u));
  // -p (u + v (a + H))
  const float2 z = split(a);
  const F2 c = add2(pair(fmaxf(z.x, -1e30f), fmaxf(z.y, -1e30f)), pair(g.entropy, g.entropy));
  return mul2(p, fma2(c, pair(-g.v, -g.v), pair(-g.u, -g.u)));
}
// load(i) gives the row's run i; elements before and after the runs, and the
// token's, are read from the row.
template <class T, bool ENT, class Load>
__device__ __forceinline__ void write_slope(const typename T::S *row, typename T::S *to, const Cut<T> &c, const Slope &g,
                                            unsigned t, unsigned threads, Load &&load) {
  using S = typename T::S;
  constexpr unsigned V = Cut<T>::V;
  const bool whole = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(to)) & 15) == 0;
  auto put = [&](unsigned at, uint4 w) {
    if (whole) {
      *reinterpret_cast<uint4 *>(to + at) = w;
    } else {
      union {
        uint4 w;
        S e[V];
      } u;
      u.w = w;
#pragma unroll
      for (unsigned j = 0; j < V; ++j) to[at + j] = u.e[j];
    }
  };
  if (g.u == 0.0f && (!ENT || g.v == 0.0f)) {
    // nothing flows back through this row, whatever its logits
    if (t < c.head) to[t] = S(0);
    for (unsigned i = t; i < c.runs; i += threads) put(c.body + i * V, make_uint4(0, 0, 0, 0));
    if (t < c.tail) to[c.after + t] = S(0);
    return;
  }
  auto many = [&](unsigned i, const auto &r) {
    constexpr int U = sizeof(r) / sizeof(r[0]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned at = c.body + (i + u * threads) * V;
      F2 d[V / 2];
#pragma unroll
      for (unsigned j = 0; j < V / 2; ++j) d[j] = slope_of_pair<ENT>(g, r[u].pair_at(j));
      union {
        uint4 w;
        S e[V];
      } out;
      if constexpr (T::code == TC_F32) {
        const float2 lo = split(d[0]), hi = split(d[1]);
        out.w = make_uint4(__float_as_uint(lo.x), __float_as_uint(lo.y), __float_as_uint(hi.x), __float_as_uint(hi.y));
      } else {
        out.w = make_uint4(narrow2<T>(d[0]), narrow2<T>(d[1]), narrow2<T>(d[2]), narrow2<T>(d[3]));
      }
      if (g.token - at < V) {
        const S special = T::store(slope_at<ENT>(g, r[u].at(g.token - at), g.token));
#pragma unroll
        for (unsigned j = 0; j < V; ++j)
          if (at + j == g.token) out.e[j] = special;
      }
      put(at, out.w);
    }
  };
  walk<T>(row, c, t, threads, load, [&](unsigned at, S e) { to[at] = T::store(slope_at<ENT>(g, T::load(e), at)); }, many);
}

struct TokenArgs {
  const void *logits;
  size_t stride, rows;
  unsigned vocab, top;
  const uint32_t *tokens;
  float *logprobs, *entropy;
  float2 *statistics;
  uint32_t *top_tokens;
  float *top_logprobs;
  const float *grad_logprobs, *grad_entropy, *kept_entropy;
  const float2 *kept_statistics;
  void *grad_logits;
  size_t grad_stride;
};

// The upstream gradients of row r: none for the logprob of a row without a
// token, or of one whose token is none of the vocabulary.
__device__ __forceinline__ Slope slope_of(const TokenArgs &a, size_t r, float2 st, float entropy) {
  Slope g;
  const bool empty = st.x == -INFINITY && st.y == 0.0f;
  g.base = base_of(st.x);
  g.log_sum = st.y;
  g.entropy = entropy;
  g.token = a.tokens ? a.tokens[r] : ~0u;
  g.u = a.grad_logprobs && g.token < a.vocab && !empty ? a.grad_logprobs[r] : 0.0f;
  g.v = a.grad_entropy && !empty ? a.grad_entropy[r] : 0.0f;
  return g;
}

enum Extra { NOTHING = 0, TOP = 1, GRADIENT = 2 };

// A block a row: the statistics in one pass, and then what is asked for.
template <class T, bool ENT, int EXTRA> __global__ void __launch_bounds__(512) token_rows(TokenArgs a) {
  using S = typename T::S;
  constexpr unsigned V = Cut<T>::V;
  __shared__ Sums room[16];
  const unsigned t = threadIdx.x, threads = blockDim.x;
  for (size_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const S *row = static_cast<const S *>(a.logits) + r * a.stride;
    const Cut<T> c(row, a.vocab);
    const unsigned token = a.tokens ? a.tokens[r] : ~0u;
    const float at_token = token < a.vocab ? T::load(row[token]) : __int_as_float(0x7fc00000);
    Running<T, ENT> run;
    // where the thread's largest element lies; its first, while all are -inf
    unsigned at = t < c.head ? t : t < c.runs ? c.body + t * V : t < c.tail ? c.after + t : ~0u;
    auto one = [&](unsigned i, S e) {
      const float v = T::load(e);
      if (v > run.m) {
        run.lift(v);
        if (EXTRA == TOP) at = i;
      }
      run.add(pair(v, -INFINITY));
    };
    auto many = [&](unsigned i, const auto &bits) {
      constexpr int U = sizeof(bits) / sizeof(bits[0]);
      const float m = largest(bits);
      if (m > run.m) {
        run.lift(m);
        if (EXTRA == TOP) {
#pragma unroll
          for (int u = U - 1; u >= 0; --u)
#pragma unroll
            for (int j = int(V) - 1; j >= 0; --j)
              if (bits[u].at(j) == m) at = c.body + (i + u * threads) * V + unsigned(j);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (unsigned j = 0; j < V / 2; ++j) run.add(bits[u].pair_at(j));
    };
    walk<T>(row, c, t, threads, from_row<T>(row, c), one, many);
    const Sums sums = run.sums();
    const Sums all = block_join<ENT>(sums, room);
    const bool empty = all.m == -INFINITY && all.s == 0.0f;
    const float2 st = make_float2(all.m, empty ? 0.0f : logf(all.s));
    const float entropy = !ENT || empty ? 0.0f : st.y - all.t / all.s;
    if (t == 0) {
      if (a.logprobs) a.logprobs[r] = token == ~0u ? 0.0f : (at_token - base_of(st.x)) - st.y;
      if (a.statistics) a.statistics[r] = st;
      if (ENT && a.entropy) a.entropy[r] = entropy;
    }
    if (EXTRA == TOP) {
      __shared__ TopRoom top;
      // a NaN among the thread's elements: `at` may not name one of value m
      const Key mine = at == ~0u || isnan(sums.s) ? 0 : key_of(sums.m, at);
      top_of_row<T>(row, c, mine, sums.m, a.top, top);
      if (t < a.top) {
        const Key k = top.best[t];
        a.top_tokens[r * a.top + t] = ~uint32_t(k);
        a.top_logprobs[r * a.top + t] = (value_of(k) - base_of(st.x)) - st.y;
      }
    }
    if (EXTRA == GRADIENT)
      write_slope<T, ENT>(row, static_cast<S *>(a.grad_logits) + r * a.grad_stride, c, slope_of(a, r, st, entropy), t, threads, from_row<T>(row, c));
    __syncthreads();
  }
}

// The gradient alone, from the statistics that the forward call left.
template <class T, bool ENT> __global__ void __launch_bounds__(512) token_slope(TokenArgs a) {
  using S = typename T::S;
  for (size_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const S *row = static_cast<const S *>(a.logits) + r * a.stride;
    const Cut<T> c(row, a.vocab);
    write_slope<T, ENT>(row, static_cast<S *>(a.grad_logits) + r * a.grad_stride, c,
                        slope_of(a, r, a.kept_statistics[r], ENT ? a.kept_entropy[r] : 0.0f), threadIdx.x, blockDim.x,
                        from_row<T>(row, c));
  }
}

int check(const char *what, size_t rows, size_t vocab, size_t stride, const char *name) {
  if (vocab == 0) return fail(TC_EINVAL, "%s: a vocabulary of no tokens", what);
  if (vocab >= TC_NO_TOKEN) return fail(TC_ERANGE, "%s: a vocabulary of %zu tokens", what, vocab);
  if (rows > 1 && stride < vocab)
    return fail(TC_EINVAL, "%s: rows of %s are %zu elements apart, fewer than the %zu tokens", what, name, stride, vocab);
  size_t end;
  if (__builtin_mul_overflow(rows, stride, &end) || __builtin_add_overflow(end, vocab, &end) || end > (size_t(1) << 60))
    return fail(TC_ERANGE, "%s: layout arithmetic of %s overflows", what, name);
  return TC_OK;
}
bool off_grid(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

unsigned threads_for(size_t vocab, size_t run) {
  const size_t want = vocab / run / 4;
  return want >= 512 ? 512 : want >= 256 ? 256 : 128;
}

}  // namespace
}  // namespace tc

using namespace tc;

extern "C" {

int tc_token_logprobs(int dtype, size_t rows, size_t vocab, const void *logits, size_t row_stride,
                      const uint32_t *tokens, float *logprobs, float *entropy, float *statistics, uint32_t top,
                      uint32_t *top_tokens, float *top_logprobs, void *stream) {
  return with_real(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (int st = check("token logprobs", rows, vocab, row_stride, "logits")) return st;
    if (top > TC_MAX_TOP || top > vocab)
      return fail(TC_EINVAL, "token logprobs: %u top tokens of %zu (at most %d)", top, vocab, TC_MAX_TOP);
    if (logprobs && !tokens) return fail(TC_EINVAL, "token logprobs: no tokens");
    if (rows == 0) return TC_OK;
    if (!logits || (top && (!top_tokens || !top_logprobs))) return fail(TC_EINVAL, "token logprobs: null pointer");
    if (off_grid(statistics, 8)) return fail(TC_EINVAL, "token logprobs: statistics are not on an 8-byte boundary");
    if (!logprobs && !entropy && !statistics && !top) return TC_OK;
    TokenArgs a{};
    a.logits = logits;
    a.stride = row_stride;
    a.rows = rows;
    a.vocab = unsigned(vocab);
    a.top = top;
    a.tokens = logprobs ? tokens : nullptr;
    a.logprobs = logprobs;
    a.entropy = entropy;
    a.statistics = reinterpret_cast<float2 *>(statistics);
    a.top_tokens = top_tokens;
    a.top_logprobs = top_logprobs;
    const unsigned grid = unsigned(std::min<size_t>(rows, 1u << 30)), threads = threads_for(vocab, 16 / sizeof(typename T::S));
    cudaStream_t on = as_stream(stream);
    if (top) {
      if (entropy) token_rows<T, true, TOP><<<grid, threads, 0, on>>>(a);
      else token_rows<T, false, TOP><<<grid, threads, 0, on>>>(a);
    } else {
      if (entropy) token_rows<T, true, NOTHING><<<grid, threads, 0, on>>>(a);
      else token_rows<T, false, NOTHING><<<grid, threads, 0, on>>>(a);
    }
    return check_launch("token logprobs");
  });
}

int tc_token_logprobs_backward(int dtype, size_t rows, size_t vocab, const void *logits, size_t row_stride,
                               const uint32_t *tokens, const float *statistics, const float *entropy,
                               const float *grad_logprobs, const float *grad_entropy, void *grad_logits,
                               size_t grad_stride, void *stream) {
  return with_real(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (int st = check("token logprobs backward", rows, vocab, row_stride, "logits")) return st;
    if (int st = check("token logprobs backward", rows, vocab, grad_stride, "grad_logits")) return st;
    if (grad_logprobs && !tokens) return fail(TC_EINVAL, "token logprobs backward: no tokens");
    if (grad_entropy && !entropy) return fail(TC_EINVAL, "token logprobs backward: no entropy");
    if (rows == 0) return TC_OK;
    if (!logits || !statistics || !grad_logits) return fail(TC_EINVAL, "token logprobs backward: null pointer");
    if (off_grid(statistics, 8)) return fail(TC_EINVAL, "token logprobs backward: statistics are not on an 8-byte boundary");
    TokenArgs a{};
    a.logits = logits;
    a.stride = row_stride;
    a.rows = rows;
    a.vocab = unsigned(vocab);
    a.tokens = tokens;
    a.kept_statistics = reinterpret_cast<const float2 *>(statistics);
    a.kept_entropy = entropy;
    a.grad_logprobs = grad_logprobs;
    a.grad_entropy = grad_entropy;
    a.grad_logits = grad_logits;
    a.grad_stride = grad_stride;
    const unsigned grid = unsigned(std::min<size_t>(rows, 1u << 30)), threads = threads_for(vocab, 16 / sizeof(typename T::S));
    if (grad_entropy) token_slope<T, true><<<grid, threads, 0, as_stream(stream)>>>(a);
    else token_slope<T, false><<<grid, threads, 0, as_stream(stream)>>>(a);
    return check_launch("token logprobs backward");
  });
}

int tc_token_loss(int dtype, size_t rows, size_t vocab, const void *logits, size_t row_stride, const uint32_t *tokens,
                  const float *grad_logprobs, const float *grad_entropy, float *logprobs, float *entropy,
                  float *statistics, void *grad_logits, size_t grad_stride, void *stream) {
  return with_real(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (int st = check("token loss", rows, vocab, row_stride, "logits")) return st;
    if (int st = check("token loss", rows, vocab, grad_stride, "grad_logits")) return st;
    if ((grad_logprobs || logprobs) && !tokens) return fail(TC_EINVAL, "token loss: no tokens");
    if (rows == 0) return TC_OK;
    if (!logits || !grad_logits) return fail(TC_EINVAL, "token loss: null pointer");
    if (off_grid(statistics, 8)) return fail(TC_EINVAL, "token loss: statistics are not on an 8-byte boundary");
    TokenArgs a{};
    a.logits = logits;
    a.stride = row_stride;
    a.rows = rows;
    a.vocab = unsigned(vocab);
    a.tokens = tokens;
    a.logprobs = logprobs;
    a.entropy = entropy;
    a.statistics = reinterpret_cast<float2 *>(statistics);
    a.grad_logprobs = grad_logprobs;
    a.grad_entropy = grad_entropy;
    a.grad_logits = grad_logits;
    a.grad_stride = grad_stride;
    const unsigned grid = unsigned(std::min<size_t>(rows, 1u << 30)), threads = threads_for(vocab, 16 / sizeof(typename T::S));
    if (entropy || grad_entropy) token_rows<T, true, GRADIENT><<<grid, threads, 0, as_stream(stream)>>>(a);
    else token_rows<T, false, GRADIENT><<<grid, threads, 0, as_stream(stream)>>>(a);
    return check_launch("token loss");
  });
}

}  // extern "C"
