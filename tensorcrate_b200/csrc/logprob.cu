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

// From here on a logit's weight is e = 2^a, a = x log2(e) - mark: one fused
// operation.  The mark is m log2(e) rounded, which shifts every a of a row by
// the same amount, known exactly, and is undone where sums are restated for
// another maximum and in what is taken from them.  That holds for |m| up to
// TAME, where the shift is below 2^-13; past it (a row masked by the type's
// lowest value, say) a = (x - m) log2(e), the difference first.  Weights below
// 2^-126 are zero.
constexpr float TAME = 1024.0f, LN2 = 0.6931471805599453f;
__device__ __forceinline__ bool tame(float m) { return fabsf(m) <= TAME; }

// The elements, none of them lower than -1e37 (f16: -65504): weightless there
// wherever m is tame, and finite, so that e a is 0.  NaNs stay.
template <class T> __device__ __forceinline__ Bits<T> lifted(Bits<T> r) {
  if constexpr (T::code == TC_F32) {
    auto up = [](uint32_t w) {
      float v;
      asm("max.NaN.f32 %0, %1, 0fFCF0BDC2;" : "=f"(v) : "f"(__uint_as_float(w)));  // -1e37
      return __float_as_uint(v);
    };
    return Bits<T>{make_uint4(up(r.w.x), up(r.w.y), up(r.w.z), up(r.w.w))};
  } else {
    auto up = [](uint32_t w) {
      uint32_t v;
      if constexpr (T::code == TC_BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(w), "r"(0xfcf0fcf0u));
      else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(v) : "r"(w), "r"(0xfbfffbffu));
      return v;
    };
    return Bits<T>{make_uint4(up(r.w.x), up(r.w.y), up(r.w.z), up(r.w.w))};
  }
}

// A thread's statistics while it walks: the maximum, and the sums of e and of
// e a, each in two halves.  The mark is that of an earlier maximum as long as
// the present one is within 8 of it (e is then below 2^12): few marks change,
// where among 32 lanes some maximum does all the time.
template <class T, bool ENT> struct Running {
  float m = -INFINITY, ref = -INFINITY, limit = -INFINITY, mark = 0.0f;
  bool wild = false;
  F2 s = 0, t = 0;
  __device__ __forceinline__ void begin(float at) {
    m = ref = at;
    wild = !tame(at) && at != -INFINITY;
    mark = at == -INFINITY || wild ? 0.0f : at * LOG2E;
    limit = at == -INFINITY || wild ? at : at + 8.0f;
  }
  __device__ __forceinline__ void lift(float to) {
    const Running old = *this;
    begin(to);
    if (old.ref == -INFINITY) return;
    float up = mark - old.mark;
    if (old.wild || wild) {  // from or to a maximum itself, of which a mark is short by its rounding
      const float rest = (old.wild ? 0.0f : fmaf(old.ref, LOG2E, -old.mark)) - (wild ? 0.0f : fmaf(to, LOG2E, -mark));
      up = fminf((to - old.ref) * LOG2E + rest, 1e20f);
    }
    const float f = exp2_of(-up);
    if (ENT) t = mul2(pair(f, f), fma2(pair(-up, -up), s, t));
    s = mul2(pair(f, f), s);
  }
  __device__ __forceinline__ void weigh(F2 a) {
    const float2 x = split(a);
    const F2 e = pair(exp2_of(x.x), exp2_of(x.y));
    s = add2(s, e);
    if (ENT) t = fma2(e, a, t);
  }
  // Elements that m is not below.
  template <int U> __device__ __forceinline__ void add(const Bits<T> (&r)[U]) {
    if (wild) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < int(Bits<T>::PAIRS); ++j) add_wild(r[u].pair_at(j));
      return;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Bits<T> b = ENT ? lifted(r[u]) : r[u];
#pragma unroll
      for (int j = 0; j < int(Bits<T>::PAIRS); ++j) weigh(fma2(b.pair_at(j), pair(LOG2E, LOG2E), pair(-mark, -mark)));
    }
  }
  __device__ __forceinline__ void add_wild(F2 v) {
    const float2 d = split(add2(v, pair(-base_of(ref), -base_of(ref))));
    const float2 e = make_float2(exp_of(d.x), exp_of(d.y));
    s = add2(s, pair(e.x, e.y));
    // 0 for an element of -inf, NaN for a NaN (e is one)
    if (ENT) t = fma2(pair(e.x, e.y), pair(fmaxf(d.x * LOG2E, -1e30f), fmaxf(d.y * LOG2E, -1e30f)), t);
  }
  __device__ __forceinline__ void add_one(float v) {
    if (wild || ref == -INFINITY) {
      add_wild(pair(v, -INFINITY));
      return;
    }
    const float a = fmaf(v, LOG2E, -mark), e = exp2_of(a);
    s = add2(s, pair(e, 0.0f));
    if (ENT) t = add2(t, pair(e * fmaxf(a, -1e30f), 0.0f));
  }
  // True where they raised the maximum.
  template <int U> __device__ __forceinline__ bool take(const Bits<T> (&r)[U]) {
    const float top = largest(r);
    const bool more = top > m;
    if (top > limit) lift(top);
    m = fmaxf(m, top);
    add(r);
    return more;
  }
  __device__ __forceinline__ bool take_one(float v) {
    const bool more = v > m;
    if (v > limit) lift(v);
    m = fmaxf(m, v);
    add_one(v);
    return more;
  }
  __device__ __forceinline__ Sums sums() const {
    const float2 a = split(s), b = split(t);
    const float off = wild || m == -INFINITY ? 0.0f : fmaf(m, LOG2E, -mark), f = exp2_of(-off), sum = a.x + a.y;
    return Sums{m, sum * f, (b.x + b.y - off * sum) * (f * LN2)};
  }
};

// A row's elements, or the part of them that one of `of` (a power of two)
// blocks has, as runs of 16 aligned bytes with the few single elements before
// and after them.
template <class T> struct Cut {
  using S = typename T::S;
  static constexpr unsigned V = 16 / sizeof(S);
  unsigned head, body, runs, after, tail;  // [0, head), runs from body, `tail` from after
  __device__ __forceinline__ Cut(const S *row, unsigned n, unsigned part = 0, unsigned of = 1) {
    const unsigned off = unsigned(reinterpret_cast<uintptr_t>(row) & 15) / unsigned(sizeof(S));
    head = min(n, (V - off) % V);
    const unsigned all = (n - head) / V, per = (all + of - 1) >> (31 - __clz(of)), from = min(all, part * per);
    body = head + from * V;
    runs = min(all - from, per);
    after = head + all * V;
    tail = part + 1 == of ? n - after : 0;
    if (part) head = 0;
  }
};

// one(index, value) for the single elements that thread t of `threads` takes,
// many(first run, bits) for its runs (`threads` apart), up to four at once, in
// ascending order.
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

// The sums of a row over the warps of the cluster's blocks (at most 64), the
// same in every thread: each warp's go to every block.  The slots of two rows
// in turn: a warp that is ahead stores a row's sums while another still reads
// the last row's.  Before the kernel's first row is joined, the blocks wait for
// one another's cluster_arrive at the kernel's start: another block's shared
// memory may be written only once that block runs.
struct Slots {
  Sums of[2][64];
};
template <bool ENT> __device__ __forceinline__ Sums row_join(Sums mine, Slots &slots, unsigned part, unsigned parts, unsigned turn,
                                                              bool first) {
  const unsigned lane = threadIdx.x & 31, warps = blockDim.x >> 5, n = parts * warps;
  Sums *all = slots.of[turn];
  mine = warp_join<ENT>(mine);
  if (parts == 1) {
    if (lane == 0) all[threadIdx.x >> 5] = mine;
    __syncthreads();
  } else {
    if (first) cluster_wait();
    if (lane < parts) {
      Sums *to = all + part * warps + (threadIdx.x >> 5);
      store_at(&to->m, lane, mine.m);
      store_at(&to->s, lane, mine.s);
      if (ENT) store_at(&to->t, lane, mine.t);
    }
    cluster_sync();
  }
  Sums v = lane < n ? all[lane] : Sums{};
  if (n > 32 && lane + 32 < n) join<ENT>(v, all[lane + 32]);
  return warp_join<ENT>(v);
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

constexpr int MAX_TOP = TC_MAX_TOP, GROUPS = 32;
static_assert(MAX_TOP <= GROUPS, "a bound needs a group for each of the top tokens");
template <int ROOM, int THREADS> struct TopRoom {
  static constexpr int room = ROOM;
  Key group[GROUPS], kept[ROOM], best[MAX_TOP], least;
  float value[GROUPS], bound;
  unsigned holders, count;
  unsigned short holder[THREADS];
};

// hit(i, rank): the rank of each of `n` values among them, the largest first
// and of equal ones the first; a warp compares a value with 32 at a time.
template <class V, class Hit>
__device__ __forceinline__ void rank_all(const V *value, unsigned n, unsigned warp, unsigned warps, Hit &&hit) {
  const unsigned lane = threadIdx.x & 31;
  for (unsigned i = warp; i < n; i += warps) {
    const V own = value[i];
    unsigned rank = 0;
    for (unsigned j = lane; j < (n + 31) / 32 * 32; j += 32)
      rank += __popc(__ballot_sync(0xffffffffu, j < n && (value[j] > own || (value[j] == own && j < i))));
    if (lane == 0) hit(i, rank);
  }
}
// The same of distinct keys, for ranks below k alone.
template <class Hit>
__device__ __forceinline__ void rank_first(const Key *key, unsigned n, unsigned k, unsigned t, unsigned threads, Hit &&hit) {
  if (n <= 64 && threads > 32) {
    rank_all(key, n, t >> 5, threads >> 5, [&](unsigned i, unsigned rank) {
      if (rank < k) hit(i, rank);
    });
    return;
  }
  for (unsigned i = t; i < n; i += threads) {  // most are soon known to be none of the first k
    const Key own = key[i];
    unsigned rank = 0;
    for (unsigned j = 0; j < n && rank < k; ++j) rank += key[j] > own;
    if (rank < k) hit(i, rank);
  }
}

// Where a thread's largest element was met: in the `runs` runs (each
// `threads` after the other) of which the first begins at element `at`, or,
// with runs = 0, at that element (~0: the thread has none).
struct Met {
  unsigned at, runs;
};

// The `k` largest keys of a row (or of a block's part of it: fewer may be
// there, 0 stands for none), in order, into room.best.  `m` is the thread's
// largest element, met at `met`; `clean` says that no NaN is among its
// elements.  The threads are a block's, or (WARP) a warp's.
//
// Each of 32 groups of threads has an element as large as its largest, so
// the k-th largest of those bounds the k-th element of the row from below; in
// rows without structure few elements more reach it, and only threads whose
// largest does (the holders) hold any.  Among equal values the index decides:
// the holders look up where their largest lies, and the k-th largest key of
// the groups, or of the holders where ties make those many, is the bound
// that elements are kept by.  The holders' elements are read again (from L2)
// and the kept ones ranked by counting.
template <class T, bool WARP, class Room>
__device__ __forceinline__ void top_of_row(const typename T::S *row, const Cut<T> &c, Met met, float m, bool clean,
                                           unsigned k, Room &room) {
  using S = typename T::S;
  constexpr unsigned V = Cut<T>::V;
  const unsigned t = WARP ? threadIdx.x & 31 : threadIdx.x, threads = WARP ? 32 : blockDim.x, lanes = threads / GROUPS;
  const unsigned warp = t >> 5, warps = threads >> 5;
  const auto load = from_row<T>(row, c);
  auto sync = [] {
    if (WARP) __syncwarp();
    else __syncthreads();
  };
  float top = m;
  for (unsigned o = 1; o < lanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (t % lanes == 0) room.value[t / lanes] = top;
  if (t == 0) room.holders = room.count = 0;
  sync();
  if (WARP) {  // a value a lane
    unsigned rank = 0;
#pragma unroll 8
    for (unsigned j = 0; j < 32; ++j) {
      const float v = __shfl_sync(0xffffffffu, m, j);
      rank += v > m || (v == m && j < t);
    }
    if (rank == k - 1) room.bound = m;
  } else {
    rank_all(room.value, GROUPS, warp, warps, [&](unsigned i, unsigned rank) {
      if (rank == k - 1) room.bound = room.value[i];
    });
  }
  sync();
  Key g = 0;
  if (m >= room.bound && met.at != ~0u) {
    room.holder[atomicAdd(&room.holders, 1u)] = (unsigned short)t;
    if (m != -INFINITY) {
      unsigned at = met.at;
      for (unsigned u = met.runs; u-- > 0;) {
        const unsigned i = (met.at - c.body) / V + u * threads;
        const Bits<T> r = load(i);
#pragma unroll
        for (int j = int(V) - 1; j >= 0; --j)
          if (r.at(j) == m) at = c.body + i * V + unsigned(j);
      }
      g = key_of(m, at);
    } else if (clean) {  // all are -inf, the first among them
      g = key_of(m, met.at);
    }
  }
  const Key own = g;
  for (unsigned o = 1; o < lanes; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
  if (t % lanes == 0) room.group[t / lanes] = g;
  sync();
  if (WARP) {
    unsigned rank = 0;
#pragma unroll 8
    for (unsigned j = 0; j < 32; ++j) rank += room.group[j] > g || (room.group[j] == g && j < t);
    if (rank == k - 1) room.least = g;
  } else {
    rank_all(room.group, GROUPS, warp, warps, [&](unsigned i, unsigned rank) {
      if (rank == k - 1) room.least = room.group[i];
    });
  }
  sync();
  const unsigned holders = room.holders;
  if (!WARP && holders > 2 * GROUPS) {
    // many equal values: the k-th largest of the holders' own keys
    if (own >= room.least && own) {
      const unsigned slot = atomicAdd(&room.count, 1u);
      if (slot < unsigned(Room::room)) room.kept[slot] = own;
    }
    __syncthreads();
    const unsigned n = room.count;
    __syncthreads();
    if (n >= k && n <= unsigned(Room::room))
      rank_first(room.kept, n, k, t, threads, [&](unsigned i, unsigned rank) {
        if (rank == k - 1) room.least = room.kept[i];
      });
    if (t == 0) room.count = 0;
    __syncthreads();
  }
  const Key least = room.least;
  const float bound = value_of(least);  // a NaN where any element may be kept
  const unsigned limit = ~uint32_t(least);  // of equal values, the last index to be kept
  auto keep = [&](unsigned at, float v) {
    if (v < bound) return;
    const Key key = key_of(v, at);
    if (key < least) return;
    const unsigned slot = atomicAdd(&room.count, 1u);
    if (slot < unsigned(Room::room)) room.kept[slot] = key;
  };
  auto keep_run = [&](unsigned i, const Bits<T> &r) {
    const Bits<T> one[1] = {r};
    const float top = largest(one);
    if (top < bound || (top == bound && c.body + i * V > limit)) return;
#pragma unroll
    for (unsigned j = 0; j < V; ++j) keep(c.body + i * V + j, r.at(j));
  };
  if (holders > threads / 8) {
    walk<T>(row, c, t, threads, load, [&](unsigned at, S e) { keep(at, T::load(e)); }, [&](unsigned i, const auto &r) {
      constexpr int U = sizeof(r) / sizeof(r[0]);
#pragma unroll
      for (int u = 0; u < U; ++u) keep_run(i + u * threads, r[u]);
    });
  } else {
    if (t < c.head) keep(t, T::load(row[t]));
    if (t < c.tail) keep(c.after + t, T::load(row[c.after + t]));
    // the holders' runs dealt out to all threads
    const unsigned all = holders * ((c.runs + threads - 1) / threads);
    for (unsigned x = t; x < all; x += threads) {
      const unsigned i = room.holder[x % holders] + x / holders * threads;
      if (i < c.runs) keep_run(i, load(i));
    }
  }
  sync();
  const unsigned count = room.count;
  if (count <= unsigned(Room::room)) {
    for (unsigned i = count + t; i < k; i += threads) room.best[i] = 0;
    rank_first(room.kept, count, k, t, threads, [&](unsigned i, unsigned rank) { room.best[rank] = room.kept[i]; });
    sync();
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
    if ((t & 31) == 0) room.group[warp] = best;
    sync();
    for (unsigned w = 0; w < warps; ++w) best = max(best, room.group[w]);
    sync();
    if (t == 0) room.best[n] = best;
    last = best;
  }
  sync();
}

// ---------------------------------------------------------------------------
// The gradient of one row, given its statistics.
// ---------------------------------------------------------------------------
struct Slope {
  float base, log_sum, entropy, u, v;  // u, v: the gradients of the logprob and of the entropy
  unsigned token;
  // With p = 2^(a - off), a = x log2(e) - mark, off what rounding the mark
  // shifted it by: the gradient is 2^a (k1 a + k2).
  bool wild;
  float mark, k1, k2;
};
template <bool ENT> __device__ __forceinline__ float slope_at(const Slope &g, float x, unsigned at) {
  const float a = (x - g.base) - g.log_sum, p = exp_of(a);
  // 1 - p without its cancellation, where p is near one
  float d = at == g.token ? -g.u * expm1f(a) : -g.u * p;
  if (ENT) d -= g.v * p * (fmaxf(a, -1e30f) + g.entropy);
  return d;
}
template <bool ENT, bool WILD> __device__ __forceinline__ F2 slope_of_pair(const Slope &g, F2 x) {
  if constexpr (!WILD) {
    const F2 a = fma2(x, pair(LOG2E, LOG2E), pair(-g.mark, -g.mark));
    const float2 y = split(a);
    const F2 p = pair(exp2_of(y.x), exp2_of(y.y));
    if (!ENT) return mul2(p, pair(g.k2, g.k2));
    return mul2(p, fma2(pair(fmaxf(y.x, -1e30f), fmaxf(y.y, -1e30f)), pair(g.k1, g.k1), pair(g.k2, g.k2)));
  }
  const F2 a = add2(add2(x, pair(-g.base, -g.base)), pair(-g.log_sum, -g.log_sum));
  const float2 y = split(mul2(a, pair(LOG2E, LOG2E)));
  const F2 p = pair(exp2_of(y.x), exp2_of(y.y));
  if (!ENT) return mul2(p, pair(-g.u, -g.u));
  // -p (u + v (a + H))
  const float2 z = split(a);
  const F2 c = add2(pair(fmaxf(z.x, -1e30f), fmaxf(z.y, -1e30f)), pair(g.entropy, g.entropy));
  return mul2(p, fma2(c, pair(-g.v, -g.v), pair(-g.u, -g.u)));
}
// The gradient at a run, but for the token's own term.
template <class T, bool ENT, bool WILD> __device__ __forceinline__ uint4 slope_run(const Slope &g, const Bits<T> &r) {
  using S = typename T::S;
  constexpr unsigned V = Cut<T>::V;
  F2 d[V / 2];
#pragma unroll
  for (unsigned j = 0; j < V / 2; ++j) d[j] = slope_of_pair<ENT, WILD>(g, r.pair_at(j));
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
  return out.w;
}
// The token's own element of the gradient: the thread that writes its run
// stores it after that run.
template <class T> struct Own {
  unsigned run = ~0u;  // the token's, where this thread has it
  typename T::S value;
  template <bool ENT>
  __device__ __forceinline__ void find(const typename T::S *row, const Cut<T> &c, const Slope &g, unsigned t, unsigned threads) {
    if (g.token < c.body || g.token - c.body >= c.runs * Cut<T>::V) return;
    const unsigned i = (g.token - c.body) / Cut<T>::V;
    if (i % threads != t) return;
    run = i;
    value = T::store(slope_at<ENT>(g, T::load(row[g.token]), g.token));
  }
  // After the runs from i, `threads` apart, U of them.
  __device__ __forceinline__ void after(unsigned i, unsigned span, typename T::S *to, unsigned token) const {
    if (run - i < span) to[token] = value;
  }
};
// A run of the gradient's row, whole where it lies on the grid as the logits do.
template <class T> __device__ __forceinline__ void put_run(typename T::S *to, uint4 w, bool whole) {
  using S = typename T::S;
  if (whole) {
    __stcs(reinterpret_cast<uint4 *>(to), w);
  } else {
    union {
      uint4 w;
      S e[Cut<T>::V];
    } u;
    u.w = w;
#pragma unroll
    for (unsigned j = 0; j < Cut<T>::V; ++j) to[j] = u.e[j];
  }
}
__device__ __forceinline__ bool same_grid(const void *a, const void *b) {
  return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}
template <bool ENT> __device__ __forceinline__ bool no_slope(const Slope &g) { return g.u == 0.0f && (!ENT || g.v == 0.0f); }
// Nothing flows back through this row, whatever its logits.
template <class T>
__device__ __forceinline__ void write_zeros(typename T::S *to, const Cut<T> &c, unsigned t, unsigned threads, bool whole) {
  using S = typename T::S;
  if (t < c.head) to[t] = S(0);
  for (unsigned i = t; i < c.runs; i += threads) put_run<T>(to + c.body + size_t(i) * Cut<T>::V, make_uint4(0, 0, 0, 0), whole);
  if (t < c.tail) to[c.after + t] = S(0);
}
template <class T, bool ENT>
__device__ __forceinline__ void write_slope(const typename T::S *row, typename T::S *to, const Cut<T> &c, const Slope &g,
                                            unsigned t, unsigned threads) {
  using S = typename T::S;
  constexpr unsigned V = Cut<T>::V;
  const bool whole = same_grid(row, to);
  if (no_slope<ENT>(g)) {
    write_zeros<T>(to, c, t, threads, whole);
    return;
  }
  Own<T> own;
  own.template find<ENT>(row, c, g, t, threads);
  auto write = [&](auto wild) {
    walk<T>(
        row, c, t, threads, from_row<T>(row, c), [&](unsigned at, S e) { to[at] = T::store(slope_at<ENT>(g, T::load(e), at)); },
        [&](unsigned i, const auto &r) {
          constexpr int U = sizeof(r) / sizeof(r[0]);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const unsigned at = c.body + (i + u * threads) * V;
            put_run<T>(to + at, slope_run<T, ENT, decltype(wild)::value>(g, r[u]), whole);
          }
          own.after(i, U * threads, to, g.token);
        });
  };
  if (g.wild) write(std::true_type{});
  else write(std::false_type{});
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
  g.wild = !tame(g.base);
  g.mark = fmaf(g.base, LOG2E, g.log_sum * LOG2E);
  const float off = fmaf(g.base, LOG2E, -g.mark) + g.log_sum * LOG2E, f = exp2_of(-off);
  g.k1 = -g.v * LN2 * f;
  g.k2 = -(g.u + g.v * (g.entropy - off * LN2)) * f;
  return g;
}

// What a row's sums say.
struct Told {
  float2 st;
  float entropy;
};
template <bool ENT> __device__ __forceinline__ Told told_by(const Sums &all) {
  const bool empty = all.m == -INFINITY && all.s == 0.0f;
  Told o;
  o.st = make_float2(all.m, empty ? 0.0f : logf(all.s));
  o.entropy = !ENT || empty ? 0.0f : o.st.y - all.t / all.s;
  return o;
}
// `at_token` is the token's logit, read before any gradient is written.
template <bool ENT>
__device__ __forceinline__ void write_told(const TokenArgs &a, size_t r, const Told &o, unsigned token, float at_token) {
  if (a.logprobs) a.logprobs[r] = token == ~0u ? 0.0f : (at_token - base_of(o.st.x)) - o.st.y;
  if (a.statistics) a.statistics[r] = o.st;
  if (ENT && a.entropy) a.entropy[r] = o.entropy;
}
__device__ __forceinline__ void write_top(const TokenArgs &a, size_t r, const Told &o, unsigned i, Key k) {
  a.top_tokens[r * a.top + i] = ~uint32_t(k);
  a.top_logprobs[r * a.top + i] = (value_of(k) - base_of(o.st.x)) - o.st.y;
}
template <class T> __device__ __forceinline__ float logit_of(const typename T::S *row, unsigned token, unsigned vocab) {
  return token < vocab ? T::load(row[token]) : __int_as_float(0x7fc00000);
}

enum Extra { NOTHING = 0, TOP = 1, GRADIENT = 2 };

// Small vocabularies: a warp holds a row, U runs a lane.  The row is read
// once, whatever is asked for but the top tokens' second look.  Bound by
// issue: 67108x1000 bf16 with entropy in 34 us (floor 21), with 5 top tokens
// in 131; the loss of 65536x1024 with entropy in 64 (floor 42).  Blocks of a
// row each take 118, 361 and 235; at 2048 tokens, the most that a warp holds,
// 32768 rows take 34 us for 73, and 73 for 139 with the loss.
template <class T, bool ENT, int EXTRA, int U> __global__ void __launch_bounds__(256) token_small(const TokenArgs a) {
  using S = typename T::S;
  constexpr unsigned V = Cut<T>::V;
  constexpr uint32_t LOW = T::code == TC_F32 ? 0xff800000u : T::code == TC_BF16 ? 0xff80ff80u : 0xfc00fc00u;  // -inf
  const unsigned lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  __shared__ std::conditional_t<EXTRA == TOP, TopRoom<256, 32>, int> rooms[EXTRA == TOP ? 8 : 1];
  for (size_t r = size_t(blockIdx.x) * warps + (threadIdx.x >> 5); r < a.rows; r += size_t(gridDim.x) * warps) {
    const S *row = static_cast<const S *>(a.logits) + r * a.stride;
    const Cut<T> c(row, a.vocab);
    const unsigned token = a.tokens ? a.tokens[r] : ~0u;
    const float at_token = logit_of<T>(row, token, a.vocab);
    Bits<T> bits[U];
    const auto load = from_row<T>(row, c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      bits[u].w = make_uint4(LOW, LOW, LOW, LOW);
      if (lane + 32 * u < c.runs) bits[u] = load(lane + 32 * u);
    }
    // the single elements: those before the runs to the first lanes, those
    // after them from lane 8 on
    const unsigned single = lane < c.head ? lane : lane >= 8 && lane - 8 < c.tail ? c.after + lane - 8 : ~0u;
    const float extra = single != ~0u ? T::load(row[single]) : -INFINITY;
    // a lane of nothing but NaNs has no largest: -inf, as one without elements
    const float in_runs = fmaxf(largest(bits), -INFINITY), m = fmaxf(in_runs, extra);
    float all_m = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) all_m = fmaxf(all_m, __shfl_xor_sync(0xffffffffu, all_m, o));
    Running<T, ENT> run;
    run.begin(all_m);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (32 * u < int(c.runs)) {
        const Bits<T> one[1] = {bits[u]};
        run.add(one);
      }
    run.add_one(extra);
    Sums sums = run.sums();
    const bool clean = !isnan(sums.s);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      sums.s += __shfl_xor_sync(0xffffffffu, sums.s, o);
      if (ENT) sums.t += __shfl_xor_sync(0xffffffffu, sums.t, o);
    }
    const Told o = told_by<ENT>(sums);
    if (lane == 0) write_told<ENT>(a, r, o, token, at_token);
    if constexpr (EXTRA == TOP) {
      auto &room = rooms[threadIdx.x >> 5];
      const unsigned mine = lane < c.runs ? (c.runs - lane + 31) / 32 : 0;
      Met met{c.body + lane * V, mine};
      if (single != ~0u && (mine == 0 || (lane < c.head ? extra >= in_runs : extra > in_runs))) met = Met{single, 0};
      else if (mine == 0) met = Met{~0u, 0};
      top_of_row<T, true>(row, c, met, m, clean, a.top, room);
      if (lane < a.top) write_top(a, r, o, lane, room.best[lane]);
      __syncwarp();
    }
    if constexpr (EXTRA == GRADIENT) {
      const Slope g = slope_of(a, r, o.st, o.entropy);
      S *to = static_cast<S *>(a.grad_logits) + r * a.grad_stride;
      const bool whole = same_grid(row, to), none = no_slope<ENT>(g);
      auto write = [&](auto wild) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const unsigned i = lane + 32 * u, at = c.body + i * V;
          if (i < c.runs)
            put_run<T>(to + at, none ? make_uint4(0, 0, 0, 0) : slope_run<T, ENT, decltype(wild)::value>(g, bits[u]), whole);
        }
      };
      Own<T> own;
      if (!none) own.template find<ENT>(row, c, g, lane, 32);
      if (g.wild) write(std::true_type{});
      else write(std::false_type{});
      if (own.run != ~0u) to[g.token] = own.value;
      if (single != ~0u) to[single] = none ? S(0) : T::store(slope_at<ENT>(g, extra, single));
    }
  }
}

// A thread's runs of the rows that its block takes, copied ahead of their use
// into slots of its own (so only it waits for them): `groups` groups of four,
// as many as a row has.
template <class T> struct Ahead {
  using S = typename T::S;
  const TokenArgs &a;
  uint4 *const slots;
  const unsigned t, threads, groups;
  size_t row;            // of the next group
  unsigned group, runs;  // of the row; the row's
  const uint4 *from;
  __device__ __forceinline__ Ahead(const TokenArgs &a, void *slots, unsigned groups)
      : a(a), slots(static_cast<uint4 *>(slots) + threadIdx.x), t(threadIdx.x), threads(blockDim.x), groups(groups),
        row(blockIdx.x), group(0) {
    place();
  }
  __device__ __forceinline__ void place() {
    if (row >= a.rows) return;
    const S *at = static_cast<const S *>(a.logits) + row * a.stride;
    const Cut<T> c(at, a.vocab);
    from = reinterpret_cast<const uint4 *>(at + c.body) + t;
    runs = c.runs;
  }
  __device__ __forceinline__ uint4 *slot(unsigned g, int u) const { return slots + (g * 4 + u) * threads; }
  // Begin the next group's copies; the group of the row before it is no
  // longer needed.
  __device__ __forceinline__ void fetch() {
    if (row < a.rows) {
      const unsigned i = group * 4 * threads;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (t + i + u * threads < runs) copy_async(uint32_t(__cvta_generic_to_shared(slot(group, u))), from + i + u * threads);
      if (++group == groups) {
        group = 0;
        row += gridDim.x;
        place();
      }
    }
    copy_commit();
  }
  // A thread's part of a group that has arrived: f(first run, bits[1 or 4])
  // for the runs that it has.
  template <class F> __device__ __forceinline__ void each(unsigned g, const Cut<T> &c, F &&f) const {
    const unsigned i = t + g * 4 * threads;
    if (i + 3 * threads < c.runs) {
      Bits<T> r[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) r[u].w = *slot(g, u);
      f(i, r);
    } else {
      for (int u = 0; u < 4; ++u)
        if (i + u * threads < c.runs) {
          Bits<T> r[1];
          r[0].w = *slot(g, u);
          f(i + u * threads, r);
        }
    }
  }
};

// Larger ones: a block a row, or a cluster's blocks, each a part of it.  Four
// 16-byte loads a thread and 1536 threads an SM cover HBM's latency (the same
// rows copied ahead through shared memory took 58 us for 56).  8192x32768 bf16
// with entropy in 93 us, 5.8 TB/s; 2048x50257 in 44 us, where 2.3 rounds of
// blocks begin and end together.  With top tokens the steps between the row's
// barriers, not HBM, take the time: 67 us with 8 of them, some rows masked to
// nothing.  (Their code spills with the registers of six blocks an SM: 77 us;
// five are kept.)
template <class T, bool ENT, int EXTRA> __global__ void __launch_bounds__(256, EXTRA == TOP ? 5 : 6) token_rows(const TokenArgs a) {
  using S = typename T::S;
  constexpr unsigned V = Cut<T>::V;
  __shared__ Slots joint;
  const unsigned t = threadIdx.x, threads = blockDim.x, part = cluster_part(), parts = cluster_parts();
  const size_t first = blockIdx.x / parts, step = gridDim.x / parts;
  unsigned turn = 0;
  if (parts > 1) cluster_arrive();  // waited for in the first row's join (every cluster has a row)
  for (size_t r = first; r < a.rows; r += step, turn ^= 1) {
    const S *row = static_cast<const S *>(a.logits) + r * a.stride;
    const Cut<T> c(row, a.vocab, part, parts);
    const unsigned token = a.tokens ? a.tokens[r] : ~0u;
    const float at_token = part == 0 && t == 0 ? logit_of<T>(row, token, a.vocab) : 0.0f;
    Running<T, ENT> run;
    // the thread's first element, while all are -inf; none: ~0
    Met met{t < c.head ? t : t < c.runs ? c.body + t * V : t < c.tail ? c.after + t : ~0u, 0};
    walk<T>(
        row, c, t, threads, from_row<T>(row, c),
        [&](unsigned i, S e) {
          if (run.take_one(T::load(e))) met = Met{i, 0};
        },
        [&](unsigned i, const auto &bits) {
          if (run.take(bits)) met = Met{c.body + i * V, unsigned(sizeof(bits) / sizeof(bits[0]))};
        });
    const Sums sums = run.sums();
    const Sums all = row_join<ENT>(sums, joint, part, parts, turn, r == first);
    const Told o = told_by<ENT>(all);
    if (part == 0 && t == 0) write_told<ENT>(a, r, o, token, at_token);
    if constexpr (EXTRA == TOP) {
      __shared__ TopRoom<1024, 256> top;
      __shared__ Key parts_best[8 * MAX_TOP];
      top_of_row<T, false>(row, c, met, sums.m, !isnan(sums.s), a.top, top);
      if (parts == 1) {
        if (t < a.top) write_top(a, r, o, t, top.best[t]);
      } else {
        // each block's top tokens to the first, which has the row's among them
        if (t < a.top) store_at(&parts_best[part * a.top + t], 0, top.best[t]);
        cluster_sync();
        if (part == 0) {
          const unsigned n = parts * a.top;
          for (unsigned i = t; i < n; i += threads) {
            const Key own = parts_best[i];
            unsigned rank = 0;
            for (unsigned j = 0; j < n; ++j) rank += parts_best[j] > own;
            if (rank < a.top && own) write_top(a, r, o, rank, own);
          }
        }
      }
      __syncthreads();
    }
  }
}

// The loss of rows that a block's shared memory holds: a row stays in its
// slots until its gradient is written from there, and the next one follows it
// group by group.  Against rows read twice (token_loss_twice), without entropy:
// f32 87 us for 98 at 16384x4096, 94 for 97 at 4096x16384; bf16 213 for 239 at
// 53687x2500, 107 for 103 at 16384x8192, 104 for 103 at 4096x32768.
template <class T, bool ENT> __global__ void __launch_bounds__(256, 3) token_loss_held(const TokenArgs a, unsigned groups) {
  using S = typename T::S;
  constexpr unsigned V = Cut<T>::V;
  extern __shared__ __align__(16) unsigned char slots[];
  __shared__ Slots joint;
  const unsigned t = threadIdx.x, threads = blockDim.x;
  Ahead<T> ring(a, slots, groups);
  for (unsigned g = 0; g < groups; ++g) ring.fetch();
  unsigned turn = 0;
  for (size_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1) {
    const S *row = static_cast<const S *>(a.logits) + r * a.stride;
    const Cut<T> c(row, a.vocab);
    const unsigned token = a.tokens ? a.tokens[r] : ~0u;
    const float at_token = t == 0 ? logit_of<T>(row, token, a.vocab) : 0.0f;
    Running<T, ENT> run;
    copy_wait<0>();
    if (t < c.head) run.take_one(T::load(row[t]));
    for (unsigned g = 0; g < groups; ++g) ring.each(g, c, [&](unsigned, const auto &bits) { run.take(bits); });
    if (t < c.tail) run.take_one(T::load(row[c.after + t]));
    const Told o = told_by<ENT>(row_join<ENT>(run.sums(), joint, 0, 1, turn, false));
    if (t == 0) write_told<ENT>(a, r, o, token, at_token);
    const Slope s = slope_of(a, r, o.st, o.entropy);
    S *to = static_cast<S *>(a.grad_logits) + r * a.grad_stride;
    const bool whole = same_grid(row, to), none = no_slope<ENT>(s);
    if (none) {
      write_zeros<T>(to, c, t, threads, whole);
    } else {
      if (t < c.head) to[t] = T::store(slope_at<ENT>(s, T::load(row[t]), t));
      if (t < c.tail) to[c.after + t] = T::store(slope_at<ENT>(s, T::load(row[c.after + t]), c.after + t));
    }
    Own<T> own;
    if (!none) own.template find<ENT>(row, c, s, t, threads);
    auto write = [&](auto wild) {
      for (unsigned g = 0; g < groups; ++g) {
        if (!none)
          ring.each(g, c, [&](unsigned i, const auto &bits) {
            constexpr int U = sizeof(bits) / sizeof(bits[0]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const unsigned at = c.body + (i + u * threads) * V;
              put_run<T>(to + at, slope_run<T, ENT, decltype(wild)::value>(s, bits[u]), whole);
            }
            own.after(i, U * threads, to, s.token);
          });
        ring.fetch();
      }
    };
    if (s.wild) write(std::true_type{});
    else write(std::false_type{});
  }
}

// Larger rows, and few: the blocks of a cluster share a row, and the second
// pass reads it from L2, which the parts of all resident blocks leave room in
// (2.1 GB of HBM traffic at 4096x131072 bf16, where blocks of whole rows made
// it 3.1).  421 us, 5.1 TB/s: the two passes' exponentials keep the special
// function unit 60% busy between the row's barriers.
template <class T, bool ENT> __global__ void __launch_bounds__(256, 4) token_loss_twice(const TokenArgs a) {
  using S = typename T::S;
  __shared__ Slots joint;
  const unsigned t = threadIdx.x, threads = blockDim.x, part = cluster_part(), parts = cluster_parts();
  const size_t first = blockIdx.x / parts, step = gridDim.x / parts;
  unsigned turn = 0;
  if (parts > 1) cluster_arrive();  // waited for in the first row's join (every cluster has a row)
  for (size_t r = first; r < a.rows; r += step, turn ^= 1) {
    const S *row = static_cast<const S *>(a.logits) + r * a.stride;
    const Cut<T> c(row, a.vocab, part, parts);
    const unsigned token = a.tokens ? a.tokens[r] : ~0u;
    const float at_token = part == 0 && t == 0 ? logit_of<T>(row, token, a.vocab) : 0.0f;
    Running<T, ENT> run;
    walk<T>(
        row, c, t, threads, from_row<T>(row, c), [&](unsigned, S e) { run.take_one(T::load(e)); },
        [&](unsigned, const auto &bits) { run.take(bits); });
    const Told o = told_by<ENT>(row_join<ENT>(run.sums(), joint, part, parts, turn, r == first));
    if (part == 0 && t == 0) write_told<ENT>(a, r, o, token, at_token);
    write_slope<T, ENT>(row, static_cast<S *>(a.grad_logits) + r * a.grad_stride, c, slope_of(a, r, o.st, o.entropy), t, threads);
  }
}

// The gradient alone, from the statistics that the forward call left, by
// blocks or (`apart`) by warps of a row each.  Bound by HBM: with entropy
// 4096x32768 f32 in 168 us, 6.4 TB/s; bf16 8192x32768 in 169, 6.3 TB/s, and
// 5341x50257 in 177, 6.1.
template <class T, bool ENT> __global__ void __launch_bounds__(512) token_slope(const TokenArgs a, bool apart) {
  using S = typename T::S;
  const unsigned threads = apart ? 32 : blockDim.x, each = blockDim.x / threads;
  const unsigned t = apart ? threadIdx.x & 31 : threadIdx.x;
  for (size_t r = size_t(blockIdx.x) * each + (apart ? threadIdx.x >> 5 : 0); r < a.rows; r += size_t(gridDim.x) * each) {
    const S *row = static_cast<const S *>(a.logits) + r * a.stride;
    const Cut<T> c(row, a.vocab);
    write_slope<T, ENT>(row, static_cast<S *>(a.grad_logits) + r * a.grad_stride, c,
                        slope_of(a, r, a.kept_statistics[r], ENT ? a.kept_entropy[r] : 0.0f), t, threads);
  }
}

// -scale * the sum of the logprobs, by one block.
template <class T> __global__ void __launch_bounds__(1024) loss_value(const float *logprobs, size_t rows, float scale, typename T::S *out) {
  __shared__ float room[32];
  float sum = 0.0f;
  for (size_t r = threadIdx.x; r < rows; r += blockDim.x) sum += logprobs[r];
  sum = block_sum(sum, room);
  if (threadIdx.x == 0) *out = T::store(-scale * sum);
}
template <class T> __global__ void __launch_bounds__(256) loss_seed(const typename T::S *adjoint, size_t rows, float scale, float *grad) {
  const float g = -scale * T::load(*adjoint);
  for (size_t r = size_t(blockIdx.x) * blockDim.x + threadIdx.x; r < rows; r += size_t(gridDim.x) * blockDim.x) grad[r] = g;
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

// Blocks of `kernel` that the GPU holds at once.
template <class K> size_t resident(K kernel, unsigned threads, size_t shared) {
  int n = 0;
  cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, int(threads), shared);
  return size_t(std::max(1, n)) * size_t(sm_count());
}

// In how many parts to cut each of `rows` rows of `runs` runs: as many as
// leave none of `slots` blocks idle and each thread two runs.  (Cutting
// further, to even out the blocks' last rows, costs more in joins.)
unsigned parts_for(size_t rows, size_t runs, unsigned threads, size_t slots) {
  unsigned parts = 1;
  while (parts < 8 && rows * parts * 2 <= slots && runs / (parts * 2) >= 2 * threads) parts *= 2;
  return parts;
}

// The most runs of a part whose row is read twice: 100 KB a block, of which
// four blocks on each of 148 SMs hold 60 MB.  In one, two and four parts, 2^28
// bf16 logits: 218, 239, 364 us at 50257 tokens (6282 runs); 218, 224, 333 at
// 53248 (6656); 218, 230, 318 at 57344; 231, 209, 265 at 65536 (8192); 245, 215,
// 242 at 98304; 256, 241, 230 at 131072.  So between 6400 and some 7500 runs two
// parts lose up to 5%.
constexpr size_t PART_RUNS = 6400;
// A warp a row up to 8 runs a lane; 2 or 4 where those do.
template <class T, bool ENT, int EXTRA> int small(const char *what, const TokenArgs &a, cudaStream_t stream) {
  const unsigned grid = unsigned(std::min<size_t>((a.rows + 7) / 8, size_t(sm_count()) * 64));
  if (a.vocab <= 64 * Cut<T>::V) token_small<T, ENT, EXTRA, 2><<<grid, 256, 0, stream>>>(a);
  else if (a.vocab <= 128 * Cut<T>::V) token_small<T, ENT, EXTRA, 4><<<grid, 256, 0, stream>>>(a);
  else token_small<T, ENT, EXTRA, 8><<<grid, 256, 0, stream>>>(a);
  return check_launch(what);
}
template <class T> bool is_small(const TokenArgs &a) { return a.vocab <= 256 * Cut<T>::V; }

template <class T, bool ENT, bool WITH_TOP> int forward(const TokenArgs &a, cudaStream_t stream) {
  constexpr int EXTRA = WITH_TOP ? TOP : NOTHING;
  if (is_small<T>(a)) return small<T, ENT, EXTRA>("token logprobs", a, stream);
  auto kernel = token_rows<T, ENT, EXTRA>;
  const size_t runs = a.vocab / Cut<T>::V;
  // Blocks of 128 threads have less to join a row, those of 256 more loads
  // ahead: 90 us for 107 at 16384x16384 bf16, 91 for 93 at 8192x32768, 106 for 92
  // at 2048x131072; f32 84 for 95 at 16384x8192 (2048 runs, as 16384 of 16
  // bits), 87 for 86 at 8192x16384.  The top tokens' steps wait for one another,
  // so many rows take smaller blocks, more of them: 8 of 2048x16384 bf16 in 31 us
  // for 34 (but 64 for 61 at 50257 and 137 for 111 at 131072); up to a row an SM
  // the larger ones, 14 for 22 us at 148x16384.
  const unsigned threads = runs >= 2048 && (!WITH_TOP || a.rows <= size_t(sm_count())) ? 256 : 128;
  const size_t slots = resident(kernel, threads, 0);
  const unsigned parts = parts_for(a.rows, runs, threads, slots);
  return launch("token logprobs", kernel, std::min<size_t>(a.rows, (1u << 30) / parts), parts, threads, 0, stream, a);
}

template <class T, bool ENT> int loss(const TokenArgs &a, cudaStream_t stream) {
  if (is_small<T>(a)) return small<T, ENT, GRADIENT>("token loss", a, stream);
  const size_t runs = a.vocab / Cut<T>::V;
  // 128 threads for 256: bf16 206 us for 282 at 32768x8192, 193 for 222 at
  // 16384x16384 (2048 runs), 236 for 206 at 8192x32768; f32 189 for 192 at
  // 16384x8192 (2048), 230 for 174 at 8192x16384.
  const unsigned threads = runs >= 2048 ? 256 : 128;
  // Sixteen runs a thread leave three blocks on an SM; with fewer rows than
  // SMs each row is better shared.
  if (runs <= 16 * size_t(threads) && a.rows > size_t(sm_count())) {
    auto kernel = token_loss_held<T, ENT>;
    const size_t groups = (runs + 4 * threads - 1) / (4 * threads), shared = groups * 4 * 16 * threads;
    static std::atomic<uint64_t> allowed{0};
    if (int st = allow_shared("token loss", reinterpret_cast<const void *>(kernel), 16 * 16 * 256, allowed)) return st;
    const unsigned grid = unsigned(std::min<size_t>(a.rows, resident(kernel, threads, shared)));
    kernel<<<grid, threads, shared, stream>>>(a, unsigned(groups));
    return check_launch("token loss");
  }
  auto kernel = token_loss_twice<T, ENT>;
  unsigned parts = parts_for(a.rows, runs, threads, resident(kernel, threads, 0));
  while (parts < 8 && runs > PART_RUNS * parts) parts *= 2;
  return launch("token loss", kernel, std::min<size_t>(a.rows, (1u << 30) / parts), parts, threads, 0, stream, a);
}

template <class T, bool ENT> int backward(const TokenArgs &a, cudaStream_t stream) {
  const bool apart = is_small<T>(a);
  const size_t runs = a.vocab / Cut<T>::V;
  // 128, 256 and 512 threads, 2^28 bf16 logits: 184, 226, 392 us at 8192 tokens
  // (1024 runs), 167, 183, 228 at 16384 (2048), 173, 169, 185 at 32768, 177, 172,
  // 170 at 65536 (8192).
  const unsigned threads = apart ? 256 : runs >= 8192 ? 512 : runs >= 2048 ? 256 : 128;
  const size_t blocks = apart ? (a.rows + 7) / 8 : a.rows;
  token_slope<T, ENT><<<unsigned(std::min<size_t>(blocks, 1u << 30)), threads, 0, stream>>>(a, apart);
  return check_launch("token logprobs backward");
}

}  // namespace

int token_loss_value(int dtype, const float *logprobs, size_t rows, double scale, void *out, cudaStream_t stream) {
  return with_real(dtype, [&](auto t) -> int {
    using T = decltype(t);
    loss_value<T><<<1, 1024, 0, stream>>>(logprobs, rows, float(scale), static_cast<typename T::S *>(out));
    return check_launch("token loss");
  });
}
int token_loss_seed(int dtype, const void *adjoint, size_t rows, double scale, float *grad, cudaStream_t stream) {
  if (rows == 0) return TC_OK;
  return with_real(dtype, [&](auto t) -> int {
    using T = decltype(t);
    loss_seed<T><<<grid_for(rows, 256), 256, 0, stream>>>(static_cast<const typename T::S *>(adjoint), rows, float(scale), grad);
    return check_launch("token loss");
  });
}
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
    cudaStream_t on = as_stream(stream);
    return entropy ? (top ? forward<T, true, true>(a, on) : forward<T, true, false>(a, on))
                   : (top ? forward<T, false, true>(a, on) : forward<T, false, false>(a, on));
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
    return grad_entropy ? backward<T, true>(a, as_stream(stream)) : backward<T, false>(a, as_stream(stream));
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
    return entropy || grad_entropy ? loss<T, true>(a, as_stream(stream)) : loss<T, false>(a, as_stream(stream));
  });
}

}  // extern "C"
