// Log probabilities of given tokens with entropy and top alternatives, and
// the gradient of the logits.
//
// With c = log2(e) / temperature, m = max x, d_v = x_v - m:
//   S = sum 2^(c d_v), U = sum d_v 2^(c d_v)
//   log p_v = d_v / temperature - ln S,  entropy = ln S - U / (S temperature)
//   dx_v = (1/temperature) (sum of the gradients that name v - p_v (G + ge (log p_v + entropy))),
//   G the sum of all gradients of the row's log probabilities, ge the entropy's.
//
// Bound: memory, the logits read once (and, for the gradient, read once more
// and written once).  The forward keeps a running maximum per thread and
// rescales S and U where a batch of values exceeds it; each value costs one
// hardware exp2 and about four other instructions (sums two at a time), below
// the memory time for 16-bit logits too.
//
// Top alternatives: each thread keeps its largest value, the batch of 4 vectors
// that held it (in shared memory) and the largest value outside that batch.  A
// value that k of the threads' largest reach bounds the k-th best of the row
// from below (from the maxima of 32 groups of threads, then by bisection, a vote
// per step), and only threads whose largest reaches it can hold alternatives:
// most of them in the kept batch; the values of those whose second reaches it
// too are read again (from L2; reading all of them again took 78 us in place of
// 65 for 20 alternatives of 4096 rows of 32000 bfloat16).  The few values that reach the
// bound are collected, and one warp sorts them.  Where equal values make more than
// fit, the whole row is read again into a list per warp.
// A key is the value's monotone 32-bit image with the complement of its index
// below it, so the order is by value and, for equal values, by the lower index.
//
// Split: a CTA of 128 or 256 threads per row, a cluster of CTAs per row where
// there are few rows (the parts meet in distributed shared memory), a warp per
// row where the rows are short.
//
// Measured on one B200 (plain copy 6.53 TB/s): 16384 rows of 32000 bfloat16
// logits take 159-172 us forward (6.1-6.6 TB/s) and 323-333 for the gradient (6.3-6.5);
// 2047 rows of 50021 take 41 us, with 5 alternatives 48, with 20 52: the
// search adds about 3 us to each row's own time, which other rows' passes
// only partly cover.  24 rows of 131072 float32 logits with 20 alternatives, on
// eight CTAs each, take 9.9 us.
#include <type_traits>

#include "lm_types.cuh"

namespace hs {
namespace {

constexpr int kShortRows = 8;  // rows of a CTA where each warp takes one
template <int W> constexpr int threads_of() { return 32 * (W == 1 ? kShortRows : W); }
constexpr int kMaxCluster = 8;
constexpr float kFloor = -150.f;  // 2^-150 is 0 in float32: a smaller exponent changes nothing

HS_DEV float max_nan(float a, float b) {  // the maximum, NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
HS_DEV float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kNegInf = -__builtin_huge_valf();

// Running (maximum, S, U) of a set of values; S and U are relative to m.
// Differences are held to `floor` = -150 / c, where 2^(c d) is 0: a masked -inf
// adds 0 to both sums, and a NaN stays one.
struct Stat {
  float m, s, u;
};
struct Scale {
  float c, floor;
};
HS_DEV float rel(float m) { return m == kNegInf ? 0.f : m; }  // nothing but -inf so far: every term is 0
// Moves (s, u) from its reference to the larger reference `to`.
HS_DEV void rescale(Stat &a, float to, Scale k) {
  const bool none = a.m == kNegInf;
  const float d = none ? 0.f : max_nan(a.m - to, k.floor);
  const float f = none ? 0.f : ex2(d * k.c);  // (a NaN s stays NaN)
  a.u = (a.u + d * a.s) * f;
  a.s *= f;
  a.m = to;
}
HS_DEV void merge(Stat &a, Stat b, Scale k) {
  const float m = fmaxf(a.m, b.m);
  if (a.m != m) rescale(a, m, k);
  if (b.m != m) rescale(b, m, k);
  a.s += b.s;
  a.u += b.u;
}
// Over groups of n lanes: the maximum first, so that each lane moves its sums once.
HS_DEV Stat reduce(Stat a, int n, Scale k) {
  float m = a.m;
  for (int o = n / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (a.m != m) rescale(a, m, k);
  for (int o = n / 2; o; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
  }
  return a;
}

// ------------------------------------------------------------------ keys
using Key = unsigned long long;  // 0: none
HS_DEV unsigned order_bits(float v) {
  const unsigned b = __float_as_uint(v + 0.0f);  // -0 counts as +0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
HS_DEV float value_of(Key k) {
  const unsigned b = (unsigned)(k >> 32);
  return __uint_as_float((b & 0x80000000u) ? b ^ 0x80000000u : ~b);
}
HS_DEV int index_of(Key k) { return (int)(0xffffffffu - (unsigned)k); }
HS_DEV Key make_key(float v, int i) { return ((Key)order_bits(v) << 32) | (0xffffffffu - (unsigned)i); }

HS_DEV Key order_pair(Key k, int o, bool keep_max) {
  const Key other = __shfl_xor_sync(0xffffffffu, k, o);
  return ((k > other) == keep_max) ? k : other;
}
// The warp's 32 keys in descending order of lanes (bitonic network).  A
// function of its own, as its code is long and used in several places.
__device__ __noinline__ Key sort_desc(Key k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o; o >>= 1) k = order_pair(k, o, ((lane & o) == 0) == ((lane & size) == 0));
  return k;
}
// The 32 largest of two descending lists, descending.
__device__ __noinline__ Key merge_desc(Key a, Key b, int lane) {
  const Key r = __shfl_sync(0xffffffffu, b, 31 - lane);
  Key k = a > r ? a : r;  // bitonic
#pragma unroll
  for (int o = 16; o; o >>= 1) k = order_pair(k, o, (lane & o) == 0);
  return k;
}

// ------------------------------------------------------------------ a row
// The row as [head scalars | 16-byte vectors | tail scalars]; CTA `rank` of
// `C` takes a contiguous share of the vectors, the first the head, the last
// the tail.  Thread j of n holds head scalar j, vectors lo+j, lo+j+n, .. and
// tail scalar j, in ascending order of index.
template <typename T> struct Row {
  static constexpr int E = 16 / (int)sizeof(T);
  const T *x;
  int head, lo, hi, tail0, ntail;
  HS_DEV Row(const T *row, int64_t V, int rank, int C) : x(row) {
    const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    const int h = off ? min((int64_t)(E - off), V) : 0;
    const int nv = (int)((V - h) / E);
    head = rank == 0 ? h : 0;
    base = h;
    lo = (int)((int64_t)nv * rank / C);
    hi = (int)((int64_t)nv * (rank + 1) / C);
    tail0 = h + nv * E;
    ntail = rank == C - 1 ? (int)(V - tail0) : 0;
  }
  int base;  // index of vector 0's first value
  HS_DEV const uint4 *vec(int i) const { return reinterpret_cast<const uint4 *>(x + base) + i; }
  HS_DEV int index(int i, int e) const { return base + i * E + e; }
};

template <typename T> HS_DEV void unpack_vec(const uint4 &c, float *v) {
  constexpr int P = PerWord<T>::value;
  unpack_word<T>(c.x, v);
  unpack_word<T>(c.y, v + P);
  unpack_word<T>(c.z, v + 2 * P);
  unpack_word<T>(c.w, v + 3 * P);
}

struct FwdArgs {
  const void *x;
  int64_t ld;
  const void *tok;
  int token64;
  int64_t ignore;
  Scale k;      // c = log2(e) / temperature
  float inv_t;  // 1 / temperature
  int top;
  float *lp, *ent, *top_lp;
  int64_t *top_id;
  float *stats;
  int64_t N, V;
  int cluster;
  int *status;
};

HS_DEV int64_t token_at(const void *tok, int token64, int64_t n) {
  return token64 ? static_cast<const int64_t *>(tok)[n] : (int64_t)static_cast<const int *>(tok)[n];
}

// The largest of U 16-byte vectors' values, NaN left out.
template <typename T, int U> HS_DEV float vec_max(const uint4 (&q)[U]) {
  if constexpr (sizeof(T) == 4) {
    float m = kNegInf;
#pragma unroll
    for (int j = 0; j < U; ++j)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(q[j].x), __uint_as_float(q[j].y)), fmaxf(__uint_as_float(q[j].z), __uint_as_float(q[j].w))));
    return m;
  } else {
    unsigned w = minus_inf_word<T>();
#pragma unroll
    for (int j = 0; j < U; ++j) w = word_max<T>(w, word_max<T>(word_max<T>(q[j].x, q[j].y), word_max<T>(q[j].z, q[j].w)));
    float v[2];
    unpack_word<T>(w, v);
    return fmaxf(v[0], v[1]);
  }
}
template <typename T> HS_DEV float vec_max(const uint4 &q) {
  const uint4 one[1] = {q};
  return vec_max<T, 1>(one);
}

// What a thread knows of its values.  S and U are kept as two partial sums
// each, for even and odd values.
template <typename T> struct Scan {
  float m = kNegInf;
  Cols<2> s = Cols<2>::all(0.f), u = Cols<2>::all(0.f);
  HS_DEV Stat stat() const {
    float a[2], b[2];
    s.get(a);
    u.get(b);
    return {m, a[0] + a[1], b[0] + b[1]};
  }
  // Moves the sums to the reference `to` >= m (from none, m = -inf, they are 0).
  HS_DEV void raise(float to, Scale k) {
    const float d = max_nan(m - to, k.floor);
    const Cols<2> f = Cols<2>::all(ex2(d * k.c));
    u = fma(Cols<2>::all(d), s, u) * f;
    s = s * f;
    m = to;
  }
  HS_DEV void add(const float *v, Cols<2> minus, Scale k) {
    float d[2];
    (Cols<2>::of(v) + minus).get(d);
    d[0] = max_nan(d[0], k.floor);
    d[1] = max_nan(d[1], k.floor);
    const Cols<2> dd = Cols<2>::of(d);
    float t[2];
    (dd * Cols<2>::all(k.c)).get(t);
    t[0] = ex2(t[0]);
    t[1] = ex2(t[1]);
    const Cols<2> e = Cols<2>::of(t);
    s = s + e;
    u = fma(e, dd, u);
  }
  HS_DEV void scalar(float v, Scale k) {
    if (v > m) raise(v, k);
    const float two[2] = {v, kNegInf};
    add(two, Cols<2>::all(-rel(m)), k);
  }
  template <int U> HS_DEV void vectors(const uint4 (&q)[U], Scale k) {
    constexpr int E = Row<T>::E;
    const float bm = vec_max<T, U>(q);
    if (bm > m) raise(bm, k);
    const Cols<2> minus = Cols<2>::all(-rel(m));
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float v[E];
      unpack_vec<T>(q[j], v);
#pragma unroll
      for (int e = 0; e < E; e += 2) add(v + e, minus, k);
    }
  }
};

constexpr int kChosen = 64, kFound = 128;  // threads read again, values collected: at most
constexpr int kBatch = 4;                 // vectors of a thread at a time

// What finding the alternatives of one row needs (chosen: the threads whose
// values are read again).
struct Finder {
  Key found[kFound];
  int nfound, nchosen, nkept;
  int chosen[kChosen];
  int2 whose[kChosen];  // threads whose best batch holds all they have, and its first vector
};
// Shared memory of a CTA: one row's, or the finders of a row per warp.
template <int W, bool TOP> struct Shared {
  Finder f[TOP && W == 1 ? kShortRows : 1];
  Stat stat[W];
  unsigned group[32];
  Key list[TOP && W > 1 ? W : 1][32];
  Stat cstat[kMaxCluster];  // written by the cluster's CTAs
  Key clist[TOP ? kMaxCluster : 1][32];
  uint4 kept[TOP ? kBatch : 1][TOP ? threads_of<W>() : 1];  // each thread's batch with its largest value
};

template <int W> HS_DEV void row_sync() {
  if (W == 1) __syncwarp(); else __syncthreads();
}
template <int W> HS_DEV int row_count(bool p) {
  return W == 1 ? __popc(__ballot_sync(0xffffffffu, p)) : __syncthreads_count(p);
}

HS_DEV unsigned remote(const void *p, int rank) {
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
HS_DEV void st_remote(const float *p, int rank, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote(p, rank)), "f"(v) : "memory");
}
HS_DEV void st_remote(const Key *p, int rank, Key v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(p, rank)), "l"(v) : "memory");
}

// W: warps per row.
template <typename T, int W, bool TOP>
__global__ void __launch_bounds__(threads_of<W>(), 1024 / threads_of<W>()) logprobs_fwd_kernel(const FwdArgs p) {
  __shared__ Shared<W, TOP> sh;
  constexpr int NT = 32 * W, U = kBatch, E = Row<T>::E;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tid = W == 1 ? lane : (int)threadIdx.x;
  const int C = W == 1 ? 1 : p.cluster, rank = (int)(blockIdx.x % C);
  const int64_t n = W == 1 ? (int64_t)blockIdx.x * kShortRows + warp : blockIdx.x / C;
  if (W == 1 && n >= p.N) return;
  const T *row = static_cast<const T *>(p.x) + n * p.ld;
  const int64_t tok = token_at(p.tok, p.token64, n);
  if (tok == p.ignore) {  // the whole cluster
    if (rank == 0) {
      if (tid == 0) {
        p.lp[n] = 0.f;
        if (p.ent) p.ent[n] = 0.f;
        if (p.stats) p.stats[2 * n] = p.stats[2 * n + 1] = 0.f;
      }
      if (TOP && tid < p.top) {
        p.top_lp[n * p.top + tid] = 0.f;
        p.top_id[n * p.top + tid] = -1;
      }
    }
    return;
  }
  __syncwarp();
  if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  const bool inside = tok >= 0 && tok < p.V;
  // the token's logit, loaded before the row: it is there when it is needed
  const float given = tid == 0 && rank == 0 && inside ? to_f32<T>(row[tok]) : 0.f;
  const Row<T> r(row, p.V, rank, C);
  Scan<T> scan;
  float second = kNegInf;  // the largest of the thread's vectors outside its best batch
  int best = -1;           // that batch's first vector
  // U vectors at a time, the next ones on their way meanwhile; -inf, which adds
  // nothing, past the end
  auto load = [&](uint4 (&q)[U], int i) {
    if (i + (U - 1) * NT < r.hi) {
#pragma unroll
      for (int k = 0; k < U; ++k) q[k] = __ldg(r.vec(i + k * NT));
    } else {
      constexpr unsigned w = minus_inf_word<T>();
#pragma unroll
      for (int k = 0; k < U; ++k) q[k] = i + k * NT < r.hi ? __ldg(r.vec(i + k * NT)) : make_uint4(w, w, w, w);
    }
  };
  auto take = [&](const uint4 (&q)[U], int i) {
    if constexpr (TOP) {
      const float bm = vec_max<T, U>(q);
      second = fmaxf(second, fminf(bm, scan.m));
      if (bm > scan.m) {
        best = i;
#pragma unroll
        for (int k = 0; k < U; ++k) sh.kept[k][threadIdx.x] = q[k];
      }
    }
    scan.template vectors<U>(q, p.k);
  };
  int at = r.lo + tid;
  if (at < r.hi) {
    uint4 q[2][U];
    load(q[0], at);
    while (true) {
      if ((at += U * NT) < r.hi) load(q[1], at);
      take(q[0], at - U * NT);
      if (at >= r.hi) break;
      if ((at += U * NT) < r.hi) load(q[0], at);
      take(q[1], at - U * NT);
      if (at >= r.hi) break;
    }
  }
  if (tid < r.head) scan.scalar(to_f32<T>(row[tid]), p.k);
  if (tid < r.ntail) scan.scalar(to_f32<T>(row[r.tail0 + tid]), p.k);

  // the row's statistics
  Stat a = reduce(scan.stat(), 32, p.k);
  if (W > 1 && lane == 0) sh.stat[warp] = a;

  Key list = 0;
  if constexpr (TOP) {
    Finder &f = sh.f[W == 1 ? warp : 0];
    if (tid == 0) f.nfound = f.nchosen = f.nkept = 0;
    if (W == 1) __syncwarp();  // before any lane counts (shuffles and votes order no memory)
    const bool some = tid < r.head || r.lo + tid < r.hi || tid < r.ntail;  // this thread holds values
    const unsigned mine = some ? order_bits(scan.m) : 0;
    // A bound that at least `top` threads reach, and not many more: the top-th
    // largest of the maxima of 32 groups of threads, raised by bisection where
    // more than a few too many reach it (large `top`, equal values).
    unsigned v = mine;
#pragma unroll
    for (int o = 1; o < W; o <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (W > 1) {
      if (lane % W == 0) sh.group[(warp * 32 + lane) / W] = v;
      __syncthreads();
      v = sh.group[lane];
    }
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)  // in descending order of lanes
#pragma unroll
      for (int o = size >> 1; o; o >>= 1) {
        const unsigned w = __shfl_xor_sync(0xffffffffu, v, o);
        v = ((lane & o) == 0) == ((lane & size) == 0) ? max(v, w) : min(v, w);
      }
    unsigned lo = __shfl_sync(0xffffffffu, v, p.top - 1), hi = __shfl_sync(0xffffffffu, v, 0);
    if (lo == 0) lo = 1;  // some groups hold nothing
    hi += 1;
    int c = row_count<W>(mine >= lo);
    while (c > p.top + 8 && hi - lo > 1) {
      const unsigned mid = lo + (hi - lo) / 2;
      const int n = row_count<W>(mine >= mid);
      if (n >= p.top) lo = mid, c = n; else hi = mid;
    }
    if (c < p.top) lo = 1;  // fewer threads with values than alternatives: all of them
    // the bound as a value (below -inf's image: everything but NaN)
    const float bound = lo <= order_bits(kNegInf) ? kNegInf : value_of((Key)lo << 32);
    auto collect = [&](float v, int at) {
      if (!(v >= bound)) return;
      const int k = atomicAdd(&f.nfound, 1);  // in any order: the keys are sorted
      if (k < kFound) f.found[k] = make_key(v, at);
    };
    auto vector = [&](const uint4 &q, int at) {
      float v[E];
      unpack_vec<T>(q, v);
      unsigned hit = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) hit |= v[e] >= bound ? 1u << e : 0u;
      if (!hit) return;
      int k = atomicAdd(&f.nfound, __popc(hit));
#pragma unroll
      for (int e = 0; e < E; ++e)
        if ((hit >> e) & 1) {
          if (k < kFound) f.found[k] = make_key(v[e], r.index(at, e));
          ++k;
        }
    };
    if (some && scan.m >= bound) {
      if (tid < r.head) collect(to_f32<T>(row[tid]), tid);
      if (tid < r.ntail) collect(to_f32<T>(row[r.tail0 + tid]), r.tail0 + tid);
      if (second >= bound) {  // beyond the best batch too
        const int at = atomicAdd(&f.nchosen, 1);
        if (at < kChosen) f.chosen[at] = tid;
      } else if (best >= 0) {
        const int at = atomicAdd(&f.nkept, 1);
        if (at < kChosen) f.whose[at] = make_int2(threadIdx.x, best);
      }
    }
    row_sync<W>();
    const int nchosen = f.nchosen, nkept = f.nkept;
    if (nchosen <= kChosen && nkept <= kChosen) {
      // the vectors of the chosen threads from memory, then the kept batches
      const int per = (r.hi - r.lo + NT - 1) / NT, all = nchosen * per, items = all + nkept * U;
      constexpr int G = W == 1 ? 1 : 3;  // loads at once
      for (int j0 = tid; j0 < items; j0 += G * NT) {
        uint4 q[G];
        int at[G];
#pragma unroll
        for (int k = 0; k < G; ++k) {
          const int j = j0 + k * NT;
          at[k] = r.hi;
          if (j < all) {
            const int t = j / per;
            at[k] = r.lo + f.chosen[t] + (j - t * per) * NT;
            if (at[k] < r.hi) q[k] = __ldg(r.vec(at[k]));
          } else if (j < items) {
            const int2 o = f.whose[(j - all) / U];
            at[k] = o.y + (j - all) % U * NT;
            q[k] = sh.kept[(j - all) % U][o.x];
          }
        }
#pragma unroll
        for (int k = 0; k < G; ++k)
          if (at[k] < r.hi) vector(q[k], at[k]);
      }
    }
    row_sync<W>();
    const int n = f.nfound;
    if (nchosen <= kChosen && nkept <= kChosen && n <= kFound) {
      if (W == 1 || warp == 0) {
        // in order by counting the larger ones
        auto rank = [&](auto keys) {
          constexpr int M = decltype(keys)::value;  // of a lane
          Key a[M];
          int before[M] = {};
#pragma unroll
          for (int i = 0; i < M; ++i) a[i] = lane + 32 * i < n ? f.found[lane + 32 * i] : 0;
#pragma unroll 4
          for (int j = 0; j < n; ++j) {
            const Key k = f.found[j];
#pragma unroll
            for (int i = 0; i < M; ++i) before[i] += k > a[i];
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < M; ++i)
            if (lane + 32 * i < n && before[i] < 32) f.found[before[i]] = a[i];
          __syncwarp();
        };
        if (n <= 64) rank(std::integral_constant<int, 2>{});
        else rank(std::integral_constant<int, kFound / 32>{});
        list = lane < n ? f.found[lane] : 0;
      }
    } else {  // too many equal values
      auto add = [&](float v, int at, bool ok) {
        const Key k = ok && !isnan(v) ? make_key(v, at) : 0;
        if (__any_sync(0xffffffffu, k > __shfl_sync(0xffffffffu, list, 31))) list = merge_desc(list, sort_desc(k, lane), lane);
      };
      if (W == 1 || warp == 0) {
        add(lane < r.head ? to_f32<T>(row[lane]) : 0.f, lane, lane < r.head);
        add(lane < r.ntail ? to_f32<T>(row[r.tail0 + lane]) : 0.f, r.tail0 + lane, lane < r.ntail);
      }
      for (int i0 = r.lo + (W == 1 ? 0 : warp * 32); i0 < r.hi; i0 += NT) {
        const int i = i0 + lane;
        const uint4 q = i < r.hi ? __ldg(r.vec(i)) : uint4{};
        const Key last = __shfl_sync(0xffffffffu, list, 31);
        if (!__any_sync(0xffffffffu, i < r.hi && order_bits(vec_max<T>(q)) >= (unsigned)(last >> 32))) continue;
        float v[E];
        unpack_vec<T>(q, v);
#pragma unroll 1
        for (int e = 0; e < E; ++e) {
          float x = v[0];
#pragma unroll
          for (int o = 1; o < E; ++o) x = e == o ? v[o] : x;
          add(x, r.index(i, e), i < r.hi);
        }
      }
      if (W > 1) {
        sh.list[warp][lane] = list;
        __syncthreads();
        if (warp == 0)
          for (int w = 1; w < W; ++w) list = merge_desc(list, sh.list[w][lane], lane);
      }
    }
  } else if (W > 1) {
    __syncthreads();
  }
  if (W > 1) {
    if (warp != 0 && C == 1) return;
    if (warp == 0) {
      a = reduce(sh.stat[lane & (W - 1)], W, p.k);
    }
    if (C > 1) {
      __syncwarp();
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA has started
      if (warp == 0) {
        if (lane == 0) {
          st_remote(&sh.cstat[rank].m, 0, a.m);
          st_remote(&sh.cstat[rank].s, 0, a.s);
          st_remote(&sh.cstat[rank].u, 0, a.u);
        }
        if (TOP) st_remote(&sh.clist[rank][lane], 0, list);
      }
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
      if (rank != 0 || warp != 0) return;
      a = sh.cstat[0];
      for (int j = 1; j < C; ++j) merge(a, sh.cstat[j], p.k);
      if (TOP) {
        list = sh.clist[0][lane];
        for (int j = 1; j < C; ++j) list = merge_desc(list, sh.clist[j][lane], lane);
      }
    }
  }
  const float kLn2 = 0.69314718055994531f;
  const bool empty = a.m == kNegInf && a.s == 0.f, bad = isnan(a.s);  // only -inf; a NaN or +inf
  const float ls = log2f(a.s);
  auto logp = [&](float x) { return empty ? kNegInf : bad ? a.s : fmaf(x - a.m, p.inv_t, -kLn2 * ls); };
  if (lane == 0) {
    if (inside) {
      p.lp[n] = logp(given);
    } else {
      p.lp[n] = __int_as_float(0x7fc00000);
      report(p.status, HS_ERR_INDEX);
    }
    if (p.ent) p.ent[n] = empty ? 0.f : kLn2 * ls - p.inv_t * (a.u / a.s);
    if (p.stats) {
      p.stats[2 * n] = bad ? a.s : a.m;
      p.stats[2 * n + 1] = ls;
    }
  }
  if (TOP && lane < p.top) {
    p.top_lp[n * p.top + lane] = logp(value_of(list));
    p.top_id[n * p.top + lane] = bad ? -1 : index_of(list);
  }
}

// ------------------------------------------------------------------ gradient
struct BwdArgs {
  const void *x;
  int64_t ld;
  const void *tok;
  int token64;
  int64_t ignore;
  float c, inv_t;
  int top;
  const float *stats, *ent, *g, *ge, *gt;
  const int64_t *top_id;
  void *dx;
  int64_t dld;
  int64_t N, V;
  int parts;  // CTAs per row
};

template <typename T, int W>
__global__ void __launch_bounds__(threads_of<W>()) logprobs_bwd_kernel(const BwdArgs p) {
  constexpr int NT = 32 * W, U = 4, E = Row<T>::E;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tid = W == 1 ? lane : (int)threadIdx.x;
  const int C = W == 1 ? 1 : p.parts, rank = (int)(blockIdx.x % C);
  const int64_t n = W == 1 ? (int64_t)blockIdx.x * kShortRows + warp : blockIdx.x / C;
  if (W == 1 && n >= p.N) return;
  const T *row = static_cast<const T *>(p.x) + n * p.ld;
  T *out = static_cast<T *>(p.dx) + n * p.dld;
  const int64_t tok = token_at(p.tok, p.token64, n);
  const float m = p.stats[2 * n], ls = p.stats[2 * n + 1];
  const bool zero = tok == p.ignore || m == kNegInf;
  const float kLn2 = 0.69314718055994531f;
  const bool named = tok >= 0 && tok < p.V;
  const float g = p.g && named ? p.g[n] : 0.f;
  float sum = g;  // G: every gradient of a log probability of this row
  if (p.gt && !zero)
    for (int j = 0; j < p.top; ++j)
      if (p.top_id[n * p.top + j] >= 0) sum += p.gt[n * p.top + j];
  const float ge = p.ge && !zero ? p.ge[n] : 0.f;
  // dx = -inv_t p (sum + ge (ln2 t + entropy)) = p (k0 + k1 t)
  const float k0 = ge != 0.f ? -p.inv_t * fmaf(ge, p.ent[n], sum) : -p.inv_t * sum, k1 = -p.inv_t * ge * kLn2;
  const Cols<2> minus = Cols<2>::all(-m), cc = Cols<2>::all(p.c), mls = Cols<2>::all(-ls), kk0 = Cols<2>::all(k0),
                kk1 = Cols<2>::all(k1);
  auto grad2 = [&](float *v) {  // two logits to their gradients
    float t[2], e[2];
    fma(Cols<2>::of(v) + minus, cc, mls).get(t);
    t[0] = max_nan(t[0], kFloor);
    t[1] = max_nan(t[1], kFloor);
    e[0] = ex2(t[0]);
    e[1] = ex2(t[1]);
    (Cols<2>::of(e) * fma(kk1, Cols<2>::of(t), kk0)).get(v);
  };
  auto grad = [&](float x) {
    float v[2] = {x, x};
    grad2(v);
    return v[0];
  };
  const Row<T> r(row, p.V, rank, C);
  // vectors where the output's row is aligned like the input's, else one value at a time
  const bool vec = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  if (tid < r.head) out[tid] = from_f32<T>(zero ? 0.f : grad(to_f32<T>(row[tid])));
  if (vec) {
    uint4 *o = reinterpret_cast<uint4 *>(out + r.base);
    auto one = [&](const uint4 &q) {
      float v[E];
      unpack_vec<T>(q, v);
#pragma unroll
      for (int e = 0; e < E; e += 2) grad2(v + e);
      constexpr int P = PerWord<T>::value;
      return make_uint4(pack_word<T>(v), pack_word<T>(v + P), pack_word<T>(v + 2 * P), pack_word<T>(v + 3 * P));
    };
    int i = r.lo + tid;
    if (zero) {
      for (; i < r.hi; i += NT) o[i] = uint4{};
    } else {
      for (; i < r.hi; i += U * NT) {
        uint4 q[U];
        if (i + (U - 1) * NT < r.hi) {
#pragma unroll
          for (int k = 0; k < U; ++k) q[k] = __ldg(r.vec(i + k * NT));
#pragma unroll
          for (int k = 0; k < U; ++k) o[i + k * NT] = one(q[k]);
        } else {
#pragma unroll
          for (int k = 0; k < U - 1; ++k)
            if (i + k * NT < r.hi) q[k] = __ldg(r.vec(i + k * NT));
#pragma unroll
          for (int k = 0; k < U - 1; ++k)
            if (i + k * NT < r.hi) o[i + k * NT] = one(q[k]);
        }
      }
    }
  } else {
    for (int i = r.index(r.lo, 0) + tid; i < r.index(r.hi, 0); i += NT) out[i] = from_f32<T>(zero ? 0.f : grad(to_f32<T>(row[i])));
  }
  if (tid < r.ntail) out[r.tail0 + tid] = from_f32<T>(zero ? 0.f : grad(to_f32<T>(row[r.tail0 + tid])));
  if (zero) return;
  // the values that the gradients name, whole: written again by the CTA that wrote them
  if (W == 1) __syncwarp(); else __syncthreads();
  const int a = rank == 0 ? 0 : r.index(r.lo, 0), b = rank == C - 1 ? (int)p.V : r.index(r.hi, 0);
  for (int j = tid; j <= p.top; j += NT) {
    const int64_t v = j < p.top ? (p.gt ? p.top_id[n * p.top + j] : -1) : (named ? tok : -1);
    if (v < a || v >= b) continue;
    float add = v == tok ? g : 0.f;
    if (p.gt)
      for (int k = 0; k < p.top; ++k)
        if (p.top_id[n * p.top + k] == v) add += p.gt[n * p.top + k];
    out[v] = from_f32<T>(fmaf(p.inv_t, add, grad(to_f32<T>(row[v]))));
  }
}

// ------------------------------------------------------------------ launch
// Warps per row.  One up to 4 KB (4096 rows of 1 KB: 3.5 us, with four warps
// 10.5), in the forward of many rows up to 8 KB (8192 of 8 KB: 16.8 against 23.5
// us); four up to 64 KB (16384 of 64 KB: 174 us, with eight 195), in the forward
// of any longer rows where they alone fill the SMs (600 rows of 100 KB with 5
// alternatives: 20.8 us, with eight 24.4; 2047: 48.5 and 53.8; but 500 of 600
// KB: 68 and 60); else eight (the gradient of 2047 rows of 100 KB: 77 us, with
// four 81).
int warps_of(bool forward, int64_t N, int64_t row_bytes) {
  if (row_bytes <= 4096 || (forward && row_bytes <= 8192 && N >= 2048)) return 1;
  return row_bytes <= 65536 || (forward && N >= 4 * 148) ? 4 : 8;
}

// CTAs per row, of 8 KB at least.  The forward's meet in a cluster, which
// pays where the rows alone leave SMs idle (24 rows of 512 KB: 7.1 us on
// eight CTAs each, 20 on one; 300 rows of 100 KB: 15.5 on one, 20.5 on two); the
// gradient's are independent.
int parts_of(bool forward, int64_t N, int64_t row_bytes) {
  int c = 1;
  while (c < (forward ? kMaxCluster : 256) && (forward ? 2 * N * c <= 2 * 148 : N * c < 4 * 148) && row_bytes / (2 * c) >= 8192) c *= 2;
  return c;
}

int check_rows(const char *who, int dtype, const void *x, int64_t ld, int token_bits, const void *tok, float temperature,
               int top, int64_t N, int64_t V) {
  if (!dtype_ok(dtype)) return fail(HS_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
  if (token_bits != 32 && token_bits != 64) return fail(HS_ERR_INVALID_ARG, "%s: token_bits is 32 or 64", who);
  if (N < 0 || V < 0) return fail(HS_ERR_INVALID_ARG, "%s: negative N or V", who);
  if (V > (int64_t)1 << 30 || N > (int64_t)1 << 27) return fail(HS_ERR_UNSUPPORTED, "%s: V above 2^30 or N above 2^27", who);
  if (!(temperature >= 1e-30f) || !(temperature <= 1e30f))
    return fail(HS_ERR_INVALID_ARG, "%s: the temperature must be positive (1e-30 to 1e30)", who);
  if (top < 0 || top > HS_MAX_TOP || top > V) return fail(HS_ERR_INVALID_ARG, "%s: top=%d outside 0..min(%d, V)", who, top, HS_MAX_TOP);
  if (N == 0) return HS_OK;
  if (V == 0) return fail(HS_ERR_INVALID_ARG, "%s: rows of no logits", who);
  if (!x || !aligned(x, dtype_bytes(dtype)) || !tok || !aligned(tok, token_bits / 8))
    return fail(HS_ERR_INVALID_ARG, "%s: null or misaligned logits or tokens", who);
  if (ld < V && N > 1) return fail(HS_ERR_INVALID_ARG, "%s: rows %lld apart hold %lld logits", who, (long long)ld, (long long)V);
  return HS_OK;
}

template <typename F> int by_type(int dtype, F f) {
  if (dtype == HS_F32) return f(float{});
  if (dtype == HS_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}

}  // namespace
}  // namespace hs

extern "C" {

int hs_token_logprobs_forward(int dtype, const void *logits, int64_t logits_ld, int token_bits, const void *tokens,
                              int64_t ignore_index, float temperature, int top, float *logprob, float *entropy,
                              float *top_logprob, int64_t *top_index, float *stats, int64_t N, int64_t V,
                              int *dev_status, hs_stream_t stream) {
  using namespace hs;
  if (int e = check_rows("hs_token_logprobs_forward", dtype, logits, logits_ld, token_bits, tokens, temperature, top, N, V)) return e;
  if (N == 0) return HS_OK;
  if (!logprob || (top && (!top_logprob || !top_index)) || !dev_status)
    return fail(HS_ERR_INVALID_ARG, "hs_token_logprobs_forward: null output or dev_status");
  FwdArgs a = {};
  a.x = logits, a.ld = logits_ld, a.tok = tokens, a.token64 = token_bits == 64, a.ignore = ignore_index;
  a.k.c = (float)(1.4426950408889634 / (double)temperature), a.k.floor = kFloor / a.k.c;
  a.inv_t = (float)(1.0 / (double)temperature);
  a.top = top, a.lp = logprob, a.ent = entropy, a.top_lp = top_logprob, a.top_id = top_index, a.stats = stats;
  a.N = N, a.V = V, a.status = dev_status;
  const int64_t bytes = V * (int64_t)dtype_bytes(dtype);
  const int warps = warps_of(true, N, bytes);
  a.cluster = warps == 1 ? 1 : parts_of(true, N, bytes);
  return by_type(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    auto kernel = warps == 1   ? (top ? logprobs_fwd_kernel<T, 1, true> : logprobs_fwd_kernel<T, 1, false>)
                  : warps == 4 ? (top ? logprobs_fwd_kernel<T, 4, true> : logprobs_fwd_kernel<T, 4, false>)
                               : (top ? logprobs_fwd_kernel<T, 8, true> : logprobs_fwd_kernel<T, 8, false>);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(warps == 1 ? (N + kShortRows - 1) / kShortRows : N * a.cluster));
    cfg.blockDim = dim3(warps == 1 ? 32 * kShortRows : 32 * warps);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)a.cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = a.cluster > 1;
    (void)cudaLaunchKernelEx(&cfg, kernel, a);
    return check_launch("logprobs_fwd_kernel");
  });
}

int hs_token_logprobs_backward(int dtype, const void *logits, int64_t logits_ld, int token_bits, const void *tokens,
                               int64_t ignore_index, float temperature, int top, const float *stats,
                               const float *entropy, const int64_t *top_index, const float *dlogprob,
                               const float *dentropy, const float *dtop_logprob, void *dlogits, int64_t dlogits_ld,
                               int64_t N, int64_t V, hs_stream_t stream) {
  using namespace hs;
  if (int e = check_rows("hs_token_logprobs_backward", dtype, logits, logits_ld, token_bits, tokens, temperature, top, N, V)) return e;
  if (N == 0) return HS_OK;
  if (!stats || !dlogits || !aligned(dlogits, dtype_bytes(dtype)) || (dentropy && !entropy) || (dtop_logprob && top && !top_index))
    return fail(HS_ERR_INVALID_ARG, "hs_token_logprobs_backward: null or misaligned tensor");
  if (dlogits_ld < V && N > 1) return fail(HS_ERR_INVALID_ARG, "hs_token_logprobs_backward: dlogits rows overlap");
  BwdArgs a = {};
  a.x = logits, a.ld = logits_ld, a.tok = tokens, a.token64 = token_bits == 64, a.ignore = ignore_index;
  a.c = (float)(1.4426950408889634 / (double)temperature), a.inv_t = (float)(1.0 / (double)temperature);
  a.top = top, a.stats = stats, a.ent = entropy, a.top_id = top_index;
  a.g = dlogprob, a.ge = dentropy, a.gt = top ? dtop_logprob : nullptr;
  a.dx = dlogits, a.dld = dlogits_ld, a.N = N, a.V = V;
  const int64_t bytes = V * (int64_t)dtype_bytes(dtype);
  const int warps = warps_of(false, N, bytes);
  a.parts = warps == 1 ? 1 : parts_of(false, N, bytes);
  const unsigned grid = (unsigned)(warps == 1 ? (N + kShortRows - 1) / kShortRows : N * a.parts);
  return by_type(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    if (warps == 1)
      logprobs_bwd_kernel<T, 1><<<grid, threads_of<1>(), 0, (cudaStream_t)stream>>>(a);
    else if (warps == 4)
      logprobs_bwd_kernel<T, 4><<<grid, threads_of<4>(), 0, (cudaStream_t)stream>>>(a);
    else
      logprobs_bwd_kernel<T, 8><<<grid, threads_of<8>(), 0, (cudaStream_t)stream>>>(a);
    return check_launch("logprobs_bwd_kernel");
  });
}

}  // extern "C"
