// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out_n = s W[tok_n],   dW[v] = s sum_{n : tok_n = v} dout_n
//
// Bound: memory.  The lookup reads N rows and writes N rows; the gradient
// reads the N rows of dout once and writes the V rows of dW once.
//
// Gradient:
//   1. The ids are sorted with their positions (stable, least significant
//      digit first, up to 9 bits a pass: two passes for any vocabulary below
//      2^18); in one launch of one cluster up to 16384 tokens, in two launches
//      per pass over the GPU beyond.
//   2. Pieces of 32 consecutive sorted entries x 32 lanes of up to 16 bytes:
//      each warp sums the runs of equal ids in its piece in float32.  A run
//      inside the piece is a finished row of dW; one that crosses a piece
//      boundary leaves its part in the workspace.  The work of a warp does not depend on
//      how often a token occurs, so a frequent token costs no more than rare
//      ones.  Further CTAs write the zero rows of the ids that a search in
//      the sorted entries does not find.
//   3. The parts of each crossing run are added in order.
// dW is therefore written once (no clearing pass), there are no atomics on
// floating-point data, and the order of every sum follows from the tokens alone.
//
// Measured on one B200 (plain copy 6.53 TB/s), ids as skewed as text: 131072
// tokens of a 131072 x 1024 bfloat16 table take 60 us for the lookup and 131 for
// the gradient, of which the sort takes 26 and the sums 88 (537 MB, 6.1 TB/s);
// 8192 tokens of 32000 x 512 float32 take 5.4 and 31 us (sort 12: two passes
// whose steps wait on one another).
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "lm_types.cuh"

namespace hs {
namespace {

constexpr int kPiece = 32;        // sorted entries per warp of the summing kernel
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortCluster = 8;   // CTAs of the sorting cluster at most
constexpr int kMaxBits = 9;       // bits of a sorting pass at most
constexpr int kAhead = 8;         // groups of 32 entries that a sorting warp loads at once

template <int BYTES> struct Chunk;  // one lane's bytes of a row
template <> struct Chunk<16> { using type = uint4; };
template <> struct Chunk<8> { using type = uint2; };
template <> struct Chunk<4> { using type = unsigned; };
template <> struct Chunk<2> { using type = unsigned short; };

// The scale as a sum of two float32, so that a float32 product with it is rounded
// once although the scale (the root of a width, say) is no float32; v * lo is kept
// finite, as it would make a NaN of an infinity (with lo = 0, or of the other
// sign).  A product that is rounded to 16 bits does without lo, which is
// 2^-25 of it.
struct Scale {
  float hi, lo;
};
template <typename T> HS_DEV float scaled(float v, Scale s) {
  if constexpr (sizeof(T) == 2) return v * s.hi;
  return fmaf(v, s.hi, fmaxf(fminf(v * s.lo, FLT_MAX), -FLT_MAX));
}
Scale make_scale(double s) {
  const float hi = (float)s;
  const double lo = s - (double)hi;
  return {hi, lo == lo && lo - lo == 0.0 ? (float)lo : 0.f};
}

template <typename T, int BYTES> HS_DEV void chunk_to_f32(const typename Chunk<BYTES>::type &c, float *v) {
  if constexpr (BYTES == 2) {
    v[0] = to_f32<T>(*reinterpret_cast<const T *>(&c));
  } else {
    const unsigned *w = reinterpret_cast<const unsigned *>(&c);
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) unpack_word<T>(w[i], v + i * PerWord<T>::value);
  }
}
template <typename T, int BYTES> HS_DEV typename Chunk<BYTES>::type chunk_of_f32(const float *v) {
  typename Chunk<BYTES>::type c;
  if constexpr (BYTES == 2) {
    *reinterpret_cast<T *>(&c) = from_f32<T>(v[0]);
  } else {
    unsigned *w = reinterpret_cast<unsigned *>(&c);
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) w[i] = pack_word<T>(v + i * PerWord<T>::value);
  }
  return c;
}

// E float32 of a part of a run, at a multiple of E (whole chunks divide a row).
template <int E> HS_DEV void load_part(const float *p, float *v) {
  if constexpr (E % 4 == 0) {
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float4 t = *reinterpret_cast<const float4 *>(p + e);
      v[e] = t.x, v[e + 1] = t.y, v[e + 2] = t.z, v[e + 3] = t.w;
    }
  } else if constexpr (E == 2) {
    const float2 t = *reinterpret_cast<const float2 *>(p);
    v[0] = t.x, v[1] = t.y;
  } else {
    v[0] = *p;
  }
}
template <int E> HS_DEV void store_part(float *p, const float *v) {
  if constexpr (E % 4 == 0) {
#pragma unroll
    for (int e = 0; e < E; e += 4) *reinterpret_cast<float4 *>(p + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
  } else if constexpr (E == 2) {
    *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
  } else {
    *p = v[0];
  }
}

// ------------------------------------------------------------------ lookup
// One thread per row chunk and four chunks per thread, a CTA's width apart.
template <typename T, int BYTES, typename TOK>
__global__ void __launch_bounds__(256) emb_lookup_kernel(const char *w, int64_t ld_bytes, const TOK *tok, Scale scale,
                                                         char *out, int64_t total, int chunks, int64_t V, int *status) {
  using C = typename Chunk<BYTES>::type;
  constexpr int E = BYTES / (int)sizeof(T);
  const int64_t i0 = (int64_t)blockIdx.x * (256 * 4) + threadIdx.x;
  const bool small = total <= 0xffffffffll;  // a 32-bit division will do
  C c[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t i = i0 + k * 256;
    if (i < total) {
      const int64_t n = small ? (int64_t)((unsigned)i / (unsigned)chunks) : i / chunks;
      const int64_t t = (int64_t)tok[n];
      if (t >= 0 && t < V) {
        c[k] = *reinterpret_cast<const C *>(w + t * ld_bytes + (i - n * chunks) * BYTES);
      } else {
        c[k] = C{};
        report(status, HS_ERR_INDEX);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t i = i0 + k * 256;
    if (i < total) {
      float v[E];
      chunk_to_f32<T, BYTES>(c[k], v);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = scaled<T>(v[e], scale);
      *reinterpret_cast<C *>(out + i * BYTES) = chunk_of_f32<T, BYTES>(v);
    }
  }
}

// Rows that are not whole 16-byte chunks: a warp per row, so that no position
// is divided by the row's length (92769 rows of 841 float16: 54 us, by the kernel above 174).
template <typename T, int BYTES, typename TOK>
__global__ void __launch_bounds__(256) emb_lookup_rows_kernel(const char *w, int64_t ld_bytes, const TOK *tok, Scale scale,
                                                              char *out, int64_t N, int chunks, int64_t V, int *status) {
  using C = typename Chunk<BYTES>::type;
  constexpr int E = BYTES / (int)sizeof(T), K = 8;
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= N) return;
  const int64_t t = (int64_t)tok[n];
  const bool inside = t >= 0 && t < V;
  if (!inside && lane == 0) report(status, HS_ERR_INDEX);
  const C *src = reinterpret_cast<const C *>(w + (inside ? t : 0) * ld_bytes);
  C *dst = reinterpret_cast<C *>(out + n * chunks * (int64_t)BYTES);
  for (int c0 = lane; c0 < chunks; c0 += 32 * K) {
    C c[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (c0 + 32 * k < chunks) c[k] = inside ? src[c0 + 32 * k] : C{};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (c0 + 32 * k < chunks) {
        float v[E];
        chunk_to_f32<T, BYTES>(c[k], v);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = scaled<T>(v[e], scale);
        dst[c0 + 32 * k] = chunk_of_f32<T, BYTES>(v);
      }
    }
  }
}

// ------------------------------------------------------------------ sort
HS_DEV void cluster_sync_all() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
HS_DEV void st_cluster_u32(const void *p, int rank, unsigned v) {
  const unsigned a = (unsigned)__cvta_generic_to_shared(p);
  asm volatile(
      "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, %1;\n\tst.shared::cluster.u32 [r], %2;\n\t}" ::"r"(a),
      "r"(rank), "r"(v)
      : "memory");
}

struct SortArgs {
  const void *tok;
  int64_t N, V, pad;
  uint2 *pair[2];     // {key, position}
  unsigned *counts;   // [CTAs][digits] of a pass (grid form)
  int passes, bits;
  int *status;
};

// One pass of a stable counting sort.  Every warp owns a contiguous part of
// the entries: it counts its digits, the counts are added up over warps, CTAs
// and digits, and it then places its entries in order, so entries of one digit
// keep their order.  Ids out of range and the padding id sort as V, last.
template <typename TOK> struct Pass {
  const SortArgs &p;
  int pass, shift, D;
  int lane, warp;
  int64_t lo, hi;  // this warp's entries
  HS_DEV Pass(const SortArgs &a, int pass_, int ctas, int rank)
      : p(a), pass(pass_), shift(pass_ * a.bits), D(1 << a.bits), lane(threadIdx.x & 31), warp(threadIdx.x >> 5) {
    const int64_t per = (p.N + (int64_t)ctas * kSortThreads - 1) / ((int64_t)ctas * kSortThreads) * 32;
    lo = min(p.N, ((int64_t)rank * kSortWarps + warp) * per);
    hi = min(p.N, lo + per);
  }
  // kAhead groups of 32 entries, all loads in flight at once
  HS_DEV void load(uint2 (&e)[kAhead], int64_t b) const {
    const uint2 *src = p.pair[(pass + 1) & 1];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t i = b + u * 32 + lane;
      e[u] = {0u, 0u};
      if (i < hi) {
        if (pass) {
          e[u] = __ldcg(src + i);
        } else {
          const int64_t t = (int64_t)static_cast<const TOK *>(p.tok)[i];
          const bool inside = t >= 0 && t < p.V;
          if (!inside) report(p.status, HS_ERR_INDEX);
          e[u] = {inside && t != p.pad ? (unsigned)t : (unsigned)p.V, (unsigned)i};
        }
      }
    }
  }
  HS_DEV unsigned digit(uint2 e) const { return (e.x >> shift) & (D - 1); }
  // Whether the warp's entries are few enough to stay in registers from
  // counting to placing.
  HS_DEV bool once() const { return hi - lo <= 32 * kAhead; }
  // adds this warp's digits to h; e: its last (or only) entries
  HS_DEV void count(unsigned *h, uint2 (&e)[kAhead]) const {
    for (int64_t b = lo; b < hi; b += 32 * kAhead) {
      load(e, b);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (b + u * 32 + lane < hi) atomicAdd(h + digit(e[u]), 1u);
    }
  }
  // the counts of the warps, [kSortWarps][D], to those of the warps before; their sum
  HS_DEV unsigned over_warps(unsigned *hist) const {
    unsigned run = 0;
#pragma unroll 8
    for (int w = 0; w < kSortWarps; ++w) {
      const unsigned c = hist[w * D + threadIdx.x];
      hist[w * D + threadIdx.x] = run;
      run += c;
    }
    return run;
  }
  // base[d]: the place of the CTA's first entry of digit d, from the thread's
  // digit's counts in all CTAs and in those before this one.  Whole CTA.
  HS_DEV void bases(unsigned *base, unsigned *wsum, unsigned all, unsigned before) const {
    unsigned inc = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    if ((int)threadIdx.x < D) {
      unsigned less = 0;
      for (int w = 0; w < warp; ++w) less += wsum[w];
      base[threadIdx.x] = less + inc - all + before;
    }
    __syncthreads();
  }
  HS_DEV void place(const unsigned *base, unsigned *h, uint2 (&e)[kAhead]) const {
    uint2 *dst = p.pair[pass & 1];
    for (int64_t b = lo; b < hi; b += 32 * kAhead) {
      if (!once()) load(e, b);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (b + u * 32 >= hi) break;
        const bool ok = b + u * 32 + lane < hi;
        const unsigned dig = digit(e[u]);
        // the lanes of the same digit, by a vote on each of its bits (with a
        // match instruction the whole sort took 82 us in place of 63)
        unsigned same = __ballot_sync(0xffffffffu, ok);
#pragma unroll
        for (int bit = 0; bit < kMaxBits; ++bit) {
          const unsigned set = __ballot_sync(0xffffffffu, (dig >> bit) & 1);
          same &= ((dig >> bit) & 1) ? set : ~set;
        }
        unsigned at = 0;
        if (ok) at = base[dig] + h[dig] + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (ok && lane == __ffs(same) - 1) h[dig] += __popc(same);
        __syncwarp();
        if (ok) dst[at] = e[u];
      }
    }
  }
};

// Few tokens: all passes in one launch of one cluster.
template <typename TOK>
__global__ void __launch_bounds__(kSortThreads, 1) emb_sort_kernel(const SortArgs p) {
  extern __shared__ __align__(16) unsigned sm[];
  __shared__ unsigned wsum[kSortWarps];
  const int D = 1 << p.bits, C = gridDim.x, rank = blockIdx.x, tid = threadIdx.x;
  unsigned *hist = sm;                         // [warps][D]
  unsigned *tot = hist + kSortWarps * D;       // [cluster][D], written by the cluster's CTAs
  unsigned *base = tot + kSortCluster * D;     // [D]
  for (int pass = 0; pass < p.passes; ++pass) {
    const Pass<TOK> q(p, pass, C, rank);
    unsigned *h = hist + q.warp * D;
    for (int i = q.lane; i < D; i += 32) h[i] = 0;
    __syncwarp();
    uint2 e[kAhead];
    q.count(h, e);
    if (pass == 0 && C > 1) cluster_sync_all();  // every CTA has started before its memory is written
    __syncthreads();
    if (tid < D) {
      const unsigned n = q.over_warps(hist);
      if (C == 1)
        tot[tid] = n;
      else
        for (int r = 0; r < C; ++r) st_cluster_u32(tot + rank * D + tid, r, n);
    }
    if (C > 1) cluster_sync_all(); else __syncthreads();
    unsigned before = 0, all = 0;
    if (tid < D) {
      for (int r = 0; r < C; ++r) {
        const unsigned c = tot[r * D + tid];
        if (r < rank) before += c;
        all += c;
      }
    }
    q.bases(base, wsum, all, before);
    q.place(base, h, e);
    if (C > 1) cluster_sync_all(); else __syncthreads();
  }
}

// Many tokens: two launches per pass over up to kSortCtas CTAs (placing
// writes 32 separate sectors per warp, which binds a single cluster's SMs: 54 us
// for 131072 tokens there).
constexpr int kSortCtas = 64;

template <typename TOK>
__global__ void __launch_bounds__(kSortThreads, 1) emb_count_kernel(const SortArgs p, int pass) {
  __shared__ unsigned h[1 << kMaxBits];
  const Pass<TOK> q(p, pass, gridDim.x, blockIdx.x);
  if ((int)threadIdx.x < q.D) h[threadIdx.x] = 0;
  __syncthreads();
  uint2 e[kAhead];
  q.count(h, e);
  __syncthreads();
  if ((int)threadIdx.x < q.D) p.counts[blockIdx.x * q.D + threadIdx.x] = h[threadIdx.x];
}
template <typename TOK>
__global__ void __launch_bounds__(kSortThreads, 1) emb_place_kernel(const SortArgs p, int pass) {
  extern __shared__ __align__(16) unsigned sm[];
  __shared__ unsigned wsum[kSortWarps], other[2][1 << kMaxBits];
  const Pass<TOK> q(p, pass, gridDim.x, blockIdx.x);
  unsigned *hist = sm, *base = hist + kSortWarps * q.D;
  unsigned *h = hist + q.warp * q.D;
  for (int i = q.lane; i < q.D; i += 32) h[i] = 0;
  __syncwarp();
  uint2 e[kAhead];
  q.count(h, e);
  // the counts of all CTAs and of those before this one, by two threads per
  // digit (the digits are at most half the threads)
  const int d = threadIdx.x & (q.D - 1), part = threadIdx.x / q.D, n = gridDim.x;
  unsigned before = 0, all = 0;
  if (part < 2) {
    const int to = part ? n : n / 2;
#pragma unroll 16
    for (int r = part ? n / 2 : 0; r < to; ++r) {
      const unsigned c = __ldcg(p.counts + r * q.D + d);
      if (r < (int)blockIdx.x) before += c;
      all += c;
    }
    if (part) other[0][d] = before, other[1][d] = all;
  }
  __syncthreads();
  if (part == 0) {
    before += other[0][d], all += other[1][d];
    q.over_warps(hist);
  }
  q.bases(base, wsum, part == 0 ? all : 0u, before);
  q.place(base, h, e);
}

// ------------------------------------------------------------------ sums of runs
struct SumArgs {
  const uint2 *pair;   // {key, position}, sorted
  const char *dout;
  char *dw;
  float *head, *tail;  // [pieces][D]: the part of a run that came in / goes on
  int64_t N, V, D, pieces;
  int slices;          // lane groups of a row, of lane_chunks a lane (joining: of one)
  int chunks;          // lane chunks of a row
  int64_t sum_blocks;  // CTAs of the sums; the others write zero rows
  int zero_ids;        // ids per warp there: 8 to 32, about 16 KB of rows
  Scale scale;
};

// The first entries with keys of at least key[0] and key[1] (N if none), by 32
// probes for each at a time.  Whole warp.
HS_DEV void first_entries(const SumArgs &p, const unsigned (&key)[2], int lane, int64_t (&a)[2]) {
  int64_t b[2] = {p.N, p.N};  // the answers lie in a..b
  a[0] = a[1] = 0;
  while (a[0] < b[0] || a[1] < b[1]) {
    int64_t by[2];
    bool under[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      by[i] = (b[i] - a[i] + 31) / 32;
      const int64_t j = a[i] + (lane + 1) * by[i] - 1;  // the last of each 32nd
      under[i] = j < b[i] && p.pair[j].x < key[i];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int below = __popc(__ballot_sync(0xffffffffu, under[i]));
      if (a[i] >= b[i]) continue;
      const int64_t from = a[i] + below * by[i];
      b[i] = min(b[i], from + by[i] - 1);
      a[i] = min(from, b[i]);
    }
  }
}

// Chunks per lane of the summing kernel: where odd rows keep the chunks small a
// lane takes several, 32 apart, so that what each entry costs is shared
// (gradient of 92769 tokens, 80727 x 841 float16: 180 us with one, 158 with four).
constexpr int lane_chunks(int bytes) { return bytes == 16 ? 1 : bytes == 8 ? 2 : 4; }

template <typename T, int BYTES>
__global__ void __launch_bounds__(256) emb_sum_kernel(const SumArgs p) {
  using C = typename Chunk<BYTES>::type;
  constexpr int E = BYTES / (int)sizeof(T), K = lane_chunks(BYTES);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row_bytes = p.D * (int64_t)sizeof(T);
  if ((int64_t)blockIdx.x >= p.sum_blocks) {
    // a few ids per warp: rows of those that do not occur
    const int64_t first = (((int64_t)blockIdx.x - p.sum_blocks) * 8 + warp) * p.zero_ids;
    if (first >= p.V) return;
    const unsigned end = (unsigned)min(p.V, first + p.zero_ids);
    unsigned none = 0xffffffffu >> (32 - (end - (unsigned)first));
    int64_t at[2];
    first_entries(p, {(unsigned)first, end}, lane, at);
    if (at[1] - at[0] <= 128) {
      for (int64_t i = at[0] + lane; i - lane < at[1]; i += 32)
        none &= ~__reduce_or_sync(0xffffffffu, i < at[1] ? 1u << (p.pair[i].x - (unsigned)first) : 0u);
    } else {  // frequent ids: a lane looks for each
      const unsigned id = (unsigned)first + lane;
      int64_t a = at[0], b = at[1];
      while (a < b) {
        const int64_t m = (a + b) / 2;
        if (p.pair[m].x < id) a = m + 1; else b = m;
      }
      none &= ~__ballot_sync(0xffffffffu, a < at[1] && p.pair[a].x == id);
    }
    const C zero = {};
    while (none) {
      const int r = __ffs(none) - 1;
      none &= none - 1;
      C *row = reinterpret_cast<C *>(p.dw + (first + r) * row_bytes);
      for (int c = lane; c < p.chunks; c += 32) row[c] = zero;
    }
    return;
  }
  const int64_t unit = (int64_t)blockIdx.x * 8 + warp;
  if (unit >= p.pieces * p.slices) return;
  const int64_t piece = unit / p.slices;
  const int chunk = (int)(unit - piece * p.slices) * (32 * K) + lane;  // and every 32nd after it
  const int64_t first = piece * kPiece, mine = first + lane;
  const unsigned none = (unsigned)p.V;
  const uint2 entry = mine < p.N ? p.pair[mine] : uint2{none, 0u};
  const unsigned key = entry.x, pos = entry.y;
  const unsigned prev = first > 0 ? p.pair[first - 1].x : none;
  const unsigned next = first + kPiece < p.N ? p.pair[first + kPiece].x : none;
  const int count = __popc(__ballot_sync(0xffffffffu, key != none));  // valid entries come first
  float acc[K][E];
#pragma unroll
  for (int q = 0; q < K; ++q)
#pragma unroll
    for (int e = 0; e < E; ++e) acc[q][e] = 0.f;
  unsigned cur = __shfl_sync(0xffffffffu, key, 0);
  bool from_prev = cur == prev;
  constexpr int U = 8;
  for (int j0 = 0; j0 < count; j0 += U) {
    C c[U][K];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned n = __shfl_sync(0xffffffffu, pos, (j0 + u) & 31);
      const char *src = p.dout + (int64_t)n * row_bytes + (int64_t)chunk * BYTES;
#pragma unroll
      for (int q = 0; q < K; ++q)
        if (chunk + 32 * q < p.chunks && j0 + u < count) c[u][q] = *reinterpret_cast<const C *>(src + 32 * BYTES * q);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j0 + u >= count) break;
#pragma unroll
      for (int q = 0; q < K; ++q) {
        float v[E];
        chunk_to_f32<T, BYTES>(c[u][q], v);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[q][e] += v[e];
      }
      const int j = j0 + u;
      const unsigned after = j + 1 < kPiece ? __shfl_sync(0xffffffffu, key, (j + 1) & 31) : next;
      if (after != cur || j + 1 == kPiece) {  // the run, or its part in this piece, ends here
        const bool goes_on = after == cur;
#pragma unroll
        for (int q = 0; q < K; ++q) {
          if (chunk + 32 * q < p.chunks) {
            if (from_prev || goes_on) {
              store_part<E>((from_prev ? p.head : p.tail) + piece * p.D + (int64_t)(chunk + 32 * q) * E, acc[q]);
            } else {
#pragma unroll
              for (int e = 0; e < E; ++e) acc[q][e] = scaled<T>(acc[q][e], p.scale);
              *reinterpret_cast<C *>(p.dw + (int64_t)cur * row_bytes + (int64_t)(chunk + 32 * q) * BYTES) = chunk_of_f32<T, BYTES>(acc[q]);
            }
          }
#pragma unroll
          for (int e = 0; e < E; ++e) acc[q][e] = 0.f;
        }
        cur = after;
        from_prev = false;
      }
    }
  }
}

// ------------------------------------------------------------------ crossing runs
// A warp per piece whose last run goes on into the next piece and began in
// this one: it adds the run's parts in order.  Runs over more than kLong
// pieces are left to the whole CTA, each warp adding a contiguous share.
constexpr int kJoinWarps = 16, kLong = 16;

template <typename T, int BYTES>
__global__ void __launch_bounds__(32 * kJoinWarps, 2) emb_join_kernel(const SumArgs p) {
  using C = typename Chunk<BYTES>::type;
  constexpr int E = BYTES / (int)sizeof(T);
  __shared__ float share[kJoinWarps][E][32];
  __shared__ int64_t long_first, long_last;
  __shared__ unsigned long_key;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t group = blockIdx.x / p.slices;
  const int chunk = (int)(blockIdx.x % p.slices) * 32 + lane;
  const bool live = chunk < p.chunks;
  const int64_t piece = group * kJoinWarps + warp;
  const unsigned none = (unsigned)p.V;
  if (threadIdx.x == 0) long_first = -1;
  __syncthreads();
  auto part = [&](const float *of, int64_t j, float *v) {
    if (live) {
      load_part<E>(of + j * p.D + (int64_t)chunk * E, v);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = 0.f;
    }
  };
  auto add_heads = [&](int64_t a, int64_t b, float *acc) {  // head parts of pieces a..b
    int64_t j = a;
    constexpr int U = E > 4 ? 4 : 8;
    for (; j + U <= b + 1; j += U) {
      float v[U][E];
#pragma unroll
      for (int u = 0; u < U; ++u) part(p.head, j + u, v[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += v[u][e];
    }
    for (; j <= b; ++j) {
      float v[E];
      part(p.head, j, v);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += v[e];
    }
  };
  auto write_row = [&](unsigned v, float *acc) {
    if (!live) return;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = scaled<T>(acc[e], p.scale);
    *reinterpret_cast<C *>(p.dw + (int64_t)v * p.D * (int64_t)sizeof(T) + (int64_t)chunk * BYTES) = chunk_of_f32<T, BYTES>(acc);
  };
  const int64_t end = (piece + 1) * kPiece;
  if (piece < p.pieces && end < p.N) {
    const unsigned k = p.pair[end - 1].x;
    const bool crosses = k != none && p.pair[end].x == k;
    const bool began = p.pair[piece * kPiece].x != k || piece == 0 || p.pair[piece * kPiece - 1].x != k;
    if (crosses && began) {
      // the run's last piece: the last whose first entry is still k (the pieces
      // of a run are consecutive), by 32 probes at a time, further and further
      // apart, then closer again
      auto probe = [&](int64_t from, int64_t by) {  // how many of from, from + by, .. (32 of them)
        const int64_t j = from + lane * by;
        return __popc(__ballot_sync(0xffffffffu, j < p.pieces && p.pair[j * kPiece].x == k));
      };
      int64_t last = piece, by = 1;
      int n = probe(piece + 1, 1);
      last += n;
      while (n == 32) {
        by *= 32;
        n = probe(last + by, by);
        last += n * by;
      }
      while (by > 1) {
        by /= 32;
        last += probe(last + by, by) * by;
      }
      if (last - piece <= kLong) {
        float acc[E];
        part(p.tail, piece, acc);
        add_heads(piece + 1, last, acc);
        write_row(k, acc);
      } else if (lane == 0) {
        long_first = piece;  // kJoinWarps <= kLong + 1 pieces hold the beginning of one such run at most
        long_last = last;
        long_key = k;
      }
    }
  }
  __syncthreads();
  if (long_first < 0) return;
  const int64_t n = long_last - long_first, per = (n + kJoinWarps - 1) / kJoinWarps;
  const int64_t a = long_first + 1 + warp * per, b = min(long_last, a + per - 1);
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (warp == 0) part(p.tail, long_first, acc);
  add_heads(a, b, acc);
#pragma unroll
  for (int e = 0; e < E; ++e) share[warp][e][lane] = acc[e];
  __syncthreads();
  if (warp == 0) {
    for (int w = 1; w < kJoinWarps; ++w)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += share[w][e][lane];
    write_row(long_key, acc);
  }
}

// ------------------------------------------------------------------ host side
// Tokens up to this many are sorted by one cluster.
constexpr int64_t kClusterSort = 16384;

struct Layout {
  size_t pair[2], counts, head, tail, total;
};
Layout layout(int64_t N, int64_t D) {
  Layout l;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += round_up(bytes, 256);
    return o;
  };
  for (int i = 0; i < 2; ++i) l.pair[i] = take((size_t)N * sizeof(uint2));
  l.counts = take(N > kClusterSort ? sizeof(unsigned) * kSortCtas << kMaxBits : 0);
  const size_t parts = (size_t)((N + kPiece - 1) / kPiece) * (size_t)D * sizeof(float);
  l.head = take(parts);
  l.tail = take(parts);
  l.total = at;
  return l;
}

// The widest lane chunk that divides the row and the alignments.
int chunk_bytes(int64_t row_bytes, std::initializer_list<const void *> ptrs, int64_t ld_bytes, size_t es) {
  int b = 16;
  auto fits = [&](int c) {
    if (row_bytes % c || ld_bytes % c) return false;
    for (const void *p : ptrs)
      if (!aligned(p, c)) return false;
    return true;
  };
  while (b > (int)es && !fits(b)) b /= 2;
  return b;
}

template <typename F> int by_chunk(int dtype, int bytes, F f) {
  auto at = [&](auto tag) -> int {
    using T = decltype(tag);
    if (bytes == 16) return f(tag, std::integral_constant<int, 16>{});
    if (bytes == 8) return f(tag, std::integral_constant<int, 8>{});
    if constexpr (sizeof(T) == 2)
      if (bytes == 2) return f(tag, std::integral_constant<int, 2>{});
    return f(tag, std::integral_constant<int, 4>{});
  };
  if (dtype == HS_F32) return at(float{});
  if (dtype == HS_BF16) return at(__nv_bfloat16{});
  return at(__half{});
}

int check_ids(const char *who, int dtype, int token_bits, const void *tokens, int64_t N, int64_t V, int64_t D,
              const int *status) {
  if (!dtype_ok(dtype)) return fail(HS_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
  if (token_bits != 32 && token_bits != 64) return fail(HS_ERR_INVALID_ARG, "%s: token_bits is 32 or 64", who);
  if (N < 0 || V < 0 || D < 0) return fail(HS_ERR_INVALID_ARG, "%s: negative N, V or D", who);
  if (N > 0x7fffffff || V > 0x7ffffffe) return fail(HS_ERR_UNSUPPORTED, "%s: N or V is 2^31 or more", who);
  if (N && (!tokens || !aligned(tokens, token_bits / 8))) return fail(HS_ERR_INVALID_ARG, "%s: null or misaligned tokens", who);
  if (!status) return fail(HS_ERR_INVALID_ARG, "%s: null dev_status", who);
  return HS_OK;
}

template <typename TOK> int sort(const SortArgs &s, cudaStream_t st) {
  constexpr size_t kWord = sizeof(unsigned);
  static std::atomic<unsigned long long> done{0}, done_place{0};
  if (s.N > kClusterSort) {
    const size_t smem = kWord * (kSortWarps + 1) << s.bits;
    if (int e = allow_dynamic_smem((const void *)emb_place_kernel<TOK>, kWord * (kSortWarps + 1) << kMaxBits, &done_place)) return e;
    const int ctas = (int)std::min<int64_t>(kSortCtas, (s.N + kSortThreads - 1) / kSortThreads);
    for (int pass = 0; pass < s.passes; ++pass) {
      emb_count_kernel<TOK><<<ctas, kSortThreads, 0, st>>>(s, pass);
      if (int e = check_launch("emb_count_kernel")) return e;
      emb_place_kernel<TOK><<<ctas, kSortThreads, smem, st>>>(s, pass);
      if (int e = check_launch("emb_place_kernel")) return e;
    }
    return HS_OK;
  }
  if (int e = allow_dynamic_smem((const void *)emb_sort_kernel<TOK>, kWord * (kSortWarps + kSortCluster + 1) << kMaxBits, &done)) return e;
  int cluster = 1;
  while (cluster < kSortCluster && (int64_t)cluster * kSortThreads < s.N) cluster *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = kWord * (kSortWarps + kSortCluster + 1) << s.bits;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  (void)cudaLaunchKernelEx(&cfg, emb_sort_kernel<TOK>, s);
  return check_launch("emb_sort_kernel");
}

}  // namespace
}  // namespace hs

extern "C" {

int hs_embedding_forward(int dtype, const void *weight, int64_t weight_ld, int token_bits, const void *tokens,
                         double scale, void *out, int64_t N, int64_t V, int64_t D, int *dev_status,
                         hs_stream_t stream) {
  using namespace hs;
  if (int e = check_ids("hs_embedding_forward", dtype, token_bits, tokens, N, V, D, dev_status)) return e;
  if (N == 0 || D == 0) return HS_OK;
  const size_t es = dtype_bytes(dtype);
  if ((V && !weight) || !out || !aligned(weight, es) || !aligned(out, es))
    return fail(HS_ERR_INVALID_ARG, "hs_embedding_forward: null or misaligned weight or out");
  if (weight_ld < D && V > 1) return fail(HS_ERR_INVALID_ARG, "hs_embedding_forward: weight_ld is below D");
  const int bytes = chunk_bytes(D * (int64_t)es, {weight, out}, V > 1 ? weight_ld * (int64_t)es : 0, es);
  const int64_t chunks = D * (int64_t)es / bytes, total = chunks * N, blocks = (total + 1023) / 1024;
  if (chunks > 0x7fff0000 || blocks > 0x7fffffff) return fail(HS_ERR_UNSUPPORTED, "hs_embedding_forward: N * D is too large");
  return by_chunk(dtype, bytes, [&](auto tag, auto b) -> int {
    using T = decltype(tag);
    constexpr int BYTES = decltype(b)::value;
    const char *w = (const char *)weight;
    const Scale sc = make_scale(scale);
    auto go = [&](auto *tok) {
      using TOK = std::remove_cv_t<std::remove_pointer_t<decltype(tok)>>;
      if constexpr (BYTES != 16) {
        if (chunks >= 96) {  // 100000 rows of 75 chunks: 22.6 us a warp per row, 21.5 by the kernel below; of 301 (60000): 19 and 42
          emb_lookup_rows_kernel<T, BYTES, TOK><<<(unsigned)((N + 7) / 8), 256, 0, (cudaStream_t)stream>>>(
              w, weight_ld * (int64_t)es, tok, sc, (char *)out, N, (int)chunks, V, dev_status);
          return;
        }
      }
      emb_lookup_kernel<T, BYTES, TOK><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(
          w, weight_ld * (int64_t)es, tok, sc, (char *)out, total, (int)chunks, V, dev_status);
    };
    if (token_bits == 64) go((const int64_t *)tokens); else go((const int *)tokens);
    return check_launch("emb_lookup_kernel");
  });
}

size_t hs_embedding_workspace_bytes(int64_t N, int64_t V, int64_t D) {
  if (N <= 0 || V <= 0 || D <= 0) return 0;
  return hs::layout(N, D).total;
}

int hs_embedding_backward(int dtype, const void *dout, int token_bits, const void *tokens, int64_t padding_idx,
                          double scale, void *dweight, int64_t N, int64_t V, int64_t D, void *workspace,
                          size_t workspace_bytes, int *dev_status, hs_stream_t stream) {
  using namespace hs;
  cudaStream_t st = (cudaStream_t)stream;
  if (int e = check_ids("hs_embedding_backward", dtype, token_bits, tokens, N, V, D, dev_status)) return e;
  if (V == 0 || D == 0) return HS_OK;
  const size_t es = dtype_bytes(dtype);
  if (!dweight || !aligned(dweight, es) || (N && !dout) || !aligned(dout, es))
    return fail(HS_ERR_INVALID_ARG, "hs_embedding_backward: null or misaligned dout or dweight");
  if (N == 0) {
    const cudaError_t e = cudaMemsetAsync(dweight, 0, (size_t)V * D * es, st);
    return e == cudaSuccess ? HS_OK : fail(HS_ERR_CUDA, "hs_embedding_backward: %s", cudaGetErrorString(e));
  }
  const Layout l = layout(N, D);
  if (!workspace || workspace_bytes < l.total || !aligned(workspace, 256))
    return fail(HS_ERR_WORKSPACE, "hs_embedding_backward: workspace %zu < %zu bytes, or not 256-byte aligned", workspace_bytes, l.total);
  char *ws = static_cast<char *>(workspace);

  SortArgs s = {};
  s.tok = tokens, s.N = N, s.V = V, s.pad = padding_idx, s.status = dev_status;
  for (int i = 0; i < 2; ++i) s.pair[i] = (uint2 *)(ws + l.pair[i]);
  int key_bits = 1;
  while ((V >> key_bits) != 0) ++key_bits;  // ids 0..V
  s.passes = (key_bits + kMaxBits - 1) / kMaxBits;
  s.bits = (key_bits + s.passes - 1) / s.passes;
  s.counts = (unsigned *)(ws + l.counts);
  if (int e = token_bits == 64 ? sort<int64_t>(s, st) : sort<int>(s, st)) return e;

  SumArgs p = {};
  p.pair = s.pair[(s.passes + 1) & 1];
  p.dout = (const char *)dout, p.dw = (char *)dweight;
  p.head = (float *)(ws + l.head), p.tail = (float *)(ws + l.tail);
  p.N = N, p.V = V, p.D = D, p.pieces = (N + kPiece - 1) / kPiece, p.scale = make_scale(scale);
  const int bytes = chunk_bytes(D * (int64_t)es, {dout, dweight}, 0, es);
  const int64_t chunks = D * (int64_t)es / bytes, wide = 32 * lane_chunks(bytes), slices = (chunks + wide - 1) / wide;
  p.sum_blocks = (p.pieces * slices + 7) / 8;
  p.zero_ids = 8;
  while (p.zero_ids < 32 && 2 * p.zero_ids * D * (int64_t)es <= 16384) p.zero_ids *= 2;
  const int64_t zero_blocks = (V + 8 * p.zero_ids - 1) / (8 * p.zero_ids), join_slices = (chunks + 31) / 32, join_blocks = (p.pieces + kJoinWarps - 1) / kJoinWarps * join_slices;
  if (chunks > 0x7fff0000 || p.sum_blocks + zero_blocks > 0x7fffffff || join_blocks > 0x7fffffff)
    return fail(HS_ERR_UNSUPPORTED, "hs_embedding_backward: N * D is too large");
  p.chunks = (int)chunks, p.slices = (int)slices;
  return by_chunk(dtype, bytes, [&](auto tag, auto b) -> int {
    using T = decltype(tag);
    constexpr int BYTES = decltype(b)::value;
    emb_sum_kernel<T, BYTES><<<(unsigned)(p.sum_blocks + zero_blocks), 256, 0, st>>>(p);
    if (int e = check_launch("emb_sum_kernel")) return e;
    if (p.pieces > 1) {
      SumArgs q = p;
      q.slices = (int)join_slices;
      emb_join_kernel<T, BYTES><<<(unsigned)join_blocks, 32 * kJoinWarps, 0, st>>>(q);
      return check_launch("emb_join_kernel");
    }
    return HS_OK;
  });
}

}  // extern "C"
