// Gated linear recurrence over time, forward and backward.
//
//   h_t = k_t f_t h_{t-1} + b_t,   k_t = 0 where a sequence starts, else 1
//   gated:  f_t = 1 / (1 + e^-z_t), b_t = (1 - f_t) x_t
//   linear: f_t and b_t are given
//
// A run of steps maps the state entering it to the state leaving it as
// h -> A h + B, and such maps compose, so the runs of a long sequence are
// summarised at once and only the maps are chained.  The backward is the same
// construction from the last step to the first on u_t = k_t f_t (g_t + u_{t+1}),
// the gradient reaching h_{t-1}:
//   e_t = g_t + u_{t+1},  dx_t = e_t (1 - f_t),  dz_t = e_t (k_t h_{t-1} - x_t) f_t (1 - f_t)
//   (linear: db_t = e_t,  df_t = e_t k_t h_{t-1}),  dh0 = u_0.
//
// Bound: memory.  The forward reads two words and writes one per element; the
// backward reads three (z, x, g) and writes two.  It does not read h: the
// forward keeps the float32 state entering each run of 16 steps (1/16 of a
// float32 tensor) and the backward recomputes the states inside the run from
// it, which moves less than reading h back and leaves no 16-bit rounding of h
// in the gradient.
//
// Split: a warp owns 16 consecutive steps of one 128-byte word row (32 lanes
// of one 32-bit word: 32 float32 or 64 16-bit columns).  The warps of a CTA
// stack along time, the CTAs of a cluster continue the stack, and a cluster
// walks the sequence in waves of 16 x warps x CTAs steps.  Each warp summarises its
// run, the maps meet in shared memory (distributed over the cluster), and
// every warp then knows its entering state and writes its outputs from the
// values it still holds, so every tensor is read and written once.  The order of
// operations follows from the shape, the tensors' strides and alignment, whether there are
// starts, and the device: a call gives the same bits each time, but not the same as one
// on another layout.  No CTA waits on one outside its own cluster.
//
// Measured on one B200, whose plain copy moves 6.53 TB/s: at T = 16384, B = 8,
// H = 1024 in bfloat16 the forward with its saved states takes 149 us (5.6 TB/s)
// and the backward 238 (5.8 TB/s), with starts 168 and 264; at T = 16384, B = 1 in
// float32 the forward takes 34 us (6.0 TB/s).  Per step of 64 bfloat16 columns the forward
// issues 43 instructions and the backward 64, two columns to a packed instruction
// where it can.
#include <float.h>

#include <algorithm>

#include <cuda.h>
#include <cudaTypedefs.h>

#include "lm_types.cuh"

// Arrays filled and read by fully unrolled loops read as "used before set" to
// the compiler's front end.
#pragma nv_diag_suppress 549

namespace hs {
namespace {

constexpr int kRun = 16;       // steps per warp and per saved state
constexpr int kFwdWarps = 16, kBwdWarps = 12;  // warps of an SM (128 and 168 registers a thread), of a CTA at most
constexpr int kMaxCluster = 8; // CTAs of a cluster along time
constexpr int kStages = 2;     // waves of inputs in shared memory
constexpr unsigned kStep = 128, kSlab = kRun * kStep;  // bytes of a step's words, and of a warp's run of one tensor

struct RecShape {
  int64_t T, n;         // steps; columns of one row
  int64_t groups;       // word-row groups of one row
  int nchunk;           // runs of 16 steps
  int waves;
  int cluster;
};

struct FwdArgs {
  RecShape s;
  const char *z, *x;
  char *h;
  const float *h0;
  float *h_n, *ckpt;
  const unsigned char *starts;
  unsigned *masks;                         // [chunks][B]: the starts of each run, for the backward
  int64_t masks_t;
  int64_t zt, zb, xt, xb, ht, hb, st, sb;  // strides in elements
  int64_t state_b;                         // row stride of h0 and h_n (columns)
  int64_t ckpt_t;                          // columns of one saved state (B * H)
  int *status;
  const char *ze, *xe;                     // ends of the tensors
  CUtensorMap zm, xm, hm;                  // where the tensors suit tiles
};

struct BwdArgs {
  RecShape s;
  const char *z, *x, *g;
  char *dz, *dx;
  const float *ckpt, *dh_n;
  float *dh0;
  const unsigned *starts;                  // [chunks][B], the forward's masks
  int64_t starts_t;
  int64_t zt, zb, xt, xb, gt, gb, dzt, dzb, dxt, dxb;
  int64_t state_b, ckpt_t;
  int *status;
  const char *ze, *xe, *ge;
  CUtensorMap zm, xm, gm, dzm, dxm;
};

HS_DEV unsigned smem_u32(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
HS_DEV void cp_async4(unsigned dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
HS_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> HS_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// The aligned forms are for a whole warp at once, whatever its lanes did before
// (polled a barrier, say, each for itself).
HS_DEV void cluster_arrive_relaxed() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
HS_DEV void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
HS_DEV void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
HS_DEV void fence_mbar_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
HS_DEV void mbar_init(uint64_t *b, int count = 1) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
HS_DEV void mbar_arrive(uint64_t *b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
HS_DEV void mbar_expect(uint64_t *b, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
// Bounded wait for a phase: past kWaitLimitNs the status word is set and the
// caller goes on (its results are void).  Once another wait has given up, this one
// lasts 10 ms more at most: the copies on their way have landed by then.
HS_DEV void mbar_wait(uint64_t *b, unsigned parity, int *status) {
  auto done = [&] {
    unsigned ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(b)), "r"(parity)
        : "memory");
    return ok != 0;
  };
  if (done()) return;
  const uint64_t t0 = globaltimer();
  unsigned n = 0;
  while (!done()) {
    if ((++n & 63u) == 0) {
      const uint64_t waited = globaltimer() - t0;
      if (waited > 10000000ull && ld_status(status) != 0) return;
      if (waited > kWaitLimitNs) {
        report(status, HS_ERR_DEVICE_TIMEOUT);
        return;
      }
    }
  }
}
HS_DEV unsigned cluster_addr(const void *p, int rank) {
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}

// A box of a [T][rows][columns] tensor into shared memory, counted on bar (out
// of range: zeros), and a warp's run back (out of range: dropped).
HS_DEV void tma_load(unsigned dst, const CUtensorMap *tm, uint64_t *bar, int col, int row, int t) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(tm), "r"(col), "r"(row), "r"(t), "r"(smem_u32(bar))
      : "memory");
}
HS_DEV void tma_store(const CUtensorMap *tm, unsigned src, int col, int row, int t) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(tm), "r"(col),
               "r"(row), "r"(t), "r"(src)
               : "memory");
}
HS_DEV void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
HS_DEV void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
HS_DEV void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// f = 1/(1+e^-z) and 1-f = e^-z/(1+e^-z), each to a few float32 ulps of its own
// size.  e^-z is held to 2^126, so that both stay finite (f is 2^-126 there and 1-f is 1;
// shut() makes such an f 0); a NaN stays one.  The reciprocal is refined by
// one Newton step (as in sigf: its rounding compounds over thousands of steps).
// gate_of() gives both from e^-z.
template <int VEC> HS_DEV void gate_of(Cols<VEC> e, Cols<VEC> &f, Cols<VEC> &om) {
  const Cols<VEC> nd = fma(e, Cols<VEC>::all(-1.f), Cols<VEC>::all(-1.f));  // -(1 + e^-z)
  float dd[VEC], r[VEC];
  nd.get(dd);
#pragma unroll
  for (int v = 0; v < VEC; ++v) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r[v]) : "f"(-dd[v]));
  const Cols<VEC> rr = Cols<VEC>::of(r);
  f = fma(rr, fma(nd, rr, Cols<VEC>::all(1.f)), rr);
  om = e * f;
}
template <int VEC> HS_DEV Cols<VEC> gate_exp(const float *z) {
  float t[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    float x = z[v] * -1.44269504088896341f;
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(126.f));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t[v]) : "f"(x));
  }
  return Cols<VEC>::of(t);
}
template <int VEC> HS_DEV void gate(const float *z, Cols<VEC> &f, Cols<VEC> &om) { gate_of<VEC>(gate_exp<VEC>(z), f, om); }

// Gates below float32's normal range are 0: nothing of the state passes, not even
// what would show beside an input of 0.
template <int VEC> HS_DEV Cols<VEC> shut(Cols<VEC> f) {
  float v[VEC];
  f.get(v);
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = v[i] <= FLT_MIN ? 0.f : v[i];
  return Cols<VEC>::of(v);
}
template <int VEC> HS_DEV Cols<VEC> least(Cols<VEC> a, Cols<VEC> b) {  // NaN left out
  float u[VEC], v[VEC];
  a.get(u);
  b.get(v);
#pragma unroll
  for (int i = 0; i < VEC; ++i) u[i] = fminf(u[i], v[i]);
  return Cols<VEC>::of(u);
}
// A product of gates, the least of them `low`: above 0 unless a gate is 0.
template <int VEC> HS_DEV Cols<VEC> open(Cols<VEC> a, Cols<VEC> low) {
  float u[VEC], v[VEC];
  a.get(u);
  low.get(v);
#pragma unroll
  for (int i = 0; i < VEC; ++i) u[i] = u[i] == 0.f && v[i] > 0.f ? 0x1p-149f : u[i];
  return Cols<VEC>::of(u);
}
template <int VEC> HS_DEV Cols<VEC> open(Cols<VEC> a) {  // of gates that are all above 0
  float u[VEC];
  a.get(u);
#pragma unroll
  for (int i = 0; i < VEC; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(u[i]) : "f"(0x1p-149f));
  return Cols<VEC>::of(u);
}
// Whether a product of gates is so small that one of them may be.
template <int VEC> HS_DEV bool tiny(Cols<VEC> a) {
  float v[VEC];
  a.get(v);
  bool r = false;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r |= v[i] <= FLT_MIN;
  return r;
}

// One lane's word of a step, copied by the lane itself.
template <typename T, int VEC> HS_DEV void fetch_word(unsigned dst, const char *src) {
  if constexpr (VEC == PerWord<T>::value) {
    cp_async4(dst, src);
  } else {  // one 16-bit value per lane: rows that are not 4-byte aligned
    const unsigned w = *reinterpret_cast<const unsigned short *>(src);
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(w) : "memory");
  }
}
HS_DEV unsigned read_raw(unsigned src) {
  unsigned w;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(src) : "memory");
  return w;
}
template <typename T, int VEC> HS_DEV void unpack_lane(unsigned w, float *v) {
  if constexpr (VEC == PerWord<T>::value) {
    unpack_word<T>(w, v);
  } else {
    float t[2];
    unpack_word<T>(w, t);
    v[0] = t[0];
  }
}
template <typename T, int VEC> HS_DEV void read_word(unsigned src, float *v) { unpack_lane<T, VEC>(read_raw(src), v); }
template <typename T> HS_DEV void stage_word(unsigned dst, const float *v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(pack_word<T>(v)) : "memory");
}
template <typename T, int VEC> HS_DEV void write_word(char *dst, const float *v) {
  if constexpr (VEC == PerWord<T>::value)
    *reinterpret_cast<unsigned *>(dst) = pack_word<T>(v);
  else
    *reinterpret_cast<T *>(dst) = from_f32<T>(v[0]);
}

// The map h -> a h + b of a run of steps, of one lane's columns.  a = -0 marks
// a run that a start lies in: nothing passes it, the map is b alone.  For a
// finite h that is what a h + b gives, so maps are chained without a look at the marks,
// and a chain of gates that ends in NaN is gone through once more with them (with a
// look at each: 80 us in place of 74 at T=16384, B=2, H=1024 float32).
template <int VEC> struct __align__(8 * VEC) Map {
  float a[VEC], b[VEC];
  HS_DEV bool cut() const { return __float_as_uint(a[0]) == 0x80000000u; }
};
template <int VEC> HS_DEV Cols<VEC> apply(const Map<VEC> &m, Cols<VEC> h) { return fma(Cols<VEC>::of(m.a), h, Cols<VEC>::of(m.b)); }
template <int VEC> HS_DEV Cols<VEC> apply_marked(const Map<VEC> &m, Cols<VEC> h) { return m.cut() ? Cols<VEC>::of(m.b) : apply(m, h); }
template <int VEC> HS_DEV bool any_nan(Cols<VEC> h) {
  float v[VEC];
  h.get(v);
  bool r = false;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r |= v[i] != v[i];
  return r;
}

// A product of gates is at most 1, and too small a one is as good as 0, as nothing
// grows again; but it is held to 2^-149 where no gate is 0, so that an infinite state
// stays one.  A product of given coefficients may be no float32 of full precision
// although the states are: growth by 1.5 a step takes 1e-20 to 1e25 in 256 steps, by
// a factor of 1e45.  Products are chained as they are all the same, and the states looked at:
//   - An infinite or NaN product leaves a state that is infinite or NaN, and so do
//     all maps after it.
//   - What a subnormal or vanished product loses is about 2^-149 of the state before
//     it: of states up to kNear below 2^-116, where steps would soon lose as much.
// Where a state along a chain is beyond kNear, infinite or NaN, the wave is chained once
// more with exact products, m 2^e with 1 <= |m| < 2 (resolve_exact; with states about 1e11
// in every wave 16384 x 8 x 1024 bfloat16 takes 250 us forward in place of 154).
constexpr float kNear = 4294967296.f;
template <int VEC> HS_DEV void largest(float &top, Cols<VEC> h) {
  float v[VEC];
  h.get(v);
#pragma unroll
  for (int i = 0; i < VEC; ++i) top = fmaxf(top, fabsf(v[i]));
}
// Of a chain whose states were at most `top`, NaN left out, and that ended in h.
template <int VEC> HS_DEV bool is_far(float top, Cols<VEC> h) {
  float v[VEC];
  h.get(v);
  bool r = !(top <= kNear);
#pragma unroll
  for (int i = 0; i < VEC; ++i) r |= !(fabsf(v[i]) <= kNear);
  return r;
}

// m 2^e; e = kAll: a map that a start lies in, of no product.
constexpr int kAll = 0x7fffffff;
template <int VEC> struct __align__(8 * VEC) Product {
  float m[VEC];
  int e[VEC];
};
// v = v' 2^x with 1 <= |v'| < 2; e becomes e + x.  Zeros, infinities and NaN stay.
HS_DEV void split(float &v, int &e) {
  const bool small = fabsf(v) < FLT_MIN;
  const unsigned w = __float_as_uint(small ? v * 16777216.f : v);
  const int x = (int)(w >> 23) & 255;
  if (x != 0 && x != 255) {
    v = __uint_as_float((w & 0x807fffffu) | 0x3f800000u);
    e += x - (small ? 127 + 24 : 127);
  }
}
HS_DEV float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
// m 2^e h + b.  Where m 2^e is a float32 of full precision, as a fused product and
// sum; else h is split too (beyond 2^252 and below 2^-252 the product is infinite and
// 0 in any case; zeros, infinities and NaN of m and h do as they would).
HS_DEV float exact_step(float m, int e, float h, float b) {
  if (e >= -126 && e <= 127) return fmaf(m * power_of_two(e), h, b);
  split(h, e);
  e = max(-252, min(252, e));
  return m * h * power_of_two(e / 2) * power_of_two(e - e / 2) + b;
}
template <int VEC> HS_DEV Cols<VEC> exact_step(const Product<VEC> &p, const float *b, Cols<VEC> h) {
  if (p.e[0] == kAll) return Cols<VEC>::of(b);
  float v[VEC];
  h.get(v);
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = exact_step(p.m[i], p.e[i], v[i], b[i]);
  return Cols<VEC>::of(v);
}
// The product of the 16 coefficients of a run: of four at a time in 64 bits, which no
// four float32 leave.
template <int VEC, typename F> HS_DEV Product<VEC> run_product(F coef) {
  Product<VEC> p;
#pragma unroll
  for (int i = 0; i < VEC; ++i) p.m[i] = 1.f, p.e[i] = 0;
#pragma unroll
  for (int k = 0; k < kRun; k += 4) {
    double d[VEC];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float c[VEC];
      coef(k + j).get(c);
#pragma unroll
      for (int i = 0; i < VEC; ++i) d[i] = j ? d[i] * (double)c[i] : (double)c[i];
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int hi = __double2hiint(d[i]), x = (hi >> 20) & 2047;
      if (x != 0 && x != 2047) {
        d[i] = __hiloint2double((hi & 0x800fffff) | 0x3ff00000, __double2loint(d[i]));
        p.e[i] += x - 1023;
      }
      p.m[i] *= (float)d[i];
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    split(p.m[i], p.e[i]);
    if (p.m[i] == 0.f || !(fabsf(p.m[i]) <= FLT_MAX)) p.e[i] = 0;
  }
  return p;
}

template <int VEC> struct __align__(4 * VEC) Exponent { int e[VEC]; };

// The maps of the warps of this CTA and of the CTAs of its cluster, each in
// two copies for alternate waves: a wave's barrier separates its writes from
// the reads of the wave two before.  The CTAs' maps arrive by asynchronous
// remote stores that complete on `bar`, so no warp waits for its own global
// stores.  A CTA sends the map of wave w+2 only after all of wave w+1 have
// arrived, and each of those was sent after its sender's last read of wave w.
template <int VEC> struct Maps {
  uint64_t *bar;   // [2], and two of the exact chains: the runs' products, the CTAs' maps
  Map<VEC> *warp;  // [2][warps][32]
  Map<VEC> *cta;   // [2][cluster][32], where the cluster has more than one CTA
  // of given coefficients, for a wave that is chained once more (one copy: a wave's
  // is done with before any warp publishes the next)
  Product<VEC> *run;   // [warps][32]
  Map<VEC> *exact;     // [cluster][32], m in the place of a
  Exponent<VEC> *pow;  // [cluster][32]
};
__host__ __device__ constexpr size_t maps_bytes(bool gated, int vec, int warps, int cluster) {
  return (size_t)32 * vec * (warps * (gated ? 16 : 24) + (cluster > 1 ? cluster * (gated ? 16 : 28) : 0));
}

// Sets up the maps behind the tiles; met by exchange_ready() before the first publish.
template <int VEC, bool GATED>
HS_DEV Maps<VEC> exchange_init(uint64_t *bar, unsigned char *behind, int warps, int warp, int lane, int cluster) {
  Maps<VEC> m;
  const int ctas = cluster > 1 ? cluster : 0;
  m.bar = bar;
  m.warp = reinterpret_cast<Map<VEC> *>(behind) + lane;
  m.cta = m.warp + 2 * warps * 32;
  m.exact = m.cta + 2 * ctas * 32;
  m.run = reinterpret_cast<Product<VEC> *>(m.exact - lane + ctas * 32) + lane;
  m.pow = reinterpret_cast<Exponent<VEC> *>(m.run - lane + warps * 32) + lane;
  if (warp == 0 && lane == 0) {
    if (cluster > 1) {
      mbar_init(&m.bar[0]);
      mbar_init(&m.bar[1]);
    }
    if (!GATED) {
      mbar_init(&m.bar[2], warps);
      mbar_init(&m.bar[3]);
    }
    if (cluster > 1 || !GATED) fence_mbar_init();
  }
  if (cluster > 1) cluster_arrive();
  return m;
}
HS_DEV void exchange_ready(int cluster) {
  if (cluster > 1) cluster_wait();  // every CTA has started and set up its barriers
}

HS_DEV void send(const void *p, int rank, const void *bar, const Map<2> &t) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(cluster_addr(p, rank)),
               "f"(t.a[0]), "f"(t.a[1]), "f"(t.b[0]), "f"(t.b[1]), "r"(cluster_addr(bar, rank))
               : "memory");
}
HS_DEV void send(const void *p, int rank, const void *bar, const Map<1> &t) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(cluster_addr(p, rank)),
               "f"(t.a[0]), "f"(t.b[0]), "r"(cluster_addr(bar, rank))
               : "memory");
}
HS_DEV void send(const void *p, int rank, const void *bar, const Exponent<2> &t) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.s32 [%0], {%1, %2}, [%3];" ::"r"(cluster_addr(p, rank)),
               "r"(t.e[0]), "r"(t.e[1]), "r"(cluster_addr(bar, rank))
               : "memory");
}
HS_DEV void send(const void *p, int rank, const void *bar, const Exponent<1> &t) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.s32 [%0], %1, [%2];" ::"r"(cluster_addr(p, rank)), "r"(t.e[0]),
               "r"(cluster_addr(bar, rank))
               : "memory");
}

// Publishes this warp's map of wave w.  SHUT: gates may be 0 (the forward's).
template <int VEC, bool GATED, bool STARTS, bool SHUT>
HS_DEV void publish(const Maps<VEC> &m, int w, int warps, int warp, int lane, int cluster, int rank, Cols<VEC> A, Cols<VEC> B,
                    bool cut) {
  const int p = w & 1;
  Map<VEC> mine;
  A.get(mine.a);
  B.get(mine.b);
  if (STARTS) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) mine.a[i] = cut ? -0.f : GATED ? mine.a[i] : mine.a[i] + 0.f;  // (a -0 by itself: +0)
  }
  const Map<VEC> *all = m.warp + p * warps * 32;
  m.warp[(p * warps + warp) * 32] = mine;
  __syncthreads();
  if (cluster == 1) return;
  if (warp == 0 && lane == 0) mbar_expect(&m.bar[p], cluster * 32 * (unsigned)sizeof(Map<VEC>));
  if (warp == warps - 1) {  // the CTA's map, to every CTA of the cluster
    Cols<VEC> ta = Cols<VEC>::all(1.f), tb = Cols<VEC>::all(0.f), least_a = ta;
    bool any = false;
    float top = 0.f, grown = 0.f, low = FLT_MAX;
#pragma unroll 4
    for (int j = 0; j < warps; ++j) {
      const Map<VEC> e = all[j * 32];
      if (STARTS) any |= e.cut();
      tb = apply(e, tb);
      ta = Cols<VEC>::of(e.a) * ta;
      if (GATED && SHUT) least_a = least<VEC>(least_a, Cols<VEC>::of(e.a));
      if (!GATED) {
        largest<VEC>(top, tb);
        largest<VEC>(grown, ta);
#pragma unroll
        for (int i = 0; i < VEC; ++i) low = fminf(low, fabsf(e.a[i]));
      }
    }
    if (GATED && STARTS && any && any_nan(tb)) {
      tb = Cols<VEC>::all(0.f);
      for (int j = 0; j < warps; ++j) tb = apply_marked(all[j * 32], tb);
    }
    if (GATED) ta = SHUT ? open<VEC>(ta, least_a) : open<VEC>(ta);
    Map<VEC> t;
    ta.get(t.a);
    tb.get(t.b);
    // (a state from before the CTA's steps that grows before a product loses it is not seen
    // in the states between CTAs)
    const bool again = !GATED && (is_far<VEC>(top, tb) || (grown > 1024.f && low < FLT_MIN));
#pragma unroll
    for (int i = 0; i < VEC; ++i) t.a[i] = again ? __int_as_float(0x7f800000) : any ? -0.f : STARTS && !GATED ? t.a[i] + 0.f : t.a[i];
    for (int r = 0; r < cluster; ++r) send(&m.cta[(p * cluster + rank) * 32], r, &m.bar[p], t);
  }
}

// Wave w's states with exact products: the state entering this warp's run, and
// in `state` the wave's entry moved to its end.  All warps of a cluster come here
// together, as all look at the same maps; should they not (a wait that gave up), the
// waits here end as all do.
template <int VEC, typename F>
HS_DEV Cols<VEC> resolve_exact(const Maps<VEC> &m, int w, int round, int warps, int warp, int lane, int cluster, int rank, bool cut, F coef,
                               Cols<VEC> &state, int *status) {
  const Map<VEC> *all = m.warp + (w & 1) * warps * 32;
  Product<VEC> mine = run_product<VEC>(coef);
  if (cut) mine.e[0] = kAll;
  m.run[warp * 32] = mine;
  __syncwarp();
  if (lane == 0) mbar_arrive(&m.bar[2]);
  mbar_wait(&m.bar[2], round & 1, status);
  auto runs = [&](int from, int to, Cols<VEC> h) {
#pragma unroll 1
    for (int j = from; j < to; ++j) h = exact_step<VEC>(m.run[j * 32], all[j * 32].b, h);
    return h;
  };
  if (cluster == 1) {
    const Cols<VEC> in = runs(0, warp, state);
    state = runs(warp, warps, in);
    return in;
  }
  if (warp == 0 && lane == 0) mbar_expect(&m.bar[3], cluster * 32 * (unsigned)(sizeof(Map<VEC>) + sizeof(Exponent<VEC>)));
  if (warp == warps - 1) {
    Map<VEC> t;
    Exponent<VEC> x;
    runs(0, warps, Cols<VEC>::all(0.f)).get(t.b);
#pragma unroll
    for (int i = 0; i < VEC; ++i) t.a[i] = 1.f, x.e[i] = 0;
    bool any = false;
#pragma unroll 1
    for (int j = 0; j < warps; ++j) {
      const Product<VEC> q = m.run[j * 32];
      any |= q.e[0] == kAll;
      if (any) break;
#pragma unroll
      for (int i = 0; i < VEC; ++i) t.a[i] *= q.m[i], x.e[i] += q.e[i];  // (up to 16 factors below 2)
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      split(t.a[i], x.e[i]);
      if (t.a[i] == 0.f || !(fabsf(t.a[i]) <= FLT_MAX)) x.e[i] = 0;
      if (any) x.e[i] = kAll;
    }
    for (int r = 0; r < cluster; ++r) {
      send(&m.exact[rank * 32], r, &m.bar[3], t);
      send(&m.pow[rank * 32], r, &m.bar[3], x);
    }
  }
  mbar_wait(&m.bar[3], round & 1, status);
  Cols<VEC> in = state;
#pragma unroll 1
  for (int r = 0; r < cluster; ++r) {
    if (r == rank) in = state;
    const Map<VEC> t = m.exact[r * 32];
    const Exponent<VEC> x = m.pow[r * 32];
    Product<VEC> q;
#pragma unroll
    for (int i = 0; i < VEC; ++i) q.m[i] = t.a[i], q.e[i] = x.e[i];
    state = exact_step<VEC>(q, t.b, state);
  }
  return runs(0, warp, in);
}

// (Lanes past the last column hold whatever lay in shared memory: what such values
// call for is not gone into.)
//
// The state entering this warp's run of wave w; `state`, the same in every
// thread of a column, moves from the wave's entry to its end.  `again`: the lanes
// that need the exact chain (of given coefficients).
template <int VEC, bool GATED, bool STARTS>
HS_DEV Cols<VEC> resolve(const Maps<VEC> &m, int w, int warps, int warp, int lane, int cluster, int rank, bool live, Cols<VEC> &state, bool &again, int *status) {
  const int p = w & 1;
  const Map<VEC> *all = m.warp + p * warps * 32;
  const Cols<VEC> entry = state;
  Cols<VEC> in = state;
  float top = 0.f;
  if (!GATED) largest<VEC>(top, state);
  if (cluster == 1) {
#pragma unroll 4
    for (int j = 0; j < warps; ++j) {
      if (j == warp) in = state;
      state = apply(all[j * 32], state);
      if (!GATED) largest<VEC>(top, state);
    }
    if (GATED && STARTS && live && any_nan(state)) {
      state = entry;
      for (int j = 0; j < warps; ++j) {
        if (j == warp) in = state;
        state = apply_marked(all[j * 32], state);
      }
    }
    again = !GATED && live && is_far<VEC>(top, state);
    return in;
  }
  mbar_wait(&m.bar[p], (w >> 1) & 1, status);
  const Map<VEC> *ctas = m.cta + p * cluster * 32;
#pragma unroll
  for (int r = 0; r < kMaxCluster; ++r) {
    if (r < cluster) {
      if (r == rank) in = state;
      state = apply(ctas[r * 32], state);
      if (!GATED) largest<VEC>(top, state);
    }
  }
#pragma unroll 4
  for (int j = 0; j < warp; ++j) in = apply(all[j * 32], in);
  if (GATED && STARTS && live && (any_nan(state) || any_nan(in))) {
    state = in = entry;
    for (int r = 0; r < cluster; ++r) {
      if (r == rank) in = state;
      state = apply_marked(ctas[r * 32], state);
    }
    for (int j = 0; j < warp; ++j) in = apply_marked(all[j * 32], in);
  }
  again = !GATED && live && is_far<VEC>(top, state);
  return in;
}

// The same, whatever the coefficients; `round` counts the exact chains.
template <int VEC, bool GATED, bool STARTS, typename F>
HS_DEV Cols<VEC> enter(const Maps<VEC> &m, int w, int &round, int warps, int warp, int lane, int cluster, int rank, bool live, bool cut, F coef,
                       Cols<VEC> &state, int *status) {
  Cols<VEC> entry = state;
  bool again;
  Cols<VEC> in = resolve<VEC, GATED, STARTS>(m, w, warps, warp, lane, cluster, rank, live, state, again, status);
  if constexpr (!GATED) {
    if (__any_sync(0xffffffffu, again)) {
      const Cols<VEC> exact = resolve_exact<VEC>(m, w, round, warps, warp, lane, cluster, rank, cut, coef, entry, status);
      if (again) in = exact, state = entry;
      ++round;
    }
  }
  return in;
}

template <int VEC> HS_DEV void load_state(const float *p, int64_t at, float *v) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = p ? p[at + i] : 0.f;
}

// ------------------------------------------------------------------ inputs
// How tensors move.  kTiles: a tile of all warps' runs comes in by one TMA copy
// per tensor and each run leaves by one (bases and strides multiples of 16
// bytes).  kRows: each lane of a warp copies one step's words of the warp's run,
// the 16-byte granules that they lie in, by one bulk copy (rows 4-byte aligned).
// kLanes: each lane copies and reads its own words (a single run, where copies
// that signal a barrier take longer; rows that are only 2-byte aligned; many
// columns, as an SM starts one row copy in about 17 cycles).
enum { kLanes, kTiles, kRows };
constexpr unsigned step_bytes(int move) { return move == kRows ? kStep + 16 : kStep; }
constexpr unsigned slab_bytes(int move) { return kRun * step_bytes(move); }

// Shared memory of a CTA: kStages x [N tensors][warps][16 steps] of inputs,
// then [outputs][warps][16 steps] with kTiles.
template <int MOVE, int N> struct Inputs {
  unsigned base, tensor;  // this lane's first word of its slab; bytes between tensors
  uint64_t *full;         // [kStages], with kRows [kStages][warps]
  int *status;
  int warp, warps;
  HS_DEV unsigned at(int w) const { return base + (unsigned)(w % kStages) * (N * tensor); }
  HS_DEV uint64_t *bar(int w) const { return full + (w % kStages) * (MOVE == kRows ? warps : 1) + (MOVE == kRows ? warp : 0); }
  // Waits until wave w is there; a warp's lanes, which poll each for itself, go on together.
  HS_DEV void wait(int w) const {
    if constexpr (MOVE == kLanes) {
      cp_wait<kStages - 1>();
    } else {
      mbar_wait(bar(w), (w / kStages) & 1, status);
      __syncwarp();
    }
  }
};

// Where a step's words begin in their 16-byte granule, for the row segment of
// a warp (the first of its words at `at` elements from base; 16 steps of any
// stride are whole granules, so every run begins alike).
template <typename T, int MOVE> struct Shift {
  unsigned o, r;
  HS_DEV Shift(const char *base, int64_t at, int64_t stride)
      : o((unsigned)(reinterpret_cast<uintptr_t>(base) + (uintptr_t)at * sizeof(T))), r((unsigned)(stride * (int64_t)sizeof(T))) {}
  HS_DEV unsigned operator()(int k) const { return MOVE == kRows ? (o + k * r) & 15 : 0; }
};

// Copies the granules of `bytes` bytes at src, but none past the tensor's end;
// what is left of the last one by the lane itself.  Returns the bytes that the
// barrier is to expect.
template <typename T> HS_DEV unsigned copy_row(unsigned dst, const char *src, unsigned bytes, const char *end, uint64_t *bar) {
  const char *from = reinterpret_cast<const char *>(reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15);
  unsigned size = (unsigned)(src + bytes - from + 15) & ~15u;
  if (from + size > end) {
    size -= 16;
    const char *q = from + size < src ? src : from + size;
    for (; q < src + bytes; q += sizeof(T)) {
      if constexpr (sizeof(T) == 4)
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + (unsigned)(q - from)), "r"(*reinterpret_cast<const unsigned *>(q)) : "memory");
      else
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + (unsigned)(q - from)), "h"(*reinterpret_cast<const unsigned short *>(q)) : "memory");
    }
    fence_async();  // these stores before the bulk copies that fill the place in later waves (the backward's)
  }
  if (size)
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(from),
                 "r"(size), "r"(smem_u32(bar))
                 : "memory");
  return size;
}

// The starts among the 16 steps of each of a warp's next 32 waves, as bits, one
// wave per lane.  Read wave by wave, the load's latency showed in every one of
// them (25% of the forward's time, 40% of the backward's).  The two halves of
// the warp read the steps of two waves at a time (neighbours in memory, where a lane
// per wave touched 32 lines a load).
// The forward leaves the masks with the saved states: the backward loads one
// word per run in place of 16 bytes (257 -> 244 us at T=16384, B=8, H=1024 bf16).
template <typename F>
HS_DEV unsigned start_masks(const unsigned char *starts, int64_t stride, int w, int waves, int lane, int64_t T, F start_of) {
  unsigned m = 0;
  bool cut[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int wave = w + 2 * j + lane / 16;
    const int64_t t = start_of(wave) + lane % 16;
    cut[j] = wave < waves && t < T && starts[t * stride] != 0;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const unsigned two = __ballot_sync(0xffffffffu, cut[j]);
    if (lane / 2 == j) m = lane & 1 ? two >> 16 : two & 0xffffu;
  }
  return m;
}

HS_DEV void barriers_init(uint64_t *full, int n, int warp, int lane) {
  if (warp == 0 && lane == 0) {
    for (int i = 0; i < n; ++i) mbar_init(full + i);
    fence_mbar_init();
    fence_async();
  }
  __syncthreads();
}

// ------------------------------------------------------------------ forward
template <typename T, int VEC, bool GATED, bool STARTS, int MOVE>
__global__ void __launch_bounds__(32 * kFwdWarps, 1) rec_fwd_kernel(const __grid_constant__ FwdArgs p) {
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ uint64_t full[kStages * kFwdWarps], swap[4];
  using C = Cols<VEC>;
  const int lane = threadIdx.x, warp = threadIdx.y, warps = blockDim.y;
  const int cluster = p.s.cluster, rank = (int)(blockIdx.x % cluster), waves = p.s.waves;
  const int64_t gid = blockIdx.x / cluster;
  const int64_t row = gid / p.s.groups;
  const int64_t col0 = (gid % p.s.groups) * 32 * VEC;
  int64_t col = col0 + lane * VEC;
  const bool live = col < p.s.n;  // VEC > 1 only where n is a multiple of VEC
  if (!live) col = p.s.n - VEC;   // reads what a live lane reads, writes nothing
  const int64_t T_ = p.s.T;
  constexpr unsigned kPitch = step_bytes(MOVE);
  Inputs<MOVE, 2> in;
  in.tensor = warps * slab_bytes(MOVE), in.full = full, in.status = p.status, in.warp = warp, in.warps = warps;
  in.base = smem_u32(dyn) + warp * slab_bytes(MOVE) + lane * 4;
  const Shift<T, MOVE> zsh(p.z, row * p.zb + col0, p.zt), xsh(p.x, row * p.xb + col0, p.xt);
  const unsigned slab = in.base + kStages * 2 * in.tensor;  // this lane's words of the outputs

  auto start_of = [&](int w) { return ((int64_t)(w * cluster + rank) * warps + warp) * kRun; };
  auto fetch = [&](int w) {
    if constexpr (MOVE == kRows) {
      if (w < waves) {  // lanes 0..15 the steps of z, 16..31 those of x
        const int64_t t = start_of(w) + lane % 16;
        const bool x = lane >= 16;
        const unsigned bytes = (unsigned)min((int64_t)kStep, (p.s.n - col0) * (int64_t)sizeof(T));
        unsigned size = 0;
        if (t < T_) {
          const int64_t at = row * (x ? p.xb : p.zb) + col0 + t * (x ? p.xt : p.zt);
          size = copy_row<T>(in.at(w) - lane * 4 + (x ? in.tensor : 0u) + lane % 16 * kPitch, (x ? p.x : p.z) + at * (int64_t)sizeof(T), bytes,
                             x ? p.xe : p.ze, in.bar(w));
        }
        size = __reduce_add_sync(0xffffffffu, size);
        if (lane == 0) mbar_expect(in.bar(w), size);
        __syncwarp();
      }
    } else if constexpr (MOVE == kTiles) {
      if (warp == 0 && lane == 0 && w < waves) {
        uint64_t *bar = in.bar(w);
        const unsigned d = in.at(w);
        const int t = (int)start_of(w);
        mbar_expect(bar, 2 * in.tensor);
        tma_load(d, &p.zm, bar, (int)col0, (int)row, t);
        tma_load(d + in.tensor, &p.xm, bar, (int)col0, (int)row, t);
      }
    } else {
      if (w < waves) {
        const int64_t t0 = start_of(w), zs = p.zt * (int64_t)sizeof(T), xs = p.xt * (int64_t)sizeof(T);
        const unsigned d = in.at(w);
        const char *zq = p.z + (row * p.zb + col) * (int64_t)sizeof(T) + t0 * zs;
        const char *xq = p.x + (row * p.xb + col) * (int64_t)sizeof(T) + t0 * xs;
        if (t0 + kRun <= T_) {
#pragma unroll
          for (int k = 0; k < kRun; ++k, zq += zs, xq += xs) {
            fetch_word<T, VEC>(d + k * kStep, zq);
            fetch_word<T, VEC>(d + in.tensor + k * kStep, xq);
          }
        } else {
#pragma unroll 1
          for (int k = 0; k < kRun && t0 + k < T_; ++k, zq += zs, xq += xs) {
            fetch_word<T, VEC>(d + k * kStep, zq);
            fetch_word<T, VEC>(d + in.tensor + k * kStep, xq);
          }
        }
      }
      cp_commit();
    }
  };
  auto starts_from = [&](int w) { return start_masks(p.starts + row * p.sb, p.st, w, waves, lane, T_, start_of); };

  const Maps<VEC> maps = exchange_init<VEC, GATED>(swap, dyn + (kStages * 2 + (MOVE == kTiles ? 1 : 0)) * in.tensor, warps, warp, lane, cluster);
  if (MOVE != kLanes) barriers_init(full, kStages * (MOVE == kRows ? warps : 1), warp, lane);
  fetch(0);
  fetch(1);
  unsigned masks = 0;
  float s0[VEC];
  load_state<VEC>(p.h0, row * p.state_b + col, s0);
  C state = C::of(s0);
  int round = 0;

  for (int w = 0; w < waves; ++w) {
    const int64_t t0 = start_of(w);
    const int len = (int)max((int64_t)0, min((int64_t)kRun, T_ - t0));
    unsigned mask = 0;
    if (STARTS) {
      if (w % 32 == 0) masks = starts_from(w);
      mask = __shfl_sync(0xffffffffu, masks, w % 32);
      if (p.masks && col0 == 0 && lane == 0 && len > 0) p.masks[(t0 / kRun) * p.masks_t + row] = mask;
    }
    in.wait(w);
    const unsigned d = in.at(w);
    C f[kRun], b[kRun];
    C A = C::all(1.f), B = C::all(0.f);
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      float zv[VEC], xv[VEC];
      read_word<T, VEC>(d + zsh(k) + k * kPitch, zv);
      read_word<T, VEC>(d + in.tensor + xsh(k) + k * kPitch, xv);
      if (GATED) {
        C om;
        gate<VEC>(zv, f[k], om);
        b[k] = om * C::of(xv);
      } else {
        f[k] = C::of(zv);
        b[k] = C::of(xv);
      }
    }
    if (len < kRun) {
#pragma unroll
      for (int k = 0; k < kRun; ++k)
        if (k >= len) f[k] = C::all(1.f), b[k] = C::all(0.f);
    }
    if (STARTS && mask) {
#pragma unroll
      for (int k = 0; k < kRun; ++k) {
        const bool cut = (mask >> k) & 1;
        if (GATED) f[k] = shut<VEC>(f[k]);
        A = cut ? C::all(0.f) : A * f[k];
        B = cut ? b[k] : fma(f[k], B, b[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kRun; ++k) {
        A = A * f[k];
        B = fma(f[k], B, b[k]);
      }
      if (GATED && live && tiny<VEC>(A)) {
        A = C::all(1.f), B = C::all(0.f);
        C low = A;
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
          f[k] = shut<VEC>(f[k]);
          A = A * f[k];
          B = fma(f[k], B, b[k]);
          low = least<VEC>(low, f[k]);
        }
        A = open<VEC>(A, low);
      }
    }
    if (w == 0) exchange_ready(cluster);
    // (every warp has read its inputs once all have published)
    publish<VEC, GATED, STARTS, true>(maps, w, warps, warp, lane, cluster, rank, A, B, mask != 0);
    fetch(w + kStages);
    C h = enter<VEC, GATED, STARTS>(maps, w, round, warps, warp, lane, cluster, rank, live, mask != 0, [&](int k) { return f[k]; }, state, p.status);
    if (len > 0) {
      if (p.ckpt && live) {
        float *c = p.ckpt + (t0 / kRun) * p.ckpt_t + row * p.state_b + col;
        float v[VEC];
        h.get(v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) c[i] = v[i];
      }
      if constexpr (MOVE == kTiles) {
        if (lane == 0) bulk_wait_read();  // the previous wave's copy has left the slab
        __syncwarp();
      }
      const int64_t hs = p.ht * (int64_t)sizeof(T);
      char *hq = p.h + (row * p.hb + col) * (int64_t)sizeof(T) + t0 * hs;
      auto put = [&](int k, bool cut) {
        h = cut ? b[k] : fma(f[k], h, b[k]);
        float v[VEC];
        h.get(v);
        if constexpr (MOVE == kTiles) {
          stage_word<T>(slab + k * kStep, v);
        } else {
          if (live && k < len) write_word<T, VEC>(hq, v);
          hq += hs;
        }
      };
      if (STARTS && mask) {
#pragma unroll
        for (int k = 0; k < kRun; ++k) put(k, (mask >> k) & 1);
      } else {
#pragma unroll
        for (int k = 0; k < kRun; ++k) put(k, false);
      }
      if constexpr (MOVE == kTiles) {
        fence_async();
        __syncwarp();
        if (lane == 0) {
          tma_store(&p.hm, slab, (int)col0, (int)row, (int)t0);
          bulk_commit();
        }
      }
    }
  }
  if (MOVE == kTiles && lane == 0) bulk_wait_read();
  // no CTA leaves before the others are done with its memory, nor is the last state
  // written where it takes the place of the first before all have read that
  if (cluster > 1) {
    if (p.h_n && p.h_n == p.h0) cluster_arrive(); else cluster_arrive_relaxed();  // (to release waits for all outputs, 1 us)
    cluster_wait();
  }
  if (p.h_n && live && rank == 0 && warp == 0) {
    float v[VEC];
    state.get(v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) p.h_n[row * p.state_b + col + i] = v[i];
  }
}

// ------------------------------------------------------------------ backward
template <typename T, int VEC, bool GATED, bool STARTS, int MOVE>
__global__ void __launch_bounds__(32 * kBwdWarps, 1) rec_bwd_kernel(const __grid_constant__ BwdArgs p) {
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ uint64_t full[kStages * kBwdWarps], swap[4];
  using C = Cols<VEC>;
  // float32 keeps both f and 1-f.  The 16-bit types have registers for one value (two
  // columns to a lane, or as many loads on their way) and keep e^-z, from which
  // gate_of() gives both again, the same bits (1-f alone would leave f with the error
  // 2^-25, all of a small gate)
  constexpr bool kBoth = GATED && sizeof(T) == 4, kExp = GATED && sizeof(T) == 2;
  const int lane = threadIdx.x, warp = threadIdx.y, warps = blockDim.y;
  const int cluster = p.s.cluster, rank = (int)(blockIdx.x % cluster), waves = p.s.waves;
  const int64_t gid = blockIdx.x / cluster;
  const int64_t row = gid / p.s.groups;
  const int64_t col0 = (gid % p.s.groups) * 32 * VEC;
  int64_t col = col0 + lane * VEC;
  const bool live = col < p.s.n;
  if (!live) col = p.s.n - VEC;
  const int64_t T_ = p.s.T;
  const bool has_g = p.g != nullptr;
  constexpr unsigned kPitch = step_bytes(MOVE);
  Inputs<MOVE, 3> in;
  in.tensor = warps * slab_bytes(MOVE), in.full = full, in.status = p.status, in.warp = warp, in.warps = warps;
  // warps go back in time, so the first warp's run is the last of a tile
  in.base = smem_u32(dyn) + (warps - 1 - warp) * slab_bytes(MOVE) + lane * 4;
  const Shift<T, MOVE> zsh(p.z, row * p.zb + col0, p.zt), xsh(p.x, row * p.xb + col0, p.xt), gsh(p.g, row * p.gb + col0, p.gt);
  const unsigned slab = in.base + kStages * 3 * in.tensor;

  // chunks from the last to the first; below 0: past the beginning, nothing
  auto chunk_of = [&](int w) { return p.s.nchunk - 1 - ((w * cluster + rank) * warps + warp); };
  auto fetch = [&](int w) {
    if constexpr (MOVE == kRows) {
      if (w < waves) {  // lanes 0..15 the steps of z, 16..31 those of x, then 0..15 those of g
        const int c = chunk_of(w);
        const int64_t t = (int64_t)c * kRun + lane % 16;
        const unsigned bytes = (unsigned)min((int64_t)kStep, (p.s.n - col0) * (int64_t)sizeof(T));
        const unsigned d = in.at(w) - lane * 4 + lane % 16 * kPitch;
        const bool x = lane >= 16;
        unsigned size = 0;
        if (c >= 0 && t < T_) {
          const int64_t at = row * (x ? p.xb : p.zb) + col0 + t * (x ? p.xt : p.zt);
          size = copy_row<T>(d + (x ? in.tensor : 0u), (x ? p.x : p.z) + at * (int64_t)sizeof(T), bytes, x ? p.xe : p.ze, in.bar(w));
          if (!x && has_g)
            size += copy_row<T>(d + 2 * in.tensor, p.g + (row * p.gb + col0 + t * p.gt) * (int64_t)sizeof(T), bytes, p.ge, in.bar(w));
        }
        size = __reduce_add_sync(0xffffffffu, size);
        if (lane == 0) mbar_expect(in.bar(w), size);
        __syncwarp();
      }
    } else if constexpr (MOVE == kTiles) {
      if (warp == warps - 1 && lane == 0 && w < waves) {  // (the warp whose slab is the tile's first)
        uint64_t *bar = in.bar(w);
        const unsigned d = in.at(w);
        const int t = chunk_of(w) * kRun;  // negative in the last wave's tail: zeros
        mbar_expect(bar, (has_g ? 3 : 2) * in.tensor);
        tma_load(d, &p.zm, bar, (int)col0, (int)row, t);
        tma_load(d + in.tensor, &p.xm, bar, (int)col0, (int)row, t);
        if (has_g) tma_load(d + 2 * in.tensor, &p.gm, bar, (int)col0, (int)row, t);
      }
    } else {
      const int c = w < waves ? chunk_of(w) : -1;
      if (c >= 0) {
        const int64_t t0 = (int64_t)c * kRun;
        const int64_t zs = p.zt * (int64_t)sizeof(T), xs = p.xt * (int64_t)sizeof(T), gs = p.gt * (int64_t)sizeof(T);
        const unsigned d = in.at(w);
        const char *zq = p.z + (row * p.zb + col) * (int64_t)sizeof(T) + t0 * zs;
        const char *xq = p.x + (row * p.xb + col) * (int64_t)sizeof(T) + t0 * xs;
        const char *gq = p.g + (row * p.gb + col) * (int64_t)sizeof(T) + t0 * gs;
        if (t0 + kRun <= T_ && has_g) {
#pragma unroll
          for (int k = 0; k < kRun; ++k, zq += zs, xq += xs, gq += gs) {
            fetch_word<T, VEC>(d + k * kStep, zq);
            fetch_word<T, VEC>(d + in.tensor + k * kStep, xq);
            fetch_word<T, VEC>(d + 2 * in.tensor + k * kStep, gq);
          }
        } else {
#pragma unroll 1
          for (int k = 0; k < kRun && t0 + k < T_; ++k, zq += zs, xq += xs, gq += gs) {
            fetch_word<T, VEC>(d + k * kStep, zq);
            fetch_word<T, VEC>(d + in.tensor + k * kStep, xq);
            if (has_g) fetch_word<T, VEC>(d + 2 * in.tensor + k * kStep, gq);
          }
        }
      }
      cp_commit();
    }
  };
  auto starts_from = [&](int w) {
    const int c = chunk_of(w + lane);
    return w + lane < waves && c >= 0 ? p.starts[c * p.starts_t + row] : 0u;
  };
  auto fetch_ckpt = [&](int w, float *h) {
    const int c = w < waves ? chunk_of(w) : -1;
    load_state<VEC>(c >= 0 ? p.ckpt : nullptr, c * p.ckpt_t + row * p.state_b + col, h);
  };

  const Maps<VEC> maps = exchange_init<VEC, GATED>(swap, dyn + (kStages * 3 + (MOVE == kTiles ? 2 : 0)) * in.tensor, warps, warp, lane, cluster);
  if (MOVE != kLanes) barriers_init(full, kStages * (MOVE == kRows ? warps : 1), warp, lane);
  fetch(0);
  fetch(1);
  float next_h[VEC], s0[VEC];
  fetch_ckpt(0, next_h);
  unsigned masks = 0;
  load_state<VEC>(p.dh_n, row * p.state_b + col, s0);
  C state = C::of(s0);
  int round = 0;
  const C one = C::all(1.f), zero = C::all(0.f);

  for (int w = 0; w < waves; ++w) {
    unsigned mask = 0;
    if (STARTS) {
      if (w % 32 == 0) masks = starts_from(w);
      mask = __shfl_sync(0xffffffffu, masks, w % 32);
    }
    C s = C::of(next_h);
    fetch_ckpt(w + 1, next_h);
    in.wait(w);
    const int c = chunk_of(w);
    const int64_t t0 = (int64_t)c * kRun;
    const unsigned d = in.at(w);
    const int len = c < 0 ? 0 : (int)min((int64_t)kRun, T_ - t0);
    // keep: 1-f, with kExp e^-z (gated) or f (linear); q: the factor of e in df; raw: g as stored
    C keep[kRun], both[kBoth ? kRun : 1], q[kRun];
    unsigned raw[kRun];
    auto coef = [&](int k) {
      if constexpr (kExp) {
        C f, om;
        gate_of<VEC>(keep[k], f, om);
        return f;
      }
      return kBoth ? both[kBoth ? k : 0] : keep[k];
    };
    auto grad = [&](int k) {
      float g[VEC];
      unpack_lane<T, VEC>(raw[k], g);
      return C::of(g);
    };
    C A = one, B = zero;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      float zv[VEC], xv[VEC];
      read_word<T, VEC>(d + zsh(k) + k * kPitch, zv);
      read_word<T, VEC>(d + in.tensor + xsh(k) + k * kPitch, xv);
      raw[k] = has_g ? read_raw(d + 2 * in.tensor + gsh(k) + k * kPitch) : 0u;
      const C x = C::of(xv);
      if (STARTS && ((mask >> k) & 1)) s = zero;
      if (GATED) {
        const C e = gate_exp<VEC>(zv);
        C f, om;
        gate_of<VEC>(e, f, om);
        q[k] = (s - x) * (f * om);
        s = fma(f, s, om * x);
        keep[k] = kExp ? e : om;
        if (kBoth) both[k] = f;
        if (kExp) {  // the run's map while f is at hand: B = sum of g_k f_0 .. f_k, up to a start
          A = STARTS && ((mask >> k) & 1) ? zero : A * f;
          B = fma(A, grad(k), B);
        }
      } else {
        q[k] = s;
        keep[k] = C::of(zv);
        s = fma(keep[k], s, x);
      }
    }
    if (len < kRun) {
#pragma unroll
      for (int k = 0; k < kRun; ++k) {
        if (k >= len) {
          keep[k] = GATED ? zero : one;
          if (kBoth) both[k] = one;
          raw[k] = 0;
        }
      }
    }
    // (what a step at a time gives: a part of a run, and gradients that are infinite or NaN)
    const bool steps = !kExp || len < kRun || (live && any_nan(B));
    if (steps) A = one, B = zero;
    if (STARTS && mask && steps) {
#pragma unroll
      for (int k = kRun - 1; k >= 0; --k) {
        const bool cut = (mask >> k) & 1;
        B = cut ? zero : coef(k) * (grad(k) + B);
        A = cut ? zero : A * coef(k);
      }
    } else if (steps) {
#pragma unroll
      for (int k = kRun - 1; k >= 0; --k) {
        const C f = coef(k);
        B = f * (grad(k) + B);
        A = A * f;
      }
    }
    if (GATED) A = open<VEC>(A);  // (2^-126 at least)
    if (w == 0) exchange_ready(cluster);
    publish<VEC, GATED, STARTS, false>(maps, w, warps, warp, lane, cluster, rank, A, B, mask != 0);
    fetch(w + kStages);
    C u = enter<VEC, GATED, STARTS>(maps, w, round, warps, warp, lane, cluster, rank, live, mask != 0, coef, state, p.status);
    if (len > 0) {
      if constexpr (MOVE == kTiles) {
        if (lane == 0) bulk_wait_read();
        __syncwarp();
      }
      const int64_t dzs = p.dzt * (int64_t)sizeof(T), dxs = p.dxt * (int64_t)sizeof(T);
      char *dzq = p.dz + (row * p.dzb + col) * (int64_t)sizeof(T) + (t0 + kRun - 1) * dzs;
      char *dxq = p.dx + (row * p.dxb + col) * (int64_t)sizeof(T) + (t0 + kRun - 1) * dxs;
      auto put = [&](int k, bool cut) {
        const C e = grad(k) + u;
        C f = kExp ? zero : coef(k), om = keep[k];
        if (kExp) gate_of<VEC>(keep[k], f, om);
        u = cut ? zero : f * e;
        float dz[VEC], dx[VEC];
        (e * q[k]).get(dz);
        (GATED ? e * om : e).get(dx);
        if constexpr (MOVE == kTiles) {
          stage_word<T>(slab + k * kStep, dz);
          stage_word<T>(slab + in.tensor + k * kStep, dx);
        } else {
          if (live && k < len) {
            write_word<T, VEC>(dzq, dz);
            write_word<T, VEC>(dxq, dx);
          }
          dzq -= dzs;
          dxq -= dxs;
        }
      };
      if (STARTS && mask) {
#pragma unroll
        for (int k = kRun - 1; k >= 0; --k) put(k, (mask >> k) & 1);
      } else {
#pragma unroll
        for (int k = kRun - 1; k >= 0; --k) put(k, false);
      }
      if constexpr (MOVE == kTiles) {
        fence_async();
        __syncwarp();
        if (lane == 0) {
          tma_store(&p.dzm, slab, (int)col0, (int)row, (int)t0);
          tma_store(&p.dxm, slab + in.tensor, (int)col0, (int)row, (int)t0);
          bulk_commit();
        }
      }
    }
  }
  if (MOVE == kTiles && lane == 0) bulk_wait_read();
  // no CTA leaves before the others are done with its memory, nor is dh0 written,
  // where it takes the place of dh_n before all have read that
  if (cluster > 1) {
    if (p.dh0 && p.dh0 == p.dh_n) cluster_arrive(); else cluster_arrive_relaxed();
    cluster_wait();
  }
  if (p.dh0 && live && rank == 0 && warp == 0) {
    float last[VEC];
    state.get(last);
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.dh0[row * p.state_b + col + v] = last[v];
  }
}

// ------------------------------------------------------------------ launch
struct Plan {
  int vec, warps, cluster, waves;
  bool flat, gated;
  int move;
  int64_t groups;  // of all rows
  size_t smem;
};

// What a wave takes, in us: `fixed` + `warp` x the CTA's warps from its inputs
// to its outputs (+ kHop through the cluster), and at least `move` x the
// resident warps of an SM for their share of the memory bandwidth (10% more where
// clusters go in step).  Fitted to runs of every split of 16-byte-aligned rows at
// T = 128..65536 and 4..2048 column groups, most of which it is within 10% of the fastest
// split at.  Rows off 16 bytes go by the same constants, up to a third from the
// fastest split (2000 x 20 x 301 float16 backward 59.9 us, best 45.9; 7179 x 3 x 364
// forward 35.4, best 27.1; 4096 x 7 x 1023 float32 133.7, best 95.8).
struct Pace {
  bool backward;
  int sm_warps;
  double fixed, warp, move;
};
constexpr double kHop = 0.45;
Pace pace_of(bool backward, int dtype) {
  if (backward) return {true, kBwdWarps, 0.55, dtype == HS_F32 ? 0.11 : 0.165, 0.24};
  return {false, kFwdWarps, 0.5, dtype == HS_F32 ? 0.075 : 0.12, 0.14};
}

// Dynamic shared memory of a CTA.
size_t smem_of(bool backward, bool gated, int move, int vec, int warps, int cluster) {
  const int inputs = backward ? 3 : 2, outputs = move != kTiles ? 0 : backward ? 2 : 1;
  return (size_t)(kStages * inputs + outputs) * warps * slab_bytes(move) + maps_bytes(gated, vec, warps, cluster);
}

// Clusters of c CTAs that run at once (a cluster stays within a GPC, so some
// SMs are left over), asked once per device.
int64_t clusters_at_once(const Pace &m, int warps, int c);

// Warps and CTAs along time: the least time by that model.  A sequence of n
// waves takes n + 1 of them, and what does not fit the SMs at once goes in
// rounds.  Many columns run as CTAs of 8 or 4 warps, whose phases overlap on an
// SM; few columns get more warps and CTAs along time.
void split_time(Plan &pl, int nchunk, const Pace &m) {
  double best = -1;
  for (int warps = 1; warps <= m.sm_warps; warps = warps < 4 ? 2 * warps : warps + 4) {
    if (warps > 1 && warps / 2 >= nchunk) break;
    if (warps < 4 && warps < nchunk) continue;  // CTAs of under 4 warps: short sequences alone
    const int most = std::min(kMaxCluster, (nchunk + warps - 1) / warps);
    for (int c = 1; c <= most; ++c) {
      const int64_t at_once = clusters_at_once(m, warps, c), full = pl.groups / at_once;
      const int waves = (nchunk + warps * c - 1) / (warps * c);
      auto wave = [&](int64_t groups) {
        const double resident = warps * (double)(groups * c) / 148;
        return std::max(m.fixed + m.warp * warps + (c > 1 ? kHop : 0.), m.move * (c > 1 ? 1.1 : 1.) * resident);
      };
      double time = (double)full * wave(at_once);
      if (pl.groups % at_once) time += wave(pl.groups % at_once);
      time *= waves + 1;
      if (best < 0 || time < 0.999 * best) best = time, pl.warps = warps, pl.cluster = c;
    }
  }
  pl.waves = (nchunk + pl.warps * pl.cluster - 1) / (pl.warps * pl.cluster);
  pl.smem = smem_of(m.backward, pl.gated, pl.move, pl.vec, pl.warps, pl.cluster);
}

struct Tensor3 {  // [T][rows][n] with contiguous n; null: not there
  const void *p;
  int64_t t, b;
};

// One row of B * H columns when every tensor stores its batch rows back to
// back and no start mask tells them apart; else B rows of H.  16-bit tensors
// move two columns per lane where every row is 4-byte aligned.
Plan make_plan(int dtype, int form, bool starts, int64_t T, int64_t B, int64_t H, const Tensor3 *ts, int n, int nchunk,
               const Pace &pace) {
  Plan pl = {};
  const int64_t es = (int64_t)dtype_bytes(dtype);
  pl.flat = !starts, pl.gated = form == HS_RECURRENCE_GATED;
  for (int i = 0; i < n; ++i)
    if (ts[i].p && ts[i].b != H && B > 1) pl.flat = false;
  const int64_t rows = pl.flat ? 1 : B, cols = pl.flat ? B * H : H;
  auto fits = [&](int64_t bytes) {
    for (int i = 0; i < n; ++i) {
      if (!ts[i].p) continue;
      if (!aligned(ts[i].p, bytes) || ts[i].t * es % bytes || (rows > 1 && ts[i].b * es % bytes)) return false;
    }
    return true;
  };
  pl.vec = dtype != HS_F32 && cols % 2 == 0 && fits(4) ? 2 : 1;
  bool whole = true, positive = true;  // strides that a tensor map can hold; that grow
  for (int i = 0; i < n; ++i) {
    if (!ts[i].p) continue;
    const int64_t t = ts[i].t * es, b = rows > 1 ? ts[i].b * es : 0;
    if (t <= 0 || t >= (int64_t)1 << 40 || (rows > 1 && (b <= 0 || b >= (int64_t)1 << 40))) whole = false;
    if (t < 0 || b < 0 || !aligned(ts[i].p, 16)) positive = false;
  }
  const int per = 32 * pl.vec;
  pl.groups = (cols + per - 1) / per * rows;
  // Rows off 16 bytes: one by one where the columns are few (7179 x 1092
  // float16, 18 groups: 35 us forward and 44 backward, by lanes 54 and 91), by lanes
  // where they are many (4096 x 7154 bfloat16, 112 groups: 59 and 102, one by one 67 and 137);
  // between those two the bound of 96 groups was not measured.
  if (nchunk > 1 && pl.vec == 4 / es) {
    if (whole && fits(16) && cols <= 0x7fffffff && B <= 0x7fffffff) pl.move = kTiles;
    else if (positive && pl.groups <= 96) pl.move = kRows;
  }
  split_time(pl, nchunk, pace);
  return pl;
}

// One past the tensor's last element.
const char *end_of(const Tensor3 &t, int dtype, int64_t T, int64_t B, int64_t H) {
  return t.p ? (const char *)t.p + ((B - 1) * t.b + (T - 1) * t.t + H) * (int64_t)dtype_bytes(dtype) : nullptr;
}

RecShape shape_of(const Plan &pl, int64_t T, int64_t B, int64_t H, int nchunk) {
  RecShape s;
  s.T = T, s.n = pl.flat ? B * H : H;
  s.groups = pl.flat ? pl.groups : pl.groups / B;
  s.nchunk = nchunk, s.waves = pl.waves, s.cluster = pl.cluster;
  return s;
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// The tensor as a map of boxes of `steps` x 1 row x one word row.
bool encode(CUtensorMap *m, const Tensor3 &t, int dtype, const Plan &pl, int64_t T, int64_t B, int64_t H, int steps) {
  if (!t.p) return true;
  const cuuint64_t es = dtype_bytes(dtype);
  const cuuint64_t dims[3] = {(cuuint64_t)(pl.flat ? B * H : H), (cuuint64_t)(pl.flat ? 1 : B), (cuuint64_t)T};
  const cuuint64_t strides[2] = {dims[1] > 1 ? (cuuint64_t)t.b * es : (cuuint64_t)t.t * es, (cuuint64_t)t.t * es};
  const cuuint32_t box[3] = {(cuuint32_t)(32 * pl.vec), 1, (cuuint32_t)steps}, elem[3] = {1, 1, 1};
  const CUtensorMapDataType type = dtype == HS_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == HS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                      : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return encoder() && encoder()(m, type, 3, const_cast<void *>(t.p), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr size_t kSmemMost = (size_t)(kStages * 3 + 2) * kBwdWarps * kSlab + maps_bytes(false, 2, kBwdWarps, kMaxCluster);
static_assert(kSmemMost + 512 <= 227 * 1024 && (kStages * 2 + 1) * kFwdWarps * kSlab + maps_bytes(false, 2, kFwdWarps, kMaxCluster) <= kSmemMost &&
                  kStages * 2 * kFwdWarps * slab_bytes(kRows) + maps_bytes(false, 2, kFwdWarps, kMaxCluster) <= kSmemMost &&
                  kStages * 3 * kBwdWarps * slab_bytes(kRows) + maps_bytes(false, 2, kBwdWarps, kMaxCluster) <= kSmemMost,
              "shared memory of a CTA, beside its barriers");

template <typename Args, typename K>
int launch(K kernel, const Args &args, const Plan &pl, cudaStream_t st, const char *what,
           std::atomic<unsigned long long> *done) {
  if (int e = allow_dynamic_smem((const void *)kernel, kSmemMost, done)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pl.groups * pl.cluster));
  cfg.blockDim = dim3(32, pl.warps);
  cfg.dynamicSmemBytes = pl.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)pl.cluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = pl.cluster > 1;
  (void)cudaLaunchKernelEx(&cfg, kernel, args);
  return check_launch(what);
}

int64_t clusters_at_once(const Pace &m, int warps, int c) {
  const int64_t ctas = (int64_t)(m.sm_warps / warps) * 148;
  static std::atomic<int> known[64][2][kFwdWarps / 4][kMaxCluster];
  int dev = 0;
  if (c == 1 || warps < 4 || cudaGetDevice(&dev) != cudaSuccess) return ctas / c;
  std::atomic<int> &k = known[dev & 63][m.backward][warps / 4 - 1][c - 1];
  int n = k.load(std::memory_order_relaxed);
  if (n) return n;
  static std::atomic<unsigned long long> done[2];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctas / c * c));
  cfg.blockDim = dim3(32, warps);
  cfg.dynamicSmemBytes = smem_of(m.backward, true, kTiles, 2, warps, c);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)c;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  auto ask = [&](auto kernel) {
    return allow_dynamic_smem((const void *)kernel, kSmemMost, &done[m.backward]) == HS_OK &&
           cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess && n > 0;
  };
  if (!(m.backward ? ask(rec_bwd_kernel<__nv_bfloat16, 2, true, false, kTiles>) : ask(rec_fwd_kernel<__nv_bfloat16, 2, true, false, kTiles>))) {
    (void)cudaGetLastError();
    n = (int)(ctas / c);
  }
  k.store(n, std::memory_order_relaxed);
  return n;
}

template <typename T, int VEC, bool GATED, bool STARTS, int MOVE> struct Kernel {
  static int run(const FwdArgs &a, const Plan &pl, cudaStream_t st) {
    static std::atomic<unsigned long long> done{0};
    return launch(rec_fwd_kernel<T, VEC, GATED, STARTS, MOVE>, a, pl, st, "rec_fwd_kernel", &done);
  }
  static int run(const BwdArgs &a, const Plan &pl, cudaStream_t st) {
    static std::atomic<unsigned long long> done{0};
    return launch(rec_bwd_kernel<T, VEC, GATED, STARTS, MOVE>, a, pl, st, "rec_bwd_kernel", &done);
  }
};

template <typename T, int VEC, int MOVE, typename Args>
int by_form(int form, const Args &a, const Plan &pl, cudaStream_t st) {
  const bool gated = form == HS_RECURRENCE_GATED, cuts = a.starts != nullptr;
  if (gated) return cuts ? Kernel<T, VEC, true, true, MOVE>::run(a, pl, st) : Kernel<T, VEC, true, false, MOVE>::run(a, pl, st);
  return cuts ? Kernel<T, VEC, false, true, MOVE>::run(a, pl, st) : Kernel<T, VEC, false, false, MOVE>::run(a, pl, st);
}
template <typename T, typename Args> int by_move(int form, const Args &a, const Plan &pl, cudaStream_t st) {
  constexpr int V = PerWord<T>::value;
  if (pl.move == kTiles) return by_form<T, V, kTiles>(form, a, pl, st);
  if (pl.move == kRows) return by_form<T, V, kRows>(form, a, pl, st);
  return pl.vec == V ? by_form<T, V, kLanes>(form, a, pl, st) : by_form<T, 1, kLanes>(form, a, pl, st);
}
template <typename Args> int dispatch(int dtype, int form, const Args &a, const Plan &pl, cudaStream_t st) {
  if (dtype == HS_F32) return by_move<float>(form, a, pl, st);
  if (dtype == HS_BF16) return by_move<__nv_bfloat16>(form, a, pl, st);
  return by_move<__half>(form, a, pl, st);
}

int check_common(const char *who, int dtype, int form, int64_t T, int64_t B, int64_t H) {
  if (!dtype_ok(dtype)) return fail(HS_ERR_INVALID_ARG, "%s: unknown dtype %d", who, dtype);
  if (form != HS_RECURRENCE_GATED && form != HS_RECURRENCE_LINEAR)
    return fail(HS_ERR_INVALID_ARG, "%s: unknown form %d", who, form);
  if (T < 0 || B < 0 || H < 0) return fail(HS_ERR_INVALID_ARG, "%s: negative T, B or H", who);
  if (T > (int64_t)1 << 30) return fail(HS_ERR_UNSUPPORTED, "%s: T=%lld is above 2^30", who, (long long)T);
  if (H > 0 && B > ((int64_t)1 << 31) / H)
    return fail(HS_ERR_UNSUPPORTED, "%s: B * H = %lld * %lld is above 2^31", who, (long long)B, (long long)H);
  return HS_OK;
}

}  // namespace
}  // namespace hs

extern "C" {

size_t hs_recurrence_checkpoint_bytes(int64_t T, int64_t B, int64_t H) {
  if (T <= 0 || B <= 0 || H <= 0) return 0;
  return (size_t)((T + hs::kRun - 1) / hs::kRun) * (size_t)B * ((size_t)H * sizeof(float) + sizeof(unsigned));
}

int hs_recurrence_forward(int dtype, int form, const void *z, int64_t z_t, int64_t z_b, const void *x, int64_t x_t,
                          int64_t x_b, const float *h0, const unsigned char *starts, int64_t starts_t,
                          int64_t starts_b, void *h, int64_t h_t, int64_t h_b, float *h_n, float *checkpoints,
                          int64_t T, int64_t B, int64_t H, int *dev_status, hs_stream_t stream) {
  using namespace hs;
  cudaStream_t st = (cudaStream_t)stream;
  if (int e = check_common("hs_recurrence_forward", dtype, form, T, B, H)) return e;
  if (B == 0 || H == 0) return HS_OK;
  if (T == 0) {
    if (!h_n || h_n == h0) return HS_OK;
    const size_t bytes = (size_t)B * H * sizeof(float);
    const cudaError_t e = h0 ? cudaMemcpyAsync(h_n, h0, bytes, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(h_n, 0, bytes, st);
    return e == cudaSuccess ? HS_OK : fail(HS_ERR_CUDA, "hs_recurrence_forward: %s", cudaGetErrorString(e));
  }
  if (!z || !x || !h || !dev_status) return fail(HS_ERR_INVALID_ARG, "hs_recurrence_forward: null z, x, h or dev_status");
  const size_t es = dtype_bytes(dtype);
  if (!aligned(z, es) || !aligned(x, es) || !aligned(h, es) || !aligned(h0, 4) || !aligned(h_n, 4) || !aligned(checkpoints, 4))
    return fail(HS_ERR_INVALID_ARG, "hs_recurrence_forward: misaligned tensor");
  const int nchunk = (int)((T + kRun - 1) / kRun);
  const Tensor3 ts[3] = {{z, z_t, z_b}, {x, x_t, x_b}, {h, h_t, h_b}};
  const Plan pl = make_plan(dtype, form, starts != nullptr, T, B, H, ts, 3, nchunk, pace_of(false, dtype));
  if (pl.groups * pl.cluster > 0x7fffffff) return fail(HS_ERR_UNSUPPORTED, "hs_recurrence_forward: too many columns");
  FwdArgs a = {};
  a.s = shape_of(pl, T, B, H, nchunk);
  a.z = (const char *)z, a.x = (const char *)x, a.h = (char *)h;
  a.ze = end_of(ts[0], dtype, T, B, H), a.xe = end_of(ts[1], dtype, T, B, H);
  a.h0 = h0, a.h_n = h_n, a.ckpt = checkpoints, a.starts = starts;
  a.zt = z_t, a.zb = z_b, a.xt = x_t, a.xb = x_b, a.ht = h_t, a.hb = h_b, a.st = starts_t, a.sb = starts_b;
  a.state_b = H, a.ckpt_t = B * H, a.status = dev_status;
  if (checkpoints && starts) a.masks = reinterpret_cast<unsigned *>(checkpoints + (int64_t)nchunk * B * H);
  a.masks_t = B;
  const int tile = pl.warps * kRun;
  if (pl.move == kTiles && !(encode(&a.zm, ts[0], dtype, pl, T, B, H, tile) && encode(&a.xm, ts[1], dtype, pl, T, B, H, tile) &&
                  encode(&a.hm, ts[2], dtype, pl, T, B, H, kRun)))
    return fail(HS_ERR_CUDA, "hs_recurrence_forward: cannot describe a tensor to TMA");
  return dispatch(dtype, form, a, pl, st);
}

int hs_recurrence_backward(int dtype, int form, const void *z, int64_t z_t, int64_t z_b, const void *x, int64_t x_t,
                           int64_t x_b, const float *checkpoints, int with_starts, const void *dh, int64_t dh_t, int64_t dh_b, const float *dh_n, void *dz,
                           int64_t dz_t, int64_t dz_b, void *dx, int64_t dx_t, int64_t dx_b, float *dh0, int64_t T,
                           int64_t B, int64_t H, int *dev_status, hs_stream_t stream) {
  using namespace hs;
  cudaStream_t st = (cudaStream_t)stream;
  if (int e = check_common("hs_recurrence_backward", dtype, form, T, B, H)) return e;
  if (B == 0 || H == 0) return HS_OK;
  if (T == 0) {
    if (!dh0 || dh0 == dh_n) return HS_OK;
    const size_t bytes = (size_t)B * H * sizeof(float);
    const cudaError_t e = dh_n ? cudaMemcpyAsync(dh0, dh_n, bytes, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(dh0, 0, bytes, st);
    return e == cudaSuccess ? HS_OK : fail(HS_ERR_CUDA, "hs_recurrence_backward: %s", cudaGetErrorString(e));
  }
  if (!z || !x || !checkpoints || !dz || !dx || !dev_status)
    return fail(HS_ERR_INVALID_ARG, "hs_recurrence_backward: null z, x, checkpoints, dz, dx or dev_status");
  const size_t es = dtype_bytes(dtype);
  if (!aligned(z, es) || !aligned(x, es) || !aligned(dh, es) || !aligned(dz, es) || !aligned(dx, es) ||
      !aligned(checkpoints, 4) || !aligned(dh_n, 4) || !aligned(dh0, 4))
    return fail(HS_ERR_INVALID_ARG, "hs_recurrence_backward: misaligned tensor");
  const int nchunk = (int)((T + kRun - 1) / kRun);
  const Tensor3 ts[5] = {{z, z_t, z_b}, {x, x_t, x_b}, {dh, dh_t, dh_b}, {dz, dz_t, dz_b}, {dx, dx_t, dx_b}};
  const Plan pl = make_plan(dtype, form, with_starts, T, B, H, ts, 5, nchunk, pace_of(true, dtype));
  if (pl.groups * pl.cluster > 0x7fffffff) return fail(HS_ERR_UNSUPPORTED, "hs_recurrence_backward: too many columns");
  BwdArgs a = {};
  a.s = shape_of(pl, T, B, H, nchunk);
  a.ze = end_of(ts[0], dtype, T, B, H), a.xe = end_of(ts[1], dtype, T, B, H), a.ge = end_of(ts[2], dtype, T, B, H);
  a.z = (const char *)z, a.x = (const char *)x, a.g = (const char *)dh, a.dz = (char *)dz, a.dx = (char *)dx;
  a.ckpt = checkpoints, a.dh_n = dh_n, a.dh0 = dh0;
  if (with_starts) a.starts = reinterpret_cast<const unsigned *>(checkpoints + (int64_t)nchunk * B * H);
  a.starts_t = B;
  a.zt = z_t, a.zb = z_b, a.xt = x_t, a.xb = x_b, a.gt = dh_t, a.gb = dh_b;
  a.dzt = dz_t, a.dzb = dz_b, a.dxt = dx_t, a.dxb = dx_b;
  a.state_b = H, a.ckpt_t = B * H, a.status = dev_status;
  const int tile = pl.warps * kRun;
  if (pl.move == kTiles && !(encode(&a.zm, ts[0], dtype, pl, T, B, H, tile) && encode(&a.xm, ts[1], dtype, pl, T, B, H, tile) &&
                  encode(&a.gm, ts[2], dtype, pl, T, B, H, tile) && encode(&a.dzm, ts[3], dtype, pl, T, B, H, kRun) &&
                  encode(&a.dxm, ts[4], dtype, pl, T, B, H, kRun)))
    return fail(HS_ERR_CUDA, "hs_recurrence_backward: cannot describe a tensor to TMA");
  return dispatch(dtype, form, a, pl, st);
}

}  // extern "C"
