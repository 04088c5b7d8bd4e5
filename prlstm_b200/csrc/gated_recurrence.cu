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
// operations is fixed by the shape alone: results are the same bit for bit
// from run to run.  No CTA waits on one outside its own cluster.
#include <float.h>

#include <algorithm>

#include "lm_types.cuh"

namespace hs {
namespace {

constexpr int kRun = 16;       // steps per warp and per saved state
constexpr int kMaxWarps = 8;   // warps of a CTA along time
constexpr int kMaxCluster = 8; // CTAs of a cluster along time
constexpr int kFwdStages = 3, kBwdStages = 2;
constexpr unsigned kStep = 128, kTensor = kRun * kStep;  // shared memory of one warp: a step, a run of one tensor

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
  int64_t zt, zb, xt, xb, ht, hb, st, sb;  // strides in elements
  int64_t state_b;                         // row stride of h0 and h_n (columns)
  int64_t ckpt_t;                          // columns of one saved state (B * H)
  int *status;
};

struct BwdArgs {
  RecShape s;
  const char *z, *x, *g;
  char *dz, *dx;
  const float *ckpt, *dh_n;
  float *dh0;
  const unsigned char *starts;
  int64_t zt, zb, xt, xb, gt, gb, dzt, dzb, dxt, dxb, st, sb;
  int64_t state_b, ckpt_t;
  int *status;
};

HS_DEV unsigned smem_u32(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
HS_DEV void cp_async4(unsigned dst, const void *src, bool valid) {
  const int n = valid ? 4 : 0;  // 0 bytes read: the word is filled with zeros
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
HS_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> HS_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
HS_DEV void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
HS_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
HS_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
HS_DEV void fence_mbar_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
HS_DEV void mbar_init(uint64_t *b) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(b)) : "memory");
}
HS_DEV void mbar_expect(uint64_t *b, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
// Bounded wait for a phase: past kWaitLimitNs, or once another wait has given
// up, the status word is set and the caller goes on (its results are void).
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
      if (ld_status(status) != 0) return;
      if (globaltimer() - t0 > kWaitLimitNs) {
        set_status(status, HS_ERR_DEVICE_TIMEOUT);
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

// The columns of one lane: one float32, or two as one pair of registers that
// sm_100a's packed float32 instructions take at once.
template <int VEC> struct Cols;
template <> struct Cols<1> {
  float v;
  HS_DEV static Cols all(float a) { return {a}; }
  HS_DEV static Cols of(const float *a) { return {a[0]}; }
  HS_DEV void get(float *a) const { a[0] = v; }
};
template <> struct Cols<2> {
  unsigned long long v;
  HS_DEV static Cols of(const float *a) {
    Cols r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a[0]), "f"(a[1]));
    return r;
  }
  HS_DEV static Cols all(float a) {
    const float t[2] = {a, a};
    return of(t);
  }
  HS_DEV void get(float *a) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a[0]), "=f"(a[1]) : "l"(v)); }
};
HS_DEV Cols<1> operator+(Cols<1> a, Cols<1> b) { return {a.v + b.v}; }
HS_DEV Cols<1> operator-(Cols<1> a, Cols<1> b) { return {a.v - b.v}; }
HS_DEV Cols<1> operator*(Cols<1> a, Cols<1> b) { return {__fmul_rn(a.v, b.v)}; }
HS_DEV Cols<1> fma(Cols<1> a, Cols<1> b, Cols<1> c) { return {fmaf(a.v, b.v, c.v)}; }
HS_DEV Cols<2> fma(Cols<2> a, Cols<2> b, Cols<2> c) {
  Cols<2> r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
HS_DEV Cols<2> operator+(Cols<2> a, Cols<2> b) {
  Cols<2> r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
HS_DEV Cols<2> operator*(Cols<2> a, Cols<2> b) {
  Cols<2> r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
HS_DEV Cols<2> operator-(Cols<2> a, Cols<2> b) { return fma(b, Cols<2>::all(-1.f), a); }

// f = 1/(1+e^-z) and 1-f = e^-z/(1+e^-z), each to a few float32 ulps of its own
// size.  e^-z is held to 2^126, so that both stay finite (f is 0 to float32's
// smallest normal number there); a NaN stays one.  The reciprocal is refined by
// one Newton step (as in sigf: its rounding compounds over thousands of steps).
template <int VEC> HS_DEV void gate(const float *z, Cols<VEC> &f, Cols<VEC> &om) {
  float t[VEC], r[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    float x = z[v] * -1.44269504088896341f;
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(126.f));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t[v]) : "f"(x));
  }
  const Cols<VEC> e = Cols<VEC>::of(t), nd = fma(e, Cols<VEC>::all(-1.f), Cols<VEC>::all(-1.f));  // -(1 + e^-z)
  float dd[VEC];
  nd.get(dd);
#pragma unroll
  for (int v = 0; v < VEC; ++v) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r[v]) : "f"(-dd[v]));
  const Cols<VEC> rr = Cols<VEC>::of(r);
  f = fma(rr, fma(nd, rr, Cols<VEC>::all(1.f)), rr);
  om = e * f;
}

// Row of one warp: base pointers advance by whole steps.
template <typename T, int VEC> HS_DEV void fetch_word(unsigned dst, const char *src, bool valid) {
  if constexpr (VEC == PerWord<T>::value) {
    cp_async4(dst, src, valid);
  } else {  // one 16-bit value per lane: rows that are not 4-byte aligned
    unsigned w = 0;
    if (valid) w = *reinterpret_cast<const unsigned short *>(src);
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(w) : "memory");
  }
}
template <typename T, int VEC> HS_DEV void read_word(unsigned src, float *v) {
  unsigned w;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(src) : "memory");
  if constexpr (VEC == PerWord<T>::value) {
    unpack_word<T>(w, v);
  } else {
    float t[2];
    unpack_word<T>(w, t);
    v[0] = t[0];
  }
}
template <typename T, int VEC> HS_DEV void write_word(char *dst, const float *v) {
  if constexpr (VEC == PerWord<T>::value)
    *reinterpret_cast<unsigned *>(dst) = pack_word<T>(v);
  else
    *reinterpret_cast<T *>(dst) = from_f32<T>(v[0]);
}

// The map h -> a h + b of a run of steps, of one lane's columns.  a = +inf
// marks a run that a start lies in: nothing passes it, the map is b alone.  (A
// product of gates is at most 1; one of given coefficients is held to the
// largest finite value, so that it leaves a zero state zero as step by step.)
template <int VEC> struct __align__(8 * VEC) Map {
  float a[VEC], b[VEC];
};
template <int VEC, bool STARTS> HS_DEV Cols<VEC> apply(const Map<VEC> &m, Cols<VEC> h) {
  const Cols<VEC> b = Cols<VEC>::of(m.b), r = fma(Cols<VEC>::of(m.a), h, b);
  return STARTS && m.a[0] == __int_as_float(0x7f800000) ? b : r;
}
template <int VEC, bool GATED> HS_DEV Cols<VEC> held(Cols<VEC> a) {
  if (GATED) return a;
  float v[VEC];
  a.get(v);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(v[i]) : "f"(FLT_MAX));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(v[i]) : "f"(-FLT_MAX));
  }
  return Cols<VEC>::of(v);
}

// The maps of the warps of this CTA and of the CTAs of its cluster, each in
// two copies for alternate waves: a wave's barrier separates its writes from
// the reads of the wave two before.  The CTAs' maps arrive by asynchronous
// remote stores that complete on `bar`, so no warp waits for its own global
// stores.  A CTA sends the map of wave w+2 only after all of wave w+1 have
// arrived, and each of those was sent after its sender's last read of wave w.
template <int VEC> struct Maps {
  Map<VEC> warp[2][kMaxWarps][32], cta[2][kMaxCluster][32];
  uint64_t bar[2];
};

// Sets up the maps; met by exchange_ready() before the first publish.
template <int VEC> HS_DEV void exchange_init(Maps<VEC> &m, int warps, int warp, int lane, int cluster) {
  Map<VEC> one;
#pragma unroll
  for (int v = 0; v < VEC; ++v) one.a[v] = 1.f, one.b[v] = 0.f;
  for (int j = warps + warp; j < kMaxWarps; j += warps) m.warp[0][j][lane] = m.warp[1][j][lane] = one;  // absent warps
  if (cluster > 1) {
    if (warp == 0 && lane == 0) {
      mbar_init(&m.bar[0]);
      mbar_init(&m.bar[1]);
      fence_mbar_init();
    }
    cluster_arrive();
  }
}
HS_DEV void exchange_ready(int cluster) {
  if (cluster > 1) cluster_wait();  // every CTA has started and set up its barriers
}

// Publishes this warp's map of wave w.
template <int VEC, bool GATED, bool STARTS>
HS_DEV void publish(Maps<VEC> &m, int w, int warps, int warp, int lane, int cluster, int rank, Cols<VEC> A, Cols<VEC> B,
                    bool cut) {
  const int p = w & 1;
  Map<VEC> mine;
  held<VEC, GATED>(A).get(mine.a);
  B.get(mine.b);
  if (STARTS && cut) mine.a[0] = __int_as_float(0x7f800000);
  m.warp[p][warp][lane] = mine;
  __syncthreads();
  if (cluster == 1) return;
  if (warp == 0 && lane == 0) mbar_expect(&m.bar[p], cluster * 32 * (unsigned)sizeof(Map<VEC>));
  if (warp == warps - 1) {  // the CTA's map, to every CTA of the cluster
    const Cols<VEC> none = Cols<VEC>::all(0.f);
    Cols<VEC> ta = Cols<VEC>::all(1.f), tb = none;
    bool any = false;
#pragma unroll
    for (int j = 0; j < kMaxWarps; ++j) {
      const Map<VEC> e = m.warp[p][j][lane];
      if (STARTS && e.a[0] == __int_as_float(0x7f800000)) any = true;
      tb = apply<VEC, STARTS>(e, tb);
      ta = held<VEC, GATED>(Cols<VEC>::of(e.a) * ta);
    }
    Map<VEC> t;
    ta.get(t.a);
    tb.get(t.b);
    if (STARTS && any) t.a[0] = __int_as_float(0x7f800000);
    for (int r = 0; r < cluster; ++r) {
      const unsigned to = cluster_addr(&m.cta[p][rank][lane], r), bar = cluster_addr(&m.bar[p], r);
      if constexpr (VEC == 2)
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to),
                     "f"(t.a[0]), "f"(t.a[1]), "f"(t.b[0]), "f"(t.b[1]), "r"(bar)
                     : "memory");
      else
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(to),
                     "f"(t.a[0]), "f"(t.b[0]), "r"(bar)
                     : "memory");
    }
  }
}

// The state entering this warp's run of wave w; `state`, the same in every
// thread of a column, moves from the wave's entry to its end.
template <int VEC, bool STARTS>
HS_DEV Cols<VEC> resolve(Maps<VEC> &m, int w, int warp, int lane, int cluster, int rank, Cols<VEC> &state, int *status) {
  const int p = w & 1;
  Cols<VEC> in = state;
  if (cluster == 1) {
#pragma unroll
    for (int j = 0; j < kMaxWarps; ++j) {
      if (j == warp) in = state;
      state = apply<VEC, STARTS>(m.warp[p][j][lane], state);
    }
    return in;
  }
  mbar_wait(&m.bar[p], (w >> 1) & 1, status);
#pragma unroll
  for (int r = 0; r < kMaxCluster; ++r) {
    if (r < cluster) {
      if (r == rank) in = state;
      state = apply<VEC, STARTS>(m.cta[p][r][lane], state);
    }
  }
#pragma unroll
  for (int j = 0; j < kMaxWarps - 1; ++j)
    if (j < warp) in = apply<VEC, STARTS>(m.warp[p][j][lane], in);
  return in;
}

template <int VEC> HS_DEV void load_state(const float *p, int64_t at, float *v) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = p ? p[at + i] : 0.f;
}

// ------------------------------------------------------------------ forward
// Shared memory: kFwdStages buffers of [2 tensors][16 steps][32 words] per warp,
// each lane's words private to it (copied in and read by the same thread).
//
// A wave is summarised before the previous one is finished: its gates and
// its map are computed while the previous wave's maps travel, then the
// previous wave's outputs are written, then its own map is published.  Between the
// two a 16-bit lane keeps 1-f alone and reads x again from shared memory
// (f = 1 - (1-f) is off by 2^-25 at most); a float32 lane keeps f and b.
template <typename T, int VEC, bool GATED, bool STARTS> struct FwdRun {
  static constexpr bool kBoth = sizeof(T) == 4;
  using C = Cols<VEC>;
  C keep[GATED || kBoth ? kRun : 1], b[kBoth ? kRun : 1];
  unsigned mask;
  C A, B;

  // gates and map of the run staged at d; steps from len on are the identity
  HS_DEV void summarise(unsigned d, int len) {
    A = C::all(1.f), B = C::all(0.f);
    auto one = [&](int k, bool cut) {
      float zv[VEC], xv[VEC];
      read_word<T, VEC>(d + k * kStep, zv);
      read_word<T, VEC>(d + kTensor + k * kStep, xv);
      C f, bb;
      if (GATED) {
        C om;
        gate<VEC>(zv, f, om);
        bb = om * C::of(xv);
        keep[k] = kBoth ? f : om;
      } else {
        f = C::of(zv);
        bb = C::of(xv);
        if (kBoth) keep[k] = f;
      }
      if (kBoth) b[k] = bb;
      A = cut ? C::all(0.f) : A * f;
      B = cut ? bb : fma(f, B, bb);
    };
    if (len < kRun) {
#pragma unroll
      for (int k = 0; k < kRun; ++k)
        if (k < len) one(k, STARTS && ((mask >> k) & 1));
    } else if (STARTS && mask) {
#pragma unroll
      for (int k = 0; k < kRun; ++k) one(k, (mask >> k) & 1);
    } else {
#pragma unroll
      for (int k = 0; k < kRun; ++k) one(k, false);
    }
  }

  // the states of the run from the one entering it
  HS_DEV void write(unsigned d, int len, C h, char *hq, int64_t hs) const {
    auto one = [&](int k, bool cut) {
      C f, bb;
      if (kBoth) {
        f = keep[k], bb = b[k];
      } else {
        float xv[VEC];
        read_word<T, VEC>(d + kTensor + k * kStep, xv);
        bb = C::of(xv);
        if (GATED) {
          f = C::all(1.f) - keep[k];
          bb = keep[k] * bb;
        } else {
          float zv[VEC];
          read_word<T, VEC>(d + k * kStep, zv);
          f = C::of(zv);
        }
      }
      h = cut ? bb : fma(f, h, bb);
      float hv[VEC];
      h.get(hv);
      write_word<T, VEC>(hq, hv);
      hq += hs;
    };
    if (len < kRun) {
#pragma unroll
      for (int k = 0; k < kRun; ++k)
        if (k < len) one(k, STARTS && ((mask >> k) & 1));
    } else if (STARTS && mask) {
#pragma unroll
      for (int k = 0; k < kRun; ++k) one(k, (mask >> k) & 1);
    } else {
#pragma unroll
      for (int k = 0; k < kRun; ++k) one(k, false);
    }
  }
};

template <typename T, int VEC, bool GATED, bool STARTS>
__global__ void __launch_bounds__(32 * kMaxWarps, 2) rec_fwd_kernel(const FwdArgs p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Maps<VEC> maps;
  using C = Cols<VEC>;
  const int lane = threadIdx.x, warp = threadIdx.y, warps = blockDim.y;
  const int cluster = p.s.cluster, rank = (int)(blockIdx.x % cluster), waves = p.s.waves;
  const int64_t gid = blockIdx.x / cluster;
  const int64_t row = gid / p.s.groups;
  int64_t col = (gid % p.s.groups) * 32 * VEC + lane * VEC;
  const bool live = col < p.s.n;  // VEC > 1 only where n is a multiple of VEC
  if (!live) col = p.s.n - VEC;   // reads what a live lane reads, writes nothing
  const int64_t T_ = p.s.T;
  const char *zp = p.z + (row * p.zb + col) * sizeof(T), *xp = p.x + (row * p.xb + col) * sizeof(T);
  char *hp = p.h + (row * p.hb + col) * sizeof(T);
  const int64_t zs = p.zt * (int64_t)sizeof(T), xs = p.xt * (int64_t)sizeof(T), hs = p.ht * (int64_t)sizeof(T);
  constexpr unsigned stage = 2 * kTensor;
  const unsigned buf = smem_u32(dyn) + warp * (kFwdStages * stage) + lane * 4;

  auto start_of = [&](int w) { return ((int64_t)(w * cluster + rank) * warps + warp) * kRun; };
  auto fetch = [&](int w) {
    if (w < waves) {
      const int64_t t0 = start_of(w);
      const unsigned d = buf + (unsigned)(w % kFwdStages) * stage;
      const char *zq = zp + t0 * zs, *xq = xp + t0 * xs;
      if (t0 + kRun <= T_) {
#pragma unroll
        for (int k = 0; k < kRun; ++k, zq += zs, xq += xs) {
          fetch_word<T, VEC>(d + k * kStep, zq, true);
          fetch_word<T, VEC>(d + kTensor + k * kStep, xq, true);
        }
      } else {
#pragma unroll 1
        for (int k = 0; k < kRun && t0 + k < T_; ++k, zq += zs, xq += xs) {
          fetch_word<T, VEC>(d + k * kStep, zq, true);
          fetch_word<T, VEC>(d + kTensor + k * kStep, xq, true);
        }
      }
    }
    cp_commit();
  };
  auto fetch_starts = [&](int w) -> unsigned {
    const int64_t t = start_of(w) + lane;
    return w < waves && lane < kRun && t < T_ ? p.starts[t * p.st + row * p.sb] : 0;
  };
  auto length = [&](int w) { return (int)max((int64_t)0, min((int64_t)kRun, T_ - start_of(w))); };
  auto staged = [&](int w) { return buf + (unsigned)(w % kFwdStages) * stage; };

  exchange_init(maps, warps, warp, lane, cluster);
  float s0[VEC];
  load_state<VEC>(p.h0, row * p.state_b + col, s0);
  C state = C::of(s0);
  unsigned next = 0;
  fetch(0);
  fetch(1);
  if (STARTS) next = fetch_starts(0);

  FwdRun<T, VEC, GATED, STARTS> run[2];
  auto summarise = [&](FwdRun<T, VEC, GATED, STARTS> &r, int w) {
    r.mask = 0;
    if (STARTS) {
      r.mask = __ballot_sync(0xffffffffu, next != 0);
      next = fetch_starts(w + 1);
    }
    r.summarise(staged(w), length(w));
  };
  auto put = [&](const FwdRun<T, VEC, GATED, STARTS> &r, int w) {
    publish<VEC, GATED, STARTS>(maps, w, warps, warp, lane, cluster, rank, r.A, r.B, r.mask != 0);
  };
  // wave w is published, wave w+1 staged; ends with w+1 published
  auto wave = [&](FwdRun<T, VEC, GATED, STARTS> &cur, FwdRun<T, VEC, GATED, STARTS> &nxt, int w) {
    fetch(w + 2);
    cp_wait<1>();
    if (w + 1 < waves) summarise(nxt, w + 1);
    const C in = resolve<VEC, STARTS>(maps, w, warp, lane, cluster, rank, state, p.status);
    const int64_t t0 = start_of(w);
    const int len = length(w);
    if (live && len > 0) {
      if (p.ckpt) {
        float *c = p.ckpt + (t0 / kRun) * p.ckpt_t + row * p.state_b + col;
        float v[VEC];
        in.get(v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) c[i] = v[i];
      }
      cur.write(staged(w), len, in, hp + t0 * hs, hs);
    }
    if (w + 1 < waves) put(nxt, w + 1);
  };
  cp_wait<1>();
  summarise(run[0], 0);
  exchange_ready(cluster);
  put(run[0], 0);
  for (int w = 0; w < waves; w += 2) {
    wave(run[0], run[1], w);
    if (w + 1 < waves) wave(run[1], run[0], w + 1);
  }
  if (p.h_n && live && rank == 0 && warp == 0) {
    float v[VEC];
    state.get(v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) p.h_n[row * p.state_b + col + i] = v[i];
  }
  if (cluster > 1) {  // no CTA leaves before the others are done with its memory
    cluster_arrive_relaxed();
    cluster_wait();
  }
}

// ------------------------------------------------------------------ backward
// Shared memory: [3 tensors][16 steps][32 words] per warp and stage; a stage is
// in use until its outputs are written (g is read twice), so the next one is
// fetched beside it.
template <typename T, int VEC, bool GATED, bool STARTS>
__global__ void __launch_bounds__(32 * kMaxWarps, 2) rec_bwd_kernel(const BwdArgs p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Maps<VEC> maps;
  // float32 keeps both f and 1-f; the 16-bit types keep 1-f alone and take
  // f = 1 - (1-f), whose error (2^-25) only enters u, far below their rounding
  constexpr bool kBoth = GATED && sizeof(T) == 4;
  const int lane = threadIdx.x, warp = threadIdx.y, warps = blockDim.y;
  const int cluster = p.s.cluster, rank = (int)(blockIdx.x % cluster);
  const int64_t gid = blockIdx.x / cluster;
  const int64_t row = gid / p.s.groups;
  int64_t col = (gid % p.s.groups) * 32 * VEC + lane * VEC;
  const bool live = col < p.s.n;
  if (!live) col = p.s.n - VEC;
  const int64_t T_ = p.s.T;
  const char *zp = p.z + (row * p.zb + col) * sizeof(T), *xp = p.x + (row * p.xb + col) * sizeof(T);
  const char *gp = p.g + (row * p.gb + col) * sizeof(T);
  char *dzp = p.dz + (row * p.dzb + col) * sizeof(T), *dxp = p.dx + (row * p.dxb + col) * sizeof(T);
  const int64_t zs = p.zt * (int64_t)sizeof(T), xs = p.xt * (int64_t)sizeof(T), gs = p.gt * (int64_t)sizeof(T);
  const int64_t dzs = p.dzt * (int64_t)sizeof(T), dxs = p.dxt * (int64_t)sizeof(T);
  constexpr unsigned stage = 3 * kTensor;
  const unsigned buf = smem_u32(dyn) + warp * (kBwdStages * stage) + lane * 4;

  exchange_init(maps, warps, warp, lane, cluster);
  float s0[VEC];
  load_state<VEC>(p.dh_n, row * p.state_b + col, s0);
  Cols<VEC> state = Cols<VEC>::of(s0);

  // chunks from the last to the first; below 0: past the beginning, nothing
  auto chunk_of = [&](int w) { return p.s.nchunk - 1 - ((w * cluster + rank) * warps + warp); };
  auto fetch = [&](int w) {
    const int c = chunk_of(w);
    const int64_t t0 = (int64_t)c * kRun;
    const unsigned d = buf + (unsigned)(w % kBwdStages) * stage;
    const char *zq = zp + t0 * zs, *xq = xp + t0 * xs, *gq = gp + t0 * gs;
    if (c >= 0 && t0 + kRun <= T_ && p.g) {
#pragma unroll
      for (int k = 0; k < kRun; ++k, zq += zs, xq += xs, gq += gs) {
        fetch_word<T, VEC>(d + k * kStep, zq, true);
        fetch_word<T, VEC>(d + kTensor + k * kStep, xq, true);
        fetch_word<T, VEC>(d + 2 * kTensor + k * kStep, gq, true);
      }
    } else if (c >= 0) {
#pragma unroll 1
      for (int k = 0; k < kRun; ++k, zq += zs, xq += xs, gq += gs) {
        const bool ok = t0 + k < T_, okg = ok && p.g;
        fetch_word<T, VEC>(d + k * kStep, ok ? zq : zp, ok);
        fetch_word<T, VEC>(d + kTensor + k * kStep, ok ? xq : xp, ok);
        fetch_word<T, VEC>(d + 2 * kTensor + k * kStep, okg ? gq : zp, okg);
      }
    }
    cp_commit();
  };
  auto fetch_starts = [&](int w) -> unsigned {
    const int64_t t = (int64_t)chunk_of(w) * kRun + lane;
    return lane < kRun && t >= 0 && t < T_ ? p.starts[t * p.st + row * p.sb] : 0;
  };
  auto fetch_ckpt = [&](int w, float *h) {
    const int c = chunk_of(w);
    load_state<VEC>(c >= 0 ? p.ckpt : nullptr, c * p.ckpt_t + row * p.state_b + col, h);
  };

  unsigned next_start = 0;
  float next_h[VEC];
  fetch(0);
  fetch_ckpt(0, next_h);
  if (STARTS) next_start = fetch_starts(0);
  for (int w = 0; w < p.s.waves; ++w) {
    if (w + 1 < p.s.waves) fetch(w + 1); else cp_commit();
    unsigned mask = 0;
    if (STARTS) {
      mask = __ballot_sync(0xffffffffu, next_start != 0);
      if (w + 1 < p.s.waves) next_start = fetch_starts(w + 1);
    }
    float h[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = next_h[v];
    if (w + 1 < p.s.waves) fetch_ckpt(w + 1, next_h);
    cp_wait<1>();
    const int c = chunk_of(w);
    const int64_t t0 = (int64_t)c * kRun;
    const unsigned d = buf + (unsigned)(w % kBwdStages) * stage;
    const int len = c < 0 ? 0 : (int)min((int64_t)kRun, T_ - t0);
    using C = Cols<VEC>;
    const C one = C::all(1.f), zero = C::all(0.f);
    // keep: 1-f (gated) or f (linear); q: the factor of e in df (set where the
    // warp has a run, c >= 0, and read only there)
#pragma nv_diag_suppress 549
    C keep[kRun], both[kBoth ? kRun : 1], q[kRun];
    auto coef = [&](int k) { return kBoth ? both[kBoth ? k : 0] : GATED ? one - keep[k] : keep[k]; };
    auto grad = [&](int k) {
      float g[VEC];
      read_word<T, VEC>(d + 2 * kTensor + k * kStep, g);
      return C::of(g);
    };
    C A = one, B = zero;
    if (c >= 0) {
      C s = C::of(h);
#pragma unroll
      for (int k = 0; k < kRun; ++k) {
        float zv[VEC], xv[VEC];
        read_word<T, VEC>(d + k * kStep, zv);
        read_word<T, VEC>(d + kTensor + k * kStep, xv);
        const C x = C::of(xv);
        if (STARTS && ((mask >> k) & 1)) s = zero;
        if (GATED) {
          C f, om;
          gate<VEC>(zv, f, om);
          q[k] = (s - x) * (f * om);
          s = fma(f, s, om * x);
          keep[k] = om;
          if (kBoth) both[k] = f;
        } else {
          q[k] = s;
          keep[k] = C::of(zv);
          s = fma(keep[k], s, x);
        }
      }
      if (len < kRun) {
#pragma unroll
        for (int k = 0; k < kRun; ++k)
          if (k >= len) {
            keep[k] = GATED ? zero : one;
            if (kBoth) both[k] = one;
          }
      }
      if (STARTS && mask) {
#pragma unroll
        for (int k = kRun - 1; k >= 0; --k) {
          const bool cut = (mask >> k) & 1;
          B = cut ? zero : coef(k) * (grad(k) + B);
          A = cut ? zero : A * coef(k);
        }
      } else {
#pragma unroll
        for (int k = kRun - 1; k >= 0; --k) {
          const C f = coef(k);
          B = f * (grad(k) + B);
          A = A * f;
        }
      }
    }
    if (w == 0) exchange_ready(cluster);
    publish<VEC, GATED, STARTS>(maps, w, warps, warp, lane, cluster, rank, A, B, mask != 0);
    C uu = resolve<VEC, STARTS>(maps, w, warp, lane, cluster, rank, state, p.status);
    if (live && len > 0) {
      char *dzq = dzp + (t0 + kRun - 1) * dzs, *dxq = dxp + (t0 + kRun - 1) * dxs;
      auto put = [&](int k, bool cut, bool write) {
        const C e = grad(k) + uu;
        uu = cut ? zero : coef(k) * e;
        if (write) {
          float dz[VEC], dx[VEC];
          (e * q[k]).get(dz);
          (GATED ? e * keep[k] : e).get(dx);
          write_word<T, VEC>(dzq, dz);
          write_word<T, VEC>(dxq, dx);
        }
        dzq -= dzs;
        dxq -= dxs;
      };
      if (len < kRun || (STARTS && mask)) {
#pragma unroll
        for (int k = kRun - 1; k >= 0; --k) put(k, STARTS && ((mask >> k) & 1), k < len);
      } else {
#pragma unroll
        for (int k = kRun - 1; k >= 0; --k) put(k, false, true);
      }
    }
  }
  if (p.dh0 && live && rank == 0 && warp == 0) {
    float last[VEC];
    state.get(last);
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.dh0[row * p.state_b + col + v] = last[v];
  }
  if (cluster > 1) {  // no CTA leaves before the others are done with its memory
    cluster_arrive_relaxed();
    cluster_wait();
  }
}

// ------------------------------------------------------------------ launch
struct Plan {
  int warps, cluster;
  size_t smem;
};

// Warps and CTAs along time: up to 8 warps as the sequence has runs for, then
// the cluster size of the least time in units of one wave: the rounds in
// which the CTAs pass through the SMs (two at a time each) times the waves of a
// round, with 1.5 for its start and end.
Plan make_plan(int64_t groups, int nchunk, int tensors, int stages) {
  Plan pl;
  pl.warps = 1;
  while (pl.warps < kMaxWarps && pl.warps < nchunk) pl.warps *= 2;
  const int64_t slots = 2 * 148;
  const int most = std::min(kMaxCluster, (nchunk + pl.warps - 1) / pl.warps);
  double best = 0;
  for (int c = 1; c <= most; ++c) {
    const int64_t rounds = (groups * c + slots - 1) / slots;
    const int waves = (nchunk + pl.warps * c - 1) / (pl.warps * c);
    const double time = (double)rounds * (waves + 1.5);
    if (c == 1 || time < best) best = time, pl.cluster = c;
  }
  pl.smem = (size_t)stages * tensors * kRun * pl.warps * 128;
  return pl;
}

template <typename Args, typename K>
int launch(K kernel, const Args &args, const Plan &pl, int64_t groups, cudaStream_t st, const char *what,
           std::atomic<unsigned long long> *done) {
  if (int e = allow_dynamic_smem((const void *)kernel, (size_t)6 * kRun * kMaxWarps * 128, done)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(groups * pl.cluster));
  cfg.blockDim = dim3(32, pl.warps);
  cfg.dynamicSmemBytes = pl.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)pl.cluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args) != cudaSuccess) return check_launch(what);
  return check_launch(what);
}

template <typename T, int VEC, bool GATED, bool STARTS> int launch_fwd(const FwdArgs &a, const Plan &pl, int64_t groups, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  return launch(rec_fwd_kernel<T, VEC, GATED, STARTS>, a, pl, groups, st, "rec_fwd_kernel", &done);
}
template <typename T, int VEC, bool GATED, bool STARTS> int launch_bwd(const BwdArgs &a, const Plan &pl, int64_t groups, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  return launch(rec_bwd_kernel<T, VEC, GATED, STARTS>, a, pl, groups, st, "rec_bwd_kernel", &done);
}

#define HS_REC_DISPATCH(FN, args)                                                                       \
  [&]() -> int {                                                                                        \
    const bool gated = form == HS_RECURRENCE_GATED, cuts = starts != nullptr;                           \
    auto go = [&](auto tag, auto vec) -> int {                                                          \
      using E = decltype(tag);                                                                          \
      constexpr int V = decltype(vec)::value;                                                           \
      if (gated) return cuts ? FN<E, V, true, true>(args, pl, groups, st) : FN<E, V, true, false>(args, pl, groups, st); \
      return cuts ? FN<E, V, false, true>(args, pl, groups, st) : FN<E, V, false, false>(args, pl, groups, st);          \
    };                                                                                                  \
    if (dtype == HS_F32) return go(float{}, std::integral_constant<int, 1>{});                          \
    if (dtype == HS_BF16)                                                                               \
      return vec == 2 ? go(__nv_bfloat16{}, std::integral_constant<int, 2>{})                           \
                      : go(__nv_bfloat16{}, std::integral_constant<int, 1>{});                          \
    return vec == 2 ? go(__half{}, std::integral_constant<int, 2>{}) : go(__half{}, std::integral_constant<int, 1>{});   \
  }()

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

// One row of B * H columns when every tensor stores its batch rows back to
// back and no start mask tells them apart; else B rows of H.
bool one_row(const void *starts, int64_t H, std::initializer_list<int64_t> batch_strides) {
  if (starts) return false;
  for (int64_t s : batch_strides)
    if (s != H) return false;
  return true;
}

// 16-bit tensors move two columns per lane where every row is 4-byte aligned.
int vec_of(int dtype, int64_t n, std::initializer_list<const void *> ptrs, std::initializer_list<int64_t> strides) {
  if (dtype == HS_F32) return 1;
  if (n % 2) return 1;
  for (const void *p : ptrs)
    if (p && !aligned(p, 4)) return 1;
  for (int64_t s : strides)
    if (s % 2) return 1;
  return 2;
}

}  // namespace
}  // namespace hs

extern "C" {

size_t hs_recurrence_checkpoint_bytes(int64_t T, int64_t B, int64_t H) {
  if (T <= 0 || B <= 0 || H <= 0) return 0;
  return (size_t)((T + hs::kRun - 1) / hs::kRun) * (size_t)B * (size_t)H * sizeof(float);
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
  const bool flat = one_row(starts, H, {z_b, x_b, h_b});
  FwdArgs a = {};
  a.s.T = T;
  a.s.n = flat ? B * H : H;
  const int vec = vec_of(dtype, a.s.n, {z, x, h}, {z_t, x_t, h_t, flat ? 0 : z_b, flat ? 0 : x_b, flat ? 0 : h_b});
  const int per = 32 * (dtype == HS_F32 ? 1 : vec);
  a.s.groups = (a.s.n + per - 1) / per;
  const int64_t groups = a.s.groups * (flat ? 1 : B);
  a.s.nchunk = (int)((T + kRun - 1) / kRun);
  const Plan pl = make_plan(groups, a.s.nchunk, 2, kFwdStages);
  if (groups * pl.cluster > 0x7fffffff) return fail(HS_ERR_UNSUPPORTED, "hs_recurrence_forward: too many columns");
  a.s.cluster = pl.cluster;
  a.s.waves = (a.s.nchunk + pl.warps * pl.cluster - 1) / (pl.warps * pl.cluster);
  a.z = (const char *)z, a.x = (const char *)x, a.h = (char *)h;
  a.h0 = h0, a.h_n = h_n, a.ckpt = checkpoints, a.starts = starts;
  a.zt = z_t, a.zb = z_b, a.xt = x_t, a.xb = x_b, a.ht = h_t, a.hb = h_b, a.st = starts_t, a.sb = starts_b;
  a.state_b = H, a.ckpt_t = B * H, a.status = dev_status;
  return HS_REC_DISPATCH(launch_fwd, a);
}

int hs_recurrence_backward(int dtype, int form, const void *z, int64_t z_t, int64_t z_b, const void *x, int64_t x_t,
                           int64_t x_b, const float *checkpoints, const unsigned char *starts, int64_t starts_t,
                           int64_t starts_b, const void *dh, int64_t dh_t, int64_t dh_b, const float *dh_n, void *dz,
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
  if (!dh) dh_t = dz_t, dh_b = dz_b;
  const bool flat = one_row(starts, H, {z_b, x_b, dh_b, dz_b, dx_b});
  BwdArgs a = {};
  a.s.T = T;
  a.s.n = flat ? B * H : H;
  const int vec = vec_of(dtype, a.s.n, {z, x, dh, dz, dx},
                         {z_t, x_t, dh_t, dz_t, dx_t, flat ? 0 : z_b, flat ? 0 : x_b, flat ? 0 : dh_b, flat ? 0 : dz_b, flat ? 0 : dx_b});
  const int per = 32 * (dtype == HS_F32 ? 1 : vec);
  a.s.groups = (a.s.n + per - 1) / per;
  const int64_t groups = a.s.groups * (flat ? 1 : B);
  a.s.nchunk = (int)((T + kRun - 1) / kRun);
  const Plan pl = make_plan(groups, a.s.nchunk, 3, kBwdStages);
  if (groups * pl.cluster > 0x7fffffff) return fail(HS_ERR_UNSUPPORTED, "hs_recurrence_backward: too many columns");
  a.s.cluster = pl.cluster;
  a.s.waves = (a.s.nchunk + pl.warps * pl.cluster - 1) / (pl.warps * pl.cluster);
  a.z = (const char *)z, a.x = (const char *)x, a.g = (const char *)dh, a.dz = (char *)dz, a.dx = (char *)dx;
  a.ckpt = checkpoints, a.dh_n = dh_n, a.dh0 = dh0, a.starts = starts;
  a.zt = z_t, a.zb = z_b, a.xt = x_t, a.xb = x_b, a.gt = dh_t, a.gb = dh_b;
  a.dzt = dz_t, a.dzb = dz_b, a.dxt = dx_t, a.dxb = dx_b, a.st = starts_t, a.sb = starts_b;
  a.state_b = H, a.ckpt_t = B * H, a.status = dev_status;
  return HS_REC_DISPATCH(launch_bwd, a);
}

}  // extern "C"
