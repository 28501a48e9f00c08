// Gated linear recurrence over a sequence, its gradient and its one-token form.
//
//   L[t] = c softplus(Lambda) s(r[t])       a[t] = exp(-L[t])
//   h[t] = a[t] h[t-1] + sqrt(1 - a[t]^2) s(i[t]) x[t],      s = sigmoid
//   where reset[t] is set the state is dropped: a[t] = 0, and sqrt(..) is 1.
//
// Gradient, from dy (and dhT for the last state), c[t] = a[t] g[t]:
//   g[t] = dy[t] + c[t+1]            dx = g beta s(i)       di = g beta x s(i) (1 - s(i))
//   dL = g (a^2 / beta s(i) x - a h[t-1])    dr = dL L (1 - s(r))
//   dLambda = c s(Lambda) sum dL s(r)        dh0 = c[1]
//
// Layout. A CTA owns 64 channels of one sequence and walks over time in tiles of
// kTile steps; each warp takes a run of consecutive steps of the tile, each lane
// two channels, so every row access of a warp is one 128-byte (bf16) or 256-byte
// (fp32) line and the arithmetic is packed two-wide. A run is reduced to (A, E),
// h_out = A h_in + E (held as A - 1), in registers; runs are joined through shared memory, tiles
// through the shared memory of a thread-block cluster whose CTAs take consecutive
// tiles of the same sequence. So each input is read once and each output written
// once, and no CTA waits for another one outside its cluster.
//
// The backward pass reads no y: it runs each tile again from the fp32 state that
// the forward pass left at the tile's start (y in bf16 would cost dLambda three
// digits), and the reverse recurrence uses the same products A.
#include <cooperative_groups.h>

#include <atomic>
#include <initializer_list>

#include "mqc_common.cuh"
#include "mqc_host.h"
#include "packed_math.cuh"

namespace cg = cooperative_groups;

namespace mqc {
namespace {

using pk::add2;
using pk::bc2;
using pk::fma2;
using pk::mul2;
using pk::neg2;

constexpr int kChan = 64;  // channels of a CTA
constexpr int kTile = MQC_GATED_SCAN_TILE;  // time steps of a tile
constexpr int kMaxCluster = 16;

// ---------------------------------------------------------------- arithmetic

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rsqrt_a(float v) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// minimum and maximum that keep a NaN
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLeastNormal = 1.17549435e-38f;

// 1 / (1 + 2^(-z log2 e)); the exponent is held at 126, where the result is 2^-126.
__device__ __forceinline__ float2 sigmoid2(float2 z) {
  const float2 e = mul2(z, bc2(-kLog2e));
  const float2 d = add2(make_float2(ex2(min_nan(e.x, 126.f)), ex2(min_nan(e.y, 126.f))), bc2(1.f));
  return make_float2(rcp(d.x), rcp(d.y));
}

// exp(-l) - 1 for l >= 0: with -l = n ln 2 + f, |f| <= ln 2 / 2, it is
// 2^n (e^f - 1) + (2^n - 1), e^f - 1 by its Taylor polynomial of degree 7
// (remainder f^8 / 8!: below 2e-8 of f). Exact to the last place near l = 0, where
// 1 - exp(-2 l) and the decay over many steps need it.
__device__ __forceinline__ float2 expm1_neg2(float2 l) {
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: the sum's low bits are the integer
  constexpr float kLn2Hi = 0.693145751953125f;  // 16 bits: n * hi is exact
  constexpr float kLn2Lo = 1.42860682030941723e-6f;
  const float2 x = make_float2(max_nan(-l.x, -87.f), max_nan(-l.y, -87.f));
  const float2 t = fma2(x, bc2(kLog2e), bc2(kMagic));
  const float2 n = add2(t, bc2(-kMagic));
  const float2 f = fma2(n, bc2(-kLn2Lo), fma2(n, bc2(-kLn2Hi), x));
  float2 p = fma2(f, bc2(1.f / 5040.f), bc2(1.f / 720.f));
  p = fma2(p, f, bc2(1.f / 120.f));
  p = fma2(p, f, bc2(1.f / 24.f));
  p = fma2(p, f, bc2(1.f / 6.f));
  p = fma2(p, f, bc2(0.5f));
  p = fma2(mul2(p, f), f, f);
  const float2 s = make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000),
                               __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000));
  return fma2(s, p, add2(s, bc2(-1.f)));
}

__device__ __forceinline__ float softplus_acc(float u) {
  return u > 20.f ? u + log1pf(expf(-u)) : log1pf(expf(u));
}

// m = a - 1 and q = 1 - a^2 of a step with L = l.
__device__ __forceinline__ void decay2(float2 l, float2& m, float2& q) {
  m = expm1_neg2(l);
  q = mul2(neg2(m), add2(m, bc2(2.f)));
}

// Products of decays are held as M = A - 1: (1 + M)(1 + m) - 1 = M + (M m + m). A
// product of fp32 numbers just below 1 loses j k 2^-48 each time, j and k their
// distances from 1 in units of 2^-24, always to the same side; over a state's
// memory of 1e4 steps that came to 4e-5 of it.
__device__ __forceinline__ float2 join_decay(float2 M, float2 m) {
  return add2(M, fma2(M, m, m));
}

// A s + E with A = 1 + M. kDrop: where M is -1 (a reset) s is dropped, also if it is
// infinite or NaN.
template <bool kDrop>
__device__ __forceinline__ float2 apply(float2 M, float2 E, float2 s) {
  float2 r = add2(s, fma2(M, s, E));
  if (kDrop) {
    if (M.x == -1.f) r.x = E.x;
    if (M.y == -1.f) r.y = E.y;
  }
  return r;
}

// 1 / sqrt(q); 0 where q is 0 or subnormal (no decay to speak of: neither the
// input's factor, 1e-19 at most, nor its slope counts)
__device__ __forceinline__ float2 inv_sqrt2(float2 q) {
  return make_float2(q.x >= kLeastNormal ? rsqrt_a(q.x) : 0.f,
                     q.y >= kLeastNormal ? rsqrt_a(q.y) : 0.f);
}

// ------------------------------------------------------------------- memory

// Two channels of one row as they are stored: one word of adjacent channels (kVec)
// or two elements 32 channels apart (any width and alignment).
template <typename T, bool kVec>
struct Pair;

template <>
struct Pair<float, true> {
  float2 v;
  __device__ __forceinline__ void load(const float* p, int, bool, bool) {
    v = __ldg(reinterpret_cast<const float2*>(p));
  }
  __device__ __forceinline__ float2 get() const { return v; }
  static __device__ __forceinline__ void store(float* p, float2 o, int, bool, bool) {
    *reinterpret_cast<float2*>(p) = o;
  }
};
template <>
struct Pair<__nv_bfloat16, true> {
  uint32_t v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int, bool, bool) {
    v = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
  __device__ __forceinline__ float2 get() const {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float2 o, int, bool, bool) {
    __nv_bfloat162 h = __floats2bfloat162_rn(o.x, o.y);
    *reinterpret_cast<__nv_bfloat162*>(p) = h;
  }
};
template <typename T>
struct Pair<T, false> {
  T a, b;
  __device__ __forceinline__ void load(const T* p, int step, bool ok0, bool ok1) {
    a = ok0 ? __ldg(p) : T(0.f);
    b = ok1 ? __ldg(p + step) : T(0.f);
  }
  __device__ __forceinline__ float2 get() const { return make_float2(to_f(a), to_f(b)); }
  static __device__ __forceinline__ void store(T* p, float2 o, int step, bool ok0, bool ok1) {
    if (ok0) QIO<T>::st1(p, o.x);
    if (ok1) QIO<T>::st1(p + step, o.y);
  }
};

// The two channels of a lane: columns c and c + step of the tensors.
struct Lane {
  int c, step;
  bool ok0, ok1;
};

template <bool kVec>
__device__ __forceinline__ Lane lane_of(int tile, int channels) {
  const int l = threadIdx.x & 31;
  Lane r;
  r.step = kVec ? 1 : 32;
  r.c = tile * kChan + (kVec ? 2 * l : l);
  r.ok0 = r.c < channels;
  r.ok1 = r.c + r.step < channels;
  return r;
}

__device__ __forceinline__ float2 load_f2(const float* p, const Lane& l) {
  if (p == nullptr) return bc2(0.f);
  return make_float2(l.ok0 ? p[l.c] : 0.f, l.ok1 ? p[l.c + l.step] : 0.f);
}
__device__ __forceinline__ void store_f2(float* p, float2 v, const Lane& l) {
  if (l.ok0) p[l.c] = v.x;
  if (l.ok1) p[l.c + l.step] = v.y;
}

struct FwdArgs {
  const void *x, *r, *i;
  int64_t xs, rs, is;  // row strides, elements
  const float* lambda;
  const float* h0;
  const uint8_t* reset;
  void* y;
  float* hT;
  float* ckpt;  // [batch][tiles][channels]: state before each tile, or NULL
  int batch, seq, channels, chan_tiles;
  float sharpness;
};

struct BwdArgs {
  const void *x, *r, *i, *dy;
  int64_t xs, rs, is, dys;
  const float* lambda;
  const uint8_t* reset;
  const float* ckpt;
  const float* dhT;
  void *dx, *dr, *di;
  float* dh0;
  float* part;  // [batch][channels] x cluster rank: sums of dL s(r)
  int batch, seq, channels, chan_tiles;
  float sharpness;
};

// ------------------------------------------------------------------- forward

constexpr int kFwdWarps = 8;

template <typename T, bool kVec, bool kReset>
__global__ void __launch_bounds__(kFwdWarps * 32)
    gated_scan_fwd_kernel(const FwdArgs p) {
  constexpr int W = kFwdWarps, S = kTile / W;
  // (A0, A1, E0, E1) of each warp's run and of each CTA's tile, double-buffered
  __shared__ float4 seg[2][W][32];
  __shared__ float4 sum[2][kMaxCluster][32];
  cg::cluster_group cluster = cg::this_cluster();
  const int csize = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int unit = int(blockIdx.x) / csize;
  const int b = unit / p.chan_tiles;
  const Lane ln = lane_of<kVec>(unit - b * p.chan_tiles, p.channels);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = (p.seq + kTile - 1) / kTile;
  const int64_t row0 = int64_t(b) * p.seq;
  const T* x = static_cast<const T*>(p.x) + row0 * p.xs + ln.c;
  const T* r = static_cast<const T*>(p.r) + row0 * p.rs + ln.c;
  const T* iv = static_cast<const T*>(p.i) + row0 * p.is + ln.c;
  T* y = static_cast<T*>(p.y) + row0 * p.channels + ln.c;
  const uint8_t* rst = kReset ? p.reset + row0 : nullptr;
  const float2 lam = load_f2(p.lambda, ln);
  const float2 rate = make_float2(p.sharpness * softplus_acc(lam.x), p.sharpness * softplus_acc(lam.y));
  float2 carry = load_f2(p.h0 ? p.h0 + int64_t(b) * p.channels : nullptr, ln);

  Pair<T, kVec> xr[S], rr[S], ir[S];
  bool rs[S];
  auto load = [&](int tile) {
    const int t0 = tile * kTile + warp * S;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int t = t0 + s;
      const bool in = t < p.seq;
      if (kReset) rs[s] = in && rst[t] != 0;
      if (in && ln.ok0) {
        xr[s].load(x + t * p.xs, ln.step, ln.ok0, ln.ok1);
        rr[s].load(r + t * p.rs, ln.step, ln.ok0, ln.ok1);
        ir[s].load(iv + t * p.is, ln.step, ln.ok0, ln.ok1);
      } else {
        xr[s] = rr[s] = ir[s] = Pair<T, kVec>{};
      }
    }
  };

  load(rank);
  if (csize > 1) cluster.sync();  // every CTA has begun before its shared memory is written
  int buf = 0;
  for (int first = 0; first < tiles; first += csize, buf ^= 1) {
    const int tile = first + rank;
    const int t0 = tile * kTile + warp * S;
    bool rs_now[S];
#pragma unroll
    for (int s = 0; s < S; ++s) rs_now[s] = kReset && rs[s];
    float2 a[S], u[S];
    float2 M = bc2(0.f), E = bc2(0.f);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float2 m, q;
      decay2(mul2(rate, sigmoid2(rr[s].get())), m, q);
      const float2 v = mul2(sigmoid2(ir[s].get()), xr[s].get());
      u[s] = mul2(mul2(q, inv_sqrt2(q)), v);
      if (t0 + s >= p.seq) {  // past the end: the state is kept
        m = bc2(0.f);
        u[s] = bc2(0.f);
      }
      a[s] = add2(m, bc2(1.f));
      if (kReset && rs_now[s]) {
        a[s] = bc2(0.f);
        u[s] = v;
        E = v;
        M = bc2(-1.f);
      } else {
        E = fma2(a[s], E, u[s]);
        M = join_decay(M, m);
      }
    }
    seg[buf][warp][lane] = make_float4(M.x, M.y, E.x, E.y);
    // the next tile's rows are on their way while this one is joined and stored
    if (first + csize < tiles) load(tile + csize);
    __syncthreads();
    // (PM, PE): the runs before this warp's; (TM, TE): the whole tile
    float2 PM = bc2(0.f), PE = bc2(0.f), TM = bc2(0.f), TE = bc2(0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w == warp) {
        PM = TM;
        PE = TE;
      }
      const float4 g = seg[buf][w][lane];
      const float2 gm = make_float2(g.x, g.y);
      TE = apply<kReset>(gm, make_float2(g.z, g.w), TE);
      TM = join_decay(TM, gm);
    }
    float2 h = carry;
    if (csize > 1) {
      if (warp < csize)
        for (int to = warp; to < csize; to += W)
          *cluster.map_shared_rank(&sum[buf][rank][lane], to) =
              make_float4(TM.x, TM.y, TE.x, TE.y);
      cluster.sync();
      for (int k = 0; k < csize; ++k) {
        if (k == rank) h = carry;
        const float4 g = sum[buf][k][lane];
        carry = apply<kReset>(make_float2(g.x, g.y), make_float2(g.z, g.w), carry);
      }
    } else {
      carry = apply<kReset>(TM, TE, carry);
    }
    if (p.ckpt != nullptr && warp == 0 && tile < tiles)
      store_f2(p.ckpt + (int64_t(b) * tiles + tile) * p.channels, h, ln);
    h = apply<kReset>(PM, PE, h);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      h = kReset && rs_now[s] ? u[s] : fma2(a[s], h, u[s]);
      const int t = t0 + s;
      if (t < p.seq && ln.ok0)
        Pair<T, kVec>::store(y + int64_t(t) * p.channels, h, ln.step, ln.ok0, ln.ok1);
    }
  }
  if (p.hT != nullptr && rank == 0 && warp == 0)
    store_f2(p.hT + int64_t(b) * p.channels, carry, ln);
}

// ------------------------------------------------------------------ backward

constexpr int kBwdWarps = 16;

template <typename T, bool kVec, bool kReset>
__global__ void __launch_bounds__(kBwdWarps * 32)
    gated_scan_bwd_kernel(const BwdArgs p) {
  constexpr int W = kBwdWarps, S = kTile / W;
  __shared__ float4 segf[2][W][32];  // (A0, A1, E0, E1) of each run
  __shared__ float2 segb[2][W][32];  // G of each run: c_out = A c_in + G
  __shared__ float4 sum[2][kMaxCluster][32];
  __shared__ float2 red[W][32];
  cg::cluster_group cluster = cg::this_cluster();
  const int csize = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int unit = int(blockIdx.x) / csize;
  const int b = unit / p.chan_tiles;
  const Lane ln = lane_of<kVec>(unit - b * p.chan_tiles, p.channels);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = (p.seq + kTile - 1) / kTile;
  const int64_t row0 = int64_t(b) * p.seq;
  const T* x = static_cast<const T*>(p.x) + row0 * p.xs + ln.c;
  const T* r = static_cast<const T*>(p.r) + row0 * p.rs + ln.c;
  const T* iv = static_cast<const T*>(p.i) + row0 * p.is + ln.c;
  const T* dy = static_cast<const T*>(p.dy) + (p.dy ? row0 * p.dys + ln.c : 0);
  const int64_t out0 = row0 * p.channels + ln.c;
  const uint8_t* rst = kReset ? p.reset + row0 : nullptr;
  const float2 lam = load_f2(p.lambda, ln);
  const float2 rate = make_float2(p.sharpness * softplus_acc(lam.x), p.sharpness * softplus_acc(lam.y));
  float2 carry = load_f2(p.dhT ? p.dhT + int64_t(b) * p.channels : nullptr, ln);
  float2 dlam = bc2(0.f);

  Pair<T, kVec> xr[S], rr[S], ir[S], gr[S];
  bool rs[S];
  float2 start;
  auto load = [&](int tile) {
    const int t0 = tile * kTile + warp * S;
    start = bc2(0.f);
    if (tile >= 0)
      start = load_f2(p.ckpt + (int64_t(b) * tiles + tile) * p.channels, ln);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int t = t0 + s;
      const bool in = t >= 0 && t < p.seq;
      if (kReset) rs[s] = in && rst[t] != 0;
      if (in && ln.ok0) {
        xr[s].load(x + t * p.xs, ln.step, ln.ok0, ln.ok1);
        rr[s].load(r + t * p.rs, ln.step, ln.ok0, ln.ok1);
        ir[s].load(iv + t * p.is, ln.step, ln.ok0, ln.ok1);
        if (p.dy != nullptr) gr[s].load(dy + t * p.dys, ln.step, ln.ok0, ln.ok1);
        else gr[s] = Pair<T, kVec>{};
      } else {
        xr[s] = rr[s] = ir[s] = gr[s] = Pair<T, kVec>{};
      }
    }
  };

  // the cluster's tiles are taken from the end: rank 0 the last of each group
  load(tiles - 1 - rank);
  if (csize > 1) cluster.sync();  // every CTA has begun before its shared memory is written
  int buf = 0;
  for (int done = 0; done < tiles; done += csize, buf ^= 1) {
    const int tile = tiles - 1 - done - rank;  // below 0: an empty tile
    const int t0 = tile * kTile + warp * S;
    float2 a[S], sr[S], si[S], xv[S], ib[S], q[S], g[S];
    bool drop[S];
    float2 M = bc2(0.f), E = bc2(0.f), G = bc2(0.f);
    const float2 h_tile = start;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      sr[s] = sigmoid2(rr[s].get());
      si[s] = sigmoid2(ir[s].get());
      xv[s] = xr[s].get();
      g[s] = gr[s].get();
      float2 m;
      decay2(mul2(rate, sr[s]), m, q[s]);
      ib[s] = inv_sqrt2(q[s]);
      drop[s] = kReset && rs[s];
      const int t = t0 + s;
      if (t < 0 || t >= p.seq) m = bc2(0.f);  // nothing there: c passes through (g is 0)
      a[s] = add2(m, bc2(1.f));
      const float2 v = mul2(si[s], xv[s]);
      if (drop[s]) {
        a[s] = bc2(0.f);
        E = v;
        M = bc2(-1.f);
      } else {
        E = fma2(a[s], E, mul2(mul2(q[s], ib[s]), v));
        M = join_decay(M, m);
      }
    }
#pragma unroll
    for (int s = S - 1; s >= 0; --s) G = drop[s] ? bc2(0.f) : mul2(a[s], add2(g[s], G));
    segf[buf][warp][lane] = make_float4(M.x, M.y, E.x, E.y);
    segb[buf][warp][lane] = G;
    if (done + csize < tiles) load(tile - csize);
    __syncthreads();
    float2 h = h_tile, PM = bc2(0.f), PG = bc2(0.f), TM = bc2(0.f), TG = bc2(0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < warp) {
        const float4 f = segf[buf][w][lane];
        h = apply<kReset>(make_float2(f.x, f.y), make_float2(f.z, f.w), h);
      }
    }
#pragma unroll
    for (int w = W - 1; w >= 0; --w) {
      if (w == warp) {
        PM = TM;
        PG = TG;
      }
      const float4 f = segf[buf][w][lane];
      const float2 fm = make_float2(f.x, f.y);
      TG = apply<kReset>(fm, segb[buf][w][lane], TG);
      TM = join_decay(TM, fm);
    }
    float2 c = carry;
    if (csize > 1) {
      if (warp < csize)
        *cluster.map_shared_rank(&sum[buf][rank][lane], warp) = make_float4(TM.x, TM.y, TG.x, TG.y);
      cluster.sync();
      for (int k = 0; k < csize; ++k) {
        if (k == rank) c = carry;
        const float4 f = sum[buf][k][lane];
        carry = apply<kReset>(make_float2(f.x, f.y), make_float2(f.z, f.w), carry);
      }
    } else {
      carry = apply<kReset>(TM, TG, carry);
    }
    c = apply<kReset>(PM, PG, c);
    // h[t-1] of each step forwards, then the gradients backwards
    float2 hp[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      hp[s] = h;
      const float2 v = mul2(si[s], xv[s]);
      h = drop[s] ? v : fma2(a[s], h, mul2(mul2(q[s], ib[s]), v));
    }
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      const int t = t0 + s;
      const float2 gs = add2(g[s], c);
      c = drop[s] ? bc2(0.f) : mul2(a[s], gs);
      const float2 beta = drop[s] ? bc2(1.f) : mul2(q[s], ib[s]);
      const float2 gb = mul2(gs, beta);
      const float2 dx = mul2(gb, si[s]);
      const float2 di = mul2(mul2(dx, xv[s]), fma2(neg2(si[s]), bc2(1.f), bc2(1.f)));
      // dL = g (a^2 / beta s(i) x - a h[t-1])
      const float2 slope = mul2(mul2(a[s], ib[s]), mul2(si[s], xv[s]));
      float2 dl = mul2(c, add2(slope, neg2(hp[s])));
      if (drop[s] || t < 0 || t >= p.seq) dl = bc2(0.f);
      const float2 ds = mul2(dl, sr[s]);
      const float2 dr = mul2(mul2(ds, rate), fma2(neg2(sr[s]), bc2(1.f), bc2(1.f)));
      dlam = add2(dlam, ds);
      if (t >= 0 && t < p.seq && ln.ok0) {
        const int64_t o = out0 + int64_t(t) * p.channels;
        Pair<T, kVec>::store(static_cast<T*>(p.dx) + o, dx, ln.step, ln.ok0, ln.ok1);
        Pair<T, kVec>::store(static_cast<T*>(p.dr) + o, dr, ln.step, ln.ok0, ln.ok1);
        Pair<T, kVec>::store(static_cast<T*>(p.di) + o, di, ln.step, ln.ok0, ln.ok1);
      }
    }
  }
  if (p.dh0 != nullptr && rank == 0 && warp == 0)
    store_f2(p.dh0 + int64_t(b) * p.channels, carry, ln);
  red[warp][lane] = dlam;
  __syncthreads();
  if (warp == 0) {
    float2 t = red[0][lane];
    for (int w = 1; w < W; ++w) t = add2(t, red[w][lane]);
    store_f2(p.part + (int64_t(b) * csize + rank) * p.channels, t, ln);
  }
}

// dLambda[ch] = c s(Lambda) sum over rows of part, in a fixed order.
__global__ void __launch_bounds__(256)
    gated_scan_dlambda_kernel(const float* __restrict__ part, const float* __restrict__ lambda,
                              float* __restrict__ out, int rows, int channels, float sharpness) {
  __shared__ float red[8][32];
  const int l = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int ch = blockIdx.x * 32 + l;
  float s = 0.f;
  if (ch < channels)
    for (int k = w; k < rows; k += 8) s += part[int64_t(k) * channels + ch];
  red[w][l] = s;
  __syncthreads();
  if (w == 0 && ch < channels) {
    for (int k = 1; k < 8; ++k) s += red[k][l];
    out[ch] = s * sharpness / (1.f + expf(-lambda[ch]));
  }
}

// ------------------------------------------------------------------ one token

template <typename T, bool kVec>
__global__ void __launch_bounds__(128)
    gated_step_kernel(const T* __restrict__ x, const T* __restrict__ r, const T* __restrict__ i,
                      int64_t xs, int64_t rs, int64_t is, const float* __restrict__ lambda,
                      float* __restrict__ h, T* __restrict__ y, int64_t batch, int channels,
                      int pairs, float sharpness) {
  const int64_t n = int64_t(blockIdx.x) * 128 + threadIdx.x;
  const int64_t b = n / pairs;
  if (b >= batch) return;
  Lane ln;
  ln.step = 1;
  ln.c = int(n - b * pairs) * 2;
  ln.ok0 = true;
  ln.ok1 = ln.c + 1 < channels;
  Pair<T, kVec> xr, rr, ir;
  xr.load(x + b * xs + ln.c, 1, true, ln.ok1);
  rr.load(r + b * rs + ln.c, 1, true, ln.ok1);
  ir.load(i + b * is + ln.c, 1, true, ln.ok1);
  float* hb = h + b * channels;
  const float2 h0 = load_f2(hb, ln);
  const float2 lam = load_f2(lambda, ln);
  const float2 rate = make_float2(sharpness * softplus_acc(lam.x), sharpness * softplus_acc(lam.y));
  float2 m, q;
  decay2(mul2(rate, sigmoid2(rr.get())), m, q);
  const float2 u = mul2(mul2(q, inv_sqrt2(q)), mul2(sigmoid2(ir.get()), xr.get()));
  const float2 hn = fma2(add2(m, bc2(1.f)), h0, u);
  store_f2(hb, hn, ln);
  Pair<T, kVec>::store(y + b * channels + ln.c, hn, 1, true, ln.ok1);
}

// ----------------------------------------------------------------------- host

// How many clusters of 1, 2, 4, 8, 16 CTAs of a kernel fit the device at once
// (asked once for each kernel and device; a repeated question gives the same answer).
struct Fit {
  std::atomic<int> known{0};
  std::atomic<int> clusters[5];
};

template <typename K>
void ask_fit(K kernel, int threads, Fit& fit) {
  cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  for (int k = 0; k < 5; ++k) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1u << k);
    cfg.blockDim = dim3(unsigned(threads));
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1u << k;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) n = 0;
    cudaGetLastError();
    fit.clusters[k].store(n);
  }
  fit.known.store(1);
}

// Cluster size: the CTAs of a cluster take consecutive tiles of one sequence. The
// one that needs the fewest rounds of a tile, by how many clusters fit at once; no
// more CTAs than tiles.
template <auto kernel>
int cluster_size(int threads, int64_t units, int tiles) {
  static Fit fits[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
  Fit& fit = fits[dev];
  if (!fit.known.load()) ask_fit(kernel, threads, fit);
  int best = 1;
  int64_t least = INT64_MAX;
  for (int k = 0; k < 5; ++k) {
    const int c = 1 << k, n = fit.clusters[k].load();
    if (c > tiles || n <= 0) break;
    const int64_t rounds = ((units + n - 1) / n) * ((tiles + c - 1) / c);
    if (rounds < least) {
      least = rounds;
      best = c;
    }
  }
  return best;
}

template <typename K, typename A>
int launch_clusters(const char* what, K kernel, const A& args, int threads, int64_t units, int c,
                    cudaStream_t st) {
  MQC_REQUIRE(units * c <= 0x7fffffffll, MQC_ERR_UNSUPPORTED, "%s: too many channel tiles", what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(units * c));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = unsigned(c);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(MQC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  return check_launch(what);
}

template <typename T, bool kVec, bool kReset>
int run_fwd(const FwdArgs& f, cudaStream_t st) {
  constexpr auto kernel = &gated_scan_fwd_kernel<T, kVec, kReset>;
  const int64_t units = int64_t(f.batch) * f.chan_tiles;
  const int c = cluster_size<kernel>(kFwdWarps * 32, units, (f.seq + kTile - 1) / kTile);
  return launch_clusters("mqc_gated_scan_fwd", kernel, f, kFwdWarps * 32, units, c, st);
}

template <typename T, bool kVec, bool kReset>
int run_bwd(const BwdArgs& f, float* dlambda, cudaStream_t st) {
  constexpr auto kernel = &gated_scan_bwd_kernel<T, kVec, kReset>;
  const int64_t units = int64_t(f.batch) * f.chan_tiles;
  const int c = cluster_size<kernel>(kBwdWarps * 32, units, (f.seq + kTile - 1) / kTile);
  if (int rc = launch_clusters("mqc_gated_scan_bwd", kernel, f, kBwdWarps * 32, units, c, st))
    return rc;
  gated_scan_dlambda_kernel<<<(f.channels + 31) / 32, 256, 0, st>>>(
      f.part, f.lambda, dlambda, f.batch * c, f.channels, f.sharpness);
  return check_launch("mqc_gated_scan_bwd (dLambda)");
}

int check_sizes(const char* what, const mqc_gated_scan_args* a) {
  MQC_REQUIRE(a != nullptr, MQC_ERR_INVALID_VALUE, "%s: args is NULL", what);
  MQC_REQUIRE(dtype_ok(a->dtype), MQC_ERR_INVALID_VALUE, "%s: dtype %d", what, a->dtype);
  MQC_REQUIRE(a->batch >= 0 && a->seq_len >= 0 && a->channels >= 0, MQC_ERR_INVALID_VALUE,
              "%s: batch %lld, seq_len %lld, channels %lld", what, (long long)a->batch,
              (long long)a->seq_len, (long long)a->channels);
  MQC_REQUIRE(a->seq_len <= 0x7fffffff - 2 * kMaxCluster * kTile && a->channels <= 0x7fffffff - kChan &&
                  a->batch <= 0x7fffffff / kMaxCluster,
              MQC_ERR_UNSUPPORTED, "%s: a size above 2^31", what);
  MQC_REQUIRE(a->sharpness > 0.f, MQC_ERR_INVALID_VALUE, "%s: sharpness %g", what,
              double(a->sharpness));
  return MQC_OK;
}

int check_inputs(const char* what, const mqc_gated_scan_args* a) {
  MQC_REQUIRE(a->x && a->r && a->i && a->lambda_, MQC_ERR_INVALID_VALUE,
              "%s: x, r, i or lambda is NULL", what);
  MQC_REQUIRE(a->x_row >= a->channels && a->r_row >= a->channels && a->i_row >= a->channels,
              MQC_ERR_INVALID_VALUE, "%s: a row stride is below channels", what);
  const uintptr_t es = dtype_size(a->dtype);
  MQC_REQUIRE(aligned(a->x, es) && aligned(a->r, es) && aligned(a->i, es) && aligned(a->lambda_, 4),
              MQC_ERR_MISALIGNED, "%s: a pointer is not aligned to its type", what);
  return MQC_OK;
}

// Adjacent channel pairs can move as one word: even widths and strides, aligned bases.
bool pairs_ok(int64_t channels, uintptr_t es, std::initializer_list<const void*> ptrs,
              std::initializer_list<int64_t> strides) {
  if (channels % 2) return false;
  for (const void* q : ptrs)
    if (!aligned(q, 2 * es)) return false;
  for (int64_t s : strides)
    if (s % 2) return false;
  return true;
}

}  // namespace
}  // namespace mqc

extern "C" {

int mqc_gated_scan_fwd(const mqc_gated_scan_args* a, void* stream) {
  using namespace mqc;
  clear_error();
  if (int rc = check_sizes("mqc_gated_scan_fwd", a)) return rc;
  if (a->batch == 0 || a->channels == 0) return MQC_OK;
  cudaStream_t st = as_stream(stream);
  if (a->seq_len == 0) {
    if (a->hT == nullptr) return MQC_OK;
    const size_t bytes = size_t(a->batch) * size_t(a->channels) * 4;
    cudaError_t e = a->h0 ? cudaMemcpyAsync(a->hT, a->h0, bytes, cudaMemcpyDeviceToDevice, st)
                          : cudaMemsetAsync(a->hT, 0, bytes, st);
    MQC_REQUIRE(e == cudaSuccess, MQC_ERR_CUDA, "mqc_gated_scan_fwd: %s", cudaGetErrorString(e));
    return MQC_OK;
  }
  if (int rc = check_inputs("mqc_gated_scan_fwd", a)) return rc;
  const uintptr_t es = dtype_size(a->dtype);
  MQC_REQUIRE(a->y && aligned(a->y, es), MQC_ERR_INVALID_VALUE,
              "mqc_gated_scan_fwd: y is NULL or misaligned");
  MQC_REQUIRE(aligned(a->h0, 4) && aligned(a->hT, 4) && aligned(a->ckpt, 4), MQC_ERR_MISALIGNED,
              "mqc_gated_scan_fwd: h0, hT or ckpt is misaligned");
  FwdArgs f = {a->x, a->r, a->i, a->x_row, a->r_row, a->i_row,
               static_cast<const float*>(a->lambda_), static_cast<const float*>(a->h0),
               static_cast<const uint8_t*>(a->reset), a->y, static_cast<float*>(a->hT),
               static_cast<float*>(a->ckpt), int(a->batch), int(a->seq_len), int(a->channels),
               int((a->channels + kChan - 1) / kChan), a->sharpness};
  const bool vec = pairs_ok(a->channels, es, {a->x, a->r, a->i, a->y}, {a->x_row, a->r_row, a->i_row});
  const bool rst = a->reset != nullptr, f32 = a->dtype == MQC_DTYPE_F32;
#define MQC_RUN(T) \
  (vec ? (rst ? run_fwd<T, true, true>(f, st) : run_fwd<T, true, false>(f, st)) \
       : (rst ? run_fwd<T, false, true>(f, st) : run_fwd<T, false, false>(f, st)))
  return f32 ? MQC_RUN(float) : MQC_RUN(__nv_bfloat16);
#undef MQC_RUN
}

size_t mqc_gated_scan_bwd_workspace_size(int64_t batch, int64_t seq_len, int64_t channels) {
  if (batch <= 0 || seq_len <= 0 || channels <= 0) return 0;
  return size_t(batch) * size_t(channels) * mqc::kMaxCluster * sizeof(float);
}

int mqc_gated_scan_bwd(const mqc_gated_scan_args* a, void* workspace, size_t workspace_bytes,
                       void* stream) {
  using namespace mqc;
  clear_error();
  if (int rc = check_sizes("mqc_gated_scan_bwd", a)) return rc;
  if (a->channels == 0) return MQC_OK;
  MQC_REQUIRE(a->dlambda && aligned(a->dlambda, 4), MQC_ERR_INVALID_VALUE,
              "mqc_gated_scan_bwd: dlambda is NULL or misaligned");
  cudaStream_t st = as_stream(stream);
  if (a->batch == 0 || a->seq_len == 0) {
    cudaError_t e = cudaMemsetAsync(a->dlambda, 0, size_t(a->channels) * 4, st);
    if (e == cudaSuccess && a->dh0 != nullptr && a->batch > 0) {
      const size_t bytes = size_t(a->batch) * size_t(a->channels) * 4;
      e = a->dhT ? cudaMemcpyAsync(a->dh0, a->dhT, bytes, cudaMemcpyDeviceToDevice, st)
                 : cudaMemsetAsync(a->dh0, 0, bytes, st);
    }
    MQC_REQUIRE(e == cudaSuccess, MQC_ERR_CUDA, "mqc_gated_scan_bwd: %s", cudaGetErrorString(e));
    return MQC_OK;
  }
  if (int rc = check_inputs("mqc_gated_scan_bwd", a)) return rc;
  const uintptr_t es = dtype_size(a->dtype);
  MQC_REQUIRE(a->ckpt && a->dx && a->dr && a->di, MQC_ERR_INVALID_VALUE,
              "mqc_gated_scan_bwd: ckpt, dx, dr or di is NULL");
  MQC_REQUIRE(a->dy == nullptr || a->dy_row >= a->channels, MQC_ERR_INVALID_VALUE,
              "mqc_gated_scan_bwd: dy's row stride is below channels");
  MQC_REQUIRE(aligned(a->dy, es) && aligned(a->dx, es) && aligned(a->dr, es) &&
                  aligned(a->di, es) && aligned(a->ckpt, 4) && aligned(a->dhT, 4) &&
                  aligned(a->dh0, 4),
              MQC_ERR_MISALIGNED, "mqc_gated_scan_bwd: a pointer is not aligned to its type");
  MQC_REQUIRE(workspace && aligned(workspace, 4) &&
                  workspace_bytes >= mqc_gated_scan_bwd_workspace_size(a->batch, a->seq_len, a->channels),
              MQC_ERR_INVALID_VALUE, "mqc_gated_scan_bwd: workspace of %zu bytes is too small",
              workspace_bytes);
  BwdArgs f = {a->x, a->r, a->i, a->dy, a->x_row, a->r_row, a->i_row, a->dy_row,
               static_cast<const float*>(a->lambda_), static_cast<const uint8_t*>(a->reset),
               static_cast<const float*>(a->ckpt), static_cast<const float*>(a->dhT), a->dx, a->dr,
               a->di, static_cast<float*>(a->dh0), static_cast<float*>(workspace), int(a->batch),
               int(a->seq_len), int(a->channels), int((a->channels + kChan - 1) / kChan),
               a->sharpness};
  float* dl = static_cast<float*>(a->dlambda);
  const bool vec = pairs_ok(a->channels, es, {a->x, a->r, a->i, a->dy, a->dx, a->dr, a->di},
                            {a->x_row, a->r_row, a->i_row, a->dy ? a->dy_row : 0});
  const bool rst = a->reset != nullptr, f32 = a->dtype == MQC_DTYPE_F32;
#define MQC_RUN(T) \
  (vec ? (rst ? run_bwd<T, true, true>(f, dl, st) : run_bwd<T, true, false>(f, dl, st)) \
       : (rst ? run_bwd<T, false, true>(f, dl, st) : run_bwd<T, false, false>(f, dl, st)))
  return f32 ? MQC_RUN(float) : MQC_RUN(__nv_bfloat16);
#undef MQC_RUN
}

int mqc_gated_scan_step(const void* x, int64_t x_row, const void* r, int64_t r_row, const void* i,
                        int64_t i_row, const void* lambda_, void* h, void* y, int64_t batch,
                        int64_t channels, float sharpness, int dtype, void* stream) {
  using namespace mqc;
  clear_error();
  MQC_REQUIRE(dtype_ok(dtype), MQC_ERR_INVALID_VALUE, "mqc_gated_scan_step: dtype %d", dtype);
  MQC_REQUIRE(batch >= 0 && channels >= 0 && channels <= 0x7ffffffe && sharpness > 0.f,
              MQC_ERR_INVALID_VALUE, "mqc_gated_scan_step: batch %lld, channels %lld, sharpness %g",
              (long long)batch, (long long)channels, double(sharpness));
  if (batch == 0 || channels == 0) return MQC_OK;
  const uintptr_t es = dtype_size(dtype);
  MQC_REQUIRE(x && r && i && lambda_ && h && y, MQC_ERR_INVALID_VALUE,
              "mqc_gated_scan_step: a pointer is NULL");
  MQC_REQUIRE(x_row >= channels && r_row >= channels && i_row >= channels, MQC_ERR_INVALID_VALUE,
              "mqc_gated_scan_step: a row stride is below channels");
  MQC_REQUIRE(aligned(x, es) && aligned(r, es) && aligned(i, es) && aligned(y, es) &&
                  aligned(lambda_, 4) && aligned(h, 4),
              MQC_ERR_MISALIGNED, "mqc_gated_scan_step: a pointer is not aligned to its type");
  const int pairs = int((channels + 1) / 2);
  const int64_t blocks = (batch * pairs + 127) / 128;
  MQC_REQUIRE(blocks <= 0x7fffffffll, MQC_ERR_UNSUPPORTED, "mqc_gated_scan_step: too large");
  const bool vec = pairs_ok(channels, es, {x, r, i, y}, {x_row, r_row, i_row});
  cudaStream_t st = as_stream(stream);
#define MQC_STEP(T, V)                                                                       \
  gated_step_kernel<T, V><<<unsigned(blocks), 128, 0, st>>>(                                 \
      static_cast<const T*>(x), static_cast<const T*>(r), static_cast<const T*>(i), x_row,   \
      r_row, i_row, static_cast<const float*>(lambda_), static_cast<float*>(h),              \
      static_cast<T*>(y), batch, int(channels), pairs, sharpness)
  if (dtype == MQC_DTYPE_F32) {
    if (vec) MQC_STEP(float, true);
    else MQC_STEP(float, false);
  } else {
    if (vec) MQC_STEP(__nv_bfloat16, true);
    else MQC_STEP(__nv_bfloat16, false);
  }
#undef MQC_STEP
  return check_launch("mqc_gated_scan_step");
}

}  // extern "C"
