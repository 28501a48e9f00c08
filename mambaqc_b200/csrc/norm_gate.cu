// The residual epilogue of a block, fused over each row, and its gradient:
//
//   out = x + scale * s(z) * P(y)        n = Q(out)         s = sigmoid
//
// P (the norm after the block's last projection) and Q (the norm before the next
// block) are LayerNorm or RMSNorm over the row with their own weight and bias; Q
// is optional, and with only Q the kernel is the norm in front of the first block.
//
// Gradient, from dout and dn (D columns, means over a row):
//   d  = dout + Qr (dn wq - m(dn wq) - nhat m(dn wq nhat))   (RMS: without the first mean)
//   dx = d     dp = d scale s(z)     dz = d scale P s(z) (1 - s(z))
//   dy = Pr (dp wp - m(dp wp) - yhat m(dp wp yhat))
//   column sums: dwp = dp yhat, dbp = dp, dscale = d s(z) P, dwq = dn nhat, dbq = dn
// out is computed again from x, y and z: reading it back would cost as much and
// would carry its rounding into dwq.
//
// Both passes are streams, bound by the row tensors' bytes. A CTA owns whole rows
// and a thread the same few columns of each, so the parameters and the five column
// sums stay in registers; the rows of the next step are loaded before this step is
// reduced. Rows are dealt to CTAs by a fixed rule and the CTAs' column sums are
// joined by a second kernel in a fixed order.
#include <type_traits>

#include "mqc_common.cuh"
#include "mqc_host.h"

namespace mqc {
namespace {

constexpr int kMaxThreads = 512;
constexpr int kMaxWarps = kMaxThreads / 32;
constexpr int kMaxWidth = MQC_NORM_GATE_MAX_WIDTH;
static_assert(kMaxWidth <= kMaxThreads * 8, "at most eight columns a thread");
constexpr int kSums = 5;  // column sums: dwp, dscale, dbp, dwq, dbq

template <typename T, int V>
struct Vec;
template <>
struct Vec<float, 4> {
  float4 v;
  __device__ __forceinline__ void load(const float* p) { v = __ldg(reinterpret_cast<const float4*>(p)); }
  __device__ __forceinline__ void get(float (&o)[4]) const { o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w; }
  static __device__ __forceinline__ void store(float* p, const float (&o)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(o[0], o[1], o[2], o[3]);
  }
};
template <>
struct Vec<__nv_bfloat16, 4> {
  uint2 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldg(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void get(float (&o)[4]) const {
    const float4 f = QIO<__nv_bfloat16>::unpack(v);
    o[0] = f.x; o[1] = f.y; o[2] = f.z; o[3] = f.w;
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&o)[4]) {
    QIO<__nv_bfloat16>::st(p, make_float4(o[0], o[1], o[2], o[3]));
  }
};
template <typename T>
struct Vec<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = __ldg(p); }
  __device__ __forceinline__ void get(float (&o)[1]) const { o[0] = to_f(v); }
  static __device__ __forceinline__ void store(T* p, const float (&o)[1]) { QIO<T>::st1(p, o[0]); }
};

// 1 / (1 + e^-v); e^-v is held below 2^126, a NaN stays one
__device__ __forceinline__ float sigmoid_s(float v) {
  float e = v * -1.44269504088896341f, d, r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(e) : "f"(e), "f"(126.f));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(e));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d + 1.f));
  return r;
}

// Sums of N values over the CTA, one barrier. `red` is used in turns of two, so a
// thread that is still reading one turn's sums is never overwritten by the next.
template <int N>
__device__ __forceinline__ void cta_sums(float (&v)[N], float (*red)[kMaxWarps][N], int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return;
  const int w = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int k = 0; k < N; ++k) red[turn][w][k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = red[turn][0][k];
  for (int j = 1; j < warps; ++j)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += red[turn][j][k];
  turn ^= 1;
}

struct FwdArgs {
  const void *x, *y, *z;
  int64_t z_row;
  const float *wp, *bp, *scale, *wq, *bq;
  void *out, *n;
  float4* stats;  // per row: mean and 1/std of P, of Q; or NULL
  int64_t rows;
  int width, layer;
  float eps;
};

// A parameter's values at this thread's columns: kept in registers where a thread
// has up to four columns, else read again (from L1 and L2) for each row, as the
// registers are needed for the rows themselves.
template <int V, int C>
struct Cols {
  static constexpr bool kKeep = V * C <= 4;
  const float* p;
  int width;
  float r[kKeep ? C : 1][V];
  __device__ __forceinline__ void read(int j, float (&o)[V]) const {
    const int c = (j * int(blockDim.x) + int(threadIdx.x)) * V;
    if (p != nullptr && c < width) {
      Vec<float, V> t;
      t.load(p + c);
      t.get(o);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = 0.f;
    }
  }
  __device__ __forceinline__ Cols(const float* ptr, int w) : p(ptr), width(w) {
    if constexpr (kKeep)
#pragma unroll
      for (int j = 0; j < C; ++j) read(j, r[j]);
  }
  __device__ __forceinline__ void get(int j, float (&o)[V]) const {
    if constexpr (kKeep) {
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = r[j][v];
    } else {
      read(j, o);
    }
  }
};

// Normalises R rows in place (u -> uhat) and returns their mean and 1/std.
template <int V, int C, int R>
__device__ __forceinline__ void normalise(float (&u)[R][C][V], int width, bool layer, float eps,
                                          float (*red)[kMaxWarps][R], int& turn, float (&mean)[R],
                                          float (&rstd)[R]) {
  const float inv = 1.f / float(width);
  if (layer) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = 0.f;
#pragma unroll
      for (int j = 0; j < C; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) mean[r] += u[r][j][v];
    }
    cta_sums<R>(mean, red, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] *= inv;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const bool in = (j * int(blockDim.x) + int(threadIdx.x)) * V < width;
#pragma unroll
        for (int v = 0; v < V; ++v) u[r][j][v] = in ? u[r][j][v] - mean[r] : 0.f;
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) mean[r] = 0.f;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    rstd[r] = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) rstd[r] = fmaf(u[r][j][v], u[r][j][v], rstd[r]);
  }
  cta_sums<R>(rstd, red, turn);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    rstd[r] = 1.f / sqrtf(fmaf(rstd[r], inv, eps));
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) u[r][j][v] *= rstd[r];
  }
}

template <typename TX, typename TY, int V, int C, int R, bool kPost>
__global__ void __launch_bounds__(kMaxThreads)
    norm_gate_fwd_kernel(const FwdArgs p) {
  __shared__ float red[2][kMaxWarps][R];
  int turn = 0;
  const int T = blockDim.x, tid = threadIdx.x;
  const bool layer = p.layer != 0, next = p.n != nullptr;
  const Cols<V, C> wps(kPost ? p.wp : nullptr, p.width), bps(kPost ? p.bp : nullptr, p.width),
      scs(kPost ? p.scale : nullptr, p.width), wqs(p.wq, p.width), bqs(p.bq, p.width);
  Vec<TX, V> xr[R][C];
  Vec<TY, V> yr[R][C], zr[R][C];
  const int64_t step = int64_t(gridDim.x) * R;
  auto load = [&](int64_t row0) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int c = (j * T + tid) * V;
        xr[r][j] = Vec<TX, V>{};
        if (kPost) yr[r][j] = zr[r][j] = Vec<TY, V>{};
        if (row0 + r < p.rows && c < p.width) {
          xr[r][j].load(static_cast<const TX*>(p.x) + (row0 + r) * p.width + c);
          if (kPost) {
            yr[r][j].load(static_cast<const TY*>(p.y) + (row0 + r) * p.width + c);
            zr[r][j].load(static_cast<const TY*>(p.z) + (row0 + r) * p.z_row + c);
          }
        }
      }
  };
  int64_t row0 = int64_t(blockIdx.x) * R;
  load(row0);
  for (; row0 < p.rows; row0 += step) {
    float u[R][C][V], o[R][C][V], mp[R], rp[R], mq[R], rq[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < C; ++j) {
        xr[r][j].get(o[r][j]);
        if (kPost) yr[r][j].get(u[r][j]);
      }
    if constexpr (kPost) {
      float gt[R][C][V];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < C; ++j) {
          zr[r][j].get(gt[r][j]);
          float sc[V];
          scs.get(j, sc);
#pragma unroll
          for (int v = 0; v < V; ++v) gt[r][j][v] = sc[v] * sigmoid_s(gt[r][j][v]);
        }
      load(row0 + step);
      normalise<V, C, R>(u, p.width, layer, p.eps, red, turn, mp, rp);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const int c = (j * T + tid) * V;
          float wp[V], bp[V];
          wps.get(j, wp);
          bps.get(j, bp);
#pragma unroll
          for (int v = 0; v < V; ++v)
            o[r][j][v] = fmaf(gt[r][j][v], fmaf(u[r][j][v], wp[v], bp[v]), o[r][j][v]);
          if (row0 + r < p.rows && c < p.width)
            Vec<TX, V>::store(static_cast<TX*>(p.out) + (row0 + r) * p.width + c, o[r][j]);
        }
    } else {
      load(row0 + step);
#pragma unroll
      for (int r = 0; r < R; ++r) mp[r] = rp[r] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) mq[r] = rq[r] = 0.f;
    if (next) {
      normalise<V, C, R>(o, p.width, layer, p.eps, red, turn, mq, rq);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const int c = (j * T + tid) * V;
          float wq[V], bq[V];
          wqs.get(j, wq);
          bqs.get(j, bq);
#pragma unroll
          for (int v = 0; v < V; ++v) o[r][j][v] = fmaf(o[r][j][v], wq[v], bq[v]);
          if (row0 + r < p.rows && c < p.width)
            Vec<TY, V>::store(static_cast<TY*>(p.n) + (row0 + r) * p.width + c, o[r][j]);
        }
    }
    if (p.stats != nullptr && tid == 0)
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (row0 + r < p.rows) p.stats[row0 + r] = make_float4(mp[r], rp[r], mq[r], rq[r]);
  }
}

struct BwdArgs {
  const void *x, *y, *z;
  int64_t z_row;
  const float *wp, *bp, *scale, *wq;
  const void *dout, *dn;
  const float4* stats;
  void *dx, *dy, *dz;
  float* part;  // [gridDim.x][kSums][width]
  int64_t rows;
  int width, layer;
};

template <typename TX, typename TY, int V, int C, int R, bool kPost>
__global__ void __launch_bounds__(kMaxThreads)
    norm_gate_bwd_kernel(const BwdArgs p) {
  __shared__ float red[2][kMaxWarps][2 * R];
  int turn = 0;
  const int T = blockDim.x, tid = threadIdx.x;
  const bool layer = p.layer != 0, next = p.dn != nullptr;
  const float inv = 1.f / float(p.width);
  const Cols<V, C> wps(kPost ? p.wp : nullptr, p.width), bps(kPost ? p.bp : nullptr, p.width),
      scs(kPost ? p.scale : nullptr, p.width), wqs(p.wq, p.width);
  float cs[kSums][C][V];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) cs[k][j][v] = 0.f;
  Vec<TX, V> xr[R][C], gr[R][C];
  Vec<TY, V> yr[R][C], zr[R][C], nr[R][C];
  float4 st[R];
  const int64_t step = int64_t(gridDim.x) * R;
  auto load = [&](int64_t row0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r;
      st[r] = row < p.rows ? __ldg(p.stats + row) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int c = (j * T + tid) * V;
        xr[r][j] = gr[r][j] = Vec<TX, V>{};
        nr[r][j] = Vec<TY, V>{};
        if (kPost) yr[r][j] = zr[r][j] = Vec<TY, V>{};
        if (row < p.rows && c < p.width) {
          const int64_t at = row * p.width + c;
          if (p.dout != nullptr) gr[r][j].load(static_cast<const TX*>(p.dout) + at);
          if (next) {
            xr[r][j].load(static_cast<const TX*>(p.x) + at);
            nr[r][j].load(static_cast<const TY*>(p.dn) + at);
          }
          if (kPost) {
            yr[r][j].load(static_cast<const TY*>(p.y) + at);
            zr[r][j].load(static_cast<const TY*>(p.z) + row * p.z_row + c);
          }
        }
      }
    }
  };
  int64_t row0 = int64_t(blockIdx.x) * R;
  load(row0);
  for (; row0 < p.rows; row0 += step) {
    // d: dout, then the whole gradient of out; yh: yhat; gt: s(z); nh: nhat; dn
    float d[R][C][V], yh[R][C][V], gt[R][C][V], nh[R][C][V], dn[R][C][V];
    float4 s4[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s4[r] = st[r];
#pragma unroll
      for (int j = 0; j < C; ++j) {
        gr[r][j].get(d[r][j]);
        if (kPost) {
          yr[r][j].get(yh[r][j]);
          zr[r][j].get(gt[r][j]);
        }
        if (next) {
          xr[r][j].get(nh[r][j]);
          nr[r][j].get(dn[r][j]);
        }
      }
    }
    load(row0 + step);
    float sums[2 * R];
    if constexpr (kPost) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            yh[r][j][v] = (yh[r][j][v] - s4[r].x) * s4[r].y;
            gt[r][j][v] = sigmoid_s(gt[r][j][v]);
          }
    }
    if (next) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int j = 0; j < C; ++j) {
          float wq[V], wp[V], bp[V], sc[V];
          wqs.get(j, wq);
          if constexpr (kPost) {
            wps.get(j, wp);
            bps.get(j, bp);
            scs.get(j, sc);
          }
#pragma unroll
          for (int v = 0; v < V; ++v) {
            float o = nh[r][j][v];
            if constexpr (kPost)
              o = fmaf(sc[v] * gt[r][j][v], fmaf(yh[r][j][v], wp[v], bp[v]), o);
            const float h = (o - s4[r].z) * s4[r].w;
            nh[r][j][v] = h;
            cs[3][j][v] = fmaf(dn[r][j][v], h, cs[3][j][v]);
            cs[4][j][v] += dn[r][j][v];
            const float w = dn[r][j][v] * wq[v];
            dn[r][j][v] = w;
            a += w;
            b = fmaf(w, h, b);
          }
        }
        sums[r] = a;
        sums[R + r] = b;
      }
      cta_sums<2 * R>(sums, red, turn);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float a = layer ? sums[r] * inv : 0.f, b = sums[R + r] * inv;
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
          for (int v = 0; v < V; ++v)
            d[r][j][v] = fmaf(s4[r].w, dn[r][j][v] - a - nh[r][j][v] * b, d[r][j][v]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int c = (j * T + tid) * V;
        if (row0 + r < p.rows && c < p.width)
          Vec<TX, V>::store(static_cast<TX*>(p.dx) + (row0 + r) * p.width + c, d[r][j]);
      }
    if constexpr (kPost) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int j = 0; j < C; ++j) {
          float dz[V], wp[V], bp[V], sc[V];
          wps.get(j, wp);
          bps.get(j, bp);
          scs.get(j, sc);
          const int c = (j * T + tid) * V;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float pv = fmaf(yh[r][j][v], wp[v], bp[v]);
            const float dg = d[r][j][v] * gt[r][j][v];       // d s(z)
            const float dp = dg * sc[v];
            dz[v] = dp * pv * (1.f - gt[r][j][v]);
            cs[0][j][v] = fmaf(dp, yh[r][j][v], cs[0][j][v]);
            cs[1][j][v] = fmaf(dg, pv, cs[1][j][v]);
            cs[2][j][v] += dp;
            const float w = dp * wp[v];
            d[r][j][v] = w;
            a += w;
            b = fmaf(w, yh[r][j][v], b);
          }
          if (row0 + r < p.rows && c < p.width)
            Vec<TY, V>::store(static_cast<TY*>(p.dz) + (row0 + r) * p.width + c, dz);
        }
        sums[r] = a;
        sums[R + r] = b;
      }
      cta_sums<2 * R>(sums, red, turn);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float a = layer ? sums[r] * inv : 0.f, b = sums[R + r] * inv;
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const int c = (j * T + tid) * V;
#pragma unroll
          for (int v = 0; v < V; ++v)
            d[r][j][v] = s4[r].y * (d[r][j][v] - a - yh[r][j][v] * b);
          if (row0 + r < p.rows && c < p.width)
            Vec<TY, V>::store(static_cast<TY*>(p.dy) + (row0 + r) * p.width + c, d[r][j]);
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kSums; ++k) {
    if ((k < 3 && !kPost) || (k >= 3 && !next)) continue;
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = (j * T + tid) * V + v;
        if (c < p.width) p.part[(int64_t(blockIdx.x) * kSums + k) * p.width + c] = cs[k][j][v];
      }
  }
}

struct SumArgs {
  const float* part;
  float* out[kSums];  // NULL: not wanted
  int ctas, width;
};

// out[k][c] = sum over CTAs of part[cta][k][c]: 32 columns a block, 8 slices of CTAs.
__global__ void __launch_bounds__(256) norm_gate_sum_kernel(const SumArgs p) {
  __shared__ float red[8][32];
  const int k = blockIdx.y;
  if (p.out[k] == nullptr) return;
  const int l = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + l;
  float s = 0.f;
  if (c < p.width)
    for (int i = w; i < p.ctas; i += 8) s += p.part[(int64_t(i) * kSums + k) * p.width + c];
  red[w][l] = s;
  __syncthreads();
  if (w == 0 && c < p.width) {
    for (int j = 1; j < 8; ++j) s += red[j][l];
    p.out[k][c] = s;
  }
}

// ----------------------------------------------------------------------- host

// Threads of a CTA (a multiple of 32) and columns a thread: C chunks of V.
struct Shape {
  int threads, chunks;
};

Shape shape_of(int width, bool vec) {
  const int groups = vec ? (width + 3) / 4 : width;
  const int most = vec ? 2 : 8;
  int c = 1;
  // 256 threads up to four columns each, then 512
  while (c < most && (groups + c - 1) / c > (c * (vec ? 4 : 1) < 4 ? 256 : kMaxThreads)) c *= 2;
  const int t = ((groups + c - 1) / c + 31) / 32 * 32;
  return {t, c};
}

constexpr int kFwdCtas = 2048 / 256;  // resident threads aimed at, in CTAs of 256
constexpr int kBwdThreads = 1024;     // per SM: each CTA leaves kSums rows of partial sums

int fwd_grid(int threads, int64_t rows, int r) {
  const int64_t most = int64_t(num_sms()) * (kFwdCtas * 256 / threads > 0 ? kFwdCtas * 256 / threads : 1);
  const int64_t want = (rows + r - 1) / r;
  return int(want < most ? want : most);
}

int bwd_grid(int threads, int64_t rows, int r) {
  int per = kBwdThreads / threads;
  if (per < 1) per = 1;
  if (per > 8) per = 8;
  const int64_t most = int64_t(num_sms()) * per, want = (rows + r - 1) / r;
  return int(want < most ? want : most);
}

constexpr int kRows = 2;  // rows a CTA works on at once where a thread has 4 columns

template <typename TX, typename TY, int V, int C, bool kPost>
int launch_fwd(const FwdArgs& f, int threads, cudaStream_t st) {
  constexpr int R = V * C <= 4 ? kRows : 1;
  norm_gate_fwd_kernel<TX, TY, V, C, R, kPost>
      <<<fwd_grid(threads, f.rows, R), threads, 0, st>>>(f);
  return check_launch("mqc_norm_gate_fwd");
}

template <typename TX, typename TY, int V, int C, bool kPost>
int launch_bwd(const BwdArgs& f, int threads, int* ctas, cudaStream_t st) {
  constexpr int R = 1;
  *ctas = bwd_grid(threads, f.rows, R);
  norm_gate_bwd_kernel<TX, TY, V, C, R, kPost><<<*ctas, threads, 0, st>>>(f);
  return check_launch("mqc_norm_gate_bwd");
}

template <typename TX, typename TY, bool kPost, typename F>
int by_shape(Shape s, bool vec, F f) {
  if (vec) {
    return s.chunks == 1 ? f(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{})
                         : f(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
  }
  switch (s.chunks) {
    case 1: return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
    case 4: return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
    default: return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
  }
}

template <typename F>
int by_types(int xd, int yd, bool post, F f) {
  const bool xf = xd == MQC_DTYPE_F32, yf = yd == MQC_DTYPE_F32;
  float a = 0;
  __nv_bfloat16 b{};
  if (xf && yf) return post ? f(a, a, std::true_type{}) : f(a, a, std::false_type{});
  if (xf) return post ? f(a, b, std::true_type{}) : f(a, b, std::false_type{});
  return post ? f(b, b, std::true_type{}) : f(b, b, std::false_type{});
}

int check(const char* what, const mqc_norm_gate_args* a, bool* post, bool* next) {
  MQC_REQUIRE(a != nullptr, MQC_ERR_INVALID_VALUE, "%s: args is NULL", what);
  MQC_REQUIRE(dtype_ok(a->x_dtype) && dtype_ok(a->y_dtype), MQC_ERR_INVALID_VALUE,
              "%s: dtype %d / %d", what, a->x_dtype, a->y_dtype);
  MQC_REQUIRE(!(a->x_dtype == MQC_DTYPE_BF16 && a->y_dtype == MQC_DTYPE_F32), MQC_ERR_UNSUPPORTED,
              "%s: a bf16 residual with fp32 branches", what);
  MQC_REQUIRE(a->rows >= 0 && a->width >= 0, MQC_ERR_INVALID_VALUE, "%s: rows %lld, width %lld",
              what, (long long)a->rows, (long long)a->width);
  MQC_REQUIRE(a->width <= kMaxWidth, MQC_ERR_UNSUPPORTED, "%s: width %lld (at most %d)", what,
              (long long)a->width, kMaxWidth);
  MQC_REQUIRE(a->norm == MQC_NORM_LAYER || a->norm == MQC_NORM_RMS, MQC_ERR_INVALID_VALUE,
              "%s: norm %d", what, a->norm);
  MQC_REQUIRE(a->eps >= 0.f, MQC_ERR_INVALID_VALUE, "%s: eps %g", what, double(a->eps));
  *post = a->y != nullptr;
  *next = a->next_weight != nullptr;
  if (a->rows == 0 || a->width == 0) return MQC_OK;
  const uintptr_t xs = dtype_size(a->x_dtype), ys = dtype_size(a->y_dtype);
  MQC_REQUIRE(*post || *next, MQC_ERR_INVALID_VALUE, "%s: neither y nor next_weight", what);
  MQC_REQUIRE(a->x != nullptr, MQC_ERR_INVALID_VALUE, "%s: x is NULL", what);
  MQC_REQUIRE(!*post || (a->z && a->weight && a->scale && a->z_row >= a->width),
              MQC_ERR_INVALID_VALUE, "%s: z, weight or scale is NULL, or z's row stride is too small",
              what);
  MQC_REQUIRE(aligned(a->x, xs) && aligned(a->y, ys) && aligned(a->z, ys) && aligned(a->weight, 4) &&
                  aligned(a->bias, 4) && aligned(a->scale, 4) && aligned(a->next_weight, 4) &&
                  aligned(a->next_bias, 4) && aligned(a->stats, 16),
              MQC_ERR_MISALIGNED, "%s: a pointer is not aligned to its type", what);
  return MQC_OK;
}

// Rows can move four columns at a time: the width and z's stride divide by four and
// every tensor is aligned to four elements.
bool vec_ok(const mqc_norm_gate_args* a) {
  const uintptr_t xs = 4 * dtype_size(a->x_dtype), ys = 4 * dtype_size(a->y_dtype);
  return a->width % 4 == 0 && (a->z == nullptr || a->z_row % 4 == 0) && aligned(a->x, xs) &&
         aligned(a->out, xs) && aligned(a->dout, xs) && aligned(a->dx, xs) && aligned(a->y, ys) &&
         aligned(a->z, ys) && aligned(a->n, ys) && aligned(a->dn, ys) && aligned(a->dy, ys) &&
         aligned(a->dz, ys) && aligned(a->weight, 16) && aligned(a->bias, 16) &&
         aligned(a->scale, 16) && aligned(a->next_weight, 16) && aligned(a->next_bias, 16);
}

}  // namespace
}  // namespace mqc

extern "C" {

int mqc_norm_gate_fwd(const mqc_norm_gate_args* a, void* stream) {
  using namespace mqc;
  clear_error();
  bool post = false, next = false;
  if (int rc = check("mqc_norm_gate_fwd", a, &post, &next)) return rc;
  if (a->rows == 0 || a->width == 0) return MQC_OK;
  const uintptr_t xs = dtype_size(a->x_dtype), ys = dtype_size(a->y_dtype);
  MQC_REQUIRE(!post || (a->out && aligned(a->out, xs)), MQC_ERR_INVALID_VALUE,
              "mqc_norm_gate_fwd: out is NULL or misaligned");
  MQC_REQUIRE(!next || (a->n && aligned(a->n, ys)), MQC_ERR_INVALID_VALUE,
              "mqc_norm_gate_fwd: n is NULL or misaligned");
  FwdArgs f = {a->x, a->y, a->z, a->z_row, a->weight, a->bias, a->scale, a->next_weight,
               a->next_bias, a->out, next ? a->n : nullptr, static_cast<float4*>(a->stats),
               a->rows, int(a->width), a->norm == MQC_NORM_LAYER, a->eps};
  const bool vec = vec_ok(a);
  const Shape s = shape_of(f.width, vec);
  return by_types(a->x_dtype, a->y_dtype, post, [&](auto tx, auto ty, auto kp) {
    using TX = decltype(tx);
    using TY = decltype(ty);
    constexpr bool kPost = decltype(kp)::value;
    return by_shape<TX, TY, kPost>(s, vec, [&](auto v, auto c) {
      return launch_fwd<TX, TY, decltype(v)::value, decltype(c)::value, kPost>(
          f, s.threads, as_stream(stream));
    });
  });
}

size_t mqc_norm_gate_bwd_workspace_size(int64_t rows, int64_t width) {
  using namespace mqc;
  if (rows <= 0 || width <= 0 || width > kMaxWidth) return 0;
  // the larger grid of the two column layouts
  const int a = bwd_grid(shape_of(int(width), true).threads, rows, 1);
  const int b = bwd_grid(shape_of(int(width), false).threads, rows, 1);
  return size_t(a > b ? a : b) * kSums * size_t(width) * sizeof(float);
}

int mqc_norm_gate_bwd(const mqc_norm_gate_args* a, void* workspace, size_t workspace_bytes,
                      void* stream) {
  using namespace mqc;
  clear_error();
  bool post = false, next = false;
  if (int rc = check("mqc_norm_gate_bwd", a, &post, &next)) return rc;
  next = next && a->dn != nullptr;
  float* outs[kSums] = {a->dweight, a->dscale, a->dbias, a->dnext_weight, a->dnext_bias};
  cudaStream_t st = as_stream(stream);
  const bool empty = a->rows == 0 || a->width == 0;
  for (int k = 0; k < kSums; ++k) {
    MQC_REQUIRE(aligned(outs[k], 4), MQC_ERR_MISALIGNED, "mqc_norm_gate_bwd: a column sum");
    // nothing reaches these sums: no rows (the row tensors may then be NULL), no y, or
    // no gradient of n
    if (outs[k] != nullptr && (empty || (k < 3 && !post) || (k >= 3 && !next))) {
      cudaError_t e = cudaMemsetAsync(outs[k], 0, size_t(a->width) * 4, st);
      MQC_REQUIRE(e == cudaSuccess, MQC_ERR_CUDA, "mqc_norm_gate_bwd: %s", cudaGetErrorString(e));
      outs[k] = nullptr;
    }
  }
  if (empty) return MQC_OK;
  const uintptr_t xs = dtype_size(a->x_dtype), ys = dtype_size(a->y_dtype);
  MQC_REQUIRE(a->stats && a->dx && (!post || (a->dy && a->dz)), MQC_ERR_INVALID_VALUE,
              "mqc_norm_gate_bwd: stats, dx, dy or dz is NULL");
  MQC_REQUIRE(aligned(a->dx, xs) && aligned(a->dout, xs) && aligned(a->dn, ys) &&
                  aligned(a->dy, ys) && aligned(a->dz, ys),
              MQC_ERR_MISALIGNED, "mqc_norm_gate_bwd: a pointer is not aligned to its type");
  MQC_REQUIRE(workspace && aligned(workspace, 4) &&
                  workspace_bytes >= mqc_norm_gate_bwd_workspace_size(a->rows, a->width),
              MQC_ERR_INVALID_VALUE, "mqc_norm_gate_bwd: workspace of %zu bytes is too small",
              workspace_bytes);
  BwdArgs f = {a->x, a->y, a->z, a->z_row, a->weight, a->bias, a->scale, a->next_weight,
               a->dout, next ? a->dn : nullptr, static_cast<const float4*>(a->stats),
               a->dx, a->dy, a->dz, static_cast<float*>(workspace), a->rows, int(a->width),
               a->norm == MQC_NORM_LAYER};
  const bool vec = vec_ok(a);
  const Shape s = shape_of(f.width, vec);
  int ctas = 0;
  int rc = by_types(a->x_dtype, a->y_dtype, post, [&](auto tx, auto ty, auto kp) {
    using TX = decltype(tx);
    using TY = decltype(ty);
    constexpr bool kPost = decltype(kp)::value;
    return by_shape<TX, TY, kPost>(s, vec, [&](auto v, auto c) {
      return launch_bwd<TX, TY, decltype(v)::value, decltype(c)::value, kPost>(f, s.threads, &ctas,
                                                                               st);
    });
  });
  if (rc) return rc;
  SumArgs q;
  q.part = f.part;
  bool any = false;
  for (int k = 0; k < kSums; ++k) {
    q.out[k] = outs[k];
    any = any || outs[k] != nullptr;
  }
  if (!any) return MQC_OK;
  q.ctas = ctas;
  q.width = f.width;
  norm_gate_sum_kernel<<<dim3((f.width + 31) / 32, kSums), 256, 0, st>>>(q);
  return check_launch("mqc_norm_gate_bwd (column sums)");
}

}  // extern "C"
