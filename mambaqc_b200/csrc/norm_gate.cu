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
// Both passes are streams, bound by the row tensors' bytes. Forward, a warp owns a row.
// Backward, a group of threads owns rows and each thread the same eight columns of
// them, so that the parameters and the five column sums stay in registers (a warp a
// row would need 120 registers for the sums alone); the rows of the next two steps are
// on their way into shared memory meanwhile. Rows are dealt to CTAs by a fixed rule and
// the CTAs' column sums are joined by a second kernel in a fixed order.
//
// Measured on one B200, LayerNorm, 8192 x 768, x fp32, y and z bf16: forward 18.7 us
// (13.5 us of bytes at 6.5 TB/s), backward 38.1 and 3.5 us (21.2); RMSNorm, 16384 x 1024,
// bf16: 30.3 (25.7), 60.3 and 3.7 us (41). The backward pass waits: 12 warps an SM (168
// registers), two sums over a group with a barrier each for every row. Slower: 128
// registers with spills (63 us), four columns a thread (44 us), 8 warps an SM (46 us).
#include <type_traits>

#include "mqc_common.cuh"
#include "mqc_host.h"
#include "packed_math.cuh"

namespace mqc {
namespace {

using pk::add2;
using pk::bc2;
using pk::fma2;
using pk::mul2;
using pk::neg2;

constexpr int kMaxThreads = 512;
constexpr int kMaxWarps = kMaxThreads / 32;
constexpr int kMaxWidth = MQC_NORM_GATE_MAX_WIDTH;
static_assert(kMaxWidth <= kMaxThreads * 8, "at most eight columns a thread");
constexpr int kBwdThreads = 384;  // threads of a backward CTA (168 registers each) unless a row needs more
constexpr int kFwdThreads = 256;  // threads of a forward CTA
constexpr int kFwdCtas = 2;       // forward CTAs an SM, at most (they keep the parameters); without: 8
constexpr int kFewRows = 8;       // rows an SM up to which a row is split over warps
constexpr int kSums = 5;  // column sums: dwp, dscale, dbp, dwq, dbq

// A thread's eight columns of a row, as four pairs. kVec: eight adjacent columns, 16 (bf16)
// or 32 (fp32) aligned bytes; else column j * threads + tid, one element at a time, of
// any width and alignment. `mask` has a bit for each column inside the row; the others
// stay as they are set at the start, zero.
constexpr int kCols = 8;

template <typename T, bool kVec>
struct Row;
template <>
struct Row<float, true> {
  float4 a, b;
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const float* p, int, uint32_t mask) {
    if (mask) {
      a = __ldg(reinterpret_cast<const float4*>(p));
      b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    }
  }
  // from two halves of a parameter in shared memory, `half` floats apart
  __device__ __forceinline__ void load_shared(const float* p, int half, uint32_t mask) {
    if (mask) {
      a = *reinterpret_cast<const float4*>(p);
      b = *reinterpret_cast<const float4*>(p + half);
    }
  }
  __device__ __forceinline__ void get(float2 (&o)[4]) const {
    o[0] = make_float2(a.x, a.y);
    o[1] = make_float2(a.z, a.w);
    o[2] = make_float2(b.x, b.y);
    o[3] = make_float2(b.z, b.w);
  }
  static __device__ __forceinline__ void store(float* p, const float2 (&o)[4], int, uint32_t mask) {
    if (mask) {
      reinterpret_cast<float4*>(p)[0] = make_float4(o[0].x, o[0].y, o[1].x, o[1].y);
      reinterpret_cast<float4*>(p)[1] = make_float4(o[2].x, o[2].y, o[3].x, o[3].y);
    }
  }
};
template <>
struct Row<__nv_bfloat16, true> {
  uint4 v;
  __device__ __forceinline__ void zero() { v = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int, uint32_t mask) {
    if (mask) v = __ldg(reinterpret_cast<const uint4*>(p));
  }
  __device__ __forceinline__ void get(float2 (&o)[4]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      o[k] = make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float2 (&o)[4], int,
                                               uint32_t mask) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      __nv_bfloat162 h = __floats2bfloat162_rn(o[k].x, o[k].y);
      w[k] = *reinterpret_cast<uint32_t*>(&h);
    }
    if (mask) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <typename T>
struct Row<T, false> {
  T v[kCols];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < kCols; ++j) v[j] = T(0.f);
  }
  __device__ __forceinline__ void load(const T* p, int step, uint32_t mask) {
#pragma unroll
    for (int j = 0; j < kCols; ++j)
      if (mask >> j & 1u) v[j] = __ldg(p + j * step);
  }
  __device__ __forceinline__ void load_shared(const T* p, int step, uint32_t mask) {
#pragma unroll
    for (int j = 0; j < kCols; ++j)
      if (mask >> j & 1u) v[j] = p[j * step];
  }
  __device__ __forceinline__ void get(float2 (&o)[4]) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = make_float2(to_f(v[2 * k]), to_f(v[2 * k + 1]));
  }
  static __device__ __forceinline__ void store(T* p, const float2 (&o)[4], int step, uint32_t mask) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (mask >> (2 * k) & 1u) QIO<T>::st1(p + 2 * k * step, o[k].x);
      if (mask >> (2 * k + 1) & 1u) QIO<T>::st1(p + (2 * k + 1) * step, o[k].y);
    }
  }
};

// 1 / (1 + e^-v); 0 where e^-v is infinite
__device__ __forceinline__ float sigmoid_s(float v) {
  const float e = v * -1.44269504088896341f;
  float d, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(e));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d + 1.f));
  return r;
}

// The threads of a CTA that share rows: `threads` of them (whole warps), group `id` of
// the CTA, with a barrier of their own.
struct Group {
  int threads, id, tid;
  __device__ __forceinline__ void sync() const {
    asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(threads) : "memory");
  }
};

// Sums of N (1 or 2) values over the group, one barrier. `red` has a row for each warp
// of the CTA and is used in turns of two, so a thread that is still reading one turn's
// sums is never overwritten by the next. Two values go through one butterfly: after
// its first step the lower lanes carry the first value and the upper ones the second.
template <int N>
__device__ __forceinline__ void group_sums(float (&v)[N], float (*red)[kMaxWarps][2], int& turn,
                                           const Group& g) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  float t = v[0];
  if constexpr (N == 2) {
    const bool up = lane >= 16;
    t = (up ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, up ? v[0] : v[1], 16);
  } else {
    t += __shfl_xor_sync(0xffffffffu, t, 16);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (g.threads == 32) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = __shfl_sync(0xffffffffu, t, 16 * k);
    return;
  }
  if ((lane & 15) == 0) red[turn][w][lane >> 4] = t;  // N = 1: twice the same sum
  g.sync();
  const int w0 = w - (g.tid >> 5), warps = g.threads >> 5;
  float2 sum = *reinterpret_cast<const float2*>(red[turn][w0]);
  for (int j = 1; j < warps; ++j) sum = add2(sum, *reinterpret_cast<const float2*>(red[turn][w0 + j]));
  v[0] = sum.x;
  if constexpr (N == 2) v[1] = sum.y;
  turn ^= 1;
}

__device__ __forceinline__ float across(const float2 (&u)[4]) {
  const float2 t = add2(add2(u[0], u[1]), add2(u[2], u[3]));
  return t.x + t.y;
}

// Where eight of a thread's columns are (the chunk-th eight), the same in every row.
template <bool kVec>
struct Place {
  int first, step;
  uint32_t mask;
  __device__ __forceinline__ Place(const Group& g, int width, int chunk = 0) {
    first = (kVec ? g.tid * kCols : g.tid) + chunk * kCols * g.threads;
    step = g.threads;
    mask = 0;
    if (kVec) {
      mask = first < width ? 0xffu : 0u;
    } else {
#pragma unroll
      for (int j = 0; j < kCols; ++j) mask |= uint32_t(first + j * step < width) << j;
    }
  }
};

// The values of a parameter at eight of a thread's columns; 0 for none.
template <bool kVec>
__device__ __forceinline__ void load_cols(const float* p, const Place<kVec>& at, float2 (&o)[4]) {
  Row<float, kVec> t;
  t.zero();
  if (p != nullptr) t.load(p + at.first, at.step, at.mask);
  t.get(o);
}

struct FwdArgs {
  const void *x, *y, *z;
  int64_t z_row;
  const float *wp, *bp, *scale, *wq, *bq;
  void *out, *n;
  float4* stats;  // per row: mean and 1/std of P, of Q; or NULL
  int64_t rows;
  int width, layer, threads;  // threads of a group
  float eps;
};

// Normalises a row in place (u -> uhat) and returns its mean and 1/std. K: chunks of
// eight columns a thread.
template <bool kVec, int K>
__device__ __forceinline__ void normalise(float2 (&u)[K][4], int width, bool layer, float eps,
                                          float (*red)[kMaxWarps][2], int& turn, const Group& g,
                                          float& mean, float& rstd) {
  const float inv = 1.f / float(width);
  float s[1];
  mean = 0.f;
  if (layer) {
    s[0] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) s[0] += across(u[j]);
    group_sums<1>(s, red, turn, g);
    mean = s[0] * inv;
  }
  float2 q = bc2(0.f);
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const Place<kVec> at(g, width, j);
    // columns outside the row count nothing: they stay zero
    const float m = kVec && !at.mask ? 0.f : -mean;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (layer) {
        u[j][k] = add2(u[j][k], bc2(m));
        if (!kVec) {
          if (!(at.mask >> (2 * k) & 1u)) u[j][k].x = 0.f;
          if (!(at.mask >> (2 * k + 1) & 1u)) u[j][k].y = 0.f;
        }
      }
      q = fma2(u[j][k], u[j][k], q);
    }
  }
  s[0] = q.x + q.y;
  group_sums<1>(s, red, turn, g);
  rstd = rsqrtf(fmaf(s[0], inv, eps));
#pragma unroll
  for (int j = 0; j < K; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) u[j][k] = mul2(u[j][k], bc2(rstd));
}

// Rows on their way into shared memory, two deep: each thread copies the columns that it
// will read itself (cp.async, 16 bytes at a time), so no barrier is needed, and a row
// takes no registers while it is in flight. Slot k of thread t is 16 bytes at
// (k * threads of the CTA + t). Only for kVec.
template <typename T>
constexpr int kSlots = int(sizeof(T)) * kCols / 16;
struct Ring {
  unsigned char* base;
  int stride;  // bytes of a stage
  __device__ __forceinline__ unsigned char* at(int stage, int slot) const {
    return base + stage * stride + (slot * int(blockDim.x) + int(threadIdx.x)) * 16;
  }
  template <typename T>
  __device__ __forceinline__ void copy(int stage, int slot, const T* src) const {
#pragma unroll
    for (int k = 0; k < kSlots<T>; ++k)
      cp_async16(at(stage, slot + k), reinterpret_cast<const unsigned char*>(src) + 16 * k, true);
  }
  template <typename T>
  __device__ __forceinline__ void read(int stage, int slot, float2 (&o)[4]) const {
    Row<T, true> r;
    if constexpr (sizeof(T) == 4) {
      r.a = *reinterpret_cast<const float4*>(at(stage, slot));
      r.b = *reinterpret_cast<const float4*>(at(stage, slot + 1));
    } else {
      r.v = *reinterpret_cast<const uint4*>(at(stage, slot));
    }
    r.get(o);
  }
};

// A row belongs to one warp where eight columns x K chunks a lane hold it (no barrier,
// and a sum's five steps serve up to 32 columns a lane), to up to four warps beyond.
// The parameters are kept in shared memory where a CTA works on several rows (K > 1):
// read from L1 for each row they missed it often enough to cost as much L2 traffic as
// the rows themselves.
template <typename TX, typename TY, bool kVec, bool kPost, int K>
__global__ void __launch_bounds__(kFwdThreads, kVec || K > 1 ? 2 : 4)
    norm_gate_fwd_kernel(const FwdArgs p) {
  __shared__ __align__(8) float red[2][kMaxWarps][2];
  extern __shared__ __align__(16) unsigned char dyn[];
  float* params = reinterpret_cast<float*>(dyn);  // [5][width]: wp, bp, scale, wq, bq
  int turn = 0;
  const Group grp = {p.threads, int(threadIdx.x) / p.threads, int(threadIdx.x) % p.threads};
  const int groups = int(blockDim.x) / p.threads;
  const bool layer = p.layer != 0, next = p.n != nullptr;
  if (K > 1) {
    for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
      // kVec: the first four of each eight columns, then the second four, so that the
      // lanes' 16-byte reads are adjacent (eight in a row are two-way bank conflicts:
      // 8192 x 768 rows 20.8 us, so 18.7)
      const int at = kVec ? (c >> 2 & 1) * (p.width / 2) + (c >> 3) * 4 + (c & 3) : c;
      params[at] = p.wp ? __ldg(p.wp + c) : 0.f;
      params[p.width + at] = p.bp ? __ldg(p.bp + c) : 0.f;
      params[2 * p.width + at] = p.scale ? __ldg(p.scale + c) : 0.f;
      params[3 * p.width + at] = p.wq ? __ldg(p.wq + c) : 0.f;
      params[4 * p.width + at] = p.bq ? __ldg(p.bq + c) : 0.f;
    }
    __syncthreads();
  }
  // the values of parameter k at eight of the thread's columns
  auto param = [&](int k, const float* ptr, const Place<kVec>& at, float2(&o)[4]) {
    if (K > 1) {
      Row<float, kVec> t;
      t.zero();
      t.load_shared(params + k * p.width + (kVec ? at.first / 2 : at.first),
                    kVec ? p.width / 2 : at.step, at.mask);
      t.get(o);
    } else {
      load_cols(ptr, at, o);
    }
  };
  for (int64_t row = int64_t(blockIdx.x) * groups + grp.id; row < p.rows;
       row += int64_t(gridDim.x) * groups) {
    Row<TX, kVec> xr[K];
    Row<TY, kVec> yr[K], zr[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const Place<kVec> at(grp, p.width, j);
      const int64_t off = row * p.width + at.first;
      xr[j].zero();
      if (kPost) {
        yr[j].zero();
        zr[j].zero();
        yr[j].load(static_cast<const TY*>(p.y) + off, at.step, at.mask);
        zr[j].load(static_cast<const TY*>(p.z) + row * p.z_row + at.first, at.step, at.mask);
      }
      xr[j].load(static_cast<const TX*>(p.x) + off, at.step, at.mask);
    }
    float2 o[K][4];
    float mp = 0.f, rp = 0.f, mq = 0.f, rq = 0.f;
    if constexpr (kPost) {
      float2 u[K][4];
#pragma unroll
      for (int j = 0; j < K; ++j) yr[j].get(u[j]);
      normalise<kVec, K>(u, p.width, layer, p.eps, red, turn, grp, mp, rp);
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const Place<kVec> at(grp, p.width, j);
        float2 gt[4], w[4], b[4], c[4];
        zr[j].get(gt);
        xr[j].get(o[j]);
        param(0, p.wp, at, w);
        param(1, p.bp, at, b);
        param(2, p.scale, at, c);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 s = mul2(c[k], make_float2(sigmoid_s(gt[k].x), sigmoid_s(gt[k].y)));
          o[j][k] = fma2(s, fma2(u[j][k], w[k], b[k]), o[j][k]);
        }
        Row<TX, kVec>::store(static_cast<TX*>(p.out) + row * p.width + at.first, o[j], at.step,
                             at.mask);
      }
    } else {
#pragma unroll
      for (int j = 0; j < K; ++j) xr[j].get(o[j]);
    }
    if (next) {
      normalise<kVec, K>(o, p.width, layer, p.eps, red, turn, grp, mq, rq);
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const Place<kVec> at(grp, p.width, j);
        float2 w[4], b[4];
        param(3, p.wq, at, w);
        param(4, p.bq, at, b);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[j][k] = fma2(o[j][k], w[k], b[k]);
        Row<TY, kVec>::store(static_cast<TY*>(p.n) + row * p.width + at.first, o[j], at.step,
                             at.mask);
      }
    }
    if (p.stats != nullptr && grp.tid == 0) p.stats[row] = make_float4(mp, rp, mq, rq);
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
  int width, layer, threads;  // threads of a group
};

// slots of x, dout, y, z, dn
template <typename TX, typename TY>
constexpr int kBwdSlots = 2 * kSlots<TX> + 3 * kSlots<TY>;

template <typename TX, typename TY, bool kVec, bool kPost, int kBound>
__global__ void __launch_bounds__(kBound)
    norm_gate_bwd_kernel(const BwdArgs p) {
  __shared__ __align__(8) float red[2][kMaxWarps][2];
  extern __shared__ __align__(16) unsigned char dyn[];  // the ring, in the end the groups' sums
  int turn = 0;
  const int groups = int(blockDim.x) / p.threads;
  const Group grp = {p.threads, int(threadIdx.x) / p.threads, int(threadIdx.x) % p.threads};
  const Place<kVec> at(grp, p.width);
  const bool layer = p.layer != 0, next = p.dn != nullptr;
  const float inv = 1.f / float(p.width);
  float2 wp[4], bp[4], sc[4], wq[4];
  load_cols(kPost ? p.wp : nullptr, at, wp);
  load_cols(kPost ? p.bp : nullptr, at, bp);
  load_cols(kPost ? p.scale : nullptr, at, sc);
  load_cols(p.wq, at, wq);
  float2 cs[kSums][4];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) cs[k][j] = bc2(0.f);
  constexpr int kX = 0, kG = kSlots<TX>, kY = 2 * kSlots<TX>;
  constexpr int kZ = kY + kSlots<TY>, kN = kZ + kSlots<TY>;
  const Ring ring = {dyn, kBwdSlots<TX, TY> * int(blockDim.x) * 16};
  const int64_t step = int64_t(gridDim.x) * groups;
  int64_t row = int64_t(blockIdx.x) * groups + grp.id;
  int stage = 0;
  float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
  auto fetch = [&](int64_t at_row, int to) {
    if (at_row < p.rows && at.mask) {
      const int64_t off = at_row * p.width + at.first;
      if (p.dout != nullptr) ring.copy(to, kG, static_cast<const TX*>(p.dout) + off);
      if (next) {
        ring.copy(to, kX, static_cast<const TX*>(p.x) + off);
        ring.copy(to, kN, static_cast<const TY*>(p.dn) + off);
      }
      if (kPost) {
        ring.copy(to, kY, static_cast<const TY*>(p.y) + off);
        ring.copy(to, kZ, static_cast<const TY*>(p.z) + at_row * p.z_row + at.first);
      }
    }
    cp_async_commit();
  };
  if (row < p.rows) st = __ldg(p.stats + row);
  if (kVec) {
    // what is never copied stays zero
    for (int k = 0; k < 2 * kBwdSlots<TX, TY>; ++k)
      *reinterpret_cast<uint4*>(ring.at(0, k)) = make_uint4(0u, 0u, 0u, 0u);
    fetch(row, 0);
    fetch(row + step, 1);
  }
  for (; row < p.rows; row += step, stage ^= 1) {
    if (kVec) cp_async_wait_group<1>();
    const int64_t off = row * p.width + at.first;
    // d: dout, then the whole gradient of out; yh: yhat; gt: s(z); nh: out, then nhat
    float2 d[4], yh[4], gt[4], nh[4], dn[4];
    const float4 s4 = st;
    if (row + step < p.rows) st = __ldg(p.stats + row + step);
    auto read = [&](auto type, int slot, const void* src, int64_t from, float2(&o)[4]) {
      using T = decltype(type);
      if constexpr (kVec) {
        ring.read<T>(stage, slot, o);
      } else {
        Row<T, kVec> t;
        t.zero();
        if (src != nullptr) t.load(static_cast<const T*>(src) + from, at.step, at.mask);
        t.get(o);
      }
    };
    float sums[2];
    read(TX{}, kG, p.dout, off, d);
    if constexpr (kPost) {
      read(TY{}, kY, p.y, off, yh);
      read(TY{}, kZ, p.z, row * p.z_row + at.first, gt);
    }
    if (next) {
      read(TX{}, kX, p.x, off, nh);
      read(TY{}, kN, p.dn, off, dn);
    }
    if (kVec) fetch(row + 2 * step, stage);
    if constexpr (kPost) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        yh[k] = mul2(add2(yh[k], bc2(-s4.x)), bc2(s4.y));
        gt[k] = make_float2(sigmoid_s(gt[k].x), sigmoid_s(gt[k].y));
      }
    }
    if (next) {
      float2 a = bc2(0.f), b = bc2(0.f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (kPost) nh[k] = fma2(mul2(sc[k], gt[k]), fma2(yh[k], wp[k], bp[k]), nh[k]);
        nh[k] = mul2(add2(nh[k], bc2(-s4.z)), bc2(s4.w));
        cs[3][k] = fma2(dn[k], nh[k], cs[3][k]);
        cs[4][k] = add2(dn[k], cs[4][k]);
        dn[k] = mul2(dn[k], wq[k]);
        a = add2(a, dn[k]);
        b = fma2(dn[k], nh[k], b);
      }
      sums[0] = a.x + a.y;
      sums[1] = b.x + b.y;
      group_sums<2>(sums, red, turn, grp);
      const float2 ma = bc2(layer ? -sums[0] * inv : 0.f), mb = bc2(-sums[1] * inv);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        d[k] = fma2(bc2(s4.w), fma2(nh[k], mb, add2(dn[k], ma)), d[k]);
    }
    Row<TX, kVec>::store(static_cast<TX*>(p.dx) + off, d, at.step, at.mask);
    if constexpr (kPost) {
      float2 dz[4], a = bc2(0.f), b = bc2(0.f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 pv = fma2(yh[k], wp[k], bp[k]);
        const float2 dg = mul2(d[k], gt[k]);  // d s(z)
        const float2 dp = mul2(dg, sc[k]);
        dz[k] = mul2(mul2(dp, pv), add2(bc2(1.f), neg2(gt[k])));
        cs[0][k] = fma2(dp, yh[k], cs[0][k]);
        cs[1][k] = fma2(dg, pv, cs[1][k]);
        cs[2][k] = add2(dp, cs[2][k]);
        d[k] = mul2(dp, wp[k]);
        a = add2(a, d[k]);
        b = fma2(d[k], yh[k], b);
      }
      Row<TY, kVec>::store(static_cast<TY*>(p.dz) + off, dz, at.step, at.mask);
      sums[0] = a.x + a.y;
      sums[1] = b.x + b.y;
      group_sums<2>(sums, red, turn, grp);
      const float2 ma = bc2(layer ? -sums[0] * inv : 0.f), mb = bc2(-sums[1] * inv);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        d[k] = mul2(bc2(s4.y), fma2(yh[k], mb, add2(d[k], ma)));
      Row<TY, kVec>::store(static_cast<TY*>(p.dy) + off, d, at.step, at.mask);
    }
  }
  // the groups add their column sums in turn, in [kSums][width] where the ring was
  if (kVec) cp_async_wait_all();
  __syncthreads();
  float* acc = reinterpret_cast<float*>(dyn);
  for (int turn_of = 0; turn_of < groups; ++turn_of) {
    if (turn_of == grp.id) {
#pragma unroll
      for (int k = 0; k < kSums; ++k) {
        if ((k < 3 && !kPost) || (k >= 3 && !next)) continue;
        float* part = p.part + (int64_t(blockIdx.x) * kSums + k) * p.width;
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          if (!(at.mask >> j & 1u)) continue;
          const int c = at.first + (kVec ? j : j * at.step);
          const float own = j & 1 ? cs[k][j >> 1].y : cs[k][j >> 1].x;
          const float sum = turn_of == 0 ? own : acc[k * p.width + c] + own;
          if (turn_of == groups - 1) part[c] = sum;
          else acc[k * p.width + c] = sum;
        }
      }
    }
    __syncthreads();
  }
}

struct SumArgs {
  const float* part;
  float* out[kSums];  // NULL: not wanted
  int ctas, width;
};

// out[k][c] = sum over CTAs of part[cta][k][c]: 32 columns a block, 16 slices of CTAs,
// four loads in flight a thread.
__global__ void __launch_bounds__(512) norm_gate_sum_kernel(const SumArgs p) {
  __shared__ float red[16][32];
  const int k = blockIdx.y;
  if (p.out[k] == nullptr) return;
  const int l = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + l;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < p.width) {
    const float* q = p.part + int64_t(k) * p.width + c;
    const int64_t row = int64_t(kSums) * p.width;
    for (int i = w; i < p.ctas; i += 64)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + 16 * j < p.ctas) s[j] += __ldg(q + (i + 16 * j) * row);
  }
  red[w][l] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (w == 0 && c < p.width) {
    float t = red[0][l];
    for (int j = 1; j < 16; ++j) t += red[j][l];
    p.out[k][c] = t;
  }
}

// ----------------------------------------------------------------------- host

// Threads that share a row: eight columns each, whole warps.
int row_threads(int64_t width) { return int((width + 32 * kCols - 1) / (32 * kCols)) * 32; }

// Groups of a CTA and CTAs of the backward pass: one CTA an SM, of as many groups as
// fit kMaxThreads, as each CTA leaves kSums rows of partial sums.
int bwd_groups(int threads) {
  return threads <= kBwdThreads ? kBwdThreads / threads : kMaxThreads / threads;
}
int bwd_grid(int threads, int64_t rows) {
  const int64_t want = (rows + bwd_groups(threads) - 1) / bwd_groups(threads);
  return int(want < num_sms() ? want : num_sms());
}

// Shared memory above the 48 KB that need no leave (asked each time: it is one host call).
template <typename K>
int allow_smem(K kernel, size_t bytes, const char* what) {
  if (bytes <= 40 * 1024) return MQC_OK;  // leaves room for the static part
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
  MQC_REQUIRE(e == cudaSuccess, MQC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return MQC_OK;
}

// Chunks of eight columns a thread has in the forward pass. With enough rows to fill the
// device a row goes to one warp (up to 1024 columns): 8192 x 768 rows, fp32 and bf16,
// 18.7 us against 23.3 with three warps a row. With few rows, and where columns are
// loaded one by one (1731 x 515 fp32: 6.7 us against 10.6), to as many warps as it has
// chunks.
template <bool kVec>
int fwd_chunks(int64_t rows, int64_t width) {
  const int64_t need = (width + 32 * kCols - 1) / (32 * kCols), most = kFwdThreads / 32;
  if (!kVec || rows <= int64_t(num_sms()) * kFewRows) return need <= most ? 1 : 2;
  return int(need < 4 ? need : 4);
}

template <typename TX, typename TY, bool kVec, bool kPost, int K>
int launch_fwd_k(FwdArgs& f, cudaStream_t st) {
  f.threads = int((f.width + 32 * kCols * K - 1) / (32 * kCols * K)) * 32;
  const int groups = kFwdThreads / f.threads, threads = groups * f.threads;
  const int64_t ctas = (f.rows + groups - 1) / groups;
  auto kernel = norm_gate_fwd_kernel<TX, TY, kVec, kPost, K>;
  const size_t smem = K > 1 ? 5 * sizeof(float) * size_t(f.width) : 0;
  if (int rc = allow_smem(kernel, smem, "mqc_norm_gate_fwd")) return rc;
  const int64_t most = int64_t(num_sms()) * (K > 1 ? kFwdCtas : 8);
  kernel<<<unsigned(ctas < most ? ctas : most), threads, smem, st>>>(f);
  return check_launch("mqc_norm_gate_fwd");
}

template <typename TX, typename TY, bool kVec, bool kPost>
int launch_fwd(FwdArgs& f, cudaStream_t st) {
  switch (fwd_chunks<kVec>(f.rows, f.width)) {
    case 1: return launch_fwd_k<TX, TY, kVec, kPost, 1>(f, st);
    case 2: return launch_fwd_k<TX, TY, kVec, kPost, 2>(f, st);
  }
  if constexpr (kVec) {
    return f.width <= 768 ? launch_fwd_k<TX, TY, kVec, kPost, 3>(f, st)
                          : launch_fwd_k<TX, TY, kVec, kPost, 4>(f, st);
  }
  return fail(MQC_ERR_UNSUPPORTED, "mqc_norm_gate_fwd: width %d", f.width);
}

template <typename TX, typename TY, bool kVec, bool kPost>
int launch_bwd(const BwdArgs& f, int* ctas, cudaStream_t st) {
  const int groups = bwd_groups(f.threads);
  *ctas = bwd_grid(f.threads, f.rows);
  const int threads = groups * f.threads;
  const size_t join = groups > 1 ? size_t(kSums) * f.width * sizeof(float) : 0;
  const size_t ring = kVec ? 2 * 16 * size_t(threads) * kBwdSlots<TX, TY> : 0;
  const size_t smem = join > ring ? join : ring;
  auto kernel = f.threads <= kBwdThreads ? norm_gate_bwd_kernel<TX, TY, kVec, kPost, kBwdThreads>
                                         : norm_gate_bwd_kernel<TX, TY, kVec, kPost, kMaxThreads>;
  if (int rc = allow_smem(kernel, smem, "mqc_norm_gate_bwd")) return rc;
  kernel<<<*ctas, threads, smem, st>>>(f);
  return check_launch("mqc_norm_gate_bwd");
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

// Rows can move eight columns at a time: the width and z's stride divide by eight and
// every tensor is aligned to 16 bytes.
bool vec_ok(const mqc_norm_gate_args* a) {
  return a->width % kCols == 0 && (a->z == nullptr || a->z_row % kCols == 0) && aligned(a->x, 16) &&
         aligned(a->out, 16) && aligned(a->dout, 16) && aligned(a->dx, 16) && aligned(a->y, 16) &&
         aligned(a->z, 16) && aligned(a->n, 16) && aligned(a->dn, 16) && aligned(a->dy, 16) &&
         aligned(a->dz, 16) && aligned(a->weight, 16) && aligned(a->bias, 16) &&
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
               a->rows, int(a->width), a->norm == MQC_NORM_LAYER, 0, a->eps};
  const bool vec = vec_ok(a);
  cudaStream_t st = as_stream(stream);
  return by_types(a->x_dtype, a->y_dtype, post, [&](auto tx, auto ty, auto kp) {
    using TX = decltype(tx);
    using TY = decltype(ty);
    constexpr bool kPost = decltype(kp)::value;
    return vec ? launch_fwd<TX, TY, true, kPost>(f, st) : launch_fwd<TX, TY, false, kPost>(f, st);
  });
}

size_t mqc_norm_gate_bwd_workspace_size(int64_t rows, int64_t width) {
  using namespace mqc;
  if (rows <= 0 || width <= 0 || width > kMaxWidth) return 0;
  return size_t(bwd_grid(row_threads(width), rows)) * kSums * size_t(width) * sizeof(float);
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
               a->norm == MQC_NORM_LAYER, row_threads(a->width)};
  const bool vec = vec_ok(a);
  int ctas = 0;
  int rc = by_types(a->x_dtype, a->y_dtype, post, [&](auto tx, auto ty, auto kp) {
    using TX = decltype(tx);
    using TY = decltype(ty);
    constexpr bool kPost = decltype(kp)::value;
    return vec ? launch_bwd<TX, TY, true, kPost>(f, &ctas, st)
               : launch_bwd<TX, TY, false, kPost>(f, &ctas, st);
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
  norm_gate_sum_kernel<<<dim3((f.width + 31) / 32, kSums), 512, 0, st>>>(q);
  return check_launch("mqc_norm_gate_bwd (column sums)");
}

}  // extern "C"
