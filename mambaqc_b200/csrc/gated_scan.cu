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
// 32 or 64 steps; each warp takes a run of consecutive steps of the tile, each lane
// two channels, so the arithmetic is packed two-wide; the tile's rows come through
// shared memory (cp.async). A run is reduced to (A, E), h_out = A h_in + E (A held as
// A - 1 from 1/2 up), in registers; runs are joined through shared memory, tiles through the
// shared memory of a thread-block cluster whose CTAs take consecutive tiles of the same
// sequence. So each input is read once and each output written once, and no CTA waits
// for another one outside its cluster.
//
// The backward pass reads no y: it runs each tile again from the fp32 state that
// the forward pass left at the tile's start (y in bf16 would cost dLambda three
// digits), and the reverse recurrence uses the same products A.
//
// Measured, bf16, 4 x 2048 x 1536 on one B200: forward 35 us, backward 68 us (and 3 for
// dLambda), where the bytes alone take 15 and 27 us at 6.5 TB/s; 1 x 32768 x 1024
// forward 129 us (41), backward 231: a round of the cluster takes 2.15 us with one CTA an
// SM, 3.1 with two and 4 with three, and clusters of 16 come to three on some SMs. With
// products of decays held as A - 1 throughout it was 34, 69, 125 and 223. Found at
// 35.3 us, before that and the short form of slow decays: neither memory bounds the forward (with
// all tiles read from the cache and nothing stored it took 34 us) nor the special
// functions (35 us without any) nor one pipe (the fullest, FMA, 46 % busy), but the
// phases of a tile between barriers: 47 instructions an element at 0.57 a cycle and
// scheduler with 24 warps an SM. Slower or the same: four CTAs an SM at 64 registers
// (40 us), every warp joining the runs for itself (38 us), an mbarrier for each rank
// (39 us; the long prefill 198), bulk copies in place of st.async (36.7 us), unpacked
// arithmetic (40 us), one reciprocal for both sigmoids (37 us), the next tile reduced
// while the exchange is under way (one barrier a round, but two CTAs an SM: 46 us; the
// long prefill 129 against 133).
//
// Backward, tiles of 32 steps: the barriers of two CTAs an SM overlap, where one CTA of
// 16 warps and tiles of 64 took 79 us (512 x 64 x 1024: 160 against 253; only 3 x 2048 x
// 1536 was faster with it, 50 us against 58, now 56). Slower: three
// CTAs an SM at 85 registers (78 us); and with tiles of 64, eight warps of eight steps
// (82 us), one joining warp of channel pairs (94 us), the states' half of the second
// pass under the exchange for one more barrier (81 us; 64 x 512 x 1024 170 against 154).
#include <cooperative_groups.h>

#include <atomic>
#include <cmath>
#include <initializer_list>
#include <type_traits>

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
constexpr int kBwdTile = MQC_GATED_SCAN_TILE;  // time steps of a tile backward, and of a checkpoint
constexpr int kRun = 8;  // steps of a warp's run forward
// Forward, sequences of up to kShort steps go in tiles of 32 (four warps), longer ones
// in tiles of 64 (eight). us with 32 and 64, bf16 (fp32): 512 x 64 x 1024 65 and 85 (89
// and 121), 256 x 128 x 1024 62 and 73 (85 and 102), 1 x 32768 x 1024 153 and 129 (224 and
// 190), 1 x 8192 x 1024 41 and 36 (59 and 50): small CTAs hide one another's loads where a
// sequence is done in a round or two, large ones take half the rounds where it is long.
// Between, neither is better throughout: 200 x 160 x 1024 60 and 83 (85 and 109), 24 x 320
// x 768 19 and 16 (both 19), 40 x 300 x 1024 39 and 32 (51 and 44), 64 x 512 x 1024 75 and
// 67 (87 and 96), 4 x 2048 x 1536 both 34 (40 and 51), 1 x 2048 x 1536 both 15 (23 and 16).
constexpr int kShort = 128;
// CTAs of a cluster: as many as the exchange's shared memory leaves room for two CTAs
// an SM beside (16 is the device's limit, above the portable 8)
template <typename T>
constexpr int kMaxCluster = sizeof(T) == 2 ? 16 : 8;

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
__device__ __forceinline__ float sqrt_a(float v) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr float kLog2e = 1.44269504088896341f;

// 1 / (1 + 2^(-z log2 e)); 0 where the power is infinite
__device__ __forceinline__ float2 sigmoid2(float2 z) {
  const float2 e = mul2(z, bc2(-kLog2e));
  const float2 d = add2(make_float2(ex2(e.x), ex2(e.y)), bc2(1.f));
  return make_float2(rcp(d.x), rcp(d.y));
}

// e^f - 1 as f + f^2 p(f), p of least relative error over the interval (weighted least
// squares, the weights moved to where the error is largest until it is level): 1.7e-8 in
// both, the coefficients rounded to fp32. Exact to the last place near 0, where
// 1 - exp(-2 l) and the decay over many steps need it. For -kNear <= f <= 0:
constexpr float kNear = 0.3465f;
__device__ __forceinline__ float2 expm1_near2(float2 f) {
  float2 p = fma2(f, bc2(0.007241870276629925f), bc2(0.04135452210903168f));
  p = fma2(p, f, bc2(0.16663089394569397f));
  p = fma2(p, f, bc2(0.49999871850013733f));
  return fma2(mul2(p, f), f, f);
}
// and for |f| <= ln 2 / 2:
__device__ __forceinline__ float2 expm1_reduced2(float2 f) {
  float2 p = fma2(f, bc2(0.0013882521307095885f), bc2(0.008366518653929234f));
  p = fma2(p, f, bc2(0.04166720062494278f));
  p = fma2(p, f, bc2(0.1666654348373413f));
  p = fma2(p, f, bc2(0.4999999701976776f));
  return fma2(mul2(p, f), f, f);
}

// a = e^v and m = e^v - 1 for v <= 0: with v = n ln 2 + f they are 2^n (e^f - 1) + 2^n and
// 2^n (e^f - 1) + (2^n - 1), so a keeps its digits where it is small and m where it is.
// The constant ln 2 is rounded: 2e-9 n in f. Below kLeast v counts as kLeast (a 1.6e-38):
// n stays in the range of an exponent, and a above 0.
constexpr float kLeast = -87.f;
__device__ __forceinline__ void exp_neg2(float2 v, float2& a, float2& m) {
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: the sum's low bits are the integer
  const float2 x = make_float2(max_nan(v.x, kLeast), max_nan(v.y, kLeast));
  const float2 t = fma2(x, bc2(kLog2e), bc2(kMagic));
  const float2 n = add2(t, bc2(-kMagic));
  const float2 p = expm1_reduced2(fma2(n, bc2(-0.693147180559945309f), x));
  const float2 s = make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000),
                               __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000));
  a = fma2(s, p, s);
  m = fma2(s, p, add2(s, bc2(-1.f)));
}

__device__ __forceinline__ float softplus_acc(float u) {
  return u > 20.f ? u + log1pf(expf(-u)) : log1pf(expf(u));
}

// a, m = a - 1 and q = 1 - a^2 = -m (m + 2) of a step with -L = v; kSmall: |v| <= kNear.
template <bool kSmall>
__device__ __forceinline__ void decay2(float2 v, float2& a, float2& m, float2& q) {
  if (kSmall) {
    m = expm1_near2(v);
    a = add2(m, bc2(1.f));
  } else {
    exp_neg2(v, a, m);
  }
  q = mul2(neg2(m), add2(m, bc2(2.f)));
}

// -c softplus(Lambda) of two channels, 0 where there is none: what s(r) is multiplied
// by to -L. As s(r) <= 1, a warp whose rates are all within kNear needs no reduction of
// the exponent (small_rates): decays of 0.7 a step and slower,
// which is where such layers start and mostly stay. Forward, slow against fast decays:
// 34.9 and 36.9 us at 4 x 2048 x 1536, 129 and 139 at 1 x 32768 x 1024; backward 68.2 and
// 70.4, 231 and 241.
__device__ __forceinline__ float2 neg_rate2(float2 lam, float sharpness, bool ok0, bool ok1) {
  return make_float2(ok0 ? -sharpness * softplus_acc(lam.x) : 0.f, ok1 ? -sharpness * softplus_acc(lam.y) : 0.f);
}
__device__ __forceinline__ bool small_rates(float2 nrate) {
  return __all_sync(0xffffffffu, nrate.x >= -kNear && nrate.y >= -kNear);
}

// Products A of decays are held as M = A - 1: (1 + M)(1 + m) - 1 = M + (M m + m). A
// product of fp32 numbers just below 1 loses j k 2^-48 each time, j and k their
// distances from 1 in units of 2^-24, always to the same side; over a state's
// memory of 1e4 steps that came to 4e-5 of it. M has 6e-8 of A at least, but only 6e-8:
// under 1/2 it is A itself that counts, multiplied up beside M (where single decays are
// above 0.7, 1 + M serves: 2e-6 of A over eight of them). A gradient carried as
// s + (M s + E) over 32 steps of decay 0.6 was 25 % off.
struct Product2 {
  float2 M, A;
};
template <bool kSmall>
__device__ __forceinline__ void join_step(Product2& t, float2 a, float2 m) {
  t.M = add2(t.M, fma2(t.M, m, m));
  if (!kSmall) t.A = mul2(t.A, a);
}

// The product of a run or a tile as one number: M (below 0) from A = 1/2 up, A (0 or
// above) under that, and kDropped with a reset in the run. A product of exactly 1 is held
// as -kTiny, which s + (M s + E) does not see.
constexpr float kDropped = -2.f;
constexpr float kTiny = 1.17549435e-38f;
__device__ __forceinline__ float product_of(float M, float A) {
  return M >= -0.5f ? fminf(M, -kTiny) : A;
}
template <bool kSmall>
__device__ __forceinline__ float2 product_of(const Product2& t) {
  const float2 A = kSmall ? add2(t.M, bc2(1.f)) : t.A;
  return make_float2(product_of(t.M.x, A.x), product_of(t.M.y, A.y));
}

// The product of a tile's runs for one channel.
template <bool kReset, int W>
__device__ __forceinline__ float tile_product(const float2 (*run)[kChan], int ch) {
  float M = 0.f, A = 1.f;
  bool dropped = false;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float D = run[w][ch].x;
    const float m = D < 0.f ? D : D - 1.f;
    A *= D < 0.f ? D + 1.f : D;
    M += fmaf(M, m, m);
    dropped = dropped || (kReset && D == kDropped);
  }
  return dropped ? kDropped : product_of(M, A);
}

// A s + E. A reset drops s whatever it is, a NaN decay in the same run notwithstanding;
// decays that multiply to nothing drop no NaN. kInfinite: s may be infinite and stays
// so, as every decay is above 0; without, the result is NaN there (the joins below look
// for one and start again with kInfinite).
template <bool kReset, bool kInfinite>
__device__ __forceinline__ float apply(float D, float E, float s) {
  // the factor of s, 1 or 0, and not s or 0: nothing else than two multiply-adds waits
  // for s (a select there cost 4 % of the backward pass)
  const float r = fmaf(D < 0.f ? 1.f : 0.f, s, fmaf(D, s, E));
  if (kReset && D == kDropped) return E;
  return kInfinite && fabsf(s) == __int_as_float(0x7f800000) ? s + E : r;
}

__device__ __forceinline__ float2 sqrt2(float2 q) { return make_float2(sqrt_a(q.x), sqrt_a(q.y)); }
// 1 / beta (9e18 at most: at beta = 0 what it multiplies is multiplied by L = 0 as well)
__device__ __forceinline__ float2 inv_beta2(float2 beta) {
  const float2 t = add2(beta, bc2(1.0842022e-19f));
  return make_float2(rcp(t.x), rcp(t.y));
}

// ------------------------------------------------------------------- memory

// Two adjacent channels. kVec: the pair is one aligned word of the tensor.
__device__ __forceinline__ float2 unpack2(const float* p) {
  return *reinterpret_cast<const float2*>(p);
}
__device__ __forceinline__ float2 unpack2(const __nv_bfloat16* p) {
  const uint32_t v = *reinterpret_cast<const uint32_t*>(p);
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <bool kVec>
__device__ __forceinline__ void store2(float* p, float2 o, bool ok0, bool ok1) {
  if (kVec) {
    if (ok0) *reinterpret_cast<float2*>(p) = o;
  } else {
    if (ok0) p[0] = o.x;
    if (ok1) p[1] = o.y;
  }
}
template <bool kVec>
__device__ __forceinline__ void store2(__nv_bfloat16* p, float2 o, bool ok0, bool ok1) {
  if (kVec) {
    if (ok0) *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(o.x, o.y);
  } else {
    if (ok0) p[0] = __float2bfloat16_rn(o.x);
    if (ok1) p[1] = __float2bfloat16_rn(o.y);
  }
}

// One tile (kRows rows of kChan channels) of a tensor into shared memory. kBytes: what
// one copy moves (16 or 4: cp.async; else single elements through registers). Rows
// from `rows` on and channels from `cols` on become zero and are not read. `src`: the
// tile's first element, or NULL for zeros.
template <typename T, int kBytes, int kThreads, int kRows>
__device__ __forceinline__ void copy_tile(T* dst, const T* src, int64_t stride, int rows, int cols) {
  constexpr int kPer = kBytes / int(sizeof(T));  // elements a copy
  constexpr int kUnits = kChan / kPer;           // copies a row
  constexpr int kEach = kRows * kUnits / kThreads;
  static_assert(kRows * kUnits % kThreads == 0 && kThreads % kUnits == 0, "whole rounds");
  const int unit = int(threadIdx.x) % kUnits, row0 = int(threadIdx.x) / kUnits;
  const int c = unit * kPer;
  const int have = min(max(cols - c, 0), kPer) * int(sizeof(T));
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int row = row0 + k * (kThreads / kUnits);
    const int bytes = row < rows && src != nullptr ? have : 0;
    T* d = dst + row * kChan + c;
    if constexpr (kBytes == 16) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(d)),
                   "l"(bytes ? src + row * stride + c : src), "r"(bytes)
                   : "memory");
    } else if constexpr (kBytes == 4) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_addr(d)),
                   "l"(bytes ? src + row * stride + c : src), "r"(bytes)
                   : "memory");
    } else {
      *d = bytes ? __ldg(src + row * stride + c) : T(0.f);
    }
  }
}

__device__ __forceinline__ float2 load_f2(const float* p, int c, bool ok0, bool ok1) {
  if (p == nullptr) return bc2(0.f);
  return make_float2(ok0 ? p[c] : 0.f, ok1 ? p[c + 1] : 0.f);
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
  int* status;
  int give_up;  // waits give up at once
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
  int* status;
  int give_up;  // waits give up at once
  int batch, seq, channels, chan_tiles;
  float sharpness;
};

// --------------------------------------------------- exchange between the CTAs

// What one thread a channel of each CTA tells all CTAs of its cluster in a round: the
// pair (D, E) of its tile, written into their shared memory with the bytes counted on
// an mbarrier there, so a round needs no barrier of the cluster and no fence that
// waits for the global stores in flight. Two buffers in turn: a CTA writes round k + 2
// only after it has every message of round k + 1, which their senders sent after
// they had read round k.
template <int kRanks>
struct Exchange {
  float2 sum[2][kRanks][kChan];
  uint64_t bar[2];
};
// A poll may sleep for up to kPollNs; after kPollLimit of them, about a second, a wait is
// given up and reported.
constexpr int kPollNs = 1000;
constexpr int kPollLimit = 1 << 20;

template <int kRanks>
__device__ __forceinline__ void exchange_init(Exchange<kRanks>* x) {
  if (threadIdx.x == 0) {
    mbar_init(&x->bar[0], 1);
    mbar_init(&x->bar[1], 1);
    fence_mbar_init();
  }
}

__device__ __forceinline__ uint32_t remote_addr(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

// Whether the round's messages are all here, after up to kPollLimit polls. (A limit
// that is an argument costs the forward pass 3 to 5 % in registers.)
__device__ __forceinline__ bool exchange_wait(uint32_t bar, uint32_t parity) {
  for (int k = 0; k < kPollLimit; ++k) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity), "n"(kPollNs)
        : "memory");
    if (done) return true;
  }
  return false;
}

// Sends this channel's pair and waits for those of all ranks; false: given up (at once,
// if asked to) and reported, after a second wait for the messages that are on their way
// to this CTA (a channel whose wait was given up sends no more).
template <int kRanks>
__device__ __forceinline__ bool exchange(Exchange<kRanks>* x, int buf, uint32_t parity, int rank, int csize,
                                         int ch, float d, float e, bool give_up, int* status) {
  if (ch == 0) mbar_arrive_expect_tx(&x->bar[buf], uint32_t(csize * kChan * sizeof(float2)));
  const uint32_t at = smem_addr(&x->sum[buf][rank][ch]), bar = smem_addr(&x->bar[buf]);
  for (int to = 0; to < csize; ++to)
    asm volatile(
        "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::
            "r"(remote_addr(at, to)),
        "f"(d), "f"(e), "r"(remote_addr(bar, to))
        : "memory");
  if (!give_up && exchange_wait(bar, parity)) return true;
  report_status(status, MQC_DEVICE_STATUS_TIMEOUT);
  exchange_wait(bar, parity);
  return false;
}

// ------------------------------------------------------------------- forward

template <typename T, int kWarps>
struct FwdSmem {
  T raw[3][kWarps * kRun][kChan];      // x, r, i of a tile
  float2 run[kWarps][kChan];          // (D, E) of each warp's run
  float start[kWarps][kChan];         // state before each run
  Exchange<kMaxCluster<T>> ex;
};

// One tile: (A) each warp reduces its run to (D, E); (B) one thread a channel joins
// the runs, exchanges the tile's pair with the cluster and hands each run its start;
// (C) each warp runs its steps again from there and stores y. The next tile's copies
// are in flight from (B) on.
template <typename T, int kBytes, bool kVec, bool kReset, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, (sizeof(T) == 2 ? 24 : 16) / kWarps)
    gated_scan_fwd_kernel(const FwdArgs p) {
  constexpr int W = kWarps, S = kRun, kThreads = W * 32, kTile = W * S;
  static_assert(kTile % kBwdTile == 0 && kBwdTile % S == 0, "checkpoints at the starts of runs");
  extern __shared__ __align__(128) unsigned char smem_raw[];
  FwdSmem<T, W>& sm = *reinterpret_cast<FwdSmem<T, W>*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int csize = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int unit = int(blockIdx.x) / csize;
  const int b = unit / p.chan_tiles;
  const int c0 = (unit - b * p.chan_tiles) * kChan;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int c = c0 + 2 * lane;
  const bool ok0 = c < p.channels, ok1 = c + 1 < p.channels;
  const int tiles = (p.seq + kTile - 1) / kTile, ckpts = (p.seq + kBwdTile - 1) / kBwdTile;
  const int64_t row0 = int64_t(b) * p.seq;
  const T* x = static_cast<const T*>(p.x) + row0 * p.xs + c0;
  const T* r = static_cast<const T*>(p.r) + row0 * p.rs + c0;
  const T* iv = static_cast<const T*>(p.i) + row0 * p.is + c0;
  T* y = static_cast<T*>(p.y) + row0 * p.channels + c;
  const uint8_t* rst = kReset ? p.reset + row0 : nullptr;
  const float2 lam = load_f2(p.lambda, c, ok0, ok1);
  const float2 nrate = neg_rate2(lam, p.sharpness, ok0, ok1);
  const bool small = small_rates(nrate);
  // the joining threads' channel and its state, passed from round to round
  const int jc = c0 + tid;
  const bool jok = tid < kChan && jc < p.channels;
  float carry = jok && p.h0 ? p.h0[int64_t(b) * p.channels + jc] : 0.f;

  auto load = [&](int tile) {
    const int64_t t0 = int64_t(tile) * kTile;
    const int rows = p.seq - int(t0), cols = p.channels - c0;
    copy_tile<T, kBytes, kThreads, kTile>(&sm.raw[0][0][0], x + t0 * p.xs, p.xs, rows, cols);
    copy_tile<T, kBytes, kThreads, kTile>(&sm.raw[1][0][0], r + t0 * p.rs, p.rs, rows, cols);
    copy_tile<T, kBytes, kThreads, kTile>(&sm.raw[2][0][0], iv + t0 * p.is, p.is, rows, cols);
  };

  if (csize > 1) exchange_init(&sm.ex);
  if (rank < tiles) load(rank);
  cp_async_commit();
  if (csize > 1) cluster.sync();  // every CTA's mbarriers are ready before they are written
  bool alive = true;
  int round = 0;
  for (int first = 0; first < tiles; first += csize, ++round) {
    const int tile = first + rank, st = round & 1;
    const int t0 = tile * kTile + warp * S;
    cp_async_wait_all();
    __syncthreads();  // the tile has landed
    float2 a[S], u[S];
    bool drop[S];
    float2 D = bc2(-kTiny), E = bc2(0.f);
    // steps past the end keep the state; whole tiles do not look for it
    auto reduce = [&](auto whole, auto slow) {
      Product2 t = {bc2(0.f), bc2(1.f)};
      bool dropped = false;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int row = warp * S + s;
        const bool in = decltype(whole)::value || t0 + s < p.seq;
        float2 m, q;
        decay2<decltype(slow)::value>(mul2(nrate, sigmoid2(unpack2(&sm.raw[1][row][2 * lane]))), a[s], m, q);
        const float2 v =
            mul2(sigmoid2(unpack2(&sm.raw[2][row][2 * lane])), unpack2(&sm.raw[0][row][2 * lane]));
        u[s] = mul2(sqrt2(q), v);
        drop[s] = kReset && in && rst[t0 + s] != 0;
        if (!in) {
          m = u[s] = bc2(0.f);
          a[s] = bc2(1.f);
        }
        if (kReset && drop[s]) {
          u[s] = E = v;
          dropped = true;
        } else {
          E = fma2(a[s], E, u[s]);
          join_step<decltype(slow)::value>(t, a[s], m);
        }
      }
      D = kReset && dropped ? bc2(kDropped) : product_of<decltype(slow)::value>(t);
    };
    const bool whole = (tile + 1) * kTile <= p.seq;
    if (whole && small) reduce(std::true_type{}, std::true_type{});
    else if (whole) reduce(std::true_type{}, std::false_type{});
    else if (tile < tiles) reduce(std::false_type{}, std::false_type{});
    *reinterpret_cast<float4*>(&sm.run[warp][2 * lane]) = make_float4(D.x, E.x, D.y, E.y);
    __syncthreads();  // the runs are there, and the tile's rows are no longer read
    if (tile + csize < tiles) load(tile + csize);
    cp_async_commit();
    if (tid < kChan) {
      if (csize > 1) {
        const float td = tile_product<kReset, W>(sm.run, tid);
        auto total = [&](auto infinite) {
          float te = 0.f;
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const float2 g = sm.run[w][tid];
            te = apply<kReset, decltype(infinite)::value>(g.x, g.y, te);
          }
          return te;
        };
        float te = total(std::false_type{});
        if (te != te) te = total(std::true_type{});
        if (alive)
          alive = exchange(&sm.ex, st, uint32_t(round >> 1) & 1u, rank, csize, tid, td, te, p.give_up != 0, p.status);
      }
      // the carry over the round, and the state before each run; true: a state was
      // infinite or NaN
      float next;
      auto place = [&](auto infinite) {
        constexpr bool kInf = decltype(infinite)::value;
        float h = carry, seen = 0.f;  // seen: 0 times the states
        next = carry;
        if (csize > 1) {
          for (int k = 0; k < csize; ++k) {
            if (k == rank) h = next;
            const float2 g = sm.ex.sum[st][k][tid];
            next = apply<kReset, kInf>(g.x, g.y, next);
            if (kReset) seen = fmaf(next, 0.f, seen);
          }
          seen = fmaf(next, 0.f, seen);
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          sm.start[w][tid] = h;
          if (w * S % kBwdTile == 0) {
            const int q = tile * (kTile / kBwdTile) + w * S / kBwdTile;
            if (p.ckpt != nullptr && jok && q < ckpts) p.ckpt[(int64_t(b) * ckpts + q) * p.channels + jc] = h;
          }
          const float2 g = sm.run[w][tid];
          h = apply<kReset, kInf>(g.x, g.y, h);
          if (kReset) seen = fmaf(h, 0.f, seen);
        }
        seen = fmaf(h, 0.f, seen);
        if (csize == 1) next = h;
        return seen != seen;
      };
      if (place(std::false_type{})) place(std::true_type{});
      carry = next;
    }
    __syncthreads();
    float2 h = *reinterpret_cast<const float2*>(&sm.start[warp][2 * lane]);
    T* yt = y + int64_t(t0) * p.channels;
    auto write = [&](auto whole) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        h = kReset && drop[s] ? u[s] : fma2(a[s], h, u[s]);
        if (decltype(whole)::value || t0 + s < p.seq) store2<kVec>(yt, h, ok0, ok1);
        yt += p.channels;
      }
    };
    if (whole) write(std::true_type{});
    else if (tile < tiles) write(std::false_type{});
  }
  if (p.hT != nullptr && rank == 0 && jok) p.hT[int64_t(b) * p.channels + jc] = carry;
  if (csize > 1) cluster.sync();  // no CTA leaves while another may still write to it
}

// ------------------------------------------------------------------ backward

constexpr int kBwdWarps = 8;

template <typename T>
struct BwdSmem {
  T raw[2][4][kBwdTile][kChan];          // x, r, i, dy of this tile and the one before it
  float2 run[kBwdWarps][kChan];       // (D, E) of each warp's run
  float back[kBwdWarps][kChan];       // G of each run: c before it = A c after it + G
  float start[kBwdWarps][kChan];      // state before each run
  float after[kBwdWarps][kChan];      // c after each run
  Exchange<kMaxCluster<T>> ex;
};

template <typename T, int kBytes, bool kVec, bool kReset>
__global__ void __launch_bounds__(kBwdWarps * 32, 2)
    gated_scan_bwd_kernel(const BwdArgs p) {
  constexpr int W = kBwdWarps, S = kBwdTile / W, kThreads = W * 32;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  BwdSmem<T>& sm = *reinterpret_cast<BwdSmem<T>*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int csize = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int unit = int(blockIdx.x) / csize;
  const int b = unit / p.chan_tiles;
  const int c0 = (unit - b * p.chan_tiles) * kChan;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int c = c0 + 2 * lane;
  const bool ok0 = c < p.channels, ok1 = c + 1 < p.channels;
  const int tiles = (p.seq + kBwdTile - 1) / kBwdTile;
  const int64_t row0 = int64_t(b) * p.seq;
  const T* x = static_cast<const T*>(p.x) + row0 * p.xs + c0;
  const T* r = static_cast<const T*>(p.r) + row0 * p.rs + c0;
  const T* iv = static_cast<const T*>(p.i) + row0 * p.is + c0;
  const T* dy = p.dy ? static_cast<const T*>(p.dy) + row0 * p.dys + c0 : nullptr;
  const int64_t out0 = row0 * p.channels + c;
  const uint8_t* rst = kReset ? p.reset + row0 : nullptr;
  const float2 lam = load_f2(p.lambda, c, ok0, ok1);
  const float2 nrate = neg_rate2(lam, p.sharpness, ok0, ok1);
  const bool small = small_rates(nrate);
  // threads 0 .. 63 join the states, 64 .. 127 the gradients, one channel each
  const int jch = tid & (kChan - 1), jc = c0 + jch;
  const bool jok = tid < 2 * kChan && jc < p.channels;
  float carry = jok && p.dhT ? p.dhT[int64_t(b) * p.channels + jc] : 0.f;
  float2 dlam = bc2(0.f);

  auto load = [&](int tile, int st) {
    const int64_t t0 = int64_t(tile) * kBwdTile;
    const int rows = p.seq - int(t0), cols = p.channels - c0;
    copy_tile<T, kBytes, kThreads, kBwdTile>(&sm.raw[st][0][0][0], x + t0 * p.xs, p.xs, rows, cols);
    copy_tile<T, kBytes, kThreads, kBwdTile>(&sm.raw[st][1][0][0], r + t0 * p.rs, p.rs, rows, cols);
    copy_tile<T, kBytes, kThreads, kBwdTile>(&sm.raw[st][2][0][0], iv + t0 * p.is, p.is, rows, cols);
    if (dy != nullptr)
      copy_tile<T, kBytes, kThreads, kBwdTile>(&sm.raw[st][3][0][0], dy + t0 * p.dys, p.dys, rows, cols);
  };
  if (dy == nullptr)
    for (int k = tid; k < 2 * kBwdTile * kChan; k += kThreads)
      sm.raw[k / (kBwdTile * kChan)][3][0][k % (kBwdTile * kChan)] = T(0.f);

  if (csize > 1) exchange_init(&sm.ex);
  // the cluster's tiles are taken from the end: rank 0 the last of each group
  if (rank < tiles) load(tiles - 1 - rank, 0);
  cp_async_commit();
  if (csize > 1) cluster.sync();  // every CTA's mbarriers are ready before they are written
  bool alive = true;
  int round = 0;
  for (int done = 0; done < tiles; done += csize, ++round) {
    const int tile = tiles - 1 - done - rank, st = round & 1;  // below 0: an empty tile
    const int t0 = tile * kBwdTile + warp * S;
    float h_tile = 0.f;
    if (jok && tid < kChan && tile >= 0)
      h_tile = p.ckpt[(int64_t(b) * tiles + tile) * p.channels + jc];
    cp_async_wait_all();
    __syncthreads();  // the tile has landed; the other buffer is no longer read
    if (tile - csize >= 0) load(tile - csize, st ^ 1);
    cp_async_commit();
    float2 a[S], sr[S], si[S], beta[S];
    bool drop[S];
    float2 D = bc2(-kTiny), E = bc2(0.f), G = bc2(0.f);
    // steps past the end pass c on (x and dy are 0 there); whole tiles do not look for it
    auto reduce = [&](auto whole, auto slow) {
      Product2 t = {bc2(0.f), bc2(1.f)};
      bool dropped = false;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int row = warp * S + s;
        const bool in = decltype(whole)::value || t0 + s < p.seq;
        float2 m, q;
        sr[s] = sigmoid2(unpack2(&sm.raw[st][1][row][2 * lane]));
        si[s] = sigmoid2(unpack2(&sm.raw[st][2][row][2 * lane]));
        decay2<decltype(slow)::value>(mul2(nrate, sr[s]), a[s], m, q);
        beta[s] = sqrt2(q);
        drop[s] = kReset && in && rst[t0 + s] != 0;
        const float2 v = mul2(si[s], unpack2(&sm.raw[st][0][row][2 * lane]));
        if (!in) {
          m = bc2(0.f);
          a[s] = bc2(1.f);
        }
        if (kReset && drop[s]) {
          E = v;
          dropped = true;
        } else {
          E = fma2(a[s], E, mul2(beta[s], v));
          join_step<decltype(slow)::value>(t, a[s], m);
        }
      }
      D = kReset && dropped ? bc2(kDropped) : product_of<decltype(slow)::value>(t);
#pragma unroll
      for (int s = S - 1; s >= 0; --s) {
        const float2 g = add2(unpack2(&sm.raw[st][3][warp * S + s][2 * lane]), G);
        G = kReset && drop[s] ? bc2(0.f) : mul2(a[s], g);
      }
    };
    const bool here = tile >= 0, whole = here && (tile + 1) * kBwdTile <= p.seq;
    if (whole && small) reduce(std::true_type{}, std::true_type{});
    else if (whole) reduce(std::true_type{}, std::false_type{});
    else if (here) reduce(std::false_type{}, std::false_type{});
    *reinterpret_cast<float4*>(&sm.run[warp][2 * lane]) = make_float4(D.x, E.x, D.y, E.y);
    *reinterpret_cast<float2*>(&sm.back[warp][2 * lane]) = G;
    __syncthreads();
    if (tid < kChan) {
      auto place = [&](auto infinite) {
        float h = h_tile, seen = 0.f;
        float2 run[W];
#pragma unroll
        for (int w = 0; w < W; ++w) run[w] = sm.run[w][jch];
#pragma unroll
        for (int w = 0; w < W; ++w) {
          sm.start[w][jch] = h;
          h = apply<kReset, decltype(infinite)::value>(run[w].x, run[w].y, h);
          if (kReset) seen = fmaf(h, 0.f, seen);
        }
        seen = fmaf(h, 0.f, seen);
        return seen != seen;
      };
      if (place(std::false_type{})) place(std::true_type{});
    } else if (tid < 2 * kChan) {
      if (csize > 1) {
        const float td = tile_product<kReset, W>(sm.run, jch);
        auto total = [&](auto infinite) {
          float tg = 0.f;
#pragma unroll
          for (int w = W - 1; w >= 0; --w)
            tg = apply<kReset, decltype(infinite)::value>(sm.run[w][jch].x, sm.back[w][jch], tg);
          return tg;
        };
        float tg = total(std::false_type{});
        if (tg != tg) tg = total(std::true_type{});
        if (alive)
          alive = exchange(&sm.ex, st, uint32_t(round >> 1) & 1u, rank, csize, jch, td, tg, p.give_up != 0, p.status);
      }
      // c over the round, and c after each run (loaded before, not between, the joins: 67.4
      // us instead of 70 at 4 x 2048 x 1536; forward, with fewer registers, it is the reverse)
      float next, D_of[W], G_of[W];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        D_of[w] = sm.run[w][jch].x;
        G_of[w] = sm.back[w][jch];
      }
      auto place = [&](auto infinite) {
        constexpr bool kInf = decltype(infinite)::value;
        float cc = carry, seen = 0.f;
        next = carry;
        if (csize > 1) {
#pragma unroll 4
          for (int k = 0; k < csize; ++k) {
            if (k == rank) cc = next;
            const float2 g = sm.ex.sum[st][k][jch];
            next = apply<kReset, kInf>(g.x, g.y, next);
            if (kReset) seen = fmaf(next, 0.f, seen);
          }
          seen = fmaf(next, 0.f, seen);
        }
#pragma unroll
        for (int w = W - 1; w >= 0; --w) {
          sm.after[w][jch] = cc;
          cc = apply<kReset, kInf>(D_of[w], G_of[w], cc);
          if (kReset) seen = fmaf(cc, 0.f, seen);
        }
        seen = fmaf(cc, 0.f, seen);
        if (csize == 1) next = cc;
        return seen != seen;
      };
      if (place(std::false_type{})) place(std::true_type{});
      carry = next;
    }
    __syncthreads();
    // h[t-1] of each step forwards, then the gradients backwards
    auto write = [&](auto whole) {
      float2 h = *reinterpret_cast<const float2*>(&sm.start[warp][2 * lane]);
      float2 cc = *reinterpret_cast<const float2*>(&sm.after[warp][2 * lane]);
      float2 term[S];  // a / beta s(i) x - h[t-1]: what c is multiplied by in dL
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const float2 v = mul2(si[s], unpack2(&sm.raw[st][0][warp * S + s][2 * lane]));
        term[s] = fma2(mul2(a[s], inv_beta2(beta[s])), v, neg2(h));
        h = kReset && drop[s] ? v : fma2(a[s], h, mul2(beta[s], v));
        if (kReset && drop[s]) beta[s] = bc2(1.f);
      }
#pragma unroll
      for (int s = S - 1; s >= 0; --s) {
        const int row = warp * S + s;
        const float2 gs = add2(unpack2(&sm.raw[st][3][row][2 * lane]), cc);
        cc = kReset && drop[s] ? bc2(0.f) : mul2(a[s], gs);
        const float2 dx = mul2(mul2(gs, beta[s]), si[s]);
        const float2 di = mul2(mul2(dx, unpack2(&sm.raw[st][0][row][2 * lane])),
                               add2(bc2(1.f), neg2(si[s])));
        float2 ds = mul2(mul2(cc, term[s]), sr[s]);
        if (kReset && drop[s]) ds = bc2(0.f);
        const float2 dr = mul2(mul2(ds, nrate), add2(sr[s], bc2(-1.f)));
        if (decltype(whole)::value || t0 + s < p.seq) {
          dlam = add2(dlam, ds);
          const int64_t o = out0 + int64_t(t0 + s) * p.channels;
          store2<kVec>(static_cast<T*>(p.dx) + o, dx, ok0, ok1);
          store2<kVec>(static_cast<T*>(p.dr) + o, dr, ok0, ok1);
          store2<kVec>(static_cast<T*>(p.di) + o, di, ok0, ok1);
        }
      }
    };
    if (whole) write(std::true_type{});
    else if (here) write(std::false_type{});
  }
  if (p.dh0 != nullptr && rank == 0 && jok && tid >= kChan) p.dh0[int64_t(b) * p.channels + jc] = carry;
  __syncthreads();
  float2(*red)[32] = reinterpret_cast<float2(*)[32]>(&sm.run[0][0]);
  red[warp][lane] = dlam;
  __syncthreads();
  if (warp == 0) {
    float2 t = red[0][lane];
    for (int w = 1; w < W; ++w) t = add2(t, red[w][lane]);
    float* q = p.part + (int64_t(b) * csize + rank) * p.channels + c;
    if (ok0) q[0] = t.x;
    if (ok1) q[1] = t.y;
  }
  if (csize > 1) cluster.sync();  // no CTA leaves while another may still write to it
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

// A thread takes two adjacent channels of one sequence.
template <typename T, bool kVec>
__global__ void __launch_bounds__(128)
    gated_step_kernel(const T* __restrict__ x, const T* __restrict__ r, const T* __restrict__ i,
                      int64_t xs, int64_t rs, int64_t is, const float* __restrict__ lambda,
                      float* __restrict__ h, T* __restrict__ y, int64_t batch, int channels,
                      int pairs, float sharpness) {
  const int64_t n = int64_t(blockIdx.x) * 128 + threadIdx.x;
  const int64_t b = n / pairs;
  if (b >= batch) return;
  const int c = int(n - b * pairs) * 2;
  const bool ok1 = c + 1 < channels;
  auto load = [&](const T* p) {
    if constexpr (kVec) return unpack2(p);
    else return make_float2(to_f(p[0]), ok1 ? to_f(p[1]) : 0.f);
  };
  const float2 xv = load(x + b * xs + c), rv = load(r + b * rs + c), iv = load(i + b * is + c);
  float* hb = h + b * channels + c;
  const float2 h0 = make_float2(hb[0], ok1 ? hb[1] : 0.f);
  const float2 lam = load_f2(lambda, c, true, ok1);
  const float2 nrate = neg_rate2(lam, sharpness, true, true);
  float2 a, m, q;
  decay2<false>(mul2(nrate, sigmoid2(rv)), a, m, q);
  const float2 u = mul2(sqrt2(q), mul2(sigmoid2(iv), xv));
  const float2 hn = fma2(a, h0, u);
  hb[0] = hn.x;
  if (ok1) hb[1] = hn.y;
  store2<kVec>(y + b * channels + c, hn, true, ok1);
}

// ----------------------------------------------------------------------- host

// How many clusters of each size of a kernel fit the device at once (asked once for
// each kernel and device; a repeated question gives the same answer).
constexpr int kSizes[] = {1, 2, 3, 4, 5, 6, 7, 8, 12, 16};
constexpr int kSizeCount = int(sizeof(kSizes) / sizeof(int));
struct Fit {
  std::atomic<int> known{0};
  std::atomic<int> clusters[kSizeCount];
};

cudaLaunchConfig_t cluster_config(cudaLaunchAttribute* at, int64_t grid, int threads, size_t smem,
                                  int c, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  at->id = cudaLaunchAttributeClusterDimension;
  at->val.clusterDim.x = unsigned(c);
  at->val.clusterDim.y = at->val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cfg;
}

template <typename K>
void ask_fit(K kernel, int threads, size_t smem, int most, Fit& fit) {
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (most > 8) cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  for (int k = 0; k < kSizeCount; ++k) {
    int n = 0;
    cudaLaunchAttribute at;
    const cudaLaunchConfig_t cfg = cluster_config(&at, kSizes[k], threads, smem, kSizes[k], nullptr);
    if (kSizes[k] > most || cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) n = 0;
    cudaGetLastError();
    fit.clusters[k].store(n);
  }
  fit.known.store(1);
}

// What a round of a tile takes in a wave of clusters, in units of what each CTA that
// shares the SM adds to it: `latency`, and the exchange between up to `few` CTAs or more.
// Fitted to bf16 at nine shapes and cluster sizes 1 to 16; us at the sizes 1, 2, 4, 8:
//   forward (units of 0.8 us)     4 x 2048 x 1536  66, 48, 35, 40  64 x 512 x 1024  68, 79, 100, 145
//   backward (units of 0.88 us)   4 x 2048 x 1536  84, 80, 68, 73  64 x 512 x 1024  120, 149, 180, 252
//                                 6 x 2048 x 1536  87, 80, 105, 108
// fp32 (sizes up to 8) goes by the same numbers: 4 x 2048 x 1536 forward 78, 52, 51, 52,
// backward 104, 92, 80, 84. Against every size at 16 shapes (1 to 512 sequences of 64 to
// 32768 steps) the size taken is within 3 % of the best in 29 of 32 bf16 and 26 of 32 fp32
// launches; farthest off: 32 x 100 x 512 forward 9.1 and 7.9 us, 3 x 2048 x 1536 forward
// 33 and 31, fp32 46 and 39, 8 x 512 x 1536 backward 39 and 36, 1 x 32768 x 1024 backward,
// fp32, 366 and 340.
struct RoundCost {
  double latency, exchange_few, exchange_more;
  int few;
};
constexpr RoundCost kFwdShortCost = {1.9, 0.4, 1.5, 5};  // tiles of 32, units of 0.43 us
constexpr RoundCost kFwdCost = {1.5, 0.4, 1.6, 2};
constexpr RoundCost kBwdCost = {0.5, 0.4, 0.9, 4};

// Launches `units` clusters, one for each 64 channels of a sequence. The CTAs of a
// cluster take consecutive tiles; of the sizes that fit (no more CTAs than tiles) it
// is the one that takes the least time by a model of waves of clusters x rounds of a
// tile x RoundCost. *size: the size taken.
template <auto kernel, typename A>
int launch_clusters(const char* what, const A& args, int threads, size_t smem, int most,
                    int64_t units, int tiles, const RoundCost& cost, cudaStream_t st, int* size) {
  static Fit fits[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  MQC_REQUIRE(e == cudaSuccess && dev >= 0 && dev < 64, MQC_ERR_CUDA, "%s: no device", what);
  Fit& fit = fits[dev];
  if (!fit.known.load()) ask_fit(kernel, threads, smem, most, fit);
  int c = 0;
  double least = 0.0;
  const double sms = num_sms();
  for (int k = 0; k < kSizeCount && (c == 0 || kSizes[k] <= tiles); ++k) {
    const int64_t n = fit.clusters[k].load(), size = kSizes[k];
    if (n <= 0) continue;
    const double exchange = size == 1 ? 0.0 : size <= cost.few ? cost.exchange_few : cost.exchange_more;
    auto wave = [&](int64_t u) {  // of u clusters
      return u == 0 ? 0.0 : cost.latency + exchange + std::ceil(double(u * size) / sms);
    };
    const double time = double((tiles + size - 1) / size) *
                        (double(units / n) * wave(n) + wave(units % n));
    if (c == 0 || time < least) {
      least = time;
      c = int(size);
    }
  }
  MQC_REQUIRE(c > 0, MQC_ERR_CUDA, "%s: the kernel does not fit the device", what);
  MQC_REQUIRE(units * c <= 0x7fffffffll, MQC_ERR_UNSUPPORTED, "%s: too many channel tiles", what);
  cudaLaunchAttribute at;
  const cudaLaunchConfig_t cfg = cluster_config(&at, units * c, threads, smem, c, st);
  e = cudaLaunchKernelEx(&cfg, kernel, args);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(MQC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  *size = c;
  return check_launch(what);
}

template <typename T, int kBytes, bool kVec, bool kReset, int kWarps>
int run_fwd_tiles(const FwdArgs& f, const RoundCost& cost, cudaStream_t st) {
  int c;
  return launch_clusters<&gated_scan_fwd_kernel<T, kBytes, kVec, kReset, kWarps>>(
      "mqc_gated_scan_fwd", f, kWarps * 32, sizeof(FwdSmem<T, kWarps>), kMaxCluster<T>,
      int64_t(f.batch) * f.chan_tiles, (f.seq + kWarps * kRun - 1) / (kWarps * kRun), cost, st, &c);
}

template <typename T, int kBytes, bool kVec, bool kReset>
int run_fwd(const FwdArgs& f, cudaStream_t st) {
  return f.seq <= kShort ? run_fwd_tiles<T, kBytes, kVec, kReset, 4>(f, kFwdShortCost, st)
                         : run_fwd_tiles<T, kBytes, kVec, kReset, 8>(f, kFwdCost, st);
}

template <typename T, int kBytes, bool kVec, bool kReset>
int run_bwd(const BwdArgs& f, float* dlambda, cudaStream_t st) {
  int c = 0;
  if (int rc = launch_clusters<&gated_scan_bwd_kernel<T, kBytes, kVec, kReset>>(
          "mqc_gated_scan_bwd", f, kBwdWarps * 32, sizeof(BwdSmem<T>), kMaxCluster<T>,
          int64_t(f.batch) * f.chan_tiles, (f.seq + kBwdTile - 1) / kBwdTile, kBwdCost, st, &c))
    return rc;
  gated_scan_dlambda_kernel<<<(f.channels + 31) / 32, 256, 0, st>>>(
      f.part, f.lambda, dlambda, f.batch * c, f.channels, f.sharpness);
  return check_launch("mqc_gated_scan_bwd (dLambda)");
}

constexpr int kLargestCluster = 16;

int check_sizes(const char* what, const mqc_gated_scan_args* a) {
  MQC_REQUIRE(a != nullptr, MQC_ERR_INVALID_VALUE, "%s: args is NULL", what);
  MQC_REQUIRE(dtype_ok(a->dtype), MQC_ERR_INVALID_VALUE, "%s: dtype %d", what, a->dtype);
  MQC_REQUIRE(a->batch >= 0 && a->seq_len >= 0 && a->channels >= 0, MQC_ERR_INVALID_VALUE,
              "%s: batch %lld, seq_len %lld, channels %lld", what, (long long)a->batch,
              (long long)a->seq_len, (long long)a->channels);
  MQC_REQUIRE(a->seq_len <= 0x7fffffff - 2 * kLargestCluster * 64 && a->channels <= 0x7fffffff - kChan &&
                  a->batch <= 0x7fffffff / kLargestCluster,
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

// Whether `group` adjacent channels can move as one word: strides and bases are
// multiples of it.
bool groups_ok(int64_t group, uintptr_t es, std::initializer_list<const void*> ptrs,
               std::initializer_list<int64_t> strides) {
  for (const void* q : ptrs)
    if (!aligned(q, group * es)) return false;
  for (int64_t s : strides)
    if (s % group) return false;
  return true;
}

// What a copy into shared memory moves at once, by alignment: 16 bytes, 4, or (bf16
// of odd stride or base) 2. Pairs of channels are stored as one word with the first
// two of bf16 and the first of fp32.
int copy_bytes(int64_t channels, uintptr_t es, std::initializer_list<const void*> in,
               std::initializer_list<const void*> out, std::initializer_list<int64_t> strides) {
  const bool pairs = channels % 2 == 0 && groups_ok(2, es, out, {});
  if (pairs && groups_ok(16 / es, es, in, strides)) return 16;
  if (es == 4 || (pairs && groups_ok(2, es, in, strides))) return 4;
  return 2;
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
               static_cast<float*>(a->ckpt), static_cast<int*>(a->status), a->give_up, int(a->batch),
               int(a->seq_len), int(a->channels), int((a->channels + kChan - 1) / kChan),
               a->sharpness};
  const int bytes = copy_bytes(a->channels, es, {a->x, a->r, a->i}, {a->y},
                               {a->x_row, a->r_row, a->i_row});
  const bool rst = a->reset != nullptr;
#define MQC_RUN(...) (rst ? run_fwd<__VA_ARGS__, true>(f, st) : run_fwd<__VA_ARGS__, false>(f, st))
  if (a->dtype == MQC_DTYPE_F32)
    return bytes == 16 ? MQC_RUN(float, 16, true) : MQC_RUN(float, 4, false);
  if (bytes == 16) return MQC_RUN(__nv_bfloat16, 16, true);
  return bytes == 4 ? MQC_RUN(__nv_bfloat16, 4, true) : MQC_RUN(__nv_bfloat16, 2, false);
#undef MQC_RUN
}

size_t mqc_gated_scan_bwd_workspace_size(int64_t batch, int64_t seq_len, int64_t channels) {
  if (batch <= 0 || seq_len <= 0 || channels <= 0) return 0;
  return size_t(batch) * size_t(channels) * mqc::kLargestCluster * sizeof(float);
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
               a->di, static_cast<float*>(a->dh0), static_cast<float*>(workspace),
               static_cast<int*>(a->status), a->give_up, int(a->batch), int(a->seq_len),
               int(a->channels), int((a->channels + kChan - 1) / kChan), a->sharpness};
  float* dl = static_cast<float*>(a->dlambda);
  const int bytes = copy_bytes(a->channels, es, {a->x, a->r, a->i, a->dy}, {a->dx, a->dr, a->di},
                               {a->x_row, a->r_row, a->i_row, a->dy ? a->dy_row : 0});
  const bool rst = a->reset != nullptr;
#define MQC_RUN(...) \
  (rst ? run_bwd<__VA_ARGS__, true>(f, dl, st) : run_bwd<__VA_ARGS__, false>(f, dl, st))
  if (a->dtype == MQC_DTYPE_F32)
    return bytes == 16 ? MQC_RUN(float, 16, true) : MQC_RUN(float, 4, false);
  if (bytes == 16) return MQC_RUN(__nv_bfloat16, 16, true);
  return bytes == 4 ? MQC_RUN(__nv_bfloat16, 4, true) : MQC_RUN(__nv_bfloat16, 2, false);
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
  const bool vec = channels % 2 == 0 && groups_ok(2, es, {x, r, i, y}, {x_row, r_row, i_row});
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
