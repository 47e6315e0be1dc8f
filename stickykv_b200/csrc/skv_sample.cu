// skv_sample: the next token of each row from its logits and a given random
// number (temperature, top-k, top-p, min-p).
//
// In descending order with ties by index every cut is a threshold: the key of
// the last kept token and how many of its equals, lowest indices first, stay.
// No sort.  A cluster holds a row in its blocks' shared memory (up to 315
// thousand float32 or 630 thousand 16-bit tokens; of a longer row every pass
// reads global memory); every 256 tokens' largest is kept beside them, and
// passes skip those below what they look for.
//   few of top-k   a value that k of those maxima reach bounds the cut; the
//                  tokens from there on, little more than k, are listed;
//   top-k, top-p   a histogram (counts, weights) over evenly spaced values
//                  below the maximum names the bin that holds the cut; the
//                  bin's tokens are listed, what lies above is summed exactly;
// the cut is then found in the list, by comparing each with each or by 8 bits of
// the keys a turn.  The sums prove that the list holds it; where it does not, or
// equals overflow the list, the row is searched bit by bit.
//
// Weights and sums are 64-bit: a draw falls between two neighbours of 10^5
// cumulative sums, and 32-bit sums would move a share of draws to a neighbour.
// Sums are taken in a fixed order, or, where the order is not fixed, as whole
// numbers of 2^-52 of the largest weight (the step of a 64-bit sum of which that
// is part), so equal calls give equal tokens.
//
// Bound: one row is latency, three to six cluster barriers (32000 tokens: greedy
// 3.3 us, top-k 50 13 us, with top-p 0.95 15 us).  Many rows: rounds of blocks,
// one an SM (16 warps; shared memory and registers hold no second), whose warps
// wait for their own last results with nobody to step in: issue at 51 %, the
// 64-bit pipe at 24 %, HBM read once (rows that fit).  128 rows x 128256 bf16 are
// two rounds: greedy 12 us, 2.8 TB/s; temperature 46 us; top-p 0.9 119 to 125 us
// (74 rows, one round: 6.6, 24, 65 us).  A block of 256 tokens of which one is
// kept is weighed whole, at a top-p cut twice.
#include <float.h>

#include <type_traits>

#include "skv_common.cuh"

namespace skv {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBlock = 256;        // tokens a warp takes at once: 8 neighbours a lane
constexpr int kBins = 1024;
constexpr int kPerThread = kBins / kThreads;
constexpr int kList = 2048;        // tokens that are searched in registers, 4 a thread
constexpr int kRanked = 192;       // listed tokens up to here are compared each with each (n^2 / 512 steps a thread; more take
                                   // three to four turns of 8 bits, about 1.5 us each)
constexpr int kLists = 4;          // made for a row at most: two for top-k, two for top-p
constexpr int kMaxCluster = 8;
constexpr uint32_t kNone = 0x007fffffu;  // key of -inf
constexpr double kUnit = 4503599627370496.0;  // 2^52: a listed weight as a whole number

struct SampleParams {
  const void* logits;
  int64_t stride;
  const float* u;
  const float* temps;
  const int32_t* ks;
  const float* ps;
  const float* mins;
  int64_t* out;
  float temp, p, min_p;
  int k, V;
  int per_cta;   // blocks of 256 tokens of a CTA
  int staged;    // the row's slice is held in shared memory
};

// Total order of the values as unsigned integers (without NaN; -0 as +0).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// 16 bytes of logits: NaN to -inf, their maximum and minimum, and as floats.
template <typename T> struct Pack;
template <> struct Pack<float> {
  static constexpr int N = 4;
  float v[4];
  __device__ __forceinline__ void clean() {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fmaxf(v[i], -INFINITY);
  }
  __device__ __forceinline__ float top() const { return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])); }
  __device__ __forceinline__ float least() const { return fminf(fminf(v[0], v[1]), fminf(v[2], v[3])); }
  __device__ __forceinline__ void floats(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = v[i];
  }
};
template <typename T2> struct Pack2 {
  static constexpr int N = 8;
  T2 v[4];
  __device__ __forceinline__ T2 top2() const { return __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3])); }
  __device__ __forceinline__ T2 least2() const { return __hmin2(__hmin2(v[0], v[1]), __hmin2(v[2], v[3])); }
};
template <> struct Pack<__half> : Pack2<__half2> {
  __device__ __forceinline__ void clean() {
    const __half2 low = __float2half2_rn(-INFINITY);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __hmax2(v[i], low);
  }
  __device__ __forceinline__ float top() const { const float2 f = __half22float2(top2()); return fmaxf(f.x, f.y); }
  __device__ __forceinline__ float least() const { const float2 f = __half22float2(least2()); return fminf(f.x, f.y); }
  __device__ __forceinline__ void floats(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<float2*>(f)[i] = __half22float2(v[i]);
  }
};
template <> struct Pack<__nv_bfloat16> : Pack2<__nv_bfloat162> {
  __device__ __forceinline__ void clean() {
    const __nv_bfloat162 low = __float2bfloat162_rn(-INFINITY);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __hmax2(v[i], low);
  }
  __device__ __forceinline__ float top() const { const float2 f = __bfloat1622float2(top2()); return fmaxf(f.x, f.y); }
  __device__ __forceinline__ float least() const { const float2 f = __bfloat1622float2(least2()); return fminf(f.x, f.y); }
  __device__ __forceinline__ void floats(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<float2*>(f)[i] = __bfloat1622float2(v[i]);
  }
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <typename A>
__device__ __forceinline__ A peer(const A* p, int rank) {  // another block's copy of a shared variable
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
  if constexpr (sizeof(A) == 8) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];\n" : "=l"(v) : "r"(a) : "memory");
    return *reinterpret_cast<A*>(&v);
  } else {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(a) : "memory");
    return *reinterpret_cast<A*>(&v);
  }
}

__device__ __forceinline__ uint4 peer4(const uint32_t* p, int rank) {
  uint32_t a;
  uint4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// What the blocks of a cluster tell one another.
struct Shared {
  uint64_t warp_best[kWarps];             // of each warp: largest key above the complement of its first block's place
  uint32_t warp_least[kWarps];            // smallest key
  uint32_t warp_min[kWarps];              // smallest of its lanes' largest keys
  uint32_t listed[kLists];
  uint32_t list_lo[kLists], list_hi[kLists];        // smallest and largest listed key
  uint32_t finite;                        // smallest key above -inf, where the row holds such
  uint32_t list_above;                    // tokens above the list
  double mass[2];                         // above the bracket; below its upper end
  double turn_d[2];                       // bit by bit search, in turns
  uint32_t turn_u[2];
  double kept;                            // mass above the threshold, of the block's tokens
  uint32_t ties;                          // equals of the threshold
  // within the block
  alignas(16) uint32_t all_min[kWarps * kMaxCluster];  // warp_min of all blocks
  uint64_t best[kMaxCluster / 2];
  uint32_t least[kMaxCluster / 2];
  uint32_t list_end[kMaxCluster];         // listed tokens of the blocks up to each
  uint32_t span_lo, span_hi, all_above;   // of all blocks' lists
  uint64_t red[2][kWarps];                // reductions, in turns
  int found, last;
  uint32_t pick_key;
  uint64_t pick_above, pick_equal;
  double found_before, carry_mass;
  uint32_t found_ties, carry_ties;
};

// w(x) = 2^((x - m) c), c = log2 e / T, in 64 bits: 2^n 2^f with n whole and
// |f| <= 1/2, the latter by the polynomial that interpolates 2^f at the 11
// Chebyshev nodes of [-1/2, 1/2] (off by 3.2e-16 of itself at most, a rounding
// or two of 64 bits; exactly 1 at 0).
// Where the exponent is above -1000 only; further down a weight counts as none.
struct Weight {
  double m, c;
  __device__ __forceinline__ double operator()(float x) const {
    const double d = (double)x - m;
    const double t = fma(d, c, 6755399441055744.0);  // 1.5 * 2^52: rounds to whole numbers
    const double f = fma(d, c, -(t - 6755399441055744.0));
    double e = 7.072585949269223e-09;
    e = fma(e, f, 1.0208690299958306e-07);
    e = fma(e, f, 1.321544258792169e-06);
    e = fma(e, f, 1.5252657260200837e-05);
    e = fma(e, f, 0.0001540353044173605);
    e = fma(e, f, 0.0013333558230164974);
    e = fma(e, f, 0.009618129107606888);
    e = fma(e, f, 0.05550410866444772);
    e = fma(e, f, 0.24022650695910097);
    e = fma(e, f, 0.69314718055995);
    e = fma(e, f, 1.0);
    return __hiloint2double(__double2hiint(e) + (__double2loint(t) << 20), __double2loint(e));
  }
};

template <typename A, typename Op>
__device__ __forceinline__ A warp_reduce(A v, Op op) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename A>
__device__ __forceinline__ A warp_prefix(A v, int n) {  // inclusive, over groups of n lanes
#pragma unroll
  for (int o = 1; o < n; o <<= 1) {
    const A d = __shfl_up_sync(0xffffffffu, v, o, n);
    if ((int)(threadIdx.x & (n - 1)) >= o) v += d;
  }
  return v;
}

struct Max { template <typename A> __device__ A operator()(A a, A b) const { return a > b ? a : b; } };
struct Min { template <typename A> __device__ A operator()(A a, A b) const { return a < b ? a : b; } };
struct Sum { template <typename A> __device__ A operator()(A a, A b) const { return a + b; } };

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Shared sh;
  __shared__ __align__(16) uint32_t hist[kBins];
  __shared__ __align__(16) float gathered[2][kBins];  // of half the cluster's blocks each
  __shared__ uint32_t list[kList];
  // of a search in the list, 8 bits a turn: weights in three parts whose sums over the list fit 32 bits each (one
  // add of 64 bits is a loop of compare-and-swap, and most listed keys share their upper digits)
  __shared__ uint32_t digits[4][3][256];
  // a short list: keys and weights
  __shared__ __align__(16) uint32_t ranked[kRanked];
  __shared__ __align__(16) unsigned long long ranked_w[kRanked];
  double* blk_mass = reinterpret_cast<double*>(smem);                       // [per_cta]
  uint32_t* blk_ties = reinterpret_cast<uint32_t*>(blk_mass + p.per_cta);   // [per_cta]
  float* blk_top = reinterpret_cast<float*>(blk_ties + p.per_cta);          // [per_cta] largest logit
  T* data = reinterpret_cast<T*>(smem + align_up((size_t)p.per_cta * 16, 16));

  uint32_t rank, size;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(size));
  const int C = (int)size, me = (int)rank;
  const int b = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = p.V;
  const T* x = (const T*)p.logits + b * p.stride;
  const float temp = p.temps ? p.temps[b] : p.temp, uniform = p.u[b], given_share = p.ps ? p.ps[b] : p.p;
  const float share = given_share <= 0.f ? FLT_MIN : given_share;  // one token, by way of the list as any other share
  const float min_p = p.mins ? p.mins[b] : p.min_p;
  const int k = min(p.ks ? p.ks[b] : p.k, V);  // from V on it cuts nothing; doubled below
  const int blk0 = me * p.per_cta;                                // first block of this CTA
  const int n_blk = max(0, min(p.per_cta, ceil_div(V, kBlock) - blk0));
  auto cluster_arrive = [&] {
    if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  };
  auto cluster_wait = [&] {
    if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
  };
  auto cluster_barrier = [&] {
    if (C > 1) {
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();
    }
  };
  // over the block: two buffers in turn, so one barrier each
  int turn_r = 0;
  auto block_reduce = [&](auto v, auto op) {
    using A = decltype(v);
    A* buf = reinterpret_cast<A*>(sh.red[turn_r++ & 1]);
    v = warp_reduce(v, op);
    if (lane == 0) buf[warp] = v;
    __syncthreads();
    v = buf[lane & (kWarps - 1)];
#pragma unroll
    for (int o = kWarps / 2; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };
  auto block_prefix = [&](auto v) {  // inclusive, over the threads
    using A = decltype(v);
    A* buf = reinterpret_cast<A*>(sh.red[turn_r++ & 1]);
    v = warp_prefix(v, 32);
    if (lane == 31) buf[warp] = v;
    __syncthreads();
    const A ends = warp_prefix(buf[lane & (kWarps - 1)], kWarps);
    const A base = __shfl_sync(0xffffffffu, ends, (warp + kWarps - 1) & (kWarps - 1));
    return warp ? base + v : v;
  };
  auto over = [&](const auto* v, auto op) {  // a variable of all blocks of the cluster, the loads in flight together
    auto r = peer(v, 0);
    decltype(r) e[kMaxCluster];
#pragma unroll
    for (int c = 1; c < kMaxCluster; ++c)
      if (c < C) e[c] = peer(v, c);
#pragma unroll
    for (int c = 1; c < kMaxCluster; ++c)
      if (c < C) r = op(r, e[c]);
    return r;
  };

  // ---- 8 neighbouring tokens a lane, of block `blk` of this CTA ------------------------------
  using P = Pack<T>;
  constexpr int kPacks = 8 / P::N;
  const bool wide = ((uintptr_t)x & 15) == 0;
  auto fetch = [&](int blk, P (&v)[kPacks]) {  // from global memory; -inf behind the row
    const int i0 = (blk0 + blk) * kBlock + lane * 8;
    if (wide && i0 + 8 <= V) {
#pragma unroll
      for (int h = 0; h < kPacks; ++h) *reinterpret_cast<uint4*>(&v[h]) = reinterpret_cast<const uint4*>(x + i0)[h];
    } else {
#pragma unroll
      for (int h = 0; h < kPacks; ++h) {
        T e[P::N];
#pragma unroll
        for (int i = 0; i < P::N; ++i)
          e[i] = i0 + h * P::N + i < V ? x[i0 + h * P::N + i] : Elt<T>::from_f32(-INFINITY);
        *reinterpret_cast<uint4*>(&v[h]) = *reinterpret_cast<uint4*>(e);
      }
    }
  };
  bool infinite = false;                       // the largest logit is +inf: such count as 0, the others as -inf
  auto finite = [&](float v) { return infinite ? (v == INFINITY ? 0.f : -INFINITY) : v; };
  auto load = [&](int blk, float (&f)[8]) {
    P v[kPacks];
    if (p.staged) {
      const uint4* s = reinterpret_cast<const uint4*>(data + blk * kBlock + lane * 8);
#pragma unroll
      for (int h = 0; h < kPacks; ++h) *reinterpret_cast<uint4*>(&v[h]) = s[h];
    } else {
      fetch(blk, v);
#pragma unroll
      for (int h = 0; h < kPacks; ++h) v[h].clean();
    }
#pragma unroll
    for (int h = 0; h < kPacks; ++h) v[h].floats(f + h * P::N);
    if (infinite) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = finite(f[i]);
    }
  };
  auto each8 = [&](float least, auto&& f) {    // every 8 tokens of a lane, of this CTA's blocks that reach `least`
    for (int blk = warp; blk < n_blk; blk += kWarps) {
      if (!(finite(blk_top[blk]) >= least)) continue;
      float v[8];
      load(blk, v);
      f(v);
    }
  };

  // ---- the largest logit --------------------------------------------------------------------
  {
    float mx = -INFINITY, mn = INFINITY;
    uint64_t best = 0;
    constexpr int kAhead = 8 / sizeof(T);  // blocks whose loads are in flight together
    for (int blk_a = warp; blk_a < n_blk; blk_a += kAhead * kWarps) {
      P ahead[kAhead][kPacks];
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
        if (blk_a + a * kWarps < n_blk) fetch(blk_a + a * kWarps, ahead[a]);
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int blk = blk_a + a * kWarps, i0 = (blk0 + blk) * kBlock + lane * 8;
        if (blk >= n_blk) break;
        P(&v)[kPacks] = ahead[a];
#pragma unroll
        for (int h = 0; h < kPacks; ++h) v[h].clean();
        if (p.staged) {
          uint4* s = reinterpret_cast<uint4*>(data + blk * kBlock + lane * 8);
#pragma unroll
          for (int h = 0; h < kPacks; ++h) s[h] = *reinterpret_cast<uint4*>(&v[h]);
        }
        float hi = v[0].top(), lo = v[0].least();
        if constexpr (kPacks > 1) hi = fmaxf(hi, v[1].top()), lo = fminf(lo, v[1].least());
        mx = fmaxf(mx, hi);
        if (i0 + 8 <= V) {
          mn = fminf(mn, lo);
        } else {  // without what fills up the last block
          float f[8];
#pragma unroll
          for (int h = 0; h < kPacks; ++h) v[h].floats(f + h * P::N);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i0 + i < V) mn = fminf(mn, f[i]);
        }
        const uint32_t key = __reduce_max_sync(0xffffffffu, key_of(hi));
        if (lane == 0) blk_top[blk] = value_of(key);
        if (key > (uint32_t)(best >> 32)) best = (uint64_t)key << 32 | ~(uint32_t)(blk0 + blk);
      }
    }
    const uint32_t lane_min = __reduce_min_sync(0xffffffffu, key_of(mx)), low = __reduce_min_sync(0xffffffffu, key_of(mn));
    if (lane == 0) {
      sh.warp_best[warp] = best;
      sh.warp_least[warp] = low;
      sh.warp_min[warp] = lane_min;
    }
    if (tid < kLists) {
      sh.listed[tid] = 0;
      sh.list_lo[tid] = 0xffffffffu;
      sh.list_hi[tid] = 0;
      sh.list_above = 0;
    }
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
  }
  cluster_barrier();
  if (tid < kWarps * kMaxCluster) {
    const bool have = tid < kWarps * C;
    const int w = tid % kWarps, c = tid / kWarps;
    uint64_t best = have ? peer(&sh.warp_best[w], c) : 0;
    uint32_t low = have ? peer(&sh.warp_least[w], c) : 0xffffffffu;
    sh.all_min[tid] = have ? peer(&sh.warp_min[w], c) : 0;
    best = warp_reduce(best, Max());
    low = __reduce_min_sync(0xffffffffu, low);
    if (lane == 0) {
      sh.best[warp] = best;
      sh.least[warp] = low;
    }
  }
  __syncthreads();
  uint64_t best = sh.best[0];
  uint32_t least_key = sh.least[0];
#pragma unroll
  for (int i = 1; i < kMaxCluster / 2; ++i) {
    best = max(best, sh.best[i]);
    least_key = min(least_key, sh.least[i]);
  }
  uint32_t top = (uint32_t)(best >> 32);
  if (top == kNone || !(temp > 0.f)) {  // nothing above -inf; greedy
    cluster_arrive();
    if (top == kNone) {
      if (me == 0 && tid == 0) p.out[b] = -1;
    } else {
      const int blk = (int)~(uint32_t)best - blk0;  // the first block that reaches it
      if (blk >= 0 && blk < n_blk && warp == 0) {
        float v[8];
        load(blk, v);
        int at = 8;
#pragma unroll
        for (int i = 7; i >= 0; --i)
          if (key_of(v[i]) == top) at = i;
        const uint32_t hit = __ballot_sync(0xffffffffu, at < 8);
        if (lane == __ffs(hit) - 1) p.out[b] = (int64_t)(blk0 + blk) * kBlock + lane * 8 + at;
      }
    }
    cluster_wait();  // no block leaves while others read its variables
    return;
  }
  if (top == 0xff800000u) {
    infinite = true;
    top = key_of(0.f);
    least_key = kNone;
  }
  const float m = value_of(top);
  const double per_t = 1.4426950408889634074 / (double)temp;
  const Weight weight{(double)m, per_t};
  // weights of keys below `low_key` count as none
  const uint32_t low_key = min(top, max(key_of(m - (float)(1000.0 / per_t)), kNone) + 1);
  auto safe_weight = [&](uint32_t key) { return key >= low_key ? weight(value_of(key)) : 0.0; };
  auto whole_weight = [&](uint32_t key) { return (uint64_t)__double2ll_rn(safe_weight(key) * kUnit); };

  // ---- search over the whole row, bit by bit (counts or masses of keys >= t, those kept) -------
  uint32_t tau = 0, ties = (uint32_t)V;  // kept: keys above tau and `ties` of its equals
  int turn = 0;
  auto count_from = [&](uint32_t t) {
    uint32_t n = 0;
    const float least = value_of(t);
    each8(least, [&](const float (&v)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) n += v[i] >= least;
    });
    n = block_reduce(n, Sum());
    if (tid == 0) sh.turn_u[turn & 1] = n;
    cluster_barrier();
    return over(&sh.turn_u[turn++ & 1], Sum());
  };
  auto mass_from = [&](uint32_t t) {
    double s = 0;
    const float least = value_of(max(max(t, tau + 1), low_key));
    each8(least, [&](const float (&v)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double e = weight(v[i]);
        if (v[i] >= least) s += e;
      }
    });
    s = block_reduce(s, Sum());
    if (tid == 0) sh.turn_d[turn & 1] = s;
    cluster_barrier();
    s = over(&sh.turn_d[turn++ & 1], Sum());
    return tau && t <= tau ? s + ties * safe_weight(tau) : s;
  };
  auto slow_mass = [&](float share) {  // tau and ties of the fewest first kept tokens that hold `share` of their mass
    const double goal = (double)share * mass_from(0);
    uint32_t t = 0;
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
      if ((t | bit) <= top && mass_from(t | bit) >= goal) t |= bit;
    const double above = mass_from(t + 1), w = safe_weight(t);
    uint32_t n = count_from(t) - count_from(t + 1);
    if (t == tau) n = ties;
    const double need = w > 0 ? ceil((goal - above) / w) : 1.0;
    tau = t;
    ties = need >= (double)n ? n : need < 1.0 ? 1u : (uint32_t)need;
  };
  auto lowest = [&]() -> float {           // the smallest logit above -inf
    if (least_key == kNone) {
      float mn = INFINITY;
      each8(-FLT_MAX, [&](const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (v[i] > -INFINITY) mn = fminf(mn, v[i]);
      });
      const uint32_t key = block_reduce(key_of(mn), Min());
      if (tid == 0) sh.finite = key;
      cluster_barrier();
      least_key = over(&sh.finite, Min());
    }
    return value_of(least_key);
  };

  // ---- histogram over evenly spaced values below the maximum ------------------------------------
  float per_unit = 0.f;                    // bins per unit of the logit
  // the distance below the maximum in bins, the last for all further down; rounded to a bin in the low bits of
  // `place`, and never falls as v falls
  auto depth = [&](float v) { return fminf((m - v) * per_unit, (float)(kBins - 1)); };
  auto place = [&](float d) { return d + 8388608.f; };  // 2^23
  auto bin_at = [&](float t) { return __float_as_uint(t) & (uint32_t)(kBins - 1); };
  // the cluster's histogram, two bins a thread: 4 bins of every other block a thread, then both halves (as floats: whole
  // numbers up to 2^24 are exact, larger ones are weights)
  static_assert(kThreads == 512 && kBins == 1024, "");
  auto gather = [&](float (&sum)[kPerThread]) {
    const int g = tid & 255, half = tid >> 8;
    uint4 e[kMaxCluster / 2];
#pragma unroll
    for (int c = 0; c < kMaxCluster / 2; ++c)
      if (2 * c + half < C) e[c] = peer4(&hist[4 * g], 2 * c + half);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kMaxCluster / 2; ++c)
      if (2 * c + half < C) s.x += (float)e[c].x, s.y += (float)e[c].y, s.z += (float)e[c].z, s.w += (float)e[c].w;
    *reinterpret_cast<float4*>(&gathered[half][4 * g]) = s;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) sum[i] = gathered[0][tid * kPerThread + i] + gathered[1][tid * kPerThread + i];
  };
  auto spread = [&](float span) {
    per_unit = span > 0.f ? (float)(kBins - 3) / span : 0.f;
    if (!(per_unit < INFINITY)) per_unit = 0.f;  // too small a span to divide by
  };
  // The list of the tokens from `low` to `high` (those kept so far), as keys,
  // over all blocks: registers, 4 a thread.  `also` sees every 8 tokens on the
  // way, but for those of blocks that do not reach `least`.
  uint32_t mine[kList / kThreads], list_lo = 0, list_hi = 0, listed_n = 0;
  int lists = 0;                           // lists made so far: each has variables of its own
  auto collect = [&](float least, float low, float high, auto&& also, auto&& done) -> uint32_t {
    const int z = lists++;
    uint32_t lo_k = 0xffffffffu, hi_k = 0;
    for (int i = tid; i < 4 * 3 * 256; i += kThreads) digits[0][0][i] = 0;
    low = fmaxf(low, tau ? value_of(tau) : -FLT_MAX);
    each8(least, [&](const float (&v)[8]) {
      also(v);
      uint32_t n = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) n += v[i] >= low && v[i] <= high;
      if (n == 0) return;
      uint32_t at = atomicAdd(&sh.listed[z], n);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v[i] >= low && v[i] <= high) {
          const uint32_t key = key_of(v[i]);
          if (at < kList) list[at] = key;
          ++at;
          lo_k = min(lo_k, key);
          hi_k = max(hi_k, key);
        }
    });
    lo_k = __reduce_min_sync(0xffffffffu, lo_k);
    hi_k = __reduce_max_sync(0xffffffffu, hi_k);
    if (lane == 0 && hi_k) {
      atomicMin(&sh.list_lo[z], lo_k);
      atomicMax(&sh.list_hi[z], hi_k);
    }
    done();
    cluster_barrier();
    if (warp == 0) {  // of each CTA, all in one round: tokens listed, the smallest and the largest, tokens above
      const int c = lane & 7, what = lane >> 3;
      const uint32_t* from = what == 0 ? &sh.listed[z] : what == 1 ? &sh.list_lo[z] : what == 2 ? &sh.list_hi[z] : &sh.list_above;
      const uint32_t got = c < C ? peer(from, c) : what == 1 ? 0xffffffffu : 0;
      const uint32_t end = warp_prefix(got, 8);  // over the 8 lanes of each kind
      uint32_t lo = got, hi = got;
#pragma unroll
      for (int o = 4; o; o >>= 1) {
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      if (what == 0) sh.list_end[c] = end;
      if (lane == 8) sh.span_lo = lo;
      if (lane == 16) sh.span_hi = hi;
      if (lane == 31) sh.all_above = end;
    }
    __syncthreads();
    list_lo = sh.span_lo;
    list_hi = sh.span_hi;
    const uint32_t n = sh.list_end[kMaxCluster - 1];
    if (n > kList) return n;
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i) {
      const uint32_t at = tid + i * kThreads;
      mine[i] = 0;
      if (at < n) {
        int c = 0;
        uint32_t first = 0;
        for (uint32_t end; at >= (end = sh.list_end[c]); ++c) first = end;
        mine[i] = peer(&list[at - first], c);
      }
    }
    listed_n = n;
    if (n <= kRanked) {
      if (tid < kRanked) ranked[tid] = mine[0];
      __syncthreads();
    }
    return n;
  };
  // The largest listed key t whose weight together with that of all larger ones
  // is `goal` or more, 8 bits a turn; `extra` counts as one more of key tau.
  // Gives the weight above t and that of t and its equals; false: all of them
  // weigh less than the goal.
  auto search = [&](const uint64_t (&w)[kList / kThreads], uint64_t extra, uint64_t goal, uint32_t& t, uint64_t& above,
                    uint64_t& equal) {
    if (listed_n <= kRanked) {  // each thread looks at all of them for its own
      if (tid < kRanked) ranked_w[tid] = w[0];
      if (tid == 0) sh.found = 0;
      __syncthreads();
      if (mine[0]) {
        uint64_t more = mine[0] < tau ? extra : 0, same = mine[0] == tau ? extra : 0;
#pragma unroll 4
        for (uint32_t j = 0; j < listed_n; j += 2) {  // behind the list: key 0, weight 0
          const uint2 key = *reinterpret_cast<const uint2*>(&ranked[j]);
          const ulonglong2 e = *reinterpret_cast<const ulonglong2*>(&ranked_w[j]);
          if (key.x > mine[0]) more += e.x;
          if (key.y > mine[0]) more += e.y;
          if (key.x == mine[0]) same += e.x;
          if (key.y == mine[0]) same += e.y;
        }
        if (more < goal && more + same >= goal) {  // its equals find the same
          sh.found = 1;
          sh.pick_key = mine[0];
          sh.pick_above = more;
          sh.pick_equal = same;
        }
      }
      __syncthreads();
      t = sh.pick_key;
      above = sh.pick_above;
      equal = sh.pick_equal;
      return sh.found != 0;
    }
    const uint32_t differ = list_lo ^ list_hi;
    int bits = differ ? 32 - __clz(differ) : 1;  // the bits above are common to all
    // 16-bit logits: the low bits follow from the upper ones (all 0, or all 1 below zero)
    constexpr int kEnd = std::is_same<T, float>::value ? 0 : std::is_same<T, __half>::value ? 13 : 16;
    bits = max(bits, kEnd + 1);
    t = list_hi;
    above = equal = 0;
    for (int turn = 0; bits > kEnd; ++turn) {
      const int d = min(bits - kEnd, 8), shift = bits - d;
      auto add = [&](uint32_t key, uint64_t e) {
        if (e && (bits == 32 || key >> bits == t >> bits)) {
          const uint32_t digit = key >> shift & 255u >> (8 - d), low = (uint32_t)e & 0x1fffff, mid = (uint32_t)(e >> 21) & 0x1fffff;
          if (low) atomicAdd(&digits[turn][0][digit], low);
          if (mid) atomicAdd(&digits[turn][1][digit], mid);
          if (e >> 42) atomicAdd(&digits[turn][2][digit], (uint32_t)(e >> 42));
        }
      };
#pragma unroll
      for (int j = 0; j < kList / kThreads; ++j)
        if (mine[j]) add(mine[j], w[j]);
      if (tid == 0) add(tau, extra);
      __syncthreads();
      // every warp finds the digit for itself: lane l holds digits 255 - 8 l and the 7 below
      uint64_t e[8], s = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int digit = 255 - 8 * lane - j;
        e[j] = digits[turn][0][digit] + ((uint64_t)digits[turn][1][digit] << 21) + ((uint64_t)digits[turn][2][digit] << 42);
        s += e[j];
      }
      uint64_t reached = above + warp_prefix(s, 32);
      const uint32_t hit = __ballot_sync(0xffffffffu, reached >= goal);
      if (!hit) return false;
      const int who = __ffs(hit) - 1;
      reached -= s;
      uint32_t digit = 0;
      uint64_t here = 0;
      bool done = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!done) {
          if (reached + e[j] >= goal) done = true, digit = 255 - 8 * lane - j, here = e[j];
          else reached += e[j];
        }
      }
      digit = __shfl_sync(0xffffffffu, digit, who);
      above = __shfl_sync(0xffffffffu, reached, who);
      equal = __shfl_sync(0xffffffffu, here, who);
      t = (bits == 32 ? 0u : t >> bits << bits) | digit << shift;
      bits = shift;
    }
    if (kEnd && !(t & 0x80000000u)) t |= (1u << kEnd) - 1;
    return true;
  };

  bool have_all = false;                   // the list holds every kept token
  const int n_all = ceil_div(V, kBlock);
  if (k > 0 && 2 * k <= min(kThreads, n_all)) {
    // few: a value that k of the row's groups of tokens reach, by the upper 20 bits of its key; all tokens from there on
    // are little more than k
    uint32_t best_of = 0, t = 0;
    for (int i = tid; i < n_all; i += kThreads) best_of = max(best_of, key_of(finite(peer(&blk_top[i % p.per_cta], i / p.per_cta))));
    for (uint32_t bit = 0x80000000u; bit > 0x800u; bit >>= 1)
      if (__syncthreads_count(best_of >= (t | bit)) >= k) t |= bit;
    const float low = value_of(max(t, kNone + 1));
    const uint32_t listed = collect(low, low, INFINITY, [](const float (&)[8]) {}, [] {});
    if (listed >= (uint32_t)k && listed <= kList) {
      uint64_t one[kList / kThreads], above, equal;
#pragma unroll
      for (int j = 0; j < kList / kThreads; ++j) one[j] = mine[j] != 0;
      search(one, 0, (uint32_t)k, tau, above, equal);
      ties = (uint32_t)k - (uint32_t)above;
      have_all = true;
    }
  }
  if (k > 0 && k < V && !have_all) {
    // a value that k tokens reach: that many lanes' largest, of the warps whose lanes do best
    const int warps = C * kWarps, need = ceil_div(k, 32);
    float low = -INFINITY;
    if (need <= warps) {
      // the need-th largest of the warps' smallest lane maxima (equal ones by place)
      uint32_t pick = 0;
      if (tid < warps) {
        const uint32_t v = sh.all_min[tid];
        int before = 0;
#pragma unroll 8
        for (int j = 0; j < warps; j += 4) {
          const uint4 o = *reinterpret_cast<const uint4*>(&sh.all_min[j]);
          before += (o.x > v || (o.x == v && j < tid)) + (o.y > v || (o.y == v && j + 1 < tid)) +
                    (o.z > v || (o.z == v && j + 2 < tid)) + (o.w > v || (o.w == v && j + 3 < tid));
        }
        if (before == need - 1) pick = v;
      }
      pick = block_reduce(pick, Max());
      low = infinite ? finite(value_of(max(pick, kNone))) : value_of(max(pick, kNone));
    }
    if (low == -INFINITY) low = lowest();
    spread(m - low);
    if (tid == 0) sh.last = -1;
    each8(low, [&](const float (&v)[8]) {  // the last bin holds all that is further down: not counted
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = depth(v[i]);
        if (d < (float)(kBins - 2)) atomicAdd(&hist[bin_at(place(d))], 1u);
      }
    });
    cluster_barrier();
    // the bin of the k-th largest, summed over the blocks
    float sums[kPerThread];
    gather(sums);
    uint32_t count[kPerThread], n = 0;  // 2^22 tokens at most: exact
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      count[i] = (uint32_t)sums[i];
      n += count[i];
    }
    uint32_t before = block_prefix(n) - n;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      if (before < (uint32_t)k && before + count[i] >= (uint32_t)k) {
        sh.last = tid * kPerThread + i;
        sh.carry_ties = before + count[i];
      }
      before += count[i];
    }
    __syncthreads();
    const int bin = sh.last;
    bool slow = true;
    if (bin >= 0) {
      // a little beyond the bin, as its ends are rounded; the counts are checked
      const float unit = per_unit > 0.f ? 1.f / per_unit : 0.f;
      const float list_low = m - ((float)bin + 0.75f) * unit, list_high = m - ((float)bin - 0.75f) * unit;
      have_all = sh.carry_ties <= kList * 3 / 4;
      uint32_t above_n = 0;
      const float high = have_all ? INFINITY : list_high;
      const uint32_t listed = collect(
          list_low, list_low, high,
          [&](const float (&v)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) above_n += v[i] > high;
          },
          [&] {
            above_n = block_reduce(above_n, Sum());
            if (tid == 0) sh.list_above = above_n;
          });
      above_n = sh.all_above;
      const uint32_t rest = (uint32_t)k - above_n;
      if (above_n < (uint32_t)k && rest <= listed) {
        if (listed <= kList) {
          uint64_t one[kList / kThreads], above, equal;
#pragma unroll
          for (int j = 0; j < kList / kThreads; ++j) one[j] = mine[j] != 0;
          search(one, 0, rest, tau, above, equal);
          ties = rest - (uint32_t)above;
          slow = false;
        } else if (list_lo == list_hi) {
          tau = list_lo;
          ties = rest;
          slow = false;
        }
      }
      if (slow) have_all = false;
    }
    if (slow && count_from(kNone + 1) > (uint32_t)k) {  // else nothing to cut
      uint32_t t = 0;
      for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
        if (count_from(t | bit) >= (uint32_t)k) t |= bit;
      ties = (uint32_t)k - count_from(t + 1);
      tau = t;
    }
  }
  if (share < 1.f) {
    uint64_t w[kList / kThreads];
    const uint64_t w_tau = tau ? whole_weight(tau) : 0;
    auto listed_weights = [&] {            // of the kept ones above tau
#pragma unroll
      for (int j = 0; j < kList / kThreads; ++j) w[j] = mine[j] > tau ? whole_weight(mine[j]) : 0;
    };
    auto cut = [&](uint64_t extra, uint64_t goal) {  // false: the listed ones do not reach the goal
      uint64_t above, equal;
      uint32_t t;
      if (!search(w, extra, goal, t, above, equal)) return false;
      const uint64_t one = whole_weight(t), need = (goal - above + one - 1) / one, have = equal / one;
      tau = t;
      ties = (uint32_t)min(need, have);
      return true;
    };
    if (have_all) {
      listed_weights();
      uint64_t s = 0;
#pragma unroll
      for (int j = 0; j < kList / kThreads; ++j) s += w[j];
      const uint64_t extra = ties * w_tau;
      s = block_reduce(s, Sum()) + extra;
      for (int i = tid; i < 4 * 3 * 256; i += kThreads) digits[0][0][i] = 0;
      __syncthreads();
      cut(extra, max(1ll, __double2ll_ru((double)share * (double)s)));
    } else {
      if (k > 0 && k < V) {
        cluster_barrier();  // the counts have been read
        for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
        cluster_barrier();
      }
      // a histogram of weights, each a whole number of 2^-14 of its bin's middle, 2^-12 where a block has more than 2^17
      // tokens (2^19 at most): all of them in one bin, each up to e^(1/60) units, stay below 2^32
      const float units = p.per_cta * kBlock > 1 << 17 ? 4096.f : 16384.f;
      // as deep as what is further down, all V tokens of it, weighs a thousandth of what the cut leaves out
      spread(fminf(m - lowest(), temp * (logf((float)V / fmaxf(1.f - share, 1e-7f)) + 7.f)));
      const float fall = per_unit > 0.f ? 1.f / (per_unit * temp) : 0.f;  // of the weight's logarithm over a bin
      if (tid == 0) sh.last = -1;
      const float kept_from = value_of(max(low_key, tau + 1));
      each8(kept_from, [&](const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float d = depth(v[i]), t = place(d), off = (t - 8388608.f - d) * fall;
          // e^off, |off| < 1/60 or so
          const float part = fmaf(fmaf(off, 0.5f, 1.f), off, 1.f) * units + 8388608.f;
          if (d < (float)(kBins - 2) && v[i] >= kept_from) atomicAdd(&hist[bin_at(t)], __float_as_uint(part) & 0x7fffffu);
        }
      });
      cluster_barrier();
      const float fall2 = fall * 1.44269504f;
      float mass[kPerThread], s = 0.f;
      gather(mass);
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        mass[i] *= exp2f(-(float)(tid * kPerThread + i) * fall2);
        s += mass[i];
      }
      float reached = block_prefix(s) - s;
      const float all = block_reduce(reached + s, Max()) + (tau ? (float)ties * (float)safe_weight(tau) * units : 0.f);
      int short_of = -1;  // the last bin that does not reach the cut
#pragma unroll
      for (int i = 0; i < kPerThread; ++i)
        if ((reached += mass[i]) < share * all) short_of = tid * kPerThread + i;
      short_of = __reduce_max_sync(0xffffffffu, short_of);
      if (lane == 0 && short_of >= 0) atomicMax(&sh.last, short_of);
      __syncthreads();
      int bin = min(sh.last + 1, kBins - 1);
      const float v_tau = tau ? value_of(tau) : -INFINITY;
      if (tau) bin = min(bin, (int)bin_at(place(depth(v_tau))));  // nothing is kept below
      const float unit = per_unit > 0.f ? 1.f / per_unit : 0.f;
      bool found = false;
      // The histogram's sums are off by 10^-7 of the whole and more: a cut at the very end of a bin, as one of some
      // thousand 16-bit rows has it, may be in the next one that holds tokens, which the exact sums tell (one such row
      // among 128, searched bit by bit instead, made 434 us of 120)
#pragma unroll 1
      for (int attempt = 0; bin >= 0 && bin < kBins; ++attempt) {
        // the bracket: that bin and a little beyond.  Exactly: the mass above it and that of all kept tokens
        const float low = m - ((float)bin + 0.65f) * unit, high = m - ((float)bin - 0.65f) * unit;
        double above = 0, rest = 0, above2 = 0, rest2 = 0;
        const uint32_t n = collect(
            kept_from, low, high,
            [&](const float (&v)[8]) {
              double e[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) e[i] = weight(v[i]);
#pragma unroll
              for (int i = 0; i < 8; i += 2) {
                if (v[i] > high) above += e[i];
                if (v[i + 1] > high) above2 += e[i + 1];
                if (v[i] <= high && v[i] >= kept_from) rest += e[i];
                if (v[i + 1] <= high && v[i + 1] >= kept_from) rest2 += e[i + 1];
              }
            },
            [&] {
              above = block_reduce(above + above2, Sum());
              rest = block_reduce(rest + rest2, Sum());
              if (tid == 0) {
                sh.mass[0] = above;
                sh.mass[1] = rest;
              }
            });
        above = over(&sh.mass[0], Sum());
        rest = over(&sh.mass[1], Sum());
        const double goal = (double)share * (above + rest + (tau ? ties * safe_weight(tau) : 0.0)) - above;
        const bool ends_here = tau && v_tau >= low && v_tau <= high;
        if (goal > 0 && goal < 1024.0 && n > 0 && n <= kList && v_tau <= high) {  // 2^10 * 2^52 and the list's 2^63 fit 64 bits
          listed_weights();
          found = cut(ends_here ? ties * w_tau : 0, (uint64_t)max(1ll, __double2ll_ru(goal * kUnit)));
        } else if (goal > 0 && n > kList && list_lo == list_hi && list_lo > tau && list_lo >= low_key) {  // equals only
          const double need = ceil(goal / weight(value_of(list_lo)));
          if (need <= (double)n) {
            tau = list_lo;
            ties = (uint32_t)need;
            found = true;
          }
        }
        if (found || attempt > 0 || (goal > 0 && n > kList)) break;
        cluster_barrier();  // what the others read of this block is written anew
        if (tid == 0) sh.last = goal > 0 ? kBins : -1;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
          const int at = tid * kPerThread + i;
          if (!(gathered[0][at] + gathered[1][at] > 0.f)) continue;
          if (goal > 0 && at > bin) atomicMin(&sh.last, at);
          if (!(goal > 0) && at < bin) atomicMax(&sh.last, at);
        }
        __syncthreads();
        bin = sh.last;
      }
      if (!found) slow_mass(share);
    }
  }

  // ---- the draw, in the vocabulary's order --------------------------------------------------------
  // kept tokens reach `from`: the smallest key whose weight is min_p or more (the largest always stays)
  uint32_t from_key = low_key;
  if (min_p >= 1.f) from_key = top;
  if (min_p > 0.f && min_p < 1.f) {
    from_key = key_of((float)((double)m + log((double)min_p) * (double)temp));
    from_key = min(max(from_key, low_key), top);
    // mostly that key; beside a border near 0, where keys lie close, it may be many millions away: steps that double, and
    // halves of what they leave
    auto heavy = [&](uint32_t key) { return weight(value_of(key)) >= (double)min_p; };
    uint32_t light = from_key, step = 1;  // in the end the key below
    if (heavy(from_key)) {
      for (; from_key > low_key; step *= 2) {
        light = from_key - min(step, from_key - low_key);
        if (!heavy(light)) break;
        from_key = light;
      }
    } else {  // the largest weighs 1
      for (;; step *= 2) {
        from_key = light + min(step, top - light);
        if (heavy(from_key)) break;
        light = from_key;
      }
    }
    while (from_key - light > 1) {
      const uint32_t mid = light + (from_key - light) / 2;
      if (heavy(mid)) from_key = mid;
      else light = mid;
    }
  }
  const double w_tau = tau >= from_key ? weight(value_of(tau)) : 0.0;
  const float from = value_of(max(from_key, tau + 1)), v_tau = value_of(max(tau, kNone));
  double kept = 0;
  uint32_t equal = 0;
  for (int blk = warp; blk < n_blk; blk += kWarps) {
    double s = 0;
    uint32_t n = 0;
    const float most = finite(blk_top[blk]);
    if (most >= from || (tau && most >= v_tau)) {
      float v[8];
      load(blk, v);
      double s2[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double e = weight(v[i]);
        if (v[i] >= from) s2[i & 1] += e;
      }
      s = s2[0] + s2[1];
      if (tau) {
#pragma unroll
        for (int i = 0; i < 8; ++i) n += v[i] == v_tau;
        n = __reduce_add_sync(0xffffffffu, n);
      }
      s = warp_reduce(s, Sum());
    }
    if (lane == 0) {
      blk_mass[blk] = s;
      blk_ties[blk] = n;
      kept += s;
      equal += n;
    }
  }
  kept = block_reduce(kept, Sum());
  equal = block_reduce(equal, Sum());
  if (tid == 0) {
    sh.kept = kept;
    sh.ties = equal;
    sh.found = 0x7fffffff;
    sh.last = -1;
  }
  cluster_barrier();
  // the CTA that holds the draw: the first whose cumulative mass exceeds it, else the last with any
  double masses[kMaxCluster], total = 0;
  uint32_t equals[kMaxCluster], ties_before = 0;
#pragma unroll
  for (int c = 0; c < kMaxCluster; ++c) {
    masses[c] = c < C ? peer(&sh.kept, c) : 0.0;
    equals[c] = c < C ? peer(&sh.ties, c) : 0;
  }
#pragma unroll
  for (int c = 0; c < kMaxCluster; ++c) {
    masses[c] += (double)min(equals[c], ties > ties_before ? ties - ties_before : 0) * w_tau;
    total += masses[c];
    ties_before += equals[c];
  }
  const double goal = (double)uniform * total;
  double sum = 0, own_before = 0;
  int owner = -1, last_owner = -1;
  uint32_t own_ties = 0;
  ties_before = 0;
#pragma unroll
  for (int c = 0; c < kMaxCluster; ++c) {
    if (c == me) own_before = sum, own_ties = ties_before;
    sum += masses[c];
    ties_before += equals[c];
    if (masses[c] > 0) last_owner = c;
    if (owner < 0 && sum > goal) owner = c;
  }
  if (owner < 0) owner = last_owner;
  cluster_arrive();  // done with the others' variables
  if (owner == me) {
    // its 256 tokens, likewise
    double before = own_before;
    uint32_t t_before = own_ties;
    for (int base = 0; base < n_blk; base += kThreads) {
      const int i = base + tid;
      const uint32_t t = i < n_blk ? blk_ties[i] : 0;
      const uint32_t t_inc = block_prefix(t), t0 = t_before + t_inc - t;
      const uint32_t left = ties > t0 ? ties - t0 : 0;
      const double mass = i < n_blk ? blk_mass[i] + (double)min(t, left) * w_tau : 0.0;
      const double inc = before + block_prefix(mass);
      if (mass > 0) {
        atomicMax(&sh.last, i);
        if (inc > goal) atomicMin(&sh.found, i);
      }
      __syncthreads();
      const bool here = sh.found != 0x7fffffff;
      const int pick = here ? sh.found : sh.last;
      if (i == pick) {
        sh.found_before = inc - mass;
        sh.found_ties = t0;
      }
      if (tid == kThreads - 1) {  // the sums so far
        sh.carry_mass = inc;
        sh.carry_ties = t_before + t_inc;
      }
      __syncthreads();
      if (here) break;
      before = sh.carry_mass;
      t_before = sh.carry_ties;
      __syncthreads();
    }
    if (warp == 0) {
      const int blk = sh.found != 0x7fffffff ? sh.found : sh.last;
      float v[8];
      double e[8], s = 0;
      uint32_t n = 0;
      load(blk, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) n += tau && v[i] == v_tau;
      uint32_t at = sh.found_ties + warp_prefix(n, 32) - n;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = v[i] >= from ? weight(v[i]) : 0.0;
        if (tau && v[i] == v_tau && at++ < ties) e[i] = w_tau;
        s += e[i];
      }
      const double inc = sh.found_before + warp_prefix(s, 32);
      const uint32_t any = __ballot_sync(0xffffffffu, s > 0), hit = __ballot_sync(0xffffffffu, s > 0 && inc > goal);
      const int who = hit ? __ffs(hit) - 1 : 31 - __clz(any);
      if (lane == who) {
        double c = inc - s;
        int chosen = -1;
        bool done = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (done || !(e[i] > 0)) continue;
          c += e[i];
          chosen = i;
          done = c > goal;
        }
        p.out[b] = (int64_t)(blk0 + blk) * kBlock + lane * 8 + chosen;
      }
    }
  }
  cluster_wait();  // no block leaves while others read its variables
}

template <typename T>
int launch(SampleParams p, int batch, cudaStream_t stream) {
  static std::atomic<uint32_t> done{0};
  constexpr int kMost = 160 * 1024;  // bytes of a row's share in shared memory, beside 36 KB of histogram and list
  const int blocks = ceil_div(p.V, kBlock);
  // a cluster at least as large as holds the row, and as large as keeps every
  // warp busy with all rows resident (a block an SM, of 124 registers a thread:
  // 33 rows on clusters of 8, two rounds, took twice as long as on 4)
  int c = 1;
  auto bytes = [&](int n) {
    const size_t per = ceil_div(blocks, n);
    return per * 16 + per * kBlock * sizeof(T);
  };
  while (c < kMaxCluster && (bytes(c) > (size_t)kMost || (c * kWarps <= blocks && (int64_t)batch * c * 2 <= 148))) c *= 2;
  p.per_cta = ceil_div(blocks, c);
  p.staged = bytes(c) <= (size_t)kMost;
  const size_t smem = p.staged ? bytes(c) : (size_t)p.per_cta * 16;
  max_smem_once(done, sample_kernel<T>, kMost);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)batch * c);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = c;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, p);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return SKV_ERR_CUDA;
  }
  return SKV_OK;
}

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" int skv_sample(const skv_sample_args* a, void* stream) {
  if (!a || a->batch <= 0 || a->vocabulary <= 0 || !a->logits || !a->uniform || !a->tokens) return SKV_ERR_INVALID_ARG;
  if (a->row_stride < 0) return SKV_ERR_INVALID_ARG;
  const int es = a->dtype == SKV_F32 ? 4 : (a->dtype == SKV_F16 || a->dtype == SKV_BF16) ? 2 : 0;
  if (!es) return SKV_ERR_UNSUPPORTED;
  if (a->vocabulary > SKV_SAMPLE_MAX_VOCABULARY || a->batch > (1 << 24)) return SKV_ERR_UNSUPPORTED;
  if ((uintptr_t)a->logits % es || (uintptr_t)a->uniform % 4 || (uintptr_t)a->tokens % 8 ||
      (uintptr_t)a->temperatures % 4 || (uintptr_t)a->top_ks % 4 || (uintptr_t)a->top_ps % 4 ||
      (uintptr_t)a->min_ps % 4)
    return SKV_ERR_MISALIGNED;
  SampleParams p{a->logits, a->row_stride, a->uniform, a->temperatures, a->top_ks, a->top_ps, a->min_ps,
                 a->tokens, a->temperature, a->top_p, a->min_p, a->top_k, a->vocabulary, 0, 0};
  const cudaStream_t s = (cudaStream_t)stream;
  if (a->dtype == SKV_F32) return launch<float>(p, a->batch, s);
  if (a->dtype == SKV_F16) return launch<__half>(p, a->batch, s);
  return launch<__nv_bfloat16>(p, a->batch, s);
}
