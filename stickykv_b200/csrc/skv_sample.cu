// skv_sample: the next token of each row from its logits and a given random
// number (temperature, top-k, top-p, min-p).
//
// In descending order with ties by index every cut is a threshold: the key of
// the last kept token and how many of its equals, lowest indices first, stay.
// No sort: a cluster holds a row in its blocks' shared memory and finds the
// threshold with one histogram over evenly spaced values (below the maximum),
// which names the bin that holds it, and a search among that bin's few tokens.
// Rows whose bin holds too many (masses of equal logits) are searched bit by
// bit over the whole row.
//
// Weights and sums are 64-bit: a draw falls between two neighbours of 10^5
// cumulative sums, and 32-bit sums would move a share of draws to a neighbour.
// Sums are taken in a fixed order, or as whole numbers where the order is not
// fixed, so equal calls give equal tokens.
//
// Bound: one row is latency (a handful of cluster barriers), many rows the
// 64-bit exponentials of a top-p cut (about 16 operations a token at 64 a clock
// and SM); HBM is read once.
#include "skv_common.cuh"

namespace skv {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBlock = 256;        // tokens a warp takes at once: 8 neighbours a lane
constexpr int kBins = 2048;
constexpr int kList = 2048;        // tokens that are searched in registers, 4 a thread
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

// Total order of the values as unsigned integers (NaN and -0 are gone by then).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.f; }

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

// What the blocks of a cluster tell one another.
struct Shared {
  uint32_t top[1], at[1], least[1];       // largest key, its first index, smallest key above -inf
  uint32_t warp_min[kWarps];              // of each warp, the smallest of its lanes' largest keys
  uint32_t listed[2];
  uint32_t list_lo[2], list_hi[2];        // smallest and largest listed key
  double mass[2];                         // above the bracket; of all
  double turn_d[2];                       // bit by bit search, in turns
  uint32_t turn_u[2];
  double kept;                            // mass above the threshold, of the block's tokens
  uint32_t ties;                          // equals of the threshold
  // within the block
  uint64_t red[kWarps];
  uint32_t red_u[kWarps];
  double red_d[kWarps];
  int found, last;
  double found_before;
  uint32_t found_ties;
};

struct Weight {  // w(x) = 2^((x - m) / T * log2 e) in 64 bits
  double m, c;
  __device__ __forceinline__ double operator()(float x) const {
    const double y = ((double)x - m) * c;
    if (x == (float)m) return 1.0;      // also where both are infinite
    if (!(y > -1000.0)) return x > -INFINITY ? exp2(y) : 0.0;  // near or below the smallest numbers
    const double t = y + 6755399441055744.0;  // 1.5 * 2^52: rounds to whole numbers
    const double f = (y - (t - 6755399441055744.0)) * 0.69314718055994530942;
    // e^f, |f| < 0.35, by its series: the first term left out is below 7e-15
    double e = 1.0 / 39916800.0;
    e = fma(e, f, 1.0 / 3628800.0);
    e = fma(e, f, 1.0 / 362880.0);
    e = fma(e, f, 1.0 / 40320.0);
    e = fma(e, f, 1.0 / 5040.0);
    e = fma(e, f, 1.0 / 720.0);
    e = fma(e, f, 1.0 / 120.0);
    e = fma(e, f, 1.0 / 24.0);
    e = fma(e, f, 1.0 / 6.0);
    e = fma(e, f, 0.5);
    e = fma(e, f, 1.0);
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
template <typename A, typename Op>
__device__ __forceinline__ A block_reduce(A v, Op op, A* buf) {
  v = warp_reduce(v, op);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = buf[threadIdx.x & (kWarps - 1)];
#pragma unroll
  for (int o = kWarps / 2; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// inclusive prefix over the block's threads
template <typename A>
__device__ __forceinline__ A block_prefix(A v, A* buf) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const A n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  __syncthreads();
  if (lane == 31) buf[warp] = v;
  __syncthreads();
  A base = 0;
  for (int w = 0; w < warp; ++w) base += buf[w];
  return base + v;
}

struct Max { template <typename A> __device__ A operator()(A a, A b) const { return a > b ? a : b; } };
struct Min { template <typename A> __device__ A operator()(A a, A b) const { return a < b ? a : b; } };
struct Sum { template <typename A> __device__ A operator()(A a, A b) const { return a + b; } };

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Shared sh;
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t list[kList];
  double* blk_mass = reinterpret_cast<double*>(smem);                       // [per_cta]
  uint32_t* blk_ties = reinterpret_cast<uint32_t*>(blk_mass + p.per_cta);   // [per_cta]
  T* data = reinterpret_cast<T*>(smem + align_up((size_t)p.per_cta * 12, 16));

  uint32_t rank, size;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(size));
  const int C = (int)size, me = (int)rank;
  const int b = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = p.V;
  const T* x = (const T*)p.logits + b * p.stride;
  const int blk0 = me * p.per_cta;                                // first block of this CTA
  const int n_blk = max(0, min(p.per_cta, ceil_div(V, kBlock) - blk0));
  auto cluster_barrier = [&] {
    if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    else __syncthreads();
  };
  auto over = [&](const auto* v, auto op) {  // a variable of all blocks of the cluster
    auto r = peer(v, 0);
    for (int c = 1; c < C; ++c) r = op(r, peer(v, c));
    return r;
  };

  // ---- a lane's 8 neighbours of block `blk` (of this CTA) --------------------------------
  const bool wide = ((uintptr_t)x & 15) == 0;
  auto fetch = [&](int blk, float (&v)[8]) {  // from global memory
    const int i0 = (blk0 + blk) * kBlock + lane * 8;
    if (wide && i0 + 8 <= V) {
      constexpr int N = 16 / sizeof(T);
#pragma unroll
      for (int h = 0; h < 8 / N; ++h) {
        const uint4 w = reinterpret_cast<const uint4*>(x + i0)[h];
        T e[N];
        *reinterpret_cast<uint4*>(e) = w;
#pragma unroll
        for (int i = 0; i < N; ++i) v[h * N + i] = clean(Elt<T>::to_f32(e[i]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i0 + i < V ? clean(Elt<T>::to_f32(x[i0 + i])) : -INFINITY;
    }
  };
  auto load = [&](int blk, float (&v)[8]) {
    if (!p.staged) return fetch(blk, v);
    const T* s = data + blk * kBlock + lane * 8;
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 8 / N; ++h) {
      T e[N];
      *reinterpret_cast<uint4*>(e) = reinterpret_cast<const uint4*>(s)[h];
#pragma unroll
      for (int i = 0; i < N; ++i) v[h * N + i] = Elt<T>::to_f32(e[i]);
    }
  };
  auto each = [&](auto&& f) {  // every token of this CTA's slice
    for (int blk = warp; blk < n_blk; blk += kWarps) {
      float v[8];
      load(blk, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) f(v[i]);
    }
  };

  // ---- the largest logit --------------------------------------------------------------------
  {
    float mx = -INFINITY, mn = INFINITY;
    int at = 0;
    for (int blk = warp; blk < n_blk; blk += kWarps) {
      float v[8];
      fetch(blk, v);
      if (p.staged) {
        T* s = data + blk * kBlock + lane * 8;
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int h = 0; h < 8 / N; ++h) {
          T e[N];
#pragma unroll
          for (int i = 0; i < N; ++i) e[i] = Elt<T>::from_f32(v[h * N + i]);
          reinterpret_cast<uint4*>(s)[h] = *reinterpret_cast<uint4*>(e);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (v[i] > mx) mx = v[i], at = (blk0 + blk) * kBlock + lane * 8 + i;
        if (v[i] > -INFINITY) mn = fminf(mn, v[i]);
      }
    }
    const uint32_t key = key_of(mx);
    const uint32_t lane_min = warp_reduce(key, Min());
    const uint32_t top = block_reduce(key, Max(), sh.red_u);
    const uint32_t first = block_reduce(key == top ? (uint32_t)at : 0xffffffffu, Min(), sh.red_u);
    const uint32_t least = block_reduce(key_of(mn), Min(), sh.red_u);
    if (lane == 0) sh.warp_min[warp] = lane_min;
    if (tid == 0) {
      sh.top[0] = top;
      sh.at[0] = first;
      sh.least[0] = least;
      sh.listed[0] = sh.listed[1] = 0;
      sh.list_lo[0] = sh.list_lo[1] = 0xffffffffu;
      sh.list_hi[0] = sh.list_hi[1] = 0;
      sh.found = 0x7fffffff;
      sh.last = -1;
    }
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
  }
  cluster_barrier();
  const uint32_t top = over(&sh.top[0], Max());
  const float temp = p.temps ? p.temps[b] : p.temp;
  if (top == kNone || !(temp > 0.f)) {  // nothing above -inf; greedy
    if (me == 0 && tid == 0) {
      uint32_t at = 0xffffffffu;
      for (int c = 0; c < C; ++c)
        if (peer(&sh.top[0], c) == top) at = min(at, peer(&sh.at[0], c));
      p.out[b] = top == kNone ? -1 : (int64_t)at;
    }
    cluster_barrier();  // no block leaves while others read its variables
    return;
  }
  const float m = value_of(top), least = value_of(over(&sh.least[0], Min()));
  const Weight weight{(double)m, 1.4426950408889634074 / (double)temp};
  auto whole_weight = [&](float v) { return (uint64_t)__double2ll_rn(weight(v) * kUnit); };

  // ---- search over the whole row, bit by bit (counts or masses of keys >= t, those kept) -------
  uint32_t tau = 0, ties = (uint32_t)V;  // kept: keys above tau and `ties` of its equals
  int turn = 0;
  auto count_from = [&](uint32_t t) {
    uint32_t n = 0;
    each([&](float v) { n += key_of(v) >= t; });
    n = block_reduce(n, Sum(), sh.red_u);
    if (tid == 0) sh.turn_u[turn & 1] = n;
    cluster_barrier();
    return over(&sh.turn_u[turn++ & 1], Sum());
  };
  auto mass_from = [&](uint32_t t) {
    double s = 0;
    each([&](float v) {
      const uint32_t k = key_of(v);
      if (k >= t && k > tau) s += weight(v);
    });
    s = block_reduce(s, Sum(), sh.red_d);
    if (tid == 0) sh.turn_d[turn & 1] = s;
    cluster_barrier();
    s = over(&sh.turn_d[turn++ & 1], Sum());
    return tau && t <= tau ? s + ties * weight(value_of(tau)) : s;
  };
  auto slow_mass = [&](float share) {  // tau and ties of the fewest first kept tokens that hold `share` of their mass
    const double goal = (double)share * mass_from(0);
    uint32_t t = 0;
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
      if ((t | bit) <= top && mass_from(t | bit) >= goal) t |= bit;
    const double above = mass_from(t + 1), w = weight(value_of(t));
    uint32_t n = count_from(t) - count_from(t + 1);
    if (t == tau) n = ties;
    const double need = w > 0 ? ceil((goal - above) / w) : 1.0;
    tau = t;
    ties = need >= (double)n ? n : need < 1.0 ? 1u : (uint32_t)need;
  };

  // ---- histogram over evenly spaced values below the maximum ------------------------------------
  float per_unit = 0.f;                    // bins per unit of the logit
  auto bin_of = [&](float v) {             // never falls as v falls
    const float d = (m - v) * per_unit;
    return d < (float)(kBins - 1) ? (int)d : kBins - 1;
  };
  // The list of the tokens in bins [lo, hi] (those kept so far), as keys, over all blocks: registers, 4 a thread.
  uint32_t mine[kList / kThreads];
  int lists = 0;                           // lists made so far: each has variables of its own
  auto collect = [&](int lo, int hi) -> uint32_t {
    const int z = lists;
    uint32_t lo_k = 0xffffffffu, hi_k = 0;
    for (int blk = warp; blk < n_blk; blk += kWarps) {
      float v[8];
      load(blk, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int bin = bin_of(v[i]);
        const uint32_t k = key_of(v[i]);
        if (bin >= lo && bin <= hi && k >= tau && k > kNone) {
          const uint32_t at = atomicAdd(&sh.listed[z], 1u);
          if (at < kList) list[at] = k;
          lo_k = min(lo_k, k);
          hi_k = max(hi_k, k);
        }
      }
    }
    lo_k = warp_reduce(lo_k, Min());
    hi_k = warp_reduce(hi_k, Max());
    if (lane == 0 && hi_k) {
      atomicMin(&sh.list_lo[z], lo_k);
      atomicMax(&sh.list_hi[z], hi_k);
    }
    cluster_barrier();
    const uint32_t n = over(&sh.listed[z], Sum());
    ++lists;
    if (n > kList) return n;
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i) {
      uint32_t at = tid + i * kThreads;
      mine[i] = 0;
      if (at < n) {
        int c = 0;
        for (uint32_t have; at >= (have = peer(&sh.listed[z], c)); ++c) at -= have;
        mine[i] = peer(&list[at], c);
      }
    }
    return n;
  };
  auto list_lo = [&] { return over(&sh.list_lo[lists - 1], Min()); };
  auto list_hi = [&] { return over(&sh.list_hi[lists - 1], Max()); };
  // The largest t with the listed weights of keys >= t at `goal` or more; `extra` counts for t <= tau.
  auto search = [&](const uint64_t (&w)[kList / kThreads], uint64_t extra, uint64_t goal, uint32_t lo, uint32_t hi) {
    // the bits that all listed keys share are known
    const uint32_t differ = lo ^ hi;
    const int bits = differ ? 32 - __clz(differ) : 0;
    uint32_t t = bits == 32 ? 0u : hi >> bits << bits;
    for (int i = bits - 1; i >= 0; --i) {
      const uint32_t c = t | 1u << i;
      uint64_t s = 0;
#pragma unroll
      for (int j = 0; j < kList / kThreads; ++j)
        if (mine[j] >= c) s += w[j];
      if (block_reduce(s, Sum(), sh.red) + (c <= tau ? extra : 0) >= goal) t = c;
    }
    // t's bits below may name a key that no token has: move up to the smallest listed key >= t
    uint32_t up = 0xffffffffu;
#pragma unroll
    for (int j = 0; j < kList / kThreads; ++j)
      if (mine[j] >= t) up = min(up, mine[j]);
    return block_reduce(up, Min(), sh.red_u);
  };
  // of the listed keys: (weights above t, equals of t)
  auto around = [&](const uint64_t (&w)[kList / kThreads], uint32_t t, uint64_t& above, uint32_t& equal) {
    uint64_t s = 0;
    uint32_t n = 0;
#pragma unroll
    for (int j = 0; j < kList / kThreads; ++j) {
      if (mine[j] > t) s += w[j];
      n += mine[j] == t;
    }
    above = block_reduce(s, Sum(), sh.red);
    equal = block_reduce(n, Sum(), sh.red_u);
  };

  const int k = p.ks ? p.ks[b] : p.k;
  const float share = p.ps ? p.ps[b] : p.p;
  bool have_all = false;                   // the list holds every kept token
  if (k > 0 && k < V) {
    // a value that k tokens reach: that many lanes' largest, of the warps whose lanes do best
    const int warps = C * kWarps, need = ceil_div(k, 32);
    float low = least;
    if (need <= warps) {
      // the need-th largest of the warps' smallest lane maxima (equal ones by place)
      uint32_t pick = 0;
      for (int i = tid; i < warps; i += kThreads) {
        const uint32_t v = peer(&sh.warp_min[i % kWarps], i / kWarps);
        int before = 0;
        for (int j = 0; j < warps; ++j) {
          const uint32_t o = peer(&sh.warp_min[j % kWarps], j / kWarps);
          before += o > v || (o == v && j < i);
        }
        if (before == need - 1) pick = v;
      }
      pick = block_reduce(pick, Max(), sh.red_u);
      if (pick > kNone) low = value_of(pick);
    }
    per_unit = m > low ? (float)(kBins - 2) / (m - low) : 0.f;
    if (!(per_unit < INFINITY)) per_unit = 0.f;   // a span too small or, with +inf, too large to divide
    each([&](float v) {
      if (v > -INFINITY) atomicAdd(&hist[bin_of(v)], 1u);
    });
    cluster_barrier();
    // the bin of the k-th largest: four bins a thread, summed over the blocks
    uint32_t n4[kBins / kThreads], n = 0;
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) {
      n4[i] = over(&hist[tid * (kBins / kThreads) + i], Sum());
      n += n4[i];
    }
    uint32_t before = block_prefix(n, sh.red_u) - n;
    if (tid == 0) sh.last = -1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) {
      if (before < (uint32_t)k && before + n4[i] >= (uint32_t)k) {
        sh.last = tid * (kBins / kThreads) + i;
        sh.found_ties = before;
      }
      before += n4[i];
    }
    __syncthreads();
    const int bin = sh.last;
    const uint32_t above = sh.found_ties;
    if (bin >= 0) {  // fewer than k tokens above -inf: nothing to cut
      uint32_t rest = (uint32_t)k;
      const uint32_t in_bin = over(&hist[bin], Sum());
      have_all = above + in_bin <= kList;
      if (!have_all) rest -= above;
      const uint32_t listed = collect(have_all ? 0 : bin, bin);
      if (listed <= kList) {
        uint64_t one[kList / kThreads];
#pragma unroll
        for (int j = 0; j < kList / kThreads; ++j) one[j] = mine[j] != 0;
        const uint32_t t = search(one, 0, rest, list_lo(), list_hi());
        uint64_t more;
        uint32_t equal;
        around(one, t, more, equal);
        tau = t;
        ties = rest - (uint32_t)more;
      } else if (list_lo() == list_hi()) {
        tau = list_lo();
        ties = rest;
      } else {
        uint32_t t = 0;
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
          if (count_from(t | bit) >= (uint32_t)k) t |= bit;
        ties = (uint32_t)k - count_from(t + 1);
        tau = t;
      }
    }
  }
  if (share < 1.f) {
    uint64_t w[kList / kThreads];
    auto listed_weights = [&] {  // of the kept ones above tau
#pragma unroll
      for (int j = 0; j < kList / kThreads; ++j) w[j] = mine[j] > tau ? whole_weight(value_of(mine[j])) : 0;
    };
    const uint64_t w_tau = tau ? whole_weight(value_of(tau)) : 0;
    auto cut = [&](uint64_t extra, uint64_t goal) {
      const uint32_t t = search(w, extra, goal, list_lo(), list_hi());
      uint64_t above;
      uint32_t equal;
      around(w, t, above, equal);
      const uint64_t wt = whole_weight(value_of(t));
      if (t == tau) equal = ties;
      const uint64_t need = wt && goal > above ? (goal - above + wt - 1) / wt : 1;
      tau = t;
      ties = need < equal ? (uint32_t)need : equal;
    };
    if (have_all) {
      listed_weights();
      uint64_t s = 0;
#pragma unroll
      for (int j = 0; j < kList / kThreads; ++j) s += w[j];
      const uint64_t extra = ties * w_tau;
      s = block_reduce(s, Sum(), sh.red) + extra;
      cut(extra, max(1ll, __double2ll_ru((double)share * (double)s)));
    } else {
      // the bracket from the histogram of weights, each as a share of its bin's largest: 2^-14 of it or less is lost
      if (k > 0 && k < V) {
        cluster_barrier();  // the counts have been read
        for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
        cluster_barrier();
      }
      const float span = fminf(m - least, 32.f * temp);  // e^-32 * 2^22 tokens weigh nothing against 2^-24
      per_unit = span > 0.f ? (float)(kBins - 2) / span : 0.f;
      if (!(per_unit < INFINITY)) per_unit = 0.f;
      const float fall = per_unit > 0.f ? 1.f / (per_unit * temp) : 0.f;  // of the weight's logarithm over a bin
      each([&](float v) {
        if (key_of(v) > max(tau, kNone)) {
          const float d = (m - v) * per_unit;
          const int bin = d < (float)(kBins - 1) ? (int)d : kBins - 1;
          const float part = bin < kBins - 1 ? expf(-(d - (float)bin) * fall) : 0.f;
          atomicAdd(&hist[bin], (uint32_t)(part * 16384.f + 0.5f));
        }
      });
      cluster_barrier();
      float s4[kBins / kThreads], s = 0.f;
#pragma unroll
      for (int i = 0; i < kBins / kThreads; ++i) {
        const int bin = tid * (kBins / kThreads) + i;
        float h = 0.f;
        for (int c = 0; c < C; ++c) h += (float)peer(&hist[bin], c);
        s4[i] = h * expf(-(float)bin * fall);
        s += s4[i];
      }
      float* red_f = reinterpret_cast<float*>(sh.red_u);
      float reached = block_prefix(s, red_f) - s;
      const float all = block_reduce(reached + s, Max(), red_f) + (tau ? (float)ties * (float)weight(value_of(tau)) * 16384.f : 0.f);
      if (tid == 0) sh.last = -1;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kBins / kThreads; ++i) {
        if (reached < share * all) atomicMax(&sh.last, tid * (kBins / kThreads) + i);
        reached += s4[i];
      }
      __syncthreads();
      const int bin = max(sh.last, 0), lo = max(0, bin - 1), hi = min(kBins - 1, bin + 1);
      // exactly: the mass above the bracket, of all kept tokens, and the bracket's tokens
      double above = 0, total = 0;
      each([&](float v) {
        if (key_of(v) > tau) {
          const double e = weight(v);
          total += e;
          if (bin_of(v) < lo) above += e;
        }
      });
      above = block_reduce(above, Sum(), sh.red_d);
      total = block_reduce(total, Sum(), sh.red_d);
      if (tid == 0) {
        sh.mass[0] = above;
        sh.mass[1] = total;
      }
      const uint32_t n = collect(lo, hi);
      above = over(&sh.mass[0], Sum());
      total = over(&sh.mass[1], Sum());
      const double extra_d = tau ? ties * weight(value_of(tau)) : 0.0;
      const double goal = (double)share * (total + extra_d) - above;
      bool found = false;
      if (n > 0 && n <= kList && goal > 0) {
        listed_weights();
        uint64_t sum = 0;
#pragma unroll
        for (int j = 0; j < kList / kThreads; ++j) sum += w[j];
        const int tau_bin = tau ? bin_of(value_of(tau)) : kBins;
        const bool ends_here = tau_bin >= lo && tau_bin <= hi;
        const uint64_t extra = ends_here ? ties * w_tau : 0;
        sum = block_reduce(sum, Sum(), sh.red) + extra;
        const uint64_t g = (uint64_t)max(1ll, __double2ll_ru(goal * kUnit));
        if (g <= sum && !(ends_here && ties > kList)) {  // more equals would not fit the whole numbers
          cut(extra, g);
          found = true;
        }
      } else if (n > kList && goal > 0 && list_lo() == list_hi() && list_lo() != tau) {  // equals only
        const double e = weight(value_of(list_lo())), need = ceil(goal / e);
        if (need <= (double)n) {
          tau = list_lo();
          ties = (uint32_t)need;
          found = true;
        }
      }
      if (!found) slow_mass(share);
    }
  }

  // ---- the draw, in the vocabulary's order --------------------------------------------------------
  const double floor_w = fminf(p.mins ? p.mins[b] : p.min_p, 1.f);  // the largest always stays
  // what is surely below the floor is not worth an exponential
  float floor_v = floor_w > 0 ? m + (float)(log(floor_w) * (double)temp) * 1.0001f - 1e-3f * temp - fabsf(m) * 1e-6f : -INFINITY;
  if (!(floor_v < INFINITY)) floor_v = -INFINITY;  // of an infinite maximum
  double kept = 0;
  uint32_t equal = 0;
  for (int blk = warp; blk < n_blk; blk += kWarps) {
    float v[8];
    load(blk, v);
    double s = 0;
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t kk = key_of(v[i]);
      n += kk == tau;
      if (kk > tau && kk > kNone && v[i] >= floor_v) {
        const double e = weight(v[i]);
        if (e >= floor_w) s += e;
      }
    }
    s = warp_reduce(s, Sum());
    n = warp_reduce(n, Sum());
    if (lane == 0) {
      blk_mass[blk] = s;
      blk_ties[blk] = n;
      kept += s;
      equal += n;
    }
  }
  kept = block_reduce(kept, Sum(), sh.red_d);
  equal = block_reduce(equal, Sum(), sh.red_u);
  if (tid == 0) {
    sh.kept = kept;
    sh.ties = equal;
    sh.found = 0x7fffffff;
    sh.last = -1;
  }
  cluster_barrier();
  double w_tau = tau ? weight(value_of(tau)) : 0.0;
  if (!(w_tau >= floor_w)) w_tau = 0.0;
  // the CTA that holds the draw: the first whose cumulative mass exceeds it, else the last with any
  double masses[kMaxCluster], total = 0;
  uint32_t before_c[kMaxCluster], ties_before = 0;
#pragma unroll
  for (int c = 0; c < kMaxCluster; ++c) {
    if (c >= C) break;
    const uint32_t t = peer(&sh.ties, c), left = ties > ties_before ? ties - ties_before : 0;
    masses[c] = peer(&sh.kept, c) + (double)min(t, left) * w_tau;
    before_c[c] = ties_before;
    total += masses[c];
    ties_before += t;
  }
  const double goal = (double)p.u[b] * total;
  double sum = 0, own_before = 0;
  int owner = -1, last_owner = -1;
  uint32_t own_ties = 0;
#pragma unroll
  for (int c = 0; c < kMaxCluster; ++c) {
    if (c >= C) break;
    if (c == me) own_before = sum, own_ties = before_c[c];
    sum += masses[c];
    if (masses[c] > 0) last_owner = c;
    if (owner < 0 && sum > goal) owner = c;
  }
  if (owner < 0) owner = last_owner;
  if (owner == me) {
    // its 256 tokens, likewise
    double before = own_before;
    uint32_t t_before = own_ties;
    for (int base = 0; base < n_blk; base += kThreads) {
      const int i = base + tid;
      const uint32_t t = i < n_blk ? blk_ties[i] : 0;
      const uint32_t t_inc = block_prefix(t, sh.red_u), t0 = t_before + t_inc - t;
      const uint32_t left = ties > t0 ? ties - t0 : 0;
      const double mass = i < n_blk ? blk_mass[i] + (double)min(t, left) * w_tau : 0.0;
      const double inc = before + block_prefix(mass, sh.red_d);
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
      // the sums so far, of the last thread
      if (tid == kThreads - 1) {
        sh.red[0] = __double_as_longlong(inc);
        sh.red[1] = t_before + t_inc;
      }
      __syncthreads();
      if (here) break;
      before = __longlong_as_double(sh.red[0]);
      t_before = (uint32_t)sh.red[1];
      __syncthreads();
    }
    if (warp == 0) {
      const int blk = sh.found != 0x7fffffff ? sh.found : sh.last;
      float v[8];
      double e[8], s = 0;
      uint32_t n = 0;
      load(blk, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) n += key_of(v[i]) == tau;
      uint32_t at = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t d = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += d;
      }
      at += sh.found_ties - n;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t kk = key_of(v[i]);
        const bool in = kk > tau || (kk == tau && at++ < ties);
        e[i] = in ? weight(v[i]) : 0.0;
        if (!(e[i] >= floor_w)) e[i] = 0.0;
        s += e[i];
      }
      double inc = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double d = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += d;
      }
      inc += sh.found_before;
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
  cluster_barrier();  // no block leaves while others read its variables
}

template <typename T>
int launch(SampleParams p, int batch, cudaStream_t stream) {
  static std::atomic<uint32_t> done{0};
  constexpr int kMost = 160 * 1024;  // of shared memory, beside the histogram and the list
  const int blocks = ceil_div(p.V, kBlock);
  // a cluster as large as keeps every block's warps busy and all rows resident
  // at once, and at least as large as holds the row
  int c = 1;
  auto bytes = [&](int n) {
    const size_t per = ceil_div(blocks, n);
    return align_up(per * 12, 16) + per * kBlock * sizeof(T);
  };
  while (c < kMaxCluster && (bytes(c) > (size_t)kMost || (2 * c * kWarps <= 2 * blocks && (int64_t)batch * c * 2 <= 2 * 148))) c *= 2;
  p.per_cta = ceil_div(blocks, c);
  p.staged = bytes(c) <= (size_t)kMost;
  const size_t smem = p.staged ? bytes(c) : align_up((size_t)p.per_cta * 12, 16);
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
