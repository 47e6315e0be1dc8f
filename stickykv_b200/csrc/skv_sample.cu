// skv_sample: the next token of each row from its logits and a given random
// number (temperature, top-k, top-p, min-p).
//
// Descending logits with ties by index make every cut a threshold: the key of
// the last kept token and how many of its equals, lowest indices first, stay.
// Weights and sums are 64-bit: a draw falls between two neighbours of 10^5
// cumulative sums, and 32-bit sums would move a share of draws to a neighbour.
#include "skv_common.cuh"

namespace skv {
namespace {

constexpr int kThreads = 1024;

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
};

// Total order of the values as unsigned integers: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) x = -INFINITY;
  x += 0.f;
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t kNone = 0x007fffffu;  // key of -inf

template <typename A, typename Op>
__device__ A block_reduce(A v, Op op, A* buf) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = buf[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// exclusive prefix over the block's threads
template <typename A>
__device__ A block_prefix(A v, A* buf) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  A inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const A n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 31) buf[warp] = inc;
  __syncthreads();
  A base = 0;
  for (int w = 0; w < warp; ++w) base += buf[w];
  const A ex = __shfl_up_sync(0xffffffffu, inc, 1);
  return base + (lane ? ex : A(0));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  __shared__ double dbuf[32];
  __shared__ uint32_t ubuf[32];
  __shared__ int found;
  const int b = blockIdx.x, tid = threadIdx.x, V = p.V;
  const T* x = (const T*)p.logits + b * p.stride;
  auto key = [&](int i) { return key_of(Elt<T>::to_f32(x[i])); };
  const auto umax = [](uint32_t a, uint32_t c) { return a > c ? a : c; };
  const auto umin = [](uint32_t a, uint32_t c) { return a < c ? a : c; };
  const auto uadd = [](uint32_t a, uint32_t c) { return a + c; };
  const auto dadd = [](double a, double c) { return a + c; };

  uint32_t top = 0;
  for (int i = tid; i < V; i += kThreads) top = umax(top, key(i));
  top = block_reduce(top, umax, ubuf);
  if (top == kNone) {  // nothing above -inf
    if (tid == 0) p.out[b] = -1;
    return;
  }
  const float temp = p.temps ? p.temps[b] : p.temp;
  if (!(temp > 0.f)) {
    uint32_t at = 0xffffffffu;
    for (int i = tid; i < V; i += kThreads)
      if (key(i) == top) at = umin(at, (uint32_t)i);
    at = block_reduce(at, umin, ubuf);
    if (tid == 0) p.out[b] = at;
    return;
  }
  const double m = value_of(top), inv = 1.0 / (double)temp;
  auto weight = [&](uint32_t k) -> double {
    if (k == top) return 1.0;
    if (k == kNone) return 0.0;
    return exp(((double)value_of(k) - m) * inv);
  };

  // kept so far: keys above `tau`, and the first `ties` of its equals
  uint32_t tau = 0, ties = (uint32_t)V;
  const int k = p.ks ? p.ks[b] : p.k;
  if (k > 0 && k < V) {
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
      uint32_t n = 0;
      for (int i = tid; i < V; i += kThreads) n += key(i) >= (tau | bit);
      if (block_reduce(n, uadd, ubuf) >= (uint32_t)k) tau |= bit;
    }
    uint32_t n = 0;
    for (int i = tid; i < V; i += kThreads) n += key(i) > tau;
    ties = (uint32_t)k - block_reduce(n, uadd, ubuf);
  }
  const float pp = p.ps ? p.ps[b] : p.p;
  if (pp < 1.f) {
    const uint32_t tau_k = tau, ties_k = ties;
    auto mass = [&](uint32_t least) {  // of the kept keys >= least
      double s = 0;
      for (int i = tid; i < V; i += kThreads) {
        const uint32_t kk = key(i);
        if (kk >= least && kk > tau_k) s += weight(kk);
      }
      s = block_reduce(s, dadd, dbuf);
      return tau_k && least <= tau_k ? s + ties_k * weight(tau_k) : s;
    };
    const double goal = (double)pp * mass(0);
    uint32_t t = 0;
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
      if ((t | bit) <= top && mass(t | bit) >= goal) t |= bit;
    // fewest of the equals of t (those kept so far) that reach the goal, one at least
    uint32_t n = 0;
    for (int i = tid; i < V; i += kThreads) n += key(i) == t;
    n = block_reduce(n, uadd, ubuf);
    if (t == tau_k) n = umin(n, ties_k);
    const double above = t == 0xffffffffu ? 0.0 : mass(t + 1), w = weight(t);
    const double need = w > 0 ? ceil((goal - above) / w) : 1.0;
    tau = umax(t, tau_k);
    ties = need >= (double)n ? n : need < 1.0 ? 1u : (uint32_t)need;
  }
  const double floor_w = fminf(p.mins ? p.mins[b] : p.min_p, 1.f);  // the largest always stays

  // vocabulary order: every thread a run of tokens
  const int run = (V + kThreads - 1) / kThreads;
  const int i0 = min(V, tid * run), i1 = min(V, i0 + run);
  uint32_t eq = 0;
  for (int i = i0; i < i1; ++i) eq += key(i) == tau;
  const uint32_t eq0 = block_prefix(eq, ubuf);
  auto walk = [&](auto&& take) {
    uint32_t rank = eq0;
    for (int i = i0; i < i1; ++i) {
      const uint32_t kk = key(i);
      bool kept = kk > tau;
      if (kk == tau) kept = rank++ < ties;
      if (!kept) continue;
      const double w = weight(kk);
      if (w >= floor_w && w > 0 && take(i, w)) return;
    }
  };
  double mine = 0;
  int last = -1;
  walk([&](int i, double w) { mine += w; last = i; return false; });
  const double before = block_prefix(mine, dbuf);
  const double total = block_reduce(mine, dadd, dbuf);
  const double goal = (double)p.u[b] * total;
  if (tid == 0) found = 0x7fffffff;
  __syncthreads();
  if (last >= 0 && before + mine > goal) {
    double s = before;
    int at = last;
    walk([&](int i, double w) {
      s += w;
      if (s > goal) { at = i; return true; }
      return false;
    });
    atomicMin(&found, at);
  }
  const int end = (int)block_reduce((uint32_t)(last + 1), umax, ubuf) - 1;  // last kept of the row
  if (tid == 0) p.out[b] = found == 0x7fffffff ? end : found;
}

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" int skv_sample(const skv_sample_args* a, void* stream) {
  if (!a || a->batch <= 0 || a->vocabulary <= 0 || !a->logits || !a->uniform || !a->tokens) return SKV_ERR_INVALID_ARG;
  if (a->row_stride < 0) return SKV_ERR_INVALID_ARG;
  const int es = a->dtype == SKV_F32 ? 4 : (a->dtype == SKV_F16 || a->dtype == SKV_BF16) ? 2 : 0;
  if (!es) return SKV_ERR_UNSUPPORTED;
  if ((uintptr_t)a->logits % es || (uintptr_t)a->uniform % 4 || (uintptr_t)a->tokens % 8 ||
      (uintptr_t)a->temperatures % 4 || (uintptr_t)a->top_ks % 4 || (uintptr_t)a->top_ps % 4 ||
      (uintptr_t)a->min_ps % 4)
    return SKV_ERR_MISALIGNED;
  SampleParams p{a->logits, a->row_stride, a->uniform, a->temperatures, a->top_ks, a->top_ps, a->min_ps,
                 a->tokens, a->temperature, a->top_p, a->min_p, a->top_k, a->vocabulary};
  const cudaStream_t s = (cudaStream_t)stream;
  if (a->dtype == SKV_F32) sample_kernel<float><<<a->batch, kThreads, 0, s>>>(p);
  else if (a->dtype == SKV_F16) sample_kernel<__half><<<a->batch, kThreads, 0, s>>>(p);
  else sample_kernel<__nv_bfloat16><<<a->batch, kThreads, 0, s>>>(p);
  SKV_CHECK_LAUNCH();
  return SKV_OK;
}
