// skv_rotary: rotary positions of queries and keys.
//
// Pair i of a head is turned by a = p * inv_freq[i].  Positions of long
// contexts reach 10^6 and more, where a 32-bit product is off by a tenth of a
// radian; the product is taken in 64 bits, in turns (a / 2 pi), reduced to
// half a turn to each side there, and only the rest goes to a 32-bit sine and
// cosine.  Both are used by every head, so a thread keeps the ones of its
// V pairs in registers and walks the heads.
//
// Bound: HBM (every value read and written once; 3 flops a value).
#include "skv_common.cuh"

namespace skv {
namespace {

struct RotaryParams {
  const char* x[2];        // queries, keys
  char* y[2];
  int64_t xs[2][3], ys[2][3];  // batch, head, token (elements)
  const int64_t* pos;
  int64_t ps_b, ps_t;
  const float* inv_freq;
  float scale;             // negative angle: sine sign in sgn
  float sgn;
  int B, T, Hq, H;         // H: query and key heads together
  int D, r, chunks, rot_chunks, heads_per_thread;
};

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T e[V]; };

// A thread owns one chunk of one token: 2V channels, as two vectors of V (the
// two halves' same channels, or 2V channels in a row when interleaved; the
// channels past the rotated ones two vectors in a row).
template <typename T, int V, bool kInter>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  using VT = Vec<T, V>;
  const int64_t id = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  const int64_t row = id / p.chunks;
  const int c = (int)(id % p.chunks);
  if (row >= (int64_t)p.B * p.T) return;
  const int b = (int)(row / p.T), t = (int)(row % p.T);
  const bool rot = c < p.rot_chunks;
  int c0, c1;              // first channels of the two vectors
  if (rot) {
    c0 = kInter ? 2 * V * c : V * c;
    c1 = kInter ? c0 + V : c0 + p.r / 2;
  } else {
    c0 = p.r + 2 * V * (c - p.rot_chunks);
    c1 = c0 + V;
  }
  const bool two = c1 < p.D;  // the last copied chunk may hold one vector
  float cs[V], sn[V];
  if (rot) {
    const double x = (double)p.pos[b * p.ps_b + t * p.ps_t];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      double turn = x * (double)p.inv_freq[V * c + i] * 0.15915494309189533577;  // 1 / (2 pi)
      turn -= rint(turn);
      float s, co;
      sincospif((float)(2.0 * turn), &s, &co);
      cs[i] = co * p.scale;
      sn[i] = s * p.scale * p.sgn;
    }
  }
  const int h0 = blockIdx.y * p.heads_per_thread, h1 = min(p.H, h0 + p.heads_per_thread);
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    const int w = h >= p.Hq;
    const int hh = w ? h - p.Hq : h;
    const T* x = (const T*)p.x[w] + b * p.xs[w][0] + hh * p.xs[w][1] + t * p.xs[w][2];
    T* y = (T*)p.y[w] + b * p.ys[w][0] + hh * p.ys[w][1] + t * p.ys[w][2];
    VT v0 = *reinterpret_cast<const VT*>(x + c0), v1 = v0;
    if (two) v1 = *reinterpret_cast<const VT*>(x + c1);
    if (rot) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // pair i: (v0[i], v1[i]), or neighbours of the 2V channels in a row
        T& e0 = kInter ? (2 * i < V ? v0.e[2 * i % V] : v1.e[2 * i % V]) : v0.e[i];
        T& e1 = kInter ? (2 * i + 1 < V ? v0.e[(2 * i + 1) % V] : v1.e[(2 * i + 1) % V]) : v1.e[i];
        const float a = Elt<T>::to_f32(e0), d = Elt<T>::to_f32(e1);
        e0 = Elt<T>::from_f32(a * cs[i] - d * sn[i]);
        e1 = Elt<T>::from_f32(d * cs[i] + a * sn[i]);
      }
    }
    *reinterpret_cast<VT*>(y + c0) = v0;
    if (two) *reinterpret_cast<VT*>(y + c1) = v1;
  }
}

// Vector width: the widest of 16, 8, 4 or 2 bytes that divides the halves and
// the copied rest of a head and to which every address is aligned.
int vector_width(const skv_rotary_args* a, int es) {
  const int half = a->rotary_dim / 2;
  for (int v = 16 / es; v > 1; v /= 2) {
    const uint64_t bytes = (uint64_t)v * es;
    bool ok = half % v == 0 && (a->head_dim - a->rotary_dim) % v == 0;
    auto fits = [&](const void* ptr, const int64_t* st) {
      if ((uintptr_t)ptr % bytes) return false;
      for (int i = 0; i < 3; ++i)
        if ((uint64_t)(st[i] * es) % bytes) return false;
      return true;
    };
    ok = ok && fits(a->q, a->q_stride) && fits(a->q_out, a->q_out_stride);
    if (a->k) ok = ok && fits(a->k, a->k_stride) && fits(a->k_out, a->k_out_stride);
    if (ok) return v;
  }
  return 1;
}

template <typename T, int V>
int launch(RotaryParams& p, bool inter, cudaStream_t stream) {
  p.rot_chunks = p.r / (2 * V);
  p.chunks = p.rot_chunks + ceil_div(p.D - p.r, 2 * V);
  const int64_t threads = (int64_t)p.B * p.T * p.chunks;
  p.heads_per_thread = p.H;
  const int64_t blocks = ceil_div64(threads, 256);
  if (blocks > 0x7fffffff) return SKV_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)blocks, ceil_div(p.H, p.heads_per_thread));
  if (inter) rotary_kernel<T, V, true><<<grid, 256, 0, stream>>>(p);
  else rotary_kernel<T, V, false><<<grid, 256, 0, stream>>>(p);
  SKV_CHECK_LAUNCH();
  return SKV_OK;
}

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" int skv_rotary(const skv_rotary_args* a, void* stream) {
  if (!a || a->batch <= 0 || a->tokens <= 0 || a->num_q_heads <= 0 || a->head_dim <= 0 || a->rotary_dim <= 0)
    return SKV_ERR_INVALID_ARG;
  if (a->rotary_dim % 2 || a->rotary_dim > a->head_dim || !a->q || !a->q_out || !a->positions || !a->inv_freq)
    return SKV_ERR_INVALID_ARG;
  if (a->k ? (a->num_kv_heads <= 0 || !a->k_out) : (a->num_kv_heads != 0)) return SKV_ERR_INVALID_ARG;
  const int es = a->dtype == SKV_F32 ? 4 : (a->dtype == SKV_F16 || a->dtype == SKV_BF16) ? 2 : 0;
  if (!es) return SKV_ERR_UNSUPPORTED;
  auto aligned = [](const void* q, int n) { return (uintptr_t)q % n == 0; };
  if (!aligned(a->q, es) || !aligned(a->q_out, es) || !aligned(a->k, es) || !aligned(a->k_out, es) ||
      !aligned(a->positions, 8) || !aligned(a->inv_freq, 4))
    return SKV_ERR_MISALIGNED;
  RotaryParams p{};
  p.x[0] = (const char*)a->q; p.x[1] = (const char*)a->k;
  p.y[0] = (char*)a->q_out; p.y[1] = (char*)a->k_out;
  for (int i = 0; i < 3; ++i) {
    p.xs[0][i] = a->q_stride[i]; p.xs[1][i] = a->k_stride[i];
    p.ys[0][i] = a->q_out_stride[i]; p.ys[1][i] = a->k_out_stride[i];
  }
  p.pos = a->positions; p.ps_b = a->position_stride[0]; p.ps_t = a->position_stride[1];
  p.inv_freq = a->inv_freq; p.scale = a->scale; p.sgn = a->inverse ? -1.f : 1.f;
  p.B = a->batch; p.T = a->tokens; p.Hq = a->num_q_heads; p.H = a->num_q_heads + a->num_kv_heads;
  p.D = a->head_dim; p.r = a->rotary_dim;
  const int v = vector_width(a, es);
  const bool inter = a->interleaved != 0;
  const cudaStream_t s = (cudaStream_t)stream;
#define SKV_ROTARY(T)                                              \
  switch (v) {                                                     \
    case 8: return launch<T, sizeof(T) == 2 ? 8 : 4>(p, inter, s); \
    case 4: return launch<T, 4>(p, inter, s);                      \
    case 2: return launch<T, 2>(p, inter, s);                      \
    default: return launch<T, 1>(p, inter, s);                     \
  }
  if (a->dtype == SKV_F32) { SKV_ROTARY(float) }
  if (a->dtype == SKV_F16) { SKV_ROTARY(__half) }
  SKV_ROTARY(__nv_bfloat16)
#undef SKV_ROTARY
}
