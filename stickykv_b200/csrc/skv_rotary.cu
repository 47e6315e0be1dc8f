// skv_rotary: rotary positions of queries and keys.
//
// Pair i of a head is turned by a = p * inv_freq[i].  Positions of long
// contexts reach 10^6 and more, where a 32-bit product is off by a tenth of a
// radian; the product is taken in 64 bits, in turns (a / 2 pi), reduced to
// half a turn to each side there, and only the rest goes to a 32-bit sine and
// cosine.  For float32 the part of the angle that 32 bits leave out is added to
// both (results are off by 4.1e-8 of their size, root mean square, without it by
// 5.6e-8; 204 us with and without for the tensors below); 16-bit results do not
// show it.
//
// A block owns 32 chunks of 2V channels, of one token or several, for four
// heads at a time: it takes the sines and cosines of its chunks once, through
// shared memory, and every thread keeps those of its chunk in registers over
// its heads, five of them in flight.
//
// Bound: HBM (every value read and written once; 3 flops a value).  4 x 8192
// tokens x 40 heads x 128 bf16, 671 MB: 103 us = 6.5 TB/s, the rate of a copy.
// A thread that takes its own sines: 118 us for 8 heads each (4 instructions a
// value go to sines), 135 us for all 40 (too few threads for the GPU); loads
// one head at a time, each waiting behind the last one's store, 127 us; 256
// threads of 64 chunks 118 us.  One token of 4 rows: 3.1 us.
#include "skv_mma.cuh"

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
  int D, r, chunks, rot_chunks, heads_per_block;
};

// A vector in registers: whole words, not one register an element.
template <int N> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };

// Turns V pairs that lie in two vectors: pair i is (v0[i], v1[i]), or
// neighbours of the 2V channels in a row.
template <typename T, int V, bool kInter, typename RT>
__device__ __forceinline__ void turn_pairs(RT& r0, RT& r1, const float (&cs)[V], const float (&sn)[V]) {
  if constexpr (sizeof(T) == 2 && V > 1) {  // two elements a word, packed and unpacked as such
    using O = mma::Op<T>;
    constexpr int W = V / 2;
    uint32_t* w0 = reinterpret_cast<uint32_t*>(&r0);
    uint32_t* w1 = reinterpret_cast<uint32_t*>(&r1);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      float a0, a1, b0, b1;
      O::unpack(w0[i], a0, a1);
      O::unpack(w1[i], b0, b1);
      if (kInter) {
        w0[i] = O::pack(a0 * cs[i] - a1 * sn[i], a1 * cs[i] + a0 * sn[i]);
        w1[i] = O::pack(b0 * cs[W + i] - b1 * sn[W + i], b1 * cs[W + i] + b0 * sn[W + i]);
      } else {
        w0[i] = O::pack(a0 * cs[2 * i] - b0 * sn[2 * i], a1 * cs[2 * i + 1] - b1 * sn[2 * i + 1]);
        w1[i] = O::pack(b0 * cs[2 * i] + a0 * sn[2 * i], b1 * cs[2 * i + 1] + a1 * sn[2 * i + 1]);
      }
    }
  } else {
    T* e0 = reinterpret_cast<T*>(&r0);
    T* e1 = reinterpret_cast<T*>(&r1);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      T& p = kInter ? (2 * i < V ? e0[2 * i % V] : e1[2 * i % V]) : e0[i];
      T& q = kInter ? (2 * i + 1 < V ? e0[(2 * i + 1) % V] : e1[(2 * i + 1) % V]) : e1[i];
      const float a = Elt<T>::to_f32(p), d = Elt<T>::to_f32(q);
      p = Elt<T>::from_f32(a * cs[i] - d * sn[i]);
      q = Elt<T>::from_f32(d * cs[i] + a * sn[i]);
    }
  }
}

constexpr int kThreads = 128, kChunks = 32, kHeads = kThreads / kChunks, kBatch = 5;

// A chunk is 2V channels of a token, as two vectors of V: the two halves' same
// channels, or 2V channels in a row when interleaved; the channels past the
// rotated ones two vectors in a row.
template <typename T, int V, bool kInter>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  using RT = typename Raw<sizeof(T) * V>::type;
  __shared__ __align__(16) float2 turns[kChunks * V];  // cosine, sine
  __shared__ double where[kChunks];                    // position / 2 pi
  __shared__ int batch[kChunks], token[kChunks], chunk[kChunks];  // batch < 0: behind the last row
  if (threadIdx.x < kChunks) {                         // the divisions, once a chunk
    const uint64_t id = blockIdx.x * (uint64_t)kChunks + threadIdx.x;
    const uint32_t row = id >> 32 ? (uint32_t)(id / p.chunks) : (uint32_t)id / p.chunks;
    const bool live = row < (uint32_t)p.B * (uint32_t)p.T;
    const int b = live ? (int)(row / (uint32_t)p.T) : -1, t = live ? (int)(row % (uint32_t)p.T) : 0;
    batch[threadIdx.x] = b;
    token[threadIdx.x] = t;
    chunk[threadIdx.x] = (int)(id - (uint64_t)row * p.chunks);
    where[threadIdx.x] = live ? (double)p.pos[b * p.ps_b + t * p.ps_t] * 0.15915494309189533577 : 0.0;
  }
  __syncthreads();
  const int mine = threadIdx.x % kChunks;
  const int b = batch[mine], t = token[mine], c = chunk[mine];
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
  for (int i = threadIdx.x; i < kChunks * V; i += kThreads) {
    const int k = chunk[i / V];
    if (k < p.rot_chunks) {
      double turn = where[i / V] * (double)p.inv_freq[V * k + i % V];
      turn -= (turn + 6755399441055744.0) - 6755399441055744.0;  // 1.5 * 2^52: rounds to whole turns
      const float a = (float)(2.0 * turn);
      float s, co;
      sincospif(a, &s, &co);
      if constexpr (sizeof(T) == 4) {  // and what the angle's rounding left over, up to 2^-25, to first order
        const float left = (float)(2.0 * turn - (double)a) * 3.14159265f, s0 = s;
        s = fmaf(co, left, s);
        co = fmaf(-s0, left, co);
      }
      turns[i] = make_float2(co * p.scale, s * p.scale * p.sgn);
    }
  }
  __syncthreads();
  if (b < 0) return;
  float cs[V], sn[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 f = turns[mine * V + i];
    cs[i] = f.x;
    sn[i] = f.y;
  }
  const int h0 = blockIdx.y * p.heads_per_block + threadIdx.x / kChunks;
  const int h1 = min(p.H, (int)(blockIdx.y + 1) * p.heads_per_block);
  // the vectors of kBatch heads come in together before any goes out: a load cannot pass a store that may be to its address
  for (int hb = h0; hb < h1; hb += kBatch * kHeads) {
    RT v[kBatch][2];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int h = hb + u * kHeads;
      if (h >= h1) break;
      const int w = h >= p.Hq, hh = w ? h - p.Hq : h;
      const T* x = (const T*)p.x[w] + b * p.xs[w][0] + hh * p.xs[w][1] + t * p.xs[w][2];
      v[u][0] = *reinterpret_cast<const RT*>(x + c0);
      if (two) v[u][1] = *reinterpret_cast<const RT*>(x + c1);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int h = hb + u * kHeads;
      if (h >= h1) break;
      const int w = h >= p.Hq, hh = w ? h - p.Hq : h;
      T* y = (T*)p.y[w] + b * p.ys[w][0] + hh * p.ys[w][1] + t * p.ys[w][2];
      if (rot) turn_pairs<T, V, kInter>(v[u][0], v[u][1], cs, sn);
      *reinterpret_cast<RT*>(y + c0) = v[u][0];
      if (two) *reinterpret_cast<RT*>(y + c1) = v[u][1];
    }
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
  const int64_t blocks = ceil_div64((int64_t)p.B * p.T * p.chunks, kChunks);
  if (blocks > 0x7fffffff || (int64_t)p.B * p.T > 0x7fffffff) return SKV_ERR_UNSUPPORTED;
  // a small call wants its heads side by side
  p.heads_per_block = align_up(p.H, kHeads);
  while (p.heads_per_block > kHeads && blocks * ceil_div(p.H, p.heads_per_block) < 8 * 148)
    p.heads_per_block = align_up(p.heads_per_block / 2, kHeads);
  const dim3 grid((unsigned)blocks, ceil_div(p.H, p.heads_per_block));
  if (inter) rotary_kernel<T, V, true><<<grid, kThreads, 0, stream>>>(p);
  else rotary_kernel<T, V, false><<<grid, kThreads, 0, stream>>>(p);
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
