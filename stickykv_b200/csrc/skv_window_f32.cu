// Window attention in float32, any number of query rows.
//
// A block owns 16 rows -- (token, query head) pairs of one kv head -- and a
// share of the keys they see; each of its 4 warps walks 8-key tiles on its own:
//   S (16 rows x 8 keys) = Q K^T,  O (16 rows x D) += P V
// on mma.sync m16n8k8 with tf32 operands.  A float32 number is the sum of two
// tf32 ones to 2^-22 of itself, so each product is three: high x high, high x
// low, low x high.  The matrix unit cuts off what it adds up, always towards
// zero, so a sum stays in it for a few products only (8 keys of O; of S the two
// halves and the small cross terms apart) and goes on in rounded 32-bit
// additions: all in it, 16000 keys came out 2e-6 off.  The orders of the contracted channels and
// keys and of the output channels are free and chosen so that every lane loads
// 4 neighbouring channels at once, and P's accumulator layout is the second
// product's operand layout: no shared memory in the loop, no exchange.
//
// Bound: the three-fold MMAs and the splitting of K and V beside them (decode of
// 18 rows, 8 kv heads, 1305 keys, head_dim 128: 58 us, 3.3 TB/s of the cache's
// bytes; a prompt of 8 x 1500 tokens, 64 heads of 128: 9.1 ms).
#include "skv_window_join.cuh"

namespace skv {
namespace {

using namespace mma;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 4, kRows = 16;

template <int D> struct F32Cfg {
  static constexpr int kBlocks = D == 128 ? 2 : 4;  // of 4 warps an SM: 255 and 128 registers
  static constexpr size_t kPart = window_part_bytes(D, kRows, kWarps);
  static constexpr size_t kStat = window_stat_bytes(kRows, kWarps);
  static constexpr int kSteps = D / 8;              // of the first product
  static constexpr size_t kSmem = kPart + kStat + (size_t)kSteps * 2 * 32 * 16;  // and the queries' operands
};

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the two terms of a number, each to the nearest
__device__ __forceinline__ uint32_t high(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;\n" : "=r"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t low(float x) { return high(x - __uint_as_float(high(x))); }

template <int D>
__global__ void __launch_bounds__(kWarps * 32, F32Cfg<D>::kBlocks)
    window_f32_kernel(const __grid_constant__ WindowParams p, int splits) {
  using C = F32Cfg<D>;
  constexpr int kPitch = window_pitch(D);
  constexpr int KL = D / 16;                   // 16-byte loads of a key by a lane: channels 16 c + 4 t4 ..
  constexpr int VW = D >= 32 ? 4 : 2;          // neighbouring channels a lane loads of a value
  constexpr int VL = D / (8 * VW);
  extern __shared__ __align__(16) unsigned char smem[];
  float* part = reinterpret_cast<float*>(smem);
  float* stat = reinterpret_cast<float*>(smem + C::kPart);
  const int split = blockIdx.x % splits, grp = blockIdx.x / splits;
  const int kh = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i8 = lane >> 2, t4 = lane & 3;
  const int G = p.Hq / p.Hkv, all_rows = p.T * G;
  const int r0 = grp * kRows, rows = min(kRows, all_rows - r0);
  const WindowRow row = window_row(p, b);
  const float* kb = (const float*)p.k + b * p.ks[0] + kh * p.ks[1];
  const float* vb = (const float*)p.v + b * p.vs[0] + kh * p.vs[1];
  const float sl2 = p.scaling * kLog2e;

  // the keys that any of the group's live queries sees, in two runs of 8-key tiles
  const int p_min = max(row.first + r0 / G, row.start);
  const int p_max = min(row.first + (r0 + rows - 1) / G, row.end - 1);
  int a0 = 0, a1 = 0, w0 = 0, w1 = 0;
  if (p_min <= p_max) {
    a0 = row.start;
    a1 = min(row.sink_end, p_max + 1);
    w0 = max(a1, p_min - p.window + 1);
    w1 = p_max + 1;
  }
  const int a_tiles = (a1 - a0 + 7) >> 3, tiles = a_tiles + ((w1 - w0 + 7) >> 3);
  const int parts = splits * kWarps, me = split * kWarps + warp;
  const int tile0 = (int)((int64_t)tiles * me / parts), tile1 = (int)((int64_t)tiles * (me + 1) / parts);

  // rows i8 and i8 + 8: their slots, and the queries' operands, both terms, through shared memory (in registers they would
  // be split again for every tile)
  uint4* qop = reinterpret_cast<uint4*>(smem + C::kPart + C::kStat);  // [step][term][lane]
  int slot[2];
  const float* src[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = r0 + i8 + 8 * e;
    slot[e] = row.first + r / G;
    src[e] = i8 + 8 * e < rows ? (const float*)p.q + b * p.qs[0] + (kh * G + r % G) * p.qs[1] + (int64_t)(r / G) * p.qs[2] + 4 * t4
                               : nullptr;
  }
  for (int c = warp; c < KL; c += kWarps) {
    float4 x[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) x[e] = src[e] ? *reinterpret_cast<const float4*>(src[e] + 16 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
    qop[(4 * c + 0) * 32 + lane] = make_uint4(high(x[0].x), high(x[1].x), high(x[0].y), high(x[1].y));
    qop[(4 * c + 1) * 32 + lane] = make_uint4(low(x[0].x), low(x[1].x), low(x[0].y), low(x[1].y));
    qop[(4 * c + 2) * 32 + lane] = make_uint4(high(x[0].z), high(x[1].z), high(x[0].w), high(x[1].w));
    qop[(4 * c + 3) * 32 + lane] = make_uint4(low(x[0].z), low(x[1].z), low(x[0].w), low(x[1].w));
  }
  __syncthreads();

  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int x = 0; x < D / 8; ++x)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[x][e] = 0.f;

  float kf[KL][4], vf[2][VL][VW];
  auto locate = [&](int tile, int& j, int& last) {
    const bool in_a = tile < a_tiles;
    j = in_a ? a0 + 8 * tile : w0 + 8 * (tile - a_tiles);
    last = (in_a ? a1 : w1) - 1;
  };
  auto load_k = [&](int tile) {  // key i8 of the tile (those past the run repeat its last)
    int j, last;
    locate(tile, j, last);
    const float* src = kb + min(j + i8, last) * p.ks[2] + 4 * t4;
#pragma unroll
    for (int c = 0; c < KL; ++c) {
      const float4 x = *reinterpret_cast<const float4*>(src + 16 * c);
      kf[c][0] = x.x; kf[c][1] = x.y; kf[c][2] = x.z; kf[c][3] = x.w;
    }
  };
  auto load_v = [&](int tile) {  // values 2 t4 and 2 t4 + 1, channels 8 VW c + VW i8 ..
    int j, last;
    locate(tile, j, last);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float* src = vb + min(j + 2 * t4 + e, last) * p.vs[2] + VW * i8;
#pragma unroll
      for (int c = 0; c < VL; ++c) {
        if constexpr (VW == 4) {
          const float4 x = *reinterpret_cast<const float4*>(src + 32 * c);
          vf[e][c][0] = x.x; vf[e][c][1] = x.y; vf[e][c][2] = x.z; vf[e][c][3] = x.w;
        } else {
          const float2 x = *reinterpret_cast<const float2*>(src + 16 * c);
          vf[e][c][0] = x.x; vf[e][c][1] = x.y;
        }
      }
    }
  };

  if (tile0 < tile1) {
    load_k(tile0);
    load_v(tile0);
  }
  for (int tile = tile0; tile < tile1; ++tile) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};         // (row i8, keys 2 t4 and + 1), (row i8 + 8, the same)
    float s2[4] = {0.f, 0.f, 0.f, 0.f}, cross[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < KL; ++c)
#pragma unroll
      for (int h = 0; h < 4; h += 2) {
        const uint4 qh = qop[(4 * c + h) * 32 + lane], ql = qop[(4 * c + h + 1) * 32 + lane];
        const uint32_t ah[4] = {qh.x, qh.y, qh.z, qh.w}, al[4] = {ql.x, ql.y, ql.z, ql.w};
        mma_tf32(cross, al, high(kf[c][h]), high(kf[c][h + 1]));
        mma_tf32(cross, ah, low(kf[c][h]), low(kf[c][h + 1]));
        mma_tf32(h ? s2 : s, ah, high(kf[c][h]), high(kf[c][h + 1]));
      }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += s2[e] + cross[e];
    if (tile + 1 < tile1) load_k(tile + 1);
    int j, last;
    locate(tile, j, last);
    const bool whole = j + 7 <= last && j + 7 <= p_min && (tile < a_tiles || j > p_max - p.window) &&
                       row.first + r0 / G >= row.start && row.first + (r0 + rows - 1) / G < row.end;
    bool grow = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = s[e] * sl2;
      if (!whole) {
        const int key = j + 2 * t4 + (e & 1), at = slot[e >> 1];
        const bool sees = key <= last && key <= at && at < row.end && at >= row.start &&
                          (key < row.sink_end || at - key < p.window);
        x = sees ? x : -INFINITY;
      }
      s[e] = x;
      grow |= x > m[e >> 1] + 8.f;
    }
    // the running maximum moves only when it is passed by 2^8 or more
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = fmaxf(s[2 * e], s[2 * e + 1]);
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        x = fmaxf(x, m[e]);
        const float f = x == -INFINITY ? 1.f : exp2f(m[e] - x);
        m[e] = x;
        l[e] *= f;
#pragma unroll
        for (int y = 0; y < D / 8; ++y) {
          o[y][2 * e] *= f;
          o[y][2 * e + 1] *= f;
        }
      }
    }
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = s[e] == -INFINITY ? 0.f : exp2f(s[e] - m[e >> 1]);
      l[e >> 1] += w[e];
    }
    // P as the operand: contracted index t4 is key 2 t4, t4 + 4 is key 2 t4 + 1
    const uint32_t ah[4] = {high(w[0]), high(w[2]), high(w[1]), high(w[3])};
    const uint32_t al[4] = {low(w[0]), low(w[2]), low(w[1]), low(w[3])};
#pragma unroll
    for (int c = 0; c < VL; ++c)
#pragma unroll
      for (int h = 0; h < VW; ++h) {           // output column i8 is channel 8 VW c + VW i8 + h
        const float v0 = vf[0][c][h], v1 = vf[1][c][h];
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        mma_tf32(x, al, high(v0), high(v1));
        mma_tf32(x, ah, low(v0), low(v1));
        mma_tf32(x, ah, high(v0), high(v1));
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c * VW + h][e] += x[e];
      }
    if (tile + 1 < tile1) load_v(tile + 1);
  }

  float* mine = part + (size_t)warp * kRows * kPitch;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float x = l[e];
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    x += __shfl_xor_sync(0xffffffffu, x, 2);
    const int r = i8 + 8 * e;
    if (t4 == 0) {
      stat[warp * kRows + r] = m[e];
      stat[(kWarps + 1 + warp) * kRows + r] = x;
    }
#pragma unroll
    for (int c = 0; c < VL; ++c)
#pragma unroll
      for (int h = 0; h < VW; ++h) {           // columns 2 t4 and 2 t4 + 1
        mine[r * kPitch + 8 * VW * c + VW * (2 * t4) + h] = o[c * VW + h][2 * e];
        mine[r * kPitch + 8 * VW * c + VW * (2 * t4 + 1) + h] = o[c * VW + h][2 * e + 1];
      }
  }
  window_join<float, D, kRows, kWarps>(p, row, b, kh, r0, rows, split, splits, part, stat);
}

template <int D>
int launch_f32(const WindowParams& p, cudaStream_t stream) {
  using C = F32Cfg<D>;
  static WindowFewState state;
  return launch_window_few(p, window_f32_kernel<D>, state, kRows, kWarps, C::kBlocks, C::kSmem, stream);
}

}  // namespace

int window_f32(const WindowParams& p, cudaStream_t stream) {
  switch (p.D) {
    case 16: return launch_f32<16>(p, stream);
    case 32: return launch_f32<32>(p, stream);
    case 64: return launch_f32<64>(p, stream);
    default: return launch_f32<128>(p, stream);
  }
}

}  // namespace skv
