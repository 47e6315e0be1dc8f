// Window attention for few query rows: decode steps and short chunks (fp16 and
// bf16), and prompts at the head dims that the tensor-memory kernel does not
// take.
//
// A block owns up to 8 * NT rows -- (token, query head) pairs of one kv head --
// and a share of the keys they see.  Each of its warps walks 16-key tiles on
// its own:
//   S^T (16 keys x 8 rows) = K Q^T,  O^T (D x 8 rows) += V^T P^T
// on mma.sync m16n8k16.  Keys go in straight from global memory in fragment
// order: the order of the contracted channels is free, so a lane loads 8
// neighbouring channels at once (the query's fragment is permuted alike), and
// V^T wants key pairs of one channel in a register, which byte permutes make
// of two rows' loads.  No shared memory, no barrier in the loop; a tile's loads
// are issued when the registers of the one before are free, and an SM's 12 or 16 warps
// keep about 100 KB in flight, three times what latency times bandwidth asks.
//
// Bound: HBM (2 * D * 2 bytes a key and kv head; the MMAs run at a few per cent
// of their rate).  Weights P enter the second product as two 16-bit terms, so
// the result carries no rounding of theirs: free where memory is the bound.
//
// Splits of one row group are the blocks of one cluster and join through
// distributed shared memory: one launch, no workspace.
#include "skv_mma.cuh"
#include "skv_window_join.cuh"

namespace skv {
namespace {

using namespace mma;

constexpr float kLog2e = 1.4426950408889634f;

template <int N> struct alignas(N * 4) Regs { uint32_t r[N]; };

template <int N>
__device__ __forceinline__ void load_regs(uint32_t* dst, const void* src) {
  const Regs<N> v = *reinterpret_cast<const Regs<N>*>(src);
#pragma unroll
  for (int i = 0; i < N; ++i) dst[i] = v.r[i];
}

template <typename T, int D, int NT>
struct FewCfg {
  static constexpr int kRows = 8 * NT;
  // head_dim 128 holds twice the registers: 12 warps an SM in three blocks (8 in two for 16 rows) instead of 16 in two
  static constexpr int kWarps = D == 128 ? 4 : 8;
  static constexpr int kBlocks = D == 128 && NT == 1 ? 3 : 2;
  static constexpr int kPitch = window_pitch(D);
  static constexpr size_t kPart = window_part_bytes(D, kRows, kWarps);
  static constexpr size_t kSmem = kPart + window_stat_bytes(kRows, kWarps);
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(FewCfg<T, D, NT>::kWarps * 32, FewCfg<T, D, NT>::kBlocks)
    window_few_kernel(const __grid_constant__ WindowParams p, int splits) {
  using C = FewCfg<T, D, NT>;
  constexpr int kWarps = C::kWarps;
  using O = Op<T>;
  constexpr int KC = D >= 32 ? 8 : 4;          // channels a lane loads of a key at once
  constexpr int KL = D / (4 * KC);             // such loads a key row
  constexpr int KR = KC / 2;                   // registers of one
  constexpr int VC = D >= 64 ? 8 : D / 8;      // the same of values
  constexpr int VL = D / (8 * VC);
  constexpr int VR = VC / 2;
  extern __shared__ __align__(16) unsigned char smem[];
  float* part = reinterpret_cast<float*>(smem);               // [warp][row][kPitch]
  float* stat = reinterpret_cast<float*>(smem + C::kPart);    // [warp + 1][row] max, then the same of sums

  const int split = blockIdx.x % splits, grp = blockIdx.x / splits;
  const int kh = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i8 = lane >> 2, t4 = lane & 3;
  const int G = p.Hq / p.Hkv, all_rows = p.T * G;
  const int r0 = grp * C::kRows, rows = min(C::kRows, all_rows - r0);
  const WindowRow row = window_row(p, b);
  const T* kb = (const T*)p.k + b * p.ks[0] + kh * p.ks[1];
  const T* vb = (const T*)p.v + b * p.vs[0] + kh * p.vs[1];
  const float sl2 = p.scaling * kLog2e;

  // slots of the group's live queries: [p_min, p_max]; none: p_max < p_min
  const int p_min = max(row.first + r0 / G, row.start);
  const int p_max = min(row.first + (r0 + rows - 1) / G, row.end - 1);
  // the keys that any of them sees, in two runs
  int a0 = 0, a1 = 0, w0 = 0, w1 = 0;
  if (p_min <= p_max) {
    a0 = row.start;
    a1 = min(row.sink_end, p_max + 1);
    w0 = max(a1, p_min - p.window + 1);
    w1 = p_max + 1;
  }
  const int a_tiles = (a1 - a0 + 15) >> 4, tiles = a_tiles + ((w1 - w0 + 15) >> 4);
  // this warp's tiles
  const int parts = splits * kWarps, me = split * kWarps + warp;
  const int tile0 = (int)((int64_t)tiles * me / parts), tile1 = (int)((int64_t)tiles * (me + 1) / parts);

  // the queries' fragments, and the slots of this lane's rows (columns 2 t4, 2 t4 + 1 of each n-tile)
  uint32_t qf[NT][KL][KR];
  int slot[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + 8 * n + i8;
    const bool live = 8 * n + i8 < rows;
    const T* q = (const T*)p.q + b * p.qs[0] + (kh * G + r % G) * p.qs[1] + (int64_t)(r / G) * p.qs[2];
#pragma unroll
    for (int c = 0; c < KL; ++c) {
      if (live) load_regs<KR>(qf[n][c], q + 4 * KC * c + KC * t4);
      else {
#pragma unroll
        for (int e = 0; e < KR; ++e) qf[n][c][e] = 0;
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) slot[n][e] = row.first + (r0 + 8 * n + 2 * t4 + e) / G;
  }

  float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int x = 0; x < D / 16; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][x][e] = 0.f;
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
  }

  uint32_t kf[2][KL][KR], vf[4][VL][VR];
  // first key of a tile and one past the last of its run; keys past it repeat the run's last one
  auto locate = [&](int tile, int& j, int& last) {
    const bool in_a = tile < a_tiles;
    j = in_a ? a0 + 16 * tile : w0 + 16 * (tile - a_tiles);
    last = (in_a ? a1 : w1) - 1;
  };
  auto load_k = [&](int tile) {
    int j, last;
    locate(tile, j, last);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const T* src = kb + min(j + i8 + 8 * e, last) * p.ks[2] + KC * t4;
#pragma unroll
      for (int c = 0; c < KL; ++c) load_regs<KR>(kf[e][c], src + 4 * KC * c);
    }
  };
  auto load_v = [&](int tile) {
    int j, last;
    locate(tile, j, last);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const T* src = vb + min(j + 2 * t4 + (e & 1) + 8 * (e >> 1), last) * p.vs[2] + VC * i8;
#pragma unroll
      for (int c = 0; c < VL; ++c) load_regs<VR>(vf[e][c], src + 8 * VC * c);
    }
  };

  if (tile0 < tile1) {
    load_k(tile0);
    load_v(tile0);
  }
  for (int tile = tile0; tile < tile1; ++tile) {
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
      for (int c = 0; c < KL; ++c)
#pragma unroll
        for (int h = 0; h < KR; h += 2)
          O::mma(s[n], kf[0][c][h], kf[1][c][h], kf[0][c][h + 1], kf[1][c][h + 1], qf[n][c][h], qf[n][c][h + 1]);
    }
    if (tile + 1 < tile1) load_k(tile + 1);
    int j, last;
    locate(tile, j, last);
    // whole tiles that every row of the group sees need no mask
    const bool whole = j + 15 <= last && j + 15 <= p_min && (tile < a_tiles || j > p_max - p.window) &&
                       row.first + r0 / G >= row.start && row.first + (r0 + rows - 1) / G < row.end;
    bool grow = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = s[n][e] * sl2;
        if (!whole) {
          const int key = j + i8 + 8 * (e >> 1), at = slot[n][e & 1];
          const bool sees = key <= last && key <= at && at < row.end && at >= row.start &&
                            (key < row.sink_end || at - key < p.window);
          x = sees ? x : -INFINITY;
        }
        s[n][e] = x;
        grow |= x > m[n][e & 1] + 8.f;
      }
    // the running maximum moves only when it is passed by 2^8 or more
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[n][e], s[n][e + 2]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
          x = fmaxf(x, m[n][e]);
          const float f = x == -INFINITY ? 1.f : ex2(m[n][e] - x);
          m[n][e] = x;
          l[n][e] *= f;
#pragma unroll
          for (int y = 0; y < D / 16; ++y) {
            o[n][y][e] *= f;
            o[n][y][e + 2] *= f;
          }
        }
    }
    uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = s[n][e] == -INFINITY ? 0.f : ex2(s[n][e] - m[n][e & 1] + weight_lift<T>());
        l[n][e & 1] += w[e];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t hi = O::pack(w[2 * e], w[2 * e + 1]);
        float h0, h1;
        O::unpack(hi, h0, h1);
        ph[n][e] = movm_t(hi);
        pl[n][e] = movm_t(O::pack(w[2 * e] - h0, w[2 * e + 1] - h1));
      }
    }
#pragma unroll
    for (int c = 0; c < VL; ++c)
#pragma unroll
      for (int h = 0; h < VR; ++h) {
        uint32_t a[4];
        a[0] = __byte_perm(vf[0][c][h], vf[1][c][h], 0x5410);
        a[1] = __byte_perm(vf[0][c][h], vf[1][c][h], 0x7632);
        a[2] = __byte_perm(vf[2][c][h], vf[3][c][h], 0x5410);
        a[3] = __byte_perm(vf[2][c][h], vf[3][c][h], 0x7632);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          O::mma(o[n][c * VR + h], a[0], a[1], a[2], a[3], ph[n][0], ph[n][1]);
          O::mma(o[n][c * VR + h], a[0], a[1], a[2], a[3], pl[n][0], pl[n][1]);
        }
      }
    if (tile + 1 < tile1) load_v(tile + 1);
  }

  // this warp's share: row 2 t4 + e of an n-tile, channels 8 VC c + VC i8 + 2 h + f at o[n][c VR + h][2 f + e]
  float* mine = part + (size_t)warp * C::kRows * C::kPitch;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[n][e];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      const int r = 8 * n + 2 * t4 + e;
      if (i8 == 0) {
        stat[warp * C::kRows + r] = m[n][e];
        stat[(kWarps + 1 + warp) * C::kRows + r] = x;
      }
#pragma unroll
      for (int c = 0; c < VL; ++c)
#pragma unroll
        for (int h = 0; h < VR; ++h)
          *reinterpret_cast<float2*>(mine + r * C::kPitch + 8 * VC * c + VC * i8 + 2 * h) =
              make_float2(o[n][c * VR + h][e], o[n][c * VR + h][2 + e]);
    }
  window_join<T, D, C::kRows, kWarps>(p, row, b, kh, r0, rows, split, splits, part, stat);
}

template <typename T, int D, int NT>
int launch_few(const WindowParams& p, cudaStream_t stream) {
  using C = FewCfg<T, D, NT>;
  static WindowFewState state;
  return launch_window_few(p, window_few_kernel<T, D, NT>, state, C::kRows, C::kWarps, C::kBlocks, C::kSmem, stream);
}

template <typename T>
int dispatch_few(const WindowParams& p, cudaStream_t stream) {
  const bool one = (int64_t)p.T * (p.Hq / p.Hkv) <= 8;
  switch (p.D) {
    case 16: return one ? launch_few<T, 16, 1>(p, stream) : launch_few<T, 16, 2>(p, stream);
    case 32: return one ? launch_few<T, 32, 1>(p, stream) : launch_few<T, 32, 2>(p, stream);
    case 64: return one ? launch_few<T, 64, 1>(p, stream) : launch_few<T, 64, 2>(p, stream);
    default: return one ? launch_few<T, 128, 1>(p, stream) : launch_few<T, 128, 2>(p, stream);
  }
}

}  // namespace

int window_few(const WindowParams& p, int dtype, cudaStream_t stream) {
  return dtype == SKV_F16 ? dispatch_few<__half>(p, stream) : dispatch_few<__nv_bfloat16>(p, stream);
}

}  // namespace skv
