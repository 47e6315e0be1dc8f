// Window attention of prompts and chunks on the 5th-generation tensor cores
// (fp16/bf16, head_dim 64 and 128).
//
// A block owns two tiles of 128 rows of one kv head; a row is a (token, query
// head) pair, the group's heads of a token side by side, so K and V are fetched
// once for all of them.  The keys that any of its rows sees form two runs, the
// first tokens (rounded up to 8) and the window, which one sequence of 128-key
// tiles covers: a few first tokens share a tile with the window's beginning.
//
//   warp 9         TMA (10 and 11 complete the warpgroup): Q once, then K and V tiles through a ring
//   warp 8         issues the MMAs:  S_t = Q_t K^T,  O_t += P_t V
//   warps 0-3/4-7  softmax of tile 0/1, a thread a row: S from tensor memory,
//                  P = exp2(S - m) back into S's columns as the second MMA's A
//                  operand; the running maximum m moves only when it is passed
//                  by 2^8, and then the row of O is rescaled in tensor memory
// While one tile is in its softmax the other one's MMAs run.  Tensor memory: S
// 2 x 128 columns, O 2 x D.
//
// P is rounded to the operands' 16 bits, its sum l is not: against 64 bits the
// result is off by 2.1e-3 of its size in bf16 (its own rounding 1.6e-3) and
// 2.6e-4 in fp16 (2.0e-4), root mean square.  A second term for what the rounding
// leaves, as skv_window_few.cu has it, gives 1.6e-3 and 2.0e-4, but half as many
// MMAs again and packing: 526 -> 583 us for 4 x 8192 tokens, head_dim 64, window
// 1024; 1970 -> 2490 us for 32768, head_dim 128, window 4096.
//
// Bound: a 128 x 128 tile takes 16384 exp2 at 16 a clock = 1024 clocks, and
// 8 * D clocks of MMA; both at once, the exponentials bound head_dim 64, the two
// are level at 128.
#include "skv_tc.cuh"
#include "skv_window_rows.cuh"

namespace skv {
namespace {

using namespace tcg;
using mma::ex2;
using mma::Op;
using mma::smem_u32;

constexpr int kRows = 128;
constexpr int kThreads = 384;
constexpr float kLog2e = 1.4426950408889634f;

template <int D> struct ManyCfg {
  static constexpr int kTile = kRows * D * 2;
  static constexpr int kHalf = kRows * 128;                  // 64 channels of a tile
  static constexpr int kStages = D == 128 ? 4 : 8;           // K and V tiles in turn
  static constexpr int kBars = 1 + 2 * kStages + 10;
  // head_dim 64 leaves room for P beside S, so that the next S need not wait for this P's product
  static constexpr bool kApart = D == 64;
  static constexpr int kO = 2 * kRows, kP = kApart ? 2 * kRows + 2 * D : 0, kPStep = kApart ? 64 : kRows;  // columns
  static constexpr size_t kSmem = (size_t)(2 + kStages) * kTile + kBars * 8 + 16 + 1024;  // + alignment
};

struct ManyMaps {
  CUtensorMap q, k, v;         // boxes of a tile's rows
  CUtensorMap k8, v8;          // of 8 rows: first tokens
  CUtensorMap k_rest, v_rest;  // of what the usual first tokens leave of a tile
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    window_many_kernel(const __grid_constant__ WindowParams p, const __grid_constant__ ManyMaps maps, int firsts) {
  using C = ManyCfg<D>;
  constexpr bool kBF = !std::is_same<T, __half>::value;
  constexpr uint32_t kIdS = idesc(kBF, kRows, kRows, false), kIdO = idesc(kBF, kRows, D, true);
  extern __shared__ unsigned char smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t sQ = base, sR = base + 2 * C::kTile, bars = sR + C::kStages * C::kTile;
  const uint32_t bQ = bars, bFull = bars + 8, bFree = bFull + 8 * C::kStages, bS = bFree + 8 * C::kStages,
                 bL = bS + 16, bP = bL + 16, bP2 = bP + 16, bO = bP2 + 16, sAddr = bO + 16, sLost = sAddr + 4;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int kh = blockIdx.y, b = blockIdx.z;
  const int G = p.Hq / p.Hkv, TQ = kRows / G;                // tokens of a tile
  const int i0 = (gridDim.x - 1 - blockIdx.x) * 2 * TQ;      // first token; the last tokens first
  const WindowRow row = window_row(p, b);

  // the keys the block's rows see: slots [a0, a0 + nA) and [w0, w0 + nB), as one sequence 0 .. A8 + nB
  // with A8 = nA rounded up to 8; and each tile's share of its 128-key tiles
  int nA = 0, A8 = 0, w0 = 0, total = 0, lo[2] = {0, 0}, hi[2] = {0, 0};
  const int a0 = row.start;
  {
    int pmin[2], pmax[2];
    for (int t = 0; t < 2; ++t) {
      const int f = i0 + t * TQ, n = min(f + TQ, p.T) - 1;   // f > n: no tokens
      pmin[t] = max(row.first + f, row.start);
      pmax[t] = f > n ? -1 : min(row.first + n, row.end - 1);
      if (pmin[t] > pmax[t]) pmin[t] = 0x7fffffff, pmax[t] = -1;
    }
    const int lo_p = min(pmin[0], pmin[1]), hi_p = max(pmax[0], pmax[1]);
    if (hi_p >= 0) {
      nA = max(0, min(row.sink_end, hi_p + 1) - a0);
      A8 = (nA + 7) & ~7;
      w0 = max(a0 + nA, lo_p - p.window + 1);
      total = A8 + hi_p + 1 - w0;
      for (int t = 0; t < 2; ++t)
        if (pmax[t] >= 0) {
          lo[t] = nA > 0 ? 0 : max(0, pmin[t] - p.window + 1 - w0) / kRows;
          hi[t] = max(A8 + pmax[t] + 1 - w0, min(nA, pmax[t] + 1 - a0));
          hi[t] = (hi[t] + kRows - 1) / kRows;
        }
    }
  }
  const int n = max(hi[0], hi[1]);

  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(sAddr));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  auto load_kv = [&](int x) {  // K_0 V_0 K_1 V_1 .. of the ring
    const int s = x % C::kStages, j = x >> 1, v0 = j * kRows;
    const bool val = x & 1;
    const uint32_t dst = sR + s * C::kTile, bar = bFull + 8 * s;
    const CUtensorMap *map = val ? &maps.v : &maps.k, *map8 = val ? &maps.v8 : &maps.k8;
    const int64_t* st = val ? p.vs : p.ks;
    const int ch = st[1] ? kh : 0, cb = st[0] ? b : 0;  // shared by all heads or rows: one entry in the map
    bar_expect(bar, C::kTile);
    if (v0 + kRows <= A8 || v0 >= A8) {
      const int slot = v0 >= A8 ? w0 + v0 - A8 : a0 + v0;
      for (int h = 0; h < D / 64; ++h) tma4(dst + h * C::kHalf, map, bar, 64 * h, slot, ch, cb);
    } else {  // both runs in one tile: first tokens 8 rows at a time; the window's in one box where there are as many as usual
      const int cut = A8 - v0;
      const bool usual = A8 == firsts;
      for (int r = 0; r < (usual ? cut : kRows); r += 8) {
        const int slot = r < cut ? a0 + v0 + r : w0 + r - cut;
        for (int h = 0; h < D / 64; ++h) tma4(dst + h * C::kHalf + r * 128, map8, bar, 64 * h, slot, ch, cb);
      }
      if (usual)
        for (int h = 0; h < D / 64; ++h)
          tma4(dst + h * C::kHalf + cut * 128, val ? &maps.v_rest : &maps.k_rest, bar, 64 * h, w0, ch, cb);
    }
  };
  if (warp == 9 && lane == 0) {
    asm volatile("st.shared.u32 [%0], %1;\n" ::"r"(sLost), "r"(0u) : "memory");
    bar_init(bQ, 1);
    for (int s = 0; s < 2 * C::kStages; ++s) bar_init(bFull + 8 * s, 1);
    for (int t = 0; t < 2; ++t) {
      bar_init(bS + 8 * t, 1);
      bar_init(bL + 8 * t, kRows);
      bar_init(bP + 8 * t, kRows);
      bar_init(bP2 + 8 * t, kRows);
      bar_init(bO + 8 * t, 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    fence_proxy();
    if (n > 0) {  // the queries are on their way before the block has met
      const int nq = i0 + TQ < p.T ? 2 : 1;
      bar_expect(bQ, nq * G * TQ * D * 2);
      for (int t = 0; t < nq; ++t)
        for (int h = 0; h < D / 64; ++h)
          tma5(sQ + t * C::kTile + h * C::kHalf, &maps.q, bQ, 64 * h, 0, i0 + t * TQ, kh, p.qs[0] ? b : 0);
      load_kv(0);
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(tmem) : "r"(sAddr));
  // a wait ran out: the rest is not waited for, and the rows are done again key by key; all rows of the block where it was
  // one of warps 8 or 9, which say so in sLost
  bool lost = false;
  auto say_lost = [&] { asm volatile("st.shared.u32 [%0], %1;\n" ::"r"(sLost), "r"(1u) : "memory"); };
  auto meet = [&] {  // the block's end, from either side of the branch
    fence_before();
    asm volatile("bar.sync 1, %0;\n" ::"n"(kThreads) : "memory");
    fence_after();
  };

  // 168 registers a thread at launch, three warpgroups: 2 x 208 + 80 of the 504 they share
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;\n" ::);
    if (warp == 9) {
      if (lane == 0 && n > 0) {
        int x = 1;
        for (; x < 2 * n; ++x) {
          const int s = x % C::kStages, use = x / C::kStages;
          if (use > 0 && !bar_wait(bFree + 8 * s, (use - 1) & 1)) break;
          load_kv(x);
        }
        lost = x < 2 * n;
        // no copy outlives the block, even where warp 8 waits no more: the last one into each place of the ring
        lost |= !bar_wait(bQ, 0);
        for (int y = max(0, x - C::kStages); y < x; ++y) lost |= !bar_wait(bFull + 8 * (y % C::kStages), (y / C::kStages) & 1);
        if (lost) say_lost();
      }
      __syncwarp();
    } else if (warp == 8) {
      if (n > 0) {
        auto wait = [&](uint32_t bar, uint32_t parity) {
          if (!lost && !bar_wait(bar, parity)) lost = true;
          lost = __any_sync(0xffffffffu, lost);
          fence_after();
        };
        auto full = [&](int x) { wait(bFull + 8 * (x % C::kStages), (x / C::kStages) & 1); };
        auto issue_s = [&](int t, int j) {
          const uint64_t q = desc_k(sQ + t * C::kTile), k = desc_k(sR + (2 * j % C::kStages) * C::kTile);
#pragma unroll
          for (int e = 0; e < D / 16; ++e) {
            const uint32_t off = ((e >> 2) * C::kHalf + (e & 3) * 32) >> 4;
            mma_ss(tmem + t * kRows, q + off, k + off, kIdS, e > 0);
          }
          commit(bS + 8 * t);
        };
        // P's first three quarters are there before the last: the product begins with them
        auto issue_o = [&](int t, int j) {
          const uint64_t v = desc_mn(sR + ((2 * j + 1) % C::kStages) * C::kTile, C::kHalf);
          const uint32_t first = j > lo[t], par = (j - lo[t]) & 1;
          wait(bP + 8 * t, par);
          full(2 * j + 1);
#pragma unroll
          for (int e = 0; e < kRows / 16; ++e) {
            if (e == 6) wait(bP2 + 8 * t, par);
            mma_ts(tmem + C::kO + t * D, tmem + C::kP + t * C::kPStep + 8 * e, v + (e * 16 * 128 >> 4), kIdO, e > 0 ? 1u : first);
          }
          commit(bO + 8 * t);
        };
        auto next_s = [&](int t, int j) {
          if (j + 1 >= lo[t] && j + 1 < hi[t]) {
            if (C::kApart && j >= lo[t]) wait(bL + 8 * t, (j - lo[t]) & 1);  // this S has been read
            full(2 * j + 2);
            issue_s(t, j + 1);
          }
        };
        wait(bQ, 0);
        full(0);
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (lo[t] == 0 && hi[t] > 0) issue_s(t, 0);
        commit(bFree);
        for (int j = 0; j < n; ++j) {
          if (C::kApart) {
#pragma unroll
            for (int t = 0; t < 2; ++t) next_s(t, j);
            if (j + 1 < n) {
              full(2 * j + 2);
              commit(bFree + 8 * ((2 * j + 2) % C::kStages));
            }
          }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j >= lo[t] && j < hi[t]) issue_o(t, j);
            if (!C::kApart) next_s(t, j);
          }
          full(2 * j + 1);
          commit(bFree + 8 * ((2 * j + 1) % C::kStages));
          if (!C::kApart && j + 1 < n) {
            full(2 * j + 2);
            commit(bFree + 8 * ((2 * j + 2) % C::kStages));
          }
        }
        if (lost) say_lost();
      }
      __syncwarp();
    }
    meet();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;\n" ::);
    const int t = warp >> 2, rl = threadIdx.x & 127;
    const int token = i0 + t * TQ + rl / G, h = kh * G + rl % G;
    const bool real = rl < TQ * G && token < p.T;            // a row of the output
    const int at = row.first + token;
    // the row's keys in the block's sequence: [0, ra) and [rb0, rb1)
    int ra = 0, rb0 = -0x40000000, rb1 = 0x7fffffff;         // rows that are none see all: no mask for their sake
    if (real) {
      rb0 = rb1 = 0;
      if (at >= row.start && at < row.end) {
        ra = min(nA, at + 1 - a0);
        rb0 = A8 + max(0, at - p.window + 1 - w0);
        rb1 = A8 + at + 1 - w0;
      }
    }
    const float sl2 = p.scaling * kLog2e;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t tS = tmem + lanes + t * kRows, tO = tmem + lanes + C::kO + t * D;
    const uint32_t tP = tmem + lanes + C::kP + t * C::kPStep;
    float m = -INFINITY, l = 0.f;
    for (int j = lo[t]; j < hi[t]; ++j) {
      const int it = j - lo[t], v0 = j * kRows;
      if (!lost && !bar_wait(bS + 8 * t, it & 1)) lost = true;
      fence_after();
      uint32_t r[kRows];
#pragma unroll
      for (int c = 0; c < 4; ++c) ld32(r + 32 * c, tS + 32 * c);
      ld_wait();
      const bool whole = (rb0 <= v0 && v0 + kRows <= rb1) || v0 + kRows <= ra;
      if (C::kApart) {
        fence_before();
        bar_arrive(bL + 8 * t);
      }
      if (!__all_sync(0xffffffffu, whole)) {  // a bit for every column that the row sees
        const int ea = ra - v0, e0 = rb0 - v0, e1 = rb1 - v0;
        auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
#pragma unroll
        for (int c = 0; c < kRows; c += 32) {
          const uint32_t seen = below(ea - c) | (below(e1 - c) & ~below(e0 - c));
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(seen >> i & 1)) r[c + i] = __float_as_uint(-INFINITY);
        }
      }
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < kRows; i += 2)
        m4[(i >> 1) & 3] = fmaxf(m4[(i >> 1) & 3], fmaxf(__uint_as_float(r[i]), __uint_as_float(r[i + 1])));
      float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
      // values of slots that no row sees may be anything: they become zeros
      if ((v0 < A8 && v0 + kRows > nA) || v0 + kRows > total) {
        const int x = 2 * j + 1, v = v0 + rl;
        if (!lost && !bar_wait(bFull + 8 * (x % C::kStages), (x / C::kStages) & 1)) lost = true;
        if ((v >= nA && v < A8) || v >= total) {
          const uint32_t dst = sR + (x % C::kStages) * C::kTile + rl * 128;
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};\n" ::"r"(dst + (c >> 3) * C::kHalf + (c & 7) * 16), "r"(0u)
                         : "memory");
        }
        fence_proxy();
      }
      mx *= sl2;
      const bool grow = mx > m + 8.f || (m == -INFINITY && mx > -INFINITY);
      if (__any_sync(0xffffffffu, grow)) {
        const float f = !grow || m == -INFINITY ? 1.f : ex2(m - mx);
        if (grow) m = mx;
        l *= f;
        if (it > 0) {  // nothing to rescale before the first product
          if (!lost && !bar_wait(bO + 8 * t, (it - 1) & 1)) lost = true;
          fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            ld32(o, tO + c);
            ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            st32(tO + c, o);
          }
        }
      }
      const float mm = m == -INFINITY ? 0.f : m;
      // P = exp2(S - m), two of the multiply-adds an instruction (scalar ones: 7 % slower)
      const float2 scale2 = make_float2(sl2, sl2), shift2 = make_float2(weight_lift<T>() - mm, weight_lift<T>() - mm);
      float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      auto weigh = [&](int i) {
        float2 x = fma2(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), scale2, shift2);
        x = make_float2(ex2(x.x), ex2(x.y));
        sum2[(i >> 1) & 1] = add2(sum2[(i >> 1) & 1], x);
        r[i >> 1] = Op<T>::pack(x.x, x.y);
      };
#pragma unroll
      for (int i = 0; i < 96; i += 2) weigh(i);
      // the product of the tile before has read its P
      if (C::kApart && it > 0 && !lost && !bar_wait(bO + 8 * t, (it - 1) & 1)) lost = true;
      st32(tP, r);
      st16(tP + 32, r + 32);
      st_wait();
      fence_before();
      bar_arrive(bP + 8 * t);
#pragma unroll
      for (int i = 96; i < kRows; i += 2) weigh(i);
      l += (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
      st16(tP + 48, r + 48);
      st_wait();
      fence_before();
      bar_arrive(bP2 + 8 * t);
    }
    // O / l
    const int last = hi[t] - lo[t] - 1;
    if (last >= 0 && !lost && !bar_wait(bO + 8 * t, last & 1)) lost = true;
    fence_after();
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* o = (T*)p.out + (((int64_t)b * p.T + token) * p.Hq + h) * D;
    bool bad = lost;
#pragma unroll 1
    for (int c = 0; c < D; c += 32) {
      uint32_t x[32];
      ld32(x, tO + c);
      ld_wait();
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float y = l == 0.f ? 0.f : __uint_as_float(x[i]) * inv;
        bad |= !(fabsf(y) < INFINITY) && l == l;
        x[i] = __float_as_uint(y);
      }
      if (real) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          uint4 w;
          w.x = Op<T>::pack(__uint_as_float(x[i]), __uint_as_float(x[i + 1]));
          w.y = Op<T>::pack(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
          w.z = Op<T>::pack(__uint_as_float(x[i + 4]), __uint_as_float(x[i + 5]));
          w.w = Op<T>::pack(__uint_as_float(x[i + 6]), __uint_as_float(x[i + 7]));
          *reinterpret_cast<uint4*>(o + c + i) = w;
        }
      }
    }
    // a key that is not finite reaches the rows that do not see it as 0 * inf:
    // rows that come out not finite are done again key by key (but for those whose own scores hold a NaN or +inf, l's
    // only way to be NaN)
    meet();  // behind the stores above
    uint32_t all;
    asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(all) : "r"(sLost) : "memory");
    uint32_t again = __ballot_sync(0xffffffffu, (bad || all) && real);
    while (again) {
      const int who = __ffs(again) - 1;
      again &= again - 1;
      window_one_row<T, D>(p, row, b, __shfl_sync(0xffffffffu, h, who), __shfl_sync(0xffffffffu, token, who), lane, 0, D);
    }
  }
}

template <typename T, int D>
int launch_many(const WindowParams& p, cudaStream_t stream) {
  using C = ManyCfg<D>;
  constexpr bool kBF = !std::is_same<T, __half>::value;
  static std::atomic<uint32_t> done{0};
  const uint64_t G = p.Hq / p.Hkv, TQ = kRows / G;
  // a dimension of one entry is never stepped over, but its stride has to be a valid one
  auto count = [](int64_t stride, int64_t n) { return stride ? (uint64_t)n : (uint64_t)1; };
  auto step = [](int64_t stride, int64_t n) { return stride && n > 1 ? (uint64_t)stride * 2 : (uint64_t)16; };
  ManyMaps maps;
  {
    const uint64_t dims[5] = {(uint64_t)D, G, (uint64_t)p.T, (uint64_t)p.Hkv, count(p.qs[0], p.B)};
    const uint64_t st[4] = {step(p.qs[1], G), step(p.qs[2], p.T), step(p.qs[1] * (int64_t)G, p.Hkv), step(p.qs[0], p.B)};
    const uint32_t box[5] = {64, (uint32_t)G, (uint32_t)TQ, 1, 1};
    if (!encode(&maps.q, kBF, 5, p.q, dims, st, box)) return SKV_ERR_CUDA;
  }
  // the usual count of first tokens, rounded up as the kernel does, and what it leaves of the tile that both runs share
  const int firsts = (int)align_up(p.sinks, 8), rest = kRows - firsts % kRows;
  CUtensorMap* const out[6] = {&maps.k, &maps.v, &maps.k8, &maps.v8, &maps.k_rest, &maps.v_rest};
  for (int i = 0; i < 6; ++i) {
    const int64_t* s = i & 1 ? p.vs : p.ks;
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)p.S, count(s[1], p.Hkv), count(s[0], p.B)};
    const uint64_t st[3] = {step(s[2], p.S), step(s[1], p.Hkv), step(s[0], p.B)};
    const uint32_t box[4] = {64, i < 2 ? (uint32_t)kRows : i < 4 ? 8u : (uint32_t)rest, 1, 1};
    if (!encode(out[i], kBF, 4, i & 1 ? p.v : p.k, dims, st, box)) return SKV_ERR_CUDA;
  }
  max_smem_once(done, window_many_kernel<T, D>, (int)C::kSmem);
  const dim3 grid((unsigned)ceil_div64(p.T, 2 * TQ), p.Hkv, p.B);
  window_many_kernel<T, D><<<grid, kThreads, C::kSmem, stream>>>(p, maps, firsts);
  SKV_CHECK_LAUNCH();
  return SKV_OK;
}

}  // namespace

// Strides that a tensor map takes: below 2^40 bytes; 0 (a tensor expanded over
// its rows or kv heads) as a dimension of one entry.  A positive scale lets the
// maximum be taken before scaling.
bool window_many_supported(const WindowParams& p) {
  if ((p.D != 64 && p.D != 128) || p.Hq / p.Hkv > kRows || !(p.scaling > 0.f) || !(p.scaling < INFINITY)) return false;
  auto below = [](int64_t stride, int64_t n) { return n == 1 || stride < ((int64_t)1 << 39); };
  auto steps = [](int64_t stride, int64_t n) { return n == 1 || stride > 0; };
  return below(p.qs[0], p.B) && below(p.qs[1] * (p.Hq / p.Hkv), p.Hkv) && below(p.qs[1], p.Hq) && below(p.qs[2], p.T) &&
         below(p.ks[0], p.B) && below(p.ks[1], p.Hkv) && below(p.ks[2], p.S) && below(p.vs[0], p.B) &&
         below(p.vs[1], p.Hkv) && below(p.vs[2], p.S) && steps(p.qs[1], p.Hq) && steps(p.qs[2], p.T) &&
         steps(p.ks[2], p.S) && steps(p.vs[2], p.S);
}

int window_many(const WindowParams& p, int dtype, cudaStream_t stream) {
  if (dtype == SKV_F16)
    return p.D == 64 ? launch_many<__half, 64>(p, stream) : launch_many<__half, 128>(p, stream);
  return p.D == 64 ? launch_many<__nv_bfloat16, 64>(p, stream) : launch_many<__nv_bfloat16, 128>(p, stream);
}

}  // namespace skv
