// The end of the few-row window kernels: a block's warps join their shares of a
// row group, then the blocks of its cluster, through distributed shared memory;
// and the launch that splits the keys over clusters.
#pragma once

#include <type_traits>

#include "skv_mma.cuh"
#include "skv_window_rows.cuh"

namespace skv {

constexpr int window_pitch(int D) { return D + 4; }  // floats a partial row: 16-byte rows, banks apart
constexpr size_t window_part_bytes(int D, int rows, int warps) { return (size_t)warps * rows * window_pitch(D) * 4; }
constexpr size_t window_stat_bytes(int rows, int warps) { return (size_t)(warps + 1) * rows * 2 * 4; }

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// part [warp][row][pitch]: sums of weights times values; stat [warp + 1][row]:
// their maxima (log2), then the same of the sums of weights.
template <typename T, int D, int kRows, int kWarps>
__device__ __forceinline__ void window_join(const WindowParams& p, const WindowRow& row, int b, int kh, int r0, int rows,
                                            int split, int splits, float* part, float* stat) {
  using mma::smem_u32;
  // the hardware's exponential is off by 2^-22, too much beside float32 results
  auto ex2 = [](float x) { return std::is_same<T, float>::value ? exp2f(x) : mma::ex2(x); };
  constexpr int kPitch = window_pitch(D);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.Hq / p.Hkv;
  __syncthreads();
  // the block's warps join into warp 0's place
  const int n_out = rows * D;
  for (int x = threadIdx.x; x < n_out; x += kWarps * 32) {
    const int r = x / D, d = x % D;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, stat[w * kRows + r]);
    float sum = 0.f, val = 0.f;
    if (mx != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(stat[w * kRows + r] - mx);
        sum += f * stat[(kWarps + 1 + w) * kRows + r];
        val += f * part[(size_t)w * kRows * kPitch + r * kPitch + d];
      }
    } else {  // no score above -inf: the sums are 0, but NaN where a score was (a maximum passes over those)
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += stat[(kWarps + 1 + w) * kRows + r];
    }
    part[r * kPitch + d] = val;
    if (d == 0) {
      stat[kWarps * kRows + r] = mx;
      stat[(2 * kWarps + 1) * kRows + r] = sum;
    }
  }
  if (splits > 1) cluster_sync();
  else __syncthreads();
  // and the cluster's blocks: each writes every splits-th row slice
  bool repair = false;
  const int per = ceil_div(n_out, splits);
  const uint32_t s_part = smem_u32(part), s_stat = smem_u32(stat);
  for (int y = threadIdx.x; y < per; y += kWarps * 32) {
    const int x = split * per + y;
    if (x >= n_out) break;
    const int r = x / D, d = x % D;
    float mx = -INFINITY, sum = 0.f, val = 0.f;
    if (splits == 1) {
      sum = stat[(2 * kWarps + 1) * kRows + r];
      val = part[r * kPitch + d];
    } else {
      for (int z = 0; z < splits; ++z) {
        const float mz = ld_cluster(s_stat + (kWarps * kRows + r) * 4, z);
        const float lz = ld_cluster(s_stat + ((2 * kWarps + 1) * kRows + r) * 4, z);
        const float vz = ld_cluster(s_part + (r * kPitch + d) * 4, z);
        if (mz == -INFINITY) {
          sum += lz;  // 0 or NaN, as above
          continue;
        }
        const float mn = fmaxf(mx, mz), f0 = ex2(mx - mn), f1 = ex2(mz - mn);
        sum = sum * f0 + lz * f1;
        val = val * f0 + vz * f1;
        mx = mn;
      }
    }
    const float res = sum == 0.f ? 0.f : val / sum;
    // (a sum of NaN is a NaN or +inf among the row's own scores, and NaN its answer; in float32 also an infinite channel,
    // whose two terms make a NaN of any score)
    repair |= !(fabsf(res) < INFINITY) && (sum == sum || std::is_same<T, float>::value);
    const int rr = r0 + r;
    st_f32((T*)p.out + (((int64_t)b * p.T + rr / G) * p.Hq + kh * G + rr % G) * D + d, res);
  }
  // a key that is not finite reaches the rows that do not see it as 0 * inf:
  // rows that come out not finite are done again key by key
  const int again = __syncthreads_or(repair);
  if (again) {
    for (int r = warp; r < rows; r += kWarps) {
      const int rr = r0 + r;
      if (r * D / per <= split && (r * D + D - 1) / per >= split)
        window_one_row<T, D>(p, row, b, kh * G + rr % G, rr / G, lane, split * per - r * D, (split + 1) * per - r * D);
    }
  }
  if (splits > 1) cluster_sync();  // no block leaves while others read its share
}

// What a kernel's limits were raised to, by device (as max_smem_once).
struct WindowFewState {
  std::atomic<uint32_t> smem{0}, wide{0};
};

template <typename K>
int launch_window_few(const WindowParams& p, K kernel, WindowFewState& state, int rows, int warps, int blocks_per_sm,
                      size_t smem, cudaStream_t stream) {
  max_smem_once(state.smem, kernel, (int)smem);
  const int G = p.Hq / p.Hkv;
  const int64_t groups = ceil_div64((int64_t)p.T * G, rows);
  const int64_t blocks = groups * p.Hkv * p.B;
  const int64_t tiles = ceil_div64(std::min<int64_t>(p.S, (int64_t)p.sinks + p.window + ceil_div(rows, G)), 16);
  // splits: as long as all blocks are resident at once and every warp has a tile
  int splits = 1;
  while (splits < 16 && blocks * splits * 2 <= blocks_per_sm * 148 && (int64_t)splits * 2 * warps <= tiles) splits *= 2;
  if (groups * splits > 0x7fffffff) return SKV_ERR_UNSUPPORTED;
  if (splits > 8) {
    int dev = 0;
    cudaGetDevice(&dev);
    const uint32_t bit = dev < 32 ? 1u << dev : 0u;
    if (!bit || !(state.wide.load(std::memory_order_relaxed) & bit)) {
      cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      state.wide.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(groups * splits), p.Hkv, p.B);
  cfg.blockDim = dim3(warps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, splits);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return SKV_ERR_CUDA;
  }
  return SKV_OK;
}

}  // namespace skv
