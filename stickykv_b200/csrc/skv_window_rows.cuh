// One row of window attention by one warp, key by key: what the tensor-core
// kernels fall back to for rows that come out not finite (so that keys a row
// does not see never reach it).
#pragma once

#include "skv_window.cuh"

namespace skv {

// Lanes over the channels, online softmax in fp32.  Writes channels [d0, d1).
template <typename T, int D>
__device__ __forceinline__ void window_one_row(const WindowParams& p, const WindowRow& row, int b, int h, int i,
                                            int lane, int d0, int d1) {
  constexpr int E = D < 32 ? 1 : D / 32;
  const int pos = row.first + i, kh = h / (p.Hq / p.Hkv);
  const T* q = (const T*)p.q + b * p.qs[0] + h * p.qs[1] + i * p.qs[2];
  const T* kb = (const T*)p.k + b * p.ks[0] + kh * p.ks[1];
  const T* vb = (const T*)p.v + b * p.vs[0] + kh * p.vs[1];
  float qr[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qr[e] = lane + 32 * e < D ? ld_f32(q + lane + 32 * e) : 0.f;
    acc[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  auto attend = [&](int j0, int j1) {
    for (int j = j0; j < j1; ++j) {
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (lane + 32 * e < D) dot += qr[e] * ld_f32(kb + j * p.ks[2] + lane + 32 * e);
      const float s = warp_sum(dot) * p.scaling;
      if (s == -INFINITY) continue;  // weighs nothing (and would be -inf - -inf below)
      const float mn = fmaxf(m, s);
      const float alpha = expf(m - mn), pr = expf(s - mn);
      l = l * alpha + pr;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (lane + 32 * e < D) acc[e] = acc[e] * alpha + pr * ld_f32(vb + j * p.vs[2] + lane + 32 * e);
      m = mn;
    }
  };
  if (pos >= row.start && pos < row.end) {
    const int sink_end = min(row.sink_end, pos + 1);
    attend(row.start, sink_end);
    attend(max(sink_end, pos - p.window + 1), pos + 1);
  }
  T* o = (T*)p.out + (((int64_t)b * p.T + i) * p.Hq + h) * D;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 32 * e;
    if (d < D && d >= d0 && d < d1) st_f32(o + d, l == 0.f ? 0.f : acc[e] / l);
  }
}

}  // namespace skv
