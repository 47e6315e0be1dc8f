// skv_window_attention: attention with a sliding window and first tokens that
// stay visible (argument checks, dispatch and the portable kernel).
//
// Query at slot p of a row whose tokens sit in [start, end) sees key j when
//   start <= j <= p < end and (j - start < sinks or p - j < window),
// i.e. the runs [start, min(start + sinks, p + 1)) and
// [max(start + sinks, p - window + 1, start), p].
#include "skv_window.cuh"

namespace skv {
namespace {

// One warp per query, lanes over the channels, online softmax in fp32.
template <typename T, int D>
__global__ void __launch_bounds__(128) window_rows_kernel(const WindowParams p) {
  constexpr int E = D < 32 ? 1 : D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x * 4 + warp, h = blockIdx.y, b = blockIdx.z;
  if (i >= p.T) return;
  const WindowRow row = window_row(p, b);
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
  for (int e = 0; e < E; ++e)
    if (lane + 32 * e < D) st_f32(o + lane + 32 * e, l == 0.f ? 0.f : acc[e] / l);
}

template <typename T>
int launch_rows(const WindowParams& p, cudaStream_t stream) {
  const dim3 grid(ceil_div(p.T, 4), p.Hq, p.B);
  switch (p.D) {
    case 16: window_rows_kernel<T, 16><<<grid, 128, 0, stream>>>(p); break;
    case 32: window_rows_kernel<T, 32><<<grid, 128, 0, stream>>>(p); break;
    case 64: window_rows_kernel<T, 64><<<grid, 128, 0, stream>>>(p); break;
    default: window_rows_kernel<T, 128><<<grid, 128, 0, stream>>>(p); break;
  }
  SKV_CHECK_LAUNCH();
  return SKV_OK;
}

int check_window(const skv_window_args* a) {
  if (!a) return SKV_ERR_INVALID_ARG;
  if (a->batch <= 0 || a->q_tokens <= 0 || a->k_slots <= 0 || a->num_q_heads <= 0 || a->num_kv_heads <= 0)
    return SKV_ERR_INVALID_ARG;
  if (a->num_q_heads % a->num_kv_heads || a->window < 1 || a->sinks < 0) return SKV_ERR_INVALID_ARG;
  if (!a->q || !a->k || !a->v || !a->out) return SKV_ERR_INVALID_ARG;
  if (a->head_dim != 16 && a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) return SKV_ERR_UNSUPPORTED;
  const int es = a->dtype == SKV_F32 ? 4 : (a->dtype == SKV_F16 || a->dtype == SKV_BF16) ? 2 : 0;
  if (!es) return SKV_ERR_UNSUPPORTED;
  // heads and rows index grid dimensions; slots and queries 31-bit sums
  if (a->batch > 65535 || a->num_q_heads > 65535 || a->k_slots > (1 << 30) || a->q_tokens > (1 << 30))
    return SKV_ERR_UNSUPPORTED;
  const void* ptrs[4] = {a->q, a->k, a->v, a->out};
  for (const void* x : ptrs)
    if ((uintptr_t)x % 16) return SKV_ERR_MISALIGNED;
  for (int i = 0; i < 3; ++i) {
    if (a->q_stride[i] < 0 || a->k_stride[i] < 0 || a->v_stride[i] < 0) return SKV_ERR_INVALID_ARG;
    if ((a->q_stride[i] * es) % 16 || (a->k_stride[i] * es) % 16 || (a->v_stride[i] * es) % 16)
      return SKV_ERR_MISALIGNED;
  }
  const int32_t* lists[3] = {a->starts, a->ends, a->query_slots};
  for (const int32_t* x : lists)
    if ((uintptr_t)x % 4) return SKV_ERR_MISALIGNED;
  return SKV_OK;
}

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" size_t skv_window_workspace_size(const skv_window_args* a) {
  if (check_window(a)) return 0;
  return 0;
}

extern "C" int skv_window_attention(const skv_window_args* a, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check_window(a);
  if (rc) return rc;
  const size_t need = skv_window_workspace_size(a);
  if (need && (!ws || ws_bytes < need)) return SKV_ERR_WORKSPACE;
  if (need && (uintptr_t)ws % 256) return SKV_ERR_MISALIGNED;
  WindowParams p{};
  p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i];
  }
  p.starts = a->starts; p.ends = a->ends; p.slots = a->query_slots;
  p.B = a->batch; p.T = a->q_tokens; p.S = a->k_slots; p.Hq = a->num_q_heads; p.Hkv = a->num_kv_heads;
  p.D = a->head_dim;
  // a window of every slot or more is no window (keeps slot arithmetic in 31 bits)
  p.window = a->window < a->k_slots ? a->window : a->k_slots;
  p.sinks = a->sinks < a->k_slots ? a->sinks : a->k_slots;
  p.scaling = a->scaling;
  const cudaStream_t s = (cudaStream_t)stream;
  switch (a->dtype) {
    case SKV_F32: return launch_rows<float>(p, s);
    case SKV_F16: return launch_rows<__half>(p, s);
    default: return launch_rows<__nv_bfloat16>(p, s);
  }
}
