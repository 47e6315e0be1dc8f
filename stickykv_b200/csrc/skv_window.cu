// skv_window_attention: attention with a sliding window and first tokens that
// stay visible: argument checks and dispatch.
//
// Query at slot p of a row whose tokens sit in [start, end) sees key j when
//   start <= j <= p < end and (j - start < sinks or p - j < window),
// i.e. the runs [start, min(start + sinks, p + 1)) and
// [max(start + sinks, p - window + 1, start), p].
#include "skv_window.cuh"

namespace skv {
int window_few(const WindowParams& p, int dtype, cudaStream_t stream);
int window_f32(const WindowParams& p, cudaStream_t stream);
bool window_many_supported(const WindowParams& p);
int window_many(const WindowParams& p, int dtype, cudaStream_t stream);
namespace {

// Which kernel takes an fp16 or bf16 call: the one that is done first by these
// estimates, in ns.  Few rows: blocks of 16 rows that read every key they see,
// 40 ps a key and block (head_dim 64; 80 at 128) over the whole GPU.  Many rows:
// rounds of a block an SM, 5 us and 1.25 us a 128-key tile (1.65 where the block
// has a second tile of rows).  Measured, few/many, 32/8 heads of 64 over 4000
// keys: 1 row, 4 tokens 10/39 us, 64 tokens 28/56, 128 tokens 46/56; 16 rows, 4
// tokens 34/41, 8 tokens 54/41, 128 tokens 629/113.
bool many_is_faster(const WindowParams& p) {
  const int64_t G = p.Hq / p.Hkv, tile = 128 / G;
  auto keys = [&](int64_t tokens) {  // that so many neighbouring tokens see
    return std::min<int64_t>(p.S, (int64_t)p.sinks + p.window + std::min<int64_t>(tokens, p.T));
  };
  const int64_t groups = ceil_div64(p.T * G, 16) * p.Hkv * p.B;
  const int64_t rounds = ceil_div64(ceil_div64(p.T, 2 * tile) * p.Hkv * p.B, 148);
  const double few = 4000.0 + 0.040 * (p.D / 64.0) * groups * keys(16 / G);
  const double many = rounds * (5000.0 + ceil_div64(keys(2 * tile), 128) * (p.T > tile ? 1650.0 : 1250.0));
  return many < few;
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
  if (a->batch > 65535 || a->num_q_heads > 65535 || a->k_slots > (1 << 29) || a->q_tokens > (1 << 29))
    return SKV_ERR_UNSUPPORTED;
  // so do the (token, head) pairs of a kv head
  if ((int64_t)a->q_tokens * (a->num_q_heads / a->num_kv_heads) > 0x7fffffff) return SKV_ERR_UNSUPPORTED;
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

extern "C" int skv_window_attention(const skv_window_args* a, void* stream) {
  const int rc = check_window(a);
  if (rc) return rc;
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
  if (a->dtype == SKV_F32) return window_f32(p, s);
  if (window_many_supported(p) && many_is_faster(p)) return window_many(p, a->dtype, s);
  return window_few(p, a->dtype, s);
}
