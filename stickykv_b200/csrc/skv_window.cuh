// Parameters and row bounds shared by the window-attention kernels.
#pragma once

#include <type_traits>

#include "skv_common.cuh"

namespace skv {

struct WindowParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;                   // [B][T][Hq][D]
  int64_t qs[3], ks[3], vs[3]; // batch, head, token (elements)
  const int32_t* starts;
  const int32_t* ends;
  const int32_t* slots;
  int B, T, S, Hq, Hkv, D, window, sinks;
  float scaling;
};

struct WindowRow {
  int start, end;   // the row's tokens, clamped to the slots there are
  int sink_end;     // one past its last always-visible token
  int first;        // slot of query 0
};

__device__ __forceinline__ WindowRow window_row(const WindowParams& p, int b) {
  WindowRow r;
  r.start = p.starts ? min(max(p.starts[b], 0), p.S) : 0;
  r.end = p.ends ? min(max(p.ends[b], 0), p.S) : p.S;
  r.sink_end = min(r.start + p.sinks, r.end);
  // slots further out than any key or query make no difference: keeps sums in 32 bits
  r.first = p.slots ? min(max(p.slots[b], -(1 << 30)), p.S) : r.end - p.T;
  return r;
}

// Weights 2^(score - m) go to fp16 times 2^7: up to 2^15 (m lags by 2^8 at
// most), and the subnormals, whose step is a constant, begin at 2^-21 of the
// largest in place of 2^-14.  The factor cancels in the quotient.
template <typename T> __device__ constexpr float weight_lift() { return std::is_same<T, __half>::value ? 7.f : 0.f; }

}  // namespace skv
