// Attention under interval masks: the forward under a window with sinks.
#include "attn_masked_fwd.cuh"

int ma_launch_window_fwd(const MaParams& p, void* ws, long long ws_bytes, cudaStream_t s) {
  return p.d <= 64 ? launch_fwd<64, true>(p, ws, ws_bytes, s) : launch_fwd<128, true>(p, ws, ws_bytes, s);
}

extern "C" int lb_window_attn_status(void* out) { return read_status(out); }
