// Attention under interval masks: the forward without a window.
#include "attn_masked_fwd.cuh"

long long ma_fwd_ws_bytes(const MaParams& p) { return fwd_ws_bytes(p); }

int ma_launch_fwd(const MaParams& p, void* ws, long long ws_bytes, cudaStream_t s) {
  return p.d <= 64 ? launch_fwd<64, false>(p, ws, ws_bytes, s) : launch_fwd<128, false>(p, ws, ws_bytes, s);
}

extern "C" int lb_masked_attn_status(void* out) { return read_status(out); }
