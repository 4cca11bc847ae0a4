// Explicit-instantiation helper of the persistent decode kernel behind a shared prefix (tails_d*.cu).
#pragma once

#include "decode_inst.cuh"

namespace b200pa {

using TailsLaunchFn = cudaError_t (*)(const DecodeParams&, const SharedPrefixParts&, int grid, int threads, size_t smem,
                                      cudaStream_t stream);

struct TailsKernelInfo {
  TailsLaunchFn fn;
  int max_warps;
  int pages_per_step;
};

template <typename QT, int KV, int D, int GP, int NT>
cudaError_t tails_launch(const DecodeParams& p, const SharedPrefixParts& pre, int grid, int threads, size_t smem,
                         cudaStream_t stream) {
  return launch_persistent<pa_decode_tails_kernel<QT, KV, D, GP, NT, decode_max_warps<KV, D, GP>()>>(grid, threads, smem,
                                                                                                stream, p, pre);
}

template <typename QT, int KV, int D>
TailsKernelInfo pick_tails(int gp, int nt) {
  constexpr int es = KV == kCache16 ? 2 : 1;
  constexpr int w1 = decode_max_warps<KV, D, 1>(), w2 = decode_max_warps<KV, D, 2>();
  if (gp == 1)
    return nt == 1 ? TailsKernelInfo{tails_launch<QT, KV, D, 1, 1>, w1, decode_pages_per_step(es, D, 1)}
                   : TailsKernelInfo{tails_launch<QT, KV, D, 1, 2>, w1, decode_pages_per_step(es, D, 2)};
  return nt == 1 ? TailsKernelInfo{tails_launch<QT, KV, D, 2, 1>, w2, decode_pages_per_step(es, D, 1)}
                 : TailsKernelInfo{tails_launch<QT, KV, D, 2, 2>, w2, decode_pages_per_step(es, D, 2)};
}

template <typename QT, int D>
TailsKernelInfo pick_tails_kv(int kv_dtype, int gp, int nt) {
  switch (kv_dtype) {
    case B200PA_KV_AUTO: return pick_tails<QT, kCache16, D>(gp, nt);
    case B200PA_KV_FP8_E4M3: return pick_tails<QT, kCacheE4M3, D>(gp, nt);
    case B200PA_KV_FP8_E5M2: return pick_tails<QT, kCacheE5M2, D>(gp, nt);
  }
  return {nullptr, 0, 1};
}

// gp: 8-head tiles per work item (1 or 2); nt: 16-token tiles per cache block (1 or 2)
template <int D>
TailsKernelInfo find_tails_for(int q_dtype, int kv_dtype, int gp, int nt) {
  if (q_dtype == B200PA_BF16) return pick_tails_kv<__nv_bfloat16, D>(kv_dtype, gp, nt);
  if (q_dtype == B200PA_F16) return pick_tails_kv<__half, D>(kv_dtype, gp, nt);
  return {nullptr, 0, 1};
}

// One finder per translation unit (defined in tails_d*.cu).
TailsKernelInfo find_tails_d32(int q_dtype, int kv_dtype, int gp, int nt);
TailsKernelInfo find_tails_d64(int q_dtype, int kv_dtype, int gp, int nt);
TailsKernelInfo find_tails_d80(int q_dtype, int kv_dtype, int gp, int nt);
TailsKernelInfo find_tails_d96(int q_dtype, int kv_dtype, int gp, int nt);
TailsKernelInfo find_tails_d112(int q_dtype, int kv_dtype, int gp, int nt);
TailsKernelInfo find_tails_d128(int q_dtype, int kv_dtype, int gp, int nt);
TailsKernelInfo find_tails_d192(int q_dtype, int kv_dtype, int gp, int nt);
TailsKernelInfo find_tails_d256(int q_dtype, int kv_dtype, int gp, int nt);

}  // namespace b200pa
