// Explicit-instantiation helper of the two kernels of shared-prefix attention (shared_prefix_*.cu).
#pragma once

#include "direct_inst.cuh"
#include "prefill_inst.cuh"
#include "shared_prefix_kernel.cuh"

namespace b200pa {

struct SharedPrefixKernels {
  // the prefix, `grid` CTAs (num_heads: query heads)
  cudaError_t (*prefix)(const SharedPrefixParams&, int num_heads, int grid, cudaStream_t stream) = nullptr;
  // what is behind it: `items` clusters
  cudaError_t (*behind)(const DecodeParams&, const SharedPrefixParts&, int items, int cluster, cudaStream_t stream) = nullptr;
  // ... where a warp takes whole items
  cudaError_t (*solo)(const DecodeParams&, const SharedPrefixParts&, int items, cudaStream_t stream) = nullptr;
  int heads = 0;        // query heads of an item of `behind`
  int ctas_per_sm = 0;  // of `behind`
  int row_tiles = 0;    // that share a K/V tile
  int keys = 0;         // of a tile
  int part_bytes = 0;   // of a row tile in the scratch
};

template <typename QT, int KV, int D>
cudaError_t shared_prefix_launch(const SharedPrefixParams& p, int num_heads, int grid, cudaStream_t stream) {
  auto kern = pa_shared_prefix_kernel<QT, KV, D>;
  constexpr int smem = PrefillShape<D>::kSmem;
  static bool done[64] = {};  // opted in to large dynamic shared memory, per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !done[dev]) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();  // do not leave the error for the next caller
      return e;
    }
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  // (the maps of the prefill kernel: a sequence is a token there)
  PrefillParams m{};
  m.q = p.q;
  m.vc = p.vc;
  m.q_stride = p.q_stride;
  m.kv_block_stride = p.kv_block_stride;
  m.kv_head_stride = p.kv_head_stride;
  m.num_tokens = p.num_seqs;
  m.num_heads = num_heads;
  m.num_kv_heads = p.num_kv_heads;
  m.group = p.group;
  m.block_size = p.block_size;
  CUtensorMap qmap, vmap = {};
  e = prefill_q_map(m, D, PrefillShape<D>::kQBox, &qmap);
  if (KV == kCache16 && e == cudaSuccess) e = prefill_v_map(m, D, &vmap);
  if (e != cudaSuccess) return e;
  return launch_dependent(kern, dim3(grid), dim3(kPrefillThreads), smem, stream, p, qmap, vmap);
}

template <typename QT, int KV, int D, int GP>
cudaError_t behind_launch(const DecodeParams& p, const SharedPrefixParts& pre, int items, int cluster, cudaStream_t stream) {
  return launch_clusters<pa_decode_behind_kernel<QT, KV, D, GP>, DirectShape<KV, D, GP>::kSmem>(items, cluster, stream, p, pre);
}

template <typename QT, int KV, int D, int GP>
cudaError_t solo_launch(const DecodeParams& p, const SharedPrefixParts& pre, int items, cudaStream_t stream) {
  constexpr int smem = DirectShape<KV, D, GP>::kSmem;
  auto kern = pa_decode_solo_kernel<QT, KV, D, GP>;
  if constexpr (smem > 40 * 1024) {
    static bool done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= 64 || !done[dev])) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
    }
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return e;
    }
  }
  return launch_dependent(kern, dim3((items + kDirectWarps - 1) / kDirectWarps), dim3(kDirectWarps * 32), smem, stream, p, pre,
                          items);
}

template <typename QT, int KV, int D>
SharedPrefixKernels shared_prefix_kernels(int group) {
  SharedPrefixKernels k;
  k.prefix = shared_prefix_launch<QT, KV, D>;
  k.behind = behind_launch<QT, KV, D, 1>;
  k.solo = solo_launch<QT, KV, D, 1>;
  k.heads = 8;
  k.ctas_per_sm = DirectShape<KV, D, 1>::kResident;
  if constexpr (D <= 128) {
    if (group > 8) {
      k.behind = behind_launch<QT, KV, D, 2>;
      k.solo = solo_launch<QT, KV, D, 2>;
      k.heads = 16;
      k.ctas_per_sm = DirectShape<KV, D, 2>::kResident;
    }
  }
  k.row_tiles = PrefillShape<D>::NQ;
  k.keys = PrefillShape<D>::KT;
  k.part_bytes = shared_prefix_part_bytes(D);
  return k;
}

template <typename QT, int D>
SharedPrefixKernels find_shared_prefix_kv(int kv_dtype, int group) {
  if (kv_dtype == B200PA_KV_AUTO) return shared_prefix_kernels<QT, kCache16, D>(group);
  if constexpr (D % 16 == 0) {
    if (kv_dtype == B200PA_KV_FP8_E4M3) return shared_prefix_kernels<QT, kCacheE4M3, D>(group);
    if (kv_dtype == B200PA_KV_FP8_E5M2) return shared_prefix_kernels<QT, kCacheE5M2, D>(group);
  }
  return {};
}

// group: query heads per kv head
template <int D>
SharedPrefixKernels find_shared_prefix_for(int q_dtype, int kv_dtype, int group) {
  if (q_dtype == B200PA_BF16) return find_shared_prefix_kv<__nv_bfloat16, D>(kv_dtype, group);
  if (q_dtype == B200PA_F16) return find_shared_prefix_kv<__half, D>(kv_dtype, group);
  return {};
}

// Defined in shared_prefix_small.cu (32 .. 80), _mid.cu (96, 112), _128.cu (120, 128), _large.cu (192, 256).
SharedPrefixKernels find_shared_prefix_small(int d, int q_dtype, int kv_dtype, int group);
SharedPrefixKernels find_shared_prefix_mid(int d, int q_dtype, int kv_dtype, int group);
SharedPrefixKernels find_shared_prefix_128(int d, int q_dtype, int kv_dtype, int group);
SharedPrefixKernels find_shared_prefix_large(int d, int q_dtype, int kv_dtype, int group);

}  // namespace b200pa
