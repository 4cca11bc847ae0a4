// Shared-prefix attention for head sizes 32, 64, 80.
#include "shared_prefix_inst.cuh"

namespace b200pa {
SharedPrefixKernels find_shared_prefix_small(int d, int q_dtype, int kv_dtype, int group) {
  switch (d) {
    case 32: return find_shared_prefix_for<32>(q_dtype, kv_dtype, group);
    case 64: return find_shared_prefix_for<64>(q_dtype, kv_dtype, group);
    case 80: return find_shared_prefix_for<80>(q_dtype, kv_dtype, group);
  }
  return {};
}
}  // namespace b200pa
