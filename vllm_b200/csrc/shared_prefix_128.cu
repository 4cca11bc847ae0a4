// Shared-prefix attention for head sizes 120, 128.
#include "shared_prefix_inst.cuh"

namespace b200pa {
SharedPrefixKernels find_shared_prefix_128(int d, int q_dtype, int kv_dtype, int group) {
  switch (d) {
    case 120: return find_shared_prefix_for<120>(q_dtype, kv_dtype, group);
    case 128: return find_shared_prefix_for<128>(q_dtype, kv_dtype, group);
  }
  return {};
}
}  // namespace b200pa
