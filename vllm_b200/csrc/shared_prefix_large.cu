// Shared-prefix attention for head sizes 192, 256.
#include "shared_prefix_inst.cuh"

namespace b200pa {
SharedPrefixKernels find_shared_prefix_large(int d, int q_dtype, int kv_dtype, int group) {
  switch (d) {
    case 192: return find_shared_prefix_for<192>(q_dtype, kv_dtype, group);
    case 256: return find_shared_prefix_for<256>(q_dtype, kv_dtype, group);
  }
  return {};
}
}  // namespace b200pa
