// Shared-prefix attention for head sizes 96, 112.
#include "shared_prefix_inst.cuh"

namespace b200pa {
SharedPrefixKernels find_shared_prefix_mid(int d, int q_dtype, int kv_dtype, int group) {
  switch (d) {
    case 96: return find_shared_prefix_for<96>(q_dtype, kv_dtype, group);
    case 112: return find_shared_prefix_for<112>(q_dtype, kv_dtype, group);
  }
  return {};
}
}  // namespace b200pa
