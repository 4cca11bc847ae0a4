// The persistent decode kernel behind a shared prefix for head size 256.
#include "tails_inst.cuh"

namespace b200pa {
TailsKernelInfo find_tails_d256(int q_dtype, int kv_dtype, int gp, int nt) {
  return find_tails_for<256>(q_dtype, kv_dtype, gp, nt);
}
}  // namespace b200pa
