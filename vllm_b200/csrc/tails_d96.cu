// The persistent decode kernel behind a shared prefix for head size 96.
#include "tails_inst.cuh"

namespace b200pa {
TailsKernelInfo find_tails_d96(int q_dtype, int kv_dtype, int gp, int nt) {
  return find_tails_for<96>(q_dtype, kv_dtype, gp, nt);
}
}  // namespace b200pa
