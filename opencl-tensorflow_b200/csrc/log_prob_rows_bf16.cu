// The passes over rows of bfloat16 scores.
#include "log_prob_rows.cuh"

namespace b2 {

int launch_rows_bf16(cudaStream_t s, const RowArgs& a, Mode mode, bool stats, bool grad, const DeviceInfo* d,
                     const char* what) {
  return launch_rows_of<__nv_bfloat16>(s, a, mode, stats, grad, d, what);
}

}  // namespace b2
