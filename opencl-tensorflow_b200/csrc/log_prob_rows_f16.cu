// The passes over rows of float16 scores.
#include "log_prob_rows.cuh"

namespace b2 {

int launch_rows_f16(cudaStream_t s, const RowArgs& a, Mode mode, bool stats, bool grad, const DeviceInfo* d,
                    const char* what) {
  return launch_rows_of<__half>(s, a, mode, stats, grad, d, what);
}

}  // namespace b2
