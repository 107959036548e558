// The RMS norm's kernels for fp16 rows.
#include "mi_rmsnorm_kernels.hpp"

namespace mi {
namespace rms {
template void forward<MI_TYPE_F16>(const Forward&, hipStream_t);
template void backward<MI_TYPE_F16>(const Backward&, hipStream_t);
}  // namespace rms
}  // namespace mi
