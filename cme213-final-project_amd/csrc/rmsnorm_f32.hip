// The RMS norm's kernels for fp32 rows.
#include "mi_rmsnorm_kernels.hpp"

namespace mi {
namespace rms {
template void forward<MI_TYPE_F32>(const Forward&, hipStream_t);
template void backward<MI_TYPE_F32>(const Backward&, hipStream_t);
}  // namespace rms
}  // namespace mi
