// The float16 kernels of varlen_kernels.h.
#include "varlen_kernels.h"

namespace dk {
namespace varlen {

template hipError_t launch<F16>(const KParams&, const Plan&, int, bool, hipStream_t);

}  // namespace varlen
}  // namespace dk
