// The norms around a block: forward, whole lots (ftc_norm_kernel.h).
#include "ftc_norm_kernel.h"

namespace ftc {
namespace norm {

void norm_forward(const Args &p, const Plan &q, hipStream_t stream) { dispatch<false, false>(p, q, stream); }

}  // namespace norm
}  // namespace ftc
