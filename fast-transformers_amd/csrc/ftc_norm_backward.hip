// The norms around a block: backward, whole lots (ftc_norm_kernel.h).
#include "ftc_norm_kernel.h"

namespace ftc {
namespace norm {

void norm_backward(const Args &p, const Plan &q, hipStream_t stream) { dispatch<true, false>(p, q, stream); }

}  // namespace norm
}  // namespace ftc
