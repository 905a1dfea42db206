// The norms around a block: backward, rows of any width (ftc_norm_kernel.h).
#include "ftc_norm_kernel.h"

namespace ftc {
namespace norm {

void norm_backward_tail(const Args &p, const Plan &q, hipStream_t stream) { dispatch<true, true>(p, q, stream); }

}  // namespace norm
}  // namespace ftc
