// The norms around a block: forward, rows of any width (ftc_norm_kernel.h).
#include "ftc_norm_kernel.h"

namespace ftc {
namespace norm {

void norm_forward_tail(const Args &p, const Plan &q, hipStream_t stream) { dispatch<false, true>(p, q, stream); }

}  // namespace norm
}  // namespace ftc
