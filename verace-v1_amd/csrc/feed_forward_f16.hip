// The feed-forward products over f16 operands.
#include "feed_forward_rows.h"

namespace vmi {
namespace prod {
int product_f16(Kind kind, Args p, hipStream_t stream) { return product_of<_Float16>(kind, p, stream); }
}  // namespace prod
}  // namespace vmi
