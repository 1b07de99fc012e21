// The feed-forward products over bf16 operands.
#include "feed_forward_rows.h"

namespace vmi {
namespace prod {
int product_bf16(Kind kind, Args p, hipStream_t stream) { return product_of<__bf16>(kind, p, stream); }
}  // namespace prod
}  // namespace vmi
