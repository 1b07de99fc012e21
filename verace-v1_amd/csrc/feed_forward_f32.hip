// The feed-forward products over f32 operands.
#include "feed_forward_rows.h"

namespace vmi {
namespace prod {
int product_f32(Kind kind, Args p, hipStream_t stream) { return product_of<float>(kind, p, stream); }
}  // namespace prod
}  // namespace vmi
