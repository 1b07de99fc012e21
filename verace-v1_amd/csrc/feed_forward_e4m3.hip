// The feed-forward products over e4m3 operands.
#include "feed_forward_rows.h"

namespace vmi {
namespace prod {
int product_e4m3(Kind kind, Args p, hipStream_t stream) { return product_of<e4m3>(kind, p, stream); }
}  // namespace prod
}  // namespace vmi
