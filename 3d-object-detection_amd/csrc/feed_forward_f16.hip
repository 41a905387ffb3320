// The feed-forward products' kernels for f16 operands (feed_forward.h).
#define FPN_FF_INSTANTIATE
#include "feed_forward_few.h"

namespace fpn {
namespace ff {

template int launch_wide<_Float16>(const Args &, int, int, bool, int, int, long, hipStream_t);
template int launch_few<_Float16>(const Args &, int, bool, int, int, hipStream_t);
template int launch_product<_Float16>(Args, int, int, bool, const Plan &, float *, hipStream_t);

}  // namespace ff
}  // namespace fpn
