// The feed-forward products' kernels for f32 operands (feed_forward.h).
#define FPN_FF_INSTANTIATE
#include "feed_forward_few.h"

namespace fpn {
namespace ff {

template int launch_wide<float>(const Args &, int, int, bool, int, int, long, hipStream_t);
template int launch_few<float>(const Args &, int, bool, int, int, hipStream_t);
template int launch_product<float>(Args, int, int, bool, const Plan &, float *, hipStream_t);

}  // namespace ff
}  // namespace fpn
