// The attention kernels over caches of one pair of types: QS_KV_BITS is the bits
// of a key's code times ten and those of a value's (88, 84, 48, 44), so that the
// four compile in parallel.
#include "qs_kv_attention_kernels.h"

namespace qskv {

template hipError_t launch_attention<QS_KV_BITS / 10, QS_KV_BITS % 10>(const AttentionArgs&, const Split&, hipStream_t);

}  // namespace qskv
