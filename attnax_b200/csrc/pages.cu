// Page operators of the paged KV cache.
#include "attn_common.cuh"
#include "host_util.h"
#include "sm100.cuh"

namespace attnb200 {
bool pages_take_status(int* status, int* notice) { return take_status_words(status, notice); }
}  // namespace attnb200
