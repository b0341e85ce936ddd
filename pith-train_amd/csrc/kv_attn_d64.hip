// Attention of new tokens to the rows of a key-value cache: heads of 64 features (see kv_attn.h).
#include "kv_attn.h"

namespace pith {

void launch_kv_attn_d64(const KVAttnParams& p, bool fp8, int row_groups, int workgroups, hipStream_t s) { launch_kv_attn<64>(p, fp8, row_groups, workgroups, s); }

}  // namespace pith
