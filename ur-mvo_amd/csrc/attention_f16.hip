// attention_f16.hip -- the attention operator's kernels for f16 tensors (attention_op.h; their barriers are lds_barrier's s_barrier).
#include "attention_op.h"

namespace urf {
hipError_t attn_forward_f16(const AttnArgs &a, int narrow, hipStream_t st) { return attn_forward_t<_Float16>(a, narrow, st); }
hipError_t attn_backward_f16(const AttnArgs &a, hipStream_t st) { return attn_backward_t<_Float16>(a, st); }
}  // namespace urf
