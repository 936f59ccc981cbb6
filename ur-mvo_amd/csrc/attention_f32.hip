// attention_f32.hip -- the attention operator's kernels for f32 tensors (attention_op.h; their barriers are lds_barrier's s_barrier).
#include "attention_op.h"

namespace urf {
hipError_t attn_forward_f32(const AttnArgs &a, int narrow, hipStream_t st) { return attn_forward_t<float>(a, narrow, st); }
hipError_t attn_backward_f32(const AttnArgs &a, hipStream_t st) { return attn_backward_t<float>(a, st); }
}  // namespace urf
