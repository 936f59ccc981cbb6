// attention_bf16.hip -- the attention operator's kernels for bf16 tensors (attention_op.h; their barriers are lds_barrier's s_barrier).
#include "attention_op.h"

namespace urf {
hipError_t attn_forward_bf16(const AttnArgs &a, int narrow, hipStream_t st) { return attn_forward_t<__bf16>(a, narrow, st); }
hipError_t attn_backward_bf16(const AttnArgs &a, hipStream_t st) { return attn_backward_t<__bf16>(a, st); }
}  // namespace urf
