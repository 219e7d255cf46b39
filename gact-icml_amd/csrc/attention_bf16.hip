// Attention's kernels for bfloat16
#include "attention.h"

template int attention_forward<bf16>(AttentionArgs, int64_t, int, bool, hipStream_t);
template int attention_backward<bf16>(AttentionArgs, int64_t, BackwardCut, BackwardCut, hipStream_t);
