// Attention's kernels for float16
#include "attention.h"

template int attention_forward<f16>(AttentionArgs, int64_t, int, bool, hipStream_t);
template int attention_backward<f16>(AttentionArgs, int64_t, BackwardCut, BackwardCut, hipStream_t);
