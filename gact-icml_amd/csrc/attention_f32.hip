// Attention's kernels for float
#include "attention.h"

template int attention_forward<float>(AttentionArgs, int64_t, int, bool, hipStream_t);
template int attention_backward<float>(AttentionArgs, int64_t, BackwardCut, BackwardCut, hipStream_t);
