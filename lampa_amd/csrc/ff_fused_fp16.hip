// The gated feed-forward block in registers (ff_fused.h) for fp16.
#include "ff_fused.h"

int ff_fused_fwd_fp16(const lampa_ff_args* a, hipStream_t s) { return fu_fwd<_Float16>(a, s); }
int ff_fused_bwd_fp16(const lampa_ff_args* a, hipStream_t s) { return fu_bwd<_Float16>(a, s); }
