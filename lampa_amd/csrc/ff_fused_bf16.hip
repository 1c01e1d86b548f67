// The gated feed-forward block in registers (ff_fused.h) for bf16.
#include "ff_fused.h"

int64_t ff_fused_workspace(const lampa_ff_args* a, int backward) { return fu_workspace(a, backward); }
int ff_fused_fwd_bf16(const lampa_ff_args* a, hipStream_t s) { return fu_fwd<__bf16>(a, s); }
int ff_fused_bwd_bf16(const lampa_ff_args* a, hipStream_t s) { return fu_bwd<__bf16>(a, s); }
