// Entry points of the gated feed-forward block.
#include "ff_common.h"

static int ff_check(const lampa_ff_args* a) {
  if (!a || a->rows < 0 || a->D < 1 || a->F < 1 || a->dtype < 0 || a->dtype > 2 || a->activation < 0 || a->activation > 2)
    return LAMPA_ERR_INVALID;
  if (a->D % 8 || a->F % 8 || a->D > (1 << 17) || a->F > (1 << 17)) return LAMPA_ERR_UNSUPPORTED;
  // a launch takes fewer than 2^32 threads along one dimension: 512 for 256 rows, 256 for a tile of 128 rows x 64 hidden columns
  if (a->rows > ((int64_t)1 << 31) - 256 || (a->rows + 127) / 128 * ((a->F + 63) / 64) >= 1 << 24) return LAMPA_ERR_UNSUPPORTED;
  return LAMPA_OK;
}
static int ff_check_operands(const lampa_ff_args* a, int64_t size) {
  if (a->rows && (!a->x || a->x_stride < a->D)) return LAMPA_ERR_INVALID;
  if (a->rows && (a->x_stride % 8 || a->x_stride > (1 << 20))) return LAMPA_ERR_UNSUPPORTED;
  if (!a->w_gate || !a->w_up || !a->w_down) return LAMPA_ERR_INVALID;
  const uintptr_t all = (uintptr_t)a->x | (uintptr_t)a->w_gate | (uintptr_t)a->w_up | (uintptr_t)a->w_down | (uintptr_t)a->y |
                        (uintptr_t)a->dy | (uintptr_t)a->dx | (uintptr_t)a->dw_gate | (uintptr_t)a->dw_up | (uintptr_t)a->dw_down |
                        (uintptr_t)a->workspace;
  if (all % 16) return LAMPA_ERR_INVALID;
  if (size && (!a->workspace || a->workspace_bytes < size)) return LAMPA_ERR_WORKSPACE;
  return LAMPA_OK;
}

extern "C" int64_t lampa_ff_workspace_bytes(const lampa_ff_args* a, int backward) {
  const int rc = ff_check(a);
  return rc != LAMPA_OK ? rc : ff_fused_takes(a) ? ff_fused_workspace(a, backward) : ff_gemm_workspace(a, backward);
}

extern "C" int lampa_ff_fwd(const lampa_ff_args* a, void* stream) {
  const int64_t size = lampa_ff_workspace_bytes(a, 0);
  if (size < 0) return (int)size;
  const int rc = ff_check_operands(a, size);
  if (rc != LAMPA_OK) return rc;
  if (a->rows && !a->y) return LAMPA_ERR_INVALID;
  if (!a->rows) return LAMPA_OK;
  hipStream_t s = (hipStream_t)stream;
  return !ff_fused_takes(a) ? ff_gemm_fwd(a, s) : a->dtype == GDR_BF16 ? ff_fused_fwd_bf16(a, s) : ff_fused_fwd_fp16(a, s);
}

// Without rows nothing is launched: the caller clears the weights' gradients itself.
extern "C" int lampa_ff_bwd(const lampa_ff_args* a, void* stream) {
  const int64_t size = lampa_ff_workspace_bytes(a, 1);
  if (size < 0) return (int)size;
  const int rc = ff_check_operands(a, size);
  if (rc != LAMPA_OK) return rc;
  if (a->rows && !a->dy) return LAMPA_ERR_INVALID;
  if (!a->rows || (!a->dx && !a->dw_gate && !a->dw_up && !a->dw_down)) return LAMPA_OK;
  hipStream_t s = (hipStream_t)stream;
  return !ff_fused_takes(a) ? ff_gemm_bwd(a, s) : a->dtype == GDR_BF16 ? ff_fused_bwd_bf16(a, s) : ff_fused_bwd_fp16(a, s);
}
