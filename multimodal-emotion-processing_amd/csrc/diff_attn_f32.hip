// The differential-attention kernels in MEP_F32.
#include "diff_attn.h"

void mep::da_run_f32(int what, const mep_diff_attn_desc& d, const mep_diff_attn_bwd_desc* b, unsigned grid, int blocks, int splits, hipStream_t st, int all, uint64_t sizes, int parts) {
    da_run<MEP_F32>(what, d, b, grid, blocks, splits, st, all, sizes, parts);
}
