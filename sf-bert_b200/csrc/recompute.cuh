// The backward pass that makes the probabilities again: what the C ABI (ops.cu), the rows' constants and the two paths share.
#pragma once
#include "attn.cuh"

namespace sfb {

struct BackwardArgs {
    const void *nt_lut, *nn_lut, *tn_lut, *q, *k, *v, *o, *dout, *mask;
    void *dq, *dk, *dv;
    int dtype;
    uint32_t bs, nt_stride;                               // nt_stride: uint2 per head of the nt_lut; p.lut_stride that of the other two
    uint32_t nn_max, tn_max;
    uint64_t in_pitch, o_pitch, do_pitch, grad_pitch;     // none is 0
    float scale;
    AttnDims p;
};

int attention_row_constants(cudaStream_t s, const void *o, const void *dout, const float *lse, float *neg_lse, float *neg_delta, int dtype, uint32_t B,
                            uint32_t L, uint32_t H, uint32_t d, uint64_t o_pitch, uint64_t do_pitch, float scale);
uint64_t simt_backward_workspace(int dtype, uint32_t bs, uint32_t nb, uint32_t blocks, uint32_t B, uint32_t H);
int simt_backward_recompute(cudaStream_t s, const BackwardArgs &a, float *neg_lse, float *neg_delta, void *blocks_ws);


// tcgen05 (attn_tc_recompute.cu): 16-bit operands, 64x64 blocks, 64-wide heads
bool tc_backward_recompute_supported(int dtype, uint32_t bs, const AttnDims &p, uint32_t nn_max, uint32_t tn_max);
int tc_backward_recompute(cudaStream_t s, const BackwardArgs &a, const float *neg_lse, const float *neg_delta);
int tc_status_recompute(uint32_t *out);
int tc_status_clear_recompute();

}  // namespace sfb
