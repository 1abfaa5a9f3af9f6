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
    float scale, inside;                                  // inside: scale_inside()
    AttnDims p;
};

// dS is an operand of 16 bits as P * (dP - delta) * inside, and dQ and dK are multiplied by what is left of the softmax scale, scale / inside, in
// fp32.  fp16 has no normal numbers below 2^-14, where most of dS of a long row or of a small loss is: multiplied by a scale of 1/8 first it loses
// three bits more (the norm of dQ's errors, 2048 causal positions, d 64, dO of 2^-5 3.6e-4 with the scale in dS and 2.9e-4 without, 2^-8 1.7e-3 and
// 3.6e-4, 2^-12 2.8e-2 and 3.7e-3; rows of 2048 keys 7.1e-4 and 3.0e-4, 5.4e-3 and 7.3e-4, 8.4e-2 and 1.1e-2).  A scale above 1 in magnitude goes in,
// for the same reason.  fp32 has the range for either; there inside is the scale.
inline float scale_inside(int dtype, float scale) { return dtype == SFB_F32 ? scale : scale > 1.f ? scale : scale < -1.f ? -scale : 1.f; }

int attention_row_constants(cudaStream_t s, const void *o, const void *dout, const float *lse, float *neg_lse, float *neg_delta, int dtype, uint32_t B,
                            uint32_t L, uint32_t H, uint32_t d, uint64_t o_pitch, uint64_t do_pitch, float inside);
uint64_t simt_backward_workspace(int dtype, uint32_t bs, uint32_t nb, uint32_t blocks, uint32_t B, uint32_t H);
int simt_backward_recompute(cudaStream_t s, const BackwardArgs &a, float *neg_lse, float *neg_delta, void *blocks_ws);

// tcgen05 (attn_tc_recompute.cu): 16-bit operands, 64x64 blocks, 64-wide heads
bool tc_backward_recompute_supported(int dtype, uint32_t bs, const AttnDims &p, uint32_t nn_max, uint32_t tn_max);
int tc_backward_recompute(cudaStream_t s, const BackwardArgs &a, const float *neg_lse, const float *neg_delta);
int tc_status_recompute(uint32_t *out);
int tc_status_clear_recompute();

}  // namespace sfb
