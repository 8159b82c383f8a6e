// Window attention with its gradients (gfx950): arguments shared by the
// kernels and their launchers.  Per window b and head h, over qkv [B, N, 3, H, D]:
//   S = scale q k^T + bias[h] + mask_b,  P = softmax(S),  out = P v
//   dP = dO v^T,  delta = rowsum(P dP) = dO . out,  dS = P (dP - delta)
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dO,  dbias[h] = sum_b dS
// A row whose scores are all -inf has P = 0: zeros out, no gradients.
#pragma once

#include <stdint.h>

#include "crumpet_common.h"

namespace crumpet {
namespace train {

enum { kNoMask = 0, kTensorMask = 1, kRegionMask = 2 };

// The shifted-window mask from the geometry: -100 between tokens of one
// window that the cyclic shift brought together from opposite ends of an axis.
struct Region {
    FastDiv plane, row;         // ws_h * ws_w, ws_w
    FastDiv grid_hw, grid_w;    // windows per plane and per row of the volume
    FastDiv windows;            // per volume
    int32_t from[3];            // first token of an axis past the seam (ws - ss)
    int32_t last[3];            // last window of an axis, -1 without a shift
};

struct AttnArgs {
    const void* qkv;            // [B, N, 3, H, D], strides sb and st, else dense
    int64_t sb, st;
    const float* bias;          // [H, N, N]
    const void* mask;           // [M, N, N], window stride mask_sb, window b reads b mod M
    int64_t mask_sb;
    int32_t mask_dtype, mode;
    uint32_t mask_batch;
    Region region;
    void* out;                  // [B, N, H, D]
    void* out_lo;               // what out's rounding left, 16-bit types only
    float* row_max;             // [B, H, N]; 0 where a row has no keys
    float* row_inv;             // [B, H, N] 1 / sum exp(S - max); 0 without keys
    const void* grad_out;       // [B, N, H, D]
    float* delta;               // [B, H, N]
    void* grad_qkv;             // [B, N, 3, H, D]
    float* grad_bias;           // [chunks, H, N, N] partial sums, or null
    uint32_t B, chunks;
    int32_t H, N;
    float scale;
};

// Per element type (attention_train_{f16,bf16,f32}.hip); D one of 16, 32, 64,
// 128.  They return a status.
int attention_forward_f16(const AttnArgs& a, int D, void* stream);
int attention_forward_bf16(const AttnArgs& a, int D, void* stream);
int attention_forward_f32(const AttnArgs& a, int D, void* stream);
int attention_backward_f16(const AttnArgs& a, int D, void* stream);
int attention_backward_bf16(const AttnArgs& a, int D, void* stream);
int attention_backward_f32(const AttnArgs& a, int D, void* stream);

}  // namespace train
}  // namespace crumpet
