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
    uint32_t grid[3];           // windows per axis, region mask
    void* out;                  // [B, N, H, D]
    void* out_lo;               // what out's rounding left, 16-bit types only
    float* row_max;             // [B, H, N]; 0 where a row has no keys.  Largest score; the tuned kernels
                                // without a mask tensor keep it in units of 1 / scale
    float* row_inv;             // [B, H, N] 1 / sum exp(S - max); 0 without keys
    const void* grad_out;       // [B, N, H, D]
    float* delta;               // [B, H, N]
    void* grad_qkv;             // [B, N, 3, H, D]
    float* grad_bias;           // [chunks, H, N, N] partial sums, or null
    uint32_t B, chunks;
    int32_t H, N;
    float scale;
};

// ---- the bias-stationary kernels (attention_train_tuned.h) -------------------------

// Windows in the order of their kind.  Region classes: which axes the window
// is last on, of those that are shifted (kind t has start[t + 1] - start[t]
// windows over all volumes).  Mask tensors: the windows of mask 0, then of
// mask 1, ...
struct Order {
    uint32_t start[9];
    FastDiv per[8], hw[8], w[8];  // windows of a kind per volume, per plane, per row
    uint32_t gh, gw, windows;     // grid of a volume
    uint32_t last[3];
    FastDiv share;                // windows of one mask
};

// Workgroups: a group of row tiles of one head, and one of `ranges` ranges of
// `per` windows.
struct Walk {
    uint32_t groups, ranges, per;
};

enum TunedPass { kForwardPass, kQueryPass, kKeyPass };

// Tiles of 16 tokens that the kernels are compiled for.
constexpr int tuned_tiles(int N) {
    return N <= 64 ? 4 : N <= 128 ? 8 : N <= 224 ? 14 : N <= 352 ? 22 : 32;
}
// Strips of a workgroup, waves that share one (each with its part of the other
// axis' tiles), waves per SIMD that the registers are allotted for.  A spilled
// tile costs more than a wave: the query pass keeps 8 registers a tile, the
// others 4, and about 100 more.  Few strips to a workgroup, so that two or more
// of them fill a CU and one computes while another waits at its barrier, except
// at head dim 32, whose rows fill the LDS.  Stage 0 (22 tiles, 1372 windows, 3
// heads of 16, fp16): query pass 305 us with {2, 2, 2}, 331 with {4, 2, 2}, 435
// with {4, 1, 1}; key pass 240 with {4, 1, 2}, 264 with {6, 2, 3}; forward 236
// with {4, 1, 2}, 242 with {6, 2, 3}.
struct Form {
    int strips, split, per_simd;
};
constexpr Form tuned_form(int tiles, int D, TunedPass pass) {
    if (tiles <= 8) return {4, 1, 2};
    if (tiles == 14)
        return pass == kForwardPass ? Form{4, 2, 2} : pass == kKeyPass ? Form{7, 1, 2} : D == 16 ? Form{3, 2, 2} : Form{4, 2, 2};
    if (tiles == 22)
        return pass == kQueryPass ? (D == 16 ? Form{2, 2, 2} : Form{4, 2, 2}) : D == 16 ? Form{4, 1, 2} : Form{8, 1, 2};
    return pass == kQueryPass ? Form{2, 4, 2} : D == 32 && pass == kKeyPass ? Form{8, 1, 2} : Form{4, 2, 2};
}
Walk tuned_walk(uint32_t B, int H, int N, int D, TunedPass pass);

int attention_tuned_f16(const AttnArgs& a, const Order& o, int D, bool grad, void* stream);
int attention_tuned_f16_mask(const AttnArgs& a, const Order& o, int D, bool grad, void* stream);
int attention_tuned_bf16(const AttnArgs& a, const Order& o, int D, bool grad, void* stream);
int attention_tuned_bf16_mask(const AttnArgs& a, const Order& o, int D, bool grad, void* stream);

// ---- the general kernels (attention_train_kernels.h) -----------------------------------

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
