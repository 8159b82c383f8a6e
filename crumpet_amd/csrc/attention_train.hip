// Window attention with gradients: argument checks, the choice of kernels and
// the C ABI (kernels: attention_train_kernels.h).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention_train.h"
#include "crumpet_hip.h"

namespace crumpet {
namespace train {
namespace {

constexpr int kThreads = 256;

// out[i] = sum over the chunks of partial[chunk][i], in order
__global__ void __launch_bounds__(kThreads)
join_kernel(float* __restrict__ out, const float* __restrict__ partial, int64_t n, uint32_t chunks) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= n) return;
    float v = 0.0f;
#pragma unroll 4
    for (uint32_t c = 0; c < chunks; ++c) v += partial[c * n + i];
    out[i] = v;
}

// Partial sums of dbias: enough that about 1024 workgroups share the windows,
// within 256 MB.
uint32_t bias_chunks(int64_t B, int64_t H, int64_t N) {
    const int64_t blocks = H * ((N + 63) / 64) * ((N + 63) / 64);
    const int64_t most = std::max<int64_t>(1, (int64_t(256) << 20) / (H * N * N * 4));
    return static_cast<uint32_t>(std::max<int64_t>(1, std::min(std::min(B, most), (1024 + blocks - 1) / blocks)));
}

int64_t rounded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// The bias-stationary kernels: 16-bit types, head dims 16 and 32, up to 512
// tokens.  Without a mask tensor they fold the scale into the bias, which
// needs a scale whose inverse is an ordinary number.  Offsets in a window's rows
// take 32 bits there.  Forward and gradients, against the general kernels: 1372
// windows of 343 tokens, three heads of 16, 794 us for 1753; 1000 of 27, six heads
// of 16, 68 for 122; 4 of 216, 24 heads of 16, 51 for 61; one of 27 and one head
// 13 for 17; 64 masks of 343, six heads of 32, 221 for 431.  (Of small calls the
// forward pass alone is 1 to 5 us slower, but both passes share the statistics.)
bool use_tuned(const AttnArgs& a, int32_t dtype, int64_t D) {
    if (a.st < 0 || a.st >= int64_t(1) << 21 || a.H > 4096) return false;
    const bool folds = a.scale >= 0x1p-20f && a.scale <= 0x1p20f;
    return dtype != CRUMPET_DTYPE_F32 && (D == 16 || D == 32) && a.N <= 512 &&
           (a.mode == kTensorMask ? a.N >= 2 : folds);  // four neighbours of a mask matrix are read at once
}

int check(AttnArgs& a, int32_t dtype, int64_t B, int64_t H, int64_t N, int64_t D, const int64_t strides[2],
          const float* bias, const void* mask, int32_t mask_dtype, int64_t mask_batch, int64_t mask_stride,
          const int64_t* region, float scale, const char* what) {
    if (dtype < 0 || dtype > 2 || (mask != nullptr && (mask_dtype < 0 || mask_dtype > 2)))
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: unknown dtype code", what);
    if (B < 0 || H < 0 || N < 0) return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: negative size", what);
    if (D != 16 && D != 32 && D != 64 && D != 128)
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: head_dim %lld is not 16, 32, 64 or 128", what, (long long)D);
    if (N > 16384 || H > 4096 || B >= (int64_t(1) << 31))
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: more than 16384 tokens, 4096 heads or 2^31 windows", what);
    if (!launch_takes(static_cast<uint64_t>(B) * H * ((N + 15) / 16) + kNumXcd, kThreads) ||
        !launch_takes((static_cast<uint64_t>(H) * N * N + kThreads - 1) / kThreads, kThreads))
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: too many windows, heads or tokens for one launch", what);
    if (B == 0 || H == 0 || N == 0) return CRUMPET_OK;
    if (bias == nullptr) return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: null bias", what);
    if (mask != nullptr && region != nullptr)
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: a mask tensor and a shifted volume exclude each other", what);
    const int64_t align = 16 / (dtype == CRUMPET_DTYPE_F32 ? 4 : 2);
    if (strides[0] % align != 0 || strides[1] % align != 0)
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: qkv rows must be 16-byte aligned", what);
    a.sb = strides[0], a.st = strides[1], a.bias = bias, a.scale = scale;
    a.B = static_cast<uint32_t>(B), a.H = static_cast<int32_t>(H), a.N = static_cast<int32_t>(N);
    a.chunks = bias_chunks(B, H, N);
    if (mask != nullptr) {
        if (mask_batch < 1 || B % mask_batch != 0)
            return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: the windows (%lld) must be a multiple of the masks (%lld)",
                        what, (long long)B, (long long)mask_batch);
        a.mode = kTensorMask, a.mask = mask, a.mask_dtype = mask_dtype;
        a.mask_batch = static_cast<uint32_t>(mask_batch), a.mask_sb = mask_stride;
    }
    if (region != nullptr) {
        const int64_t *volume = region, *ws = region + 3, *ss = region + 6;
        int64_t nw[3];
        for (int i = 0; i < 3; ++i) {
            if (ws[i] < 1 || volume[i] < 1 || volume[i] % ws[i] != 0)
                return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: the volume must be divisible by window_size", what);
            if (ss[i] < 0 || ss[i] >= ws[i])
                return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: shift_size must lie in [0, window_size)", what);
            nw[i] = volume[i] / ws[i];
            if (ws[i] > N || nw[i] > B) break;
        }
        if (ws[0] > N || ws[1] > N || ws[2] > N || ws[0] * ws[1] * ws[2] != N)
            return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: N = %lld is not the window volume", what, (long long)N);
        if (nw[0] > B || nw[1] > B || nw[2] > B || nw[0] * nw[1] > B || B % (nw[0] * nw[1] * nw[2]) != 0)
            return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: the windows (%lld) must be a multiple of the volume's", what,
                        (long long)B);
        Region& r = a.region;
        r.plane.init(static_cast<uint32_t>(ws[1] * ws[2]));
        r.row.init(static_cast<uint32_t>(ws[2]));
        r.grid_hw.init(static_cast<uint32_t>(nw[1] * nw[2]));
        r.grid_w.init(static_cast<uint32_t>(nw[2]));
        r.windows.init(static_cast<uint32_t>(nw[0] * nw[1] * nw[2]));
        for (int i = 0; i < 3; ++i) {
            r.from[i] = static_cast<int32_t>(ws[i] - ss[i]);
            r.last[i] = ss[i] > 0 ? static_cast<int32_t>(nw[i] - 1) : -1;
        }
        if (ss[0] > 0 || ss[1] > 0 || ss[2] > 0) {
            a.mode = kRegionMask;
            for (int i = 0; i < 3; ++i) a.grid[i] = static_cast<uint32_t>(nw[i]);
        }
    }
    if (use_tuned(a, dtype, D)) a.chunks = tuned_walk(a.B, a.H, a.N, static_cast<int>(D), kQueryPass).ranges;
    return CRUMPET_OK;
}

Order order_of(const AttnArgs& a) {
    Order o;
    o.share.init(a.mode == kTensorMask ? a.B / a.mask_batch : 1);
    // without a mask: one kind, one row of windows
    uint32_t n[3] = {1, 1, a.B};
    bool shifted[3] = {};
    if (a.mode == kRegionMask) {
        for (int i = 0; i < 3; ++i) n[i] = a.grid[i], shifted[i] = a.region.last[i] >= 0;
    }
    o.gh = n[1], o.gw = n[2], o.windows = n[0] * n[1] * n[2];
    const uint32_t volumes = a.B / o.windows;
    o.start[0] = 0;
    for (uint32_t t = 0; t < 8; ++t) {
        uint32_t m[3];
        for (int i = 0; i < 3; ++i) m[i] = t >> i & 1 ? (shifted[i] ? 1 : 0) : shifted[i] ? n[i] - 1 : n[i];
        const uint32_t count = m[0] * m[1] * m[2];
        o.start[t + 1] = o.start[t] + count * volumes;
        o.per[t].init(std::max(1u, count));
        o.hw[t].init(std::max(1u, m[1] * m[2]));
        o.w[t].init(std::max(1u, m[2]));
    }
    for (int i = 0; i < 3; ++i) o.last[i] = n[i] - 1;
    return o;
}

int run_tuned(const AttnArgs& a, int32_t dtype, int D, bool grad, void* stream) {
    const Order o = order_of(a);
    if (a.mode == kTensorMask)
        return dtype == CRUMPET_DTYPE_F16 ? attention_tuned_f16_mask(a, o, D, grad, stream)
                                          : attention_tuned_bf16_mask(a, o, D, grad, stream);
    return dtype == CRUMPET_DTYPE_F16 ? attention_tuned_f16(a, o, D, grad, stream)
                                      : attention_tuned_bf16(a, o, D, grad, stream);
}

bool misaligned(std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return true;
    return false;
}

}  // namespace

// As many ranges as keep every CU's workgroups in one round.
Walk tuned_walk(uint32_t B, int H, int N, int D, TunedPass pass) {
    const Form f = tuned_form(tuned_tiles(N), D, pass);
    const uint32_t tiles = static_cast<uint32_t>((N + 15) / 16);
    Walk w;
    w.groups = (tiles + f.strips - 1) / f.strips;
    const uint32_t units = w.groups * static_cast<uint32_t>(H);
    // workgroups that a CU holds: by waves and by LDS (rows, the strips' sums, the key pass' statistics)
    const int rows = tuned_tiles(N) * 16, values = D / 4 * (pass == kKeyPass ? 2 : 1) + 2;
    const int lds = 8 * rows * D + 512 * f.strips * (f.split - 1) * values + (pass == kKeyPass ? 32 * rows : rows);
    const uint32_t resident = std::max(1, std::min(4 * f.per_simd / (f.strips * f.split), 163840 / lds));
    const uint32_t ranges = std::max(1u, std::min(B, 256 * resident / units));
    w.per = (B + ranges - 1) / ranges;
    w.ranges = (B + w.per - 1) / w.per;
    return w;
}

}  // namespace train
}  // namespace crumpet

using namespace crumpet;
using namespace crumpet::train;

extern "C" int crumpet_window_attention(void* out, void* out_rest, float* row_max, float* row_inv, const void* qkv,
                                        const int64_t qkv_strides[2], int32_t dtype, int64_t B, int64_t heads,
                                        int64_t N, int64_t head_dim, const float* bias, const void* mask,
                                        int32_t mask_dtype, int64_t mask_batch, int64_t mask_stride,
                                        const int64_t* region, float scale, void* stream) {
    const char* what = "window_attention";
    AttnArgs a = {};
    const int st = train::check(a, dtype, B, heads, N, head_dim, qkv_strides, bias, mask, mask_dtype, mask_batch,
                                mask_stride, region, scale, what);
    if (st != CRUMPET_OK || B == 0 || heads == 0 || N == 0) return st;
    if (out == nullptr || qkv == nullptr || (row_max == nullptr) != (row_inv == nullptr))
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: null tensor", what);
    if (misaligned({out, out_rest, qkv}))
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: pointers must be 16-byte aligned", what);
    a.out = out, a.out_lo = out_rest, a.row_max = row_max, a.row_inv = row_inv, a.qkv = qkv;
    const int D = static_cast<int>(head_dim);
    if (use_tuned(a, dtype, D)) return run_tuned(a, dtype, D, false, stream);
    if (dtype == CRUMPET_DTYPE_F16) return attention_forward_f16(a, D, stream);
    if (dtype == CRUMPET_DTYPE_BF16) return attention_forward_bf16(a, D, stream);
    return attention_forward_f32(a, D, stream);
}

extern "C" int64_t crumpet_window_attention_workspace(int64_t B, int64_t heads, int64_t N) {
    if (B < 0 || heads < 0 || N < 0 || B >= (int64_t(1) << 31) || heads > 4096 || N > 16384) return -1;
    if (B == 0 || heads == 0 || N == 0) return 0;
    uint32_t chunks = bias_chunks(B, heads, N);
    for (int D = 16; D <= 32 && N <= 512; D *= 2)
        chunks = std::max(chunks, tuned_walk(static_cast<uint32_t>(B), static_cast<int>(heads), static_cast<int>(N), D,
                                             kQueryPass).ranges);
    return rounded(B * heads * N * 4) + chunks * heads * N * N * 4;
}

extern "C" int crumpet_window_attention_backward(void* grad_qkv, float* grad_bias, const void* grad_out, const void* out,
                                                 const void* out_rest, const float* row_max, const float* row_inv,
                                                 const void* qkv, const int64_t qkv_strides[2], int32_t dtype,
                                                 int64_t B, int64_t heads, int64_t N, int64_t head_dim,
                                                 const float* bias, const void* mask, int32_t mask_dtype,
                                                 int64_t mask_batch, int64_t mask_stride, const int64_t* region,
                                                 float scale, void* workspace, void* stream) {
    const char* what = "window_attention_backward";
    AttnArgs a = {};
    const int st = train::check(a, dtype, B, heads, N, head_dim, qkv_strides, bias, mask, mask_dtype, mask_batch,
                                mask_stride, region, scale, what);
    if (st != CRUMPET_OK || B == 0 || heads == 0 || N == 0) return st;
    if (grad_qkv == nullptr || grad_out == nullptr || out == nullptr || row_max == nullptr || row_inv == nullptr ||
        qkv == nullptr || workspace == nullptr || (dtype != CRUMPET_DTYPE_F32 && out_rest == nullptr))
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: null tensor", what);
    if (misaligned({grad_qkv, grad_out, out, out_rest, qkv, workspace}))
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: pointers must be 16-byte aligned", what);
    a.out = const_cast<void*>(out), a.out_lo = const_cast<void*>(out_rest), a.qkv = qkv;
    a.row_max = const_cast<float*>(row_max), a.row_inv = const_cast<float*>(row_inv);
    a.grad_out = grad_out, a.grad_qkv = grad_qkv;
    char* ws = static_cast<char*>(workspace);
    a.delta = reinterpret_cast<float*>(ws);
    float* partial = reinterpret_cast<float*>(ws + rounded(B * heads * N * 4));
    if (grad_bias != nullptr) a.grad_bias = a.chunks == 1 ? grad_bias : partial;
    const int D = static_cast<int>(head_dim);
    int rc;
    if (use_tuned(a, dtype, D)) rc = run_tuned(a, dtype, D, true, stream);
    else if (dtype == CRUMPET_DTYPE_F16) rc = attention_backward_f16(a, D, stream);
    else if (dtype == CRUMPET_DTYPE_BF16) rc = attention_backward_bf16(a, D, stream);
    else rc = attention_backward_f32(a, D, stream);
    if (rc != CRUMPET_OK || grad_bias == nullptr || a.chunks == 1) return rc;
    const int64_t n = heads * N * N;
    join_kernel<<<static_cast<uint32_t>((n + kThreads - 1) / kThreads), kThreads, 0, static_cast<hipStream_t>(stream)>>>(
        grad_bias, partial, n, a.chunks);
    return check_launch(what);
}
