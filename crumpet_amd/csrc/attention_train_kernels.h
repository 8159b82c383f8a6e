// General kernels of the window attention with gradients: any N, head dims 16
// to 128, fp32, fp16 and bf16, every mask form.  One template per element type
// (attention_train_{f16,bf16,f32}.hip).
//
// A workgroup of 4 waves owns one (window, head) and 64 rows, 16 per wave, and
// walks the other axis in chunks staged in LDS.  The forward pass and dq own
// queries and compute S^T = K Q^T (a lane holds 4 keys of one query); dk and
// dv own keys and compute S = Q K^T (4 queries of one key).  Either way the
// lane's P and dS are the B operand of the products that follow, and the A
// operands are LDS transpose reads of the staged rows.  dbias owns a 64 x 64
// tile of one head and walks the windows, so that its sums stay in registers.
//
// Scores, softmax, delta and dS are fp32; P and dS are rounded to the input
// type only as operands of the products whose results are rounded to it too.
// dbias sums the unrounded dS, and delta enters it in fp32: for training the
// product P v takes P as its rounded value and the rest, and out is kept with
// its rest (round_and_rest).  dbias is then off by 3e-7 in fp16 and 3 to 9e-7
// in bf16; with P rounded once it is 2e-5 and 2e-4.
//
// Rows, and the bias before them, are requested a chunk or window ahead: with 16
// windows of 1000 tokens and six heads of 128 in bf16 the four kernels take 210,
// 231, 498 and 245 us for 297, 314, 632 and 416.
//
// Measured on 64 windows of 343 tokens and six heads of 16 in fp32: forward 60
// us, dq 74, dk and dv 119, dbias 79.  fp32 products (154 TFLOP/s at the most)
// and the softmax share the issue slots: matrix cores 44, 54, 43 and 40% busy,
// VALU 52, 51, 36 and 46%.
#pragma once

#include <algorithm>

#include "attention_train.h"
#include "train_mma.h"

namespace crumpet {
namespace train {
namespace {

constexpr int kThreads = 256;

template <typename T, int D>
struct Tile {
    static constexpr int kRows = sizeof(T) * D >= 512 ? 32 : 64;  // staged rows per chunk
    static constexpr int kLd = D + 16 / static_cast<int>(sizeof(T));
    static constexpr int kSlices = D / 16;
};

// Region class of a token: which seams it lies past, of those its window has.
__device__ __forceinline__ uint32_t seams(const Region& r, uint32_t b) {
    uint32_t q, win, wd, rest, wh, ww;
    r.windows.divmod(b, q, win);
    r.grid_hw.divmod(win, wd, rest);
    r.grid_w.divmod(rest, wh, ww);
    return (static_cast<int>(wd) == r.last[0] ? 1u : 0u) | (static_cast<int>(wh) == r.last[1] ? 2u : 0u) |
           (static_cast<int>(ww) == r.last[2] ? 4u : 0u);
}
__device__ __forceinline__ uint32_t token_class(const Region& r, uint32_t seam, uint32_t token) {
    uint32_t d, rest, h, w;
    r.plane.divmod(token, d, rest);
    r.row.divmod(rest, h, w);
    const uint32_t past = (static_cast<int>(d) >= r.from[0] ? 1u : 0u) | (static_cast<int>(h) >= r.from[1] ? 2u : 0u) |
                          (static_cast<int>(w) >= r.from[2] ? 4u : 0u);
    return past & seam;
}

// Four neighbours at any address: one wide load, at any alignment of an element.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Four {
    T v[4];
};

// What one (window, head) adds to a score.
struct Terms {
    const float* bias;   // [N, N] of the head
    const void* mask;    // the tensor
    int64_t mask_at;     // first element of the window's mask
    uint32_t seam;

    __device__ __forceinline__ Terms(const AttnArgs& a, uint32_t b, int h)
        : bias(a.bias + static_cast<int64_t>(h) * a.N * a.N), mask(a.mask), mask_at(0), seam(0) {
        if (a.mode == kTensorMask) mask_at = static_cast<int64_t>(b % a.mask_batch) * a.mask_sb;
        if (a.mode == kRegionMask) seam = seams(a.region, b);
    }
    // The bias of query q and keys k .. k + 3, and of queries q .. q + 3 and key
    // k; read before a chunk's scores and before the next chunk's rows are
    // requested, since loads come back in order.
    __device__ __forceinline__ f32x4 of_row(const AttnArgs& a, int q, int k) const {
        const float* at = bias + static_cast<uint32_t>(q * a.N + k);  // N^2 is below 2^29
        f32x4 v = {};
        if (k + 4 <= a.N) {
            const Four<float> b = *reinterpret_cast<const Four<float>*>(at);
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = b.v[r];
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (k + r < a.N) v[r] = at[r];
        }
        return v;
    }
    __device__ __forceinline__ f32x4 of_column(const AttnArgs& a, int q, int k) const {
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = bias[static_cast<uint32_t>((q + r < a.N ? q + r : a.N - 1) * a.N + k)];
        return v;
    }
    // Scores of query q and keys k .. k + 3; keys past N are -inf.  b: their bias,
    // cls: the region classes of the keys.
    __device__ __forceinline__ f32x4 of_query(const AttnArgs& a, f32x4 qk, f32x4 b, int q, int k, uint32_t cq,
                                              const uint32_t* cls) const {
        const int64_t at = static_cast<int64_t>(q) * a.N + k;
        f32x4 s;
        if (k + 4 <= a.N) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] = __builtin_fmaf(qk[r], a.scale, b[r]);
            if (a.mode == kTensorMask) {
                if (a.mask_dtype == CRUMPET_DTYPE_F32) add<float>(s, at);
                else if (a.mask_dtype == CRUMPET_DTYPE_F16) add<_Float16>(s, at);
                else add<__bf16>(s, at);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[r] = -__builtin_inff();
                if (k + r >= a.N) continue;
                s[r] = __builtin_fmaf(qk[r], a.scale, b[r]);
                if (a.mode == kTensorMask) s[r] += load_float(mask, a.mask_dtype, mask_at + at + r);
            }
        }
        if (seam) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] -= cq != cls[r] ? 100.0f : 0.0f;
        }
        return s;
    }
    // Scores of queries q .. q + 3 and key k; rows past N are anything.
    __device__ __forceinline__ f32x4 of_key(const AttnArgs& a, f32x4 qk, f32x4 b, int q, int k, const uint32_t* cls,
                                            uint32_t ck) const {
        f32x4 s;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t at = static_cast<int64_t>(q + r < a.N ? q + r : a.N - 1) * a.N + k;
            s[r] = __builtin_fmaf(qk[r], a.scale, b[r]);
            if (a.mode == kTensorMask) s[r] += load_float(mask, a.mask_dtype, mask_at + at);
            if (seam) s[r] -= ck != cls[r] ? 100.0f : 0.0f;
        }
        return s;
    }

private:
    template <typename M>
    __device__ __forceinline__ void add(f32x4& s, int64_t at) const {
        const Four<M> m = *reinterpret_cast<const Four<M>*>(static_cast<const M*>(mask) + mask_at + at);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] += static_cast<float>(m.v[r]);
    }
};

template <typename T>
__device__ __forceinline__ const T* token_row(const AttnArgs& a, uint32_t b, int token, int which, int h, int D) {
    return static_cast<const T*>(a.qkv) + static_cast<int64_t>(b) * a.sb + static_cast<int64_t>(token) * a.st +
           (static_cast<int64_t>(which) * a.H + h) * D;
}

// Rows row0 .. row0 + kRows - 1 (those past N repeat the last one) on their way
// into LDS: requested a chunk ahead, stored when the chunk before is done.
template <typename T, int D>
struct Staged {
    typedef Tile<T, D> L;
    static constexpr int kPieces = D / 4, kEach = L::kRows * kPieces / kThreads;
    static_assert(kEach * kThreads == L::kRows * kPieces);
    typename Mma<T>::x4 v[kEach];
    __device__ __forceinline__ void fetch(const T* first, int64_t stride, int row0, int N) {
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            const int i = threadIdx.x + u * kThreads, row = row0 + i / kPieces;
            v[u] = load4<T>(first + (row < N ? row : N - 1) * stride + i % kPieces * 4);
        }
    }
    __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            const int i = threadIdx.x + u * kThreads;
            *reinterpret_cast<typename Mma<T>::x4*>(lds + i / kPieces * L::kLd + i % kPieces * 4) = v[u];
        }
    }
};

template <typename T, int D>
struct Rows {  // a lane's fragments of 16 rows: row col, columns 16 s + 4 g ..
    typename Mma<T>::x4 v[D / 16];
    __device__ __forceinline__ void load(const T* row, int g) {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) v[s] = load4<T>(row + 16 * s + 4 * g);
    }
};

// rows row0 .. + 15 of the staged tile (A) times the lane's rows (B)
template <typename T, int D>
__device__ __forceinline__ f32x4 product(const T* lds, int row0, const Rows<T, D>& b, int col, int g) {
    f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
        c = Mma<T>::mma16(load4<T>(lds + (row0 + col) * Tile<T, D>::kLd + 16 * s + 4 * g), b.v[s], c);
    return c;
}

// acc[d][lane's row] += staged rows row0 .. + 15 transposed (A) times w (B)
template <typename T, int D>
__device__ __forceinline__ void accumulate(f32x4* acc, const T* lds, int row0, typename Mma<T>::x4 w, int col, int g) {
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
        acc[s] = Mma<T>::mma16(load_transposed<T>(lds, Tile<T, D>::kLd, row0, 16 * s, col, g), w, acc[s]);
}

__device__ __forceinline__ float weight(float s, float top) { return __builtin_amdgcn_exp2f((s - top) * kLog2e); }

// (window, head, block) of a workgroup; blocks of one (window, head) share an XCD
__device__ __forceinline__ bool owner(const AttnArgs& a, uint32_t blocks, uint32_t& b, int& h, uint32_t& block) {
    uint32_t chunk;
    const uint32_t all = a.B * static_cast<uint32_t>(a.H) * blocks;
    if (!xcd_chunk(blockIdx.x, gridDim.x, all, chunk)) return false;
    block = chunk % blocks;
    const uint32_t bh = chunk / blocks;
    h = static_cast<int>(bh % a.H);
    b = bh / a.H;
    return true;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attn_forward_kernel(const AttnArgs a, uint32_t blocks) {
    typedef Tile<T, D> L;
    __shared__ __attribute__((aligned(16))) T k_lds[L::kRows * L::kLd];
    __shared__ __attribute__((aligned(16))) T v_lds[L::kRows * L::kLd];
    __shared__ uint32_t cls[L::kRows];
    uint32_t b, block;
    int h;
    if (!owner(a, blocks, b, h, block)) return;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int q0 = static_cast<int>(block) * 64 + (threadIdx.x >> 6) * 16 + col;
    const int q = q0 < a.N ? q0 : a.N - 1;
    const Terms terms(a, b, h);
    const uint32_t cq = terms.seam ? token_class(a.region, terms.seam, q) : 0;
    Rows<T, D> qr;
    qr.load(token_row<T>(a, b, q, 0, h, D), g);
    f32x4 acc[L::kSlices] = {};
    float top = -__builtin_inff(), total = 0.0f;
    const T *k_at = token_row<T>(a, b, 0, 1, h, D), *v_at = token_row<T>(a, b, 0, 2, h, D);
    Staged<T, D> ks, vs;
    ks.fetch(k_at, a.st, 0, a.N), vs.fetch(v_at, a.st, 0, a.N);
    for (int k0 = 0; k0 < a.N; k0 += L::kRows) {
        __syncthreads();
        ks.store(k_lds), vs.store(v_lds);
        if (threadIdx.x < L::kRows)
            cls[threadIdx.x] = terms.seam && k0 + static_cast<int>(threadIdx.x) < a.N
                                   ? token_class(a.region, terms.seam, k0 + threadIdx.x) : 0;
        __syncthreads();
        f32x4 bias[L::kRows / 16];
#pragma unroll
        for (int t = 0; t < L::kRows / 16; ++t) bias[t] = terms.of_row(a, q, k0 + 16 * t + 4 * g);
        if (k0 + L::kRows < a.N) {
            ks.fetch(k_at, a.st, k0 + L::kRows, a.N);
            vs.fetch(v_at, a.st, k0 + L::kRows, a.N);
        }
        f32x4 s[L::kRows / 16];
        float high = top;
#pragma unroll
        for (int t = 0; t < L::kRows / 16; ++t) {
            const int i = 16 * t + 4 * g;
            s[t] = terms.of_query(a, product<T, D>(k_lds, 16 * t, qr, col, g), bias[t], q, k0 + i, cq, cls + i);
#pragma unroll
            for (int r = 0; r < 4; ++r) high = fmaxf(high, s[t][r]);
        }
        high = max_groups(high);
        // a row without keys so far: exp(-inf - 0) = 0
        const float used = high == -__builtin_inff() ? 0.0f : high;
        const float fade = weight(top, used);
        top = high;
        total *= fade;
#pragma unroll
        for (int d = 0; d < L::kSlices; ++d) acc[d] *= fade;
#pragma unroll
        for (int t = 0; t < L::kRows / 16; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[t][r] = weight(s[t][r], used);
                total += s[t][r];
            }
            const typename Mma<T>::x4 hi = round4<T>(s[t]);
            accumulate<T, D>(acc, v_lds, 16 * t, hi, col, g);
            if constexpr (sizeof(T) == 2) {
                if (a.out_lo != nullptr)
                    accumulate<T, D>(acc, v_lds, 16 * t, round4<T>(s[t] - wide4<T>(hi)), col, g);
            }
        }
    }
    total = sum_groups(total);
    if (q0 >= a.N) return;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int64_t at = (static_cast<int64_t>(b) * a.N + q) * a.H + h;
#pragma unroll
    for (int d = 0; d < L::kSlices; ++d) {
        typename Mma<T>::x4 hi, lo;
        round_and_rest<T>(acc[d] * inv, hi, lo);
        *reinterpret_cast<typename Mma<T>::x4*>(static_cast<T*>(a.out) + at * D + 16 * d + 4 * g) = hi;
        if constexpr (sizeof(T) == 2) {
            if (a.out_lo != nullptr)
                *reinterpret_cast<typename Mma<T>::x4*>(static_cast<T*>(a.out_lo) + at * D + 16 * d + 4 * g) = lo;
        }
    }
    if (g == 0 && a.row_max != nullptr) {
        const int64_t row = (static_cast<int64_t>(b) * a.H + h) * a.N + q;
        a.row_max[row] = top == -__builtin_inff() ? 0.0f : top;
        a.row_inv[row] = inv;
    }
}

// dO . out over the lane's row.  out comes as its rounded value and the rest:
// the rounding alone (2^-9 in bf16) would show in the fp32 sums of dbias.
template <typename T, int D>
__device__ __forceinline__ float row_delta(const AttnArgs& a, int64_t at, const Rows<T, D>& go, int g) {
    Rows<T, D> o, lo;
    o.load(static_cast<const T*>(a.out) + at * D, g);
    if constexpr (sizeof(T) == 2) lo.load(static_cast<const T*>(a.out_lo) + at * D, g);
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x;
            if constexpr (sizeof(T) == 2)
                x = with_rest<T>(o.v[s][e], lo.v[s][e]);
            else
                x = o.v[s][e];
            sum = __builtin_fmaf(x, static_cast<float>(go.v[s][e]), sum);
        }
    }
    return sum_groups(sum);
}

// dq, and delta for the kernels after it.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attn_grad_q_kernel(const AttnArgs a, uint32_t blocks) {
    typedef Tile<T, D> L;
    __shared__ __attribute__((aligned(16))) T k_lds[L::kRows * L::kLd];
    __shared__ __attribute__((aligned(16))) T v_lds[L::kRows * L::kLd];
    __shared__ uint32_t cls[L::kRows];
    uint32_t b, block;
    int h;
    if (!owner(a, blocks, b, h, block)) return;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int q0 = static_cast<int>(block) * 64 + (threadIdx.x >> 6) * 16 + col;
    const int q = q0 < a.N ? q0 : a.N - 1;
    const Terms terms(a, b, h);
    const uint32_t cq = terms.seam ? token_class(a.region, terms.seam, q) : 0;
    const int64_t at = (static_cast<int64_t>(b) * a.N + q) * a.H + h;
    const int64_t row = (static_cast<int64_t>(b) * a.H + h) * a.N + q;
    Rows<T, D> qr, go;
    qr.load(token_row<T>(a, b, q, 0, h, D), g);
    go.load(static_cast<const T*>(a.grad_out) + at * D, g);
    const float delta = row_delta<T, D>(a, at, go, g);
    const float top = a.row_max[row], inv = a.row_inv[row];
    f32x4 acc[L::kSlices] = {};
    const T *k_at = token_row<T>(a, b, 0, 1, h, D), *v_at = token_row<T>(a, b, 0, 2, h, D);
    Staged<T, D> ks, vs;
    // Not in fp32: its rows' registers cost a wave (64 windows of 343 tokens, six
    // heads of 16: 80 us for 72).  fp16, heads of 64: 95 us for 128.
    constexpr bool kAhead = sizeof(T) == 2;
    if constexpr (kAhead) ks.fetch(k_at, a.st, 0, a.N), vs.fetch(v_at, a.st, 0, a.N);
    for (int k0 = 0; k0 < a.N; k0 += L::kRows) {
        if constexpr (!kAhead) ks.fetch(k_at, a.st, k0, a.N), vs.fetch(v_at, a.st, k0, a.N);
        __syncthreads();
        ks.store(k_lds), vs.store(v_lds);
        if (threadIdx.x < L::kRows)
            cls[threadIdx.x] = terms.seam && k0 + static_cast<int>(threadIdx.x) < a.N
                                   ? token_class(a.region, terms.seam, k0 + threadIdx.x) : 0;
        __syncthreads();
        f32x4 bias[L::kRows / 16];
        if constexpr (kAhead) {
#pragma unroll
            for (int t = 0; t < L::kRows / 16; ++t) bias[t] = terms.of_row(a, q, k0 + 16 * t + 4 * g);
            if (k0 + L::kRows < a.N) {
                ks.fetch(k_at, a.st, k0 + L::kRows, a.N);
                vs.fetch(v_at, a.st, k0 + L::kRows, a.N);
            }
        }
#pragma unroll
        for (int t = 0; t < L::kRows / 16; ++t) {
            const int i = 16 * t + 4 * g;
            if constexpr (!kAhead) bias[t] = terms.of_row(a, q, k0 + i);
            f32x4 s = terms.of_query(a, product<T, D>(k_lds, 16 * t, qr, col, g), bias[t], q, k0 + i, cq, cls + i);
            const f32x4 dp = product<T, D>(v_lds, 16 * t, go, col, g);
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] = k0 + i + r < a.N ? weight(s[r], top) * inv * (dp[r] - delta) : 0.0f;
            accumulate<T, D>(acc, k_lds, 16 * t, round4<T>(s), col, g);
        }
    }
    if (q0 >= a.N) return;
    T* to = static_cast<T*>(a.grad_qkv) + ((static_cast<int64_t>(b) * a.N + q) * 3 * a.H + h) * D;
#pragma unroll
    for (int d = 0; d < L::kSlices; ++d)
        *reinterpret_cast<typename Mma<T>::x4*>(to + 16 * d + 4 * g) = round4<T>(acc[d] * a.scale);
    if (g == 0) a.delta[row] = delta;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attn_grad_kv_kernel(const AttnArgs a, uint32_t blocks) {
    typedef Tile<T, D> L;
    __shared__ __attribute__((aligned(16))) T q_lds[L::kRows * L::kLd];
    __shared__ __attribute__((aligned(16))) T o_lds[L::kRows * L::kLd];
    __shared__ float top[L::kRows], inv[L::kRows], delta[L::kRows];
    __shared__ uint32_t cls[L::kRows];
    uint32_t b, block;
    int h;
    if (!owner(a, blocks, b, h, block)) return;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int k0 = static_cast<int>(block) * 64 + (threadIdx.x >> 6) * 16 + col;
    const int k = k0 < a.N ? k0 : a.N - 1;
    const Terms terms(a, b, h);
    const uint32_t ck = terms.seam ? token_class(a.region, terms.seam, k) : 0;
    const int64_t first = (static_cast<int64_t>(b) * a.H + h) * a.N;
    const T* go = static_cast<const T*>(a.grad_out) + (static_cast<int64_t>(b) * a.N * a.H + h) * D;
    Rows<T, D> kr, vr;
    kr.load(token_row<T>(a, b, k, 1, h, D), g);
    vr.load(token_row<T>(a, b, k, 2, h, D), g);
    f32x4 dk[L::kSlices] = {}, dv[L::kSlices] = {};
    const T* q_at = token_row<T>(a, b, 0, 0, h, D);
    Staged<T, D> qs, os;
    float top_next = 0.0f, inv_next = 0.0f, delta_next = 0.0f;
    const auto fetch = [&](int q0) {
        qs.fetch(q_at, a.st, q0, a.N), os.fetch(go, static_cast<int64_t>(a.H) * D, q0, a.N);
        if (threadIdx.x < L::kRows) {
            const int q = q0 + static_cast<int>(threadIdx.x);
            const int64_t row = first + (q < a.N ? q : a.N - 1);
            top_next = a.row_max[row], inv_next = a.row_inv[row], delta_next = a.delta[row];
        }
    };
    fetch(0);
    for (int q0 = 0; q0 < a.N; q0 += L::kRows) {
        __syncthreads();
        qs.store(q_lds), os.store(o_lds);
        if (threadIdx.x < L::kRows) {
            const int q = q0 + static_cast<int>(threadIdx.x);
            top[threadIdx.x] = top_next, inv[threadIdx.x] = inv_next, delta[threadIdx.x] = delta_next;
            cls[threadIdx.x] = q < a.N && terms.seam ? token_class(a.region, terms.seam, q) : 0;
        }
        __syncthreads();
        f32x4 bias[L::kRows / 16];
#pragma unroll
        for (int t = 0; t < L::kRows / 16; ++t) bias[t] = terms.of_column(a, q0 + 16 * t + 4 * g, k);
        if (q0 + L::kRows < a.N) fetch(q0 + L::kRows);
#pragma unroll
        for (int t = 0; t < L::kRows / 16; ++t) {
            const int first = 16 * t + 4 * g;
            f32x4 p = terms.of_key(a, product<T, D>(q_lds, 16 * t, kr, col, g), bias[t], q0 + first, k, cls + first, ck);
            f32x4 ds = product<T, D>(o_lds, 16 * t, vr, col, g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = first + r;
                p[r] = q0 + i < a.N ? weight(p[r], top[i]) * inv[i] : 0.0f;
                ds[r] = q0 + i < a.N ? p[r] * (ds[r] - delta[i]) : 0.0f;
            }
            accumulate<T, D>(dv, o_lds, 16 * t, round4<T>(p), col, g);
            accumulate<T, D>(dk, q_lds, 16 * t, round4<T>(ds), col, g);
        }
    }
    if (k0 >= a.N) return;
    T* to = static_cast<T*>(a.grad_qkv) + ((static_cast<int64_t>(b) * a.N + k) * 3 * a.H + a.H + h) * D;
#pragma unroll
    for (int d = 0; d < L::kSlices; ++d) {
        *reinterpret_cast<typename Mma<T>::x4*>(to + 16 * d + 4 * g) = round4<T>(dk[d] * a.scale);
        *reinterpret_cast<typename Mma<T>::x4*>(to + static_cast<int64_t>(a.H) * D + 16 * d + 4 * g) = round4<T>(dv[d]);
    }
}

// A 64-query by kRows-key tile of one head's dbias over the windows
// chunk, chunk + chunks, ...
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attn_grad_bias_kernel(const AttnArgs a, uint32_t qblocks, uint32_t kblocks) {
    typedef Tile<T, D> L;
    __shared__ __attribute__((aligned(16))) T k_lds[L::kRows * L::kLd];
    __shared__ __attribute__((aligned(16))) T v_lds[L::kRows * L::kLd];
    __shared__ uint32_t cls[L::kRows];
    uint32_t id = blockIdx.x;
    const int k0 = static_cast<int>(id % kblocks) * L::kRows;
    id /= kblocks;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int q0 = static_cast<int>(id % qblocks) * 64 + (threadIdx.x >> 6) * 16 + col;
    id /= qblocks;
    const int h = static_cast<int>(id % a.H);
    const uint32_t chunk = id / a.H;
    const int q = q0 < a.N ? q0 : a.N - 1;
    f32x4 acc[L::kRows / 16] = {};
    Staged<T, D> ks, vs;
    Rows<T, D> qn, gn;
    float delta_next = 0.0f, top_next = 0.0f, inv_next = 0.0f;
    const auto fetch = [&](uint32_t b) {
        const int64_t at = (static_cast<int64_t>(b) * a.N + q) * a.H + h;
        const int64_t row = (static_cast<int64_t>(b) * a.H + h) * a.N + q;
        ks.fetch(token_row<T>(a, b, 0, 1, h, D), a.st, k0, a.N);
        vs.fetch(token_row<T>(a, b, 0, 2, h, D), a.st, k0, a.N);
        qn.load(token_row<T>(a, b, q, 0, h, D), g);
        gn.load(static_cast<const T*>(a.grad_out) + at * D, g);
        delta_next = a.delta[row], top_next = a.row_max[row], inv_next = a.row_inv[row];
    };
    if (chunk < a.B) fetch(chunk);
    // the same for every window
    f32x4 bias[L::kRows / 16];
#pragma unroll
    for (int t = 0; t < L::kRows / 16; ++t) bias[t] = Terms(a, 0, h).of_row(a, q, k0 + 16 * t + 4 * g);
    for (uint32_t b = chunk; b < a.B; b += a.chunks) {
        const Terms terms(a, b, h);
        const uint32_t cq = terms.seam ? token_class(a.region, terms.seam, q) : 0;
        const Rows<T, D> qr = qn, go = gn;
        const float delta = delta_next, top = top_next, inv = inv_next;
        __syncthreads();
        ks.store(k_lds), vs.store(v_lds);
        if (threadIdx.x < L::kRows)
            cls[threadIdx.x] = terms.seam && k0 + static_cast<int>(threadIdx.x) < a.N
                                   ? token_class(a.region, terms.seam, k0 + threadIdx.x) : 0;
        __syncthreads();
        if (a.B - b > a.chunks) fetch(b + a.chunks);
#pragma unroll
        for (int t = 0; t < L::kRows / 16; ++t) {
            const int i = 16 * t + 4 * g;
            const f32x4 s = terms.of_query(a, product<T, D>(k_lds, 16 * t, qr, col, g), bias[t], q, k0 + i, cq, cls + i);
            const f32x4 dp = product<T, D>(v_lds, 16 * t, go, col, g);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (k0 + i + r < a.N) acc[t][r] += weight(s[r], top) * inv * (dp[r] - delta);
        }
    }
    if (q0 >= a.N) return;
    float* to = a.grad_bias + ((static_cast<int64_t>(chunk) * a.H + h) * a.N + q) * a.N;
#pragma unroll
    for (int t = 0; t < L::kRows / 16; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int k = k0 + 16 * t + 4 * g + r;
            if (k < a.N) to[k] = acc[t][r];
        }
    }
}

// ---- launchers ------------------------------------------------------------------

template <typename T, int D>
int forward(const AttnArgs& a, hipStream_t stream) {
    const uint32_t blocks = (a.N + 63) / 64;
    const uint32_t grid = xcd_launch_count(a.B * static_cast<uint32_t>(a.H) * blocks);
    attn_forward_kernel<T, D><<<grid, kThreads, 0, stream>>>(a, blocks);
    return check_launch("window_attention");
}

template <typename T, int D>
int backward(const AttnArgs& a, hipStream_t stream) {
    typedef Tile<T, D> L;
    const uint32_t blocks = (a.N + 63) / 64, kblocks = (a.N + L::kRows - 1) / L::kRows;
    const uint32_t grid = xcd_launch_count(a.B * static_cast<uint32_t>(a.H) * blocks);
    attn_grad_q_kernel<T, D><<<grid, kThreads, 0, stream>>>(a, blocks);
    attn_grad_kv_kernel<T, D><<<grid, kThreads, 0, stream>>>(a, blocks);
    if (a.grad_bias != nullptr)
        attn_grad_bias_kernel<T, D><<<a.chunks * static_cast<uint32_t>(a.H) * blocks * kblocks, kThreads, 0, stream>>>(
            a, blocks, kblocks);
    return check_launch("window_attention_backward");
}

template <typename T>
int forward_any(const AttnArgs& a, int D, void* s) {
    hipStream_t stream = static_cast<hipStream_t>(s);
    switch (D) {
        case 16: return forward<T, 16>(a, stream);
        case 32: return forward<T, 32>(a, stream);
        case 64: return forward<T, 64>(a, stream);
        default: return forward<T, 128>(a, stream);
    }
}

template <typename T>
int backward_any(const AttnArgs& a, int D, void* s) {
    hipStream_t stream = static_cast<hipStream_t>(s);
    switch (D) {
        case 16: return backward<T, 16>(a, stream);
        case 32: return backward<T, 32>(a, stream);
        case 64: return backward<T, 64>(a, stream);
        default: return backward<T, 128>(a, stream);
    }
}

}  // namespace
}  // namespace train
}  // namespace crumpet
