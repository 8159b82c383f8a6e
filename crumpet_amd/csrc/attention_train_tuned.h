// Window attention with gradients for windows of up to 16 NT tokens, 16-bit
// types, head dims 16 and 32: the bias-stationary kernels.
//
// The bias (with the mask of the window's kind) is the same for many windows,
// so a wave keeps it in registers: it owns 16 queries (forward, dq and dbias)
// or 16 keys (dk and dv) of one head, NT tiles of 16 x 16 fp32 values, and
// walks a range of windows; in the dbias kernel the sums of dS over the range
// stay in another NT tiles.  Windows are visited grouped by kind (region class
// or mask), so the tiles are rebuilt a few times per range.  The rows of the
// other axis pass through double-buffered LDS, requested a window ahead.
//
// Products: S^T = K Q^T starting from the tiles, which hold (bias + mask) /
// scale, so that neither costs an instruction, P = exp2(S scale log2 e - lse).
// Queries are columns in the forward and dq kernels, keys in the dk and dv
// kernel; the result layout of one product is the B operand of the next, and
// transposes come from LDS transpose reads.  The forward pass computes S
// twice (largest score, then weights) rather than hold it: matrix products
// are cheap beside the exponentials here.
#pragma once

#include <algorithm>
#include <type_traits>

#include "attention_train.h"
#include "train_mma.h"

namespace crumpet {
namespace train {
namespace {


struct Place {
    uint32_t b, kind;
};

template <bool kMask>
__device__ __forceinline__ Place place_of(const AttnArgs& a, const Order& o, uint32_t i) {
    Place p;
    if constexpr (kMask) {
        uint32_t m, j;
        o.share.divmod(i, m, j);
        p.b = j * a.mask_batch + m, p.kind = m;
    } else {
        uint32_t t = 0;
#pragma unroll
        for (int s = 1; s < 8; ++s) t += i >= o.start[s] ? 1u : 0u;
        uint32_t outer, r, wd, wh, ww, rest;
        o.per[t].divmod(i - o.start[t], outer, r);
        o.hw[t].divmod(r, wd, rest);
        o.w[t].divmod(rest, wh, ww);
        if (t & 1) wd = o.last[0];
        if (t & 2) wh = o.last[1];
        if (t & 4) ww = o.last[2];
        p.b = outer * o.windows + (wd * o.gh + wh) * o.gw + ww, p.kind = t;
    }
    p.b = __builtin_amdgcn_readfirstlane(p.b);
    p.kind = __builtin_amdgcn_readfirstlane(p.kind);
    return p;
}

template <typename T, int D>
struct Lds {
    // 16-byte pieces of a row; at head dim 32 they are permuted by the row so
    // that fragment and transpose reads of 16 rows meet distinct banks
    static __device__ __forceinline__ int at(int row, int c) {
        if constexpr (D == 16) return row * 16 + c * 8;
        const int sw = ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
        return row * 32 + ((c ^ sw) << 3);
    }
};

// The lane's operand of 16 rows at full depth: row col, D / 4 dims.
template <typename T, int D>
struct Operand;
template <typename T>
struct Operand<T, 16> {
    typename Mma<T>::x4 v;
    __device__ __forceinline__ void load(const T* row, int g) { v = load4<T>(row + 4 * g); }
    __device__ __forceinline__ void load_lds(const T* tile, int row0, int col, int g) {
        v = load4<T>(tile + (row0 + col) * 16 + 4 * g);
    }
    __device__ __forceinline__ float dim(int e) const { return static_cast<float>(v[e]); }
};
template <typename T>
struct Operand<T, 32> {
    typename Mma<T>::x8 v;
    __device__ __forceinline__ void load(const T* row, int g) {
        v = *reinterpret_cast<const typename Mma<T>::x8*>(row + 8 * g);
    }
    __device__ __forceinline__ void load_lds(const T* tile, int row0, int col, int g) {
        v = *reinterpret_cast<const typename Mma<T>::x8*>(tile + Lds<T, 32>::at(row0 + col, g));
    }
    __device__ __forceinline__ float dim(int e) const { return static_cast<float>(v[e]); }
};
template <typename T, int D>
__device__ __forceinline__ f32x4 multiply(const Operand<T, D>& x, const Operand<T, D>& y, f32x4 c) {
    if constexpr (D == 16)
        return Mma<T>::mma16(x.v, y.v, c);
    else
        return Mma<T>::mma32(x.v, y.v, c);
}

template <typename T>
__device__ __forceinline__ typename Mma<T>::x8 join(typename Mma<T>::x4 lo, typename Mma<T>::x4 hi) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Transposed rows of two 16-row tiles (the depth of one 32-deep product) at
// dims 16 s .. + 15.
template <typename T, int D>
__device__ __forceinline__ typename Mma<T>::x8 transposed_pair(const T* tile, int row0, int s, int col, int g) {
    typedef __attribute__((address_space(3))) i16x4 LdsI16x4;
    i16x4 r[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = row0 + 16 * i + 4 * g + (col >> 2);
        const T* at = tile + Lds<T, D>::at(row, 2 * s + ((col & 3) >> 1)) + 4 * (col & 1);
        r[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)(const_cast<T*>(at)));
    }
    return join<T>(__builtin_bit_cast(typename Mma<T>::x4, r[0]), __builtin_bit_cast(typename Mma<T>::x4, r[1]));
}

// Rows of one matrix of a window on their way into LDS: each thread's pieces.
template <typename T, int D, int NT, int W>
struct Pieces {
    static constexpr int kAll = NT * 16 * (D / 8), kThreads = W * 64, kEach = (kAll + kThreads - 1) / kThreads;
    typedef typename Mma<T>::x8 X8;
    X8 v[kEach];
    __device__ __forceinline__ void load(const T* first, int64_t stride, int N) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int p = threadIdx.x + i * kThreads, r = p / (D / 8), c = p % (D / 8);
            if (kAll % kThreads != 0 && p >= kAll) break;
            v[i] = *reinterpret_cast<const X8*>(first + (r < N ? r : N - 1) * stride + c * 8);
        }
    }
    __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int p = threadIdx.x + i * kThreads, r = p / (D / 8), c = p % (D / 8);
            if (kAll % kThreads != 0 && p >= kAll) break;
            *reinterpret_cast<X8*>(lds + Lds<T, D>::at(r, c)) = v[i];
        }
    }
};

template <typename T>
__device__ __forceinline__ const T* rows_of(const AttnArgs& a, uint32_t b, int which, int h, int D) {
    return static_cast<const T*>(a.qkv) + static_cast<int64_t>(b) * a.sb + (static_cast<int64_t>(which) * a.H + h) * D;
}

// Which seams a token lies past, for every token.
__device__ __forceinline__ void token_sides(const AttnArgs& a, uint8_t* side, int tokens) {
    for (int i = threadIdx.x; i < tokens; i += blockDim.x) {
        uint32_t d, rest, h, w;
        a.region.plane.divmod(static_cast<uint32_t>(i), d, rest);
        a.region.row.divmod(rest, h, w);
        side[i] = (static_cast<int>(d) >= a.region.from[0] ? 1 : 0) | (static_cast<int>(h) >= a.region.from[1] ? 2 : 0) |
                  (static_cast<int>(w) >= a.region.from[2] ? 4 : 0);
    }
}

// The unrolled loops over the tiles are straight-line code, which the compiler
// would otherwise start all of at once, in registers that it does not have.
__device__ __forceinline__ void tiles_in_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Computed here, not where it is next used: otherwise the sums of a whole
// window wait for its end, and with them every term.
template <typename V>
__device__ __forceinline__ void settled(V& v) {
    asm volatile("" : "+v"(v));
}

template <int NT, bool kKeysInLanes, typename M>
__device__ __forceinline__ void add_mask(f32x4* tile, const M* mask, int N, int mine, int g) {
    asm volatile("" : "+v"(mine), "+v"(g));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int other = 16 * t + 4 * g + r, o = other < N ? other : N - 1;
            tile[t][r] += static_cast<float>(mask[kKeysInLanes ? o * N + mine : mine * N + o]);
        }
        tiles_in_order();
    }
}

// The stationary tiles.  Folded (no mask tensor): (bias + region mask) / scale,
// the start of the score product; with a mask tensor: bias + mask, added in
// score units, so that the type's lowest value stays what it is.  Keys past N
// are -inf.  kKeysInLanes: a lane's column is its key and its rows are queries.
template <int NT, bool kMask, bool kKeysInLanes>
__device__ __forceinline__ void build_tiles(f32x4* tile, const AttnArgs& a, int h, uint32_t kind, int row, int g,
                                            const uint8_t* side, float per_scale) {
    const float* bias = a.bias + static_cast<int64_t>(h) * a.N * a.N;
    int mine = row < a.N ? row : a.N - 1;
    // keeps the addresses of all tiles from being computed ahead of the walk
    // and held in registers through it
    asm volatile("" : "+v"(mine), "+v"(g));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int other = 16 * t + 4 * g + r;
            const bool in = other < a.N;
            const int o = in ? other : a.N - 1;
            float v = bias[kKeysInLanes ? o * a.N + mine : mine * a.N + o];
            if constexpr (!kMask) {
                if ((side[o] ^ side[mine]) & kind) v -= 100.0f;
                v *= per_scale;
            }
            tile[t][r] = in || kKeysInLanes ? v : -__builtin_inff();
        }
        tiles_in_order();
    }
    if constexpr (kMask) {
        const int64_t first = static_cast<int64_t>(kind) * a.mask_sb;
        if (a.mask_dtype == CRUMPET_DTYPE_F32)
            add_mask<NT, kKeysInLanes>(tile, static_cast<const float*>(a.mask) + first, a.N, mine, g);
        else if (a.mask_dtype == CRUMPET_DTYPE_F16)
            add_mask<NT, kKeysInLanes>(tile, static_cast<const _Float16*>(a.mask) + first, a.N, mine, g);
        else
            add_mask<NT, kKeysInLanes>(tile, static_cast<const __bf16*>(a.mask) + first, a.N, mine, g);
    }
}

// Beyond this a score's products no longer cancel to a few bits when they are
// subtracted after scaling: take the difference first.
constexpr float kLargeLog2 = 1024.0f;

// (range, group, head) of a workgroup: those of one range share an XCD.
__device__ __forceinline__ bool walk_of(const AttnArgs& a, const Walk& w, uint32_t& range, uint32_t& group, int& h) {
    uint32_t chunk;
    const uint32_t units = w.groups * static_cast<uint32_t>(a.H);
    if (!xcd_chunk(blockIdx.x, gridDim.x, units * w.ranges, chunk)) return false;
    range = chunk / units;
    const uint32_t unit = chunk % units;
    h = static_cast<int>(unit / w.groups);
    group = unit % w.groups;
    return true;
}

// Score of an accumulator value, less the row's largest, times log2 e, plus
// `plus`: the exponent of a weight.
template <bool kMask, bool kLarge>
struct Exponent {
    float scale, c2;   // score = acc scale (+ tile); acc c2 = folded score log2 e
    // top: folded: in units of acc; else in score units.  off = top c2 - plus
    __device__ __forceinline__ float operator()(float acc, float tile, float top, float plus, float off) const {
        if constexpr (kMask)
            return __builtin_fmaf(__builtin_fmaf(acc, scale, tile) - top, kLog2e, plus);
        else if constexpr (kLarge)
            return __builtin_fmaf(acc - top, c2, plus);
        else
            return __builtin_fmaf(acc, c2, -off);
    }
};

template <typename T, int D, int NT, int W, bool kMask>
__global__ void __launch_bounds__(W * 64) attn_forward_tuned_kernel(const AttnArgs a, const Order o, const Walk w) {
    typedef typename Mma<T>::x4 X4;
    constexpr int kTile = NT * 16 * D;
    constexpr int kOut = D / 16;
    __shared__ __attribute__((aligned(16))) T k_lds[2][kTile];
    __shared__ __attribute__((aligned(16))) T v_lds[2][kTile];
    __shared__ uint8_t side[kMask ? 4 : NT * 16];
    uint32_t range, group;
    int h;
    if (!walk_of(a, w, range, group, h)) return;
    const uint32_t begin = range * w.per, end = std::min(a.B, begin + w.per);
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int strip = static_cast<int>(group) * W + (threadIdx.x >> 6);
    const int q0 = strip * 16 + col, q = q0 < a.N ? q0 : a.N - 1;
    const bool active = strip * 16 < a.N;
    const float per_scale = 1.0f / a.scale, c2 = a.scale * kLog2e;
    if constexpr (!kMask) token_sides(a, side, std::min(a.N, NT * 16));
    f32x4 tile[NT];
    uint32_t kind = ~0u;
    Pieces<T, D, NT, W> kp, vp;
    Operand<T, D> qn;
    Place p = place_of<kMask>(a, o, begin);
    kp.load(rows_of<T>(a, p.b, 1, h, D), a.st, a.N);
    vp.load(rows_of<T>(a, p.b, 2, h, D), a.st, a.N);
    qn.load(rows_of<T>(a, p.b, 0, h, D) + q * a.st, g);
    kp.store(k_lds[0]);
    vp.store(v_lds[0]);
    __syncthreads();
    for (uint32_t i = begin; i < end; ++i) {
        const int buf = (i - begin) & 1;
        const Place here = p;
        Operand<T, D> qr = qn;
        const bool more = i + 1 < end;
        if (more) {
            p = place_of<kMask>(a, o, i + 1);
            kp.load(rows_of<T>(a, p.b, 1, h, D), a.st, a.N);
            vp.load(rows_of<T>(a, p.b, 2, h, D), a.st, a.N);
            qn.load(rows_of<T>(a, p.b, 0, h, D) + q * a.st, g);
        }
        if (active) {
            if (here.kind != kind) {
                kind = here.kind;
                build_tiles<NT, kMask, false>(tile, a, h, kind, q, g, side, per_scale);
            }
            const T *kl = k_lds[buf], *vl = v_lds[buf];
            const auto score = [&](int t) {
                Operand<T, D> kr;
                kr.load_lds(kl, 16 * t, col, g);
                return multiply<T, D>(kr, qr, kMask ? f32x4{} : tile[t]);
            };
            float top = -__builtin_inff();
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const f32x4 s = score(t);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    top = fmaxf(top, kMask ? __builtin_fmaf(s[r], a.scale, tile[t][r]) : s[r]);
                if (t % 4 == 3) tiles_in_order();
            }
            top = max_groups(top);
            const float used = top == -__builtin_inff() ? 0.0f : top;  // a row without keys
            // the scores are computed again below, not kept in registers
            asm volatile("" : "+v"(qr.v));
            f32x4 acc[kOut] = {};
            float total = 0.0f;
            const auto weigh = [&](auto large) {
                const Exponent<kMask, decltype(large)::value> exponent = {a.scale, c2};
                const float off = used * c2;
#pragma unroll
                for (int t = 0; t < NT; t += 2) {
                    X4 hi[2], lo[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        f32x4 s = score(t + u);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            s[r] = __builtin_amdgcn_exp2f(exponent(s[r], tile[t + u][r], used, 0.0f, off));
                            total += s[r];
                        }
                        settled(total);
                        hi[u] = round4<T>(s);
                        lo[u] = round4<T>(s - wide4<T>(hi[u]));
                    }
#pragma unroll
                    for (int s = 0; s < kOut; ++s) {
                        const typename Mma<T>::x8 vt = transposed_pair<T, D>(vl, 16 * t, s, col, g);
                        acc[s] = Mma<T>::mma32(vt, join<T>(hi[0], hi[1]), acc[s]);
                        acc[s] = Mma<T>::mma32(vt, join<T>(lo[0], lo[1]), acc[s]);
                    }
                    tiles_in_order();
                }
            };
            if (!kMask && __any(fabsf(used * c2) > kLargeLog2))
                weigh(std::true_type{});
            else
                weigh(std::false_type{});
            total = sum_groups(total);
            if (q0 < a.N) {
                const float inv = total == 0.0f ? 0.0f : 1.0f / total;
                const int64_t at = ((static_cast<int64_t>(here.b) * a.N + q) * a.H + h) * D;
#pragma unroll
                for (int s = 0; s < kOut; ++s) {
                    const f32x4 out = acc[s] * inv;
                    const X4 hi = round4<T>(out);
                    *reinterpret_cast<X4*>(static_cast<T*>(a.out) + at + 16 * s + 4 * g) = hi;
                    if (a.out_lo != nullptr)
                        *reinterpret_cast<X4*>(static_cast<T*>(a.out_lo) + at + 16 * s + 4 * g) =
                            round4<T>(out - wide4<T>(hi));
                }
                if (g == 0 && a.row_max != nullptr) {
                    const int64_t row = (static_cast<int64_t>(here.b) * a.H + h) * a.N + q;
                    a.row_max[row] = used;
                    a.row_inv[row] = inv;
                }
            }
        }
        if (more) {
            kp.store(k_lds[buf ^ 1]);
            vp.store(v_lds[buf ^ 1]);
            __syncthreads();
        }
    }
}

// dq, delta and a range's share of dbias.
template <typename T, int D, int NT, int W, bool kMask>
__global__ void __launch_bounds__(W * 64) attn_grad_q_tuned_kernel(const AttnArgs a, const Order o, const Walk w) {
    typedef typename Mma<T>::x4 X4;
    constexpr int kTile = NT * 16 * D;
    constexpr int kOut = D / 16;
    __shared__ __attribute__((aligned(16))) T k_lds[2][kTile];
    __shared__ __attribute__((aligned(16))) T v_lds[2][kTile];
    __shared__ uint8_t side[kMask ? 4 : NT * 16];
    uint32_t range, group;
    int h;
    if (!walk_of(a, w, range, group, h)) return;
    const uint32_t begin = range * w.per, end = std::min(a.B, begin + w.per);
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int strip = static_cast<int>(group) * W + (threadIdx.x >> 6);
    const int q0 = strip * 16 + col, q = q0 < a.N ? q0 : a.N - 1;
    const bool active = strip * 16 < a.N;
    const float per_scale = 1.0f / a.scale, c2 = a.scale * kLog2e;
    if constexpr (!kMask) token_sides(a, side, std::min(a.N, NT * 16));
    f32x4 tile[NT], sums[NT] = {};
    uint32_t kind = ~0u;
    Pieces<T, D, NT, W> pieces;
    Operand<T, D> qn, gn;
    const auto fetch_rows = [&](uint32_t b) {
        qn.load(rows_of<T>(a, b, 0, h, D) + q * a.st, g);
        gn.load(static_cast<const T*>(a.grad_out) + ((static_cast<int64_t>(b) * a.N + q) * a.H + h) * D, g);
    };
    Place p = place_of<kMask>(a, o, begin);
    pieces.load(rows_of<T>(a, p.b, 1, h, D), a.st, a.N);
    fetch_rows(p.b);
    pieces.store(k_lds[0]);
    pieces.load(rows_of<T>(a, p.b, 2, h, D), a.st, a.N);
    pieces.store(v_lds[0]);
    __syncthreads();
    for (uint32_t i = begin; i < end; ++i) {
        const int buf = (i - begin) & 1;
        const Place here = p;
        const Operand<T, D> qr = qn, go = gn;
        const bool more = i + 1 < end;
        // the row's statistics and output, then the next window's rows
        const int64_t row = (static_cast<int64_t>(here.b) * a.H + h) * a.N + q;
        const int64_t at = ((static_cast<int64_t>(here.b) * a.N + q) * a.H + h) * D;
        Operand<T, D> out, rest;
        out.load(static_cast<const T*>(a.out) + at, g);
        rest.load(static_cast<const T*>(a.out_lo) + at, g);
        const float top = a.row_max[row], inv = a.row_inv[row];
        if (more) {
            p = place_of<kMask>(a, o, i + 1);
            pieces.load(rows_of<T>(a, p.b, 1, h, D), a.st, a.N);
            fetch_rows(p.b);
        }
        float delta = 0.0f;
#pragma unroll
        for (int e = 0; e < D / 4; ++e) delta = __builtin_fmaf(out.dim(e) + rest.dim(e), go.dim(e), delta);
        delta = sum_groups(delta);
        f32x4 acc[kOut] = {};
        const auto half = [&](auto large, int from, int to) {
            const Exponent<kMask, decltype(large)::value> exponent = {a.scale, c2};
            const float plus = __builtin_amdgcn_logf(inv), off = top * c2 - plus;
            const T *kl = k_lds[buf], *vl = v_lds[buf];
#pragma unroll
            for (int t = 0; t < NT; t += 2) {
                if (t < from || t >= to) continue;
                X4 ds[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    Operand<T, D> kr, vr;
                    kr.load_lds(kl, 16 * (t + u), col, g);
                    vr.load_lds(vl, 16 * (t + u), col, g);
                    f32x4 s = multiply<T, D>(kr, qr, kMask ? f32x4{} : tile[t + u]);
                    const f32x4 dp = multiply<T, D>(vr, go, f32x4{-delta, -delta, -delta, -delta});
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[r] = __builtin_amdgcn_exp2f(exponent(s[r], tile[t + u][r], top, plus, off)) * dp[r];
                        sums[t + u][r] += s[r];
                    }
                    settled(sums[t + u]);
                    ds[u] = round4<T>(s);
                }
#pragma unroll
                for (int s = 0; s < kOut; ++s)
                    acc[s] = Mma<T>::mma32(transposed_pair<T, D>(kl, 16 * t, s, col, g), join<T>(ds[0], ds[1]), acc[s]);
                tiles_in_order();
            }
        };
        constexpr int kHalf = NT / 4 * 2;
        const bool large = !kMask && __any(fabsf(top * c2) > kLargeLog2);
        if (active) {
            if (here.kind != kind) {
                kind = here.kind;
                build_tiles<NT, kMask, false>(tile, a, h, kind, q, g, side, per_scale);
            }
            half(std::true_type{}, 0, kHalf);
        }
        if (more) {
            pieces.store(k_lds[buf ^ 1]);
            pieces.load(rows_of<T>(a, p.b, 2, h, D), a.st, a.N);
        }
        if (active) {
            half(std::true_type{}, kHalf, NT);
            if (q0 < a.N) {
                T* to = static_cast<T*>(a.grad_qkv) + ((static_cast<int64_t>(here.b) * a.N + q) * 3 * a.H + h) * D;
#pragma unroll
                for (int s = 0; s < kOut; ++s)
                    *reinterpret_cast<X4*>(to + 16 * s + 4 * g) = round4<T>(acc[s] * a.scale);
                if (g == 0) a.delta[row] = delta;
            }
        }
        if (more) {
            pieces.store(v_lds[buf ^ 1]);
            __syncthreads();
        }
    }
    if (!active || q0 >= a.N || a.grad_bias == nullptr) return;
    float* to = a.grad_bias + ((static_cast<int64_t>(range) * a.H + h) * a.N + q) * a.N;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int k = 16 * t + 4 * g + r;
            if (k < a.N) to[k] = sums[t][r];
        }
    }
}

// dk and dv: a wave owns 16 keys.
template <typename T, int D, int NT, int W, bool kMask>
__global__ void __launch_bounds__(W * 64) attn_grad_kv_tuned_kernel(const AttnArgs a, const Order o, const Walk w) {
    typedef typename Mma<T>::x4 X4;
    constexpr int kTile = NT * 16 * D, kRows = NT * 16, kEach = (kRows + W * 64 - 1) / (W * 64);
    constexpr int kOut = D / 16;
    __shared__ __attribute__((aligned(16))) T q_lds[2][kTile];
    __shared__ __attribute__((aligned(16))) T o_lds[2][kTile];
    // per query: largest score, log2 of 1 / sum, -delta
    __shared__ __attribute__((aligned(16))) float top_lds[2][kRows], plus_lds[2][kRows], delta_lds[2][kRows];
    __shared__ uint8_t side[kMask ? 4 : kRows];
    uint32_t range, group;
    int h;
    if (!walk_of(a, w, range, group, h)) return;
    const uint32_t begin = range * w.per, end = std::min(a.B, begin + w.per);
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int strip = static_cast<int>(group) * W + (threadIdx.x >> 6);
    const int k0 = strip * 16 + col, k = k0 < a.N ? k0 : a.N - 1;
    const bool active = strip * 16 < a.N;
    const float per_scale = 1.0f / a.scale, c2 = a.scale * kLog2e;
    if constexpr (!kMask) token_sides(a, side, std::min(a.N, kRows));
    f32x4 tile[NT];
    uint32_t kind = ~0u;
    Pieces<T, D, NT, W> qp, op;
    float top_r[kEach], plus_r[kEach], delta_r[kEach];
    Operand<T, D> kn, vn;
    const auto fetch = [&](uint32_t b) {
        const T* first = static_cast<const T*>(a.grad_out) + (static_cast<int64_t>(b) * a.N * a.H + h) * D;
        qp.load(rows_of<T>(a, b, 0, h, D), a.st, a.N);
        op.load(first, static_cast<int64_t>(a.H) * D, a.N);
        kn.load(rows_of<T>(a, b, 1, h, D) + k * a.st, g);
        vn.load(rows_of<T>(a, b, 2, h, D) + k * a.st, g);
        const int64_t row = (static_cast<int64_t>(b) * a.H + h) * a.N;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int r = threadIdx.x + i * W * 64;
            const bool in = r < a.N;
            const int64_t at = row + (in ? r : a.N - 1);
            top_r[i] = in ? a.row_max[at] : 0.0f;
            plus_r[i] = in ? a.row_inv[at] : 0.0f;  // queries past N: log2 0 = -inf, no weight
            delta_r[i] = in ? a.delta[at] : 0.0f;
        }
    };
    const auto keep = [&](int buf) {
        qp.store(q_lds[buf]);
        op.store(o_lds[buf]);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int r = threadIdx.x + i * W * 64;
            if (r >= kRows) break;
            top_lds[buf][r] = top_r[i];
            plus_lds[buf][r] = __builtin_amdgcn_logf(plus_r[i]);
            delta_lds[buf][r] = -delta_r[i];
        }
    };
    Place p = place_of<kMask>(a, o, begin);
    fetch(p.b);
    keep(0);
    __syncthreads();
    for (uint32_t i = begin; i < end; ++i) {
        const int buf = (i - begin) & 1;
        const Place here = p;
        const Operand<T, D> kr = kn, vr = vn;
        const bool more = i + 1 < end;
        if (more) {
            p = place_of<kMask>(a, o, i + 1);
            fetch(p.b);
        }
        if (active) {
            if (here.kind != kind) {
                kind = here.kind;
                build_tiles<NT, kMask, true>(tile, a, h, kind, k, g, side, per_scale);
            }
            const T *ql = q_lds[buf], *ol = o_lds[buf];
            const Exponent<kMask, true> exponent = {a.scale, c2};
            f32x4 dk[kOut] = {}, dv[kOut] = {};
#pragma unroll
            for (int t = 0; t < NT; t += 2) {
                X4 pw[2], ds[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int first = 16 * (t + u) + 4 * g;
                    Operand<T, D> qr, go;
                    qr.load_lds(ql, 16 * (t + u), col, g);
                    go.load_lds(ol, 16 * (t + u), col, g);
                    const f32x4 top = *reinterpret_cast<const f32x4*>(&top_lds[buf][first]);
                    const f32x4 plus = *reinterpret_cast<const f32x4*>(&plus_lds[buf][first]);
                    const f32x4 delta = *reinterpret_cast<const f32x4*>(&delta_lds[buf][first]);
                    f32x4 s = multiply<T, D>(qr, kr, kMask ? f32x4{} : tile[t + u]);
                    f32x4 dp = multiply<T, D>(go, vr, delta);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[r] = __builtin_amdgcn_exp2f(exponent(s[r], tile[t + u][r], top[r], plus[r], 0.0f));
                        dp[r] *= s[r];
                    }
                    pw[u] = round4<T>(s);
                    ds[u] = round4<T>(dp);
                }
#pragma unroll
                for (int s = 0; s < kOut; ++s) {
                    dv[s] = Mma<T>::mma32(transposed_pair<T, D>(ol, 16 * t, s, col, g), join<T>(pw[0], pw[1]), dv[s]);
                    dk[s] = Mma<T>::mma32(transposed_pair<T, D>(ql, 16 * t, s, col, g), join<T>(ds[0], ds[1]), dk[s]);
                }
                tiles_in_order();
            }
            if (k0 < a.N) {
                const int64_t hd = static_cast<int64_t>(a.H) * D;
                T* to = static_cast<T*>(a.grad_qkv) + ((static_cast<int64_t>(here.b) * a.N + k) * 3 * a.H + h) * D + hd;
#pragma unroll
                for (int s = 0; s < kOut; ++s) {
                    *reinterpret_cast<X4*>(to + 16 * s + 4 * g) = round4<T>(dk[s] * a.scale);
                    *reinterpret_cast<X4*>(to + hd + 16 * s + 4 * g) = round4<T>(dv[s]);
                }
            }
        }
        if (more) {
            keep(buf ^ 1);
            __syncthreads();
        }
    }
}

// ---- launchers ------------------------------------------------------------------

template <typename T, int D, int NT, bool kMask>
void launch_forward(const AttnArgs& a, const Order& o, hipStream_t s) {
    constexpr int W = tuned_waves(NT, kForwardPass);
    const Walk w = tuned_walk(a.B, a.H, a.N, kForwardPass);
    const uint32_t grid = xcd_launch_count(w.groups * static_cast<uint32_t>(a.H) * w.ranges);
    attn_forward_tuned_kernel<T, D, NT, W, kMask><<<grid, W * 64, 0, s>>>(a, o, w);
}

template <typename T, int D, int NT, bool kMask>
void launch_backward(const AttnArgs& a, const Order& o, hipStream_t s) {
    constexpr int W = tuned_waves(NT, kQueryPass), V = tuned_waves(NT, kKeyPass);
    const Walk w = tuned_walk(a.B, a.H, a.N, kQueryPass), v = tuned_walk(a.B, a.H, a.N, kKeyPass);
    const uint32_t heads = static_cast<uint32_t>(a.H);
    attn_grad_q_tuned_kernel<T, D, NT, W, kMask>
        <<<xcd_launch_count(w.groups * heads * w.ranges), W * 64, 0, s>>>(a, o, w);
    attn_grad_kv_tuned_kernel<T, D, NT, V, kMask>
        <<<xcd_launch_count(v.groups * heads * v.ranges), V * 64, 0, s>>>(a, o, v);
}

template <typename T, int D, bool kMask>
void launch_tuned(const AttnArgs& a, const Order& o, bool grad, hipStream_t s) {
#define CRUMPET_TILES(NT)                          \
    case NT:                                       \
        if (grad)                                  \
            launch_backward<T, D, NT, kMask>(a, o, s); \
        else                                       \
            launch_forward<T, D, NT, kMask>(a, o, s);  \
        break;
    switch (tuned_tiles(a.N)) {
        CRUMPET_TILES(4) CRUMPET_TILES(8) CRUMPET_TILES(14) CRUMPET_TILES(22) CRUMPET_TILES(32)
    }
#undef CRUMPET_TILES
}

template <typename T, bool kMask>
int tuned_any(const AttnArgs& a, const Order& o, int D, bool grad, void* stream) {
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (D == 16)
        launch_tuned<T, 16, kMask>(a, o, grad, s);
    else
        launch_tuned<T, 32, kMask>(a, o, grad, s);
    return check_launch(grad ? "window_attention_backward" : "window_attention");
}

}  // namespace
}  // namespace train
}  // namespace crumpet
