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
//
// Measured on 1372 windows of 343 tokens and three heads of 16 in fp16: forward
// 241 us, dq and dbias 308, dk and dv 255, the join of dbias 7.  Issue bounds
// them, not memory (364 MB in all): VALU 55, 47 and 60% busy, the matrix cores
// 26, 13 and 19%, with two waves a SIMD, all that the registers of the tiles
// leave.  Of the forward pass 51 us are the rests of P, which make dbias exact
// to fp32, 23 the pass for the largest score.  Without a mask tensor a range
// rebuilds its tiles a few times, which is nothing; with one it does so for
// every few windows: 128 windows, 64 masks, six heads of 32 in bf16 take 104,
// 118 and 97 us, about half of it waiting for rows of bias and mask.
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
    return p;
}

// The places of a walk's windows: each lane works out one of the next 64, the
// divisions of which would hold up every window otherwise.
template <bool kMask>
struct Places {
    Place mine;
    uint32_t begin, end;
    __device__ __forceinline__ Places(uint32_t b, uint32_t e) : mine(), begin(b), end(e) {}
    __device__ __forceinline__ Place at(const AttnArgs& a, const Order& o, uint32_t i) {
        const uint32_t n = i - begin;
        if (n % 64 == 0) {
            const uint32_t w = i + (threadIdx.x & 63);
            mine = place_of<kMask>(a, o, w < end ? w : end - 1);
        }
        Place p;
        p.b = __builtin_amdgcn_readlane(mine.b, n % 64);
        p.kind = __builtin_amdgcn_readlane(mine.kind, n % 64);
        return p;
    }
};

template <typename T, int D>
struct Lds {
    // 16-byte pieces of a row; at head dim 32 they are permuted by the row so
    // that fragment and transpose reads of 16 rows meet distinct banks
    static __device__ __forceinline__ int piece(int row, int c) {
        return D == 16 ? c : c ^ (((row >> 2) & 1) << 1 | ((row >> 3) & 1));
    }
    static __device__ __forceinline__ int at(int row, int c) { return row * D + piece(row, c) * 8; }
};

// Two views of a tile for the even and the odd 16 rows: a merged read of both
// (ds_read2st64_b64) meets the same banks twice and takes 32 cycles for 8.
template <typename T>
struct Halves {
    const T* of[2];
    __device__ __forceinline__ Halves(const T* tile, int step) {
        uint32_t other = step;
        asm volatile("" : "+v"(other));
        of[0] = tile, of[1] = tile + other;
    }
};

// The lane's operand of 16 rows at full depth: row col, D / 4 dims.
template <typename T, int D>
struct Operand;
template <typename T>
struct Operand<T, 16> {
    typename Mma<T>::x4 v;
    __device__ __forceinline__ void load(const T* first, uint32_t row, int g) { v = load4<T>(first + (row + 4 * g)); }
    __device__ __forceinline__ void load_lds(const T* tile, int row0, int col, int g) {
        v = load4<T>(tile + (row0 + col) * 16 + 4 * g);
    }
    __device__ __forceinline__ float dim(int e) const { return static_cast<float>(v[e]); }
};
template <typename T>
struct Operand<T, 32> {
    typename Mma<T>::x8 v;
    __device__ __forceinline__ void load(const T* first, uint32_t row, int g) {
        v = *reinterpret_cast<const typename Mma<T>::x8*>(first + (row + 8 * g));
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

template <typename T, int D>
__device__ __forceinline__ typename Mma<T>::x4 transposed_one(const T* tile, int row0, int s, int col, int g) {
    typedef __attribute__((address_space(3))) i16x4 LdsI16x4;
    const T* at = tile + Lds<T, D>::at(row0 + 4 * g + (col >> 2), 2 * s + ((col & 3) >> 1)) + 4 * (col & 1);
    return __builtin_bit_cast(typename Mma<T>::x4,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)(const_cast<T*>(at))));
}

// Addresses: a base that is the same for the wave (scalar registers) plus a
// 32-bit offset of the lane, which stays the same from window to window.

// Rows of one matrix of a window on their way into LDS, without passing through
// registers: load j of a wave fills the 64 16-byte slots from 64 j, in slot
// order, with the pieces that belong there.
template <typename T, int D, int NT, int W>
struct Rows {
    static constexpr int kLoads = NT * 16 * (D / 8) / 64, kEach = (kLoads + W - 1) / W;
    uint32_t of[kEach];  // where the lane's pieces lie in the matrix, bytes
    uint32_t bytes;
    int wave;
    __device__ __forceinline__ Rows(uint32_t stride, int N) {
        wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
        bytes = (static_cast<uint32_t>(N - 1) * stride + D) * sizeof(T);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int slot = (wave + i * W) * 64 + (threadIdx.x & 63), r = slot / (D / 8);
            of[i] = (static_cast<uint32_t>(r < N ? r : N - 1) * stride + Lds<T, D>::piece(r, slot % (D / 8)) * 8) * sizeof(T);
        }
    }
    __device__ __forceinline__ void load(const T* first, uint32_t to) const {
        const u32x4 buffer = buffer_of(first, bytes);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (wave + i * W < kLoads) load_to_lds(buffer, to + (wave + i * W) * 1024, of[i]);
    }
};

template <typename T>
__device__ __forceinline__ const T* rows_of(const AttnArgs& a, uint32_t b, int which, int h, int D) {
    return static_cast<const T*>(a.qkv) + static_cast<int64_t>(b) * a.sb + (static_cast<int64_t>(which) * a.H + h) * D;
}

// First element of a window's and head's rows in [B, N, H, D].
template <int D>
__device__ __forceinline__ int64_t heads_row(const AttnArgs& a, uint32_t b, int h) {
    return (static_cast<int64_t>(b) * a.N * a.H + h) * D;
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

// v = hi + lo to twice the type's precision: hi rounded towards zero in fp16
// (one packed conversion; the rest is exact all the same).
template <typename T>
__device__ __forceinline__ void split(f32x4 v, typename Mma<T>::x4& hi, typename Mma<T>::x4& lo) {
    if constexpr (std::is_same<T, _Float16>::value) {
        typedef __fp16 h16x2 __attribute__((ext_vector_type(2)));
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const f16x2 a = __builtin_bit_cast(f16x2, static_cast<h16x2>(__builtin_amdgcn_cvt_pkrtz(v[0], v[1])));
        const f16x2 b = __builtin_bit_cast(f16x2, static_cast<h16x2>(__builtin_amdgcn_cvt_pkrtz(v[2], v[3])));
        hi = __builtin_shufflevector(a, b, 0, 1, 2, 3);
        f32x4 rest;
        // v - hi in one step: v_fma_mix_f32 takes the fp16 half as it is
        const uint32_t pair[2] = {__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(rest[e]) : "v"(pair[e >> 1]), "v"(v[e]));
            asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
                : "=v"(rest[e + 1])
                : "v"(pair[e >> 1]), "v"(v[e + 1]));
        }
        lo = round4<T>(rest);
    } else {
        hi = round4<T>(v);
        lo = round4<T>(v - wide4<T>(hi));
    }
}

constexpr float kLargest = 3.40282347e38f;

// The unrolled loops over the tiles are straight-line code, which the compiler
// would otherwise start all of at once, in registers that it does not have.
__device__ __forceinline__ void tiles_in_order() {
    asm volatile("" ::: "memory");
}

// Computed here, not where it is next used: otherwise the sums of a whole
// window wait for its end, and with them every term.
template <typename V>
__device__ __forceinline__ void settled(V& v) {
    asm volatile("" : "+v"(v));
}

// Four neighbours that lie anywhere (rows of an odd length): one load.
template <typename E>
struct __attribute__((packed, aligned(sizeof(E)))) Neighbours {
    E v[4];
};

// bias + mask for a lane whose rows are keys, -inf past N (N >= 2).  All rows
// of the bias are on their way at once, straight into the tiles, and the mask's
// 6 tiles at a time.  A read may run into the next query's row, never past
// the matrix: the last query's last keys are read singly afterwards.
template <int NT, typename M>
__device__ __forceinline__ void add_rows(f32x4* tile, const float* bias, const M* mask, int N, int mine, int first) {
    asm volatile("" : "+v"(mine), "+v"(first));
    const uint32_t row = static_cast<uint32_t>(mine * N + first), last = static_cast<uint32_t>(N * N - 4);
    const auto place = [&](int t) { return row + 16 * t < last ? row + 16 * t : last; };
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const Neighbours<float> b = *reinterpret_cast<const Neighbours<float>*>(bias + place(t));
#pragma unroll
        for (int r = 0; r < 4; ++r) tile[t][r] = b.v[r];
    }
    tiles_in_order();
#pragma unroll
    for (int t0 = 0; t0 < NT; t0 += 6) {
        Neighbours<M> m[6];
#pragma unroll
        for (int u = 0; u < 6 && t0 + u < NT; ++u)
            m[u] = *reinterpret_cast<const Neighbours<M>*>(mask + place(t0 + u));
#pragma unroll
        for (int u = 0; u < 6 && t0 + u < NT; ++u) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                tile[t0 + u][r] = 16 * (t0 + u) + first + r < N ? tile[t0 + u][r] + static_cast<float>(m[u].v[r])
                                                                : -__builtin_inff();
        }
        tiles_in_order();
    }
    if (mine + 1 < N) return;
    asm volatile("" : "+v"(first));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int at = 16 * t + first;
        if (at >= N || at + 4 <= N) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (at + r < N) tile[t][r] = bias[mine * N + at + r] + static_cast<float>(mask[mine * N + at + r]);
    }
}
// The same for a lane whose column is a key; rows past N are the last one's.
template <int NT, typename M>
__device__ __forceinline__ void add_columns(f32x4* tile, const float* bias, const M* mask, int N, int mine, int first) {
    asm volatile("" : "+v"(mine), "+v"(first));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int other = 16 * t + first + r, o = other < N ? other : N - 1;
            tile[t][r] = bias[o * N + mine] + static_cast<float>(mask[o * N + mine]);
        }
        if (t % 2 == 1) tiles_in_order();
    }
}

// The stationary tiles.  Folded (no mask tensor): (bias + region mask) / scale,
// the start of the score product; with a mask tensor: bias + mask, added in
// score units, so that the type's lowest value stays what it is.  Keys past N
// are -inf.  kKeysInLanes: a lane's column is its key and its rows are queries.
// first: the other axis' index of the lane's first value.
template <int NT, bool kMask, bool kKeysInLanes>
__device__ __forceinline__ void build_tiles(f32x4* tile, const AttnArgs& a, int h, uint32_t kind, int mine, int first,
                                            const uint8_t* side, float per_scale) {
    const float* bias = a.bias + static_cast<int64_t>(h) * a.N * a.N;
    // keeps the addresses of all tiles from being computed ahead of the walk
    // and held in registers through it
    asm volatile("" : "+v"(mine), "+v"(first));
    if constexpr (kMask) {
        const int64_t at = static_cast<int64_t>(kind) * a.mask_sb;
        const auto add = [&](auto mask) {
            if constexpr (kKeysInLanes)
                add_columns<NT>(tile, bias, mask + at, a.N, mine, first);
            else
                add_rows<NT>(tile, bias, mask + at, a.N, mine, first);
        };
        if (a.mask_dtype == CRUMPET_DTYPE_F32)
            add(static_cast<const float*>(a.mask));
        else if (a.mask_dtype == CRUMPET_DTYPE_F16)
            add(static_cast<const _Float16*>(a.mask));
        else
            add(static_cast<const __bf16*>(a.mask));
    } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int other = 16 * t + first + r;
                const bool in = other < a.N;
                const int o = in ? other : a.N - 1;
                float v = bias[kKeysInLanes ? o * a.N + mine : mine * a.N + o];
                if ((side[o] ^ side[mine]) & kind) v -= 100.0f;
                // fp32's lowest value stays finite: a row of it has equal weights
                const float folded = fminf(fmaxf(v * per_scale, -kLargest), kLargest);
                v = fabsf(v) <= kLargest ? folded : v;
                tile[t][r] = in || kKeysInLanes ? v : -__builtin_inff();
            }
            tiles_in_order();
        }
    }
}

// Lane (col, g)'s value for row 4 g + r, from the lane of its group that holds it.
__device__ __forceinline__ float of_row(float v, int r) {
    const int bits = __float_as_int(v);
    int got = bits;
    switch (r) {  // DPP row_newbcast
        case 0: got = __builtin_amdgcn_update_dpp(0, bits, 0x150, 0xf, 0xf, true); break;
        case 1: got = __builtin_amdgcn_update_dpp(0, bits, 0x151, 0xf, 0xf, true); break;
        case 2: got = __builtin_amdgcn_update_dpp(0, bits, 0x152, 0xf, 0xf, true); break;
        default: got = __builtin_amdgcn_update_dpp(0, bits, 0x153, 0xf, 0xf, true); break;
    }
    return __int_as_float(got);
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

// Where a wave stands: kSplit waves share the 16 rows of a strip, each with
// kSpan of the NT tiles of the other axis.
template <int NT, int S, int kSplit>
struct Share {
    static constexpr int kSpan = NT / kSplit;
    int lane, col, g, local, part, row0, row, first;
    bool active, leads;
    __device__ __forceinline__ Share(const AttnArgs& a, uint32_t group) {
        const int wave = threadIdx.x >> 6;
        lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
        local = wave / kSplit, part = wave % kSplit;
        const int strip = static_cast<int>(group) * S + local;
        row0 = strip * 16 + col, row = row0 < a.N ? row0 : a.N - 1;
        active = strip * 16 < a.N;
        leads = part == 0;
        first = part * kSpan;  // first tile of the other axis
    }
};

// Sums that the other waves of a strip hand to the one that leads it: written
// at the end of a window, read after the barrier that ends it, in two copies
// so that the next window's do not meet them.
template <int S, int kSplit, int kValues>
struct Handover {
    static constexpr int kFloats = kSplit > 1 ? 2 * S * (kSplit - 1) * kValues * 64 : 1;
    float* lds;
    int at;
    __device__ __forceinline__ Handover(float* l, int local, int lane) : lds(l), at(local * (kSplit - 1) * kValues * 64 + lane) {}
    __device__ __forceinline__ float& value(int copy, int part, int v) const {
        return lds[copy * S * (kSplit - 1) * kValues * 64 + at + ((part - 1) * kValues + v) * 64];
    }
};

// The transposed rows of `count` tiles (1 or 2) at row0, to be added up with
// weights: acc[d][lane's column] += rows times w.
template <typename T, int D>
struct Turned {
    typename Mma<T>::x8 v[D / 16];
    __device__ __forceinline__ void load(const T* lds, int row0, int count, int col, int g) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            if (count == 2) {
                v[d] = transposed_pair<T, D>(lds, row0, d, col, g);
            } else {
                const typename Mma<T>::x4 one = transposed_one<T, D>(lds, row0, d, col, g);
                v[d] = join<T>(one, one);
            }
        }
    }
    __device__ __forceinline__ void add(f32x4* acc, int count, const typename Mma<T>::x4* w) const {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            if (count == 2)
                acc[d] = Mma<T>::mma32(v[d], join<T>(w[0], w[1]), acc[d]);
            else
                acc[d] = Mma<T>::mma16(__builtin_shufflevector(v[d], v[d], 0, 1, 2, 3), w[0], acc[d]);
        }
    }
};

template <typename T, int D, int NT, int S, int kSplit, int kWaves, bool kMask>
__global__ void __launch_bounds__(S* kSplit * 64) __attribute__((amdgpu_waves_per_eu(kWaves)))
attn_forward_tuned_kernel(const AttnArgs a, const Order o, const Walk w) {
    typedef typename Mma<T>::x4 X4;
    typedef Share<NT, S, kSplit> Mine;
    constexpr int kTile = NT * 16 * D, W = S * kSplit, kOut = D / 16, kSpan = Mine::kSpan;
    typedef Handover<S, kSplit, 4 * kOut + 2> Hand;
    __shared__ __attribute__((aligned(16))) T k_lds[2][kTile];
    __shared__ __attribute__((aligned(16))) T v_lds[2][kTile];
    __shared__ float hand_lds[Hand::kFloats];
    __shared__ uint8_t side[kMask ? 4 : NT * 16];
    uint32_t range, group;
    int h;
    if (!walk_of(a, w, range, group, h)) return;
    const uint32_t begin = range * w.per, end = std::min(a.B, begin + w.per);
    const Mine me(a, group);
    const int col = me.col, g = me.g, q = me.row;
    const Hand hand(hand_lds, me.local, me.lane);
    const float per_scale = 1.0f / a.scale, c2 = a.scale * kLog2e;
    const float unit = kMask ? kLog2e : c2;  // of `top`, to log2
    if constexpr (!kMask) token_sides(a, side, std::min(a.N, NT * 16));
    X4 ones;
#pragma unroll
    for (int e = 0; e < 4; ++e) ones[e] = static_cast<T>(1.0f);
    f32x4 tile[kSpan];
    uint32_t kind = ~0u;
    Operand<T, D> qn;
    Places<kMask> places(begin, end);
    Place p = places.at(a, o, begin);
    const Rows<T, D, NT, W> rows(static_cast<uint32_t>(a.st), a.N);
    const uint32_t mine = static_cast<uint32_t>(q) * static_cast<uint32_t>(a.st);
    const auto fetch = [&](uint32_t b, int buf) {
        rows.load(rows_of<T>(a, b, 1, h, D), lds_address(k_lds[0]) + buf * kTile * sizeof(T));
        rows.load(rows_of<T>(a, b, 2, h, D), lds_address(v_lds[0]) + buf * kTile * sizeof(T));
        qn.load(rows_of<T>(a, b, 0, h, D), mine, g);
    };
    fetch(p.b, 0);
    f32x4 acc[kOut];
    float top, total;
    // joins the strip's parts and stores the window's rows
    const auto finish = [&](uint32_t b, int copy) {
        float most = top;
#pragma unroll
        for (int i = 1; i < kSplit; ++i) most = fmaxf(most, hand.value(copy, i, 0));
        const float used = most == -__builtin_inff() ? 0.0f : most;  // a row without keys
        const float f = __builtin_amdgcn_exp2f((top - used) * unit);
        total *= f;
#pragma unroll
        for (int d = 0; d < kOut; ++d) acc[d] *= f;
#pragma unroll
        for (int i = 1; i < kSplit; ++i) {
            const float e = __builtin_amdgcn_exp2f((hand.value(copy, i, 0) - used) * unit);
            total = __builtin_fmaf(hand.value(copy, i, 1), e, total);
#pragma unroll
            for (int v = 0; v < 4 * kOut; ++v)
                acc[v >> 2][v & 3] = __builtin_fmaf(hand.value(copy, i, 2 + v), e, acc[v >> 2][v & 3]);
        }
        if (me.row0 >= a.N) return;
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        const int64_t at = heads_row<D>(a, b, h);
        T *to = static_cast<T*>(a.out) + at, *to_lo = static_cast<T*>(a.out_lo) + at;
#pragma unroll
        for (int d = 0; d < kOut; ++d) {
            const uint32_t lane_at = static_cast<uint32_t>(q) * (a.H * D) + 16 * d + 4 * g;
            X4 hi, lo;
            round_and_rest<T>(acc[d] * inv, hi, lo);
            *reinterpret_cast<X4*>(to + lane_at) = hi;
            if (a.out_lo != nullptr) *reinterpret_cast<X4*>(to_lo + lane_at) = lo;
        }
        if (g == 0 && a.row_max != nullptr) {
            const int64_t row = (static_cast<int64_t>(b) * a.H + h) * a.N;
            (a.row_max + row)[static_cast<uint32_t>(q)] = used;
            (a.row_inv + row)[static_cast<uint32_t>(q)] = inv;
        }
    };
    wait_vmem();
    __syncthreads();
    uint32_t before = 0;  // the window before this one
    for (uint32_t i = begin; i < end; ++i) {
        const int buf = (i - begin) & 1;
        const Place here = p;
        const Operand<T, D> qr = qn;
        const bool more = i + 1 < end;
        if (more) {
            p = places.at(a, o, i + 1);
            fetch(p.b, buf ^ 1);
        }
        if (me.active) {
            if (me.leads && i > begin) finish(before, buf ^ 1);
            before = here.b;
            if (here.kind != kind) {
                kind = here.kind;
                build_tiles<kSpan, kMask, false>(tile, a, h, kind, q, 16 * me.first + 4 * g, side, per_scale);
            }
            const T* vl = v_lds[buf] + me.first * 16 * D;
            const Halves<T> kl(k_lds[buf] + me.first * 16 * D, 16 * D);
            // LDS reads run one step ahead of the products on them
            const auto start = [&](int t) { return kMask ? f32x4{} : tile[t]; };
            Operand<T, D> kr[2];
            const auto read = [&](int t) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    if (t + u < kSpan) kr[u].load_lds(kl.of[u], 16 * t, col, g);
            };
            top = -__builtin_inff();
            read(0);
#pragma unroll
            for (int t = 0; t < kSpan; t += 2) {
                f32x4 s[2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    if (t + u < kSpan) s[u] = multiply<T, D>(kr[u], qr, start(t + u));
                read(t + 2 < kSpan ? t + 2 : 0);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (t + u < kSpan)
                            top = fmaxf(top, kMask ? __builtin_fmaf(s[u][r], a.scale, tile[t + u][r]) : s[u][r]);
                }
                tiles_in_order();
            }
            top = max_groups(top);
            const float used = top == -__builtin_inff() ? 0.0f : top;
            // the sum of the weights as one more row of the product
            f32x4 sum = {};
#pragma unroll
            for (int d = 0; d < kOut; ++d) acc[d] = f32x4{};
            const auto weigh = [&](auto large) {
                const Exponent<kMask, decltype(large)::value> exponent = {a.scale, c2};
                const float off = used * c2;
#pragma unroll
                for (int t = 0; t < kSpan; t += 2) {
                    const int count = t + 1 < kSpan ? 2 : 1;
                    f32x4 s[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        if (u < count) s[u] = multiply<T, D>(kr[u], qr, start(t + u));
                    if (t + 2 < kSpan) read(t + 2);
                    Turned<T, D> vt;
                    vt.load(vl, 16 * t, count, col, g);
                    X4 hi[2], lo[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (u >= count) continue;
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            s[u][r] = __builtin_amdgcn_exp2f(exponent(s[u][r], tile[t + u][r], used, 0.0f, off));
                        split<T>(s[u], hi[u], lo[u]);
                    }
                    if (count == 2) {
                        sum = Mma<T>::mma32(join<T>(ones, ones), join<T>(hi[0], hi[1]), sum);
                        sum = Mma<T>::mma32(join<T>(ones, ones), join<T>(lo[0], lo[1]), sum);
                    } else {
                        sum = Mma<T>::mma16(ones, hi[0], sum);
                        sum = Mma<T>::mma16(ones, lo[0], sum);
                    }
                    vt.add(acc, count, hi);
                    vt.add(acc, count, lo);
                    tiles_in_order();
                }
            };
            if (!kMask && __any(fabsf(used * c2) > kLargeLog2))
                weigh(std::true_type{});
            else
                weigh(std::false_type{});
            total = sum[0];
            if (kSplit > 1 && !me.leads) {
                hand.value(buf, me.part, 0) = top;
                hand.value(buf, me.part, 1) = total;
#pragma unroll
                for (int v = 0; v < 4 * kOut; ++v) hand.value(buf, me.part, 2 + v) = acc[v >> 2][v & 3];
            }
        }
        wait_vmem();
        __syncthreads();
    }
    if (me.active && me.leads && end > begin) finish(before, (end - 1 - begin) & 1);
}

// dq, delta and a range's share of dbias.
template <typename T, int D, int NT, int S, int kSplit, int kWaves, bool kMask>
__global__ void __launch_bounds__(S* kSplit * 64) __attribute__((amdgpu_waves_per_eu(kWaves)))
attn_grad_q_tuned_kernel(const AttnArgs a, const Order o, const Walk w) {
    typedef typename Mma<T>::x4 X4;
    typedef Share<NT, S, kSplit> Mine;
    constexpr int kTile = NT * 16 * D, W = S * kSplit, kOut = D / 16, kSpan = Mine::kSpan;
    typedef Handover<S, kSplit, 4 * kOut> Hand;
    __shared__ __attribute__((aligned(16))) T k_lds[2][kTile];
    __shared__ __attribute__((aligned(16))) T v_lds[2][kTile];
    __shared__ float hand_lds[Hand::kFloats];
    __shared__ uint8_t side[kMask ? 4 : NT * 16];
    uint32_t range, group;
    int h;
    if (!walk_of(a, w, range, group, h)) return;
    const uint32_t begin = range * w.per, end = std::min(a.B, begin + w.per);
    const Mine me(a, group);
    const int col = me.col, g = me.g, q = me.row;
    const Hand hand(hand_lds, me.local, me.lane);
    const float per_scale = 1.0f / a.scale, c2 = a.scale * kLog2e;
    if constexpr (!kMask) token_sides(a, side, std::min(a.N, NT * 16));
    f32x4 tile[kSpan], sums[kSpan] = {};
    uint32_t kind = ~0u;
    // the window ahead: the lane's rows and their statistics
    Operand<T, D> qn, gn, out_n, rest_n;
    float top_n, inv_n;
    const Rows<T, D, NT, W> rows(static_cast<uint32_t>(a.st), a.N);
    const uint32_t mine = static_cast<uint32_t>(q) * static_cast<uint32_t>(a.st);
    const uint32_t mine_out = static_cast<uint32_t>(q) * (a.H * D);
    const auto fetch = [&](uint32_t b, int buf) {
        rows.load(rows_of<T>(a, b, 1, h, D), lds_address(k_lds[0]) + buf * kTile * sizeof(T));
        rows.load(rows_of<T>(a, b, 2, h, D), lds_address(v_lds[0]) + buf * kTile * sizeof(T));
        qn.load(rows_of<T>(a, b, 0, h, D), mine, g);
        const int64_t row = (static_cast<int64_t>(b) * a.H + h) * a.N, at = heads_row<D>(a, b, h);
        gn.load(static_cast<const T*>(a.grad_out) + at, mine_out, g);
        out_n.load(static_cast<const T*>(a.out) + at, mine_out, g);
        rest_n.load(static_cast<const T*>(a.out_lo) + at, mine_out, g);
        top_n = (a.row_max + row)[static_cast<uint32_t>(q)];
        inv_n = (a.row_inv + row)[static_cast<uint32_t>(q)];
    };
    Places<kMask> places(begin, end);
    Place p = places.at(a, o, begin);
    fetch(p.b, 0);
    f32x4 acc[kOut];
    const auto finish = [&](uint32_t b, int copy) {
#pragma unroll
        for (int i = 1; i < kSplit; ++i) {
#pragma unroll
            for (int v = 0; v < 4 * kOut; ++v) acc[v >> 2][v & 3] += hand.value(copy, i, v);
        }
        if (me.row0 >= a.N) return;
        T* to = static_cast<T*>(a.grad_qkv) + (static_cast<int64_t>(b) * a.N * 3 * a.H + h) * D;
#pragma unroll
        for (int d = 0; d < kOut; ++d)
            *reinterpret_cast<X4*>(to + (3 * mine_out + 16 * d + 4 * g)) = round4<T>(acc[d] * a.scale);
    };
    wait_vmem();
    __syncthreads();
    uint32_t before = 0;
    for (uint32_t i = begin; i < end; ++i) {
        const int buf = (i - begin) & 1;
        const Place here = p;
        const Operand<T, D> qr = qn, go = gn;
        const bool more = i + 1 < end;
        const Operand<T, D> out = out_n, rest = rest_n;
        const float top = top_n, inv = inv_n;
        if (more) {
            p = places.at(a, o, i + 1);
            fetch(p.b, buf ^ 1);
        }
        if (me.active) {
            if (me.leads && i > begin) finish(before, buf ^ 1);
            before = here.b;
            if (here.kind != kind) {
                kind = here.kind;
                build_tiles<kSpan, kMask, false>(tile, a, h, kind, q, 16 * me.first + 4 * g, side, per_scale);
            }
            float delta = 0.0f;
#pragma unroll
            for (int e = 0; e < D / 4; ++e) delta = __builtin_fmaf(with_rest<T>(out.v[e], rest.v[e]), go.dim(e), delta);
            delta = sum_groups(delta);
            if (me.leads && g == 0 && me.row0 < a.N)
                (a.delta + (static_cast<int64_t>(here.b) * a.H + h) * a.N)[static_cast<uint32_t>(q)] = delta;
            const float plus = __builtin_amdgcn_logf(inv), off = top * c2 - plus;
#pragma unroll
            for (int d = 0; d < kOut; ++d) acc[d] = f32x4{};
            const T* kt = k_lds[buf] + me.first * 16 * D;
            const Halves<T> kl(kt, 16 * D), vl(v_lds[buf] + me.first * 16 * D, 16 * D);
            const auto walk = [&](auto large) {
                const Exponent<kMask, decltype(large)::value> exponent = {a.scale, c2};
                Operand<T, D> kr[2], vr[2];
                const auto read = [&](int t) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (t + u >= kSpan) continue;
                        kr[u].load_lds(kl.of[u], 16 * t, col, g);
                        vr[u].load_lds(vl.of[u], 16 * t, col, g);
                    }
                };
                read(0);
#pragma unroll
                for (int t = 0; t < kSpan; t += 2) {
                    const int count = t + 1 < kSpan ? 2 : 1;
                    f32x4 s[2], dp[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (u >= count) continue;
                        s[u] = multiply<T, D>(kr[u], qr, kMask ? f32x4{} : tile[t + u]);
                        dp[u] = multiply<T, D>(vr[u], go, f32x4{-delta, -delta, -delta, -delta});
                    }
                    if (t + 2 < kSpan) read(t + 2);
                    Turned<T, D> k_turned;
                    k_turned.load(kt, 16 * t, count, col, g);
                    X4 ds[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (u >= count) continue;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            s[u][r] = __builtin_amdgcn_exp2f(exponent(s[u][r], tile[t + u][r], top, plus, off)) * dp[u][r];
                            sums[t + u][r] += s[u][r];
                        }
                        settled(sums[t + u]);
                        ds[u] = round4<T>(s[u]);
                    }
                    k_turned.add(acc, count, ds);
                    tiles_in_order();
                }
            };
            if (!kMask && __any(fabsf(top * c2) > kLargeLog2))
                walk(std::true_type{});
            else
                walk(std::false_type{});
            if (kSplit > 1 && !me.leads) {
#pragma unroll
                for (int v = 0; v < 4 * kOut; ++v) hand.value(buf, me.part, v) = acc[v >> 2][v & 3];
            }
        }
        wait_vmem();
        __syncthreads();
    }
    if (!me.active) return;
    if (me.leads && end > begin) finish(before, (end - 1 - begin) & 1);
    if (me.row0 >= a.N || a.grad_bias == nullptr) return;
    float* to = a.grad_bias + ((static_cast<int64_t>(range) * a.H + h) * a.N + q) * a.N;
#pragma unroll
    for (int t = 0; t < kSpan; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int k = 16 * (me.first + t) + 4 * g + r;
            if (k < a.N) to[k] = sums[t][r];
        }
    }
}

// dk and dv: a strip is 16 keys, the other axis the queries.
template <typename T, int D, int NT, int S, int kSplit, int kWaves, bool kMask>
__global__ void __launch_bounds__(S* kSplit * 64) __attribute__((amdgpu_waves_per_eu(kWaves)))
attn_grad_kv_tuned_kernel(const AttnArgs a, const Order o, const Walk w) {
    typedef typename Mma<T>::x4 X4;
    typedef Share<NT, S, kSplit> Mine;
    constexpr int kTile = NT * 16 * D, W = S * kSplit, kOut = D / 16, kSpan = Mine::kSpan;
    constexpr int kRows = NT * 16, kEach = (kRows + W * 64 - 1) / (W * 64);
    typedef Handover<S, kSplit, 8 * kOut> Hand;
    __shared__ __attribute__((aligned(16))) T q_lds[2][kTile];
    __shared__ __attribute__((aligned(16))) T o_lds[2][kTile];
    __shared__ float hand_lds[Hand::kFloats];
    // per query: largest score and log2 of 1 / sum (lse: both as one, in units
    // of the accumulator), delta; per wave: whether it saw a large score
    __shared__ float top_lds[2][kRows], plus_lds[2][kRows], lse_lds[kMask ? 1 : 2][kRows], delta_lds[2][kRows];
    __shared__ uint32_t large_lds[2][W];
    __shared__ uint8_t side[kMask ? 4 : kRows];
    uint32_t range, group;
    int h;
    if (!walk_of(a, w, range, group, h)) return;
    const uint32_t begin = range * w.per, end = std::min(a.B, begin + w.per);
    const Mine me(a, group);
    const int col = me.col, g = me.g, k = me.row;
    const Hand hand(hand_lds, me.local, me.lane);
    const float per_scale = 1.0f / a.scale, c2 = a.scale * kLog2e;
    if constexpr (!kMask) token_sides(a, side, std::min(a.N, kRows));
    f32x4 tile[kSpan];
    uint32_t kind = ~0u;
    float top_r[kEach], inv_r[kEach], delta_r[kEach];
    Operand<T, D> kn, vn;
    const Rows<T, D, NT, W> rows(static_cast<uint32_t>(a.st), a.N), out_rows(static_cast<uint32_t>(a.H * D), a.N);
    const uint32_t mine = static_cast<uint32_t>(k) * static_cast<uint32_t>(a.st);
    const auto fetch = [&](uint32_t b, int buf) {
        rows.load(rows_of<T>(a, b, 0, h, D), lds_address(q_lds[0]) + buf * kTile * sizeof(T));
        out_rows.load(static_cast<const T*>(a.grad_out) + heads_row<D>(a, b, h),
                      lds_address(o_lds[0]) + buf * kTile * sizeof(T));
        kn.load(rows_of<T>(a, b, 1, h, D), mine, g);
        vn.load(rows_of<T>(a, b, 2, h, D), mine, g);
        const int64_t row = (static_cast<int64_t>(b) * a.H + h) * a.N;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int r = threadIdx.x + i * W * 64;
            const bool in = r < a.N;
            const uint32_t at = in ? r : a.N - 1;
            top_r[i] = in ? (a.row_max + row)[at] : 0.0f;
            inv_r[i] = in ? (a.row_inv + row)[at] : 0.0f;  // queries past N: log2 0 = -inf, no weight
            delta_r[i] = in ? (a.delta + row)[at] : 0.0f;
        }
    };
    const auto keep = [&](int buf) {
        bool large = false;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int r = threadIdx.x + i * W * 64;
            if (r >= kRows) break;
            const float plus = __builtin_amdgcn_logf(inv_r[i]);
            top_lds[buf][r] = top_r[i];
            plus_lds[buf][r] = plus;
            if constexpr (!kMask) lse_lds[buf][r] = top_r[i] - plus * (1.0f / c2);
            delta_lds[buf][r] = delta_r[i];
            large = large || fabsf(top_r[i] * c2) > kLargeLog2;
        }
        if constexpr (!kMask) {
            large = __any(large);
            if (me.lane == 0) large_lds[buf][threadIdx.x >> 6] = large ? 1 : 0;
        }
    };
    Places<kMask> places(begin, end);
    Place p = places.at(a, o, begin);
    fetch(p.b, 0);
    keep(0);
    f32x4 dk[kOut], dv[kOut];
    const auto finish = [&](uint32_t b, int copy) {
#pragma unroll
        for (int i = 1; i < kSplit; ++i) {
#pragma unroll
            for (int v = 0; v < 4 * kOut; ++v) {
                dk[v >> 2][v & 3] += hand.value(copy, i, v);
                dv[v >> 2][v & 3] += hand.value(copy, i, 4 * kOut + v);
            }
        }
        if (me.row0 >= a.N) return;
        const uint32_t hd = static_cast<uint32_t>(a.H * D);
        T* to = static_cast<T*>(a.grad_qkv) + (static_cast<int64_t>(b) * a.N * 3 * a.H + a.H + h) * D;
#pragma unroll
        for (int d = 0; d < kOut; ++d) {
            const uint32_t at = 3 * hd * static_cast<uint32_t>(k) + 16 * d + 4 * g;
            *reinterpret_cast<X4*>(to + at) = round4<T>(dk[d] * a.scale);
            *reinterpret_cast<X4*>(to + hd + at) = round4<T>(dv[d]);
        }
    };
    wait_vmem();
    __syncthreads();
    uint32_t before = 0;
    for (uint32_t i = begin; i < end; ++i) {
        const int buf = (i - begin) & 1;
        const Place here = p;
        const Operand<T, D> kr = kn, vr = vn;
        const bool more = i + 1 < end;
        if (more) {
            p = places.at(a, o, i + 1);
            fetch(p.b, buf ^ 1);
        }
        if (me.active) {
            if (me.leads && i > begin) finish(before, buf ^ 1);
            before = here.b;
            if (here.kind != kind) {
                kind = here.kind;
                build_tiles<kSpan, kMask, true>(tile, a, h, kind, k, 16 * me.first + 4 * g, side, per_scale);
            }
            const T *qt = q_lds[buf] + me.first * 16 * D, *ot = o_lds[buf] + me.first * 16 * D;
            const Halves<T> ql(qt, 16 * D), ol(ot, 16 * D);
            const int stat = 16 * me.first + 4 * g + (col & 3);
#pragma unroll
            for (int d = 0; d < kOut; ++d) dk[d] = dv[d] = f32x4{};
            const auto walk = [&](auto large) {
                // with a mask tensor, and with large scores, top and plus apart
                constexpr bool kApart = kMask || decltype(large)::value;
                const Exponent<kMask, true> exponent = {a.scale, c2};
                Operand<T, D> qr[2], go[2];
                float top[2], plus[2], delta[2];
                // a lane holds the statistics of query 4 g + col % 4 of a tile
                const auto read = [&](int t) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (t + u >= kSpan) continue;
                        const int at = stat + 16 * (t + u);
                        qr[u].load_lds(ql.of[u], 16 * t, col, g);
                        go[u].load_lds(ol.of[u], 16 * t, col, g);
                        top[u] = kApart ? top_lds[buf][at] : lse_lds[kMask ? 0 : buf][at];
                        if (kApart) plus[u] = plus_lds[buf][at];
                        delta[u] = delta_lds[buf][at];
                    }
                };
                read(0);
#pragma unroll
                for (int t = 0; t < kSpan; t += 2) {
                    const int count = t + 1 < kSpan ? 2 : 1;
                    f32x4 s[2], dp[2];
                    float top_t[2], plus_t[2], delta_t[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (u >= count) continue;
                        s[u] = multiply<T, D>(qr[u], kr, kMask ? f32x4{} : tile[t + u]);
                        dp[u] = multiply<T, D>(go[u], vr, f32x4{});
                        top_t[u] = top[u], delta_t[u] = delta[u];
                        if (kApart) plus_t[u] = plus[u];
                    }
                    if (t + 2 < kSpan) read(t + 2);
                    Turned<T, D> o_turned, q_turned;
                    o_turned.load(ot, 16 * t, count, col, g);
                    q_turned.load(qt, 16 * t, count, col, g);
                    X4 pw[2], ds[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (u >= count) continue;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float e = kApart ? exponent(s[u][r], tile[t + u][r], of_row(top_t[u], r),
                                                              of_row(plus_t[u], r), 0.0f)
                                                   : (s[u][r] - of_row(top_t[u], r)) * c2;
                            s[u][r] = __builtin_amdgcn_exp2f(e);
                            dp[u][r] = (dp[u][r] - of_row(delta_t[u], r)) * s[u][r];
                        }
                        pw[u] = round4<T>(s[u]);
                        ds[u] = round4<T>(dp[u]);
                    }
                    o_turned.add(dv, count, pw);
                    q_turned.add(dk, count, ds);
                    tiles_in_order();
                }
            };
            if (!kMask && __any(me.lane < W && large_lds[buf][me.lane < W ? me.lane : 0] != 0))
                walk(std::true_type{});
            else
                walk(std::false_type{});
            if (kSplit > 1 && !me.leads) {
#pragma unroll
                for (int v = 0; v < 4 * kOut; ++v) {
                    hand.value(buf, me.part, v) = dk[v >> 2][v & 3];
                    hand.value(buf, me.part, 4 * kOut + v) = dv[v >> 2][v & 3];
                }
            }
        }
        if (more) keep(buf ^ 1);
        wait_vmem();
        __syncthreads();
    }
    if (me.active && me.leads && end > begin) finish(before, (end - 1 - begin) & 1);
}

// ---- launchers ------------------------------------------------------------------

template <typename T, int D, int NT, bool kMask>
void launch_forward(const AttnArgs& a, const Order& o, hipStream_t s) {
    constexpr Form f = tuned_form(NT, D, kForwardPass);
    const Walk w = tuned_walk(a.B, a.H, a.N, D, kForwardPass);
    const uint32_t grid = xcd_launch_count(w.groups * static_cast<uint32_t>(a.H) * w.ranges);
    attn_forward_tuned_kernel<T, D, NT, f.strips, f.split, f.per_simd, kMask>
        <<<grid, f.strips * f.split * 64, 0, s>>>(a, o, w);
}

template <typename T, int D, int NT, bool kMask>
void launch_backward(const AttnArgs& a, const Order& o, hipStream_t s) {
    constexpr Form f = tuned_form(NT, D, kQueryPass), e = tuned_form(NT, D, kKeyPass);
    const Walk w = tuned_walk(a.B, a.H, a.N, D, kQueryPass), v = tuned_walk(a.B, a.H, a.N, D, kKeyPass);
    const uint32_t heads = static_cast<uint32_t>(a.H);
    attn_grad_q_tuned_kernel<T, D, NT, f.strips, f.split, f.per_simd, kMask>
        <<<xcd_launch_count(w.groups * heads * w.ranges), f.strips * f.split * 64, 0, s>>>(a, o, w);
    attn_grad_kv_tuned_kernel<T, D, NT, e.strips, e.split, e.per_simd, kMask>
        <<<xcd_launch_count(v.groups * heads * v.ranges), e.strips * e.split * 64, 0, s>>>(a, o, v);
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
