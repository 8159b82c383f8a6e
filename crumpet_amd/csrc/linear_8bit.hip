// A linear layer whose input is kept in 8 bits for the backward pass (gfx950):
//   y = act(x) W^T + b,   dx = (dy W) act'(x^),   dW = dy^T act(x^),   db = sum dy
// with act the identity or the exact GELU and x^ the 8-bit copy of x: for every
// row and 32 columns whole numbers up to 127 times 2^e, e the least integer
// >= -126 with 127 2^e >= the group's largest magnitude.  A power of two makes
// both directions exact: the copy is x rounded to a multiple of 2^e, nothing
// else, and an exponent is one byte.  A group with an infinity or NaN is kept
// as NaN (exponent byte -128).
//
// Kept are 33/32 bytes a value instead of 2 for x and 2 more for act(x).
//
// Products are v_mfma_f32_16x16x32, fp32 accumulation, one rounding at the
// end; act(x) and act(x^) are rounded to the input type once, as operands.
// Weights are the A operand, rows of x the B operand, so a lane ends with 4
// neighbouring output features of one row and x passes from memory straight
// into B fragments: a 32-deep product is one quantisation group, spread over the
// 4 lane groups.  The weights, which a workgroup's waves share, pass through
// LDS.
//
// Measured, with the GELU, 442368 rows of 192 to 48 in fp16: forward 98 us
// (300 MB, 3.1 TB/s, VALU 87% busy: the GELU and the codes are 28 instructions a
// value), dx 103 us (300 MB, VALU 80%), dW and db 98 us (VALU 95%: the GELU
// again) and 7 for their sums, which one chunk of rows does without.  Without it the same forward pass takes 84 us.
// Where products bound it: 27648 rows of 192 to 768 in 32 us (250 TFLOP/s);
// a step's loads are a step ahead of the products, which is too short a time
// for more.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "crumpet_common.h"
#include "crumpet_hip.h"
#include "train_mma.h"

namespace crumpet {
namespace train {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 32;
constexpr int kNaN = -128;  // exponent byte of a group that is not finite

__device__ __forceinline__ float power_of_two(int e) {
    return e == kNaN ? __builtin_nanf("") : __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// GELU(x) = x Phi(x) and its derivative Phi(x) + x phi(x), with the normal
// distribution from its tail, Phi(-|x|) = erfc(|x| / sqrt 2) / 2 = u(t)
// exp(-x^2 / 2), t = 1 / (1 + p |x| / sqrt 2): formula 7.1.26 of Abramowitz &
// Stegun, Handbook of Mathematical Functions (|error| of erfc <= 1.5e-7, far
// below a 16-bit result's rounding).  The arithmetic of these two bounds the
// kernels, so it is written for few instructions.
struct Tail {
    float u, bell;
    __device__ __forceinline__ explicit Tail(float x) {
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f * 0.70710678f, fabsf(x), 1.0f));
        float p = __builtin_fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
        p = __builtin_fmaf(p, t, 0.5f * 1.421413741f);
        p = __builtin_fmaf(p, t, 0.5f * -0.284496736f);
        p = __builtin_fmaf(p, t, 0.5f * 0.254829592f);
        u = p * t;
        bell = __builtin_amdgcn_exp2f(x * x * (-0.5f * kLog2e));
    }
};
template <bool kGelu>
__device__ __forceinline__ float act(float x) {
    if constexpr (kGelu) {
        const Tail n(x);
        const float low = n.u * n.bell;
        return x * (x > 0.0f ? 1.0f - low : low);
    }
    return x;
}
template <bool kGelu>
__device__ __forceinline__ float act_grad(float x) {
    if constexpr (kGelu) {
        // 1/2 +- (1/2 - Phi(-|x|) + |x| phi(x)), phi(x) = bell / sqrt(2 pi)
        const Tail n(x);
        return 0.5f + copysignf(__builtin_fmaf(n.bell, __builtin_fmaf(0.39894228f, fabsf(x), -n.u), 0.5f), x);
    }
    return 1.0f;
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// The V at a 32-bit byte offset of the lane's from a base of the workgroup's,
// which keeps the address out of the lane's arithmetic.
template <typename V, typename P>
__device__ __forceinline__ __attribute__((address_space(1))) V& at(P* base, uint32_t bytes) {
    typedef std::conditional_t<std::is_const_v<P>, const char, char> Byte;
    typedef __attribute__((address_space(1))) Byte GlobalByte;
    typedef __attribute__((address_space(1))) V GlobalV;
    return *(GlobalV*)((GlobalByte*)(base) + bytes);
}

// Codes of 8 of a group's 32 values (the other lanes of the row hold the
// rest), and the group's exponent.  Magnitudes compare as their 16 bits, NaN
// above everything.
template <typename T>
__device__ __forceinline__ u32x2 quantise(typename Mma<T>::x8 v, int& e) {
    const u32x4 raw = __builtin_bit_cast(u32x4, v);
    uint32_t top = 0;  // in the upper half
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t hi = raw[i] & 0x7fff0000u, lo = (raw[i] & 0x7fffu) << 16, more = hi > lo ? hi : lo;
        top = top > more ? top : more;
    }
    top = max_groups(top);
    const uint32_t bits =
        __float_as_uint(static_cast<float>(__builtin_bit_cast(T, static_cast<unsigned short>(top >> 16))));
    // the largest magnitude is 1.f 2^k; 127 = 1.984375 2^6
    const int k = static_cast<int>(bits >> 23) - 127;
    e = k - ((bits & 0x7fffffu) > 0x7e0000u ? 5 : 6);
    e = e < -126 ? -126 : e;
    if (bits >= 0x7f800000u) {
        e = kNaN;
        return u32x2{};
    }
    const float up = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    // x 2^-e + 1.5 2^23 is the rounded code in the low bits of the mantissa
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        c[i] = __float_as_uint(__builtin_fmaf(static_cast<float>(v[i]), up, 12582912.0f));
    u32x2 codes;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t lo = __builtin_amdgcn_perm(c[4 * i + 1], c[4 * i], 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(c[4 * i + 3], c[4 * i + 2], 0x0c0c0400u);
        codes[i] = hi << 16 | lo;
    }
    return codes;
}

// Four codes times the group's step: (code + 128) step - 128 step, exact, with
// one conversion of an unsigned byte each.  In the last groups 128 steps
// overflow fp32 (bf16), and the copy of a number next to the type's largest is
// rounded up to what the type does not hold (64 2^10, 64 2^122): as an operand
// it is the largest number.
template <typename T>
__device__ __forceinline__ f32x4 values_of(uint32_t codes, float step) {
    constexpr bool kHalf = std::is_same_v<T, _Float16>;
    constexpr float kLate = kHalf ? 0x1p10f : 0x1p121f, kMost = kHalf ? 65504.0f : 0x1.fep127f;
    const uint32_t u = codes ^ 0x80808080u;
    f32x4 v;
    if (step >= kLate) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = (static_cast<float>((u >> (8 * i)) & 0xffu) - 128.0f) * step;
            v[i] = fminf(fmaxf(x, -kMost), kMost);
        }
        return v;
    }
    const float less = -128.0f * step;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(static_cast<float>((u >> (8 * i)) & 0xffu), step, less);
    return v;
}

struct RowsArgs {
    const void* x;        // [rows, K]
    const void* w;        // [n_out, K]
    const void* b;        // [n_out] or null
    void* y;              // [rows, n_out]
    int8_t* codes;        // forward: [rows, K] or null; backward: [rows, n_out], read
    int8_t* exps;         // [rows, ceil(columns / 32)]
    int64_t rows;
    int32_t K, n_out;
};

constexpr int kStep = 2 * kGroup;  // columns of a step

// A step's weights in LDS: row 16 n + m is feature 4 NT (m / 4) + 4 n + m % 4 of
// the block, so that a lane ends with 4 NT neighbouring features of its row.
// The 16-byte pieces of a row are permuted by it, so that 8 lanes of a fragment
// read meet distinct banks.  Straight from memory: load j fills rows 8 j .. + 7.
template <typename T, int NT>
struct Weights {
    static constexpr int kEach = (2 * NT + 3) / 4;
    const T* first;
    uint32_t bytes;
    int wave, piece, row[kEach];
    __device__ __forceinline__ Weights(const RowsArgs& a, int n0, int lane) {
        wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
        first = static_cast<const T*>(a.w) + static_cast<int64_t>(n0) * a.K;
        const int features = std::min(16 * NT, a.n_out - n0);
        bytes = static_cast<uint32_t>(features) * a.K * sizeof(T);
        piece = ((lane & 7) ^ (lane >> 3)) * 8;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int at = 8 * (wave + 4 * i) + (lane >> 3), n = at >> 4, m = at & 15;
            row[i] = std::min(4 * NT * (m >> 2) + 4 * n + (m & 3), features - 1) * a.K;
        }
    }
    __device__ __forceinline__ void load(const RowsArgs& a, T* to, int k0) const {
        const u32x4 buffer = buffer_of(first, bytes);
        const uint32_t lds = lds_address(to);
        const int k = std::min(k0 + piece, a.K - 8);  // a short step's pieces past K: some other of the row
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (wave + 4 * i < 2 * NT) load_to_lds(buffer, lds + (wave + 4 * i) * 1024, (row[i] + k) * sizeof(T));
    }
    static __device__ __forceinline__ int fragment(int s, int n, int col, int g) {
        return (16 * n + col) * kStep + ((4 * s + g) ^ (col & 7)) * 8;
    }
};

// y = f(x) w^T.  Forward: f = act, the bias added, codes written by the first
// column block.  Backward (x = dy, w = W^T): y times act' of the codes at y's
// place.  A wave owns 16 R rows, a workgroup 64 R rows and 16 NT columns; all
// addresses are a base of the workgroup's and a 32-bit offset of the lane's
// that the loops leave alone.
template <typename T, int NT, int R, bool kGelu, bool kForward>
__global__ void __launch_bounds__(kThreads) linear_8bit_rows_kernel(const RowsArgs a, uint32_t row_blocks, uint32_t blocks) {
    typedef typename Mma<T>::x4 X4;
    typedef typename Mma<T>::x8 X8;
    __shared__ __attribute__((aligned(16))) T w_lds[2][NT * 16 * kStep];
    uint32_t id;
    if (!xcd_chunk(blockIdx.x, gridDim.x, row_blocks * blocks, id)) return;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int n0 = static_cast<int>(id % blocks) * 16 * NT;
    const int64_t block0 = static_cast<int64_t>(id / blocks) * 64 * R;
    const int row0 = (threadIdx.x >> 6) * 16 * R + col;
    const int rows = static_cast<int>(std::min<int64_t>(64 * R, a.rows - block0));
    const int groups = (a.K + kGroup - 1) / kGroup;
    const bool keep = kForward && n0 == 0 && a.codes != nullptr;
    const T* x_at = static_cast<const T*>(a.x) + block0 * a.K;
    uint32_t x_of[R];
#pragma unroll
    for (int r = 0; r < R; ++r) x_of[r] = (std::min(row0 + 16 * r, rows - 1) * a.K + 8 * g) * sizeof(T);
    Weights<T, NT> weights(a, n0, lane);
    const int out_groups = (a.n_out + kGroup - 1) / kGroup;
    const int f0 = 4 * NT * g;  // the lane's features, from n0
    T* y_at = static_cast<T*>(a.y) + block0 * a.n_out + n0;
    // two tiles are 8 neighbouring features of one group: 16 bytes, aligned where
    // NT is even
    constexpr int kEach = NT % 2 == 0 ? 2 : 1;
    const auto place = [&](int n, int r) { return static_cast<uint32_t>((row0 + 16 * r) * a.n_out + f0 + 4 * n); };
    // the backward pass' codes, on their way while the products are formed
    uint32_t codes[NT][R] = {};
    int8_t exps[NT][R] = {};
    if constexpr (!kForward && kGelu) {
        const int8_t* codes_at = a.codes + block0 * a.n_out + n0;
        const int8_t* exps_at = a.exps + block0 * out_groups;
#pragma unroll
        for (int n = 0; n < NT; n += kEach) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (row0 + 16 * r >= rows || n0 + f0 + 4 * n >= a.n_out) continue;
                exps[n][r] = at<const int8_t>(exps_at, (row0 + 16 * r) * out_groups + (n0 + f0 + 4 * n) / kGroup);
                if constexpr (kEach == 2) {
                    if (n0 + f0 + 4 * n + 4 < a.n_out) {
                        const u32x2 both = at<const u32x2>(codes_at, place(n, r));
                        codes[n][r] = both[0], codes[n + 1][r] = both[1];
                        continue;
                    }
                }
                codes[n][r] = at<const uint32_t>(codes_at, place(n, r));
            }
        }
    }
    // Two groups a step, so that a row's 128-byte lines are read at once, x and
    // the weights a step ahead.  K is a multiple of 16: the last step may be
    // short.
    X8 xv[2][R];
    const auto fetch = [&](int k0) {
        weights.load(a, w_lds[k0 / kStep & 1], k0);
        // a new scalar base each time, not a vector pointer that is advanced
        asm volatile("" : "+s"(x_at));
        if (k0 + kStep <= a.K) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int s = 0; s < 2; ++s) xv[s][r] = at<const X8>(x_at + k0 + s * kGroup, x_of[r]);
            }
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    xv[s][r] = X8{};
                    if (k0 + s * kGroup + 8 * g < a.K) xv[s][r] = at<const X8>(x_at + k0 + s * kGroup, x_of[r]);
                }
            }
        }
    };
    f32x4 acc[NT][R] = {};
    fetch(0);
    for (int k0 = 0; k0 < a.K; k0 += kStep) {
        wait_vmem();
        __syncthreads();
        X8 x[2][R];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int r = 0; r < R; ++r) x[s][r] = xv[s][r];
        }
        if constexpr (kForward) {
            // before the next step's loads, so that the wait for them does not
            // begin with these stores
            if (keep) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int k = k0 + s * kGroup;
                    if (k >= a.K) break;
                    int8_t* codes_at = a.codes + block0 * a.K + k;
                    int8_t* exps_at = a.exps + block0 * groups + k / kGroup;
                    asm volatile("" : "+s"(codes_at), "+s"(exps_at));
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        int e;
                        const u32x2 codes = quantise<T>(x[s][r], e);
                        if (row0 + 16 * r < rows) {
                            if (k + 8 * g < a.K) at<u32x2>(codes_at, x_of[r] / sizeof(T)) = codes;
                            if (g == 0) at<int8_t>(exps_at, (row0 + 16 * r) * groups) = static_cast<int8_t>(e);
                        }
                    }
                }
            }
        }
        if (k0 + kStep < a.K) fetch(k0 + kStep);
        const T* tile = w_lds[k0 / kStep & 1];
        const bool whole = k0 + kStep <= a.K;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (k0 + s * kGroup >= a.K) break;
            if constexpr (kForward && kGelu) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[s][r][i] = static_cast<T>(act<true>(static_cast<float>(x[s][r][i])));
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                X8 w = *reinterpret_cast<const X8*>(tile + weights.fragment(s, n, col, g));
                // past K lies some other weight, which zeros in x need not silence
                if (!whole && k0 + s * kGroup + 8 * g >= a.K) w = X8{};
#pragma unroll
                for (int r = 0; r < R; ++r) acc[n][r] = Mma<T>::mma32(w, x[s][r], acc[n][r]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; n += kEach) {
        if (n0 + f0 + 4 * n >= a.n_out) continue;
        const bool pair = kEach == 2 && n0 + f0 + 4 * n + 4 < a.n_out;
        f32x4 b[kEach] = {};
        if constexpr (kForward) {
            if (a.b != nullptr) {
                const T* b_at = static_cast<const T*>(a.b) + n0;
                b[0] = wide4<T>(at<const X4>(b_at, (f0 + 4 * n) * sizeof(T)));
                if constexpr (kEach == 2)
                    if (pair) b[1] = wide4<T>(at<const X4>(b_at, (f0 + 4 * n + 4) * sizeof(T)));
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (row0 + 16 * r >= rows) continue;
            f32x4 v[kEach];
#pragma unroll
            for (int u = 0; u < kEach; ++u) v[u] = acc[n + u][r] + b[u];
            if constexpr (!kForward && kGelu) {
                const float step = power_of_two(exps[n][r]);
#pragma unroll
                for (int u = 0; u < kEach; ++u) {
                    const f32x4 x = values_of<T>(codes[n + u][r], step);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[u][i] *= act_grad<true>(x[i]);
                }
            }
            const X4 lo = round4<T>(v[0]);
            if constexpr (kEach == 2) {
                if (pair) {
                    at<X8>(y_at, place(n, r) * sizeof(T)) = __builtin_shufflevector(lo, round4<T>(v[1]), 0, 1, 2, 3, 4, 5, 6, 7);
                    continue;
                }
            }
            at<X4>(y_at, place(n, r) * sizeof(T)) = lo;
        }
    }
}

// out [K, n] = in [n, K]; 32 x 32 tiles through LDS.
template <typename T>
__global__ void __launch_bounds__(kThreads) transpose_kernel(T* __restrict__ out, const T* __restrict__ in, int32_t n, int32_t K) {
    __shared__ T tile[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int k0 = blockIdx.x * 32, n0 = blockIdx.y * 32;
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        if (n0 + y + i < n && k0 + x < K) tile[y + i][x] = in[static_cast<int64_t>(n0 + y + i) * K + k0 + x];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        if (k0 + y + i < K && n0 + x < n) out[static_cast<int64_t>(k0 + y + i) * n + n0 + x] = tile[x][y + i];
}

struct WeightArgs {
    const void* dy;          // [rows, n_out]
    const int8_t* codes;     // [rows, K]
    const int8_t* exps;
    float* partial;          // [chunks, n_out K + n_out], or null with one chunk:
    void *dw, *db;           // the results, each or null
    int64_t rows, per;       // rows of a chunk
    int32_t K, n_out;
    uint32_t kblocks, nblocks;
};

// A chunk of rows' share of a 64 x 128 tile of dW = dy^T act(x^), and of db.
// Both operands are read along the rows, so they pass through LDS, row-major,
// and come back by transpose reads; the depth's order is the same permutation
// on both sides.  The codes become act(x^) on their way into LDS, once for
// each value and column block.
template <typename T, bool kGelu>
__global__ void __launch_bounds__(kThreads) linear_8bit_weight_kernel(const WeightArgs a) {
    typedef typename Mma<T>::x4 X4;
    typedef typename Mma<T>::x8 X8;
    constexpr int kRows = 64, kN = 64, kK = 128, kLdN = kN + 8, kLdK = kK + 8;
    __shared__ __attribute__((aligned(16))) T dy_lds[kRows * kLdN];
    __shared__ __attribute__((aligned(16))) T x_lds[kRows * kLdK];
    uint32_t id = blockIdx.x;
    const uint32_t kb = id % a.kblocks;
    id /= a.kblocks;
    const int n0 = static_cast<int>(id % a.nblocks) * kN, k0 = static_cast<int>(kb) * kK;
    const int64_t chunk = id / a.nblocks;
    const int64_t begin = chunk * a.per, end = std::min<int64_t>(a.rows, begin + a.per);
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    const int groups = (a.K + kGroup - 1) / kGroup;
    const bool sum_dy = kb == 0 && wave == 0;
    f32x4 acc[4][2] = {}, db[4] = {};
    X8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = static_cast<T>(1.0f);
    // the rows of the next step, on their way while this one's are multiplied
    X8 dy_next[2];
    u32x4 codes_next[2];
    int e_next[2];
    // addresses: a base of the step's and an offset of the lane's
    uint32_t dy_of[2], x_of[2], e_of[2];
    bool dy_in[2], x_in[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int p = threadIdx.x + i * kThreads, r = p >> 3, c = p & 7;
        dy_of[i] = (r * a.n_out + c * 8) * sizeof(T), dy_in[i] = n0 + c * 8 < a.n_out;
        x_of[i] = r * a.K + c * 16, x_in[i] = k0 + c * 16 < a.K;
        e_of[i] = r * groups + c / 2;
    }
    const auto fetch = [&](int64_t r0) {
        const T* dy_at = static_cast<const T*>(a.dy) + r0 * a.n_out + n0;
        const int8_t* x_at = a.codes + r0 * a.K + k0;
        const int8_t* e_at = a.exps + r0 * groups + k0 / kGroup;
        asm volatile("" : "+s"(dy_at), "+s"(x_at), "+s"(e_at));
        const int rows = static_cast<int>(std::min<int64_t>(kRows, end - r0));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            dy_next[i] = X8{};
            codes_next[i] = u32x4{};
            e_next[i] = 0;
            if ((threadIdx.x + i * kThreads) >> 3 >= rows) continue;
            if (dy_in[i]) dy_next[i] = at<const X8>(dy_at, dy_of[i]);
            if (x_in[i]) {
                codes_next[i] = at<const u32x4>(x_at, x_of[i]);
                e_next[i] = at<const int8_t>(e_at, e_of[i]);
            }
        }
    };
    if (begin < end) fetch(begin);
    for (int64_t r0 = begin; r0 < end; r0 += kRows) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int p = threadIdx.x + i * kThreads, r = p >> 3, c = p & 7;
            *reinterpret_cast<X8*>(dy_lds + r * kLdN + c * 8) = dy_next[i];
            X8 v[2];
            const float step = power_of_two(e_next[i]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const f32x4 x = values_of<T>(codes_next[i][w], step);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[w >> 1][4 * (w & 1) + e] = static_cast<T>(act<kGelu>(x[e]));
            }
            *reinterpret_cast<X8*>(x_lds + r * kLdK + c * 16) = v[0];
            *reinterpret_cast<X8*>(x_lds + r * kLdK + c * 16 + 8) = v[1];
        }
        if (r0 + kRows < end) fetch(r0 + kRows);
        __syncthreads();
#pragma unroll
        for (int s = 0; s < kRows; s += 32) {
            X8 av[4], bv[2];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const X4 lo = load_transposed<T>(dy_lds, kLdN, s, 16 * n, col, g);
                const X4 hi = load_transposed<T>(dy_lds, kLdN, s + 16, 16 * n, col, g);
                av[n] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int c = 32 * wave + 16 * t;
                const X4 lo = load_transposed<T>(x_lds, kLdK, s, c, col, g);
                const X4 hi = load_transposed<T>(x_lds, kLdK, s + 16, c, col, g);
                bv[t] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                if (sum_dy) db[n] = Mma<T>::mma32(av[n], ones, db[n]);
#pragma unroll
                for (int t = 0; t < 2; ++t) acc[n][t] = Mma<T>::mma32(av[n], bv[t], acc[n][t]);
            }
        }
    }
    const auto put = [&](auto* weights, auto* sums) {
        typedef std::remove_reference_t<decltype(*sums)> To;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int f = n0 + 16 * n + 4 * g + r;
                if (f >= a.n_out) continue;
                if (weights != nullptr) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int k = k0 + 32 * wave + 16 * t + col;
                        if (k < a.K) weights[static_cast<int64_t>(f) * a.K + k] = static_cast<To>(acc[n][t][r]);
                    }
                }
                if (sum_dy && col == 0 && sums != nullptr) sums[f] = static_cast<To>(db[n][r]);
            }
        }
    };
    if (a.partial == nullptr) {
        put(static_cast<T*>(a.dw), static_cast<T*>(a.db));
        return;
    }
    float* to = a.partial + chunk * (static_cast<int64_t>(a.n_out) * a.K + a.n_out);
    put(to, to + static_cast<int64_t>(a.n_out) * a.K);
}

// Sums of the chunks: 32 numbers by 8 groups of chunks per workgroup, each group
// and then the groups in order; the first `weights` sums go to dw, the rest to
// db.
template <typename T>
__global__ void __launch_bounds__(kThreads) linear_8bit_join_kernel(T* dw, T* db, const float* __restrict__ partial,
                                                                   int64_t weights, int64_t all, int64_t chunks) {
    __shared__ float lds[8][33];
    const int x = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + x;
    float v = 0.0f;
    if (i < all) {
#pragma unroll 8
        for (int64_t c = part; c < chunks; c += 8) v += partial[c * all + i];
    }
    lds[part][x] = v;
    __syncthreads();
    if (part != 0 || i >= all) return;
    v = 0.0f;
#pragma unroll
    for (int p = 0; p < 8; ++p) v += lds[p][x];
    if (i < weights) {
        if (dw != nullptr) dw[i] = static_cast<T>(v);
    } else if (db != nullptr) {
        db[i - weights] = static_cast<T>(v);
    }
}

template <typename T, int R, bool kGelu, bool kForward>
int rows_launch(const RowsArgs& a, hipStream_t s) {
    // Tiles of a block at the most.  A GELU on the way in is computed by every
    // column block, so they are wide (110592 rows of 384 to 96: 58 us for 84 with
    // 4); otherwise registers for more waves count (442368 rows of 48 to 192, dx:
    // 117 us with 4, 129 with 6).
    constexpr int kMost = kForward && kGelu && R == 2 ? 8 : 4;
    const int tiles = a.n_out / 16;
    const uint32_t row_blocks = static_cast<uint32_t>((a.rows + 64 * R - 1) / (64 * R));
    const int blocks = (tiles + kMost - 1) / kMost, nt = (tiles + blocks - 1) / blocks;
    const uint32_t grid = xcd_launch_count(row_blocks * static_cast<uint32_t>(blocks));
#define CRUMPET_ROWS(NT)                                                                                             \
    case NT:                                                                                                         \
        if constexpr (NT <= kMost)                                                                                   \
            linear_8bit_rows_kernel<T, NT, R, kGelu, kForward><<<grid, kThreads, 0, s>>>(                            \
                a, row_blocks, static_cast<uint32_t>(blocks));                                                       \
        break;
    switch (nt) {
        CRUMPET_ROWS(1) CRUMPET_ROWS(2) CRUMPET_ROWS(3) CRUMPET_ROWS(4) CRUMPET_ROWS(5) CRUMPET_ROWS(6)
        CRUMPET_ROWS(7) CRUMPET_ROWS(8)
    }
#undef CRUMPET_ROWS
    return check_launch("linear_8bit");
}

// Rows of a wave: 32, or 16 where the wider grid would leave compute units with
// fewer than two workgroups and a step's latency is what counts.  Features 1536
// to 384, no activation: 864 rows 47 us against 27, 6912 rows (162 workgroups) 53
// against 38; 110592 rows of 384 to 96 (864 workgroups) 51 against 52, and with
// the GELU, which narrower blocks repeat, 62 against 79.
template <typename T, bool kGelu, bool kForward>
int rows_product(const RowsArgs& a, hipStream_t s) {
    const int64_t wide = (a.rows + 127) / 128 * ((a.n_out + 127) / 128);
    return wide < 512 ? rows_launch<T, 1, kGelu, kForward>(a, s) : rows_launch<T, 2, kGelu, kForward>(a, s);
}

struct Split {
    uint32_t kblocks, nblocks;
    int64_t chunks, per;
};
Split split_rows(int64_t rows, int64_t K, int64_t n_out) {
    Split p;
    p.kblocks = static_cast<uint32_t>((K + 127) / 128);
    p.nblocks = static_cast<uint32_t>((n_out + 63) / 64);
    // about 1024 workgroups, none with fewer than 256 rows
    const int64_t want = std::max<int64_t>(1, 1024 / (static_cast<int64_t>(p.kblocks) * p.nblocks));
    const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>(want, (rows + 255) / 256));
    p.per = ((rows + chunks - 1) / chunks + 63) / 64 * 64;
    p.chunks = std::max<int64_t>(1, (rows + p.per - 1) / p.per);
    return p;
}

int check(int32_t dtype, int64_t rows, int64_t K, int64_t n_out, int32_t activation, const char* what) {
    if (dtype != CRUMPET_DTYPE_F16 && dtype != CRUMPET_DTYPE_BF16)
        return fail(dtype == CRUMPET_DTYPE_F32 ? CRUMPET_ERR_UNSUPPORTED : CRUMPET_ERR_INVALID_ARGUMENT,
                    "%s: dtype must be float16 or bfloat16", what);
    if (rows < 0 || K < 0 || n_out < 0) return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: negative size", what);
    if (activation != 0 && activation != 1)
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: activation is 0 (none) or 1 (gelu)", what);
    if (K < 16 || n_out < 16 || K % 16 != 0 || n_out % 16 != 0 || K > 65536 || n_out > 65536)
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: features in (%lld) and out (%lld) must be multiples of 16 up to 65536",
                    what, (long long)K, (long long)n_out);
    const uint64_t row_blocks = (static_cast<uint64_t>(rows) + 127) / 128;
    // blocks of 4 tiles at the least
    if (!launch_takes(row_blocks * ((std::max(K, n_out) / 16 + 3) / 4) + kNumXcd, kThreads))
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: too many rows for one launch", what);
    return CRUMPET_OK;
}

bool misaligned(std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return true;
    return false;
}

template <typename T>
int backward(void* dx, void* dw, void* db, const void* dy, const int8_t* codes, const int8_t* exps, int64_t rows,
             int64_t K, int64_t n_out, const void* w, int32_t activation, char* workspace, hipStream_t s) {
    const int32_t k = static_cast<int32_t>(K), n = static_cast<int32_t>(n_out);
    if (dx != nullptr) {
        T* wt = reinterpret_cast<T*>(workspace);
        transpose_kernel<T><<<dim3((k + 31) / 32, (n + 31) / 32), kThreads, 0, s>>>(wt, static_cast<const T*>(w), n, k);
        RowsArgs a = {};
        a.x = dy, a.w = wt, a.y = dx, a.rows = rows, a.K = n, a.n_out = k;
        a.codes = const_cast<int8_t*>(codes), a.exps = const_cast<int8_t*>(exps);
        const int rc = activation ? rows_product<T, true, false>(a, s) : rows_product<T, false, false>(a, s);
        if (rc != CRUMPET_OK) return rc;
    }
    if (dw == nullptr && db == nullptr) return CRUMPET_OK;
    const Split p = split_rows(rows, K, n_out);
    WeightArgs a = {};
    a.dy = dy, a.codes = codes, a.exps = exps, a.rows = rows, a.per = p.per, a.K = k, a.n_out = n;
    a.dw = dw, a.db = db;
    if (p.chunks > 1) a.partial = reinterpret_cast<float*>(workspace + (K * n_out * 2 + 255) / 256 * 256);
    a.kblocks = p.kblocks, a.nblocks = p.nblocks;
    const uint32_t grid = static_cast<uint32_t>(p.chunks) * p.kblocks * p.nblocks;
    if (activation)
        linear_8bit_weight_kernel<T, true><<<grid, kThreads, 0, s>>>(a);
    else
        linear_8bit_weight_kernel<T, false><<<grid, kThreads, 0, s>>>(a);
    if (p.chunks == 1) return check_launch("linear_8bit_backward");
    const int64_t all = n_out * K + n_out;
    linear_8bit_join_kernel<T><<<static_cast<uint32_t>((all + 31) / 32), kThreads, 0, s>>>(
        static_cast<T*>(dw), static_cast<T*>(db), a.partial, n_out * K, all, p.chunks);
    return check_launch("linear_8bit_backward");
}

}  // namespace
}  // namespace train
}  // namespace crumpet

using namespace crumpet;
using namespace crumpet::train;

extern "C" int crumpet_linear_8bit(void* y, int8_t* codes, int8_t* exponents, const void* x, int32_t dtype,
                                   int64_t rows, int64_t K, const void* weight, const void* bias, int64_t n_out,
                                   int32_t activation, void* stream) {
    const char* what = "linear_8bit";
    const int st = train::check(dtype, rows, K, n_out, activation, what);
    if (st != CRUMPET_OK || rows == 0) return st;
    if (y == nullptr || x == nullptr || weight == nullptr || (codes == nullptr) != (exponents == nullptr))
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: null tensor", what);
    if (train::misaligned({y, codes, x, weight, bias}))
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: pointers must be 16-byte aligned", what);
    RowsArgs a = {};
    a.x = x, a.w = weight, a.b = bias, a.y = y, a.codes = codes, a.exps = exponents;
    a.rows = rows, a.K = static_cast<int32_t>(K), a.n_out = static_cast<int32_t>(n_out);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == CRUMPET_DTYPE_F16)
        return activation ? rows_product<_Float16, true, true>(a, s) : rows_product<_Float16, false, true>(a, s);
    return activation ? rows_product<__bf16, true, true>(a, s) : rows_product<__bf16, false, true>(a, s);
}

extern "C" int64_t crumpet_linear_8bit_workspace(int64_t rows, int64_t K, int64_t n_out) {
    if (train::check(CRUMPET_DTYPE_F16, rows, K, n_out, 0, "linear_8bit_workspace") != CRUMPET_OK) return -1;
    if (rows == 0) return 0;
    return (K * n_out * 2 + 255) / 256 * 256 + split_rows(rows, K, n_out).chunks * (n_out * K + n_out) * 4;
}

extern "C" int crumpet_linear_8bit_backward(void* grad_x, void* grad_weight, void* grad_bias, const void* grad_y,
                                            int32_t dtype, const int8_t* codes, const int8_t* exponents, int64_t rows,
                                            int64_t K, const void* weight, int64_t n_out, int32_t activation,
                                            void* workspace, void* stream) {
    const char* what = "linear_8bit_backward";
    const int st = train::check(dtype, rows, K, n_out, activation, what);
    if (st != CRUMPET_OK || rows == 0) return st;
    if (grad_y == nullptr || codes == nullptr || exponents == nullptr || weight == nullptr || workspace == nullptr)
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: null tensor", what);
    if (train::misaligned({grad_x, grad_y, codes, weight, workspace}))
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: pointers must be 16-byte aligned", what);
    char* ws = static_cast<char*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == CRUMPET_DTYPE_F16)
        return train::backward<_Float16>(grad_x, grad_weight, grad_bias, grad_y, codes, exponents, rows, K, n_out,
                                         weight, activation, ws, s);
    return train::backward<__bf16>(grad_x, grad_weight, grad_bias, grad_y, codes, exponents, rows, K, n_out, weight,
                                   activation, ws, s);
}
