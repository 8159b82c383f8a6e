// The residual sum of a block's branch with the norms around it (gfx950), over
// rows of C channels in S samples:
//   y' = post ? norm(y) w_p + b_p : y
//   x1 = x + k[sample] gate y',   h = norm(x1) w + b
// with norm a LayerNorm or an RMS norm, and its gradients.
//
// Everything is bound by HBM: one pass each way, a row in the registers of a
// group of lanes (8 to 64 lanes of a wave, or the workgroup), 8 channels a
// lane and load where C allows.  The backward pass reads x and y again and
// computes x1 and both norms anew, so that nothing but the inputs is kept for
// it and no rounded sum enters the gradients: x1 and h come from the same fp32
// values, each rounded once.  Sums over channels and rows are fp32, in a fixed
// order: each workgroup sums its rows' parameter gradients in registers and
// writes one row of partial sums, which a second kernel adds up.
//
// Measured: [4, 110592, 48], fp32 stream and fp16 branch, layer norm, drop path:
// forward 46 us (255 MB, 5.5 TB/s), gradients 78 us (382 MB, 4.9 TB/s), their
// sums 5.  [3, 4001, 768] bf16, rms norms before and after, a gate a sample:
// forward 18 us (74 MB, 4.1 TB/s), gradients 48 us (111 MB, 2.3 TB/s): 252
// registers a lane leave two waves to a SIMD, and six to twelve rows to a wave
// are too few to hide the chain of two norms and their gradients.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "crumpet_common.h"
#include "crumpet_hip.h"

namespace crumpet {
namespace {

constexpr int kThreads = 256;
constexpr int kSums = 5;  // w, b, gate, w_p, b_p

struct NormArgs {
    const void *x, *y;
    const float *pw, *pb, *gate, *scale, *w, *b;  // each may be null but w
    void *sum, *out;                              // forward
    const void *gsum, *gout;                      // backward; gsum or gout may be null
    void *gx, *gy;
    float* partial;                               // [S * chunks, kSums, C]
    uint32_t S, T, chunks;                        // samples, rows of a sample, workgroups of a sample
    int32_t C;
    int32_t gate_stride;                          // 0 or C
    int32_t post, rms;
    float eps, post_eps;
};

template <typename T, int E>
__device__ __forceinline__ void load_row(const T* p, float* v) {
    if constexpr (E == 1) {
        v[0] = static_cast<float>(p[0]);
    } else {
        typedef T TE __attribute__((ext_vector_type(E)));
        const TE t = *reinterpret_cast<const TE*>(p);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = static_cast<float>(t[e]);
    }
}
template <typename T, int E>
__device__ __forceinline__ void store_row(T* p, const float* v) {
    if constexpr (E == 1) {
        p[0] = static_cast<T>(v[0]);
    } else {
        typedef T TE __attribute__((ext_vector_type(E)));
        TE t;
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = static_cast<T>(v[e]);
        *reinterpret_cast<TE*>(p) = t;
    }
}

// v plus that of another lane: DPP within 16 lanes, half-wave swaps beyond, which
// take a few cycles where a shuffle through LDS takes dozens; a row's sums follow
// one on another.
template <int kCtrl>
__device__ __forceinline__ float add_dpp(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xf, 0xf, true));
}
__device__ __forceinline__ float add_halves(float v, bool of_32) {
    const uint32_t bits = __float_as_uint(v);
    const auto both = of_32 ? __builtin_amdgcn_permlane32_swap(bits, bits, false, false)
                            : __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}

// Sum over the G lanes of a row; G = 256 takes a round through LDS.
template <int G>
__device__ __forceinline__ float row_sum(float v, float* lds) {
    static_assert(G == 8 || G == 16 || G == 32 || G == 64 || G == 256);
    v = add_dpp<0xb1>(v);   // lane ^ 1
    v = add_dpp<0x4e>(v);   // lane ^ 2
    v = add_dpp<0x141>(v);  // the other four of 8
    if constexpr (G >= 16) v = add_dpp<0x140>(v);  // the other 8 of 16
    if constexpr (G >= 32) v = add_halves(v, false);
    if constexpr (G >= 64) v = add_halves(v, true);
    if constexpr (G == 256) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0] + lds[1] + lds[2] + lds[3];
    }
    return v;
}

// One lane's share of a row: NV vectors of E channels, vector i at channel
// (i G + lane) E.
template <int E, int NV, int G>
struct Lane {
    int at[NV];
    bool in[NV];
    __device__ __forceinline__ explicit Lane(int C) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            at[i] = (i * G + static_cast<int>(threadIdx.x) % G) * E;
            in[i] = at[i] < C;  // C is a multiple of E
        }
    }
    // dflt where there is no row; 0 past it, so that a product with it ends
    // what sums over the row must not see
    template <typename T>
    __device__ __forceinline__ void load(const T* row, float* v, float dflt = 0.0f) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (row != nullptr && in[i]) {
                load_row<T, E>(row + at[i], v + i * E);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) v[i * E + e] = in[i] ? dflt : 0.0f;
            }
        }
    }
    // The same in two steps: a row on its way, and its numbers.
    template <typename T>
    struct Ahead {
        typedef T Many __attribute__((ext_vector_type(E == 1 ? 2 : E)));
        std::conditional_t<E == 1, T, Many> v[NV];
    };
    template <typename T>
    __device__ __forceinline__ void fetch(const T* row, Ahead<T>& to) const {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (in[i]) to.v[i] = *reinterpret_cast<const std::remove_reference_t<decltype(to.v[i])>*>(row + at[i]);
    }
    template <typename T>
    __device__ __forceinline__ void widen(const Ahead<T>& from, float* v) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                T one;
                if constexpr (E == 1)
                    one = from.v[i];
                else
                    one = from.v[i][e];
                v[i * E + e] = in[i] ? static_cast<float>(one) : 0.0f;
            }
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(T* row, const float* v) const {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (in[i]) store_row<T, E>(row + at[i], v + i * E);
    }
    // v -> (v - mean) r, or v r without the mean; returns r = 1 / deviation
    __device__ __forceinline__ float normalise(float* v, int C, bool rms, float eps, float* lds) const {
        const float per = 1.0f / static_cast<float>(C);
        float mean = 0.0f;
        if (!rms) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < NV * E; ++i) s += v[i];
            mean = row_sum<G>(s, lds) * per;
        }
        float q = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float& t = v[i * E + e];
                t = in[i] ? t - mean : 0.0f;
                q = __builtin_fmaf(t, t, q);
            }
        }
        const float r = 1.0f / sqrtf(row_sum<G>(q, lds) * per + eps);
#pragma unroll
        for (int i = 0; i < NV * E; ++i) v[i] *= r;
        return r;
    }
    // g (gradient of the normed values n, 0 past the row) -> gradient of the
    // values, anything past the row
    __device__ __forceinline__ void normalise_grad(float* g, const float* n, float r, int C, bool rms, float* lds) const {
        const float per = 1.0f / static_cast<float>(C);
        float a = 0.0f, c = 0.0f;
#pragma unroll
        for (int i = 0; i < NV * E; ++i) {
            a += g[i];
            c = __builtin_fmaf(g[i], n[i], c);
        }
        a = rms ? 0.0f : row_sum<G>(a, lds) * per;
        c = row_sum<G>(c, lds) * per;
#pragma unroll
        for (int i = 0; i < NV * E; ++i) g[i] = r * (g[i] - a - n[i] * c);
    }
};

template <typename Tx, typename Ty, int E, int NV, int G>
__global__ void __launch_bounds__(kThreads) residual_norm_kernel(const NormArgs a) {
    __shared__ float lds[4];
    constexpr int kRows = kThreads / G, kN = NV * E;
    const Lane<E, NV, G> lane(a.C);
    const uint32_t sample = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const float k = a.scale != nullptr ? a.scale[sample] : 1.0f;
    float w[kN], b[kN], kg[kN];
    lane.load(a.w, w, 1.0f);
    lane.load(a.b, b);
    lane.load(a.gate != nullptr ? a.gate + static_cast<int64_t>(sample) * a.gate_stride : nullptr, kg, 1.0f);
#pragma unroll
    for (int i = 0; i < kN; ++i) kg[i] *= k;
    const uint32_t step = a.chunks * kRows;
    // every lane of a workgroup-wide row takes part in each round
    typename Lane<E, NV, G>::template Ahead<Tx> x_next = {};
    typename Lane<E, NV, G>::template Ahead<Ty> y_next = {};
    const auto fetch = [&](uint32_t t) {
        const int64_t row = (static_cast<int64_t>(sample) * a.T + t) * a.C;
        lane.fetch(static_cast<const Tx*>(a.x) + row, x_next);
        lane.fetch(static_cast<const Ty*>(a.y) + row, y_next);
    };
    // rows a round ahead: [3, 4001, 768] bf16 18 us for 22
    uint32_t t = chunk * kRows + threadIdx.x / G;
    if (t < a.T) fetch(t);
    for (; t < a.T; t += step) {
        const int64_t row = (static_cast<int64_t>(sample) * a.T + t) * a.C;
        float x[kN], y[kN];
        lane.widen(x_next, x);
        lane.widen(y_next, y);
        if (t + step < a.T) fetch(t + step);
        if (a.post) {
            float pw[kN], pb[kN];
            lane.load(a.pw, pw, 1.0f);
            lane.load(a.pb, pb);
            lane.normalise(y, a.C, a.rms, a.post_eps, lds);
#pragma unroll
            for (int i = 0; i < kN; ++i) y[i] = __builtin_fmaf(y[i], pw[i], pb[i]);
        }
#pragma unroll
        for (int i = 0; i < kN; ++i) x[i] = __builtin_fmaf(kg[i], y[i], x[i]);
        lane.store(static_cast<Tx*>(a.sum) + row, x);
        lane.normalise(x, a.C, a.rms, a.eps, lds);
#pragma unroll
        for (int i = 0; i < kN; ++i) x[i] = __builtin_fmaf(x[i], w[i], b[i]);
        lane.store(static_cast<Ty*>(a.out) + row, x);
    }
}

// Parameters are loaded where they are used, again if need be: they come from
// the cache, and rows, their norms and the sums fill the registers.
template <typename Tx, typename Ty, int E, int NV, int G, bool kPost>
__global__ void __launch_bounds__(kThreads) residual_norm_grad_kernel(const NormArgs a) {
    constexpr int kRows = kThreads / G, kN = NV * E, kCols = G * kN, kMine = kPost ? kSums : 3;
    __shared__ float lds[kRows > 1 ? kThreads * kN : 4];
    const Lane<E, NV, G> lane(a.C);
    const uint32_t sample = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const float k = a.scale != nullptr ? a.scale[sample] : 1.0f;
    const float* gate = a.gate != nullptr ? a.gate + static_cast<int64_t>(sample) * a.gate_stride : nullptr;
    float sums[kMine][kN] = {};
    const uint32_t step = a.chunks * kRows;
    // Rows a round ahead where a lane holds one vector ([4, 110592, 48], fp32 and
    // fp16: 78 us for 85); two fill the registers ([3, 4001, 768] bf16 with both
    // norms: 57 for 48).
    constexpr bool kAhead = kN <= 8;
    typename Lane<E, NV, G>::template Ahead<Tx> x_next = {}, sum_next = {};
    typename Lane<E, NV, G>::template Ahead<Ty> y_next = {}, out_next = {};
    const auto fetch = [&](uint32_t t) {
        const int64_t row = (static_cast<int64_t>(sample) * a.T + t) * a.C;
        lane.fetch(static_cast<const Tx*>(a.x) + row, x_next);
        lane.fetch(static_cast<const Ty*>(a.y) + row, y_next);
        if (a.gout != nullptr) lane.fetch(static_cast<const Ty*>(a.gout) + row, out_next);
        if (a.gsum != nullptr) lane.fetch(static_cast<const Tx*>(a.gsum) + row, sum_next);
    };
    uint32_t t = chunk * kRows + threadIdx.x / G;
    if (kAhead && t < a.T) fetch(t);
    for (; t < a.T; t += step) {
        const int64_t row = (static_cast<int64_t>(sample) * a.T + t) * a.C;
        float n[kN], y[kN], gx[kN], other[kN], yr = 0.0f;
        if constexpr (kAhead) {
            lane.widen(x_next, n);
            lane.widen(y_next, y);
            lane.widen(out_next, gx);
            lane.widen(sum_next, other);
            if (t + step < a.T) fetch(t + step);
        } else {
            lane.load(static_cast<const Tx*>(a.x) + row, n);
            lane.load(static_cast<const Ty*>(a.y) + row, y);
            lane.load(a.gout != nullptr ? static_cast<const Ty*>(a.gout) + row : nullptr, gx);
            lane.load(a.gsum != nullptr ? static_cast<const Tx*>(a.gsum) + row : nullptr, other);
        }
        if constexpr (kPost) yr = lane.normalise(y, a.C, a.rms, a.post_eps, lds);
        // y' = y p + b, made again where it is needed again
        const auto branch = [&](float* u) {
            if constexpr (kPost) {
                float p[kN];
                lane.load(a.pw, p, 1.0f);
                lane.load(a.pb, u);
#pragma unroll
                for (int i = 0; i < kN; ++i) u[i] = __builtin_fmaf(y[i], p[i], u[i]);
            } else {
#pragma unroll
                for (int i = 0; i < kN; ++i) u[i] = y[i];
            }
        };
        {
            float kg[kN], u[kN];
            lane.load(gate, kg, 1.0f);
            branch(u);
#pragma unroll
            for (int i = 0; i < kN; ++i) n[i] = __builtin_fmaf(k * kg[i], u[i], n[i]);
        }
        const float r = lane.normalise(n, a.C, a.rms, a.eps, lds);
        {
            float w[kN];
            lane.load(a.w, w, 1.0f);
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                sums[0][i] = __builtin_fmaf(gx[i], n[i], sums[0][i]);
                sums[1][i] += gx[i];
                gx[i] *= w[i];
            }
        }
        lane.normalise_grad(gx, n, r, a.C, a.rms, lds);
#pragma unroll
        for (int i = 0; i < kN; ++i) gx[i] += other[i];
        lane.store(static_cast<Tx*>(a.gx) + row, gx);
        {
            float kg[kN], u[kN];
            lane.load(gate, kg, 1.0f);
            branch(u);
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                sums[2][i] = __builtin_fmaf(gx[i] * k, u[i], sums[2][i]);
                gx[i] *= k * kg[i];
            }
        }
        if constexpr (kPost) {
            float p[kN];
            lane.load(a.pw, p, 1.0f);
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                sums[3][i] = __builtin_fmaf(gx[i], y[i], sums[3][i]);
                sums[4][i] += gx[i];
                gx[i] *= p[i];
            }
            lane.normalise_grad(gx, y, yr, a.C, a.rms, lds);
        }
        lane.store(static_cast<Ty*>(a.gy) + row, gx);
    }
    if (a.partial == nullptr) return;
    float* to = a.partial + static_cast<int64_t>(blockIdx.x) * kSums * a.C;
#pragma unroll
    for (int s = 0; s < kMine; ++s) {
        // uniform over the launch: the sums that somebody reads
        if (s == 2 && a.gate == nullptr) continue;
        if constexpr (kRows > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    lds[(threadIdx.x / G) * kCols + lane.at[i] + e] = sums[s][i * E + e];
            }
            __syncthreads();
            for (int c = threadIdx.x; c < a.C; c += kThreads) {
                float v = 0.0f;
                for (int i = 0; i < kRows; ++i) v += lds[i * kCols + c];
                to[s * a.C + c] = v;
            }
        } else {
            lane.store(to + s * a.C, sums[s]);
        }
    }
}

// Sums of the partial rows: 16 columns by 64 groups of rows per workgroup.
constexpr int kParts = 64;
struct SumArgs {
    const float* partial;
    float* out[kSums];     // null where nobody asked
    int32_t per_sample[kSums];
    uint32_t S, chunks;
    int32_t C;
};

__global__ void __launch_bounds__(kParts * 16) residual_norm_sums_kernel(const SumArgs a) {
    __shared__ float lds[kParts][17];
    const int which = static_cast<int>(blockIdx.y);
    if (a.out[which] == nullptr) return;
    const uint32_t samples = a.per_sample[which] ? a.S : 1u;
    if (blockIdx.z >= samples) return;
    const uint32_t rows = a.per_sample[which] ? a.chunks : a.chunks * a.S;
    const int c = static_cast<int>(blockIdx.x) * 16 + static_cast<int>(threadIdx.x & 15), part = threadIdx.x >> 4;
    const float* from = a.partial + (static_cast<int64_t>(blockIdx.z) * rows * kSums + which) * a.C + c;
    float v = 0.0f;
    if (c < a.C) {
#pragma unroll 4
        for (uint32_t r = part; r < rows; r += kParts) v += from[static_cast<int64_t>(r) * kSums * a.C];
    }
    lds[part][threadIdx.x & 15] = v;
    __syncthreads();
    if (part != 0 || c >= a.C) return;
    v = 0.0f;
#pragma unroll 8
    for (int i = 0; i < kParts; ++i) v += lds[i][threadIdx.x];
    a.out[which][static_cast<int64_t>(blockIdx.z) * a.C + c] = v;
}

template <typename Tx, typename Ty, int E, int NV, int G>
void launch(const NormArgs& a, bool grad, hipStream_t s) {
    if (grad && a.post)
        residual_norm_grad_kernel<Tx, Ty, E, NV, G, true><<<a.S * a.chunks, kThreads, 0, s>>>(a);
    else if (grad)
        residual_norm_grad_kernel<Tx, Ty, E, NV, G, false><<<a.S * a.chunks, kThreads, 0, s>>>(a);
    else
        residual_norm_kernel<Tx, Ty, E, NV, G><<<a.S * a.chunks, kThreads, 0, s>>>(a);
}

// Lanes of a row: the fewest that hold it in one vector each, then more
// vectors.  Rows of other lengths go one channel at a time.
struct Shape {
    int E, G;
};
Shape shape_of(int64_t C) {
    if (C % 8 == 0) return {8, C <= 64 ? 8 : C <= 128 ? 16 : C <= 256 ? 32 : C <= 1024 ? 64 : 256};
    return {1, C <= 64 ? 16 : C <= 1024 ? 64 : 256};
}

template <typename Tx, typename Ty>
void launch_shape(const NormArgs& a, bool grad, hipStream_t s) {
    const int C = a.C;
    if (C % 8 == 0) {
        if (C <= 64) return launch<Tx, Ty, 8, 1, 8>(a, grad, s);
        if (C <= 128) return launch<Tx, Ty, 8, 1, 16>(a, grad, s);
        if (C <= 256) return launch<Tx, Ty, 8, 1, 32>(a, grad, s);
        if (C <= 512) return launch<Tx, Ty, 8, 1, 64>(a, grad, s);
        if (C <= 1024) return launch<Tx, Ty, 8, 2, 64>(a, grad, s);
        if (C <= 2048) return launch<Tx, Ty, 8, 1, 256>(a, grad, s);
        if (C <= 4096) return launch<Tx, Ty, 8, 2, 256>(a, grad, s);
        return launch<Tx, Ty, 8, 4, 256>(a, grad, s);
    }
    if (C <= 64) return launch<Tx, Ty, 1, 4, 16>(a, grad, s);
    if (C <= 256) return launch<Tx, Ty, 1, 4, 64>(a, grad, s);
    if (C <= 1024) return launch<Tx, Ty, 1, 16, 64>(a, grad, s);
    return launch<Tx, Ty, 1, 16, 256>(a, grad, s);
}

int dispatch(const NormArgs& a, int32_t x_dtype, int32_t dtype, bool grad, hipStream_t s, const char* what) {
    if (x_dtype == CRUMPET_DTYPE_F32) {
        if (dtype == CRUMPET_DTYPE_F32) launch_shape<float, float>(a, grad, s);
        else if (dtype == CRUMPET_DTYPE_F16) launch_shape<float, _Float16>(a, grad, s);
        else launch_shape<float, __bf16>(a, grad, s);
    } else if (dtype == CRUMPET_DTYPE_F16) {
        launch_shape<_Float16, _Float16>(a, grad, s);
    } else {
        launch_shape<__bf16, __bf16>(a, grad, s);
    }
    return check_launch(what);
}

int check(int32_t x_dtype, int32_t dtype, int64_t samples, int64_t tokens, int64_t C, int32_t kind, const char* what) {
    if (dtype < 0 || dtype > 2 || x_dtype < 0 || x_dtype > 2)
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: unknown dtype code", what);
    if (x_dtype != dtype && x_dtype != CRUMPET_DTYPE_F32)
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: x is float32 or of the branch's type", what);
    if (kind != 0 && kind != 1) return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: norm is 0 (layer) or 1 (rms)", what);
    if (samples < 0 || tokens < 0) return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: negative size", what);
    if (C < 1 || C > 8192 || (C % 8 != 0 && C > 4096))
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: C = %lld is outside 1 .. 8192 (4096 where no multiple of 8)", what,
                    (long long)C);
    if (samples >= (int64_t(1) << 20) || tokens >= (int64_t(1) << 31))
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: more than 2^20 samples or 2^31 tokens", what);
    return CRUMPET_OK;
}

bool misaligned(std::initializer_list<const void*> ptrs, int64_t C) {
    if (C % 8 != 0) return false;  // one channel at a time
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return true;
    return false;
}

// Workgroups of a sample: about 1024 in all, none without a row.  Fewer leave
// compute units idle (768: the gradients of [4, 110592, 48] take 98 us for 84),
// more write more partial sums (2048: those of [3, 4001, 768] take 62 us for 54).
uint32_t chunks_of(int64_t samples, int64_t tokens, int64_t C) {
    const int64_t rows = kThreads / shape_of(C).G;
    const int64_t most = (tokens + rows - 1) / rows;
    return static_cast<uint32_t>(std::max<int64_t>(1, std::min<int64_t>(most, (1024 + samples - 1) / samples)));
}

}  // namespace
}  // namespace crumpet

using namespace crumpet;

extern "C" int crumpet_residual_norm(void* sum, void* out, const void* x, int32_t x_dtype, const void* y, int32_t dtype,
                                     int64_t samples, int64_t tokens, int64_t C, int32_t norm, int32_t post,
                                     const float* post_weight, const float* post_bias, const float* gate,
                                     int32_t gate_per_sample, const float* scale, const float* weight,
                                     const float* bias, float eps, void* stream) {
    const char* what = "residual_norm";
    const int st = check(x_dtype, dtype, samples, tokens, C, norm, what);
    if (st != CRUMPET_OK) return st;
    if (samples == 0 || tokens == 0) return CRUMPET_OK;
    if (sum == nullptr || out == nullptr || x == nullptr || y == nullptr)
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: null tensor", what);
    if (misaligned({sum, out, x, y, post_weight, post_bias, gate, weight, bias}, C))
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: pointers must be 16-byte aligned where C is a multiple of 8", what);
    NormArgs a = {};
    a.x = x, a.y = y, a.pw = post_weight, a.pb = post_bias, a.gate = gate, a.scale = scale, a.w = weight, a.b = bias;
    a.sum = sum, a.out = out;
    a.S = static_cast<uint32_t>(samples), a.T = static_cast<uint32_t>(tokens), a.C = static_cast<int32_t>(C);
    a.chunks = chunks_of(samples, tokens, C);
    a.gate_stride = gate_per_sample ? a.C : 0;
    a.post = post, a.rms = norm, a.eps = eps, a.post_eps = eps;
    return dispatch(a, x_dtype, dtype, false, static_cast<hipStream_t>(stream), what);
}

extern "C" int64_t crumpet_residual_norm_workspace(int64_t samples, int64_t tokens, int64_t C) {
    if (samples < 0 || samples >= (int64_t(1) << 20) || tokens < 0 || tokens >= (int64_t(1) << 31) || C < 1 || C > 8192)
        return -1;
    if (samples == 0 || tokens == 0) return 0;
    return samples * chunks_of(samples, tokens, C) * kSums * C * static_cast<int64_t>(sizeof(float));
}

extern "C" int crumpet_residual_norm_backward(
    void* grad_x, void* grad_y, float* grad_weight, float* grad_bias, float* grad_gate, float* grad_post_weight,
    float* grad_post_bias, const void* grad_sum, const void* grad_out, const void* x, int32_t x_dtype, const void* y,
    int32_t dtype, int64_t samples, int64_t tokens, int64_t C, int32_t norm, int32_t post, const float* post_weight,
    const float* post_bias, const float* gate, int32_t gate_per_sample, const float* scale, const float* weight,
    float eps, void* workspace, void* stream) {
    const char* what = "residual_norm_backward";
    const int st = check(x_dtype, dtype, samples, tokens, C, norm, what);
    if (st != CRUMPET_OK) return st;
    if (samples == 0 || tokens == 0) return CRUMPET_OK;
    if (grad_x == nullptr || grad_y == nullptr || x == nullptr || y == nullptr)
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: null tensor", what);
    if (misaligned({grad_x, grad_y, grad_sum, grad_out, x, y, post_weight, post_bias, gate, weight}, C))
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: pointers must be 16-byte aligned where C is a multiple of 8", what);
    if ((grad_gate != nullptr && gate == nullptr) || ((grad_post_weight != nullptr || grad_post_bias != nullptr) && !post))
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: gradient of a parameter that is not there", what);
    if (gate_per_sample && samples > 65535)
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: more than 65535 samples with a gate of their own", what);
    const bool sums = grad_weight != nullptr || grad_bias != nullptr || grad_gate != nullptr ||
                      grad_post_weight != nullptr || grad_post_bias != nullptr;
    if (sums && workspace == nullptr) return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: null workspace", what);
    NormArgs a = {};
    a.x = x, a.y = y, a.pw = post_weight, a.pb = post_bias, a.gate = gate, a.scale = scale, a.w = weight;
    a.gsum = grad_sum, a.gout = grad_out, a.gx = grad_x, a.gy = grad_y;
    a.partial = sums ? static_cast<float*>(workspace) : nullptr;
    a.S = static_cast<uint32_t>(samples), a.T = static_cast<uint32_t>(tokens), a.C = static_cast<int32_t>(C);
    a.chunks = chunks_of(samples, tokens, C);
    a.gate_stride = gate_per_sample ? a.C : 0;
    a.post = post, a.rms = norm, a.eps = eps, a.post_eps = eps;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int rc = dispatch(a, x_dtype, dtype, true, s, what);
    if (rc != CRUMPET_OK || !sums) return rc;
    SumArgs f = {};
    f.partial = a.partial;
    float* outs[kSums] = {grad_weight, grad_bias, grad_gate, grad_post_weight, grad_post_bias};
    for (int i = 0; i < kSums; ++i) f.out[i] = outs[i];
    f.per_sample[2] = gate_per_sample;
    f.S = a.S, f.chunks = a.chunks, f.C = a.C;
    const uint32_t deep = grad_gate != nullptr && gate_per_sample ? a.S : 1u;
    residual_norm_sums_kernel<<<dim3((a.C + 15) / 16, kSums, deep), kParts * 16, 0, s>>>(f);
    return check_launch(what);
}
