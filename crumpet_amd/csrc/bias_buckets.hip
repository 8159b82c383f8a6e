// A learned bias by buckets (gfx950): bias[h, p] = table[index[p], h] over the
// P pairs of query and key, and the table's gradient, the sum over the pairs of
// each bucket.
//
// The gradient takes the pairs sorted by bucket (stable), cut into segments of
// at most kSegment pairs that never cross a bucket: one wave per segment and
// head (or four heads) sums its pairs in a fixed order, without atomics.  Where every bucket
// fits one segment (the offsets of a window: 2,197 buckets of at most 343
// pairs) that sum is the result; longer ones (few buckets over long sequences)
// are partial sums, which a second kernel adds up.
//
// Traffic: the bias written and its gradient read once, the index and the order
// once per head or four.  The gradient is bound by its gather, a request for
// every pair and head: for 512 x 512 pairs of 24 heads in fp32 (25 MB) 29 us,
// 0.9 TB/s, and the bias 15 us, 1.7 TB/s.  Neighbours of a window's bucket lie a
// row apart, so wider loads have nothing to join.
#include <hip/hip_runtime.h>

#include "crumpet_common.h"
#include "crumpet_hip.h"

namespace crumpet {
namespace {

constexpr int kThreads = 256;
constexpr int kSegment = 2048;

// Four neighbouring pairs at any address (a head's row begins at a multiple of
// P): one wide access, which the memory takes at any alignment of an element.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Four {
    T v[4];
};

// Bits are copied, so one form per element size.  A workgroup writes `pairs`
// pairs of one head, 4 a thread and step.  Where there is work for 256 of them
// at 16384 pairs each, and the head's column of the table fits, the column waits
// in LDS (kLds), since a gather of table rows touches one line a lane; smaller
// calls gather, 1024 pairs to a workgroup: 512 x 512 pairs of 24 heads 13 us from
// LDS, 28 gathered; 343 x 343 of 3 heads 3.4 gathered, 7.4 from LDS.  An index
// outside the table reads as 0.
constexpr int64_t kManyPairs = 16384, kFewPairs = 1024;
constexpr int kColumn = 16384;  // bytes of LDS for a column

template <typename T, bool kLds>
__global__ void __launch_bounds__(kThreads)
bucket_bias_kernel(T* __restrict__ out, const T* __restrict__ table, const int32_t* __restrict__ index, int64_t P,
                   int32_t L, int32_t H, int32_t pairs) {
    __shared__ T column[kLds ? kColumn / sizeof(T) : 1];
    const int h = static_cast<int>(blockIdx.y);
    if constexpr (kLds) {
        for (int l = threadIdx.x; l < L; l += kThreads) column[l] = table[static_cast<int64_t>(l) * H + h];
        __syncthreads();
    }
    const auto value = [&](int32_t l) {
        if (static_cast<uint32_t>(l) >= static_cast<uint32_t>(L)) return T(0);
        return kLds ? column[l] : table[static_cast<int64_t>(l) * H + h];
    };
    const int64_t first = static_cast<int64_t>(blockIdx.x) * pairs;
    const int64_t last = first + pairs < P ? first + pairs : P;
    T* to = out + h * P;
    for (int64_t p = first + threadIdx.x * 4; p < last; p += kThreads * 4) {
        if (p + 4 <= last) {
            const Four<int32_t> l = *reinterpret_cast<const Four<int32_t>*>(index + p);
            Four<T> v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v.v[e] = value(l.v[e]);
            *reinterpret_cast<Four<T>*>(to + p) = v;
        } else {
            for (int64_t i = p; i < last; ++i) to[i] = value(index[i]);
        }
    }
}

// segments [n, 2]: first pair (in sorted order) and one past the last.  A wave
// sums its segment for kHeads heads at once: they share the reads of the order,
// and their own wait together.
template <typename T, typename To, int kHeads>
__global__ void __launch_bounds__(kThreads)
bucket_sum_kernel(To* __restrict__ out, const T* __restrict__ grad, const int32_t* __restrict__ order,
                  const int32_t* __restrict__ segments, int64_t P, int32_t H, uint32_t n) {
    // the workgroups of the same heads share an XCD, and its L2 their pairs
    const uint32_t groups = (n + kThreads / 64 - 1) / (kThreads / 64);
    uint32_t chunk;
    if (!xcd_chunk(blockIdx.x, gridDim.x, groups * static_cast<uint32_t>((H + kHeads - 1) / kHeads), chunk)) return;
    const uint32_t unit = chunk % groups * (kThreads / 64) + (threadIdx.x >> 6);
    const int h = static_cast<int>(chunk / groups) * kHeads, lane = threadIdx.x & 63;
    if (unit >= n) return;
    const int64_t from = segments[2 * unit] < 0 ? 0 : segments[2 * unit];
    const int64_t to = segments[2 * unit + 1] < P ? segments[2 * unit + 1] : P;
    const T* g[kHeads];
    float v[kHeads] = {};
#pragma unroll
    for (int k = 0; k < kHeads; ++k) g[k] = grad + (h + k < H ? h + k : h) * P;
#pragma unroll 4
    for (int64_t i = from + lane; i < to; i += 64) {
        const uint32_t p = static_cast<uint32_t>(order[i]);
        if (p >= P) continue;
#pragma unroll
        for (int k = 0; k < kHeads; ++k) v[k] += static_cast<float>(g[k][p]);
    }
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) v[k] += __shfl_xor(v[k], m);
        if (lane == 0 && h + k < H) out[static_cast<int64_t>(unit) * H + h + k] = static_cast<To>(v[k]);
    }
}

// firsts [L + 1]: each bucket's segments
template <typename To>
__global__ void __launch_bounds__(kThreads)
bucket_join_kernel(To* __restrict__ out, const float* __restrict__ partial, const int32_t* __restrict__ firsts,
                   int64_t L, int32_t H, uint32_t n) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (i >= L * H) return;
    const int64_t l = i / H;
    const int32_t h = static_cast<int32_t>(i % H);
    const int64_t from = firsts[l] < 0 ? 0 : firsts[l], to = firsts[l + 1] < n ? firsts[l + 1] : n;
    float v = 0.0f;
    for (int64_t s = from + lane; s < to; s += 64) v += partial[s * H + h];
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    if (lane == 0) out[i] = static_cast<To>(v);
}

int check(int32_t dtype, int64_t buckets, int64_t heads, int64_t pairs, const char* what) {
    if (dtype < 0 || dtype > 2) return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: unknown dtype code", what);
    if (buckets < 0 || heads < 0 || pairs < 0) return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: negative size", what);
    if (buckets >= (int64_t(1) << 31) || pairs >= (int64_t(1) << 31) || heads > 65535)
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: more than 2^31 buckets or pairs, or 65535 heads", what);
    return CRUMPET_OK;
}

template <typename T>
void forward(void* out, const void* table, const int32_t* index, int64_t L, int64_t H, int64_t P, hipStream_t s) {
    const bool lds = P * H >= 256 * kManyPairs && L <= static_cast<int64_t>(kColumn / sizeof(T));
    const int64_t pairs = lds ? kManyPairs : kFewPairs;
    const dim3 grid(static_cast<uint32_t>((P + pairs - 1) / pairs), static_cast<uint32_t>(H));
    T* o = static_cast<T*>(out);
    const T* t = static_cast<const T*>(table);
    const int32_t l = static_cast<int32_t>(L), h = static_cast<int32_t>(H);
    if (lds)
        bucket_bias_kernel<T, true><<<grid, kThreads, 0, s>>>(o, t, index, P, l, h, static_cast<int32_t>(pairs));
    else
        bucket_bias_kernel<T, false><<<grid, kThreads, 0, s>>>(o, t, index, P, l, h, static_cast<int32_t>(pairs));
}

// Four heads at a time where segments are long: 1000 x 1501 pairs of 12 heads in
// 32 buckets 34 us for 42.  A window's short ones lie scattered over its matrix,
// of which the L2 then holds four: 24 heads of 512 x 512 37 us for 29.
template <typename T, typename To>
void sum(To* out, const T* grad, const int32_t* order, const int32_t* segments, int64_t P, int64_t H, int64_t n,
         bool by_four, hipStream_t s) {
    const int32_t h = static_cast<int32_t>(H);
    const uint32_t units = static_cast<uint32_t>(n), groups = (units + 3) / 4;
    const uint32_t grid = xcd_launch_count(groups * static_cast<uint32_t>(by_four ? (H + 3) / 4 : H));
    if (by_four)
        bucket_sum_kernel<T, To, 4><<<grid, kThreads, 0, s>>>(out, grad, order, segments, P, h, units);
    else
        bucket_sum_kernel<T, To, 1><<<grid, kThreads, 0, s>>>(out, grad, order, segments, P, h, units);
}

template <typename T>
int backward(void* grad_table, const void* grad, int64_t L, int64_t H, int64_t P, const int32_t* order,
             const int32_t* segments, int64_t n, const int32_t* firsts, float* partial, hipStream_t s) {
    const T* g = static_cast<const T*>(grad);
    if (firsts == nullptr) {  // one segment a bucket
        sum(static_cast<T*>(grad_table), g, order, segments, P, H, n, false, s);
    } else {
        if (n > 0) sum(partial, g, order, segments, P, H, n, H >= 4, s);
        bucket_join_kernel<T><<<static_cast<uint32_t>((L * H + 3) / 4), kThreads, 0, s>>>(
            static_cast<T*>(grad_table), partial, firsts, L, static_cast<int32_t>(H), static_cast<uint32_t>(n));
    }
    return check_launch("bucket_bias_backward");
}

}  // namespace
}  // namespace crumpet

using namespace crumpet;

extern "C" int64_t crumpet_bucket_segment(void) { return kSegment; }

extern "C" int crumpet_bucket_bias(void* out, const void* table, int32_t dtype, const int32_t* index, int64_t buckets,
                                   int64_t heads, int64_t pairs, void* stream) {
    const int st = check(dtype, buckets, heads, pairs, "bucket_bias");
    if (st != CRUMPET_OK || heads == 0 || pairs == 0) return st;
    if (out == nullptr || table == nullptr || index == nullptr)
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "bucket_bias: null tensor");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == CRUMPET_DTYPE_F32)
        forward<uint32_t>(out, table, index, buckets, heads, pairs, s);
    else
        forward<uint16_t>(out, table, index, buckets, heads, pairs, s);
    return check_launch("bucket_bias");
}

extern "C" int crumpet_bucket_bias_backward(void* grad_table, const void* grad, int32_t dtype, int64_t buckets,
                                            int64_t heads, int64_t pairs, const int32_t* order, const int32_t* segments,
                                            int64_t segment_count, const int32_t* firsts, void* workspace,
                                            void* stream) {
    const char* what = "bucket_bias_backward";
    const int st = check(dtype, buckets, heads, pairs, what);
    if (st != CRUMPET_OK || heads == 0 || buckets == 0) return st;
    if (grad_table == nullptr || segments == nullptr || (pairs > 0 && (grad == nullptr || order == nullptr)))
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: null tensor", what);
    if (segment_count < 0 || segment_count >= (int64_t(1) << 31) || (firsts == nullptr && segment_count != buckets))
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: segments do not match the buckets", what);
    if (firsts != nullptr && workspace == nullptr)
        return fail(CRUMPET_ERR_INVALID_ARGUMENT, "%s: null workspace", what);
    if (!launch_takes(static_cast<uint64_t>(buckets) * heads / 4 + 1, kThreads) ||
        !launch_takes((static_cast<uint64_t>(segment_count) / 4 + 1) * heads + kNumXcd, kThreads))
        return fail(CRUMPET_ERR_UNSUPPORTED, "%s: too many buckets or segments for one launch", what);
    hipStream_t s = static_cast<hipStream_t>(stream);
    float* partial = static_cast<float*>(workspace);
    switch (dtype) {
        case CRUMPET_DTYPE_F32:
            return backward<float>(grad_table, grad, buckets, heads, pairs, order, segments, segment_count, firsts,
                                   partial, s);
        case CRUMPET_DTYPE_F16:
            return backward<_Float16>(grad_table, grad, buckets, heads, pairs, order, segments, segment_count, firsts,
                                      partial, s);
        default:
            return backward<__bf16>(grad_table, grad, buckets, heads, pairs, order, segments, segment_count, firsts,
                                    partial, s);
    }
}
