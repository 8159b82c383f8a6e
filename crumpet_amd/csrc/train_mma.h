// 16x16 matrix products of the training kernels (gfx950), one wave each.
//
// Layout of v_mfma_f32_16x16x16 and of the 16-deep product made of four
// v_mfma_f32_16x16x4_f32: lane (col = lane & 15, g = lane >> 4) holds
//   A[m = col][k = 4 g + e],  B[k = 4 g + e][n = col],  e = 0..3,
//   D[m = 4 g + r][n = col],  r = 0..3.
// D has the form of a B operand whose depth is D's row, so a product's result
// feeds the next one without leaving the registers.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "crumpet_common.h"
#include "crumpet_hip.h"

namespace crumpet {
namespace train {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Mma;

template <>
struct Mma<_Float16> {
    typedef _Float16 x4 __attribute__((ext_vector_type(4)));
    typedef _Float16 x8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 mma16(x4 a, x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mma32(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

template <>
struct Mma<__bf16> {
    typedef __bf16 x4 __attribute__((ext_vector_type(4)));
    typedef __bf16 x8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 mma16(x4 a, x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4, a), __builtin_bit_cast(i16x4, b), c,
                                                         0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mma32(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

template <>
struct Mma<float> {
    typedef f32x4 x4;
    static __device__ __forceinline__ f32x4 mma16(x4 a, x4 b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

template <typename T>
__device__ __forceinline__ typename Mma<T>::x4 load4(const T* p) {
    return *reinterpret_cast<const typename Mma<T>::x4*>(p);
}

template <typename T>
__device__ __forceinline__ typename Mma<T>::x4 round4(f32x4 v) {
    typename Mma<T>::x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = static_cast<T>(v[e]);
    return o;
}

template <typename T>
__device__ __forceinline__ f32x4 wide4(typename Mma<T>::x4 v) {
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = static_cast<float>(v[e]);
    return o;
}

// An fp32 number kept as its rounding to T and a second value of 16 bits.  fp16:
// the rounding of what is left, 2^-22 of the number.  bf16, whose rest would be
// short at 2^-17: the bits below it, fp32's own, as a whole number in
// [-2^15, 2^15) of fp32 steps (a tie that rounds down is one step less).
//
// v passes through the asm so that both see one number: a product formed anew
// inside a fused conversion to fp16 rounds a near tie the other way, and lo
// would not belong to hi.
template <typename T>
__device__ __forceinline__ void round_and_rest(f32x4 v, typename Mma<T>::x4& hi, typename Mma<T>::x4& lo) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float x = v[e];
        asm("" : "+v"(x));
        v[e] = x;
    }
    hi = round4<T>(v);
    if constexpr (sizeof(T) == 2 && !std::is_same_v<T, _Float16>) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const T top = hi[e];
            const int left = static_cast<int>(__float_as_uint(v[e]) -
                                              (static_cast<uint32_t>(__builtin_bit_cast(unsigned short, top)) << 16));
            lo[e] = __builtin_bit_cast(T, static_cast<short>(left < 0x7fff ? left : 0x7fff));
        }
    } else {
        lo = round4<T>(v - wide4<T>(hi));
    }
}
template <typename T>
__device__ __forceinline__ float with_rest(T hi, T lo) {
    if constexpr (sizeof(T) == 2 && !std::is_same_v<T, _Float16>) {
        const uint32_t top = static_cast<uint32_t>(__builtin_bit_cast(unsigned short, hi)) << 16;
        return __uint_as_float(top + static_cast<uint32_t>(static_cast<int>(__builtin_bit_cast(short, lo))));
    } else {
        return static_cast<float>(hi) + static_cast<float>(lo);
    }
}

// The lane's A fragment of the transpose of rows row0 .. row0 + 15 at columns
// c0 .. c0 + 15 of a row-major LDS tile: [row0 + 4 g + e][c0 + col].  The
// 16-bit transpose read hands lane (col, g) element col % 4 of the 8-byte
// vectors that lanes 4 e + col / 4 of its group address.  fp32 reads one value
// at a time.
template <typename T>
__device__ __forceinline__ typename Mma<T>::x4 load_transposed(const T* tile, int ld, int row0, int c0, int col, int g) {
    if constexpr (sizeof(T) == 2) {
        typedef __attribute__((address_space(3))) i16x4 LdsI16x4;
        const T* at = tile + (row0 + 4 * g + (col >> 2)) * ld + c0 + 4 * (col & 3);
        const i16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)(const_cast<T*>(at)));
        return __builtin_bit_cast(typename Mma<T>::x4, r);
    } else {
        typename Mma<T>::x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = tile[(row0 + 4 * g + e) * ld + c0 + col];
        return r;
    }
}

// 16 bytes per lane from a buffer straight into LDS, at lds_addr + 16 * lane
// (lds_addr the same for the wave).  Inline asm, so that the compiler does not
// wait for it before unrelated LDS reads; the caller waits (wait_vmem) before
// the barrier that publishes the rows.  M0 is an operand, so the compiler
// writes it; the wait states are those that the load needs after scalar writes
// of M0 and vector writes of the descriptor's registers, which the compiler
// does not insert around asm.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_to_lds(u32x4 buffer, uint32_t lds_addr, uint32_t offset) {
    asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                 :
                 : "v"(offset), "s"(buffer), "{m0}"(lds_addr)
                 : "memory");
}
// All vector memory of the wave is done, what the compiler does not see too.
__device__ __forceinline__ void wait_vmem() {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0) expcnt(7) lgkmcnt(15)
}
// A buffer of `bytes` from `first`, the same for the wave.
__device__ __forceinline__ u32x4 buffer_of(const void* first, uint32_t bytes) {
    const uint64_t at = reinterpret_cast<uintptr_t>(first);
    u32x4 b;
    b[0] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at));
    b[1] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32) & 0xffffu);
    b[2] = __builtin_amdgcn_readfirstlane(bytes);
    b[3] = 0x00020000;
    return b;
}
template <typename T>
__device__ __forceinline__ uint32_t lds_address(const T* p) {
    typedef __attribute__((address_space(3))) const T LdsT;
    return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsT*)p)));
}

// The same lane's values of two groups of 16, in some order: l and l ^ 16, l and
// l ^ 32; no round trip through LDS.
struct Two {
    uint32_t a, b;
};
__device__ __forceinline__ Two pair16(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return {r[0], r[1]};
}
__device__ __forceinline__ Two pair32(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return {r[0], r[1]};
}
// Over the 4 lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float sum_groups(float x) {
    Two t = pair16(__float_as_uint(x));
    t = pair32(__float_as_uint(__uint_as_float(t.a) + __uint_as_float(t.b)));
    return __uint_as_float(t.a) + __uint_as_float(t.b);
}
__device__ __forceinline__ float max_groups(float x) {
    Two t = pair16(__float_as_uint(x));
    t = pair32(__float_as_uint(fmaxf(__uint_as_float(t.a), __uint_as_float(t.b))));
    return fmaxf(__uint_as_float(t.a), __uint_as_float(t.b));
}
__device__ __forceinline__ uint32_t max_groups(uint32_t x) {
    Two t = pair16(x);
    t = pair32(t.a > t.b ? t.a : t.b);
    return t.a > t.b ? t.a : t.b;
}

__device__ __forceinline__ float load_float(const void* p, int32_t dtype, int64_t i) {
    if (dtype == CRUMPET_DTYPE_F32) return static_cast<const float*>(p)[i];
    if (dtype == CRUMPET_DTYPE_F16) return static_cast<float>(static_cast<const _Float16*>(p)[i]);
    return static_cast<float>(static_cast<const __bf16*>(p)[i]);
}

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace
}  // namespace train
}  // namespace crumpet
