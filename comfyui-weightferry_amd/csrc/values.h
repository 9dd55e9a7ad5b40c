// Values of the three float types as the row-wise kernels move them: 16-byte packs loaded and stored at the alignment of
// one value (the compiler emits one 128-bit access: gfx950 takes unaligned global addresses), a masked form for a row's
// last, partial pack, and sums and maxima over a 64-lane wave.
#pragma once

#include "wf_common.h"

namespace wf {

template <int D> struct ValueType { typedef uint16_t T; };
template <> struct ValueType<WF_F32> { typedef float T; };
template <int D> using value_t = typename ValueType<D>::T;

inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
inline int value_bytes(int dt) { return dt == WF_F32 ? 4 : 2; }
inline bool known_dtype(int dt) { return dt == WF_F16 || dt == WF_BF16 || dt == WF_F32; }

template <int D>
__device__ __forceinline__ float to_f32(value_t<D> v) {
    if constexpr (D == WF_F16) return f16_bits_to_f32(v);
    else if constexpr (D == WF_BF16) return __uint_as_float((uint32_t)v << 16);
    else return v;
}

template <int D>
__device__ __forceinline__ value_t<D> from_f32(float x) {
    if constexpr (D == WF_F16) return __builtin_bit_cast(uint16_t, (_Float16)x);
    else if constexpr (D == WF_BF16) return __builtin_bit_cast(uint16_t, (__bf16)x);
    else return x;
}

// a single value of a run-time type (parameters that may be float32 next to 16-bit activations)
__device__ __forceinline__ float load_value(const void* p, int64_t i, int dt) {
    if (dt == WF_F32) return static_cast<const float*>(p)[i];
    const uint16_t v = static_cast<const uint16_t*>(p)[i];
    return dt == WF_BF16 ? __uint_as_float((uint32_t)v << 16) : f16_bits_to_f32(v);
}
__device__ __forceinline__ void store_value(void* p, int64_t i, int dt, float x) {
    if (dt == WF_F32) static_cast<float*>(p)[i] = x;
    else static_cast<uint16_t*>(p)[i] = dt == WF_BF16 ? from_f32<WF_BF16>(x) : from_f32<WF_F16>(x);
}

// 16 bytes of values: VEC of them
template <int D>
struct Pack {
    static constexpr int VEC = 16 / (int)sizeof(value_t<D>);
    uint32_t w[4];

    __device__ __forceinline__ float get(int i) const {
        if constexpr (D == WF_F32) return __uint_as_float(w[i]);
        else if constexpr (D == WF_BF16) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else return f16_bits_to_f32(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
    }
    // values 2 i and 2 i + 1 (16-bit types), or value i (float32)
    __device__ __forceinline__ void put(const float (&v)[VEC]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (D == WF_F32) w[i] = __float_as_uint(v[i]);
            else if constexpr (D == WF_BF16) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
            else w[i] = pack_f16(v[2 * i], v[2 * i + 1]);
        }
    }
    __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }

    // the first n of VEC values at p (zeros for the others); n may be anything, p only its value's alignment
    __device__ __forceinline__ void load(const value_t<D>* p, int n) {
        if (n >= VEC) {
            __builtin_memcpy(w, p, 16);
        } else {
            zero();
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                if (i >= n) continue;
                if constexpr (D == WF_F32) w[i] = __float_as_uint(p[i]);
                else w[i / 2] |= (uint32_t)p[i] << (16 * (i & 1));
            }
        }
    }
    // the same past the caches' ordinary replacement, for outputs that no launch reads back at once
    __device__ __forceinline__ void store_streamed(value_t<D>* p, int n) const {
        typedef uint32_t quad __attribute__((ext_vector_type(4), aligned(2)));
        if (n >= VEC) __builtin_nontemporal_store((quad){w[0], w[1], w[2], w[3]}, reinterpret_cast<quad*>(p));
        else store(p, n);
    }
    __device__ __forceinline__ void store(value_t<D>* p, int n) const {
        if (n >= VEC) {
            __builtin_memcpy(p, w, 16);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                if (i >= n) continue;
                if constexpr (D == WF_F32) p[i] = __uint_as_float(w[i]);
                else p[i] = (uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2]);
            }
        }
    }
};

// VEC values of type D or float32 (f32 set) at index i of p, the first n of them
template <int VEC>
__device__ __forceinline__ void load_params(float (&v)[VEC], const void* p, int64_t i, int n, int dt) {
    if (dt == WF_F32) {
        const float* q = static_cast<const float*>(p) + i;
        if (n >= VEC) __builtin_memcpy(v, q, VEC * 4);
        else
#pragma unroll
            for (int e = 0; e < VEC; e++) v[e] = e < n ? q[e] : 0.0f;
    } else {
        const uint16_t* q = static_cast<const uint16_t*>(p) + i;
        uint16_t h[VEC];
        if (n >= VEC) __builtin_memcpy(h, q, VEC * 2);
        else
#pragma unroll
            for (int e = 0; e < VEC; e++) h[e] = e < n ? q[e] : (uint16_t)0;
        if (dt == WF_BF16)
#pragma unroll
            for (int e = 0; e < VEC; e++) v[e] = __uint_as_float((uint32_t)h[e] << 16);
        else
#pragma unroll
            for (int e = 0; e < VEC; e++) v[e] = f16_bits_to_f32(h[e]);
    }
}

// the sum over the wave's 64 lanes in every lane: within rows of 16 lanes by DPP, the four rows by scalar reads; always
// the same order
template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_value(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ float wave_sum(float v) {
    v += dpp_move<0xB1>(v);      // quad_perm [1, 0, 3, 2]
    v += dpp_move<0x4E>(v);      // quad_perm [2, 3, 0, 1]
    v += dpp_move<0x141>(v);     // row_half_mirror
    v += dpp_move<0x140>(v);     // row_mirror
    return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}
// the largest of non-negative floats (or NaN) by their bits: NaN is above infinity, so it wins
__device__ __forceinline__ float wave_max_bits(float v) {
    auto up = [](float a, float b) {
        const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
        return __uint_as_float(x > y ? x : y);
    };
    v = up(v, dpp_move<0xB1>(v));
    v = up(v, dpp_move<0x4E>(v));
    v = up(v, dpp_move<0x141>(v));
    v = up(v, dpp_move<0x140>(v));
    return up(up(lane_value(v, 0), lane_value(v, 16)), up(lane_value(v, 32), lane_value(v, 48)));
}

}  // namespace wf
