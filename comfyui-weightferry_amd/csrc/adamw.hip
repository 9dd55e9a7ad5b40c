// One AdamW step over many tensors for gfx950, the moments held in float32 or in 8 bits.
//
//   m' = b1 m + (1 - b1) g,  v' = b2 v + (1 - b2) g^2
//   p' = (1 - lr decay) p - (lr / (1 - b1^t)) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Bound by memory: parameters and moments are read and written once, gradients read once. The tensors of a call are one
// launch (up to kAdamTensors of them), whatever their sizes: their addresses travel in the kernel's arguments and each
// workgroup finds its tensor by a binary search over the tensors' first workgroups, in scalar registers.
//
// The moments are flat arrays over all tensors, each tensor starting on a whole block of 256 values. In 8 bits a block's
// 256 codes share a float32 scale, the block's largest magnitude: m = sign(q) (q / 127)^2 s, and v through its root,
// u = (q / 255)^2 s, v = u^2. The square spreads the codes so that values far below a block's largest keep relative
// precision; a v that is not zero keeps a code that is not zero, so that no later step divides by eps alone. The step
// itself uses the new moments before they are rounded. A wave holds a whole block (4 values a lane), so the largest is a
// wave reduction and nothing is read twice. A gradient that is not finite makes its block's scales so, and the block's
// moments NaN from then on.
//
// The moments and their codes are defined to the bit: products, sums, quotients and roots rounded correctly one by one (no
// contraction), in the order written here. Correct quotients and roots are a dozen instructions each, and with them the
// 8-bit step was bound by the vector unit (118 instructions a value: 141.6 M bfloat16 values 431 us). So a code is
// computed by the hardware's one-ulp reciprocal and root first, which decides it unless the unrounded code lies within
// 2^-11 of a half -- four times what the two ways can differ by -- and only then the correct way, for the four values of a
// lane: 278 us, 5.1 TB/s. The parameter's step uses the one-ulp forms throughout; its error is far below the parameter's own
// rounding.

#include <cmath>
#include <type_traits>

#include "grids.h"
#include "values.h"

namespace wf {

constexpr int kBlock = 256;               // values that share a scale: 64 lanes of 4
constexpr int kAdamTensors = 96;          // tensors a launch (its arguments stay below 4 KiB)
constexpr int kSpan = 2;                  // blocks a wave (2, 4, 8: 71, 77, 88 us for 14.7 M float32 values in 8 bits)
constexpr int kAdamWg = 4 * kSpan;        // blocks a workgroup of 4 waves

struct AdamTable {
    void* p[kAdamTensors];
    const void* g[kAdamTensors];
    int64_t n[kAdamTensors];              // values
    uint32_t block[kAdamTensors];         // the tensor's first block of the moments
    uint32_t wg[kAdamTensors + 1];        // its first workgroup
    int count;
};

struct AdamConst {
    float b1, b1c, b2, b2c, keep, rate, root, eps;   // b1c = 1 - b1; keep = 1 - lr decay; rate = lr / (1 - b1^t); root
};                                                   // = 1 / sqrt(1 - b2^t)

// 4 values at p (the alignment of one value), the first n of them; STREAM: past the caches' ordinary replacement
template <int D, bool STREAM>
__device__ __forceinline__ void load4(float (&v)[4], const value_t<D>* p, int n) {
    typedef value_t<D> quad __attribute__((ext_vector_type(4), aligned(sizeof(value_t<D>))));
    quad r = {0, 0, 0, 0};
    if (n >= 4) {
        if constexpr (STREAM) r = __builtin_nontemporal_load(reinterpret_cast<const quad*>(p));
        else r = *reinterpret_cast<const quad*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < n) r[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = to_f32<D>(r[i]);
}
template <int D, bool STREAM>
__device__ __forceinline__ void store4(const float (&v)[4], value_t<D>* p, int n) {
    typedef value_t<D> quad __attribute__((ext_vector_type(4), aligned(sizeof(value_t<D>))));
    quad r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = from_f32<D>(v[i]);
    if (n >= 4) {
        if constexpr (STREAM) __builtin_nontemporal_store(r, reinterpret_cast<quad*>(p));
        else *reinterpret_cast<quad*>(p) = r;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < n) p[i] = r[i];
    }
}

__device__ __forceinline__ float avg_value(int q, float scale) {
    const float c = (float)q * (1.0f / 127.0f);
    return c * fabsf(c) * scale;
}
__device__ __forceinline__ float sq_value(uint32_t q, float scale) {
    const float c = (float)q * (1.0f / 255.0f);
    const float u = c * c * scale;
    return u * u;
}
// 4 codes rint(most * sqrt(x / s)) of a block with the largest x s; x: the magnitudes to one ulp, exact(i) to the bit
// (valid for largest values above `low`: there the values whose magnitude the hardware's root may lose code to 0 either way)
template <typename F>
__device__ __forceinline__ void codes(int (&q)[4], const float (&x)[4], float s, float low, float most, F&& exact) {
#pragma unroll
    for (int i = 0; i < 4; i++) q[i] = 0;
    if (!(s > 0.0f && s <= 3.402823466e+38f)) return;              // an empty block, or one that is not finite
    bool close = !(s > low && s < 1e30f);
    const float inv = __builtin_amdgcn_rcpf(s);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float t = __builtin_amdgcn_sqrtf(x[i] * inv) * most, r = rintf(t);
        q[i] = (int)r;
        close = close || fabsf(t - r) > 0.5f - 0x1p-11f;
    }
    if (close)
#pragma unroll
        for (int i = 0; i < 4; i++) q[i] = (int)rintf(sqrtf(exact(i) / s) * most);
}

template <int D, bool EIGHT, bool STREAM>
__global__ __launch_bounds__(256) void adamw(AdamTable t, AdamConst k, void* __restrict__ m_, void* __restrict__ v_,
                                             float* __restrict__ ms, float* __restrict__ vs) {
    int lo = 0, hi = t.count - 1;                        // the last tensor whose first workgroup is not past this one
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.wg[mid] <= blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n = t.n[lo];
    value_t<D>* p = static_cast<value_t<D>*>(t.p[lo]);
    const value_t<D>* g = static_cast<const value_t<D>*>(t.g[lo]);
    const int64_t b0 = ((int64_t)(blockIdx.x - t.wg[lo]) * 4 + wave) * kSpan;      // of the tensor
    float pv[kSpan][4], gv[kSpan][4], mv[kSpan][4], vv[kSpan][4];
#pragma unroll
    for (int b = 0; b < kSpan; b++) {
        if ((b0 + b) * kBlock >= n) break;
        const int64_t at = (b0 + b) * kBlock + 4 * lane, blk = t.block[lo] + b0 + b, sat = blk * kBlock + 4 * lane;
        const int left = (int)min<int64_t>(4, n - at);
        load4<D, STREAM>(gv[b], g + at, left);
        load4<D, STREAM>(pv[b], p + at, left);
        if constexpr (EIGHT) {
            const uint32_t qm = *reinterpret_cast<const uint32_t*>(static_cast<const int8_t*>(m_) + sat);
            const uint32_t qv = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(v_) + sat);
            const float sm = ms[blk], sv = vs[blk];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                mv[b][i] = avg_value((int8_t)(qm >> (8 * i)), sm);
                vv[b][i] = sq_value(qv >> (8 * i) & 255u, sv);
            }
        } else {
            load4<WF_F32, STREAM>(mv[b], static_cast<const float*>(m_) + sat, 4);
            load4<WF_F32, STREAM>(vv[b], static_cast<const float*>(v_) + sat, 4);
        }
    }
#pragma unroll
    for (int b = 0; b < kSpan; b++) {
        if ((b0 + b) * kBlock >= n) break;
        const int64_t at = (b0 + b) * kBlock + 4 * lane, blk = t.block[lo] + b0 + b, sat = blk * kBlock + 4 * lane;
        const int left = (int)min<int64_t>(4, n - at);
        float am[4], u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            mv[b][i] = mv[b][i] * k.b1 + gv[b][i] * k.b1c;
            vv[b][i] = vv[b][i] * k.b2 + gv[b][i] * gv[b][i] * k.b2c;
            am[i] = fabsf(mv[b][i]);
            u[i] = __builtin_amdgcn_sqrtf(vv[b][i]);
            if (vv[b][i] > 0.0f && vv[b][i] < 1e-30f) u[i] = sqrtf(vv[b][i]);      // (the hardware's drops subnormals)
            const float denom = u[i] * k.root + k.eps;
            pv[b][i] = pv[b][i] * k.keep - mv[b][i] * __builtin_amdgcn_rcpf(denom) * k.rate;
        }
        store4<D, STREAM>(pv[b], p + at, left);
        if constexpr (EIGHT) {
            uint32_t bm = 0, bv = 0;                               // the largest by their bits: NaN above infinity
#pragma unroll
            for (int i = 0; i < 4; i++) {
                bm = max(bm, __float_as_uint(am[i]));
                bv = max(bv, __float_as_uint(vv[b][i]) & 0x7fffffffu);
            }
            // (the root is monotonic, rounded too: the largest root is the root of the largest)
            const float sm = wave_max_bits(__uint_as_float(bm)), su = sqrtf(wave_max_bits(__uint_as_float(bv)));
            int a[4], c[4];
            codes(a, am, sm, 1e-30f, 127.0f, [&](int i) { return am[i]; });
            codes(c, u, su, 1e-11f, 255.0f, [&](int i) { return sqrtf(vv[b][i]); });
            const int least = su > 0.0f && su <= 3.402823466e+38f ? 1 : 0;
            uint32_t qm = 0, qv = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (vv[b][i] > 0.0f) c[i] = max(c[i], least);
                qm |= (uint32_t)((mv[b][i] < 0.0f ? -a[i] : a[i]) & 255) << (8 * i);
                qv |= (uint32_t)(c[i] & 255) << (8 * i);
            }
            *reinterpret_cast<uint32_t*>(static_cast<int8_t*>(m_) + sat) = qm;
            *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(v_) + sat) = qv;
            if (lane == 0) {
                ms[blk] = sm;
                vs[blk] = su;
            }
        } else {
            store4<WF_F32, STREAM>(mv[b], static_cast<float*>(m_) + sat, 4);
            store4<WF_F32, STREAM>(vv[b], static_cast<float*>(v_) + sat, 4);
        }
    }
}

// the values that 8-bit codes stand for: 4 a thread (values: a multiple of 256)
__global__ __launch_bounds__(256) void adamw_values(const int8_t* __restrict__ m, const uint8_t* __restrict__ v,
                                                    const float* __restrict__ ms, const float* __restrict__ vs,
                                                    float4* __restrict__ mo, float4* __restrict__ vo, int64_t quads) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= quads) return;
    const uint32_t qm = reinterpret_cast<const uint32_t*>(m)[i], qv = reinterpret_cast<const uint32_t*>(v)[i];
    const float sm = ms[i / 64], sv = vs[i / 64];
    mo[i] = make_float4(avg_value((int8_t)qm, sm), avg_value((int8_t)(qm >> 8), sm), avg_value((int8_t)(qm >> 16), sm),
                        avg_value((int8_t)(qm >> 24), sm));
    vo[i] = make_float4(sq_value(qv & 255u, sv), sq_value(qv >> 8 & 255u, sv), sq_value(qv >> 16 & 255u, sv),
                        sq_value(qv >> 24, sv));
}

}  // namespace wf

extern "C" int wf_adamw(const int64_t* table, int64_t count, int dt, int bits, void* exp_avg, void* exp_avg_sq,
                        float* avg_scale, float* sq_scale, int64_t blocks, int64_t step, double lr, double beta1,
                        double beta2, double eps, double weight_decay, void* stream) {
    using namespace wf;
    if (count < 0 || (count && !table) || step < 1 || blocks < 0 || !(beta1 >= 0 && beta1 < 1) ||
        !(beta2 >= 0 && beta2 < 1) || !(eps >= 0)) {
        set_error("wf_adamw: bad arguments (count %lld, step %lld, betas %g %g, eps %g)", (long long)count,
                  (long long)step, beta1, beta2, eps);
        return WF_EINVAL;
    }
    if (!known_dtype(dt) || (bits != 8 && bits != 32)) {
        set_error("wf_adamw: dtype code %d, %d bits", dt, bits);
        return WF_EUNSUPPORTED;
    }
    if (blocks >= (1LL << 32)) { set_error("wf_adamw: 2^40 values or more"); return WF_EUNSUPPORTED; }
    // every tensor lies in the moments and is addressed as its type asks before anything is launched
    int64_t block = 0;
    const uintptr_t size = value_bytes(dt);
    for (int64_t i = 0; i < count; i++) {
        const int64_t n = table[3 * i + 2];
        if (n < 0 || n > (1LL << 40) || (n && (!table[3 * i] || !table[3 * i + 1])) || table[3 * i] % (int64_t)size ||
            table[3 * i + 1] % (int64_t)size) {
            set_error("wf_adamw: tensor %lld: %lld values, null or misaligned", (long long)i, (long long)n);
            return WF_EINVAL;
        }
        block += (n + kBlock - 1) / kBlock;
    }
    if (block != blocks) {
        set_error("wf_adamw: the tensors take %lld blocks of 256 values, the moments hold %lld", (long long)block,
                  (long long)blocks);
        return WF_EINVAL;
    }
    if (blocks == 0) return WF_OK;
    if (!exp_avg || !exp_avg_sq || !aligned(exp_avg, 16) || !aligned(exp_avg_sq, 16) ||
        (bits == 8 && (!avg_scale || !sq_scale))) {
        set_error("wf_adamw: moments null or not 16-byte aligned");
        return WF_EINVAL;
    }
    AdamConst k;
    k.b1 = (float)beta1, k.b1c = (float)(1 - beta1), k.b2 = (float)beta2, k.b2c = (float)(1 - beta2);
    k.keep = (float)(1 - lr * weight_decay);
    k.rate = (float)(lr / (1 - std::pow(beta1, (double)step)));
    k.root = (float)(1 / std::sqrt(1 - std::pow(beta2, (double)step)));
    k.eps = (float)eps;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    // float32 moments past what the 256 MB last-level cache could keep for the next step go by it: 141.6 M bfloat16 values
    // (3.1 GB) 525 against 577 us; 14.7 M float32 values (0.4 GB) 75 against 66. In 8 bits no difference.
    const bool stream_past = (double)blocks * kBlock * (16 + 3 * (double)size) > 1e9;
    AdamTable t;
    int64_t tensor = 0, before = 0;                       // blocks of the tensors before `tensor`
    auto values = [&](int64_t i) { return table[3 * i + 2]; };
    auto part = [&](int c, int64_t i, int64_t done, int64_t part_blocks, uint32_t wg) {
        for (; tensor < i; tensor++) before += (values(tensor) + kBlock - 1) / kBlock;
        t.p[c] = reinterpret_cast<char*>(table[3 * i]) + done * kBlock * size;
        t.g[c] = reinterpret_cast<const char*>(table[3 * i + 1]) + done * kBlock * size;
        t.n[c] = std::min(values(i) - done * kBlock, part_blocks * kBlock);
        t.block[c] = (uint32_t)(before + done);
        t.wg[c] = wg;
    };
    auto launch = [&](int parts, uint32_t wgs) {
        t.count = parts;
        t.wg[parts] = wgs;
        auto go = [&](auto d) {
            constexpr int D = decltype(d)::value;
            if (bits == 8) adamw<D, true, false><<<dim3(wgs), 256, 0, s>>>(t, k, exp_avg, exp_avg_sq, avg_scale, sq_scale);
            else if (stream_past)
                adamw<D, false, true><<<dim3(wgs), 256, 0, s>>>(t, k, exp_avg, exp_avg_sq, avg_scale, sq_scale);
            else adamw<D, false, false><<<dim3(wgs), 256, 0, s>>>(t, k, exp_avg, exp_avg_sq, avg_scale, sq_scale);
        };
        if (dt == WF_F16) go(std::integral_constant<int, WF_F16>{});
        else if (dt == WF_BF16) go(std::integral_constant<int, WF_BF16>{});
        else go(std::integral_constant<int, WF_F32>{});
    };
    over_tensors(count, kBlock, kAdamWg, kAdamTensors, kGridMost, values, part, launch);
    WF_LAUNCH_CHECK("wf_adamw launch");
    return WF_OK;
}

extern "C" int wf_adamw_values(const int8_t* exp_avg, const uint8_t* exp_avg_sq, const float* avg_scale,
                               const float* sq_scale, int64_t blocks, float* avg, float* sq, void* stream) {
    using namespace wf;
    if (blocks < 0) { set_error("wf_adamw_values: %lld blocks", (long long)blocks); return WF_EINVAL; }
    if (blocks == 0) return WF_OK;
    if (!exp_avg || !exp_avg_sq || !avg_scale || !sq_scale || !avg || !sq || !aligned(exp_avg, 16) ||
        !aligned(exp_avg_sq, 16) || !aligned(avg, 16) || !aligned(sq, 16) || blocks >= (1LL << 32)) {
        set_error("wf_adamw_values: null or misaligned pointer");
        return WF_EINVAL;
    }
    over_grids((blocks + 3) / 4, kGridMost, [&](int64_t wg, uint32_t n) {              // (a workgroup reads 4 blocks)
        const int64_t b = 4 * wg;
        adamw_values<<<dim3(n), 256, 0, static_cast<hipStream_t>(stream)>>>(
            exp_avg + b * kBlock, exp_avg_sq + b * kBlock, avg_scale + b, sq_scale + b,
            reinterpret_cast<float4*>(avg + b * kBlock), reinterpret_cast<float4*>(sq + b * kBlock), (blocks - b) * 64);
    });
    WF_LAUNCH_CHECK("wf_adamw_values launch");
    return WF_OK;
}
