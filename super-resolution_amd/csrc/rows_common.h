// Shared pieces of the row operators (linear, layer norm, dropout): storage conversion, activations and their slopes.
#pragma once
#include "common.h"

namespace srmi {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return bf2f(v); }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) { return f2bf(v); }

// V consecutive elements as f32, at any element's address: global memory takes unaligned 16-byte accesses on this target
// (aligned ones are faster where rows allow them, nothing else changes).
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
template <int V>
__device__ __forceinline__ void load_vec(const float* p, float* o) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        const f32x4 q = *(const f32x4_any*)(p + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i + j] = q[j];
    }
}
template <int V>
__device__ __forceinline__ void load_vec(const bf16_t* p, float* o) {
    if constexpr (V == 4) {
        const u32x2 q = *(const u32x2_any*)p;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            o[2 * j] = __builtin_bit_cast(float, q[j] << 16);
            o[2 * j + 1] = __builtin_bit_cast(float, q[j] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 8) {
            const u32x4 q = *(const u32x4_any*)(p + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[i + 2 * j] = __builtin_bit_cast(float, q[j] << 16);
                o[i + 2 * j + 1] = __builtin_bit_cast(float, q[j] & 0xffff0000u);
            }
        }
    }
}
// W times 16 bytes (or 8 bytes) to any element's address; `past`: past the caches (below)
template <int W>
__device__ __forceinline__ void put(u32x4_any* p, const u32x4* v, bool past) {
    if (past) {
        asm volatile("");                    // (keeps the compiler from merging the two kinds of store into ordinary ones)
#pragma unroll
        for (int i = 0; i < W; ++i) __builtin_nontemporal_store(v[i], p + i);
        asm volatile("");
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) p[i] = v[i];
    }
}
__device__ __forceinline__ void put(u32x2_any* p, const u32x2& v, bool past) {
    if (past) {
        asm volatile("");
        __builtin_nontemporal_store(v, p);
        asm volatile("");
    } else {
        *p = v;
    }
}
// An output larger than the eight L2s together is stored past them: nothing of it is there when it is read, and the operands that are read
// next to it stay.  147456 x 256 bf16 (75 MB): layer norm's backward pass 40 us against 48, dropout 34 + 26 against 42 + 31; a
// 16384 x 4096 product 450 against 470.  Smaller ones are better left in the caches: 9216 x 1024 (19 MB) of dz written past
// them cost the product that reads it 16.4 us instead of 14.4, and the kernel that writes it gained nothing.
constexpr size_t STREAM_BYTES = 32u << 20;
template <int V>
__device__ __forceinline__ void store_vec(float* p, const float* v, bool past = false) {
    if constexpr (V == 1) {
        p[0] = v[0];
    } else {
        u32x4 q[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i) q[i] = __builtin_bit_cast(u32x4, f32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]});
        put<V / 4>((u32x4_any*)p, q, past);
    }
}
template <int V>
__device__ __forceinline__ void store_vec(bf16_t* p, const float* v, bool past = false) {
    if constexpr (V == 4) {
        put((u32x2_any*)p, u32x2{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3])}, past);
    } else {
        static_assert(V == 8, "one 16-byte store");
        const u32x4 q = {pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7])};
        put<1>((u32x4_any*)p, &q, past);
    }
}

// What the forward pass keeps of a pre-activation for the backward pass: f32 for f32 rows; for bf16 rows an IEEE half - the same two bytes,
// but 11 significant bits, so that act'(z) adds nothing visible to the one rounding of dz = dy act'(z) (with bf16 the gradients'
// error grew from 1.41 to 1.6 times that of one rounding).  Beyond +-65504 it is an infinity, where every slope has the
// same limit as at 100.
template <typename T> struct KeptZ { typedef float type; };
template <> struct KeptZ<bf16_t> { typedef _Float16 type; };
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
template <int V>
__device__ __forceinline__ void store_vec(_Float16* p, const float* v, bool past = false) {
    if constexpr (V == 1) {
        p[0] = (_Float16)v[0];
    } else if constexpr (V == 4) {
        put((u32x2_any*)p, __builtin_bit_cast(u32x2, f16x4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]}), past);
    } else {
        f16x8 h;
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = (_Float16)v[j];
        const u32x4 q = __builtin_bit_cast(u32x4, h);
        put<1>((u32x4_any*)p, &q, past);
    }
}

// 16 bytes of storage as f32
__device__ __forceinline__ void unpack(const u32x4& q, float* o, float) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned v = q[j];
        o[j] = __builtin_bit_cast(float, v);
    }
}
__device__ __forceinline__ void unpack(const u32x4& q, float* o, bf16_t) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned v = q[j];
        o[2 * j] = __builtin_bit_cast(float, v << 16);
        o[2 * j + 1] = __builtin_bit_cast(float, v & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack(const u32x4& q, float* o, _Float16) {
    const f16x8 h = __builtin_bit_cast(f16x8, q);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (float)h[j];
}
// eight elements as they lie in memory: loads whose conversion comes later do not wait for one another
template <typename T>
struct Raw8 {
    u32x4 q[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int h = 0; h < (int)sizeof(T) / 2; ++h) q[h] = ((const u32x4_any*)p)[h];
    }
    __device__ __forceinline__ void get(float* o) const {
#pragma unroll
        for (int h = 0; h < (int)sizeof(T) / 2; ++h) unpack(q[h], o + 4 * h, T());
    }
};

// The first `left` (1 .. V - 1) of V elements, zeros behind them.  Past the last one it is loaded again: loads that each stand behind a
// test of their own would wait for one another.
template <int V, typename T>
__device__ __forceinline__ void load_some(const T* p, int left, float* o) {
    T t[V];
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = p[min(j, left - 1)];
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = j < left ? to_f32(t[j]) : 0.f;
}

// exp and division of the epilogues.  Where the result is stored in bf16 (half a step = 2^-8 of the value) the hardware's
// 2^x and reciprocal, a few 2^-23 off, are enough; f32 results take the library's functions.
template <bool FAST> __device__ __forceinline__ float exp_(float v) {
    if constexpr (FAST) return __builtin_amdgcn_exp2f(v * 1.442695040888963f);
    else return expf(v);
}
template <bool FAST> __device__ __forceinline__ float div_(float a, float b) {
    if constexpr (FAST) return a * __builtin_amdgcn_rcpf(b);
    else return a / b;
}
template <bool FAST> __device__ __forceinline__ float logistic(float v) { return div_<FAST>(1.f, 1.f + exp_<FAST>(-v)); }

// E = exp(-z^2 / 2) and q = Phi(-|z|) for bf16 results: q = E u P(u), u = 1 / (1 + 0.38 |z|), P of degree 4 fitted to
// Phi(-t) exp(t^2 / 2) on t in [0, 14] for the least relative error, 3.5e-5 (the storage rounds by up to 3.9e-3); the same
// relative error holds far out, where 1 + erf(z / sqrt 2) would cancel, at a third of an erf's instructions.
__device__ __forceinline__ void normal_tail(float z, float& E, float& q) {
    const float t = fabsf(z);
    E = __builtin_amdgcn_exp2f(-0.72134752044448170f * t * t);
    const float u = __builtin_amdgcn_rcpf(1.f + 0.38f * t);
    q = E * u * (0.15122523f + u * (0.157829f + u * (0.09198039f + u * (0.18887625f - u * 0.0899284f))));
}
// infinities to where every activation has its limit (NaN stays)
__device__ __forceinline__ float bounded(float z, float most) { return fabsf(z) > most ? copysignf(most, z) : z; }

constexpr float GELU_2C = 1.5957691216057308f;      // 2 sqrt(2 / pi)
constexpr float GELU_K = 0.044715f;

// act(z).  gelu = z Phi(z); its tanh form is z * logistic(2 sqrt(2/pi) (z + 0.044715 z^3)) since (1 + tanh u)/2 = logistic(2u):
// no cancellation for negative z.
template <bool FAST>
__device__ __forceinline__ float row_act(float z, int act, float param) {
    switch (act) {
        case SRMI_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
        case SRMI_ACT_LRELU: return z >= 0.f ? z : z * param;
        case SRMI_ACT_TANH:
            if constexpr (FAST) {                              // (1 - e) / (1 + e) cancels near 0: three terms of the series there
                const float t = fabsf(z), e = exp_<true>(-2.f * t), s = z * z;
                const float far = (1.f - e) * __builtin_amdgcn_rcpf(1.f + e);
                return t < 0.06f ? z * (1.f - s * (0.33333333f - s * 0.13333333f)) : copysignf(far, z);
            } else {
                return tanhf(z);
            }
        case SRMI_ACT_SIGMOID: return logistic<FAST>(z);
        case SRMI_ACT_GELU:
            if constexpr (FAST) {
                float E, q;
                const float t = fabsf(z) > 100.f ? 100.f : fabsf(z);           // (NaN stays)
                normal_tail(t, E, q);
                return __builtin_amdgcn_fmed3f(z, 0.f, __builtin_inff()) - t * q;
            } else {
                return 0.5f * z * erfcf(-0.70710678118654752f * z);
            }
        case SRMI_ACT_GELU_TANH: return z * logistic<FAST>(GELU_2C * (z + GELU_K * z * z * z));
        case SRMI_ACT_SILU: return z * logistic<FAST>(z);
        default: return z;
    }
}

// d act / d z at z, its limit at infinities; at the kinks torch's: 0 counts as negative.  tanh and sigmoid from e = exp(-k|z|): 1 - t^2
// and s (1 - s) would cancel for large |z|.
template <bool FAST>
__device__ __forceinline__ float row_act_slope(float z, int act, float param) {
    z = bounded(z, 100.f);
    switch (act) {
        case SRMI_ACT_RELU: return z <= 0.f ? 0.f : 1.f;
        case SRMI_ACT_LRELU: return z > 0.f ? 1.f : param;
        case SRMI_ACT_TANH: {
            const float e = exp_<FAST>(-2.f * fabsf(z)), d = 1.f + e;
            return div_<FAST>(4.f * e, d * d);
        }
        case SRMI_ACT_SIGMOID: {
            const float e = exp_<FAST>(-fabsf(z)), d = 1.f + e;
            return div_<FAST>(e, d * d);
        }
        case SRMI_ACT_GELU:
            if constexpr (FAST) {
                float E, q;
                normal_tail(z, E, q);
                return (z < 0.f ? q : 1.f - q) + z * 0.3989422804014327f * E;
            } else {
                return 0.5f * erfcf(-0.70710678118654752f * z) + z * 0.3989422804014327f * expf(-0.5f * z * z);
            }
        case SRMI_ACT_GELU_TANH: {
            const float s = logistic<FAST>(GELU_2C * (z + GELU_K * z * z * z));
            return s + z * s * (1.f - s) * GELU_2C * (1.f + 3.f * GELU_K * z * z);
        }
        case SRMI_ACT_SILU: {
            const float s = logistic<FAST>(z);
            return s + z * s * (1.f - s);
        }
        default: return 1.f;
    }
}

__device__ __forceinline__ bool is_kink(int act) { return act == SRMI_ACT_RELU || act == SRMI_ACT_LRELU; }

// v = act(v) / g *= act'(z) for V values: one branch on the (uniform) activation, not one per value
#define SRMI_ROW_ACTS(CASE) \
    CASE(SRMI_ACT_RELU) CASE(SRMI_ACT_LRELU) CASE(SRMI_ACT_TANH) CASE(SRMI_ACT_SIGMOID) CASE(SRMI_ACT_GELU) CASE(SRMI_ACT_GELU_TANH) CASE(SRMI_ACT_SILU)
template <int V, bool FAST>
__device__ __forceinline__ void row_act_vec(float* v, int act, float param) {
    switch (act) {
#define SRMI_CASE(CODE) \
    case CODE: { _Pragma("unroll") for (int j = 0; j < V; ++j) v[j] = row_act<FAST>(v[j], CODE, param); break; }
        SRMI_ROW_ACTS(SRMI_CASE)
#undef SRMI_CASE
        default: break;
    }
}
template <int V, bool FAST>
__device__ __forceinline__ void row_slope_vec(float* g, const float* z, int act, float param) {
    switch (act) {
#define SRMI_CASE(CODE) \
    case CODE: { _Pragma("unroll") for (int j = 0; j < V; ++j) g[j] *= row_act_slope<FAST>(z[j], CODE, param); break; }
        SRMI_ROW_ACTS(SRMI_CASE)
#undef SRMI_CASE
        default: break;
    }
}
#undef SRMI_ROW_ACTS

}  // namespace srmi
