// Linear products with few rows (a handful of tokens, one batch of a classifier): the time is one pass over the weights.
//
// Every wave streams weights from memory straight into matrix-core operands - each weight is used once per row tile, LDS would only
// add a hop.  The sum over the contracted axis is divided over the eight waves of a workgroup, which add their accumulators
// in LDS in wave order, and (thin_fwd_kernel) over workgroups, whose sums gemm_join_kernel adds in split order.
// A lane loads 16 bytes along a row and the contraction order is permuted to match on both operands, so every load is a full
// 16 bytes: 64-byte runs along k for x w^T, 256-byte runs along the output for dz w and dz^T x.
// f32 products run on the f32 matrix instruction: exact products, f32 sums, no workspace copies of the operands.
#pragma once
#include "rows_gemm.h"

namespace srmi {

constexpr int THIN_WAVES = 8;

__device__ __forceinline__ bf16x8 thin_load(const bf16_t* p) { return __builtin_bit_cast(bf16x8, *(const u32x4_any*)p); }
__device__ __forceinline__ f32x4 thin_load(const float* p) { return *(const f32x4_any*)p; }
// 16 bytes of a row from column k on, zeros past K
__device__ __forceinline__ bf16x8 thin_load(const bf16_t* row, long long k, long long K) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if (k + 8 <= K) v = *(const u32x4_any*)(row + k);
    else if (k < K) {
        u16x8 t = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (k + j < K) t[j] = row[k + j];
        v = __builtin_bit_cast(u32x4, t);
    }
    return __builtin_bit_cast(bf16x8, v);
}
__device__ __forceinline__ f32x4 thin_load(const float* row, long long k, long long K) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (k + 4 <= K) v = *(const f32x4_any*)(row + k);
    else if (k < K) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (k + j < K) v[j] = row[k + j];
    }
    return v;
}
__device__ __forceinline__ f32x4 thin_mac(const bf16x8& a, const bf16x8& b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 thin_mac(const f32x4& a, const f32x4& b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
template <typename T> struct ThinVec;
template <> struct ThinVec<bf16_t> { typedef bf16x8 type; };
template <> struct ThinVec<float> { typedef f32x4 type; };

struct ThinArgs {
    TileArgs t;                   // a, b unused; tiles_n: column tiles of the launch, splits, part, epilogue
    const void* x; long long ldx; // rows operand [M, K] (dz [M, N] in the backward)
    const void* w; long long ldw; // weights [N, K]
};

// y[m, n] = epilogue(sum_k x[m, k] w[n, k]); workgroup: 16 columns, 16 MT rows, one split of k
template <typename T, int MT>
__global__ __launch_bounds__(64 * THIN_WAVES) void thin_fwd_kernel(ThinArgs p) {
    typedef typename ThinVec<T>::type vec;
    constexpr int V = 16 / (int)sizeof(T), STEPS = 64 / (4 * V), AHEAD = sizeof(T) == 4 || MT > 1 ? 2 : 4;      // loads of a chunk of 64 k, chunks in flight
    __shared__ f32x4 red[THIN_WAVES][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int tile = blockIdx.x % p.t.tiles_n, split = blockIdx.x / p.t.tiles_n, n0 = tile * 16;
    const long long m0 = (long long)blockIdx.y * (16 * MT);
    const long long K = p.t.K;
    // rows past the end repeat the last one: their results are not stored
    const T* wr = (const T*)p.w + (long long)min(n0 + r, p.t.N - 1) * p.ldw + V * q;
    const T* xr[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long long m = m0 + 16 * i + r;
        xr[i] = (const T*)p.x + (m < p.t.M ? m : p.t.M - 1) * p.ldx + V * q;
    }
    const int chunks = (int)((K + 63) / 64);
    const int c0 = (int)((long long)chunks * split / p.t.splits), c1 = (int)((long long)chunks * (split + 1) / p.t.splits);
    const int whole = min(c1, (int)(K / 64));                               // chunks without a ragged end
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // AHEAD chunks of the wave are in flight while one is multiplied; past the split: nothing is loaded or multiplied
    vec fw[AHEAD][STEPS], fx[AHEAD][MT][STEPS];
    auto load = [&](int u, int c) {
        if (c < whole) {
            const long long k = (long long)c * 64;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) fw[u][s] = thin_load(wr + k + 4 * V * s);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int s = 0; s < STEPS; ++s) fx[u][i][s] = thin_load(xr[i] + k + 4 * V * s);
        } else if (c < c1) {
            const long long k = (long long)c * 64, left = K - V * q;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) fw[u][s] = thin_load(wr, k + 4 * V * s, left);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int s = 0; s < STEPS; ++s) fx[u][i][s] = thin_load(xr[i], k + 4 * V * s, left);
        }
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) load(u, c0 + wave + u * THIN_WAVES);
    for (int c = c0 + wave; c < c1; c += THIN_WAVES * AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (c + u * THIN_WAVES >= c1) break;
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[i] = thin_mac(fw[u][s], fx[u][i][s], acc[i]);
            load(u, c + (AHEAD + u) * THIN_WAVES);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) red[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave >= MT) return;
    f32x4 sum = red[0][wave][lane];
#pragma unroll
    for (int k = 1; k < THIN_WAVES; ++k) sum += red[k][wave][lane];
    // the lane holds columns 4 q .. 4 q + 3 of row r of row tile `wave`
    const long long m = m0 + 16 * wave + r;
    const int n = n0 + 4 * q;
    if (m >= p.t.M || n >= p.t.N) return;
    if (p.t.splits > 1) {
        *(f32x4*)(p.t.part + ((size_t)split * p.t.M + m) * p.t.part_ld + n) = sum;
    } else {
        float v[4] = {sum[0], sum[1], sum[2], sum[3]}, bias[4];
        load_bias<T, 4>(p.t, n, bias);
        row_epilogue<T, 4>(p.t, v, bias, m, n);
    }
}

// dx[m, k] = sum_n dz[m, n] w[n, k], f32, at most 16 rows; workgroup: 64 columns
__global__ __launch_bounds__(64 * THIN_WAVES) void thin_dgrad_kernel(ThinArgs p) {
    __shared__ f32x4 red[THIN_WAVES][4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int k0 = blockIdx.x * 64, N = (int)p.t.K;                         // contracted: the N of the layer
    const float* w = (const float*)p.w;
    const float* zr = (const float*)p.x + min(r, (int)p.t.M - 1) * p.ldx;
    f32x4 acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int chunks = (N + 15) / 16;
    const bool whole = k0 + 64 <= p.t.N;
    for (int c = wave; c < chunks; c += 2 * THIN_WAVES) {
        f32x4 fz[2], fw[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int n = (c + u * THIN_WAVES) * 16 + 4 * q;                // contraction element s of lane group q: n + s
            fz[u] = thin_load(zr, n, N);
            if (whole) {
#pragma unroll
                for (int s = 0; s < 4; ++s) fw[u][s] = thin_load(w + (long long)min(n + s, N - 1) * p.ldw + k0 + 4 * r);
            } else {
#pragma unroll
                for (int s = 0; s < 4; ++s) fw[u][s] = thin_load(w + (long long)min(n + s, N - 1) * p.ldw, k0 + 4 * r, p.t.N);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int n = (c + u * THIN_WAVES) * 16 + 4 * q;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (n + s >= N) fw[u][s] = f32x4{0.f, 0.f, 0.f, 0.f};        // the repeated last row, which might not be finite
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fw[u][s][j], fz[u][s], acc[j], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) red[wave][j][lane] = acc[j];
    __syncthreads();
    // element i of tile j of lane (r, q): column k0 + 16 q + 4 i + j of row r; wave i < 4 adds up and stores those four columns
    const int i = wave;
    if (i >= 4) return;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = 0.f;
#pragma unroll
        for (int k = 0; k < THIN_WAVES; ++k) v[j] += ((const float*)&red[k][j][lane])[i];
    }
    const int k = k0 + 16 * q + 4 * i;
    if (r >= p.t.M || k >= p.t.N) return;
    float* y = (float*)p.t.y + r * p.t.ldy + k;
    if (k + 4 <= p.t.N) store_vec<4>(y, v);
    else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (k + j < p.t.N) y[j] = v[j];
    }
}

// dw[n, k] = sum_m dz[m, n] x[m, k], f32, few m; wave: 64 n x 64 k, bound by the store of dw
__global__ __launch_bounds__(256) void thin_wgrad_kernel(ThinArgs p, const float* x, long long ldx) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int M = (int)p.t.K, N = (int)p.t.M, K = p.t.N;                     // dw is [N, K]
    const unsigned kb = (K + 255) / 256;
    const int n0 = (int)(blockIdx.x / kb) * 64, k0 = (int)(blockIdx.x % kb * 4 + wave) * 64;
    if (k0 >= K) return;
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int m = q; m - q < M; m += 4) {
        const bool in = m < M;
        const f32x4 fx = in ? thin_load(x + m * ldx, k0 + 4 * r, K) : f32x4{0.f, 0.f, 0.f, 0.f};
        float fz[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) fz[i] = in && n0 + 16 * i + r < N ? ((const float*)p.x)[m * p.ldx + n0 + 16 * i + r] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fz[i], fx[j], acc[i][j], 0, 0, 0);
    }
    // element e of tile (i, j): row n0 + 16 i + 4 q + e, column k0 + 4 r + j
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int n = n0 + 16 * i + 4 * q + e, k = k0 + 4 * r;
            if (n >= N || k >= K) continue;
            const float v[4] = {acc[i][0][e], acc[i][1][e], acc[i][2][e], acc[i][3][e]};
            float* y = (float*)p.t.y + n * p.t.ldy + k;
            if (k + 4 <= K) store_vec<4>(y, v);
            else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (k + j < K) y[j] = v[j];
            }
        }
}

}  // namespace srmi
