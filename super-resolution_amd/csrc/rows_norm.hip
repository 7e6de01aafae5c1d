// Layer norm over the last axis, forward and backward.
//
//   mean = sum x / C,  rstd = 1 / sqrt(sum (x - mean)^2 / C + eps),  xh = (x - mean) rstd,  y = xh w + b
//   g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// HBM-bound: x is read once and stays in registers for both moments (the variance is summed from the deviations, not as
// E[x^2] - mean^2, which cancels), y is written once.  A row belongs to LANES lanes of one wave - 8 for 64 bf16 channels, 64
// from 512 up - so that every lane moves 16 B and narrow maps still fill the wave.  All statistics are f32.
// The backward keeps dw / db of a lane's columns in registers over all the rows its group visits, adds the groups of a
// workgroup in LDS and stores ONE partial row per workgroup; a second launch adds the partial rows in index order.  No
// atomics: the same input gives the same bits.
#include "rows_common.h"

namespace srmi {

struct NormArgs {
    const void* x; long long ldx;
    const void* w; const void* b;      // [C] or NULL
    void* y;                           // dense [rows, C]; the backward's dx
    float* mean; float* rstd;          // [rows]; NULL in a forward whose statistics nobody keeps
    const void* dy; long long lddy;
    float* part;                       // [gridDim.x][2][C]: dw, db
    long long rows;
    int C, p_bf16;
    float eps;
};

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

template <int V>
__device__ __forceinline__ void load_param(const void* p, int p_bf16, int c, float* o) {
    if (p_bf16) load_vec<V>((const bf16_t*)p + c, o);
    else load_vec<V>((const float*)p + c, o);
}

template <typename T, int LANES, int V, int ITER>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormArgs a) {
    const int l = threadIdx.x % LANES;
    const long long ngroups = (long long)gridDim.x * (256 / LANES);
    float w[ITER * V], b[ITER * V];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (i * LANES + l) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) { w[i * V + j] = 1.f; b[i * V + j] = 0.f; }
        if (c < a.C) {
            if (a.w) load_param<V>(a.w, a.p_bf16, c, w + i * V);
            if (a.b) load_param<V>(a.b, a.p_bf16, c, b + i * V);
        }
    }
    const float inv = 1.f / (float)a.C;
    for (long long r = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; r < a.rows; r += ngroups) {
        const T* x = (const T*)a.x + r * a.ldx;
        float v[ITER * V], s = 0.f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (i * LANES + l) * V;
            if (c < a.C) load_vec<V>(x + c, v + i * V);
            else {
#pragma unroll
                for (int j = 0; j < V; ++j) v[i * V + j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) s += v[i * V + j];
        }
        const float mean = group_sum<LANES>(s) * inv;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if ((i * LANES + l) * V < a.C) {
#pragma unroll
                for (int j = 0; j < V; ++j) { v[i * V + j] -= mean; q += v[i * V + j] * v[i * V + j]; }
            }
        }
        const float rstd = 1.f / sqrtf(group_sum<LANES>(q) * inv + a.eps);
        T* y = (T*)a.y + r * (long long)a.C;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (i * LANES + l) * V;
            if (c < a.C) {
                float o[V];
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] = v[i * V + j] * rstd * w[i * V + j] + b[i * V + j];
                store_vec<V>(y + c, o);
            }
        }
        if (a.mean && l == 0) { a.mean[r] = mean; a.rstd[r] = rstd; }
    }
}

template <typename T, int LANES, int V, int ITER>
__global__ __launch_bounds__(256) void norm_bwd_kernel(NormArgs a) {
    constexpr int G = 256 / LANES;
    __shared__ float red[G > 1 ? G : 1][LANES * V];
    const int l = threadIdx.x % LANES, gr = threadIdx.x / LANES;
    const long long ngroups = (long long)gridDim.x * G;
    float w[ITER * V], dw[ITER * V], db[ITER * V];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (i * LANES + l) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) { w[i * V + j] = 1.f; dw[i * V + j] = 0.f; db[i * V + j] = 0.f; }
        if (c < a.C && a.w) load_param<V>(a.w, a.p_bf16, c, w + i * V);
    }
    const float inv = 1.f / (float)a.C;
    for (long long r = (long long)blockIdx.x * G + gr; r < a.rows; r += ngroups) {
        const T* x = (const T*)a.x + r * a.ldx;
        const T* dy = (const T*)a.dy + r * a.lddy;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float xh[ITER * V], g[ITER * V], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (i * LANES + l) * V;
            if (c < a.C) {
                load_vec<V>(x + c, xh + i * V);
                load_vec<V>(dy + c, g + i * V);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int k = i * V + j;
                    xh[k] = (xh[k] - mean) * rstd;
                    dw[k] += g[k] * xh[k];
                    db[k] += g[k];
                    g[k] *= w[k];
                    s1 += g[k];
                    s2 += g[k] * xh[k];
                }
            }
        }
        if (a.y) {
            const float c1 = group_sum<LANES>(s1) * inv, c2 = group_sum<LANES>(s2) * inv;
            T* dx = (T*)a.y + r * (long long)a.C;
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                const int c = (i * LANES + l) * V;
                if (c < a.C) {
                    float o[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) o[j] = rstd * (g[i * V + j] - c1 - xh[i * V + j] * c2);
                    store_vec<V>(dx + c, o);
                }
            }
        }
    }
    if (!a.part) return;
    float* slot = a.part + (size_t)blockIdx.x * 2 * a.C;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j) red[gr][l * V + j] = which ? db[i * V + j] : dw[i * V + j];
            __syncthreads();
            for (int k = threadIdx.x; k < LANES * V; k += 256) {
                const int c = i * LANES * V + k;
                if (c < a.C) {
                    float s = 0.f;
#pragma unroll
                    for (int q = 0; q < G; ++q) s += red[q][k];
                    slot[which * a.C + c] = s;
                }
            }
        }
    }
}

// ---- rows too wide for registers: a workgroup per row, the row re-read from L1 / L2 ------------------------------------
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = group_sum<64>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

template <typename T, int V>
__global__ __launch_bounds__(256) void norm_wide_fwd_kernel(NormArgs a) {
    __shared__ float red[4];
    const float inv = 1.f / (float)a.C;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.ldx;
        T* y = (T*)a.y + r * (long long)a.C;
        float s = 0.f;
        for (int c = threadIdx.x * V; c < a.C; c += 256 * V) {
            float v[V];
            load_vec<V>(x + c, v);
#pragma unroll
            for (int j = 0; j < V; ++j) s += v[j];
        }
        const float mean = block_sum(s, red) * inv;
        float q = 0.f;
        for (int c = threadIdx.x * V; c < a.C; c += 256 * V) {
            float v[V];
            load_vec<V>(x + c, v);
#pragma unroll
            for (int j = 0; j < V; ++j) { v[j] -= mean; q += v[j] * v[j]; }
        }
        const float rstd = 1.f / sqrtf(block_sum(q, red) * inv + a.eps);
        for (int c = threadIdx.x * V; c < a.C; c += 256 * V) {
            float v[V], w[V], b[V];
            load_vec<V>(x + c, v);
#pragma unroll
            for (int j = 0; j < V; ++j) { w[j] = 1.f; b[j] = 0.f; }
            if (a.w) load_param<V>(a.w, a.p_bf16, c, w);
            if (a.b) load_param<V>(a.b, a.p_bf16, c, b);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (v[j] - mean) * rstd * w[j] + b[j];
            store_vec<V>(y + c, v);
        }
        if (a.mean && threadIdx.x == 0) { a.mean[r] = mean; a.rstd[r] = rstd; }
    }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void norm_wide_dx_kernel(NormArgs a) {
    __shared__ float red[4];
    const float inv = 1.f / (float)a.C;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.ldx;
        const T* dy = (const T*)a.dy + r * a.lddy;
        T* dx = (T*)a.y + r * (long long)a.C;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (int pass = 0; pass < 2; ++pass) {
            float c1 = 0.f, c2 = 0.f;
            if (pass) { c1 = block_sum(s1, red) * inv; c2 = block_sum(s2, red) * inv; }
            for (int c = threadIdx.x * V; c < a.C; c += 256 * V) {
                float xh[V], g[V], w[V];
                load_vec<V>(x + c, xh);
                load_vec<V>(dy + c, g);
#pragma unroll
                for (int j = 0; j < V; ++j) w[j] = 1.f;
                if (a.w) load_param<V>(a.w, a.p_bf16, c, w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    xh[j] = (xh[j] - mean) * rstd;
                    g[j] *= w[j];
                    if (!pass) { s1 += g[j]; s2 += g[j] * xh[j]; }
                    else g[j] = rstd * (g[j] - c1 - xh[j] * c2);
                }
                if (pass) store_vec<V>(dx + c, g);
            }
        }
    }
}

// dw / db of wide rows: workgroup (strip of 256 V columns, slot of rows); a lane owns V columns of the strip
template <typename T, int V>
__global__ __launch_bounds__(256) void norm_wide_dw_kernel(NormArgs a) {
    const int c = ((int)blockIdx.y * 256 + threadIdx.x) * V;
    if (c >= a.C) return;
    float dw[V], db[V];
#pragma unroll
    for (int j = 0; j < V; ++j) dw[j] = db[j] = 0.f;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        float x[V], dy[V];
        load_vec<V>((const T*)a.x + r * a.ldx + c, x);
        load_vec<V>((const T*)a.dy + r * a.lddy + c, dy);
        const float mean = a.mean[r], rstd = a.rstd[r];
#pragma unroll
        for (int j = 0; j < V; ++j) { dw[j] += dy[j] * ((x[j] - mean) * rstd); db[j] += dy[j]; }
    }
    float* slot = a.part + (size_t)blockIdx.x * 2 * a.C;
    store_vec<V>(slot + c, dw);
    if constexpr (V == 1) slot[a.C + c] = db[0];
    else store_vec<V>(slot + a.C + c, db);
}

// out[c] = sum over slots of part[slot][c], n columns; 32 columns x 8 slot lanes per workgroup, slots added in index order
// within a lane and the 8 lanes in index order.  Two outputs: columns [0, n0) to o0, [n0, n) to o1.
__global__ __launch_bounds__(256) void slot_sum_kernel(const float* part, int slots, int n, int n0, void* o0, void* o1, int out_bf16) {
    __shared__ float red[8][32];
    const int cl = threadIdx.x & 31, sl = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cl;
    float s = 0.f;
    if (c < n) {
        for (int k = sl; k < slots; k += 8) s += part[(size_t)k * n + c];
    }
    red[sl][cl] = s;
    __syncthreads();
    if (sl == 0 && c < n) {
#pragma unroll
        for (int k = 1; k < 8; ++k) s += red[k][cl];
        void* o = c < n0 ? o0 : o1;
        const int i = c < n0 ? c : c - n0;
        if (o) {
            if (out_bf16) ((bf16_t*)o)[i] = f2bf(s);
            else ((float*)o)[i] = s;
        }
    }
}

int slot_sum_launch(const float* part, int slots, int n, int n0, void* o0, void* o1, int out_bf16, hipStream_t s) {
    if (n == 0) return SRMI_OK;
    hipLaunchKernelGGL(slot_sum_kernel, dim3((n + 31) / 32), dim3(256), 0, s, part, slots, n, n0, o0, o1, out_bf16);
    return hip_check(hipGetLastError(), "slot_sum");
}

// ---- host ------------------------------------------------------------------------------------------------------------
// 16-byte accesses need every row of every operand on a 16-byte boundary and whole vectors per row
static bool norm_aligned(const NormArgs& a, int esz) {
    const int v = 16 / esz;
    uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.dy | (uintptr_t)a.w | (uintptr_t)a.b | (uintptr_t)a.part;
    return (bits & 15) == 0 && a.C % v == 0 && a.ldx % v == 0 && a.lddy % v == 0;
}

static constexpr int NORM_WIDE_V = 2048, NORM_WIDE_1 = 1024;      // widest row of the register kernels: vector / scalar accesses

int norm_slots(long long rows, int C) {
    (void)C;
    const long long want = (rows + 7) / 8;
    return (int)(want < 1 ? 1 : want > 512 ? 512 : want);
}

template <bool BWD, typename T, int LANES, int V, int ITER>
static void norm_go(const NormArgs& a, int slots, hipStream_t s) {
    const long long rpb = 256 / LANES;
    long long grid = (a.rows + rpb - 1) / rpb;
    if constexpr (BWD) {
        if (a.part || grid > slots) grid = slots;
        hipLaunchKernelGGL((norm_bwd_kernel<T, LANES, V, ITER>), dim3((unsigned)grid), dim3(256), 0, s, a);
    } else {
        if (grid > 2048) grid = 2048;
        hipLaunchKernelGGL((norm_fwd_kernel<T, LANES, V, ITER>), dim3((unsigned)grid), dim3(256), 0, s, a);
    }
}

template <bool BWD, typename T>
static void norm_dispatch(const NormArgs& a, bool vec, int slots, hipStream_t s) {
    const int C = a.C;
    constexpr int V = 16 / (int)sizeof(T);
    if (vec) {
        if (C <= 8 * V) norm_go<BWD, T, 8, V, 1>(a, slots, s);
        else if (C <= 16 * V) norm_go<BWD, T, 16, V, 1>(a, slots, s);
        else if (C <= 32 * V) norm_go<BWD, T, 32, V, 1>(a, slots, s);
        else if (C <= 64 * V) norm_go<BWD, T, 64, V, 1>(a, slots, s);
        else if (C <= 128 * V) norm_go<BWD, T, 64, V, 2>(a, slots, s);
        else if (C <= 256 * V) norm_go<BWD, T, 64, V, 4>(a, slots, s);
        else if constexpr (V == 4) norm_go<BWD, T, 64, V, 8>(a, slots, s);
    } else {
        if (C <= 16) norm_go<BWD, T, 16, 1, 1>(a, slots, s);
        else if (C <= 64) norm_go<BWD, T, 64, 1, 1>(a, slots, s);
        else if (C <= 128) norm_go<BWD, T, 64, 1, 2>(a, slots, s);
        else if (C <= 256) norm_go<BWD, T, 64, 1, 4>(a, slots, s);
        else if (C <= 512) norm_go<BWD, T, 64, 1, 8>(a, slots, s);
        else norm_go<BWD, T, 64, 1, 16>(a, slots, s);
    }
}

template <bool BWD, typename T>
static void norm_wide(const NormArgs& a, bool vec, int slots, hipStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    const unsigned grid = (unsigned)(a.rows > 4096 ? 4096 : a.rows);
    if constexpr (BWD) {
        if (a.y) {
            if (vec) hipLaunchKernelGGL((norm_wide_dx_kernel<T, V>), dim3(grid), dim3(256), 0, s, a);
            else hipLaunchKernelGGL((norm_wide_dx_kernel<T, 1>), dim3(grid), dim3(256), 0, s, a);
        }
        if (a.part) {
            if (vec) hipLaunchKernelGGL((norm_wide_dw_kernel<T, V>), dim3(slots, (a.C + 256 * V - 1) / (256 * V)), dim3(256), 0, s, a);
            else hipLaunchKernelGGL((norm_wide_dw_kernel<T, 1>), dim3(slots, (a.C + 255) / 256), dim3(256), 0, s, a);
        }
    } else {
        if (vec) hipLaunchKernelGGL((norm_wide_fwd_kernel<T, V>), dim3(grid), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((norm_wide_fwd_kernel<T, 1>), dim3(grid), dim3(256), 0, s, a);
    }
}

static void fill_args(NormArgs* a, const srmi_norm_desc& d, const void* x, const void* w, const void* b) {
    a->x = x; a->ldx = d.ldx; a->w = w; a->b = b; a->rows = d.rows; a->C = d.C; a->p_bf16 = d.param_dtype == SRMI_BF16; a->eps = d.eps;
    a->dy = nullptr; a->lddy = 0; a->part = nullptr;
}

int norm_fwd(const srmi_norm_desc& d, const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, hipStream_t s) {
    NormArgs a;
    fill_args(&a, d, x, w, b);
    a.y = y; a.mean = mean; a.rstd = rstd;
    const bool vec = norm_aligned(a, d.dtype == SRMI_BF16 ? 2 : 4);
    const bool wide = d.C > (vec ? NORM_WIDE_V : NORM_WIDE_1);
    if (d.dtype == SRMI_BF16) { if (wide) norm_wide<false, bf16_t>(a, vec, 0, s); else norm_dispatch<false, bf16_t>(a, vec, 0, s); }
    else { if (wide) norm_wide<false, float>(a, vec, 0, s); else norm_dispatch<false, float>(a, vec, 0, s); }
    return hip_check(hipGetLastError(), "layer_norm_fwd");
}

size_t norm_workspace_bytes(const srmi_norm_desc& d) { return (size_t)norm_slots(d.rows, d.C) * 2 * d.C * sizeof(float); }

int norm_bwd(const srmi_norm_desc& d, const void* x, const void* w, const float* mean, const float* rstd, const void* dy, void* dx,
             void* dw, void* db, float* ws, hipStream_t s) {
    NormArgs a;
    fill_args(&a, d, x, w, nullptr);
    a.y = dx; a.mean = (float*)mean; a.rstd = (float*)rstd; a.dy = dy; a.lddy = d.lddy;
    a.part = dw || db ? ws : nullptr;
    const int slots = norm_slots(d.rows, d.C);
    const bool vec = norm_aligned(a, d.dtype == SRMI_BF16 ? 2 : 4);
    const bool wide = d.C > (vec ? NORM_WIDE_V : NORM_WIDE_1);
    if (d.dtype == SRMI_BF16) { if (wide) norm_wide<true, bf16_t>(a, vec, slots, s); else norm_dispatch<true, bf16_t>(a, vec, slots, s); }
    else { if (wide) norm_wide<true, float>(a, vec, slots, s); else norm_dispatch<true, float>(a, vec, slots, s); }
    const int rc = hip_check(hipGetLastError(), "layer_norm_bwd");
    if (rc || !a.part) return rc;
    return slot_sum_launch(ws, slots, 2 * d.C, d.C, dw, db, d.param_dtype == SRMI_BF16, s);
}

}  // namespace srmi
