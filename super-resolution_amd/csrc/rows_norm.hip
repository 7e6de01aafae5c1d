// Layer norm over the last axis, forward and backward.
//
//   mean = sum x / C,  rstd = 1 / sqrt(sum (x - mean)^2 / C + eps),  xh = (x - mean) rstd,  y = xh w + b
//   g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// HBM-bound: x is read once and stays in registers for both moments (the variance is summed from the deviations, not as
// E[x^2] - mean^2, which cancels), y is written once.  A row belongs to LANES lanes of one wave - 8 for 64 bf16 channels, 64
// from 512 up - so that every lane moves 16 B and narrow maps still fill the wave; above four chunks a lane (2048 bf16, 1024 f32
// columns) to the four waves of a workgroup (4096 x 4096 bf16, against re-reading the row: forward 12.7 us / 17, backward 24 + 6 /
// 56 + 4 with dw in a pass of its own; 16384 x 8192: 92 / 137, 150 + 11 / 294 + 11; f32 16384 x 2048, against 32 values a lane of
// one wave: backward 64 / 87.  Four chunks a lane of one wave, bf16 16384 x 2048: backward 36 / 44 with one chunk of four waves).
// All statistics are f32.
// The backward keeps dw / db of a lane's columns in registers over all the rows its group visits, adds the groups of a
// workgroup in LDS and stores ONE partial row per workgroup; a second launch adds the partial rows in index order.  No
// atomics: the same input gives the same bits.
//
// 147456 x 256 bf16: forward 26 us (5.8 TB/s), backward 40 us (5.6 TB/s) + 6 for the partial rows; 8281 x 771 f32, rows off the line
// boundaries: 12.8 and 17.9 us (4.0 and 4.3 TB/s), + 4.
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
    bool past;                         // y goes past the caches
};

// sums over a row's lanes: part of a wave, or (256) the workgroup, whose four waves meet in `red`
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
struct Sum2 { float a, b; };
template <int LANES>
__device__ __forceinline__ Sum2 group_sum2(float a, float b, float (*red)[4]) {
    if constexpr (LANES <= 64) {
        return {lane_sum<LANES>(a), lane_sum<LANES>(b)};
    } else {
        a = lane_sum<64>(a);
        b = lane_sum<64>(b);
        __syncthreads();                     // the sums before these have been read
        if ((threadIdx.x & 63) == 0) { red[0][threadIdx.x >> 6] = a; red[1][threadIdx.x >> 6] = b; }
        __syncthreads();
        return {red[0][0] + red[0][1] + red[0][2] + red[0][3], red[1][0] + red[1][1] + red[1][2] + red[1][3]};
    }
}
template <int LANES>
__device__ __forceinline__ float group_sum(float v, float* red) {
    if constexpr (LANES <= 64) {
        return lane_sum<LANES>(v);
    } else {
        v = lane_sum<64>(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        return red[0] + red[1] + red[2] + red[3];
    }
}

// A lane's chunks of a row, 16 bytes each as they lie in memory (rows need no alignment: rows_common.h), zeros past C.  Apart from the
// conversion so that all loads of a row are on their way before the first is looked at: a lane's second chunk may lie past the
// row's end, and behind that test a conversion would wait for its own load alone.  TAIL: the row's last columns, C % V of
// them, are one lane's chunk number C / V / LANES.
__device__ __forceinline__ u32x4 load_tail(const float* p, int left) {
    float t[4];
    load_some<4>(p, left, t);
    return __builtin_bit_cast(u32x4, f32x4{t[0], t[1], t[2], t[3]});
}
__device__ __forceinline__ u32x4 load_tail(const bf16_t* p, int left) {
    u32x4 q;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned lo = p[min(2 * j, left - 1)], hi = p[min(2 * j + 1, left - 1)];
        q[j] = (2 * j < left ? lo : 0u) | (2 * j + 1 < left ? hi << 16 : 0u);
    }
    return q;
}
template <int LANES, int ITER, bool TAIL, typename T>
__device__ __forceinline__ void load_row(const T* p, int l, int C, u32x4* raw) {
    constexpr int V = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (i * LANES + l) * V;
        raw[i] = u32x4{0u, 0u, 0u, 0u};
        if (c + (TAIL ? V : 1) <= C) raw[i] = *(const u32x4_any*)(p + c);
        else if (TAIL && ITER == 1 && c < C) raw[i] = load_tail(p + c, C - c);
    }
    if constexpr (TAIL && ITER > 1) {                                    // one copy of these loads, not one for every chunk
        const int last = C / V;
        if (l == last % LANES) {
            const u32x4 q = load_tail(p + last * V, C - last * V);
#pragma unroll
            for (int i = 0; i < ITER; ++i)
                if (i == last / LANES) raw[i] = q;
        }
    }
}
template <int V, bool TAIL, typename T>
__device__ __forceinline__ void load_cols(const T* p, int c, int C, float* o) {
    if (!TAIL || c + V <= C) load_vec<V>(p + c, o);
    else load_some<V>(p + c, C - c, o);
}
template <int V, bool TAIL, typename T>
__device__ __forceinline__ void store_cols(T* p, int c, int C, const float* o, bool past = false) {
    if (!TAIL || c + V <= C) store_vec<V>(p + c, o, past);
    else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j < C) p[c + j] = from_f32<T>(o[j]);
    }
}
template <int V, bool TAIL>
__device__ __forceinline__ void load_param(const void* p, int p_bf16, int c, int C, float* o) {
    if (p_bf16) load_cols<V, TAIL>((const bf16_t*)p, c, C, o);
    else load_cols<V, TAIL>((const float*)p, c, C, o);
}

template <typename T, int LANES, int ITER, bool TAIL>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ float red[4];
    const int l = threadIdx.x % LANES;
    const long long ngroups = (long long)gridDim.x * (256 / LANES);
    float w[ITER * V], b[ITER * V];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (i * LANES + l) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) { w[i * V + j] = 1.f; b[i * V + j] = 0.f; }
        if (c < a.C) {
            if (a.w) load_param<V, TAIL>(a.w, a.p_bf16, c, a.C, w + i * V);
            if (a.b) load_param<V, TAIL>(a.b, a.p_bf16, c, a.C, b + i * V);
        }
    }
    const float inv = 1.f / (float)a.C;
    for (long long r = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; r < a.rows; r += ngroups) {
        const T* x = (const T*)a.x + r * a.ldx;
        u32x4 raw[ITER];
        load_row<LANES, ITER, TAIL>(x, l, a.C, raw);
        float v[ITER * V], s = 0.f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            unpack(raw[i], v + i * V, T());
#pragma unroll
            for (int j = 0; j < V; ++j) s += v[i * V + j];
        }
        const float mean = group_sum<LANES>(s, red) * inv;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if ((i * LANES + l) * V < a.C) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    v[i * V + j] -= mean;
                    if (!TAIL || (i * LANES + l) * V + j < a.C) q += v[i * V + j] * v[i * V + j];
                }
            }
        }
        const float rstd = 1.f / sqrtf(group_sum<LANES>(q, red) * inv + a.eps);
        T* y = (T*)a.y + r * (long long)a.C;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (i * LANES + l) * V;
            if (c < a.C) {
                float o[V];
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] = v[i * V + j] * rstd * w[i * V + j] + b[i * V + j];
                store_cols<V, TAIL>(y, c, a.C, o, a.past);
            }
        }
        if (a.mean && l == 0) { a.mean[r] = mean; a.rstd[r] = rstd; }
    }
}

template <typename T, int LANES, int ITER, bool TAIL>
__global__ __launch_bounds__(256, 2) void norm_bwd_kernel(NormArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    constexpr int G = 256 / LANES;
    __shared__ float red[G][LANES * V];
    __shared__ float sums[2][4];
    const int l = threadIdx.x % LANES, gr = threadIdx.x / LANES;
    const long long ngroups = (long long)gridDim.x * G;
    float w[ITER * V], dw[ITER * V], db[ITER * V];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (i * LANES + l) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) { w[i * V + j] = 1.f; dw[i * V + j] = 0.f; db[i * V + j] = 0.f; }
        if (c < a.C && a.w) load_param<V, TAIL>(a.w, a.p_bf16, c, a.C, w + i * V);
    }
    const float inv = 1.f / (float)a.C;
    for (long long r = (long long)blockIdx.x * G + gr; r < a.rows; r += ngroups) {
        const T* x = (const T*)a.x + r * a.ldx;
        const T* dy = (const T*)a.dy + r * a.lddy;
        const float mean = a.mean[r], rstd = a.rstd[r];
        u32x4 rx[ITER], rg[ITER];                                       // 0 past the end: adds nothing below
        load_row<LANES, ITER, TAIL>(x, l, a.C, rx);
        load_row<LANES, ITER, TAIL>(dy, l, a.C, rg);
        float xh[ITER * V], g[ITER * V], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (i * LANES + l) * V;
            if (c < a.C) {
                unpack(rx[i], xh + i * V, T());
                unpack(rg[i], g + i * V, T());
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
            const Sum2 t = group_sum2<LANES>(s1, s2, sums);
            const float c1 = t.a * inv, c2 = t.b * inv;
            T* dx = (T*)a.y + r * (long long)a.C;
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                const int c = (i * LANES + l) * V;
                if (c < a.C) {
                    float o[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) o[j] = rstd * (g[i * V + j] - c1 - xh[i * V + j] * c2);
                    store_cols<V, TAIL>(dx, c, a.C, o, a.past);
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
template <typename T>
__global__ __launch_bounds__(256) void norm_wide_fwd_kernel(NormArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ float red[4];
    const float inv = 1.f / (float)a.C;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.ldx;
        T* y = (T*)a.y + r * (long long)a.C;
        float s = 0.f;
        for (int c = threadIdx.x * V; c < a.C; c += 256 * V) {
            float v[V];
            load_cols<V, true>(x, c, a.C, v);
#pragma unroll
            for (int j = 0; j < V; ++j) s += v[j];
        }
        const float mean = group_sum<256>(s, red) * inv;
        float q = 0.f;
        for (int c = threadIdx.x * V; c < a.C; c += 256 * V) {
            float v[V];
            load_cols<V, true>(x, c, a.C, v);
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < a.C) { v[j] -= mean; q += v[j] * v[j]; }
        }
        const float rstd = 1.f / sqrtf(group_sum<256>(q, red) * inv + a.eps);
        for (int c = threadIdx.x * V; c < a.C; c += 256 * V) {
            float v[V], w[V], b[V];
            load_cols<V, true>(x, c, a.C, v);
#pragma unroll
            for (int j = 0; j < V; ++j) { w[j] = 1.f; b[j] = 0.f; }
            if (a.w) load_param<V, true>(a.w, a.p_bf16, c, a.C, w);
            if (a.b) load_param<V, true>(a.b, a.p_bf16, c, a.C, b);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (v[j] - mean) * rstd * w[j] + b[j];
            store_cols<V, true>(y, c, a.C, v, a.past);
        }
        if (a.mean && threadIdx.x == 0) { a.mean[r] = mean; a.rstd[r] = rstd; }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void norm_wide_dx_kernel(NormArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ float red[2][4];
    const float inv = 1.f / (float)a.C;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.ldx;
        const T* dy = (const T*)a.dy + r * a.lddy;
        T* dx = (T*)a.y + r * (long long)a.C;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (int pass = 0; pass < 2; ++pass) {
            float c1 = 0.f, c2 = 0.f;
            if (pass) {
                const Sum2 t = group_sum2<256>(s1, s2, red);
                c1 = t.a * inv;
                c2 = t.b * inv;
            }
            for (int c = threadIdx.x * V; c < a.C; c += 256 * V) {
                float xh[V], g[V], w[V];
                load_cols<V, true>(x, c, a.C, xh);
                load_cols<V, true>(dy, c, a.C, g);
#pragma unroll
                for (int j = 0; j < V; ++j) w[j] = 1.f;
                if (a.w) load_param<V, true>(a.w, a.p_bf16, c, a.C, w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    xh[j] = (xh[j] - mean) * rstd;
                    g[j] *= w[j];
                    if (!pass) { s1 += g[j]; s2 += g[j] * xh[j]; }
                    else g[j] = rstd * (g[j] - c1 - xh[j] * c2);
                }
                if (pass) store_cols<V, true>(dx, c, a.C, g, a.past);
            }
        }
    }
}

// dw / db of wide rows: workgroup (strip of 256 V columns, slot of rows); a lane owns V columns of the strip
template <typename T>
__global__ __launch_bounds__(256) void norm_wide_dw_kernel(NormArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    const int c = ((int)blockIdx.y * 256 + threadIdx.x) * V;
    if (c >= a.C) return;
    float dw[V], db[V];
#pragma unroll
    for (int j = 0; j < V; ++j) dw[j] = db[j] = 0.f;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        float x[V], dy[V];
        load_cols<V, true>((const T*)a.x + r * a.ldx, c, a.C, x);
        load_cols<V, true>((const T*)a.dy + r * a.lddy, c, a.C, dy);
        const float mean = a.mean[r], rstd = a.rstd[r];
#pragma unroll
        for (int j = 0; j < V; ++j) { dw[j] += dy[j] * ((x[j] - mean) * rstd); db[j] += dy[j]; }
    }
    float* slot = a.part + (size_t)blockIdx.x * 2 * a.C;
    store_cols<V, true>(slot, c, a.C, dw);
    store_cols<V, true>(slot + a.C, c, a.C, db);
}

// out[c] = sum over slots of part[slot][c], n columns.  16 columns x 64 lanes per workgroup: lane k adds slots k, k + 64, ... in order, then
// four lanes at a time and the sixteen sums are added in order.  (Many lanes per column because the launch waits on memory, not on
// bandwidth: 512 slots of 512 columns took 20 us with 8 lanes.)  Two outputs: columns [0, n0) to o0, [n0, n) to o1.
// A launch has fewer than 2^32 threads, 64 for a column: the widest rows (n = 2^26) walk the grid more than once.
__global__ __launch_bounds__(1024) void slot_sum_kernel(const float* part, int slots, int n, int n0, void* o0, void* o1, int out_bf16) {
    __shared__ float red[64][17];
    const int cl = threadIdx.x & 15, sl = threadIdx.x >> 4;
    for (int c0 = blockIdx.x * 16; c0 < n; c0 += gridDim.x * 16) {
        const int c = c0 + cl;
        float s = 0.f;
        if (c < n) {
#pragma unroll 4
            for (int k = sl; k < slots; k += 64) s += part[(size_t)k * n + c];
        }
        red[sl][cl] = s;
        __syncthreads();
        if (sl < 16) s = red[4 * sl][cl] + red[4 * sl + 1][cl] + red[4 * sl + 2][cl] + red[4 * sl + 3][cl];
        __syncthreads();
        if (sl < 16) red[sl][cl] = s;
        __syncthreads();
        if (sl == 0 && c < n) {
#pragma unroll
            for (int k = 1; k < 16; ++k) s += red[k][cl];
            void* o = c < n0 ? o0 : o1;
            const int i = c < n0 ? c : c - n0;
            if (o) {
                if (out_bf16) ((bf16_t*)o)[i] = f2bf(s);
                else ((float*)o)[i] = s;
            }
        }
        __syncthreads();                     // red is written again
    }
}

int slot_sum_launch(const float* part, int slots, int n, int n0, void* o0, void* o1, int out_bf16, hipStream_t s) {
    if (n == 0) return SRMI_OK;
    const int blocks = (n + 15) / 16, most = 1 << 21;
    hipLaunchKernelGGL(slot_sum_kernel, dim3(blocks < most ? blocks : most), dim3(1024), 0, s, part, slots, n, n0, o0, o1, out_bf16);
    return hip_check(hipGetLastError(), "slot_sum");
}

// ---- host ------------------------------------------------------------------------------------------------------------
static constexpr int NORM_WIDE = 8192;      // widest row kept in registers: 32 values a lane; the re-reading kernels take what is wider

static int norm_lanes(int C, int dtype) {
    const int v = dtype == SRMI_BF16 ? 8 : 4;
    return C <= 8 * v ? 8 : C <= 16 * v ? 16 : C <= 32 * v ? 32 : C <= 256 * v ? 64 : 256;
}

// Workgroups of the backward = partial rows of dw / db: eight per CU where there are rows for them (147456 x 256 bf16: 58 us with 512
// workgroups, 47 with 2048, 40 with dx past the caches) and the partial rows stay below an eighth of x's bytes.
int norm_slots(const srmi_norm_desc& d) {
    const long long esz = d.dtype == SRMI_BF16 ? 2 : 4, per = 256 / norm_lanes(d.C, d.dtype);
    long long most = d.rows * esz / 64;
    // rows of a workgroup's width: two per CU at least (4096 x 4096 bf16: 33 + 5 us with 256 workgroups, 24 + 6 with 512)
    const int least = per == 1 ? 512 : 64;
    most = most < least ? least : most > 2048 ? 2048 : most;
    // wide rows: a workgroup owns a strip of columns of its rows, so fewer slots fill the chip
    const long long strips = d.C > NORM_WIDE ? (d.C * esz + 4095) / 4096 : 1;
    if (most > 2048 / strips) most = 2048 / strips;
    if (most < 1) most = 1;
    const long long want = (d.rows + per - 1) / per;
    return (int)(want < 1 ? 1 : want > most ? most : want);
}

template <bool BWD, typename T, int LANES, int ITER, bool TAIL>
static void norm_go(const NormArgs& a, int slots, hipStream_t s) {
    const long long rpb = 256 / LANES;
    long long grid = (a.rows + rpb - 1) / rpb;
    if constexpr (BWD) {
        if (a.part || grid > slots) grid = slots;
        hipLaunchKernelGGL((norm_bwd_kernel<T, LANES, ITER, TAIL>), dim3((unsigned)grid), dim3(256), 0, s, a);
    } else {
        if (grid > 2048) grid = 2048;
        hipLaunchKernelGGL((norm_fwd_kernel<T, LANES, ITER, TAIL>), dim3((unsigned)grid), dim3(256), 0, s, a);
    }
}

template <bool BWD, typename T, bool TAIL>
static void norm_rows(const NormArgs& a, int slots, hipStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    const int C = a.C;
    switch (norm_lanes(C, V == 8 ? SRMI_BF16 : SRMI_F32)) {
        case 8: norm_go<BWD, T, 8, 1, TAIL>(a, slots, s); return;
        case 16: norm_go<BWD, T, 16, 1, TAIL>(a, slots, s); return;
        case 32: norm_go<BWD, T, 32, 1, TAIL>(a, slots, s); return;
        default: break;
    }
    if (C <= 64 * V) norm_go<BWD, T, 64, 1, TAIL>(a, slots, s);
    else if (C <= 128 * V) norm_go<BWD, T, 64, 2, TAIL>(a, slots, s);
    else if (C <= 256 * V) norm_go<BWD, T, 64, 4, TAIL>(a, slots, s);
    else if (C <= 512 * V) norm_go<BWD, T, 256, 2, TAIL>(a, slots, s);
    else if (C <= 1024 * V) norm_go<BWD, T, 256, 4, TAIL>(a, slots, s);
    else if constexpr (V == 4) norm_go<BWD, T, 256, 8, TAIL>(a, slots, s);
}

template <bool BWD, typename T>
static void norm_wide(const NormArgs& a, int slots, hipStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    const unsigned grid = (unsigned)(a.rows > 4096 ? 4096 : a.rows);
    if constexpr (BWD) {
        if (a.y && grid) hipLaunchKernelGGL((norm_wide_dx_kernel<T>), dim3(grid), dim3(256), 0, s, a);
        if (a.part) hipLaunchKernelGGL((norm_wide_dw_kernel<T>), dim3(slots, (a.C + 256 * V - 1) / (256 * V)), dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL((norm_wide_fwd_kernel<T>), dim3(grid), dim3(256), 0, s, a);
    }
}

template <bool BWD, typename T>
static void norm_dispatch(const NormArgs& a, int slots, hipStream_t s) {
    if (a.C > NORM_WIDE) norm_wide<BWD, T>(a, slots, s);
    else if (a.C % (16 / (int)sizeof(T))) norm_rows<BWD, T, true>(a, slots, s);
    else norm_rows<BWD, T, false>(a, slots, s);
}

static void fill_args(NormArgs* a, const srmi_norm_desc& d, const void* x, const void* w, const void* b) {
    a->x = x; a->ldx = d.ldx; a->w = w; a->b = b; a->rows = d.rows; a->C = d.C; a->p_bf16 = d.param_dtype == SRMI_BF16; a->eps = d.eps;
    a->dy = nullptr; a->lddy = 0; a->part = nullptr;
    a->past = (size_t)d.rows * d.C * (d.dtype == SRMI_BF16 ? 2 : 4) > STREAM_BYTES;
}

int norm_fwd(const srmi_norm_desc& d, const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, hipStream_t s) {
    NormArgs a;
    fill_args(&a, d, x, w, b);
    a.y = y; a.mean = mean; a.rstd = rstd;
    if (d.dtype == SRMI_BF16) norm_dispatch<false, bf16_t>(a, 0, s);
    else norm_dispatch<false, float>(a, 0, s);
    return hip_check(hipGetLastError(), "layer_norm_fwd");
}

size_t norm_workspace_bytes(const srmi_norm_desc& d) { return (size_t)norm_slots(d) * 2 * d.C * sizeof(float); }

int norm_bwd(const srmi_norm_desc& d, const void* x, const void* w, const float* mean, const float* rstd, const void* dy, void* dx,
             void* dw, void* db, float* ws, hipStream_t s) {
    NormArgs a;
    fill_args(&a, d, x, w, nullptr);
    a.y = dx; a.mean = (float*)mean; a.rstd = (float*)rstd; a.dy = dy; a.lddy = d.lddy;
    a.part = dw || db ? ws : nullptr;
    const int slots = norm_slots(d);
    if (d.dtype == SRMI_BF16) norm_dispatch<true, bf16_t>(a, slots, s);
    else norm_dispatch<true, float>(a, slots, s);
    const int rc = hip_check(hipGetLastError(), "layer_norm_bwd");
    if (rc || !a.part) return rc;
    return slot_sum_launch(ws, slots, 2 * d.C, d.C, dw, db, d.param_dtype == SRMI_BF16, s);
}

}  // namespace srmi
