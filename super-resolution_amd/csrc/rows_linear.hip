// Linear layers on rows: y = act(x w^T + b) + residual, and the backward pass.
//
//   z = x w^T + b          [M, N] = [M, K] [N, K]^T
//   dz = dy act'(z)        db = sum_m dz
//   dx = dz w              [M, K] = [M, N] [N, K]
//   dw = dz^T x            [N, K] = [M, N]^T [M, K]
//
// All three products are one kernel over operands addressed by (row, k) strides, accumulated in f32 on the matrix cores.
#include "rows_common.h"

namespace srmi {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

int slot_sum_launch(const float* part, int slots, int n, int n0, void* o0, void* o1, int out_bf16, hipStream_t s);

struct GemmArgs {
    const void* a; const void* b;                       // element (row, k) at row * s?r + k * s?k
    long long sar, sak, sbr, sbk;
    long long M; int N; long long K;
    const void* bias; const void* residual; void* y; void* z;
    long long ldr, ldy;                                 // z is dense [M, N]
    int act; float act_param;
};

constexpr int SG_T = 64, SG_K = 32;

template <typename T>
__global__ __launch_bounds__(256) void gemm_small_kernel(GemmArgs p) {
    constexpr bool BF = sizeof(T) == 2;
    constexpr int PITCH = SG_K + (BF ? 8 : 4);
    __shared__ __align__(16) T As[SG_T][PITCH], Bs[SG_T][PITCH];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long m0 = (long long)blockIdx.x * SG_T;
    const int n0 = blockIdx.y * SG_T;
    const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
    f32x4 acc[2][2] = {};
    for (long long k0 = 0; k0 < p.K; k0 += SG_K) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < SG_T * SG_K / 256; ++i) {
            const int e = tid + 256 * i;
            int r, k;
            if (p.sak == 1) { r = e / SG_K; k = e % SG_K; } else { r = e % SG_T; k = e / SG_T; }
            As[r][k] = m0 + r < p.M && k0 + k < p.K ? ((const T*)p.a)[(m0 + r) * p.sar + (k0 + k) * p.sak] : (T)0;
            if (p.sbk == 1) { r = e / SG_K; k = e % SG_K; } else { r = e % SG_T; k = e / SG_T; }
            Bs[r][k] = n0 + r < p.N && k0 + k < p.K ? ((const T*)p.b)[(n0 + r) * p.sbr + (k0 + k) * p.sbk] : (T)0;
        }
        __syncthreads();
        if constexpr (BF) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const bf16x8 fb = *(const bf16x8*)&Bs[wn + 16 * j + (lane & 15)][8 * (lane >> 4)];
                    const bf16x8 fa = *(const bf16x8*)&As[wm + 16 * i + (lane & 15)][8 * (lane >> 4)];
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb, fa, acc[i][j], 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int k = 0; k < SG_K; k += 4)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(Bs[wn + 16 * j + (lane & 15)][k + (lane >> 4)],
                                                                          As[wm + 16 * i + (lane & 15)][k + (lane >> 4)], acc[i][j], 0, 0, 0);
        }
    }
    // the column operand is MFMA's first: a lane holds four consecutive n of one m
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const long long m = m0 + wm + 16 * i + (lane & 15);
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = n0 + wn + 16 * j + 4 * (lane >> 4) + e;
                if (n >= p.N) continue;
                float v = acc[i][j][e];
                if (p.bias) v += to_f32(((const T*)p.bias)[n]);
                if (p.z) ((T*)p.z)[m * p.N + n] = from_f32<T>(v);
                v = row_act<BF>(v, p.act, p.act_param);
                if (p.residual) v += to_f32(((const T*)p.residual)[m * p.ldr + n]);
                ((T*)p.y)[m * p.ldy + n] = from_f32<T>(v);
            }
    }
}

template <typename T>
static int gemm(const GemmArgs& p, hipStream_t s) {
    if (p.M == 0 || p.N == 0) return SRMI_OK;
    const long long gx = (p.M + SG_T - 1) / SG_T;
    const int gy = (p.N + SG_T - 1) / SG_T;
    hipLaunchKernelGGL((gemm_small_kernel<T>), dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, s, p);
    return hip_check(hipGetLastError(), "linear gemm");
}

// ---- dz = dy * act'(saved) and the partial column sums of dz ----------------------------------------------------------
// Workgroup (slot of rows, strip of columns): TX lanes across columns, 256 / TX rows at a time; the sums of a workgroup's rows
// are added in LDS and stored as one partial row, a second launch adds the partial rows in index order.  db sums the f32
// products, before dz is rounded to its storage type.
struct DzArgs {
    const void* dy; long long lddy;
    const void* saved;                // dense [M, N]: z, or y where its sign says the same
    void* dz;                         // dense [M, N] or NULL (act none: dz is dy)
    float* part;                      // [gridDim.x][N] or NULL
    long long M; int N;
    int act; float act_param;
    int tx;
};

template <typename T, int V>
__global__ __launch_bounds__(256) void linear_dz_kernel(DzArgs p) {
    __shared__ float red[256 * V];
    const int tx = threadIdx.x & (p.tx - 1), ty = threadIdx.x / p.tx, ny = 256 / p.tx;
    const int c = ((int)blockIdx.y * p.tx + tx) * V;
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.f;
    if (c < p.N) {
        for (long long m = (long long)blockIdx.x * ny + ty; m < p.M; m += (long long)gridDim.x * ny) {
            float g[V];
            load_vec<V>((const T*)p.dy + m * p.lddy + c, g);
            if (p.dz) {
                float z[V];
                load_vec<V>((const T*)p.saved + m * p.N + c, z);
#pragma unroll
                for (int j = 0; j < V; ++j) g[j] *= row_act_slope<sizeof(T) == 2>(z[j], p.act, p.act_param);
                store_vec<V>((T*)p.dz + m * p.N + c, g);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += g[j];
        }
    }
    if (!p.part) return;
#pragma unroll
    for (int j = 0; j < V; ++j) red[threadIdx.x * V + j] = sum[j];
    __syncthreads();
    if (ty == 0 && c < p.N) {
        for (int q = 1; q < ny; ++q)
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += red[(q * p.tx + tx) * V + j];
#pragma unroll
        for (int j = 0; j < V; ++j) p.part[(size_t)blockIdx.x * p.N + c + j] = sum[j];
    }
}

static int dz_slots(long long M) { return (int)(M < 8 ? 1 : M / 8 > 256 ? 256 : M / 8); }

template <typename T>
static int dz_launch(DzArgs& p, hipStream_t s) {
    if (p.N == 0) return SRMI_OK;
    constexpr int V = 16 / (int)sizeof(T);
    const bool vec = (((uintptr_t)p.dy | (uintptr_t)p.saved | (uintptr_t)p.dz) & 15) == 0 && p.N % V == 0 && p.lddy % V == 0;
    const int v = vec ? V : 1;
    p.tx = 1;
    while (p.tx < 256 && p.tx * v < p.N) p.tx *= 2;
    const dim3 grid(dz_slots(p.M), (p.N + p.tx * v - 1) / (p.tx * v));
    if (vec) hipLaunchKernelGGL((linear_dz_kernel<T, V>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((linear_dz_kernel<T, 1>), grid, dim3(256), 0, s, p);
    return hip_check(hipGetLastError(), "linear dz");
}

// ---- entry points' bodies ---------------------------------------------------------------------------------------------
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t linear_workspace_bytes(const srmi_linear_desc& d, int pass) {
    if (pass == SRMI_PASS_FWD) return 0;
    const size_t esz = d.dtype == SRMI_BF16 ? 2 : 4;
    size_t n = up256((size_t)dz_slots(d.M) * d.N * sizeof(float));
    if (d.act != SRMI_ACT_NONE) n += up256((size_t)d.M * d.N * esz);
    return n;
}

template <typename T>
static int linear_fwd_t(const srmi_linear_desc& d, const void* x, const void* w, const void* bias, const void* residual, void* y, void* z,
                        hipStream_t s) {
    GemmArgs p;
    p.a = x; p.sar = d.ldx; p.sak = 1;
    p.b = w; p.sbr = d.ldw; p.sbk = 1;
    p.M = d.M; p.N = d.N; p.K = d.K;
    p.bias = bias; p.residual = residual; p.ldr = d.ldr; p.y = y; p.ldy = d.N; p.z = z;
    p.act = d.act; p.act_param = d.act_param;
    return gemm<T>(p, s);
}

int linear_fwd(const srmi_linear_desc& d, const void* x, const void* w, const void* bias, const void* residual, void* y, void* z, void* ws,
               hipStream_t s) {
    (void)ws;
    return d.dtype == SRMI_BF16 ? linear_fwd_t<bf16_t>(d, x, w, bias, residual, y, z, s)
                                : linear_fwd_t<float>(d, x, w, bias, residual, y, z, s);
}

template <typename T>
static int linear_bwd_t(const srmi_linear_desc& d, const void* x, const void* w, const void* saved, const void* dy, void* dx, void* dw,
                        void* db, char* ws, hipStream_t s) {
    float* part = (float*)ws;
    ws += up256((size_t)dz_slots(d.M) * d.N * sizeof(float));
    const void* dz = dy;
    long long lddz = d.lddy;
    int rc = SRMI_OK;
    const bool act = d.act != SRMI_ACT_NONE;
    if (db || (act && d.M > 0)) {
        DzArgs q;
        q.dy = dy; q.lddy = d.lddy; q.saved = saved; q.dz = act ? ws : nullptr; q.part = db ? part : nullptr;
        q.M = d.M; q.N = d.N; q.act = d.act; q.act_param = d.act_param;
        if ((rc = dz_launch<T>(q, s))) return rc;
        if (db && (rc = slot_sum_launch(part, dz_slots(d.M), d.N, d.N, db, nullptr, sizeof(T) == 2, s))) return rc;
        if (act) { dz = ws; lddz = d.N; }
    }
    GemmArgs p = {};
    p.act = SRMI_ACT_NONE;
    if (dx) {
        p.a = dz; p.sar = lddz; p.sak = 1;
        p.b = w; p.sbr = 1; p.sbk = d.ldw;
        p.M = d.M; p.N = d.K; p.K = d.N;
        p.y = dx; p.ldy = d.K;
        if ((rc = gemm<T>(p, s))) return rc;
    }
    if (dw) {
        p.a = dz; p.sar = 1; p.sak = lddz;
        p.b = x; p.sbr = 1; p.sbk = d.ldx;
        p.M = d.N; p.N = d.K; p.K = d.M;
        p.y = dw; p.ldy = d.K;
        if ((rc = gemm<T>(p, s))) return rc;
    }
    return SRMI_OK;
}

int linear_bwd(const srmi_linear_desc& d, const void* x, const void* w, const void* saved, const void* dy, void* dx, void* dw, void* db,
               void* ws, hipStream_t s) {
    return d.dtype == SRMI_BF16 ? linear_bwd_t<bf16_t>(d, x, w, saved, dy, dx, dw, db, (char*)ws, s)
                                : linear_bwd_t<float>(d, x, w, saved, dy, dx, dw, db, (char*)ws, s);
}

}  // namespace srmi
