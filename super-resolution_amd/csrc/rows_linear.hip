// Linear layers on rows: y = act(x w^T + b) + residual, and the backward pass.
//
//   z = x w^T + b          [M, N] = [M, K] [N, K]^T
//   dz = dy act'(z)        db = sum_m dz
//   dx = dz w              [M, K] = [M, N] [N, K]
//   dw = dz^T x            [N, K] = [M, N]^T [M, K]
//
// All three are the tile product of rows_gemm.h.  bf16 operands whose rows lie on 16-byte boundaries are read in place; others, and f32
// operands (as three bf16 planes), are first laid out in the workspace: one pass over M K + N K elements in front of M N K
// multiplications.  Few rows take the products of rows_thin.h, which read every operand once, in place, whatever its alignment.
#include "rows_thin.h"

namespace srmi {

int slot_sum_launch(const float* part, int slots, int n, int n0, void* o0, void* o1, int out_bf16, hipStream_t s);

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static int up8(int n) { return (n + 7) & ~7; }

// ---- the tile product: shape -> tile, split ------------------------------------------------------------------------------
enum { TILE_256 = 0, TILE_128 = 1, TILE_32 = 2 };
struct TilePlan { int kind, bm, bn, tiles_m, tiles_n, splits; size_t part_bytes; };

static TilePlan tile_plan(long long M, int N, long long K, int terms) {
    TilePlan t;
    const long long steps = terms * ((K + GK - 1) / GK);
    const long long tiles256 = ((M + 255) / 256) * ((N + 255) / 256);
    t.kind = M <= 32 ? TILE_32 : tiles256 >= 200 && steps >= 8 ? TILE_256 : TILE_128;
#ifdef FORCE_KIND
    if (M > 32) t.kind = FORCE_KIND;
#endif
    t.bm = t.kind == TILE_256 ? 256 : t.kind == TILE_128 ? 128 : 32;
    t.bn = t.kind == TILE_256 ? 256 : 128;
    const long long tm = (M + t.bm - 1) / t.bm, tn = (N + t.bn - 1) / t.bn, tiles = tm * tn;
    t.tiles_m = (int)(tm > 0x7fffffff ? 0x7fffffff : tm);
    t.tiles_n = (int)tn;
    t.splits = 1;
    if (tiles < 256) {
        long long s = 512 / (tiles ? tiles : 1);
        if (s > steps / 4) s = steps / 4;
        t.splits = (int)(s < 1 ? 1 : s > 128 ? 128 : s);
    }
    t.part_bytes = t.splits > 1 ? up256((size_t)t.splits * M * up8(N) * sizeof(float)) : 0;
    return t;
}

template <typename T>
static int join(const TileArgs& p, hipStream_t s) {
    const long long n8 = p.M * (p.part_ld / 8);
    const bool wide = p.splits >= 8;
    const long long g = wide ? (n8 + 31) / 32 : (n8 + 255) / 256;
    const dim3 grid((unsigned)(g > 4096 ? 4096 : g));
    if (wide) hipLaunchKernelGGL((gemm_join_kernel<T, 8>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((gemm_join_kernel<T, 1>), grid, dim3(256), 0, s, p);
    return hip_check(hipGetLastError(), "linear join");
}

template <int BM, int BN, int WM, int WN, int NSTAGE, bool PIPE, bool AT, bool BT, typename T>
static int tile_go(const TileArgs& p, hipStream_t s) {
    const dim3 grid((unsigned)((long long)p.tiles_m * p.tiles_n * p.splits)), block(64 * WM * WN);
    constexpr size_t lds = (size_t)NSTAGE * (BM + BN) * GK * 2;
    if (p.splits > 1) {
        hipLaunchKernelGGL((gemm_tile_kernel<BM, BN, WM, WN, AT, BT, NSTAGE, PIPE, T, true>), grid, block, lds, s, p);
        return join<T>(p, s);
    } else {
        hipLaunchKernelGGL((gemm_tile_kernel<BM, BN, WM, WN, AT, BT, NSTAGE, PIPE, T, false>), grid, block, lds, s, p);
    }
    return hip_check(hipGetLastError(), "linear product");
}

template <bool AT, bool BT, typename T>
static int tile_gemm(TileArgs& p, float* part, hipStream_t s) {
    if (p.M == 0 || p.N == 0) return SRMI_OK;
    const TilePlan t = tile_plan(p.M, p.N, p.K, p.terms);
    if ((long long)t.tiles_m * t.tiles_n * t.splits > 0x7fffffff) { set_error("linear: more than 2^31 tiles"); return SRMI_EUNSUPPORTED; }
    p.tiles_m = t.tiles_m; p.tiles_n = t.tiles_n; p.splits = t.splits;
    p.part = part; p.part_ld = up8(p.N);
    switch (t.kind) {
        case TILE_256: return tile_go<256, 256, 2, 4, 2, true, AT, BT, T>(p, s);
        case TILE_128: return tile_go<128, 128, 2, 2, 2, false, AT, BT, T>(p, s);
        default: return tile_go<32, 128, 1, 4, 3, true, AT, BT, T>(p, s);
    }
}

// ---- few rows ----------------------------------------------------------------------------------------------------------------
constexpr int THIN_ROWS = 64;
static bool thin_fwd(const srmi_linear_desc& d) { return d.M <= THIN_ROWS; }
static bool thin_bwd(const srmi_linear_desc& d) { return d.M <= THIN_ROWS && d.dtype == SRMI_F32; }

// splits of k: one if a workgroup's eight waves have no more than four chunks of 64 each (then the call is one launch), else as many as
// give two workgroups per CU without leaving a wave without work
static int thin_splits(int N, int K) {
    const int tiles = (N + 15) / 16, chunks = (K + 63) / 64;
    if (chunks <= 32 || tiles == 0) return 1;
    const int s = 512 / tiles, most = chunks / 8;
    return s < 1 ? 1 : s < most ? s : most;
}
static size_t thin_part_bytes(const srmi_linear_desc& d) {
    const int s = thin_splits(d.N, d.K);
    return s > 1 ? up256((size_t)s * d.M * up8(d.N) * sizeof(float)) : 0;
}

template <typename T>
static int thin_fwd_go(const srmi_linear_desc& d, const void* x, const void* w, const TileArgs& t, float* part, hipStream_t s) {
    ThinArgs p;
    p.t = t;
    p.t.tiles_n = (d.N + 15) / 16;
    p.t.splits = thin_splits(d.N, d.K);
    p.t.part = part; p.t.part_ld = up8(d.N);
    p.x = x; p.ldx = d.ldx; p.w = w; p.ldw = d.ldw;
    const dim3 grid((unsigned)(p.t.tiles_n * p.t.splits)), block(64 * THIN_WAVES);
    if (d.M <= 16) hipLaunchKernelGGL((thin_fwd_kernel<T, 1>), grid, block, 0, s, p);
    else if (d.M <= 32) hipLaunchKernelGGL((thin_fwd_kernel<T, 2>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((thin_fwd_kernel<T, 4>), grid, block, 0, s, p);
    const int rc = hip_check(hipGetLastError(), "linear fwd");
    return rc || p.t.splits == 1 ? rc : join<T>(p.t, s);
}

// dx and dw of f32 layers; dz: f32 rows
static int thin_bwd_go(const srmi_linear_desc& d, const float* dz, long long lddz, const void* x, const void* w, void* dx, void* dw, hipStream_t s) {
    ThinArgs p = {};
    p.x = dz; p.ldx = lddz; p.w = w; p.ldw = d.ldw;
    if (dx && d.M > 0 && d.K > 0) {
        p.t.M = d.M; p.t.N = d.K; p.t.K = d.N; p.t.y = dx; p.t.ldy = d.K;
        const dim3 grid((d.K + 63) / 64), block(64 * THIN_WAVES);
        if (d.M <= 16) hipLaunchKernelGGL((thin_dgrad_kernel<1>), grid, block, 0, s, p);
        else if (d.M <= 32) hipLaunchKernelGGL((thin_dgrad_kernel<2>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((thin_dgrad_kernel<4>), grid, block, 0, s, p);
    }
    if (dw && d.N > 0 && d.K > 0) {
        p.t.M = d.N; p.t.N = d.K; p.t.K = d.M; p.t.y = dw; p.t.ldy = d.K;
        hipLaunchKernelGGL(thin_wgrad_kernel, dim3((d.K + 255) / 256, (d.N + 63) / 64), dim3(256), 0, s, p, (const float*)x, (long long)d.ldx);
    }
    return hip_check(hipGetLastError(), "linear bwd");
}

// ---- operands -------------------------------------------------------------------------------------------------------------
struct Operand { const bf16_t* p; long long ld, plane; };

static bool in_place(const srmi_linear_desc& d, int cols, long long ld) {
    return d.dtype == SRMI_BF16 && d.align >= 16 && cols % 8 == 0 && ld % 8 == 0 && ld <= GEMM_MAX_LD;
}
static size_t packed_bytes(const srmi_linear_desc& d, long long rows, int cols) {
    return up256((size_t)rows * up8(cols) * (d.dtype == SRMI_BF16 ? 2 : 6));
}

template <typename T>
static int operand(const srmi_linear_desc& d, const void* src, long long ld, long long rows, int cols, char*& ws, Operand* o, hipStream_t s) {
    if (in_place(d, cols, ld)) { *o = Operand{(const bf16_t*)src, ld, 0}; return SRMI_OK; }
    *o = Operand{(const bf16_t*)ws, up8(cols), rows * up8(cols)};
    ws += packed_bytes(d, rows, cols);
    const long long n = rows * (up8(cols) / 8);
    if (n == 0) return SRMI_OK;
    const long long g = (n + 255) / 256;
    hipLaunchKernelGGL((pack_rows_kernel<T>), dim3((unsigned)(g > 8192 ? 8192 : g)), dim3(256), 0, s, (const T*)src, ld, rows, cols,
                       (bf16_t*)o->p, up8(cols), o->plane);
    return hip_check(hipGetLastError(), "linear operand layout");
}

// ---- dz = dy * act'(saved) in the products' form, and the partial column sums of dz --------------------------------------------
// Workgroup (slot of rows, strip of columns): tx lanes of 8 columns, 256 / tx rows at a time; the sums of a workgroup's rows
// are added in LDS and stored as one partial row, a second launch adds the partial rows in index order.  db sums the f32
// products, before dz is rounded to bf16 (the matrix cores' operand type: half a step of 2^-8 per term of dx and dw, as in y itself).
struct DzArgs {
    const void* dy; long long lddy;
    const void* saved;                // dense [M, N]: z, or y where its sign says the same; NULL: act'(z) = 1
    bf16_t* dz; int ldz; long long plane;      // [M, ldz] planes, zeros behind column N; NULL: only the sums are wanted
    float* dzf;                       // f32 with few rows: dense [M, N] instead
    float* part;                      // [gridDim.x][N] or NULL
    long long M; int N;
    int act; float act_param;
    int tx;
};

template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(DzArgs p) {
    __shared__ float red[256 * 8];
    const int tx = threadIdx.x & (p.tx - 1), ty = threadIdx.x / p.tx, ny = 256 / p.tx;
    const int c = ((int)blockIdx.y * p.tx + tx) * 8;
    float sum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] = 0.f;
    const bool whole = c + 8 <= p.N;
    if (c < p.N) {
        for (long long m = (long long)blockIdx.x * ny + ty; m < p.M; m += (long long)gridDim.x * ny) {
            float g[8];
            const T* dy = (const T*)p.dy + m * p.lddy + c;
            if (whole) load_vec<8>(dy, g);
            else {
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] = c + j < p.N ? to_f32(dy[j]) : 0.f;
            }
            if (p.saved) {
                float z[8];
                const T* sv = (const T*)p.saved + m * p.N + c;
                if (whole) load_vec<8>(sv, z);
                else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[j] = c + j < p.N ? to_f32(sv[j]) : 0.f;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] *= row_act_slope<sizeof(T) == 2>(z[j], p.act, p.act_param);
            }
            if constexpr (sizeof(T) == 4) {
                if (p.dzf) {
                    float* o = p.dzf + m * p.N + c;
                    if (whole) store_vec<8>(o, g);
                    else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (c + j < p.N) o[j] = g[j];
                    }
                }
            }
            if (p.dz) store_planes8<T>(p.dz + m * p.ldz + c, p.plane, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += g[j];
        }
    }
    if (!p.part) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) red[threadIdx.x * 8 + j] = sum[j];
    __syncthreads();
    if (ty == 0 && c < p.N) {
        for (int q = 1; q < ny; ++q)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += red[(q * p.tx + tx) * 8 + j];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < p.N) p.part[(size_t)blockIdx.x * p.N + c + j] = sum[j];
    }
}

static int dz_slots(long long M) { return (int)(M < 8 ? 1 : M / 8 > 256 ? 256 : M / 8); }

template <typename T>
static int dz_launch(DzArgs& p, hipStream_t s) {
    if (p.N == 0) return SRMI_OK;
    p.tx = 1;
    while (p.tx < 256 && p.tx * 8 < p.N) p.tx *= 2;
    const dim3 grid(dz_slots(p.M), (p.N + p.tx * 8 - 1) / (p.tx * 8));
    hipLaunchKernelGGL((linear_dz_kernel<T>), grid, dim3(256), 0, s, p);
    return hip_check(hipGetLastError(), "linear dz");
}

// ---- entry points' bodies ---------------------------------------------------------------------------------------------------
static int terms_of(const srmi_linear_desc& d) { return d.dtype == SRMI_BF16 ? 1 : 6; }
static bool own_dz(const srmi_linear_desc& d) { return d.act != SRMI_ACT_NONE || !in_place(d, d.N, d.lddy); }

size_t linear_workspace_bytes(const srmi_linear_desc& d, int pass) {
    size_t n = 0;
    if (pass == SRMI_PASS_FWD && thin_fwd(d)) return thin_part_bytes(d);
    if (pass == SRMI_PASS_BWD && thin_bwd(d))
        return up256((size_t)dz_slots(d.M) * d.N * sizeof(float)) + (d.act != SRMI_ACT_NONE ? up256((size_t)d.M * d.N * sizeof(float)) : 0);
    if (!in_place(d, d.K, d.ldx)) n += packed_bytes(d, d.M, d.K);
    if (!in_place(d, d.K, d.ldw)) n += packed_bytes(d, d.N, d.K);
    if (pass == SRMI_PASS_FWD) return n + tile_plan(d.M, d.N, d.K, terms_of(d)).part_bytes;
    n += up256((size_t)dz_slots(d.M) * d.N * sizeof(float));
    if (own_dz(d)) n += packed_bytes(d, d.M, d.N);
    const size_t pd = tile_plan(d.M, d.K, d.N, terms_of(d)).part_bytes, pw = tile_plan(d.N, d.K, d.M, terms_of(d)).part_bytes;
    return n + (pd > pw ? pd : pw);
}

template <typename T>
static int linear_fwd_t(const srmi_linear_desc& d, const void* x, const void* w, const void* bias, const void* residual, void* y, void* z,
                        char* ws, hipStream_t s) {
    TileArgs p = {};
    p.M = d.M; p.N = d.N; p.K = d.K; p.terms = terms_of(d);
    p.bias = bias; p.residual = residual; p.ldr = d.ldr; p.y = y; p.ldy = d.N; p.z = z;
    p.act = d.act; p.act_param = d.act_param;
    if (thin_fwd(d)) return thin_fwd_go<T>(d, x, w, p, (float*)ws, s);
    Operand a, b;
    int rc;
    if ((rc = operand<T>(d, x, d.ldx, d.M, d.K, ws, &a, s))) return rc;
    if ((rc = operand<T>(d, w, d.ldw, d.N, d.K, ws, &b, s))) return rc;
    p.a = a.p; p.lda = a.ld; p.pa = a.plane;
    p.b = b.p; p.ldb = b.ld; p.pb = b.plane;
    return tile_gemm<false, false, T>(p, (float*)ws, s);
}

int linear_fwd(const srmi_linear_desc& d, const void* x, const void* w, const void* bias, const void* residual, void* y, void* z, void* ws,
               hipStream_t s) {
    return d.dtype == SRMI_BF16 ? linear_fwd_t<bf16_t>(d, x, w, bias, residual, y, z, (char*)ws, s)
                                : linear_fwd_t<float>(d, x, w, bias, residual, y, z, (char*)ws, s);
}

template <typename T>
static int linear_bwd_t(const srmi_linear_desc& d, const void* x, const void* w, const void* saved, const void* dy, void* dx, void* dw,
                        void* db, char* ws, hipStream_t s) {
    int rc;
    float* part = (float*)ws;
    ws += up256((size_t)dz_slots(d.M) * d.N * sizeof(float));
    Operand dz = {(const bf16_t*)dy, d.lddy, 0}, o;
    const bool thin = thin_bwd(d), own = !thin && own_dz(d) && (dx || dw);
    float* dzf = thin && d.act != SRMI_ACT_NONE && (dx || dw) ? (float*)ws : nullptr;
    if (own) {
        dz = Operand{(const bf16_t*)ws, up8(d.N), d.M * up8(d.N)};
        ws += packed_bytes(d, d.M, d.N);
    }
    if (db || ((own || dzf) && d.M > 0)) {
        DzArgs q = {};
        q.dy = dy; q.lddy = d.lddy; q.saved = d.act != SRMI_ACT_NONE ? saved : nullptr;
        q.dz = own ? (bf16_t*)dz.p : nullptr; q.ldz = up8(d.N); q.plane = dz.plane; q.dzf = dzf;
        q.part = db ? part : nullptr;
        q.M = d.M; q.N = d.N; q.act = d.act; q.act_param = d.act_param;
        if ((rc = dz_launch<T>(q, s))) return rc;
        if (db && (rc = slot_sum_launch(part, dz_slots(d.M), d.N, d.N, db, nullptr, sizeof(T) == 2, s))) return rc;
    }
    if (thin) return thin_bwd_go(d, dzf ? dzf : (const float*)dy, dzf ? d.N : d.lddy, x, w, dx, dw, s);
    TileArgs p = {};
    p.act = SRMI_ACT_NONE;
    p.terms = terms_of(d);
    p.a = dz.p; p.lda = dz.ld; p.pa = dz.plane;
    if (dx) {
        if ((rc = operand<T>(d, w, d.ldw, d.N, d.K, ws, &o, s))) return rc;
        p.b = o.p; p.ldb = o.ld; p.pb = o.plane;
        p.M = d.M; p.N = d.K; p.K = d.N;
        p.y = dx; p.ldy = d.K;
        if ((rc = tile_gemm<false, true, T>(p, (float*)ws, s))) return rc;
    }
    if (dw) {
        if ((rc = operand<T>(d, x, d.ldx, d.M, d.K, ws, &o, s))) return rc;
        p.b = o.p; p.ldb = o.ld; p.pb = o.plane;
        p.M = d.N; p.N = d.K; p.K = d.M;
        p.y = dw; p.ldy = d.K;
        if ((rc = tile_gemm<true, true, T>(p, (float*)ws, s))) return rc;
    }
    return SRMI_OK;
}

int linear_bwd(const srmi_linear_desc& d, const void* x, const void* w, const void* saved, const void* dy, void* dx, void* dw, void* db,
               void* ws, hipStream_t s) {
    return d.dtype == SRMI_BF16 ? linear_bwd_t<bf16_t>(d, x, w, saved, dy, dx, dw, db, (char*)ws, s)
                                : linear_bwd_t<float>(d, x, w, saved, dy, dx, dw, db, (char*)ws, s);
}

bool linear_too_wide(const srmi_linear_desc& d) { return d.N > GEMM_MAX_LD || d.K > GEMM_MAX_LD; }

}  // namespace srmi
