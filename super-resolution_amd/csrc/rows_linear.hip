// Linear layers on rows: y = act(x w^T + b) + residual, and the backward pass.
//
//   z = x w^T + b          [M, N] = [M, K] [N, K]^T
//   dz = dy act'(z)        db = sum_m dz
//   dx = dz w              [M, K] = [M, N] [N, K]
//   dw = dz^T x            [N, K] = [M, N]^T [M, K]
//
// All three are tile products: bf16 operands whose rows lie on 16-byte boundaries take gemm_tile_kernel, f32 ones and others
// gemm_staged_kernel (rows_gemm.h).  Few rows take the products of rows_thin.h.  Nothing is re-laid out in memory.
#include "rows_thin.h"

namespace srmi {

int slot_sum_launch(const float* part, int slots, int n, int n0, void* o0, void* o1, int out_bf16, hipStream_t s);

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static int up8(int n) { return (n + 7) & ~7; }

// ---- the tile product: shape -> kernel, tile, split --------------------------------------------------------------------------
enum TileKind { TILE_256, TILE_128, TILE_128_SHORT, TILE_32, STAGED_128, STAGED_64 };
struct TilePlan { TileKind kind; int bm; long long tiles_m; int tiles_n, splits; size_t part_bytes; };

// direct: both operands can be read by the DMA
static TilePlan tile_plan(bool direct, long long M, int N, long long K) {
    TilePlan t;
    auto tiles = [&](int bm, int bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
    const long long steps = (K + (direct ? 64 : SK) - 1) / (direct ? 64 : SK);
    // bf16 by the length of K, in steps of 64.  256 x 256 tiles, one workgroup per CU, if they fill the chip: 1280-1380 TFLOP/s at 4096^3
    // and 8192^3, where 128 x 128 reach 1070 (4864 x 4096 x 4096, 304 tiles: 177 us against 170; 6400, 400 tiles: 183 against 214).
    // 128 x 128 with 32 k per stage keep four workgroups per CU and hide a short K's prologue and epilogue behind each other: 36864 x
    // 256 -> 1024 in 36 us against 41 with 64 k per stage (two workgroups); those win from K = 2048 on (4096^3: 128 against 187 us).
    if (direct) t.kind = M <= 32 ? TILE_32 : steps >= 8 && tiles(256, 256) >= 200 ? TILE_256 : steps >= 32 ? TILE_128 : TILE_128_SHORT;
    // the larger tile needs half the LDS traffic (190 against 120 TFLOP/s in f32), if it leaves every CU two workgroups of eight steps
    else t.kind = M >= 8 && N >= 8 && tiles(128, 128) * (steps < 8 ? 1 : steps / 8) >= 512 ? STAGED_128 : STAGED_64;
    const int bm = t.bm = t.kind == TILE_256 ? 256 : t.kind == TILE_32 ? 32 : t.kind == STAGED_64 ? 64 : 128;
    const int bn = t.kind == TILE_256 ? 256 : t.kind == STAGED_64 ? 64 : 128;
    t.tiles_m = (M + bm - 1) / bm;
    t.tiles_n = (N + bn - 1) / bn;
    t.splits = 1;
    const long long n = t.tiles_m * t.tiles_n;
    // split K where the tiles leave CUs without work, into as many workgroups as are resident (two per CU, three of the small tiles; one
    // of 256 x 256, which are chosen only where they fill the chip)
    if (t.kind != TILE_256 && n > 0 && n <= (t.kind == STAGED_64 ? 384 : 256)) {
        const long long s = (t.kind == STAGED_64 ? 768 : 512) / n, most = steps / (t.kind == STAGED_128 ? 8 : 4);
        t.splits = (int)(s < most ? (s < 128 ? s : 128) : most);
        if (t.splits < 1) t.splits = 1;
    }
    t.part_bytes = t.splits > 1 ? up256((size_t)t.splits * M * up8(N) * sizeof(float)) : 0;
    return t;
}

template <typename T>
static bool stream_past(long long rows, long long cols) { return (size_t)rows * cols * sizeof(T) > STREAM_BYTES; }

template <typename T>
static int join(const TileArgs& p, const SlotSum& other, hipStream_t s) {
    const long long n8 = p.M * (p.part_ld / 8);
    const bool wide = p.splits >= 8;
    const long long g = wide ? (n8 + 31) / 32 : (n8 + 255) / 256;
    const unsigned blocks = (unsigned)(g > 4096 ? 4096 : g);
    const dim3 grid(blocks + (other.part ? (other.n + 15) / 16 : 0));
    if (wide) hipLaunchKernelGGL((gemm_join_kernel<T, 8>), grid, dim3(256), 0, s, p, blocks, other);
    else hipLaunchKernelGGL((gemm_join_kernel<T, 1>), grid, dim3(256), 0, s, p, blocks, other);
    return hip_check(hipGetLastError(), "linear join");
}
static int slot_sum(const SlotSum& q, int out_bf16, hipStream_t s) {
    return q.part ? slot_sum_launch(q.part, q.slots, q.n, q.n, q.out, nullptr, out_bf16, s) : SRMI_OK;
}

template <int BM, int BN, int WM, int WN, int GK, int NSTAGE, bool PIPE, bool AT, bool BT, typename T>
static void tile_go(const TileArgs& p, unsigned grid, hipStream_t s) {
    constexpr size_t stages = (size_t)NSTAGE * (BM + BN) * GK * 2, ep = epilogue_bytes(WM * WN, BN / WN), lds = stages > ep ? stages : ep;
    if constexpr (BM < 256) {
        if (p.splits > 1) {
            hipLaunchKernelGGL((gemm_tile_kernel<BM, BN, WM, WN, AT, BT, GK, NSTAGE, PIPE, T, true>), dim3(grid), dim3(64 * WM * WN), lds, s, p);
            return;
        }
    }
    hipLaunchKernelGGL((gemm_tile_kernel<BM, BN, WM, WN, AT, BT, GK, NSTAGE, PIPE, T, false>), dim3(grid), dim3(64 * WM * WN), lds, s, p);
}
template <int B, bool AT, bool BT, bool NARROW, typename T>
static void staged_go(const TileArgs& p, unsigned grid, hipStream_t s) {
    if (p.splits > 1) hipLaunchKernelGGL((gemm_staged_kernel<B, AT, BT, NARROW, T, true>), dim3(grid), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((gemm_staged_kernel<B, AT, BT, NARROW, T, false>), dim3(grid), dim3(256), 0, s, p);
}

// the product's launch for the rows that `p` names
template <bool AT, bool BT, typename T>
static int tile_launch(const TilePlan& t, const TileArgs& p, hipStream_t s) {
    const unsigned g = (unsigned)p.tiles_m * p.tiles_n * p.splits;
    if constexpr (sizeof(T) == 2) {
        switch (t.kind) {
            case TILE_256: tile_go<256, 256, 2, 4, 64, 2, true, AT, BT, T>(p, g, s); break;
            case TILE_128: tile_go<128, 128, 2, 2, 64, 2, true, AT, BT, T>(p, g, s); break;
            case TILE_128_SHORT: tile_go<128, 128, 2, 2, 32, 2, false, AT, BT, T>(p, g, s); break;
            case TILE_32: tile_go<32, 128, 1, 4, 64, 3, true, AT, BT, T>(p, g, s); break;
            default: break;
        }
    }
    const bool narrow = (AT && p.M < 8) || (BT && p.N < 8);
    if (t.kind == STAGED_128) staged_go<128, AT, BT, false, T>(p, g, s);
    else if (t.kind == STAGED_64 && !narrow) staged_go<64, AT, BT, false, T>(p, g, s);
    else if constexpr (AT || BT) {
        if (t.kind == STAGED_64) staged_go<64, AT, BT, true, T>(p, g, s);
    }
    return hip_check(hipGetLastError(), "linear product");
}

// A launch has fewer than 2^32 threads, of which a workgroup has 512 at most.
constexpr long long LAUNCH_GROUPS = 0xffffffffll / 512;

// other: partial rows that are to be added as well, by the join if there is one
template <bool AT, bool BT, typename T>
static int tile_gemm(bool direct, TileArgs& p, float* part, hipStream_t s, const SlotSum& other = {}) {
    if (p.M == 0 || p.N == 0) return slot_sum(other, sizeof(T) == 2, s);
    const TilePlan t = tile_plan(direct, p.M, p.N, p.K);
    p.tiles_n = t.tiles_n; p.splits = t.splits;
    p.part = part; p.part_ld = up8(p.N);
    p.past = stream_past<T>(p.M, p.N);
    // more tiles than a launch may have workgroups (they are not split then): runs of whole tile rows, one launch each
    const long long most = LAUNCH_GROUPS / ((long long)t.tiles_n * t.splits), per = t.tiles_m < most ? t.tiles_m : most;
    int rc = SRMI_OK;
    for (long long t0 = 0; t0 < t.tiles_m && !rc; t0 += per) {
        const long long m0 = t0 * t.bm, left = p.M - m0;
        TileArgs q = p;
        q.tiles_m = (int)(t.tiles_m - t0 < per ? t.tiles_m - t0 : per);
        if (per < t.tiles_m) {
            q.M = left < per * t.bm ? left : per * t.bm;
            q.a = (const T*)p.a + (AT ? m0 : m0 * p.lda);
            q.y = (T*)p.y + m0 * p.ldy;
            if (p.z) q.z = (typename KeptZ<T>::type*)p.z + m0 * p.N;
            if (p.residual) q.residual = (const T*)p.residual + m0 * p.ldr;
        }
        rc = tile_launch<AT, BT, T>(t, q, s);
    }
    return rc ? rc : t.splits == 1 ? slot_sum(other, sizeof(T) == 2, s) : join<T>(p, other, s);
}

// ---- few rows ----------------------------------------------------------------------------------------------------------------
// Forward: where the call then is one launch (bf16, 24 x 1024 -> 4096: 5.4 us against 4.6 + 4.5 of a split tile product and its join;
// 48 x 1024 -> 1024: 6.6 against 5.5 + 4.0; f32, 24 x 333 -> 515: 5.9 against 7.5 + 3.4, but 48 x 1024 -> 1024 13.3 against 6.0 + 4.1),
// and for one tile of rows where the operands do not take the DMA (f32, 16 x 18432 -> 1024: 22 + 4 us against 30 + 5; with
// the DMA, bf16: 11.8 + 4.1 against 10.0 + 5.1; f32, 32 x 4096 -> 4096: 31 + 4 against 26 + 4).
// f32 backward of one tile of rows: dx and dw of 16 x 18432 -> 1024 20 + 20 us against 39 + 28 of the tile products; of 32 x 4096 ->
// 4096 51 + 24 against 31 + 25.
constexpr int THIN_ROWS = 16;
static bool thin_short(int K) { return K <= 2048; }       // four chunks of 64 for each of a workgroup's eight waves
static bool thin_bwd(const srmi_linear_desc& d) { return d.M <= THIN_ROWS && d.dtype == SRMI_F32; }

// splits of k otherwise: as many as give two workgroups per CU without leaving a wave without work
static int thin_splits(int N, int K) {
    const int tiles = (N + 15) / 16, chunks = (K + 63) / 64;
    if (thin_short(K) || tiles == 0) return 1;
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
    p.t.past = stream_past<T>(d.M, d.N);
    p.t.tiles_n = (d.N + 15) / 16;
    p.t.splits = thin_splits(d.N, d.K);
    p.t.part = part; p.t.part_ld = up8(d.N);
    p.x = x; p.ldx = d.ldx; p.w = w; p.ldw = d.ldw;
    const dim3 grid((unsigned)(p.t.tiles_n * p.t.splits)), block(64 * THIN_WAVES);
    if (d.M <= 16) hipLaunchKernelGGL((thin_fwd_kernel<T, 1>), grid, block, 0, s, p);
    else if (d.M <= 32) hipLaunchKernelGGL((thin_fwd_kernel<T, 2>), grid, block, 0, s, p);
    else if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((thin_fwd_kernel<T, 4>), grid, block, 0, s, p);
    const int rc = hip_check(hipGetLastError(), "linear fwd");
    return rc || p.t.splits == 1 ? rc : join<T>(p.t, SlotSum{}, s);
}

// dx and dw of f32 layers; dz: f32 rows
static int thin_bwd_go(const srmi_linear_desc& d, const float* dz, long long lddz, const void* x, const void* w, void* dx, void* dw, hipStream_t s) {
    ThinArgs p = {};
    p.x = dz; p.ldx = lddz; p.w = w; p.ldw = d.ldw;
    if (dx && d.M > 0 && d.K > 0) {
        p.t.M = d.M; p.t.N = d.K; p.t.K = d.N; p.t.y = dx; p.t.ldy = d.K;
        hipLaunchKernelGGL(thin_dgrad_kernel, dim3((d.K + 63) / 64), dim3(64 * THIN_WAVES), 0, s, p);
    }
    if (dw && d.N > 0 && d.K > 0) {
        p.t.M = d.N; p.t.N = d.K; p.t.K = d.M; p.t.y = dw; p.t.ldy = d.K;
        hipLaunchKernelGGL(thin_wgrad_kernel, dim3((unsigned)((d.K + 255) / 256) * ((d.N + 63) / 64)), dim3(256), 0, s, p, (const float*)x, (long long)d.ldx);
    }
    return hip_check(hipGetLastError(), "linear bwd");
}

// rows the DMA can read: 16-byte aligned, whole chunks (zeros behind the last column count as columns)
static bool dma_rows(const srmi_linear_desc& d, int cols, long long ld) {
    return d.dtype == SRMI_BF16 && d.align >= 16 && cols % 8 == 0 && ld % 8 == 0 && ld <= GEMM_MAX_LD;
}

// ---- dz = dy * act'(saved) and the partial column sums of dz -----------------------------------------------------------------
// Workgroup (slot of rows, strip of columns): tx lanes of 8 columns, 256 / tx rows at a time; the sums of a workgroup's rows
// are added in LDS and stored as one partial row; slot_sum_block (or a launch of its own) adds the partial rows in index order.  db sums the f32
// products, before dz is rounded to bf16 (the matrix cores' operand type: half a step of 2^-8 per term of dx and dw, as in y itself).
struct DzArgs {
    const void* dy; long long lddy;
    const void* saved;                // dense [M, N]: KeptZ<T> z, or y where its sign says the same; NULL: act'(z) = 1
    void* dz; int ldz;                // [M, ldz], zeros behind column N; NULL: only the sums are wanted
    float* part; void* db;            // partial rows [gridDim.x][N], or the sums themselves (one workgroup per strip); both NULL: not wanted
    long long M; int N;
    int act; float act_param;
    int tx;
    bool past;                        // dz goes past the caches
};

template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(DzArgs p) {
    __shared__ float red[256 * 8];
    const int tx = threadIdx.x & (p.tx - 1), ty = threadIdx.x / p.tx, ny = 256 / p.tx;
    const int c = ((int)blockIdx.y * p.tx + tx) * 8;
    float sum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] = 0.f;
    const bool whole = c + 8 <= p.N, kink = is_kink(p.act);
    if (c < p.N) {
        for (long long m = (long long)blockIdx.x * ny + ty; m < p.M; m += (long long)gridDim.x * ny) {
            typedef typename KeptZ<T>::type Z;
            const T* dy = (const T*)p.dy + m * p.lddy + c;
            const Z* sv = p.saved ? (const Z*)p.saved + m * p.N + c : nullptr;
            Raw8<T> rg;
            Raw8<Z> rz;
            if (whole) {
                rg.load(dy);
                if (sv) rz.load(sv);
            }
            float g[8];
            if (whole) rg.get(g);
            else load_some<8>(dy, p.N - c, g);
            if (sv) {
                float z[8];
                if (sizeof(T) == 2 && kink) {
                    // y (bf16) or z (half) may have been kept: sign bit and zero are the same in both
                    short h[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[j] = whole ? (short)(rz.q[0][j / 2] >> (16 * (j & 1))) : ((const short*)sv)[min(j, p.N - c - 1)];
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[j] = (h[j] & 0x7fff) == 0 ? 0.f : h[j] < 0 ? -1.f : 1.f;
                } else if (whole) {
                    rz.get(z);
                } else {
                    load_some<8>(sv, p.N - c, z);
                }
                row_slope_vec<8, sizeof(T) == 2>(g, z, p.act, p.act_param);
            }
            if (p.dz) store_vec<8>((T*)p.dz + m * p.ldz + c, g, p.past);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += g[j];
        }
    }
    if (!p.part && !p.db) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) red[threadIdx.x * 8 + j] = sum[j];
    __syncthreads();
    if (ty == 0 && c < p.N) {
        for (int q = 1; q < ny; ++q)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += red[(q * p.tx + tx) * 8 + j];
        if (p.db) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < p.N) ((T*)p.db)[c + j] = from_f32<T>(sum[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < p.N) p.part[(size_t)blockIdx.x * p.N + c + j] = sum[j];
        }
    }
}

// lanes of 8 columns per row (a power of two), and workgroups of rows = partial rows of db.  One per pass up to eight workgroups per CU
// (36864 x 1024 gelu, 226 MB: 148 us with 256 workgroups, 43 with 1024); up to 128 rows one workgroup walks them all, 32 at a time, and
// no second launch adds anything.
static int dz_tx(long long M, int N) {
    int tx = 1;
    while (tx < (M <= 128 ? 8 : 256) && tx * 8 < N) tx *= 2;
    return tx;
}
static int dz_slots(long long M, int N) {
    if (M <= 128) return 1;
    const int tx = dz_tx(M, N), strips = N / (tx * 8) + 1;
    const long long want = (M + 256 / tx - 1) / (256 / tx), most = 2048 / strips < 64 ? 64 : 2048 / strips;
    return (int)(want < 1 ? 1 : want > most ? most : want);
}

template <typename T>
static int dz_launch(DzArgs& p, hipStream_t s) {
    if (p.N == 0) return SRMI_OK;
    p.tx = dz_tx(p.M, p.N);
    p.past = stream_past<T>(p.M, p.ldz);
    const dim3 grid(dz_slots(p.M, p.N), (p.N + p.tx * 8 - 1) / (p.tx * 8));
    hipLaunchKernelGGL((linear_dz_kernel<T>), grid, dim3(256), 0, s, p);
    return hip_check(hipGetLastError(), "linear dz");
}

// ---- entry points' bodies ---------------------------------------------------------------------------------------------------
static bool own_dz(const srmi_linear_desc& d) { return d.act != SRMI_ACT_NONE; }
static bool dma_fwd(const srmi_linear_desc& d) { return dma_rows(d, d.K, d.ldx) && dma_rows(d, d.K, d.ldw); }
static bool thin_fwd(const srmi_linear_desc& d) {
    return thin_short(d.K) ? d.M <= (d.dtype == SRMI_BF16 ? 64 : 32) : d.M <= THIN_ROWS && !dma_fwd(d);
}
static bool dma_dz(const srmi_linear_desc& d) { return own_dz(d) ? d.dtype == SRMI_BF16 : dma_rows(d, d.N, d.lddy); }
static bool dma_dx(const srmi_linear_desc& d) { return dma_dz(d) && dma_rows(d, d.K, d.ldw); }
static bool dma_dw(const srmi_linear_desc& d) { return dma_dz(d) && dma_rows(d, d.K, d.ldx); }
static size_t db_bytes(const srmi_linear_desc& d) { return up256((size_t)dz_slots(d.M, d.N) * d.N * sizeof(float)); }
static size_t dz_bytes(const srmi_linear_desc& d) { return own_dz(d) ? up256((size_t)d.M * up8(d.N) * (d.dtype == SRMI_BF16 ? 2 : 4)) : 0; }

// backward: [partial db][dz][split sums of dx, then of dw]
size_t linear_workspace_bytes(const srmi_linear_desc& d, int pass) {
    if (pass == SRMI_PASS_FWD) return thin_fwd(d) ? thin_part_bytes(d) : tile_plan(dma_fwd(d), d.M, d.N, d.K).part_bytes;
    const size_t n = db_bytes(d) + dz_bytes(d);
    if (thin_bwd(d)) return n;
    const size_t px = tile_plan(dma_dx(d), d.M, d.K, d.N).part_bytes, pw = tile_plan(dma_dw(d), d.N, d.K, d.M).part_bytes;
    return n + (px > pw ? px : pw);
}

template <typename T>
static int linear_fwd_t(const srmi_linear_desc& d, const void* x, const void* w, const void* bias, const void* residual, void* y, void* z,
                        float* ws, hipStream_t s) {
    TileArgs p = {};
    p.M = d.M; p.N = d.N; p.K = d.K;
    p.bias = bias; p.residual = residual; p.ldr = d.ldr; p.y = y; p.ldy = d.N; p.z = z;
    p.act = d.act; p.act_param = d.act_param;
    if (thin_fwd(d)) return thin_fwd_go<T>(d, x, w, p, ws, s);
    p.a = x; p.lda = d.ldx;
    p.b = w; p.ldb = d.ldw;
    return tile_gemm<false, false, T>(dma_fwd(d), p, ws, s);
}

int linear_fwd(const srmi_linear_desc& d, const void* x, const void* w, const void* bias, const void* residual, void* y, void* z, void* ws,
               hipStream_t s) {
    return d.dtype == SRMI_BF16 ? linear_fwd_t<bf16_t>(d, x, w, bias, residual, y, z, (float*)ws, s)
                                : linear_fwd_t<float>(d, x, w, bias, residual, y, z, (float*)ws, s);
}

template <typename T>
static int linear_bwd_t(const srmi_linear_desc& d, const void* x, const void* w, const void* saved, const void* dy, void* dx, void* dw,
                        void* db, char* ws, hipStream_t s) {
    int rc;
    float* part = (float*)ws;
    const void* dz = dy;
    long long lddz = d.lddy;
    DzArgs q = {};
    if (own_dz(d) && (dx || dw)) {
        dz = q.dz = ws + db_bytes(d);
        lddz = q.ldz = up8(d.N);
    }
    SlotSum sum = {};
    if (db || (q.dz && d.M > 0)) {
        q.dy = dy; q.lddy = d.lddy; q.saved = own_dz(d) ? saved : nullptr;
        const int slots = dz_slots(d.M, d.N);
        q.part = db && slots > 1 ? part : nullptr;
        q.db = db && slots == 1 ? db : nullptr;
        q.M = d.M; q.N = d.N; q.act = d.act; q.act_param = d.act_param;
        if ((rc = dz_launch<T>(q, s))) return rc;
        if (q.part) sum = {part, slots, d.N, db};
    }
    if (thin_bwd(d)) return thin_bwd_go(d, (const float*)dz, lddz, x, w, dx, dw, s);
    part = (float*)(ws + db_bytes(d) + dz_bytes(d));
    TileArgs p = {};
    p.act = SRMI_ACT_NONE;
    p.a = dz; p.lda = lddz;
    if (dx) {
        p.b = w; p.ldb = d.ldw;
        p.M = d.M; p.N = d.K; p.K = d.N;
        p.y = dx; p.ldy = d.K;
        if ((rc = tile_gemm<false, true, T>(dma_dx(d), p, part, s))) return rc;
    }
    if (dw) {
        p.b = x; p.ldb = d.ldx;
        p.M = d.N; p.N = d.K; p.K = d.M;
        p.y = dw; p.ldy = d.K;
        return tile_gemm<true, true, T>(dma_dw(d), p, part, s, sum);
    }
    return slot_sum(sum, sizeof(T) == 2, s);
}

int linear_bwd(const srmi_linear_desc& d, const void* x, const void* w, const void* saved, const void* dy, void* dx, void* dw, void* db,
               void* ws, hipStream_t s) {
    return d.dtype == SRMI_BF16 ? linear_bwd_t<bf16_t>(d, x, w, saved, dy, dx, dw, db, (char*)ws, s)
                                : linear_bwd_t<float>(d, x, w, saved, dy, dx, dw, db, (char*)ws, s);
}

bool linear_too_wide(const srmi_linear_desc& d) { return d.N > GEMM_MAX_LD || d.K > GEMM_MAX_LD; }

}  // namespace srmi
