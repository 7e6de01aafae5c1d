// The tile product of the row operators: C[m, n] = sum_k A(m, k) B(n, k), bf16 operands, f32 sums on the matrix cores.
//
// A workgroup owns a BM x BN tile and walks K in steps of GK (64, or 32 where K is short).  Operand tiles go straight from memory to LDS
// (buffer_load_dwordx4 ... lds: no register round trip), up to NSTAGE steps ahead of the step being multiplied, with one barrier
// per step.  An operand may be stored along k ([row][k], like x and w in x w^T) or across it ([k][row], like w in dz w and both
// operands of dz^T x): the second kind is read from LDS with the transposing read (ds_read_b64_tr_b16), so that no operand is ever
// re-laid out in memory.
//
// LDS layouts, both free of bank conflicts:
//   along k    rows of GK / 8 16-byte chunks, chunk c of row r at position c ^ chunk_key(r);
//   across k   one row per k, columns in 32-byte pairs of chunks, pair p of row k at position p ^ ((k & 3) | (k >> 3 & 1) << 2):
//              the eight k rows that half a wave's transposing read touches fall on eight different pairs.
// The DMA writes LDS linearly, so the permutation is applied to the global address of each lane.
// Rows and k past the operand's end are lanes whose buffer offset is out of range: the hardware returns zeros.
//
// Operands this kernel cannot take - f32, or bf16 rows off 16-byte boundaries - go through gemm_staged_kernel: the same tiles and fragments,
// loaded through registers at any alignment.  f32 values are split there into three bf16 (x = hi + mid + lo to 24 bits) and
// multiplied as six products hi hi, hi mid, mid hi, hi lo, mid mid, lo hi: the matrix cores run bf16 sixteen times as fast as f32, the
// dropped products are below 2^-22 of the largest and of either sign.  bf16 has nothing below 2^-133: operands under 2^-110 are taken to the
// nearest multiple of that, instead of to 24 bits.  hi hi has an accumulator of its own, so that a sum over K is
// rounded once per 32 k as an f32 sum would be, not six times.
#pragma once
#include "rows_common.h"

namespace srmi {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
typedef __attribute__((address_space(3))) void* lds_ptr;

constexpr unsigned OUT_OF_RANGE = 0x80000000u;       // buffer offset = the resource's size: reads zeros
constexpr long long GEMM_MAX_LD = 1 << 22;           // a tile's offsets stay below 2^31 bytes

struct TileArgs {
    const void* a; const void* b;                    // rows operand [M, K] and column operand [N, K], stored along or across k
    long long lda, ldb;                              // row strides in elements
    long long M, K; int N;
    int tiles_m, tiles_n, splits;
    float* part; int part_ld;                        // split sums: [splits][M][part_ld]
    // epilogue
    const void* bias; const void* residual; void* y; void* z;
    long long ldr, ldy;                              // z is dense [M, N]
    int act; float act_param;
    bool past;                                       // y and z go past the caches
};

// act(v + bias) + residual for V columns of one row, stored as T; z, where wanted, on the way
template <typename T, int V>
__device__ __forceinline__ void row_epilogue(const TileArgs& p, float* v, const float* bias, long long m, int n) {
    constexpr bool FAST = sizeof(T) == 2;
    float q[V];
    Raw8<T> raw;                                      // of the residual, on its way during the activation
    const T* r = p.residual ? (const T*)p.residual + m * p.ldr + n : nullptr;
    if (V == 8 && r && n + V <= p.N) raw.load(r);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += bias[j];
    if (p.z) {
        auto* z = (typename KeptZ<T>::type*)p.z + m * p.N + n;
        float k[V];
#pragma unroll
        for (int j = 0; j < V; ++j) k[j] = v[j];
        if (sizeof(T) == 2 && is_kink(p.act)) {      // their slope asks whether z > 0, of every z: below the least half a positive one is kept as that
#pragma unroll
            for (int j = 0; j < V; ++j) k[j] = v[j] > 0.f ? fmaxf(v[j], 0x1p-24f) : v[j];
        }
        if (n + V <= p.N) store_vec<V>(z, k, p.past);
        else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (n + j < p.N) store_vec<1>(z + j, k + j);
        }
    }
    row_act_vec<V, FAST>(v, p.act, p.act_param);
    if (r) {
        if (n + V <= p.N) {
            if constexpr (V == 8) raw.get(q);
            else load_vec<V>(r, q);
        } else load_some<V>(r, p.N - n, q);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += q[j];
    }
    T* y = (T*)p.y + m * p.ldy + n;
    if (n + V <= p.N) store_vec<V>(y, v, p.past);
    else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (n + j < p.N) y[j] = from_f32<T>(v[j]);
    }
}

template <typename T, int V>
__device__ __forceinline__ void load_bias(const TileArgs& p, int n, float* bias) {
    const T* b = (const T*)p.bias + n;
    if (p.bias && n + V <= p.N) load_vec<V>(b, bias);
    else if (p.bias && n < p.N) load_some<V>(b, p.N - n, bias);
    else {
#pragma unroll
        for (int j = 0; j < V; ++j) bias[j] = 0.f;
    }
}

// 1 KiB of an operand tile: lane l's 16 bytes go to LDS byte `dst` + 16 l.  (The resource may come from a v_readfirstlane: five
// wait states before the load reads it.)
__device__ __forceinline__ void dma_1k(const u32x4& rsrc, unsigned voff, unsigned dst) {
    unsigned keep;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %3\n\t"
        "s_nop 2\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "v"(voff), "s"(rsrc), "s"(dst)
        : "memory");
}

// resource over [base, base + 2^31): lanes outside their operand use OUT_OF_RANGE
__device__ __forceinline__ u32x4 tile_rsrc(unsigned long long base) {
    return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)base), (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(base >> 32)),
                 OUT_OF_RANGE, 0x00020000u};
}

// along k: the permutation of a row's 16-byte chunks.  The 16 lanes that a ds_read_b128 serves at a time then hit sixteen different
// chunks of the 256 bytes of banks: rows of 128 bytes (64 k) take r mod 8, rows of 64 bytes 0, 2, 3, 1 by r / 4 mod 4.
template <int GK>
__device__ __forceinline__ int chunk_key(int r) {
    if constexpr (GK == 64) return r & 7;
    const int g = r >> 2 & 3;
    return (((g ^ (g >> 1)) & 1) << 1) | (g >> 1);
}

// Staging of one operand: R rows, NW waves, T: stored across k
template <int R, int NW, bool T, int GK>
struct TileLoader {
    static constexpr int UNITS = R * GK / 512 / NW;   // KiB per wave and step
    static constexpr int CPR = R / 8;                 // chunks per k row (T)
    unsigned voff[UNITS];
    int kk[T ? UNITS : 1];                            // k of the lane's chunk inside the step
    const bf16_t* base; long long ld;
    static_assert(R * GK % (512 * NW) == 0, "whole KiB per wave");

    // row0: the tile's first row; rows: rows of the operand
    __device__ __forceinline__ void init(const bf16_t* p, long long ld_, long long row0, long long rows, int wave, int lane) {
        ld = ld_;
        base = T ? p + row0 : p + row0 * ld_;
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int u = i * NW + wave;
            if constexpr (T) {
                const int k = u * (64 / CPR) + lane / CPR, pos = lane % CPR;
                const int pair = (pos >> 1) ^ (((k & 3) | ((k >> 3 & 1) << 2)) & (CPR / 2 - 1));
                const int c = 2 * pair + (pos & 1);
                kk[i] = k;
                voff[i] = row0 + 8 * c < rows ? (unsigned)(k * ld_ * 2 + 16 * c) : OUT_OF_RANGE;
            } else {
                const int r = u * (512 / GK) + lane / (GK / 8), c = (lane % (GK / 8)) ^ chunk_key<GK>(r);
                kk[0] = 8 * c;                       // (the key repeats every unit: one chunk per lane)
                voff[i] = row0 + r < rows ? (unsigned)(r * ld_ * 2 + 16 * c) : OUT_OF_RANGE;
            }
        }
    }
    // address of step `step` (GK k each), and the distance to the next step
    __device__ __forceinline__ unsigned long long at(long long step) const { return (unsigned long long)(uintptr_t)base + 2 * step * GK * (T ? ld : 1); }
    __device__ __forceinline__ unsigned long long stride() const { return 2 * GK * (unsigned long long)(T ? ld : 1); }
    // request the wave's i-th KiB; klim: k of the step that exist, lds: byte address of the tile
    __device__ __forceinline__ void issue(int i, const u32x4& rsrc, int klim, unsigned lds, int wave) const {
        dma_1k(rsrc, kk[T ? i : 0] < klim ? voff[i] : OUT_OF_RANGE, __builtin_amdgcn_readfirstlane(lds + (unsigned)((i * NW + wave) * 1024)));
    }
};

// Fragments of one operand for the wave: NT tiles of 16 rows starting at row w0 (a multiple of 16 NT) of the LDS tile
template <int R, int NT, bool T, int GK>
struct TileReader {
    unsigned addr[T ? NT : GK / 32];
    __device__ __forceinline__ void init(int w0, int lane) {
        const int r = lane & 15, q = lane >> 4;
        if constexpr (T) {
            // lane's address: k row 8 q + (r >> 2), four columns at 4 (r & 3); it receives column r, k = 8 q .. 8 q + 3
            const int f = ((r >> 2) | ((q & 1) << 2)) & (R / 16 - 1);
#pragma unroll
            for (int t = 0; t < NT; ++t) addr[t] = (unsigned)((8 * q + (r >> 2)) * 2 * R + (((w0 / 16 + t) ^ f) * 32) + 8 * (r & 3));
        } else {
#pragma unroll
            for (int h = 0; h < GK / 32; ++h) addr[h] = (unsigned)((w0 + r) * 2 * GK + (((4 * h + q) ^ chunk_key<GK>(r)) * 16));
        }
    }
    // fragment of tile t, k half h (32 k)
    __device__ __forceinline__ bf16x8 get(const unsigned char* tile, int t, int h) const {
        if constexpr (T) {
            const unsigned char* p = tile + addr[t] + h * (32 * 2 * R);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(lds_ptr)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(lds_ptr)(p + 4 * 2 * R));
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            return *(const bf16x8*)(tile + addr[h] + t * (32 * GK));
        }
    }
};

// workgroup -> (tile, split).  Consecutive workgroups go to the 8 XCDs in turn; each XCD gets a contiguous run of work so that its
// L2 sees neighbouring tiles: splits outermost (an XCD reads its own range of k), then groups of 8 row tiles.
__device__ __forceinline__ void tile_of_block(const TileArgs& p, int& tm, int& tn, int& split) {
    const unsigned nblk = gridDim.x, x = blockIdx.x & 7, per = nblk >> 3, rest = nblk & 7;
    unsigned id = x * per + (x < rest ? x : rest) + (blockIdx.x >> 3);
    const unsigned tiles = (unsigned)p.tiles_m * p.tiles_n;
    split = id / tiles;
    id -= split * tiles;
    const unsigned band = 8u * p.tiles_n, g = id / band;
    const unsigned first = g * 8, rows = min(8u, (unsigned)p.tiles_m - first);
    const unsigned in = id - g * band;
    tm = first + in % rows;
    tn = in / rows;
}

constexpr int ER = 32;                                // rows of a wave's tile per epilogue pass
constexpr int epilogue_bytes(int waves, int wtn) { return waves * ER * (wtn + 4) * 4; }      // reuses the operand stages

// The wave's accumulators (tile at row m0, column n0): split sums as they are, or the finished output
template <int WTM, int WTN, typename T, bool PART>
__device__ __forceinline__ void tile_store(const TileArgs& p, const f32x4 (&acc)[WTM / 16][WTN / 16], unsigned char* lds, int split, int wave,
                                           int lane, long long m0, int n0) {
    constexpr int MT = WTM / 16, NT = WTN / 16, EP = WTN + 4;
    // a lane holds columns 4 q .. 4 q + 3 (q = lane / 16) of row lane % 16 of every 16 x 16 tile
    const int r = lane & 15, q = lane >> 4;
    if constexpr (PART) {
        float* part = p.part + (size_t)split * p.M * p.part_ld;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const long long m = m0 + 16 * i + r;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int n = n0 + 16 * j + 4 * q;
                if (m < p.M && n < p.part_ld) *(f32x4*)(part + m * p.part_ld + n) = acc[i][j];
            }
        }
    } else {
        // through LDS, 32 rows of the wave at a time, to whole rows: each lane then has 8 columns of one row, and 8 neighbouring
        // lanes of a 64-column wave tile write whole 128-byte lines
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        float* st = (float*)lds + wave * (ER * EP);
        constexpr int LPR = WTN / 8, RPI = 64 / LPR;          // lanes per row, rows per step
        const int c = (lane % LPR) * 8, n = n0 + c;
        float bias[8];
        load_bias<T, 8>(p, n, bias);
#pragma unroll 1
        for (int pass = 0; pass < WTM / ER; ++pass) {
#pragma unroll
            for (int w = 0; w < WTM / ER; ++w) {
                if (w != pass) continue;
#pragma unroll
                for (int i = 0; i < ER / 16; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) *(f32x4*)(st + (16 * i + r) * EP + 16 * j + 4 * q) = acc[w * (ER / 16) + i][j];
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1
            for (int it = 0; it < ER / RPI; ++it) {
                const int row = it * RPI + lane / LPR;
                const long long m = m0 + pass * ER + row;
                float v[8];
                load_vec<8>(st + row * EP + c, v);
                if (m < p.M && n < p.N) row_epilogue<T, 8>(p, v, bias, m, n);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
}

// (two waves per SIMD as a bound keeps the accumulators out of the AGPRs, between which and the VGPRs the compiler otherwise moves them
// every step)
template <int BM, int BN, int WM, int WN, bool AT, bool BT, int GK, int NSTAGE, bool PIPE, typename T, bool PART>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_tile_kernel(TileArgs p) {
    constexpr int NW = WM * WN, WTM = BM / WM, WTN = BN / WN, MT = WTM / 16, NT = WTN / 16;
    constexpr int STAGE = (BM + BN) * GK * 2;
    constexpr int U = (BM + BN) * GK / 512 / NW;              // DMA instructions per wave and step
    extern __shared__ __align__(1024) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tm, tn, split;
    tile_of_block(p, tm, tn, split);
    const long long m0 = (long long)tm * BM;
    const int n0 = tn * BN;
    const int wm = (wave / WN) * WTM, wn = (wave % WN) * WTN;

    TileLoader<BM, NW, AT, GK> la;
    TileLoader<BN, NW, BT, GK> lb;
    la.init((const bf16_t*)p.a, p.lda, m0, p.M, wave, lane);
    lb.init((const bf16_t*)p.b, p.ldb, n0, p.N, wave, lane);
    TileReader<BM, MT, AT, GK> ra;
    TileReader<BN, NT, BT, GK> rb;
    ra.init(wm, lane);
    rb.init(wn, lane);

    const int ksteps = (int)((p.K + GK - 1) / GK), klast = (int)(p.K - (long long)(ksteps - 1) * GK);
    int kstep = (int)((long long)ksteps * split / p.splits);                    // the next step to request
    const int nsteps = (int)((long long)ksteps * (split + 1) / p.splits) - kstep, kend = kstep + nsteps;
    const unsigned lds0 = (unsigned)(uintptr_t)(lds_ptr)lds;
    unsigned long long at_a = la.at(kstep), at_b = lb.at(kstep);
    const unsigned long long inc_a = la.stride(), inc_b = lb.stride();
    u32x4 rsa, rsb;
    int klim;
    unsigned dst;
    auto step_setup = [&](int buf) {
        rsa = tile_rsrc(at_a);
        rsb = tile_rsrc(at_b);
        klim = kstep >= kend ? 0 : kstep + 1 == ksteps ? klast : GK;          // past the end: every lane out of range, zeros nobody multiplies
        dst = lds0 + (unsigned)(buf * STAGE);
        ++kstep;
        at_a += inc_a;
        at_b += inc_b;
    };
    auto request = [&](int i) {
        if (i < TileLoader<BM, NW, AT, GK>::UNITS) la.issue(i, rsa, klim, dst, wave);
        else lb.issue(i - TileLoader<BM, NW, AT, GK>::UNITS, rsb, klim, dst + BM * GK * 2, wave);
    };
    auto issue = [&](int buf) {
        step_setup(buf);
#pragma unroll
        for (int i = 0; i < U; ++i) request(i);
    };

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    bf16x8 fa[PIPE ? 2 : 1][MT], fb[PIPE ? 2 : 1][NT];
    // share i of MT of a half's reads
    auto read = [&](int h, int buf, int i) {
        const unsigned char* ta = lds + buf * STAGE;
        const unsigned char* tb = ta + BM * GK * 2;
#pragma unroll
        for (int j = i * NT / MT; j < (i + 1) * NT / MT; ++j) fb[PIPE ? h : 0][j] = rb.get(tb, j, h);
        fa[PIPE ? h : 0][i] = ra.get(ta, i, h);
    };
    auto multiply = [&](int h, int i) {
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[PIPE ? h : 0][j], fa[PIPE ? h : 0][i], acc[i][j], 0, 0, 0);
    };
    int buf = 0;
    if constexpr (PIPE) {
        // Two halves of 32 k per step, their fragments double-buffered in registers: while the matrix cores work on one half, the other
        // half's LDS reads are under way.  Half-way through a step the wave has read all of it: the barrier there both publishes the
        // next step's tiles and frees this step's for the request NSTAGE steps ahead.
#pragma unroll
        for (int i = 0; i < NSTAGE; ++i) issue(i);
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NSTAGE - 1) * U) : "memory");
#pragma unroll
        for (int i = 0; i < MT; ++i) read(0, 0, i);
        for (int s = 0; s < nsteps; ++s) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                read(1, buf, i);
                if (i == MT / 2) step_setup(buf);
                multiply(0, i);
                __builtin_amdgcn_sched_barrier(0);
            }
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NSTAGE - 2) * U) : "memory");
            buf = buf + 1 == NSTAGE ? 0 : buf + 1;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                read(0, buf, i);
#pragma unroll
                for (int k = i * U / MT; k < (i + 1) * U / MT; ++k) request(k);
                multiply(1, i);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    } else {
        // several workgroups per CU hide each other's waits: read, multiply, one barrier per step
#pragma unroll
        for (int i = 0; i < NSTAGE - 1; ++i) issue(i);
        int wbuf = NSTAGE - 1;
        for (int s = 0; s < nsteps; ++s) {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NSTAGE - 2) * U) : "memory");
            issue(wbuf);
            wbuf = wbuf + 1 == NSTAGE ? 0 : wbuf + 1;
#pragma unroll
            for (int h = 0; h < GK / 32; ++h) {
                const unsigned char* ta = lds + buf * STAGE;
                const unsigned char* tb = ta + BM * GK * 2;
#pragma unroll
                for (int i = 0; i < MT; ++i) fa[0][i] = ra.get(ta, i, h);
#pragma unroll
                for (int j = 0; j < NT; ++j) fb[0][j] = rb.get(tb, j, h);
#pragma unroll
                for (int i = 0; i < MT; ++i) multiply(0, i);
            }
            buf = buf + 1 == NSTAGE ? 0 : buf + 1;
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");       // the requests past the end, before LDS is used again or given back

    tile_store<WTM, WTN, T, PART>(p, acc, lds, split, wave, lane, m0 + wm, n0 + wn);
}

// Adds the split sums and applies the epilogue; 8 columns of a row belong to SL lanes, lane k of which adds splits k, k + SL, ... in
// order (their loads are independent: with few outputs and many splits the launch is bound by memory latency), then lane 0 adds
// the SL sums in order.
// The workgroups behind the first `blocks` add another call's partial rows (db's, see linear_dz_kernel): 16 columns and 16 lanes each, lane
// k adds rows k, k + 16, ... in order, then the lanes are added in order.  One launch instead of two (4 us and the gap between them).
struct SlotSum {
    const float* part; int slots, n;      // [slots][n]
    void* out;
};
template <typename T>
__device__ __forceinline__ void slot_sum_block(const SlotSum& s, unsigned block, float (*red)[17]) {
    const int cl = threadIdx.x & 15, sl = threadIdx.x >> 4, c = (int)block * 16 + cl;
    float v = 0.f;
    if (c < s.n) {
#pragma unroll 16
        for (int k = sl; k < s.slots; k += 16) v += s.part[(size_t)k * s.n + c];
    }
    red[sl][cl] = v;
    __syncthreads();
    if (sl == 0 && c < s.n) {
#pragma unroll
        for (int k = 1; k < 16; ++k) v += red[k][cl];
        ((T*)s.out)[c] = from_f32<T>(v);
    }
}

template <typename T, int SL>
__global__ __launch_bounds__(256) void gemm_join_kernel(TileArgs p, unsigned blocks, SlotSum other) {
    constexpr int G = 256 / SL;
    __shared__ f32x4 red[SL > 1 ? 256 : 1][2];
    __shared__ float rows[16][17];
    if (blockIdx.x >= blocks) {
        slot_sum_block<T>(other, blockIdx.x - blocks, rows);
        return;
    }
    const int cols = p.part_ld / 8, g = threadIdx.x % G, sl = threadIdx.x / G;
    const long long n8 = p.M * cols;
    const size_t slot = (size_t)p.M * p.part_ld;
    for (long long e0 = (long long)blockIdx.x * G; e0 < n8; e0 += (long long)blocks * G) {
        const long long e = e0 + g, m = e / cols;
        const int n = (int)(e - m * cols) * 8;
        f32x4 v0 = {0.f, 0.f, 0.f, 0.f}, v1 = v0;
        if (e < n8) {
            const float* s = p.part + m * p.part_ld + n;
            for (int k = sl; k < p.splits; k += SL) {
                v0 += *(const f32x4*)(s + k * slot);
                v1 += *(const f32x4*)(s + k * slot + 4);
            }
        }
        if constexpr (SL > 1) {
            __syncthreads();
            red[threadIdx.x][0] = v0;
            red[threadIdx.x][1] = v1;
            __syncthreads();
            if (sl == 0) {
#pragma unroll
                for (int k = 1; k < SL; ++k) {
                    v0 += red[k * G + g][0];
                    v1 += red[k * G + g][1];
                }
            }
        }
        if (e < n8 && sl == 0) {
            float v[8], bias[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = v0[j]; v[4 + j] = v1[j]; }
            load_bias<T, 8>(p, n, bias);
            row_epilogue<T, 8>(p, v, bias, m, n);
        }
    }
}

// ---- operands through registers ------------------------------------------------------------------------------------------
constexpr int SK = 32;                                // k per step

// two f32 -> the high, middle and low bf16 pairs.  hi is cut, not rounded (no overflow at the largest values, and an infinity or NaN
// leaves a NaN in the rest), mid and lo are rounded: what is dropped has either sign.
__device__ __forceinline__ void split3(float x0, float x1, unsigned& hi, unsigned& mid, unsigned& lo) {
    const unsigned b0 = __builtin_bit_cast(unsigned, x0), b1 = __builtin_bit_cast(unsigned, x1);
    hi = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
    const float r0 = x0 - __builtin_bit_cast(float, b0 & 0xffff0000u), r1 = x1 - __builtin_bit_cast(float, b1 & 0xffff0000u);
    mid = pack_bf2(r0, r1);
    lo = pack_bf2(r0 - __builtin_bit_cast(float, mid << 16), r1 - __builtin_bit_cast(float, mid & 0xffff0000u));
}

// One step's share of a thread: R x 32 of an operand over 256 threads, chunks of 8 values
template <typename E, int R>
struct StagedChunks {
    u32x4 v[R / 64][sizeof(E) == 4 ? 2 : 1];
    static_assert(R % 64 == 0, "whole chunks per thread");
};

// Where the thread's chunks lie.  load(): a whole step, no tests - rows past the end repeat the last one along k, and across k the last
// chunk runs over its row's end; what either produces is not stored.  load_last(): the last step of the operand, element by
// element where a chunk is partial, zeros past K.  NARROW (across k, fewer than 8 columns): a chunk could run past the last row
// from more than one row up, so every step is loaded that way.  LDS planes of bf16 are laid out as TileLoader's.
template <typename E, int R, bool T, bool NARROW>
struct StagedOperand {
    static constexpr int P = sizeof(E) == 4 ? 3 : 1, H = sizeof(E) == 4 ? 2 : 1, CH = R / 64, CPR = R / 8, PLANE = R * SK * 2;
    const E* p[CH];                    // of the step that is loaded next
    long long inc, rows;
    int k, K, col[CH];                 // k and K from the first step on

    __device__ __forceinline__ void init(const void* base, long long ld, long long row0, long long rows_, long long k0, long long K_, int tid) {
        rows = rows_; k = 0; K = (int)(K_ - k0 < 0x7fffffff ? K_ - k0 : 0x7fffffff);
        inc = T ? SK * ld : SK;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int e = tid + 256 * i;
            long long r = T ? row0 + 8 * (e % CPR) : row0 + e / 4;
            if (r >= rows) r = T ? (rows - 1) / 8 * 8 : rows - 1;
            if constexpr (T) {
                p[i] = (const E*)base + (k0 + e / CPR) * ld + r;
                col[i] = (int)(rows - r < 8 ? rows - r : 8);                  // columns of the chunk that exist
            } else {
                p[i] = (const E*)base + r * ld + k0 + 8 * (e % 4);
            }
        }
    }
    __device__ __forceinline__ void step() {
        k += SK;
#pragma unroll
        for (int i = 0; i < CH; ++i) p[i] += inc;
    }
    __device__ __forceinline__ void load(StagedChunks<E, R>& c, int tid) {
        if constexpr (NARROW && T) {
            load_last(c, tid);
            step();
        } else {
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int h = 0; h < H; ++h) c.v[i][h] = *(const u32x4_any*)(p[i] + 4 * h);
            step();
        }
    }
    // `ahead`: steps between the current one and the one to load
    __device__ __forceinline__ void load_last(StagedChunks<E, R>& c, int tid, int ahead = 0) const {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int e = tid + 256 * i, kk = k + ahead * SK + (T ? e / CPR : 8 * (e % 4));
            const E* q = p[i] + ahead * inc;
            const int left = T ? (kk < K ? col[i] : 0) : K - kk;
#pragma unroll
            for (int h = 0; h < H; ++h) c.v[i][h] = u32x4{0u, 0u, 0u, 0u};
            if (left >= 8) {
#pragma unroll
                for (int h = 0; h < H; ++h) c.v[i][h] = *(const u32x4_any*)(q + 4 * h);
            } else if (left > 0) {
                if constexpr (sizeof(E) == 4) {
#pragma unroll
                    for (int j = 0; j < 7; ++j)
                        if (j < left) c.v[i][j / 4][j % 4] = ((const unsigned*)q)[j];
                } else {
                    u16x8 o = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 7; ++j)
                        if (j < left) o[j] = q[j];
                    c.v[i][0] = __builtin_bit_cast(u32x4, o);
                }
            }
        }
    }
    static __device__ __forceinline__ void store(const StagedChunks<E, R>& ch, unsigned char* tile, int tid) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int e = tid + 256 * i;
            int at;
            if constexpr (T) {
                const int k = e / CPR, c = e % CPR;
                at = k * 2 * R + ((((c >> 1) ^ (((k & 3) | ((k >> 3 & 1) << 2)) & (R / 16 - 1))) * 2 + (c & 1)) * 16);
            } else {
                const int r = e / 4;
                at = r * 64 + (((e % 4) ^ chunk_key<SK>(r)) * 16);
            }
            if constexpr (sizeof(E) == 4) {
                u32x4 o[3];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned q0 = ch.v[i][j >> 1][2 * (j & 1)], q1 = ch.v[i][j >> 1][2 * (j & 1) + 1];
                    unsigned hi, mid, lo;
                    split3(__builtin_bit_cast(float, q0), __builtin_bit_cast(float, q1), hi, mid, lo);
                    o[0][j] = hi; o[1][j] = mid; o[2][j] = lo;
                }
#pragma unroll
                for (int t = 0; t < 3; ++t) *(u32x4*)(tile + t * PLANE + at) = o[t];
            } else {
                *(u32x4*)(tile + at) = ch.v[i][0];
            }
        }
    }
};

template <int R, int NT, bool T>
struct StagedReader {
    unsigned addr[T ? NT : 1];
    __device__ __forceinline__ void init(int w0, int lane) {
        const int r = lane & 15, q = lane >> 4;
        if constexpr (T) {
            const int f = ((r >> 2) | ((q & 1) << 2)) & (R / 16 - 1);
#pragma unroll
            for (int t = 0; t < NT; ++t) addr[t] = (unsigned)((8 * q + (r >> 2)) * 2 * R + (((w0 / 16 + t) ^ f) * 32) + 8 * (r & 3));
        } else {
            addr[0] = (unsigned)((w0 + r) * 64 + ((q ^ chunk_key<SK>(r)) * 16));
        }
    }
    __device__ __forceinline__ bf16x8 get(const unsigned char* plane, int t) const {
        if constexpr (T) {
            const unsigned char* p = plane + addr[t];
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(lds_ptr)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(lds_ptr)(p + 4 * 2 * R));
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            return *(const bf16x8*)(plane + addr[0] + t * 1024);
        }
    }
};

template <int B, typename T>
constexpr int staged_lds() {
    constexpr int tiles = (sizeof(T) == 4 ? 3 : 1) * 2 * B * SK * 2 * (B == 64 ? 2 : 1), ep = epilogue_bytes(4, B / 2);
    return tiles > ep ? tiles : ep;
}

// B x B tile, four waves of B/2 x B/2; the next D steps' operands wait in registers while this step's are multiplied (a small tile's step
// is shorter than a memory access)
template <int B, bool AT, bool BT, bool NARROW, typename T, bool PART>
__global__ __launch_bounds__(256, 2) void gemm_staged_kernel(TileArgs p) {
    constexpr int WT = B / 2, MT = WT / 16, P = sizeof(T) == 4 ? 3 : 1, PLANE = B * SK * 2, D = B == 64 ? 3 : 1;
    __shared__ __align__(1024) unsigned char lds[staged_lds<B, T>()];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int tm, tn, split;
    tile_of_block(p, tm, tn, split);
    const long long m0 = (long long)tm * B;
    const int n0 = tn * B, wm = (wave >> 1) * WT, wn = (wave & 1) * WT;
    StagedReader<B, MT, AT> ra;
    StagedReader<B, MT, BT> rb;
    ra.init(wm, lane);
    rb.init(wn, lane);
    const long long ksteps = (p.K + SK - 1) / SK;
    const long long s0 = ksteps * split / p.splits;
    const int nsteps = (int)(ksteps * (split + 1) / p.splits - s0);
    // whole steps, then the operand's last step if it is this split's
    const bool tail = nsteps > 0 && s0 + nsteps == ksteps;
    const int full = nsteps - tail;
    StagedOperand<T, B, AT, NARROW> sa;
    StagedOperand<T, B, BT, NARROW> sb;
    sa.init(p.a, p.lda, m0, p.M, s0 * SK, p.K, tid);
    sb.init(p.b, p.ldb, n0, p.N, s0 * SK, p.K, tid);
    StagedChunks<T, B> ca[D], cb[D];
    f32x4 acc[MT][MT], low[P == 3 ? MT : 1][P == 3 ? MT : 1];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            if constexpr (P == 3) low[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    // the last step's chunks come first where registers allow it: their latency would stand alone at the end
    StagedChunks<T, B> la, lb;
    if (B == 64 && tail) {
        sa.load_last(la, tid, full);
        sb.load_last(lb, tid, full);
    }
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (d < full) {
            sa.load(ca[d], tid);
            sb.load(cb[d], tid);
        }
    constexpr int SET = 2 * P * PLANE;                                  // LDS of one step
    auto multiply = [&](const unsigned char* ta) {
        const unsigned char* tb = ta + P * PLANE;
        bf16x8 fb[P][MT];
#pragma unroll
        for (int t = 0; t < P; ++t)
#pragma unroll
            for (int j = 0; j < MT; ++j) fb[t][j] = rb.get(tb + t * PLANE, j);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            bf16x8 fa[P];
#pragma unroll
            for (int t = 0; t < P; ++t) fa[t] = ra.get(ta + t * PLANE, i);
            if constexpr (P == 3) {
#pragma unroll
                for (int u = 0; u < 5; ++u) {                  // mid mid, lo hi, hi lo, mid hi, hi mid
                    constexpr int UA[5] = {1, 2, 0, 1, 0}, UB[5] = {1, 0, 2, 0, 1};
#pragma unroll
                    for (int j = 0; j < MT; ++j) low[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[UB[u]][j], fa[UA[u]], low[i][j], 0, 0, 0);
                }
            }
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[0][j], fa[0], acc[i][j], 0, 0, 0);
        }
    };
    int buf = 0;
    for (int s = 0; s < full; s += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (s + d >= full) break;
            // two sets of LDS tiles where they fit (B = 64): a set is written again only after the barrier behind its reads
            if constexpr (B != 64) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            sa.store(ca[d], lds + buf, tid);
            sb.store(cb[d], lds + buf + P * PLANE, tid);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (s + d + D < full) {
                sa.load(ca[d], tid);
                sb.load(cb[d], tid);
            }
            multiply(lds + buf);
            if constexpr (B == 64) buf ^= SET;
        }
    }
    if (tail) {
        if constexpr (B != 64) {
            sa.load_last(la, tid);
            sb.load_last(lb, tid);
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        sa.store(la, lds, tid);
        sb.store(lb, lds + P * PLANE, tid);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        multiply(lds);
    }
    if constexpr (P == 3) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[i][j] += low[i][j];
    }
    tile_store<WT, WT, T, PART>(p, acc, lds, split, wave, lane, m0 + wm, n0 + wn);
}

}  // namespace srmi
