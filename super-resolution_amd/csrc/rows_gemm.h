// The tile product of the row operators: C[m, n] = sum_k A(m, k) B(n, k), bf16 operands, f32 sums on the matrix cores.
//
// A workgroup owns a BM x BN tile and walks K in steps of 64.  Operand tiles go straight from memory to LDS
// (buffer_load_dwordx4 ... lds: no register round trip), up to NSTAGE steps ahead of the step being multiplied, with one barrier
// per step.  An operand may be stored along k ([row][k], like x and w in x w^T) or across it ([k][row], like w in dz w and both
// operands of dz^T x): the second kind is read from LDS with the transposing read (ds_read_b64_tr_b16), so that no operand is ever
// re-laid out in memory.
//
// LDS layouts, both free of bank conflicts:
//   along k    128-byte rows of eight 16-byte chunks, chunk c of row r at position c ^ (r & 7);
//   across k   one row per k, columns in 32-byte pairs of chunks, pair p of row k at position p ^ ((k & 3) | (k >> 3 & 1) << 2):
//              the eight k rows that half a wave's transposing read touches fall on eight different pairs.
// The DMA writes LDS linearly, so the permutation is applied to the global address of each lane.
// Rows and k past the operand's end are lanes whose buffer offset is out of range: the hardware returns zeros.
//
// f32 operands arrive as three bf16 planes (x = hi + mid + lo exactly, to 24 bits); the six products hi hi, hi mid, mid hi, hi lo,
// mid mid, lo hi are six passes over K with the plane pointers exchanged, smallest first, which leaves the rounding of an
// f32 sum over K (the dropped products are below 2^-24 of the largest).
#pragma once
#include "rows_common.h"

namespace srmi {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
typedef __attribute__((address_space(3))) void* lds_ptr;

constexpr int GK = 64;                               // k per step
constexpr unsigned OUT_OF_RANGE = 0x80000000u;       // buffer offset = the resource's size: reads zeros
constexpr long long GEMM_MAX_LD = 1 << 22;           // a tile's offsets stay below 2^31 bytes

struct TileArgs {
    const bf16_t* a; const bf16_t* b;
    long long lda, ldb;                              // row strides in elements, multiples of 8
    long long pa, pb;                                // distance of the planes (f32)
    long long M, K; int N;
    int terms;                                       // 1, or 6 for f32 planes
    int tiles_m, tiles_n, splits;
    float* part; int part_ld;                        // split sums: [splits][M][part_ld]
    // epilogue
    const void* bias; const void* residual; void* y; void* z;
    long long ldr, ldy;                              // z is dense [M, N]
    int act; float act_param;
};

// act(v + bias) + residual for V columns of one row, stored as T
template <typename T, int V>
__device__ __forceinline__ void row_epilogue(const TileArgs& p, float* v, const float* bias, long long m, int n) {
    constexpr bool FAST = sizeof(T) == 2;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += bias[j];
    const bool whole = n + V <= p.N;
    if (p.z) {
        T* z = (T*)p.z + m * p.N + n;
        if (whole) store_vec<V>(z, v);
        else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (n + j < p.N) z[j] = from_f32<T>(v[j]);
        }
    }
    switch (p.act) {
#define SRMI_ROW_ACT(CODE)                                                              \
    case CODE: {                                                                        \
        _Pragma("unroll") for (int j = 0; j < V; ++j) v[j] = row_act<FAST>(v[j], CODE, p.act_param); \
        break;                                                                          \
    }
        SRMI_ROW_ACT(SRMI_ACT_RELU)
        SRMI_ROW_ACT(SRMI_ACT_LRELU)
        SRMI_ROW_ACT(SRMI_ACT_TANH)
        SRMI_ROW_ACT(SRMI_ACT_SIGMOID)
        SRMI_ROW_ACT(SRMI_ACT_GELU)
        SRMI_ROW_ACT(SRMI_ACT_GELU_TANH)
        SRMI_ROW_ACT(SRMI_ACT_SILU)
#undef SRMI_ROW_ACT
        default: break;
    }
    T* y = (T*)p.y + m * p.ldy + n;
    if (p.residual) {
        const T* r = (const T*)p.residual + m * p.ldr + n;
        float q[V];
        if (whole) load_vec<V>(r, q);
        else {
#pragma unroll
            for (int j = 0; j < V; ++j) q[j] = n + j < p.N ? to_f32(r[j]) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += q[j];
    }
    if (whole) store_vec<V>(y, v);
    else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (n + j < p.N) y[j] = from_f32<T>(v[j]);
    }
}

template <typename T, int V>
__device__ __forceinline__ void load_bias(const TileArgs& p, int n, float* bias) {
#pragma unroll
    for (int j = 0; j < V; ++j) bias[j] = p.bias && n + j < p.N ? to_f32(((const T*)p.bias)[n + j]) : 0.f;
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

// Staging of one operand: R rows, NW waves, T: stored across k
template <int R, int NW, bool T>
struct TileLoader {
    static constexpr int UNITS = R / 8 / NW;          // KiB per wave and step
    static constexpr int CPR = R / 8;                 // chunks per k row (T)
    unsigned voff[UNITS];
    int kk[T ? UNITS : 1];                            // k of the lane's chunk inside the step
    const bf16_t* base; long long ld;
    static_assert(R % (8 * NW) == 0, "whole KiB per wave");

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
                const int r = 8 * u + (lane >> 3), c = (lane & 7) ^ (lane >> 3);
                kk[0] = 8 * c;
                voff[i] = row0 + r < rows ? (unsigned)(r * ld_ * 2 + 16 * c) : OUT_OF_RANGE;
            }
        }
    }
    // address of step `step` (64 k each) in the plane at element offset `plane`, and the distance to the next step
    __device__ __forceinline__ unsigned long long at(long long step, long long plane) const {
        return (unsigned long long)(uintptr_t)base + 2 * (plane + step * GK * (T ? ld : 1));
    }
    __device__ __forceinline__ unsigned long long stride() const { return 2 * GK * (unsigned long long)(T ? ld : 1); }
    // request the wave's i-th KiB; klim: k of the step that exist, lds: byte address of the tile
    __device__ __forceinline__ void issue(int i, const u32x4& rsrc, int klim, unsigned lds, int wave) const {
        dma_1k(rsrc, kk[T ? i : 0] < klim ? voff[i] : OUT_OF_RANGE, __builtin_amdgcn_readfirstlane(lds + (unsigned)((i * NW + wave) * 1024)));
    }
};

// Fragments of one operand for the wave: NT tiles of 16 rows starting at row w0 (a multiple of 16 NT) of the LDS tile
template <int R, int NT, bool T>
struct TileReader {
    unsigned addr[T ? NT : 2];
    __device__ __forceinline__ void init(int w0, int lane) {
        const int r = lane & 15, q = lane >> 4;
        if constexpr (T) {
            // lane's address: k row 8 q + (r >> 2), four columns at 4 (r & 3); it receives column r, k = 8 q .. 8 q + 3
            const int f = ((r >> 2) | ((q & 1) << 2)) & (R / 16 - 1);
#pragma unroll
            for (int t = 0; t < NT; ++t) addr[t] = (unsigned)((8 * q + (r >> 2)) * 2 * R + (((w0 / 16 + t) ^ f) * 32) + 8 * (r & 3));
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) addr[h] = (unsigned)((w0 + r) * 128 + (((4 * h + q) ^ (r & 7)) * 16));
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
            return *(const bf16x8*)(tile + addr[h] + t * 2048);
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

template <int BM, int BN, int WM, int WN, bool AT, bool BT, int NSTAGE, bool PIPE, typename T, bool PART>
__global__ __launch_bounds__(64 * WM * WN) void gemm_tile_kernel(TileArgs p) {
    constexpr int NW = WM * WN, WTM = BM / WM, WTN = BN / WN, MT = WTM / 16, NT = WTN / 16;
    constexpr int STAGE = (BM + BN) * GK * 2;
    constexpr int U = (BM + BN) / 8 / NW;                     // DMA instructions per wave and step
    constexpr int ER = 32;                                    // rows per epilogue pass
    constexpr int EP = WTN + 4;                               // floats per staged row
    static_assert(NW * ER * EP * 4 <= NSTAGE * STAGE, "the epilogue reuses the operand stages");
    extern __shared__ __align__(1024) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tm, tn, split;
    tile_of_block(p, tm, tn, split);
    const long long m0 = (long long)tm * BM;
    const int n0 = tn * BN;
    const int wm = (wave / WN) * WTM, wn = (wave % WN) * WTN;

    TileLoader<BM, NW, AT> la;
    TileLoader<BN, NW, BT> lb;
    la.init(p.a, p.lda, m0, p.M, wave, lane);
    lb.init(p.b, p.ldb, n0, p.N, wave, lane);
    TileReader<BM, MT, AT> ra;
    TileReader<BN, NT, BT> rb;
    ra.init(wm, lane);
    rb.init(wn, lane);

    const int ksteps = (int)((p.K + GK - 1) / GK);
    const long long total = (long long)p.terms * ksteps;
    const long long s_begin = total * split / p.splits, s_end = total * (split + 1) / p.splits;
    const unsigned lds0 = (unsigned)(uintptr_t)(lds_ptr)lds;

    // the next step to request: its place in the pass over k (f32: which pass over the planes, 5 = hi hi), and what its requests need
    constexpr bool PLANES = sizeof(T) == 4;
    int term = PLANES ? (int)(s_begin / (ksteps > 0 ? ksteps : 1)) : 5;
    int kstep = PLANES ? (int)(s_begin - (long long)term * ksteps) : (int)s_begin;
    const int klast = (int)(p.K - (long long)(ksteps - 1) * GK), nsteps = (int)(s_end - s_begin);
    auto plane_a = [&] { return PLANES ? (0x001012 >> (4 * term) & 3) * p.pa : 0; };      // planes of (2,0) (1,1) (0,2) (1,0) (0,1) (0,0)
    auto plane_b = [&] { return PLANES ? (0x010210 >> (4 * term) & 3) * p.pb : 0; };
    unsigned long long at_a = la.at(kstep, plane_a()), at_b = lb.at(kstep, plane_b());
    const unsigned long long inc_a = la.stride(), inc_b = lb.stride();
    u32x4 rsa, rsb;
    int klim, left = nsteps;
    unsigned dst;
    auto step_setup = [&](int buf) {
        rsa = tile_rsrc(at_a);
        rsb = tile_rsrc(at_b);
        klim = left <= 0 ? 0 : kstep + 1 == ksteps ? klast : GK;      // past the end: every lane out of range, zeros nobody multiplies
        --left;
        dst = lds0 + (unsigned)(buf * STAGE);
        ++kstep;
        at_a += inc_a;
        at_b += inc_b;
        if (PLANES && kstep == ksteps) {
            kstep = 0;
            ++term;
            at_a = la.at(0, plane_a());
            at_b = lb.at(0, plane_b());
        }
    };
    auto request = [&](int i) {
        if (i < TileLoader<BM, NW, AT>::UNITS) la.issue(i, rsa, klim, dst, wave);
        else lb.issue(i - TileLoader<BM, NW, AT>::UNITS, rsb, klim, dst + BM * GK * 2, wave);
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
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < MT; ++i) read(h, buf, i);
#pragma unroll
                for (int i = 0; i < MT; ++i) multiply(h, i);
            }
            buf = buf + 1 == NSTAGE ? 0 : buf + 1;
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");       // the requests past the end, before LDS is used again or given back

    // a lane holds columns 4 q .. 4 q + 3 (q = lane / 16) of row lane % 16 of every 16 x 16 tile
    const int r = lane & 15, q = lane >> 4;
    if constexpr (PART) {
        float* part = p.part + (size_t)split * p.M * p.part_ld;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const long long m = m0 + wm + 16 * i + r;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int n = n0 + wn + 16 * j + 4 * q;
                if (m < p.M && n < p.part_ld) *(f32x4*)(part + m * p.part_ld + n) = acc[i][j];
            }
        }
    } else {
        // through LDS, 32 rows of the wave at a time, to whole rows: each lane then has 8 columns of one row, and 8 neighbouring
        // lanes of a 64-column wave tile write whole 128-byte lines
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        float* st = (float*)lds + wave * (ER * EP);
        constexpr int LPR = WTN / 8, RPI = 64 / LPR;          // lanes per row, rows per step
        const int c = (lane % LPR) * 8, n = n0 + wn + c;
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
                const long long m = m0 + wm + pass * ER + row;
                float v[8];
                const f32x4 v0 = *(const f32x4*)(st + row * EP + c), v1 = *(const f32x4*)(st + row * EP + c + 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) { v[j] = v0[j]; v[4 + j] = v1[j]; }
                if (m < p.M && n < p.N) row_epilogue<T, 8>(p, v, bias, m, n);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
}

// Adds the split sums and applies the epilogue; 8 columns of a row belong to SL lanes, lane k of which adds splits k, k + SL, ... in
// order (their loads are independent: with few outputs and many splits the launch is bound by memory latency), then lane 0 adds
// the SL sums in order.
template <typename T, int SL>
__global__ __launch_bounds__(256) void gemm_join_kernel(TileArgs p) {
    constexpr int G = 256 / SL;
    __shared__ f32x4 red[SL > 1 ? 256 : 1][2];
    const int cols = p.part_ld / 8, g = threadIdx.x % G, sl = threadIdx.x / G;
    const long long n8 = p.M * cols;
    const size_t slot = (size_t)p.M * p.part_ld;
    for (long long e0 = (long long)blockIdx.x * G; e0 < n8; e0 += (long long)gridDim.x * G) {
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

// ---- operands in the kernel's form -------------------------------------------------------------------------------------
// x as three bf16 values whose sum is x to 24 bits (rounded, not cut: the dropped products of two operands then have either sign).
// Values that would round to infinity are cut; an infinity or NaN stays in the first value.
__device__ __forceinline__ void split3(float x, bf16_t* o) {
    bf16_t h = f2bf(x);
    const bool finite = (__builtin_bit_cast(unsigned, x) & 0x7f800000u) != 0x7f800000u;
    if (finite && (h & 0x7f80) == 0x7f80) h = (bf16_t)(__builtin_bit_cast(unsigned, x) >> 16);
    const float r1 = finite ? x - bf2f(h) : 0.f;
    const bf16_t m = f2bf(r1);
    o[0] = h;
    o[1] = m;
    o[2] = f2bf(r1 - bf2f(m));
}

// 8 values -> `planes` bf16 planes at dst, dst + plane, ...
template <typename T>
__device__ __forceinline__ void store_planes8(bf16_t* dst, long long plane, const float* v) {
    if constexpr (sizeof(T) == 2) {
        store_vec<8>(dst, v);
    } else {
        bf16_t o[8][3];
#pragma unroll
        for (int j = 0; j < 8; ++j) split3(v[j], o[j]);
#pragma unroll
        for (int t = 0; t < 3; ++t) {
            u16x8 q;
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = o[j][t];
            *(u16x8*)(dst + t * plane) = q;
        }
    }
}

// [rows, cols] of T with any row stride -> bf16 plane(s) [rows, ld], ld = cols rounded up to 8, zeros behind the columns
template <typename T>
__global__ __launch_bounds__(256) void pack_rows_kernel(const T* src, long long src_ld, long long rows, int cols, bf16_t* dst, int ld,
                                                        long long plane) {
    const int c8 = ld / 8;
    const long long n = rows * c8;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256) {
        const long long r = e / c8;
        const int c = (int)(e - r * c8) * 8;
        const T* s = src + r * src_ld + c;
        float v[8];
        if (c + 8 <= cols) load_vec<8>(s, v);
        else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? to_f32(s[j]) : 0.f;
        }
        store_planes8<T>(dst + r * ld + c, plane, v);
    }
}

}  // namespace srmi
