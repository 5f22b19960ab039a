// Tile product on the gfx950 matrix cores shared by the wide softmax head (dense_ce.hip) and the Dense weight gradient
// from 8-bit activations (act8.hip):   D[a][b] = sum_k A[a][k] B[b][k],  bf16 operands, fp32 accumulators in registers.
//
// Each operand comes in one of two memory orders:
//   row order    A[a][k], k contiguous        LDS tile [rows][64 k], 128-byte rows
//   column order A[k][a], a contiguous        LDS tile [64 k][cols]; ds_read_b64_tr_b16 transposes on the way out
// so the three products of a linear layer (forward, input gradient, weight gradient) need no transposed copies.
//
// Staging is LDS-DMA (buffer_load_dwordx4 ... lds): one wave-instruction fills 1 KiB of LDS linearly, so the swizzle
// that keeps the fragment reads free of bank conflicts is applied on the SOURCE side, lane by lane:
//   row order:    16-byte slot of row r holds k-group  slot ^ (r & 7)
//   column order: the four k rows a 16-lane group transposes, times the two groups of a 32-lane half, are eight rows
//                 whose 32-byte units must fall into eight different units of the 256-byte bank row: unit ^ f(k row)
// Rows, columns and k groups beyond the operand fetch an out-of-range offset, which writes zeros.
// One barrier per step (64 deep; 32 where both operands come in column order and more blocks are to fit a CU); the DMA
// of the next STAGES - 1 steps is in flight across it, retired by a counted vmcnt.
// The DMA is inline asm because behind the builtin the compiler drains vmcnt in front of every transposing LDS read
// (it cannot tell it from a reader of the buffer in flight); it has no register output, only LDS, and every wait for
// it is the explicit one in front of the barrier.
#pragma once
#include "common.h"
#include <atomic>

typedef unsigned int gt_u32x4 __attribute__((ext_vector_type(4)));

constexpr int GT_BK = 64;                        // reduction depth of one stage
constexpr unsigned GT_OOB = 0xFFFFFFF0u;         // a buffer offset no descriptor here reaches

__device__ __forceinline__ void gt_dma16(gt_u32x4 rs, unsigned voff, unsigned lds_base) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(rs), "s"(lds_base));
}

// the same for memory that nobody reads again soon: non-temporal, it displaces nothing
__device__ __forceinline__ void gt_dma16_once(gt_u32x4 rs, unsigned voff, unsigned lds_base) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(rs), "s"(lds_base));
}

__device__ __forceinline__ s16x4 gt_tr_read(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(p));
}

// One operand of a tile: `p` the tensor, `ld` elements per memory row.  Row order: rows [0, n) of length >= k_end.
// Column order: k rows [0, k_end) of which columns [0, n) are real.  n and ld are multiples of 8 in column order, k_end
// and ld in row order (16-byte groups are all in or all out).
// once: operand A is read by one tile only and not wanted in the caches (tiles of at most 128 in b; the others ignore it)
struct GtOperand {
    const bf16_t* p;
    long ld;
    int n;
    bool once = false;
};

// TR = column order.  T rows (columns) per tile, NW waves in the block, BK the depth of a stage.
template <int T, int NW, bool TR, int BK = GT_BK>
struct GtStage {
    static_assert(TR || BK == 64, "row order: 128-byte LDS rows");
    static constexpr int PIECES = T * BK / 512;                       // 1-KiB pieces per stage
    static constexpr int P = (PIECES + NW - 1) / NW;                  // per wave (fewer pieces than waves: some are
    static_assert(PIECES % NW == 0 || NW % PIECES == 0, "tile");      //  fetched twice, so every wave counts alike)
    static constexpr int BYTES = T * BK * 2;
    static constexpr int SLOTS = TR ? T / 8 : 8;                      // 16-byte slots per LDS row
    static constexpr int RPP = 64 / SLOTS;                            // LDS rows per piece

    unsigned voff[P];
    int chunk_k;                                                      // row order: this lane's k group * 8
    unsigned long base;
    long step_bytes;
    int left;                                                         // reduction elements not yet issued
    long ld2;

    // f(k row) of the column-order swizzle, in 32-byte units (T / 16 units per LDS row)
    static __device__ __forceinline__ int swz(int r) {
        if (T >= 128) return (r & 3) | ((r >> 1) & 4);
        if (T == 64) return ((r >> 1) & 1) | ((r >> 2) & 2);
        if (T == 32) return (r >> 3) & 1;
        return 0;
    }

    __device__ __forceinline__ void init(const GtOperand& o, int t0, int k0, int k1, int wave, int lane) {
        ld2 = o.ld * 2;
        left = k1 - k0;
        const int rl = lane / SLOTS, slot = lane % SLOTS;
        chunk_k = TR ? 0 : (slot ^ (rl & 7)) * 8;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int piece = PIECES >= NW ? wave * P + i : wave % PIECES;
            const int row = piece * RPP + rl;
            if (TR) {
                const int col = (slot ^ (swz(row) << 1)) * 8;
                voff[i] = t0 + col < o.n ? (unsigned)(row * ld2) + col * 2u : GT_OOB;
            } else {
                voff[i] = t0 + row < o.n ? (unsigned)(row * ld2) + chunk_k * 2u : GT_OOB;
            }
        }
        base = (unsigned long)o.p + (TR ? (long)k0 * ld2 + (long)t0 * 2 : (long)t0 * ld2 + (long)k0 * 2);
        step_bytes = TR ? BK * ld2 : BK * 2;
    }

    // DMA of the next step into LDS at byte address `lds` (uniform); steps past the end write zeros
    template <bool ONCE = false>
    __device__ __forceinline__ void issue(unsigned lds, int wave) {
        unsigned num = 0x7FFFFFF0u;
        if (TR) {                       // k rows past the end lie beyond the descriptor
            const long b = left > 0 ? (long)left * ld2 : 0;
            // the last row's real columns end before its pitch does: the descriptor may stop at the row's end because
            // `base` starts t0 columns in and columns >= n were sent out of range in init
            num = b < 0x7FFFFFF0L ? (unsigned)b : 0x7FFFFFF0u;
        }
        const gt_u32x4 rs = {(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)base),
                             (unsigned)__builtin_amdgcn_readfirstlane((int)((unsigned)(base >> 32) & 0xffffu)),
                             (unsigned)__builtin_amdgcn_readfirstlane((int)num), 0x00020000u};
        const bool in = TR || chunk_k < left;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int piece = PIECES >= NW ? wave * P + i : wave % PIECES;
            if (ONCE) gt_dma16_once(rs, in ? voff[i] : GT_OOB, lds + piece * 1024);
            else gt_dma16(rs, in ? voff[i] : GT_OOB, lds + piece * 1024);
        }
        base += step_bytes;
        left -= BK;
    }
};

// Fragment readers: 16 rows x 32 k per fragment, lane (fr = lane & 15, fq = lane >> 4) holds row fr, k = 8 fq .. + 7.
template <int T, bool TR>
struct GtFrag {
    int off;                            // lane's byte offset of fragment 0, k half 0 (column order: before the unit XOR)
    int unit;                           // column order: f(k row), in 32-byte units
    __device__ __forceinline__ void init(int wave_t0, int lane) {
        const int fr = lane & 15, fq = lane >> 4;
        if (TR) {
            const int row = 8 * fq + (fr >> 2);
            unit = GtStage<T, 1, true>::swz(row);
            off = row * (T * 2) + wave_t0 * 2 + (fr & 3) * 8;
        } else {
            off = (wave_t0 + fr) * 128 + ((fq ^ (fr & 7)) * 16);
            unit = 0;
        }
    }
    // wave_u0 = wave_t0 / 16 (units are XOR-ed with the absolute unit index inside the LDS row)
    __device__ __forceinline__ bf16x8_t load(const char* tile, int i, int kk, int wave_u0) const {
        if (TR) {
            const int u = ((wave_u0 + i) ^ unit) - wave_u0;
            const char* p = tile + off + u * 32 + kk * 32 * (T * 2);
            const s16x4 lo = gt_tr_read(p), hi = gt_tr_read(p + 4 * (T * 2));
            const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            return __builtin_bit_cast(bf16x8_t, v);
        }
        return *(const bf16x8_t*)(tile + (off ^ (kk * 64)) + i * 2048);
    }
};

// The block's tile: BA x BB outputs, WA x WB waves.  Lane (fr, fq) of fragment pair (i, j) holds
// D[wave_a0 + 16 i + 4 fq + e][wave_b0 + 16 j + fr], e = 0..3.
// SCHED: what keeps the fragment reads and the matrix instructions of a half step apart.  One run, 8192 x 4096 x 32768,
// TFLOP/s of the three products (row x row, column x row, column x column order), each DMA split as below:
//   0 nothing            1258  1278  1080
//   1 raised priority    1210  1236  1221
//   2 scheduling fence   1184  1306  1200
enum GtSched { GT_PLAIN = 0, GT_PRIO = 1, GT_FENCE = 2 };

template <int BA, int BB, int WA, int WB, bool TA, bool TB, int STAGES, int SCHED, int BK = GT_BK>
struct GtTile {
    static constexpr int NW = WA * WB, NTHR = 64 * NW;
    static constexpr int NA = BA / WA / 16, NB = BB / WB / 16;
    using SA = GtStage<BA, NW, TA, BK>;
    using SB = GtStage<BB, NW, TB, BK>;
    static constexpr int STAGE_BYTES = SA::BYTES + SB::BYTES;
    static constexpr int LDS_BYTES = STAGES * STAGE_BYTES;
    static constexpr int P = SA::P + SB::P;
    static_assert(NA >= 1 && NB >= 1 && LDS_BYTES <= 159 * 1024, "tile");

    // per_half(k, bv): called with the B fragments of every 32-deep half step (k counts from k0)
    template <typename F>
    static __device__ __forceinline__ void run(const GtOperand& A, const GtOperand& B, int a0, int b0, int k0, int k1,
                                               char* smem, f32x4 (&acc)[NA][NB], F&& per_half) {
        auto zero = [](f32x4 (&c)[NA][NB]) { clear(c); };
        if (BB <= 128 && A.once) run_from<true>(A, B, a0, b0, k0, k1, smem, acc, zero, per_half);
        else run_from<false>(A, B, a0, b0, k0, k1, smem, acc, zero, per_half);
    }
    static __device__ __forceinline__ void clear(f32x4 (&c)[NA][NB]) {
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) c[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    // init(acc): what the sums start from, called while the first steps are on their way
    // two loops: a branch at every issue cost the tiles of 128 rows 2 %
    template <bool ONCE, typename I, typename F>
    static __device__ __forceinline__ void run_from(const GtOperand& A, const GtOperand& B, int a0, int b0, int k0, int k1,
                                               char* smem, f32x4 (&acc)[NA][NB], I&& init, F&& per_half) {
        const int lane = threadIdx.x & 63;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wa = wave % WA, wb = wave / WA;
        SA sa; SB sb;
        sa.init(A, a0, k0, k1, wave, lane);
        sb.init(B, b0, k0, k1, wave, lane);
        GtFrag<BA, TA> fa; GtFrag<BB, TB> fb;
        fa.init(wa * (BA / WA), lane);
        fb.init(wb * (BB / WB), lane);
        const unsigned lds0 = (unsigned)(unsigned long)(__attribute__((address_space(3))) char*)smem;
        const int nsteps = (k1 - k0 + BK - 1) / BK;
#pragma unroll
        for (int d = 0; d < STAGES - 1; ++d) {
            sa.template issue<ONCE>(lds0 + d * STAGE_BYTES, wave);
            sb.issue(lds0 + d * STAGE_BYTES + SA::BYTES, wave);
        }
        init(acc);
        int cur = 0, nxt = STAGES - 1;
        for (int s = 0; s < nsteps; ++s) {
            // this wave's share of step s has landed and its reads of the buffer that is refilled below have returned;
            // the barrier makes both true of every wave
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * P) : "memory");
            // A's DMA here, B's between the half steps: issued together (eight instructions on a full queue) they held up
            // the first fragment reads of the step; 4 - 9 % on all three products
            sa.template issue<ONCE>(lds0 + nxt * STAGE_BYTES, wave);
            const char* ta = smem + cur * STAGE_BYTES;
            const char* tb = ta + SA::BYTES;
#pragma unroll
            for (int kk = 0; kk < BK / 32; ++kk) {
                bf16x8_t av[NA], bv[NB];
#pragma unroll
                for (int i = 0; i < NA; ++i) av[i] = fa.load(ta, i, kk, wa * (BA / WA / 16));
#pragma unroll
                for (int j = 0; j < NB; ++j) bv[j] = fb.load(tb, j, kk, wb * (BB / WB / 16));
                if (SCHED == GT_FENCE) __builtin_amdgcn_sched_barrier(0);
                if (SCHED == GT_PRIO) __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int i = 0; i < NA; ++i)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av[i], bv[j], acc[i][j], 0, 0, 0);
                if (SCHED == GT_PRIO) __builtin_amdgcn_s_setprio(0);
                per_half(s * BK + kk * 32, bv);
                if (kk == 0) sb.issue(lds0 + nxt * STAGE_BYTES + SA::BYTES, wave);
            }
            if (++cur == STAGES) cur = 0;
            if (++nxt == STAGES) nxt = 0;
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // LDS is free for the epilogue
    }
};

// Blocks are numbered so that one XCD (hardware index = id % 8, each with its own L2) works on neighbouring tiles: it
// owns a contiguous share of a linear order that walks the reduction's splits, inside a split strips `gb` tiles wide in
// b, a outermost inside a strip.  (Split outermost: an XCD then reads its slice of both operands once.  With the splits
// in the grid's y the input gradient of 1237 x 776 x 30011 took 96 us instead of 73.)
struct GtMap { int na, nb, ns, gb; };
__device__ __forceinline__ bool gt_map(const GtMap& m, int id, int& ta, int& tb, int& split) {
    const int tiles = m.na * m.nb, total = tiles * m.ns;
    const int per = (total + 7) >> 3;
    int lin = (id & 7) * per + (id >> 3);
    if ((id >> 3) >= per || lin >= total) return false;
    split = lin / tiles;
    lin -= split * tiles;
    const int strip = lin / (m.na * m.gb);
    const int w = min(m.gb, m.nb - strip * m.gb);
    const int in = lin - strip * m.na * m.gb;
    ta = in / w;
    tb = strip * m.gb + in % w;
    return true;
}

// ---- host side
static inline GtMap gt_make_map(int na, int nb, int ns, int gb) {
    GtMap m; m.na = na; m.nb = nb; m.ns = ns; m.gb = gb < nb ? gb : nb;
    return m;
}
static inline unsigned gt_grid(const GtMap& m) { return (unsigned)(((long)m.na * m.nb * m.ns + 7) / 8 * 8); }
// gt_map counts in int, and the runtime takes a launch's threads modulo 2^32 without an error; `more`: blocks beside the tiles
static inline bool gt_map_ok(const GtMap& m, int threads, long more = 0) {
    return ((long)m.na * m.nb * m.ns + 8 + more) * threads < (1L << 32);
}

// dynamic LDS above 64 KiB has to be asked for, once per kernel and device
template <auto Kern>
static int gt_lds(size_t bytes) {
    constexpr int MOST = 159 * 1024;           // a kilobyte is left for a kernel's static LDS
    if (bytes > MOST) return -2;
    if (bytes <= 64 * 1024) return 0;
    static std::atomic<unsigned long> done{0};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return -8;
    const unsigned long bit = 1ul << (dev & 63);
    if (done.load() & bit) return 0;
    if (hipFuncSetAttribute((const void*)Kern, hipFuncAttributeMaxDynamicSharedMemorySize, MOST) != hipSuccess) return -8;
    done.fetch_or(bit);
    return 0;
}
static inline int gt_launched() { return hipGetLastError() == hipSuccess ? 0 : -9; }
