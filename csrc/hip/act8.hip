// Activations kept in 8 bits between the forward and the backward pass, and the backward kernels that read them.
//
// Format: 32 consecutive elements (memory order) share a power-of-two scale 2^e, e the smallest integer from -119 to 121
// with max |x| <= 127 2^e; a code is x 2^-e rounded to the nearest integer (ties to even) -- +-1 where that would be 0
// for an x that is not 0, +-127 where it would be more (the largest bf16 number only).  33 bytes instead of 64.
//   * Integers with a block scale: the error is at most half a step, 2^-7 .. 2^-8 of the block's largest value; e4m3
//     in the same 8 bits has three mantissa bits, ~5 x the rms error on activations.
//   * Power-of-two scales: code * 2^e is exact in bf16 (7 bits times a power of two), so what the backward pass reads
//     is the same number in every kernel, and x 2^-e is exact, so packing is reproducible to the bit.
//   * No non-zero value becomes zero: the sign survives, so act'(y) of relu / leaky relu is exact from the code.
//   * A block that holds a NaN or an infinity cannot be represented: scale byte 255, all of it reads as NaN.
#include "gemm_tile.h"

#define A8_MIN 8              // smallest scale byte, e + 127 (e = -119: code * 2^e stays a normal number)
#define A8_MAX 248            // 127 * 2^121 is finite, 64 * 2^122 is not
#define A8_BAD 255

// 2^e of a scale byte; 255 -> NaN
__device__ __forceinline__ float a8_scale(unsigned byte) {
    return byte == A8_BAD ? NAN : __uint_as_float(byte << 23);
}
// eight codes (two dwords) to fp32 values
__device__ __forceinline__ void a8_unpack8(uint2 c, float s, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = (float)(int)(signed char)(c.x >> (8 * i)) * s;
        f[4 + i] = (float)(int)(signed char)(c.y >> (8 * i)) * s;
    }
}

// ------------------------------------------------------------------------------------------------ pack / unpack
// A lane packs 8 elements, four lanes share a block; n8 = elements / 8.
// NT: the output goes past the caches.  For tensors that the last level cache (256 MiB) cannot hold until they are read again
// (there and back, 4096 x 32 x 32 x 64: 339 -> 324 us, 16384 x 8192: 161 -> 150); smaller ones stay where the next kernel
// finds them (a weight gradient of 16384 x 4096 x 4096 whose unpacked x did not: 444 -> 452).
typedef unsigned int a8_u32x2 __attribute__((ext_vector_type(2)));
constexpr long A8_CACHED8 = (256L << 20) / 16;
template <bool NT>
__global__ __launch_bounds__(256) void pack8_kernel(const uint4* __restrict__ x, uint2* __restrict__ codes,
                                                    uint8_t* __restrict__ scales, long n8) {
    constexpr int U = 4;
    const long stride = (long)gridDim.x * 256;
    // every lane of a four-lane block stays in the loop together: i0 runs over multiples of 256 per block
    for (long i0 = blockIdx.x * 256L; i0 < n8; i0 += stride * U) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long i = i0 + u * stride + threadIdx.x;
            v[u] = i < n8 ? x[i] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long i = i0 + u * stride + threadIdx.x;
            const unsigned w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
            unsigned m = 0;                                  // largest |x| as bf16 bits (monotone as integers)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                m = max(m, w[k] & 0x7fffu);
                m = max(m, (w[k] >> 16) & 0x7fffu);
            }
            m = max(m, (unsigned)__shfl_xor((int)m, 1, 64));
            m = max(m, (unsigned)__shfl_xor((int)m, 2, 64));
            // |x| = (128 + mant) 2^(ef - 134): half of 128 + mant fits in 127 unless mant is 127
            const int ef = m >> 7, mant = m & 127;
            const int byte = m >= 0x7f80u ? A8_BAD : min(A8_MAX, max(A8_MIN, ef - 6 + (mant == 127)));
            const float inv = m >= 0x7f80u ? 0.f : __uint_as_float((unsigned)(254 - byte) << 23);
            unsigned o[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const unsigned h = (k & 1) ? w[k >> 1] & 0xffff0000u : w[k >> 1] << 16;
                // round to integer by adding 1.5 * 2^23: the low byte of the sum is the two's complement code
                const float t = __builtin_amdgcn_fmed3f(__uint_as_float(h) * inv, -127.f, 127.f);
                unsigned q = __float_as_uint(t + 12582912.f) & 0xffu;
                if (q == 0 && (h << 1) != 0) q = (h >> 31) ? 0xffu : 1u;
                o[k >> 2] |= q << (8 * (k & 3));
            }
            if (m >= 0x7f80u) o[0] = o[1] = 0;
            if (i < n8) {
                if (NT) __builtin_nontemporal_store((a8_u32x2){o[0], o[1]}, (a8_u32x2*)(codes + i));
                else codes[i] = make_uint2(o[0], o[1]);
                if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
            }
        }
    }
}

template <bool NT>
__global__ __launch_bounds__(256) void unpack8_kernel(const uint2* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                      uint4* __restrict__ y, long n8) {
    constexpr int U = 4;
    const long stride = (long)gridDim.x * 256;
    for (long i0 = blockIdx.x * 256L + threadIdx.x; i0 < n8; i0 += stride * U) {
        uint2 c[U];
        unsigned b[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long i = min(i0 + u * stride, n8 - 1);
            c[u] = codes[i];
            b[u] = scales[i >> 2];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long i = i0 + u * stride;
            float f[8];
            a8_unpack8(c[u], a8_scale(b[u]), f);
            if (i >= n8) continue;
            const uint4 o = pack8(f);
            if (NT) __builtin_nontemporal_store((gt_u32x4){o.x, o.y, o.z, o.w}, (gt_u32x4*)(y + i));
            else y[i] = o;
        }
    }
}

// ------------------------------------------------------------------------------------------------ activation backward
// dx = dy act'(y), y from its codes: 5.03 instead of 6 bytes per element
template <int K>
__global__ __launch_bounds__(256) void act_bwd8_kernel(const uint4* __restrict__ dy, const uint2* __restrict__ codes,
                                                       const uint8_t* __restrict__ scales, uint4* __restrict__ dx,
                                                       long n8, int act, float alpha) {
    constexpr int U = 4;
    const long stride = (long)gridDim.x * 256;
    for (long i0 = blockIdx.x * 256L + threadIdx.x; i0 < n8; i0 += stride * U) {
        uint4 d[U];
        uint2 c[U];
        unsigned b[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long i = min(i0 + u * stride, n8 - 1);
            d[u] = dy[i];
            c[u] = codes[i];
            b[u] = scales[i >> 2];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long i = i0 + u * stride;
            float f[8], g[8];
            a8_unpack8(c[u], a8_scale(b[u]), f);
            unpack8(d[u], g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float t = act_grad_y_k<K>(f[e], act, alpha);
                g[e] *= f[e] == f[e] ? t : NAN;              // (a comparison would turn a NaN into a slope)
            }
            if (i < n8) dx[i] = pack8(g);
        }
    }
}

// ------------------------------------------------------------------------------------------------ Dense weight gradient
// dw[o][k] = sum_r dy[r][o] xh[r][k],   db[o] = sum_r dy[r][o]
//
// Both operands are read with the reduction (rows) outermost: dy by LDS-DMA in column order (gemm_tile.h), x from its codes
// through registers -- 8 codes and their scale byte become 8 bf16 values, exactly, on the way into the same LDS layout.
// Codes of step s + 2 are fetched, those of s + 1 converted, between the two halves of step s; the conversion (2.5 vector
// instructions per element) hides behind the other wave's matrix instructions.  The products are exact and the sums fp32.
struct Wg8Args {
    const signed char* codes; const uint8_t* scales; GtOperand dy;      // [R][K], one scale per 32 codes; [R][Op]
    GtOperand x;                     // [R][K] bf16: the codes unpacked beforehand (large products)
    int R, K, O;
    int nsplit, per_split;           // rows per split, a multiple of 64
    float* dw; float* db;            // final, or slabs [nsplit][O][K] / [nsplit][O]
    GtMap map;
};

template <int T, int NTHR>
struct A8Stage {
    static constexpr int U = T * GT_BK / 8 / NTHR, UPR = T / 8;      // 8-code units per thread, units per row
    static constexpr int BYTES = T * GT_BK * 2;
    static_assert(U >= 1 && UPR * GT_BK == U * NTHR, "tile");
    typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
    unsigned off[U];                 // code offset of unit u in the step's 64 x K codes
    const signed char* c; const uint8_t* s;
    long ld;
    int left;
    u32x2_t code[U];
    unsigned scale[U];

    __device__ __forceinline__ void init(const Wg8Args& a, int t0, int r0, int r1) {
        ld = a.K;
        left = r1 - r0;
        c = a.codes + (long)r0 * a.K;                        // r0 is a multiple of 64: r0 K is one of 512
        s = a.scales + ((long)r0 * a.K >> 5);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = u * NTHR + threadIdx.x, col = t0 + i % UPR * 8;
            off[u] = col < a.K ? (unsigned)(i / UPR * ld + col) : GT_OOB;
        }
    }
    // the codes of the next step (rows past the end: zeros) into registers
    __device__ __forceinline__ void fetch() {
        const long n = left > 0 ? (left < GT_BK ? left : GT_BK) * ld : 0;
        const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc((void*)c, 0, (int)n, 0x00020000);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)s, 0, (int)((n + 31) >> 5), 0x00020000);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            code[u] = __builtin_amdgcn_raw_buffer_load_b64(rc, off[u], 0, 0);
            // past the last code no scale either: the last block may be a partial one, and marked 255 (NaN) it would reach
            // the features that its unused rest stands for
            scale[u] = __builtin_amdgcn_raw_buffer_load_b8(rs, off[u] < (unsigned)n ? off[u] >> 5 : GT_OOB, 0, 0);
        }
        c += GT_BK * ld;
        s += 2 * ld;
        left -= GT_BK;
    }
    __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = u * NTHR + threadIdx.x, row = i / UPR, slot = i % UPR;
            float f[8];
            a8_unpack8(make_uint2(code[u][0], code[u][1]), a8_scale(scale[u]), f);
            *(uint4*)(tile + row * (T * 2) + (slot ^ (GtStage<T, 1, true>::swz(row) << 1)) * 16) = pack8(f);
        }
    }
};

// db: one more product per dy fragment j, against a fragment whose row 4 j is ones: one accumulator holds all of them
template <int NB>
__device__ __forceinline__ void wg8_ones(const bf16x8_t (&bv)[NB], f32x4& bacc, int fr) {
    static_assert(NB <= 4, "rows of the bias accumulator");
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const short one = fr == 4 * j ? 0x3f80 : 0;
        const s16x8 ones = {one, one, one, one, one, one, one, one};
        bacc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, ones), bv[j], bacc, 0, 0, 0);
    }
}
template <int NA, int NB>
__device__ __forceinline__ void wg8_store(const Wg8Args& a, const f32x4 (&acc)[NA][NB], const f32x4& bacc, bool do_db,
                                          int split, int wk, int wo, int fq) {
    float* dw = a.dw + (long)split * a.O * a.K;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int o = wo + 16 * j;
        if (o >= a.O) continue;
        if (do_db && fq == j) a.db[(long)split * a.O + o] = bacc[0];
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int k = wk + 16 * i;
            if (k >= a.K) continue;
            const f32x4 d = acc[i][j];
            *(float4*)(dw + (long)o * a.K + k) = make_float4(d[0], d[1], d[2], d[3]);
        }
    }
}

template <int BA, int BB, int WA, int WB>
__global__ __launch_bounds__(64 * WA * WB, (BA * BB >= 65536 ? 2 : 1)) void dense_wgrad8_kernel(const Wg8Args a) {
    constexpr int NW = WA * WB, NA = BA / WA / 16, NB = BB / WB / 16;
    using SA = A8Stage<BA, 64 * NW>;
    using SB = GtStage<BB, NW, true>;
    constexpr int STAGE = SA::BYTES + SB::BYTES;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int ta, tb, split;
    if (!gt_map(a.map, blockIdx.x, ta, tb, split)) return;
    const int k0 = ta * BA, o0 = tb * BB;
    const int r0 = split * a.per_split, r1 = min(r0 + a.per_split, a.R);
    const int lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wa = wave % WA, wb = wave / WA;
    const bool do_db = ta == 0 && wa == 0 && a.db;
    const unsigned lds0 = (unsigned)(unsigned long)(__attribute__((address_space(3))) char*)smem;
    SA sa;
    SB sb;
    sa.init(a, k0, r0, r1);
    sb.init(a.dy, o0, r0, r1, wave, lane);
    GtFrag<BA, true> fa;
    GtFrag<BB, true> fb;
    fa.init(wa * (BA / WA), lane);
    fb.init(wb * (BB / WB), lane);
    f32x4 acc[NA][NB], bacc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

    sa.fetch();
    sa.store(smem);
    sa.fetch();
    sb.issue(lds0 + SA::BYTES, wave);
    const int nsteps = (r1 - r0 + GT_BK - 1) / GT_BK;
    for (int st = 0; st < nsteps; ++st) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int cur = (st & 1) * STAGE, nxt = STAGE - cur;
        const char* t = smem + cur;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            bf16x8_t av[NA], bv[NB];
#pragma unroll
            for (int i = 0; i < NA; ++i) av[i] = fa.load(t, i, kk, wa * NA);
#pragma unroll
            for (int j = 0; j < NB; ++j) bv[j] = fb.load(t + SA::BYTES, j, kk, wb * NB);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int i = 0; i < NA; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av[i], bv[j], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_s_setprio(0);
            if (do_db) wg8_ones<NB>(bv, bacc, fr);
            if (kk == 0) {
                sa.store(smem + nxt);
                sa.fetch();
                sb.issue(lds0 + nxt + SA::BYTES, wave);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // the last (empty) fetch has landed
    wg8_store<NA, NB>(a, acc, bacc, do_db, split, k0 + wa * (BA / WA) + 4 * fq, o0 + wb * (BB / WB) + fr, fq);
}

// The same product with x unpacked to bf16 beforehand: both operands by LDS-DMA
template <int BA, int BB, int WA, int WB>
__global__ __launch_bounds__(64 * WA * WB, (BA * BB >= 65536 ? 2 : 1)) void dense_wgrad8_dma_kernel(const Wg8Args a) {
    using T = GtTile<BA, BB, WA, WB, true, true, 2, GT_PRIO>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int ta, tb, split;
    if (!gt_map(a.map, blockIdx.x, ta, tb, split)) return;
    const int k0 = ta * BA, o0 = tb * BB;
    const int r0 = split * a.per_split, r1 = min(r0 + a.per_split, a.R);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const int wa = wave % WA, wb = wave / WA;
    const bool do_db = ta == 0 && wa == 0 && a.db;
    f32x4 acc[T::NA][T::NB], bacc = {0.f, 0.f, 0.f, 0.f};
    T::run(a.x, a.dy, k0, o0, r0, r1, smem, acc, [&](int, const bf16x8_t (&bv)[T::NB]) {
        if (do_db) wg8_ones<T::NB>(bv, bacc, fr);
    });
    wg8_store<T::NA, T::NB>(a, acc, bacc, do_db, split, k0 + wa * (BA / WA) + 4 * fq, o0 + wb * (BB / WB) + fr, fq);
}

// sums of the row splits, in split order: n weight gradients (four per thread), then O bias gradients
__global__ __launch_bounds__(256) void wgrad8_finish_kernel(const float* __restrict__ slab, const float* __restrict__ bslab,
                                                            float* __restrict__ dw, float* __restrict__ db, long n, int O,
                                                            int nsplit) {
    const long t0 = blockIdx.x * 256L + threadIdx.x, stride = gridDim.x * 256L;
    for (long i = t0 * 4; i < n; i += stride * 4) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        int k = 0;
        for (; k + 7 < nsplit; k += 8) {                      // eight loads in flight
            float4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = *(const float4*)(slab + (k + u) * n + i);
#pragma unroll
            for (int u = 0; u < 8; ++u) { s.x += v[u].x; s.y += v[u].y; s.z += v[u].z; s.w += v[u].w; }
        }
        for (; k < nsplit; ++k) {
            const float4 v = *(const float4*)(slab + k * n + i);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        *(float4*)(dw + i) = s;
    }
    for (long i = t0; i < O; i += stride) {
        float s = 0.f;
        for (int k = 0; k < nsplit; ++k) s += bslab[(long)k * O + i];
        db[i] = s;
    }
}

// ------------------------------------------------------------------------------------------------ host side
static int a8_grid(long n8) {
    const long b = (n8 + 1023) / 1024;                       // four 8-element units per thread
    return (int)(b < 1 ? 1 : (b > 8192 ? 8192 : b));
}

DDL_API int ddl_pack8(const void* x, void* codes, void* scales, long n, hipStream_t s) {
    if (n <= 0 || (n & 7)) return -1;
    constexpr auto kern = pack8_kernel<false>, once = pack8_kernel<true>;
    (n / 8 >= A8_CACHED8 ? once : kern)<<<a8_grid(n / 8), 256, 0, s>>>((const uint4*)x, (uint2*)codes, (uint8_t*)scales, n / 8);
    return gt_launched();
}

DDL_API int ddl_unpack8(const void* codes, const void* scales, void* y, long n, hipStream_t s) {
    if (n <= 0 || (n & 7)) return -1;
    constexpr auto kern = unpack8_kernel<false>, once = unpack8_kernel<true>;
    (n / 8 >= A8_CACHED8 ? once : kern)<<<a8_grid(n / 8), 256, 0, s>>>((const uint2*)codes, (const uint8_t*)scales, (uint4*)y, n / 8);
    return gt_launched();
}

DDL_API int ddl_act_bwd8(const void* dy, const void* codes, const void* scales, void* dx, long n, int act, float alpha,
                         hipStream_t s) {
    if (n <= 0 || (n & 7)) return -1;
#define A8_CALL(A) act_bwd8_kernel<A><<<a8_grid(n / 8), 256, 0, s>>>((const uint4*)dy, (const uint2*)codes, \
                                                                    (const uint8_t*)scales, (uint4*)dx, n / 8, act, alpha)
    ACT1_DISPATCH(act, A8_CALL);
#undef A8_CALL
    return gt_launched();
}

template <int BA, int BB, int WA, int WB, bool DMA>
static int launch_wgrad8(Wg8Args& a, hipStream_t s) {
    constexpr auto kern = DMA ? dense_wgrad8_dma_kernel<BA, BB, WA, WB> : dense_wgrad8_kernel<BA, BB, WA, WB>;
    constexpr int lds = 2 * (BA + BB) * GT_BK * 2;
    if (int rc = gt_lds<kern>(lds)) return rc;
    a.map = gt_make_map((a.K + BA - 1) / BA, (a.O + BB - 1) / BB, a.nsplit, 4);
    if (!gt_map_ok(a.map, 64 * WA * WB)) return -1;
    kern<<<gt_grid(a.map), 64 * WA * WB, lds, s>>>(a);
    return gt_launched();
}

// Tile and row splits of a call, by their estimated time: 64-row steps plus a block's start and end in rounds of the blocks
// that share a CU (1000 x 6272 x 128, 196 tiles: one block per CU 15.5 us, 4 splits and as many blocks per CU 18.7), the
// splits' partial sums written and read once, and the unpacking.  Reading the codes in the product saves 3 bytes per element
// of x but costs 2.5 vector instructions per element and output tile (kernels' time: 1000 x 6272 x 128 20 us, unpacked first
// 27; 512 x 1024 x 1024 12 and 16; 4096 x 2048 x 2048 77 and 62; 16384 x 4096 x 4096 854 and 487).
struct Wg8Plan { int tile, ns, per; };                       // tile: see ddl_dense_wgrad8
static Wg8Plan wg8_plan(int R, int K, int O, int force) {
    static const int edge[4] = {64, 128, 128, 256}, fit[4] = {4, 2, 2, 1};      // blocks that share a CU,
    static const double step_us[4][4] = {{0.67, 0.8, 1.06, 1.28}, {1.42, 1.78}, {1.1, 1.2}, {1.75}};      // and a step of so many
    const int steps = (R + 63) / 64;
    Wg8Plan p = {0, 1, steps * 64};
    double best = 0;
    for (int t = 0; t < 4; ++t) {
        if (force >= 0 && t != force) continue;
        const long tiles = (long)((K + edge[t] - 1) / edge[t]) * ((O + edge[t] - 1) / edge[t]);
        for (int want = 1; want <= 64 && (want == 1 || want <= steps / 4); ++want) {
            const int per = (steps + want - 1) / want, ns = (steps + per - 1) / per;
            const long cu = (tiles * ns + 255) / 256, rest = cu % fit[t];
            const double us = (cu / fit[t] * step_us[t][fit[t] - 1] + (rest ? step_us[t][rest - 1] : 0.0)) * (per + 4.0) +
                              (ns > 1 ? 2.5 + ns * 8.0 * O * K / 7e6 : 0.0) +
                              (t >= 2 ? 4.0 + 3.0 * R * K / 4.5e6 : 0.0);
            if (best == 0 || us < best) { best = us; p = {t, ns, per * 64}; }
        }
    }
    return p;
}
// partial sums, 256-byte multiples (the unpacked x follows them)
static long wg8_slabs(const Wg8Plan& p, int K, int O) {
    return p.ns > 1 ? (((long)p.ns * O * K + (long)p.ns * O) * 4 + 255) / 256 * 256 : 0;
}
static bool wg8_unpacks(const Wg8Plan& p) { return p.tile >= 2; }

static bool wg8_range_ok(int R, int K, int Op, int O) {
    return R > 0 && K > 0 && (K & 7) == 0 && Op > 0 && (Op & 7) == 0 && O > 0 && O <= Op && (long)K * 128 < (1L << 31) &&
           (long)Op * 128 < (1L << 31);
}

// Bytes of workspace (the row splits' partial sums; 0: none).  Negative: sizes outside the kernels' range.
DDL_API long ddl_dense_wgrad8_workspace(int R, int K, int Op, int O, int force_tile) {
    if (!wg8_range_ok(R, K, Op, O) || force_tile > 3) return -1;
    const Wg8Plan p = wg8_plan(R, K, O, force_tile);
    return wg8_slabs(p, K, O) + (wg8_unpacks(p) ? 2L * R * K : 0);
}

// codes [R][K] with their scales, dy [R][Op] bf16 -> dw [O][K], db [O] fp32.  Tiles: 0 = 64 x 64 and 1 = 128 x 128 from the
// codes, 2 = 128 x 128 and 3 = 256 x 256 from x unpacked into the workspace; force_tile -1: by the sizes
DDL_API int ddl_dense_wgrad8(const void* codes, const void* scales, const void* dy, int R, int K, int Op, int O, float* dw,
                             float* db, void* ws, long ws_bytes, int force_tile, hipStream_t s) {
    if (!wg8_range_ok(R, K, Op, O) || force_tile > 3) return -1;
    const Wg8Plan p = wg8_plan(R, K, O, force_tile);
    const long n = (long)O * K, slabs = wg8_slabs(p, K, O);
    if (ws_bytes < slabs + (wg8_unpacks(p) ? 2L * R * K : 0)) return -3;
    Wg8Args a;
    a.codes = (const signed char*)codes; a.scales = (const uint8_t*)scales; a.dy = {(const bf16_t*)dy, Op, Op};
    a.R = R; a.K = K; a.O = O; a.nsplit = p.ns; a.per_split = p.per;
    a.dw = p.ns > 1 ? (float*)ws : dw;
    a.db = p.ns > 1 ? (float*)ws + p.ns * n : db;
    a.x = {(const bf16_t*)((char*)ws + slabs), K, K};
    int rc;
    if (wg8_unpacks(p)) {
        rc = ddl_unpack8(codes, scales, (char*)ws + slabs, (long)R * K, s);
        if (rc) return rc;
    }
    switch (p.tile) {
        case 0: rc = launch_wgrad8<64, 64, 2, 2, false>(a, s); break;
        case 1: rc = launch_wgrad8<128, 128, 2, 2, false>(a, s); break;
        case 2: rc = launch_wgrad8<128, 128, 2, 2, true>(a, s); break;
        default: rc = launch_wgrad8<256, 256, 2, 4, true>(a, s);
    }
    if (rc == 0 && p.ns > 1) {
        const long nb = (n + O + 1023) / 1024;
        wgrad8_finish_kernel<<<(int)(nb > 4096 ? 4096 : nb), 256, 0, s>>>(a.dw, a.db, dw, db, n, O, p.ns);
        rc = gt_launched();
    }
    return rc;
}
