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
                codes[i] = make_uint2(o[0], o[1]);
                if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
            }
        }
    }
}

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
            if (i < n8) y[i] = pack8(f);
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
struct Wg8Args {
    GtOperand x, dy;                 // column order over the rows: [R][K], [R][Op]
    int R, K, O;
    int nsplit, per_split;           // rows per split, a multiple of 64
    float* dw; float* db;            // final, or slabs [nsplit][O][K] / [nsplit][O]
    GtMap map;
};

template <int BA, int BB, int WA, int WB, int STAGES>
__global__ __launch_bounds__(64 * WA * WB, (BA * BB >= 65536 ? 2 : 1)) void dense_wgrad8_kernel(const Wg8Args a) {
    using T = GtTile<BA, BB, WA, WB, true, true, STAGES, GT_PRIO>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int ta, tb, split;
    if (!gt_map(a.map, blockIdx.x, ta, tb, split)) return;
    const int k0 = ta * BA, o0 = tb * BB;
    const int r0 = split * a.per_split, r1 = min(r0 + a.per_split, a.R);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const int wa = wave % WA, wb = wave / WA;
    const bool do_db = ta == 0 && wa == 0 && a.db;
    f32x4 acc[T::NA][T::NB], bacc = {0.f, 0.f, 0.f, 0.f};
    static_assert(T::NB <= 4, "rows of the bias accumulator");
    T::run(a.x, a.dy, k0, o0, r0, r1, smem, acc, [&](int, const bf16x8_t (&bv)[T::NB]) {
        if (do_db) {                 // db: one more product per fragment j, against a fragment whose row 4 j is ones
#pragma unroll
            for (int j = 0; j < T::NB; ++j) {
                const short one = fr == 4 * j ? 0x3f80 : 0;
                const s16x8 ones = {one, one, one, one, one, one, one, one};
                bacc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, ones), bv[j], bacc, 0, 0, 0);
            }
        }
    });
    float* dw = a.dw + (long)split * a.O * a.K;
    float* db = a.db ? a.db + (long)split * a.O : nullptr;
    const int wk = k0 + wa * (BA / WA) + 4 * fq, wo = o0 + wb * (BB / WB) + fr;
#pragma unroll
    for (int j = 0; j < T::NB; ++j) {
        const int o = wo + 16 * j;
        if (o >= a.O) continue;
        if (do_db && fq == j) db[o] = bacc[0];
#pragma unroll
        for (int i = 0; i < T::NA; ++i) {
            const int k = wk + 16 * i;
            if (k >= a.K) continue;
            const f32x4 d = acc[i][j];
            *(float4*)(dw + (long)o * a.K + k) = make_float4(d[0], d[1], d[2], d[3]);
        }
    }
}

// sums of the row splits, in split order
__global__ __launch_bounds__(256) void wgrad8_finish_kernel(const float* __restrict__ slab, float* __restrict__ out,
                                                            long n, int nsplit) {
    for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += gridDim.x * 256L) {
        float s = 0.f;
        int k = 0;
        for (; k + 3 < nsplit; k += 4) {
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = slab[(long)(k + u) * n + i];
#pragma unroll
            for (int u = 0; u < 4; ++u) s += v[u];
        }
        for (; k < nsplit; ++k) s += slab[(long)k * n + i];
        out[i] = s;
    }
}

// ------------------------------------------------------------------------------------------------ host side
static int a8_grid(long n8) {
    const long b = (n8 + 1023) / 1024;                       // four 8-element units per thread
    return (int)(b < 1 ? 1 : (b > 8192 ? 8192 : b));
}

DDL_API int ddl_pack8(const void* x, void* codes, void* scales, long n, hipStream_t s) {
    if (n <= 0 || (n & 7)) return -1;
    pack8_kernel<<<a8_grid(n / 8), 256, 0, s>>>((const uint4*)x, (uint2*)codes, (uint8_t*)scales, n / 8);
    return gt_launched();
}

DDL_API int ddl_unpack8(const void* codes, const void* scales, void* y, long n, hipStream_t s) {
    if (n <= 0 || (n & 7)) return -1;
    unpack8_kernel<<<a8_grid(n / 8), 256, 0, s>>>((const uint2*)codes, (const uint8_t*)scales, (uint4*)y, n / 8);
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

template <int BA, int BB, int WA, int WB, int STAGES>
static int launch_wgrad8(Wg8Args& a, hipStream_t s) {
    using T = GtTile<BA, BB, WA, WB, true, true, STAGES, GT_PRIO>;
    constexpr auto kern = dense_wgrad8_kernel<BA, BB, WA, WB, STAGES>;
    if (int rc = gt_lds<kern>(T::LDS_BYTES)) return rc;
    a.map = gt_make_map((a.K + BA - 1) / BA, (a.O + BB - 1) / BB, a.nsplit, 4);
    kern<<<gt_grid(a.map), T::NTHR, T::LDS_BYTES, s>>>(a);
    return gt_launched();
}

// x [R][K], dy [R][Op]; tile: 0 = 256 x 256, 1 = 128 x 128, 2 = 64 x 64.  `slab_w` / `slab_b` hold the row splits' partial sums.
DDL_API int ddl_dense_wgrad8(const void* x, const void* dy, int R, int K, int Op, int O, int nsplit, int per_split,
                             float* dw, float* db, float* slab_w, float* slab_b, int tile, hipStream_t s) {
    if (R <= 0 || K <= 0 || (K & 7) || (Op & 7) || O <= 0 || O > Op || nsplit < 1 || (per_split & 63) ||
        (long)nsplit * per_split < R || (long)(nsplit - 1) * per_split >= R || (nsplit > 1 && (!slab_w || (db && !slab_b))) ||
        (long)K * 128 >= (1L << 31) || (long)Op * 128 >= (1L << 31)) return -1;
    Wg8Args a;
    a.x = {(const bf16_t*)x, K, K}; a.dy = {(const bf16_t*)dy, Op, Op};
    a.R = R; a.K = K; a.O = O; a.nsplit = nsplit; a.per_split = per_split;
    a.dw = nsplit > 1 ? slab_w : dw;
    a.db = nsplit > 1 ? (db ? slab_b : nullptr) : db;
    int rc;
    switch (tile) {
        case 0: rc = launch_wgrad8<256, 256, 2, 4, 2>(a, s); break;
        case 1: rc = launch_wgrad8<128, 128, 2, 2, 2>(a, s); break;
        case 2: rc = launch_wgrad8<64, 64, 2, 2, 4>(a, s); break;
        default: return -4;
    }
    if (rc == 0 && nsplit > 1) {
        const long n = (long)O * K, nb = (n + 255) / 256;
        wgrad8_finish_kernel<<<(int)(nb > 4096 ? 4096 : nb), 256, 0, s>>>(slab_w, dw, n, nsplit);
        if (db) wgrad8_finish_kernel<<<(O + 255) / 256, 256, 0, s>>>(slab_b, db, O, nsplit);
        rc = gt_launched();
    }
    return rc;
}
