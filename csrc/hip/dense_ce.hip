// Dense(K -> V) + softmax cross entropy for any number of classes: loss, row losses and the gradients of x, w and b
// without ever holding the logits [N][V].
//
//   z = x w^T + b      lse_r = log sum_v e^{z_rv}      row_r = lse_r - z_{r,label}      loss = mean over labelled rows
//   dl = (softmax(z) - onehot) / count                  dx = dl w      dw = dl^T x      db = sum_r dl
//
// Three matrix products, 6 N K V operations, no recomputation.  Rows are taken in pieces whose workspace (2 bytes per
// row and class) is bounded by the caller; scoring keeps nothing at all.
//
//  1. `ce_logits`: z tile = w x^T on the matrix cores; the epilogue turns it into E = 2^{z log2(e) - c} and per row and
//     wave tile the sum of the fp32 E.  E is stored in bf16 (the precision a bf16 gradient of the logits would have).
//     c is 0 whenever the tile's largest exponent lies in [-64, 64]: bf16 has the exponent range of fp32, so a common
//     reference of 0 loses nothing, and 2^64 times 2^20 classes times the weights stays far inside fp32.  Only outside
//     that range does a tile take its own maximum.
//  2. `ce_rows`, one block per row: the row's reference (0, or the largest c), S = sum_v E, the row loss, and
//       g = 1 / (S count),   E[label] = -(1 - p_label) S   (so that g E = dl holds for every class),   x' = bf16(g x).
//     A tile whose own c differs from the row's is rescaled here by a power of two; with logits of ordinary size no
//     tile is.  Dividing by S through g instead of rewriting E saves a pass over the piece (2 x 2 bytes per element,
//     20 % of the step at K = 1024).
//  3. `ce_dx`: dx = g (E w), split over the classes when the tiles of [N][K] do not fill the chip.
//  4. `ce_dw`: dw = E^T x', and db = E^T g out of the same fragments (g as two bf16 terms, hi + lo).
//
// Rows whose label is negative take no part: E = 0, x' = 0, dx = 0 whatever their x holds.
// Every sum has a fixed order: the results of two calls are the same bits.
#include "gemm_tile.h"

#define CE_LOG2E 1.44269504088896340736f
#define CE_LN2 0.69314718055994530942f

struct CeRow { float g; float live; };

// ------------------------------------------------------------------------------------------------ 1. logits
struct CeLogitsArgs {
    GtOperand w, x;                  // row order: [V][K], [N][K]
    const float* bias; const long* labels;
    int N, V, K, Vp;                 // Vp: pitch of E, columns V .. Vp are zero-filled (Vp % 64 == 0)
    bf16_t* E;                       // [N][Vp] or nullptr (scoring)
    float2* stats; int nst;          // [N][nst] (c, sum) per wave tile
    float* zt;                       // [N] logit of the label
    const long* labels_all; int n_all; float* count;      // block 0 counts the labelled rows of the whole batch
    GtMap map;
};

template <int BA, int BB, int WA, int WB, int STAGES, bool STORE>
__global__ __launch_bounds__(64 * WA * WB, (BA * BB >= 65536 ? 2 : 1)) void ce_logits_kernel(const CeLogitsArgs a) {
    using T = GtTile<BA, BB, WA, WB, false, false, STAGES>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x;
    if (blockIdx.x == 0 && a.count) {
        int c = 0;
        for (int i = tid; i < a.n_all; i += T::NTHR) c += a.labels_all[i] >= 0;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
        int* red = (int*)smem;
        if ((tid & 63) == 0) red[tid >> 6] = c;
        __syncthreads();
        if (tid == 0) {
            int t = 0;
            for (int w = 0; w < T::NW; ++w) t += red[w];
            *a.count = (float)(t > 0 ? t : 1);
        }
        __syncthreads();
    }
    int ta, tb;
    if (!gt_map(a.map, blockIdx.x, ta, tb)) return;
    const int v0 = ta * BA, r0 = tb * BB;
    f32x4 acc[T::NA][T::NB];
    T::run(a.w, a.x, v0, r0, 0, a.K, smem, acc, [](int, const bf16x8_t (&)[T::NB]) {});

    const int lane = tid & 63, wave = tid >> 6, fr = lane & 15, fq = lane >> 4;
    const int wa = wave % WA, wb = wave / WA;
    const int wv = v0 + wa * (BA / WA), wr = r0 + wb * (BB / WB);
    float bias[T::NA][4];
#pragma unroll
    for (int i = 0; i < T::NA; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int v = wv + 16 * i + 4 * fq + e;
            bias[i][e] = v < a.V ? (a.bias ? a.bias[v] : 0.f) : -INFINITY;
        }
    constexpr int PITCH = BA * 2 + 16;
    char* lrow = smem + (size_t)(wb * (BB / WB)) * PITCH + wa * (BA / WA) * 2;
#pragma unroll
    for (int j = 0; j < T::NB; ++j) {
        const int r = wr + 16 * j + fr;
        const long lab = r < a.N ? a.labels[r] : -1;
        const bool live = (unsigned long)lab < (unsigned long)a.V;
        const int lrel = live ? (int)lab - wv - 4 * fq : -1;
        float zt = 0.f, m = -INFINITY;
        bool mine = false;
#pragma unroll
        for (int i = 0; i < T::NA; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float z = acc[i][j][e] + bias[i][e];
                const bool hit = lrel == 16 * i + e;
                zt = hit ? z : zt;
                mine |= hit;
                acc[i][j][e] = z;
                m = fmaxf(m, z);
            }
        if (mine) a.zt[r] = zt;
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        // the tile's reference, in powers of two (m: fmaxf drops NaNs; a NaN logit still reaches the sum below)
        const float m2 = m * CE_LOG2E;
        float c = 0.f;
        if (fabsf(m2) > 64.f && fabsf(m2) < INFINITY) c = rintf(m2);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < T::NA; ++i) {
            float e4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                e4[e] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], CE_LOG2E, -c));
                if (!live) e4[e] = 0.f;
                s += e4[e];
            }
            if (STORE)
                *(uint2*)(lrow + (16 * j + fr) * PITCH + (16 * i + 4 * fq) * 2) =
                    make_uint2(pack2bf(e4[0], e4[1]), pack2bf(e4[2], e4[3]));
        }
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (fq == 0 && r < a.N) a.stats[(long)r * a.nst + ta * WA + wa] = make_float2(c, s);
    }
    if (!STORE) return;
    __syncthreads();
    // E tile: 16-byte stores along the classes
    constexpr int CPR = BA / 8;
    for (int u = tid; u < BB * CPR; u += T::NTHR) {
        const int row = u / CPR, c8 = u % CPR;
        const int r = r0 + row, v = v0 + c8 * 8;
        if (r < a.N && v < a.Vp) *(uint4*)(a.E + (long)r * a.Vp + v) = *(const uint4*)(smem + row * PITCH + c8 * 16);
    }
}

// ------------------------------------------------------------------------------------------------ 2. rows
struct CeRowsArgs {
    const float2* stats; int nst; int wave_cols;      // classes per stats entry
    const float* zt; const long* labels; const float* count;
    int N, V, K, Vp;
    bf16_t* E; const bf16_t* x; bf16_t* xs;           // xs = bf16(g x)
    float* rows; float* g; bf16_t* g2; int g2_pitch;  // g2[0] + g2[1] = g in two bf16 terms
};

__device__ __forceinline__ float ce_block_max(float v, float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) r = fmaxf(r, red[w]);
    __syncthreads();
    return r;
}
__device__ __forceinline__ float ce_block_sum(float v, float* red) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) r += red[w];
    __syncthreads();
    return r;
}
// 2^d for whole d, exact (0 below the normal range: such a term is 2^-126 of the row's largest)
__device__ __forceinline__ float ce_pow2(float d) { return d < -126.f ? 0.f : ldexpf(1.f, (int)d); }

// loss of a row from its reference, its sum and its label's logit
__device__ __forceinline__ float ce_row_loss(float cref, float S, float zt) {
    const float lse = __logf(S) + cref * CE_LN2;
    return lse < INFINITY ? lse - zt : NAN;
}

template <bool GRAD>
__global__ __launch_bounds__(256) void ce_rows_kernel(const CeRowsArgs a) {
    __shared__ float red[4];
    const int r = blockIdx.x, tid = threadIdx.x;
    const long lab = a.labels[r];
    const bool live = (unsigned long)lab < (unsigned long)a.V;
    if (!live) {
        if (tid == 0) a.rows[r] = lab < 0 ? 0.f : NAN;        // a label past the last class is an error, not padding
        if (GRAD) {
            if (tid == 0) { a.g[r] = 0.f; a.g2[r] = 0; a.g2[a.g2_pitch + r] = 0; }
            for (int k = tid * 8; k < a.K; k += 256 * 8) *(uint4*)(a.xs + (long)r * a.K + k) = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    const float2* st = a.stats + (long)r * a.nst;
    float cref = -INFINITY;
    for (int t = tid; t < a.nst; t += 256) {
        const float2 v = st[t];
        if (v.y != 0.f) cref = fmaxf(cref, v.x);
    }
    cref = ce_block_max(cref, red);
    if (cref == -INFINITY) cref = 0.f;                        // no class left: S = 0
    float S = 0.f;
    int other = 0;                                            // a tile with a reference of its own
    for (int t = tid; t < a.nst; t += 256) {
        const float2 v = st[t];
        if (v.y == 0.f) continue;
        S += v.x == cref ? v.y : v.y * ce_pow2(v.x - cref);
        other |= v.x != cref;
    }
    S = ce_block_sum(S, red);
    const float zt = a.zt[r];
    const float loss = ce_row_loss(cref, S, zt);
    if (tid == 0) a.rows[r] = loss;
    if (!GRAD) return;
    bf16_t* E = a.E + (long)r * a.Vp;
    if (__syncthreads_or(other)) {                            // bring those tiles to the row's reference
        for (int t = 0; t < a.nst; ++t) {
            const float2 v = st[t];
            if (v.y == 0.f || v.x == cref) continue;
            const float f = ce_pow2(v.x - cref);
            const int v1 = min((t + 1) * a.wave_cols, a.V);
            for (int c = t * a.wave_cols + tid; c < v1; c += 256) E[c] = f2bf(bf2f(E[c]) * f);
        }
        __syncthreads();                                      // the label's entry is written below
    }
    // no class left (S = 0) or an infinite logit: the softmax does not exist and the row's gradient is NaN
    const float g = (S > 0.f && S < INFINITY) ? 1.f / (S * *a.count) : NAN;
    if (tid == 0) {
        E[lab] = f2bf(expm1f(-loss) * S);                     // -(1 - p) S
        a.g[r] = g;
        const bf16_t hi = f2bf(g);
        a.g2[r] = hi;
        a.g2[a.g2_pitch + r] = f2bf(g - bf2f(hi));
    }
    for (int k = tid * 8; k < a.K; k += 256 * 8) {
        float f[8];
        unpack8(*(const uint4*)(a.x + (long)r * a.K + k), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= g;
        *(uint4*)(a.xs + (long)r * a.K + k) = pack8(f);
    }
}

// mean of the row losses over the labelled rows, fp64 in a fixed order
__global__ __launch_bounds__(1024) void ce_mean_kernel(const float* rows, const float* count, int N, float* loss) {
    __shared__ double red[16];
    double s = 0.0;
    for (int i = threadIdx.x; i < N; i += 1024) s += (double)rows[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < 16; ++w) t += red[w];
        *loss = (float)(t / (double)*count);
    }
}

// ------------------------------------------------------------------------------------------------ 3. dx
struct CeDxArgs {
    GtOperand w, e;                  // w column order over the classes ([V][K], columns K), E row order [N][Vp]
    int N, V, K;
    int nsplit, per_split;           // classes per split (a multiple of 64)
    const float* g; bf16_t* dx; float* slab;      // slab [nsplit][N][K] when nsplit > 1
    GtMap map;
};

template <int BA, int BB, int WA, int WB, int STAGES>
__global__ __launch_bounds__(64 * WA * WB, (BA * BB >= 65536 ? 2 : 1)) void ce_dx_kernel(const CeDxArgs a) {
    using T = GtTile<BA, BB, WA, WB, true, false, STAGES>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int ta, tb;
    if (!gt_map(a.map, blockIdx.x, ta, tb)) return;
    const int k0 = ta * BA, r0 = tb * BB;
    const int v0 = blockIdx.y * a.per_split, v1 = min(v0 + a.per_split, a.V);
    f32x4 acc[T::NA][T::NB];
    T::run(a.w, a.e, k0, r0, v0, v1, smem, acc, [](int, const bf16x8_t (&)[T::NB]) {});
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const int wk = k0 + (wave % WA) * (BA / WA) + 4 * fq, wr = r0 + (wave / WA) * (BB / WB) + fr;
#pragma unroll
    for (int j = 0; j < T::NB; ++j) {
        const int r = wr + 16 * j;
        if (r >= a.N) continue;
        const float g = a.g[r];
#pragma unroll
        for (int i = 0; i < T::NA; ++i) {
            const int k = wk + 16 * i;
            if (k >= a.K) continue;
            const f32x4 d = acc[i][j];
            if (a.slab) {
                *(float4*)(a.slab + ((long)blockIdx.y * a.N + r) * a.K + k) = make_float4(d[0], d[1], d[2], d[3]);
            } else {
                uint2 o = make_uint2(pack2bf(d[0] * g, d[1] * g), pack2bf(d[2] * g, d[3] * g));
                if (g == 0.f) o = make_uint2(0, 0);
                *(uint2*)(a.dx + (long)r * a.K + k) = o;
            }
        }
    }
}

__global__ __launch_bounds__(256) void ce_dx_finish_kernel(const float* __restrict__ slab, const float* __restrict__ g,
                                                           bf16_t* __restrict__ dx, int N, int K, int nsplit) {
    const long MK = (long)N * K;
    for (long i = (blockIdx.x * 256L + threadIdx.x) * 4; i < MK; i += gridDim.x * 1024L) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        int k = 0;
        for (; k + 3 < nsplit; k += 4) {                       // four loads in flight, added in split order
            float4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = *(const float4*)(slab + (long)(k + u) * MK + i);
#pragma unroll
            for (int u = 0; u < 4; ++u) { s.x += v[u].x; s.y += v[u].y; s.z += v[u].z; s.w += v[u].w; }
        }
        for (; k < nsplit; ++k) {
            const float4 v = *(const float4*)(slab + (long)k * MK + i);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        const float gr = g[i / K];
        uint2 o = make_uint2(pack2bf(s.x * gr, s.y * gr), pack2bf(s.z * gr, s.w * gr));
        if (gr == 0.f) o = make_uint2(0, 0);
        *(uint2*)(dx + i) = o;
    }
}

// ------------------------------------------------------------------------------------------------ 4. dw, db
struct CeDwArgs {
    GtOperand xs, e;                 // column order over the rows: x' [N][K] (columns K), E [N][Vp] (columns Vp)
    int N, V, K;
    const bf16_t* g2; int g2_pitch;  // zero behind row N up to a multiple of 64
    const float* acc_w; const float* acc_b;       // earlier row pieces ([V][K], [V]) or nullptr
    void* dw; void* db; int out_bf16;             // this piece's output: fp32 (possibly the accumulator) or bf16
    GtMap map;
};

template <int BA, int BB, int WA, int WB, int STAGES>
__global__ __launch_bounds__(64 * WA * WB, (BA * BB >= 65536 ? 2 : 1)) void ce_dw_kernel(const CeDwArgs a) {
    using T = GtTile<BA, BB, WA, WB, true, true, STAGES>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int ta, tb;
    if (!gt_map(a.map, blockIdx.x, ta, tb)) return;
    const int k0 = ta * BA, v0 = tb * BB;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const int wa = wave % WA, wb = wave / WA;
    const bool do_db = ta == 0 && wa == 0;                     // wave-uniform
    f32x4 acc[T::NA][T::NB], bacc[T::NB];
#pragma unroll
    for (int j = 0; j < T::NB; ++j) bacc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    // db = E^T g: one more matrix instruction per B fragment against a fragment whose rows 0 and 1 are g's two terms
    T::run(a.xs, a.e, k0, v0, 0, a.N, smem, acc, [&](int k, const bf16x8_t (&bv)[T::NB]) {
        if (do_db) {
            const s16x8 gv = *(const s16x8*)(a.g2 + (fr & 1) * a.g2_pitch + k + 8 * fq);
            const s16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
            const bf16x8_t ga = __builtin_bit_cast(bf16x8_t, fr < 2 ? gv : z);
#pragma unroll
            for (int j = 0; j < T::NB; ++j) bacc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ga, bv[j], bacc[j], 0, 0, 0);
        }
    });
    const int wk = k0 + wa * (BA / WA) + 4 * fq, wv = v0 + wb * (BB / WB) + fr;
#pragma unroll
    for (int j = 0; j < T::NB; ++j) {
        const int v = wv + 16 * j;
        if (v >= a.V) continue;
        if (do_db && fq == 0 && a.db) {
            float b = bacc[j][0] + bacc[j][1];
            if (a.acc_b) b += a.acc_b[v];
            if (a.out_bf16) ((bf16_t*)a.db)[v] = f2bf(b);
            else ((float*)a.db)[v] = b;
        }
#pragma unroll
        for (int i = 0; i < T::NA; ++i) {
            const int k = wk + 16 * i;
            if (k >= a.K) continue;
            f32x4 d = acc[i][j];
            const long o = (long)v * a.K + k;
            if (a.acc_w) {
                const float4 p = *(const float4*)(a.acc_w + o);
                d[0] += p.x; d[1] += p.y; d[2] += p.z; d[3] += p.w;
            }
            if (a.out_bf16) *(uint2*)((bf16_t*)a.dw + o) = make_uint2(pack2bf(d[0], d[1]), pack2bf(d[2], d[3]));
            else *(float4*)((float*)a.dw + o) = make_float4(d[0], d[1], d[2], d[3]);
        }
    }
}

// ------------------------------------------------------------------------------------------------ host side
template <int BA, int BB, int WA, int WB, int STAGES, bool STORE>
static int launch_logits(CeLogitsArgs& a, hipStream_t s) {
    using T = GtTile<BA, BB, WA, WB, false, false, STAGES>;
    size_t lds = T::LDS_BYTES, out = (size_t)BB * (BA * 2 + 16);
    if (STORE && out > lds) lds = out;
    constexpr auto kern = ce_logits_kernel<BA, BB, WA, WB, STAGES, STORE>;
    if (int rc = gt_lds<kern>(lds)) return rc;
    a.nst = (a.V + BA - 1) / BA * WA;
    a.map = gt_make_map((a.V + BA - 1) / BA, (a.N + BB - 1) / BB, 8);
    kern<<<gt_grid(a.map), T::NTHR, lds, s>>>(a);
    return gt_launched();
}

// tile: 0 = 256 classes x 256 rows, 1 = 128 x 128, 2 = 128 x 32, 3 = 32 x 32
DDL_API int ddl_ce_stats_cols(int V, int tile) {
    const int cols = tile == 3 ? 16 : (tile == 2 ? 32 : (tile == 1 ? 64 : 128));
    const int ba = tile == 3 ? 32 : (tile == 0 ? 256 : 128);
    return (V + ba - 1) / ba * (ba / cols);
}

DDL_API int ddl_ce_logits(const void* w, const void* x, const float* bias, const long* labels, int N, int V, int K,
                          int Vp, void* E, void* stats, float* zt, const long* labels_all, int n_all, float* count,
                          int tile, hipStream_t s) {
    if (N <= 0 || V <= 0 || K <= 0 || (K & 7) || (Vp & 63) || Vp < V || (long)K * 512 >= (1L << 31)) return -1;
    CeLogitsArgs a;
    a.w = {(const bf16_t*)w, K, V}; a.x = {(const bf16_t*)x, K, N};
    a.bias = bias; a.labels = labels; a.N = N; a.V = V; a.K = K; a.Vp = Vp;
    a.E = (bf16_t*)E; a.stats = (float2*)stats; a.zt = zt;
    a.labels_all = labels_all; a.n_all = n_all; a.count = count;
    switch (tile) {
        case 0: return E ? launch_logits<256, 256, 2, 4, 2, true>(a, s) : launch_logits<256, 256, 2, 4, 2, false>(a, s);
        case 1: return E ? launch_logits<128, 128, 2, 2, 2, true>(a, s) : launch_logits<128, 128, 2, 2, 2, false>(a, s);
        case 2: return E ? launch_logits<128, 32, 4, 1, 4, true>(a, s) : launch_logits<128, 32, 4, 1, 4, false>(a, s);
        case 3: return E ? launch_logits<32, 32, 2, 1, 4, true>(a, s) : launch_logits<32, 32, 2, 1, 4, false>(a, s);
        default: return -4;
    }
}

DDL_API int ddl_ce_rows(const void* stats, int nst, int wave_cols, const float* zt, const long* labels,
                        const float* count, int N, int V, int K, int Vp, void* E, const void* x, void* xs, float* rows,
                        float* g, void* g2, int g2_pitch, hipStream_t s) {
    if (N <= 0 || V <= 0 || K <= 0 || (K & 7) || nst <= 0) return -1;
    CeRowsArgs a;
    a.stats = (const float2*)stats; a.nst = nst; a.wave_cols = wave_cols; a.zt = zt; a.labels = labels; a.count = count;
    a.N = N; a.V = V; a.K = K; a.Vp = Vp; a.E = (bf16_t*)E; a.x = (const bf16_t*)x; a.xs = (bf16_t*)xs; a.rows = rows;
    a.g = g; a.g2 = (bf16_t*)g2; a.g2_pitch = g2_pitch;
    if (E) ce_rows_kernel<true><<<N, 256, 0, s>>>(a);
    else ce_rows_kernel<false><<<N, 256, 0, s>>>(a);
    return gt_launched();
}

DDL_API int ddl_ce_mean(const float* rows, const float* count, int N, float* loss, hipStream_t s) {
    if (N <= 0) return -1;
    ce_mean_kernel<<<1, 1024, 0, s>>>(rows, count, N, loss);
    return gt_launched();
}

template <int BA, int BB, int WA, int WB, int STAGES>
static int launch_dx(CeDxArgs& a, hipStream_t s) {
    using T = GtTile<BA, BB, WA, WB, true, false, STAGES>;
    constexpr auto kern = ce_dx_kernel<BA, BB, WA, WB, STAGES>;
    if (int rc = gt_lds<kern>(T::LDS_BYTES)) return rc;
    a.map = gt_make_map((a.K + BA - 1) / BA, (a.N + BB - 1) / BB, 8);
    kern<<<dim3(gt_grid(a.map), a.nsplit), T::NTHR, T::LDS_BYTES, s>>>(a);
    return gt_launched();
}

// tile: 0 = 256 features x 256 rows, 1 = 128 x 128, 2 = 128 x 32
DDL_API int ddl_ce_dx(const void* w, const void* E, int N, int V, int K, int Vp, int nsplit, int per_split,
                      const float* g, void* dx, float* slab, int tile, hipStream_t s) {
    if (N <= 0 || V <= 0 || K <= 0 || (K & 7) || (Vp & 63) || Vp < V || nsplit < 1 || (per_split & 63) ||
        (long)nsplit * per_split < V || (long)(nsplit - 1) * per_split >= V || (nsplit > 1 && !slab) ||
        (long)Vp * 512 >= (1L << 31) || (long)K * 128 >= (1L << 31)) return -1;
    CeDxArgs a;
    a.w = {(const bf16_t*)w, K, K}; a.e = {(const bf16_t*)E, Vp, N};
    a.N = N; a.V = V; a.K = K; a.nsplit = nsplit; a.per_split = per_split; a.g = g; a.dx = (bf16_t*)dx;
    a.slab = nsplit > 1 ? slab : nullptr;
    int rc;
    switch (tile) {
        case 0: rc = launch_dx<256, 256, 2, 4, 2>(a, s); break;
        case 1: rc = launch_dx<128, 128, 2, 2, 2>(a, s); break;
        case 2: rc = launch_dx<128, 32, 4, 1, 4>(a, s); break;
        default: return -4;
    }
    if (rc == 0 && nsplit > 1) {
        const long MK = (long)N * K, nb = (MK + 1023) / 1024;
        ce_dx_finish_kernel<<<(int)(nb > 2048 ? 2048 : nb), 256, 0, s>>>(slab, g, (bf16_t*)dx, N, K, nsplit);
    }
    return rc;
}

template <int BA, int BB, int WA, int WB, int STAGES>
static int launch_dw(CeDwArgs& a, hipStream_t s) {
    using T = GtTile<BA, BB, WA, WB, true, true, STAGES>;
    constexpr auto kern = ce_dw_kernel<BA, BB, WA, WB, STAGES>;
    if (int rc = gt_lds<kern>(T::LDS_BYTES)) return rc;
    a.map = gt_make_map((a.K + BA - 1) / BA, (a.V + BB - 1) / BB, 4);
    kern<<<gt_grid(a.map), T::NTHR, T::LDS_BYTES, s>>>(a);
    return gt_launched();
}

// tile: 0 = 256 features x 256 classes, 1 = 128 x 128
DDL_API int ddl_ce_dw(const void* xs, const void* E, int N, int V, int K, int Vp, const void* g2, int g2_pitch,
                      const float* acc_w, const float* acc_b, void* dw, void* db, int out_bf16, int tile,
                      hipStream_t s) {
    if (N <= 0 || V <= 0 || K <= 0 || (K & 7) || (Vp & 63) || Vp < V || g2_pitch < (N + 63) / 64 * 64 ||
        (long)Vp * 128 >= (1L << 31) || (long)K * 128 >= (1L << 31)) return -1;
    CeDwArgs a;
    a.xs = {(const bf16_t*)xs, K, K}; a.e = {(const bf16_t*)E, Vp, Vp};
    a.N = N; a.V = V; a.K = K; a.g2 = (const bf16_t*)g2; a.g2_pitch = g2_pitch;
    a.acc_w = acc_w; a.acc_b = acc_b; a.dw = dw; a.db = db; a.out_bf16 = out_bf16;
    switch (tile) {
        case 0: return launch_dw<256, 256, 2, 4, 2>(a, s);
        case 1: return launch_dw<128, 128, 2, 2, 2>(a, s);
        default: return -4;
    }
}
