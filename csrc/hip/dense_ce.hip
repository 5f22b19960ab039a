// Dense(K -> V) + softmax cross entropy for any number of classes: loss, row losses and the gradients of x, w and b.  The logits
// [N][V] are not kept: scoring keeps a reference and a sum per row and wave tile, a step their exponentials in bf16 (2.15 GB for
// 8192 x 131072: as much as bf16 logits, half of fp32 ones).
//
//   z = x w^T + b      lse_r = log sum_v e^{z_rv}      row_r = lse_r - z_{r,label}      loss = mean over labelled rows
//   dl = (softmax(z) - onehot) / count                  dx = dl w      dw = dl^T x      db = sum_r dl
//
// Three matrix products, 6 N K V operations, no recomputation.  Rows are taken in pieces whose workspace (2 bytes per
// row and class; scoring: 8 per row and wave tile) is bounded by the caller; each piece reads w and writes an fp32 dw once more
// (2048 x 2048 x 32000 in 1, 2, 4, 8 pieces: 733, 897, 1208, 2003 us; 8192 x 4096 x 131072 in 1, 2, 4: 20.5, 21.4, 23.4 ms).
//
//  1. `ce_logits`: z tile = w x^T on the matrix cores; the epilogue turns it into E = 2^{z log2(e) - c} and per row and
//     wave tile the sum of the fp32 E.  E is stored in bf16 (the precision a bf16 gradient of the logits would have).
//     c is 0 whenever the tile's sum lies in [2^-64, 2^64]: bf16 has the exponent range of fp32, so a common reference of 0
//     loses nothing, and 2^64 times 2^20 classes times the weights stays far inside fp32.  Only outside that range does a
//     tile take its own maximum.
//  2. `ce_rows`, one block per row: the row's reference (0, or the largest c), S = sum_v E, the row loss, and
//       g = 1 / (S count),   E[label] = bf16(-(1 - p_label) S)   (g E = dl holds for every class),   x' = bf16(g x).
//     A tile whose own c differs from the row's is rescaled here by a power of two; with logits of ordinary size no
//     tile is.  Dividing by S through g instead of rewriting E saves a pass over the piece (2 x 2 bytes per element,
//     20 % of the step at K = 1024).
//  3. `ce_labels`: with many classes the label's entry -(1 - p) is most of a row's gradient, and so most of what the two
//     roundings (E, x') cost.  The label terms are therefore made exact: what the products get wrong there,
//       dw[label] += -(1 - p)/count x - bf16(..) x',   db[label] and dx alike,
//     is summed per class in row order (ranks counted in `ce_logits`, whose first blocks do nothing else) and added in
//     the products' epilogues.  Measured against 64 bits (8192 x 4096 x 131072, bf16 outputs): dw 0.0027 -> 0.0018 where
//     the output's own rounding is 0.0017.  fp32 outputs show the roundings of the other entries: rms of dw 5e-5 (512 x 1024
//     x 20000) to 4e-4 (1000 x 64 x 128), of db 4e-5 to 1.5e-4.  Both are the price of bf16 matrix operands, 16 x the rate of
//     fp32 ones; the losses carry neither.
//  4. `ce_dx`: dx = g (E w), split over the classes when the tiles of [N][K] do not fill the chip.
//  5. `ce_dw`: dw = E^T x', and db = E^T g out of the same fragments (g as two bf16 terms, hi + lo).
//
// Rows whose label is negative take no part: E = 0, x' = 0, dx = 0 whatever their x holds.
// Every sum has a fixed order: the results of two calls are the same bits.
#include "gemm_tile.h"

#define CE_LOG2E 1.44269504088896340736f
#define CE_LN2 0.69314718055994530942f
#define CE_LN2_REST -2.12194440054690583e-4f      // log 2 - 355 / 512
constexpr long CE_CACHE = 256L << 20;      // the last level cache, shared by the whole chip
constexpr int CE_NT = 2;                   // a raw buffer store's policy: non-temporal

// What the later kernels need of a row: the gradient of its logits is g E, plus `rest` in the label's class.
struct CeRow { float g, hi, tg, rest; int label; int pad[3]; };      // hi = E[label], tg = dl[label], rest = tg - hi g
static_assert(sizeof(CeRow) == 32, "two 16-byte loads");

// ------------------------------------------------------------------------------------------------ 1. logits
struct CeLogitsArgs {
    GtOperand w, x;                  // row order: [V][K], [N][K]
    const float* bias; const long* labels;
    int N, V, K, Vp;                 // Vp: pitch of E, columns V .. Vp are zero-filled (Vp % 64 == 0)
    bf16_t* E;                       // [N][Vp] or nullptr (scoring)
    float2* stats; int nst;          // [N][nst] (c, sum) per wave tile
    float* zt;                       // [N] logit of the label
    const long* labels_all; int n_all; float* count;      // block 0 counts the labelled rows of the whole batch
    int* order;                      // [N] rows sorted by (label, row), unlabelled ones last (training)
    int2* slot;                      // [V] reset to -1 (training)
    int nrank;                       // blocks in front of the tiles that do the counting and ranking (a multiple of 8)
    GtMap map;
};

// Block `b` of the first nrank: the ranks of rows 32 b .. 32 b + 31 among all labels (stable, so the order is unique)
// and, in block 0, the number of labelled rows.  N^2 comparisons against labels in LDS: 3 us for 8192 rows.
#define CE_RANK_ROWS 32
template <int NTHR>
__device__ __forceinline__ void ce_rank(const CeLogitsArgs& a, char* smem, int b) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (b == 0 && a.count) {
        int c = 0;
        constexpr int U = 8;                                  // loads in flight
        for (int i = tid; i < a.n_all; i += NTHR * U) {
            long l[U];
#pragma unroll
            for (int u = 0; u < U; ++u) l[u] = a.labels_all[min(i + u * NTHR, a.n_all - 1)];
#pragma unroll
            for (int u = 0; u < U; ++u) c += l[u] >= 0 && i + u * NTHR < a.n_all;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
        int* red = (int*)smem;
        if (lane == 0) red[wave] = c;
        __syncthreads();
        if (tid == 0) {
            int t = 0;
            for (int w = 0; w < NTHR / 64; ++w) t += red[w];
            *a.count = (float)(t > 0 ? t : 1);
        }
        __syncthreads();
    }
    const int r0 = b * CE_RANK_ROWS;
    if (!a.order || r0 >= a.N) return;
    int* lab = (int*)smem;                                   // CE_MAX_ROWS entries at most: 32 KiB
    constexpr int U = 8;
    for (int i = tid; i < a.N; i += NTHR * U) {
        long l[U];
#pragma unroll
        for (int u = 0; u < U; ++u) l[u] = a.labels[min(i + u * NTHR, a.N - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * NTHR < a.N) lab[i + u * NTHR] = (unsigned long)l[u] < (unsigned long)a.V ? (int)l[u] : 0x7fffffff;
    }
    __syncthreads();
    constexpr int PER = CE_RANK_ROWS / (NTHR / 64);           // rows of a wave, all compared with a label read once
    int mine[PER], c[PER];
#pragma unroll
    for (int q = 0; q < PER; ++q) {
        mine[q] = lab[min(r0 + wave * PER + q, a.N - 1)];
        c[q] = 0;
    }
    // rows in front of the block's count when their label is not larger, rows behind it when it is smaller (r0 is a multiple
    // of 32: only the 64 rows around it need the row number itself)
    const int lo = r0 & ~63, hi = lo + 64;
    for (int i = lane; i < lo; i += 64) {
        const int l = lab[i];
#pragma unroll
        for (int q = 0; q < PER; ++q) c[q] += l <= mine[q];
    }
    if (lo + lane < a.N) {
        const int i = lo + lane, l = lab[i];
#pragma unroll
        for (int q = 0; q < PER; ++q) c[q] += l < mine[q] || (l == mine[q] && i < r0 + wave * PER + q);
    }
    for (int i = hi + lane; i < a.N; i += 64) {
        const int l = lab[i];
#pragma unroll
        for (int q = 0; q < PER; ++q) c[q] += l < mine[q];
    }
#pragma unroll
    for (int q = 0; q < PER; ++q) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) c[q] += __shfl_xor(c[q], o, 64);
        if (lane == 0 && r0 + wave * PER + q < a.N) a.order[c[q]] = r0 + wave * PER + q;
    }
}

template <int BA, int BB, int WA, int WB, int STAGES, bool STORE>
__global__ __launch_bounds__(64 * WA * WB, (BA * BB >= 65536 ? 2 : 1)) void ce_logits_kernel(const CeLogitsArgs a) {
    using T = GtTile<BA, BB, WA, WB, false, false, STAGES, GT_PLAIN>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x;
    if ((int)blockIdx.x < a.nrank) {
        ce_rank<T::NTHR>(a, smem, blockIdx.x);
        return;
    }
    int ta, tb, one;
    if (!gt_map(a.map, blockIdx.x - a.nrank, ta, tb, one)) return;
    const int v0 = ta * BA, r0 = tb * BB;
    if (STORE && tb == 0)
        for (int i = tid; i < BA; i += T::NTHR)
            if (v0 + i < a.V) a.slot[v0 + i] = make_int2(-1, -1);
    // the tile's biases (in powers of two; no class there: -inf, E = 0) and labels, one of each per thread: fetched here, their
    // latency is the loop's, and handed round through LDS behind it (read where they are used: 512 x 1024 x 50021 71 us, 66 so,
    // 2048 x 512 x 32000 99 and 87; all of a lane's own in registers across the loop: 74 and 101)
    static_assert(BA <= T::NTHR && BB <= T::NTHR, "tile");
    const float my_bias = tid < BA && v0 + tid < a.V && a.bias ? a.bias[v0 + tid] : 0.f;
    const long my_label = tid < BB && r0 + tid < a.N ? a.labels[r0 + tid] : -1;
    f32x4 acc[T::NA][T::NB];
    T::run(a.w, a.x, v0, r0, 0, a.K, smem, acc, [](int, const bf16x8_t (&)[T::NB]) {});
    constexpr int PITCH = BA * 2 + 16;
    float* tile_bias = (float*)(smem + (STORE ? BB * PITCH : 0));      // behind E's patch, in the stages' place
    int* tile_label = (int*)(tile_bias + BA);
    if (tid < BA) tile_bias[tid] = v0 + tid < a.V ? my_bias * CE_LOG2E : -INFINITY;
    if (tid < BB) tile_label[tid] = (unsigned long)my_label < (unsigned long)a.V ? (int)my_label : -1;
    __syncthreads();

    const int lane = tid & 63, wave = tid >> 6, fr = lane & 15, fq = lane >> 4;
    const int wa = wave % WA, wb = wave / WA;
    const int wv = v0 + wa * (BA / WA), wr = r0 + wb * (BB / WB);
    // The epilogue is as long as eight steps of the loop if every element pays for a maximum, a label test and a live test
    // (512 x 1024 x 50021: 75 us with them, 68 without), so the common case does a multiply-add, an exponential and a
    // sum per element; which wave tiles need more shows in the sum and in two votes.
    f32x4 bias[T::NA];
#pragma unroll
    for (int i = 0; i < T::NA; ++i) bias[i] = *(const f32x4*)(tile_bias + wa * (BA / WA) + 16 * i + 4 * fq);
    char* lrow = smem + (size_t)(wb * (BB / WB)) * PITCH + wa * (BA / WA) * 2;
#pragma unroll
    for (int j = 0; j < T::NB; ++j) {
        const int r = wr + 16 * j + fr;
        const int lab = tile_label[wb * (BB / WB) + 16 * j + fr];
        const bool live = lab >= 0;
        const int lrel = live ? lab - wv - 4 * fq : -1;           // the label's position among this lane's classes
        if (__any((unsigned)lrel < (unsigned)(BA / WA) && (lrel & 15) < 4)) {
            float zt = 0.f;
            bool mine = false;
#pragma unroll
            for (int i = 0; i < T::NA; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool hit = lrel == 16 * i + e;
                    zt = hit ? acc[i][j][e] : zt;
                    mine |= hit;
                }
            if (mine) a.zt[r] = zt + (a.bias ? a.bias[lab] : 0.f);
        }
        float s = 0.f, c = 0.f;
        auto pass = [&](float cref) {
            s = 0.f;
#pragma unroll
            for (int i = 0; i < T::NA; ++i) {
                float e4[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    e4[e] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], CE_LOG2E, bias[i][e]) - cref);
                    s += e4[e];
                }
                if (STORE)
                    *(uint2*)(lrow + (16 * j + fr) * PITCH + (16 * i + 4 * fq) * 2) =
                        make_uint2(pack2bf(e4[0], e4[1]), pack2bf(e4[2], e4[3]));
            }
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
        };
        pass(0.f);
        if (__any(live && !(s >= 0x1p-64f && s <= 0x1p64f))) {
            // some row's largest exponent is far from 0 (or its classes are masked, or a logit is not finite): it takes its own
            // maximum as reference (m: fmaxf drops NaNs; a NaN logit still reaches the sum)
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < T::NA; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) m = fmaxf(m, fmaf(acc[i][j][e], CE_LOG2E, bias[i][e]));
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            if (!(s >= 0x1p-64f && s <= 0x1p64f) && fabsf(m) < INFINITY) c = rintf(m);
            pass(c);
        }
        if (__any(!live)) {          // rows without a label (their x may hold anything) take no part
            if (!live) s = 0.f;
            if (STORE && !live)
#pragma unroll
                for (int i = 0; i < T::NA; ++i)
                    *(uint2*)(lrow + (16 * j + fr) * PITCH + (16 * i + 4 * fq) * 2) = make_uint2(0, 0);
        }
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
    const bf16_t* w; const float* bias;
    int N, V, K, Vp;
    bf16_t* E; const bf16_t* x; bf16_t* xs;           // xs = bf16(g x)
    float* rows; CeRow* row; bf16_t* g2; int g2_pitch;      // g2[0] + g2[1] = g in two bf16 terms, zero behind row N
    float* loss;                     // scoring a single row: its loss is the mean
};

// 2^d for whole d, exact (0 below the normal range: such a term is 2^-126 of the row's largest)
__device__ __forceinline__ float ce_pow2(float d) { return d < -126.f ? 0.f : ldexpf(1.f, (int)d); }

// Loss of a row from its reference, its sum and its label's logit: log(S 2^cref) - zt.  With S = m 2^e the whole powers of two
// leave as (e + cref) log 2 in two terms (355 / 512 and the rest, Cody and Waite: the first product is exact below 2^15), so
// the difference is rounded at its own size, not at that of the logarithm (rows of 9 x 1958 x 156: 1.1e-6 -> 7e-7 off).
__device__ __forceinline__ float ce_row_loss(float cref, float S, float zt) {
    if (!(S >= 0x1p-126f && S < INFINITY)) {                  // no class left, or a logit that is not finite
        const float lse = __logf(S) + cref * CE_LN2;
        return lse < INFINITY ? lse - zt : NAN;
    }
    const unsigned b = __float_as_uint(S) - 0x3f350000u;      // m in [0.707, 1.414)
    const float m = __uint_as_float((b & 0x7fffffu) + 0x3f350000u), n = (float)((int)b >> 23) + cref;
    return fmaf(n, 355.f / 512.f, -zt) + (__logf(m) + n * CE_LN2_REST);
}

// The label's logit once more, by a tree: the products' chain of K / 32 additions is most of a row loss' error (9 x 1958 x 156:
// 7e-7, so 2e-7, plain fp32 3e-7; 300 x 4096 x 3000: 5e-7, 0.9e-7, 1e-6; 1 us of a step).  This thread's part of x_r w_label
__device__ __forceinline__ float ce_label_dot(const CeRowsArgs& a, int r, long lab, int t, int threads) {
    float d = 0.f;
    for (int k = t * 8; k < a.K; k += threads * 8) {
        float f[8], g[8];
        unpack8(*(const uint4*)(a.x + (long)r * a.K + k), f);
        unpack8(*(const uint4*)(a.w + lab * a.K + k), g);
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = fmaf(f[e], g[e], f[e + 4] * g[e + 4]);
        d += (p[0] + p[1]) + (p[2] + p[3]);
    }
    return d;
}
// it takes the place of the tiles' value z, in the sum S as well: a label that is most of S has to cancel
__device__ __forceinline__ void ce_refine(float cref, float& S, float& z, float better) {
    const float d = z - better;
    if (fabsf(d) < 0.5f) {                                    // finite, both of them
        S -= __builtin_amdgcn_exp2f(fmaf(better, CE_LOG2E, -cref)) * expm1f(d);
        z = better;
    }
}

// (reference, sum) of a row's tiles: running maximum and sum, entries with sum 0 (no class) left out
struct CeSum {
    float c, s, lo;                                           // lo: the smallest reference seen
    __device__ __forceinline__ void add(float oc, float os, float olo) {
        if (os == 0.f) return;
        const float m = fmaxf(c, oc);
        s = (s == 0.f ? 0.f : (c == m ? s : s * ce_pow2(c - m))) + (oc == m ? os : os * ce_pow2(oc - m));
        c = m;
        lo = fminf(lo, olo);
    }
    __device__ __forceinline__ void wave() {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) add(__shfl_xor(c, o, 64), __shfl_xor(s, o, 64), __shfl_xor(lo, o, 64));
    }
};

template <bool GRAD, int NTHR>
__global__ __launch_bounds__(NTHR) void ce_rows_kernel(const CeRowsArgs a) {
    __shared__ float red[NTHR / 64][4];
    const int r = blockIdx.x, tid = threadIdx.x;
    if (GRAD && r == 0)
        for (int i = a.N + tid; i < a.g2_pitch; i += NTHR) a.g2[i] = a.g2[a.g2_pitch + i] = 0;
    const long lab = a.labels[r];
    const bool live = (unsigned long)lab < (unsigned long)a.V;
    if (!live) {
        const float v = lab < 0 ? 0.f : NAN;                  // a label past the last class is an error, not padding
        if (tid == 0) {
            a.rows[r] = v;
            if (a.loss) *a.loss = v;
        }
        if (GRAD) {
            if (tid == 0) { a.row[r] = CeRow{0.f, 0.f, 0.f, 0.f, -1, {0, 0, 0}}; a.g2[r] = 0; a.g2[a.g2_pitch + r] = 0; }
            for (int k = tid * 8; k < a.K; k += NTHR * 8) *(uint4*)(a.xs + (long)r * a.K + k) = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    const float2* st = a.stats + (long)r * a.nst;
    float dot = ce_label_dot(a, r, lab, tid, NTHR), zt = a.zt[r];
    CeSum t = {-INFINITY, 0.f, INFINITY};
    for (int i = tid; i < a.nst; i += NTHR) {
        const float2 v = st[i];
        t.add(v.x, v.y, v.x);
    }
    t.wave();
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
    if ((tid & 63) == 0) { red[tid >> 6][0] = t.c; red[tid >> 6][1] = t.s; red[tid >> 6][2] = t.lo; red[tid >> 6][3] = dot; }
    __syncthreads();
    t = {red[0][0], red[0][1], red[0][2]};
    dot = red[0][3];
    for (int w = 1; w < NTHR / 64; ++w) {
        t.add(red[w][0], red[w][1], red[w][2]);
        dot += red[w][3];
    }
    const float cref = t.s == 0.f ? 0.f : t.c;                // no class left: S = 0
    float S = t.s;
    ce_refine(cref, S, zt, a.bias ? dot + a.bias[lab] : dot);
    const float loss = ce_row_loss(cref, S, zt);
    if (tid == 0) {
        a.rows[r] = loss;
        if (a.loss) *a.loss = loss;
    }
    if (!GRAD) return;
    bf16_t* E = a.E + (long)r * a.Vp;
    // bring the tiles with a reference of their own to the row's.  One statistic after the other, and only rows that have such a
    // tile (a logit past 44, a stretch of classes switched off by a finite value) pay: 512 x 1024 x 50021 with a twentieth of
    // the classes at -1e9 258 us, at -inf 211; 4096 x 2048 x 32768 1522 and 1414
    if (t.s != 0.f && t.lo != cref) {
        for (int i = 0; i < a.nst; ++i) {
            const float2 v = st[i];
            if (v.y == 0.f || v.x == cref) continue;
            const float f = ce_pow2(v.x - cref);
            const int v1 = min((i + 1) * a.wave_cols, a.V);
            for (int c = i * a.wave_cols + tid; c < v1; c += NTHR) E[c] = f2bf(bf2f(E[c]) * f);
        }
        __syncthreads();                                      // the label's entry is written below
    }
    // no class left (S = 0) or an infinite logit: the softmax does not exist and the row's gradient is NaN
    const float g = (S > 0.f && S < INFINITY) ? 1.f / (S * *a.count) : NAN;
    if (tid == 0) {
        const float q = expm1f(-loss);                        // -(1 - p)
        const bf16_t el = f2bf(q * S), hi = f2bf(g), lo = f2bf(g - bf2f(hi));
        E[lab] = el;
        const float tg = q / *a.count;
        a.row[r] = CeRow{g, bf2f(el), tg, tg - bf2f(el) * g, (int)lab, {0, 0, 0}};
        a.g2[r] = hi;
        a.g2[a.g2_pitch + r] = lo;
    }
    for (int k = tid * 8; k < a.K; k += NTHR * 8) {
        float f[8];
        unpack8(*(const uint4*)(a.x + (long)r * a.K + k), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= g;
        *(uint4*)(a.xs + (long)r * a.K + k) = pack8(f);
    }
}

// mean of the row losses over the labelled rows, fp64 in a fixed order; one block of NTHR threads
template <int NTHR>
__device__ __forceinline__ void ce_mean(const float* rows, const float* count, int N, float* loss, double (&red)[NTHR / 64]) {
    double s = 0.0;
    constexpr int U = 8;                                      // loads in flight (one at a time: 56 us of 8000 x 64 x 65)
    for (int i = threadIdx.x; i < N; i += NTHR * U) {
        float v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = rows[min(i + u * NTHR, N - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u) s += i + u * NTHR < N ? (double)v[u] : 0.0;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < NTHR / 64; ++w) t += red[w];
        *loss = (float)(t / (double)*count);
    }
}
__global__ __launch_bounds__(1024) void ce_mean_kernel(const float* rows, const float* count, int N, float* loss) {
    __shared__ double red[16];
    ce_mean<1024>(rows, count, N, loss, red);
}

// Scoring a few rows of few tiles: row losses (a wave each) and their mean in one block instead of two launches.  With
// 2048 statistics for each of 32 rows the one block took 40 us and the two launches 6; it is for short ones only.
#define CE_FEW_STATS 256
#define CE_FEW_ROWS 32
__global__ __launch_bounds__(1024) void ce_score_few_kernel(const CeRowsArgs a, float* loss) {
    const int lane = threadIdx.x & 63;
    for (int r = threadIdx.x >> 6; r < a.N; r += 16) {
        const long lab = a.labels[r];
        float v = lab < 0 ? 0.f : NAN;
        if ((unsigned long)lab < (unsigned long)a.V) {
            const float2* st = a.stats + (long)r * a.nst;
            float dot = ce_label_dot(a, r, lab, lane, 64), zt = a.zt[r];
            CeSum t = {-INFINITY, 0.f, INFINITY};
            for (int i = lane; i < a.nst; i += 64) {
                const float2 p = st[i];
                t.add(p.x, p.y, p.x);
            }
            t.wave();
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
            const float cref = t.s == 0.f ? 0.f : t.c;
            ce_refine(cref, t.s, zt, a.bias ? dot + a.bias[lab] : dot);
            v = ce_row_loss(cref, t.s, zt);
        }
        if (lane == 0) a.rows[r] = v;
    }
    __syncthreads();
    __shared__ double red[16];
    ce_mean<1024>(a.rows, a.count, a.N, loss, red);
}

// ------------------------------------------------------------------------------------------------ 3. label terms
// Rows in sorted order, in windows of 64 positions: the rows of one class inside a window are a run; its first position i
// sums it (ascending) into L[i].  slot[class] holds its first and its last run; those between start at the windows'.
// Windows bound a block's work whatever the labels are (8000 rows, 1000 of them of one class: 340 us with a block per class,
// 20 so).  256 threads.  Block 0, in front of them all, takes the mean of the row losses.
#define CE_RUN 64
struct CeLabelsArgs {
    const CeRow* row; const int* order; const bf16_t* x; const bf16_t* xs; int N, K;
    int2* slot; float* L; float* Lb;                         // [V], [N][K], [N]
    const float* rows_all; const float* count; int n_all; float* loss;      // loss nullptr: not the last piece
};

// LDS of a block (the caller's: static LDS here would be every dx tile's, and cost the small ones their second block per CU)
struct CeLabelsLds { union { double mean[4]; struct { float s[256][8]; float b[256]; }; }; };

__device__ __forceinline__ void ce_labels(const CeLabelsArgs& a, int i, int chunk, CeLabelsLds& lds) {
    if (i == 0) {                                             // (the longest block starts first)
        if (a.loss && chunk == 0) ce_mean<256>(a.rows_all, a.count, a.n_all, a.loss, lds.mean);
        return;
    }
    --i;
    const int lab = a.row[a.order[i]].label;
    if (lab < 0) return;
    const bool fresh = i == 0 || a.row[a.order[i - 1]].label != lab;
    if (!fresh && i % CE_RUN != 0) return;
    int width = 8;
    while (width < 256 && width * 8 < a.K) width *= 2;
    const int tid = threadIdx.x, lane = tid & 63, g = tid / width;
    const int k = (chunk * 256 + (tid & (width - 1))) * 8;
    const bool on = k < a.K;
    const int end = min((i / CE_RUN + 1) * CE_RUN, a.N);      // of the window
    const int q = i + lane < end ? a.order[i + lane] : a.order[i];
    const CeRow c = a.row[q];                                 // a lane per row: the loop's loads do not wait for each other
    const unsigned long m = __ballot(i + lane < end && c.label == lab);
    const int n = m == ~0ul ? 64 : __builtin_ctzl(~m);        // the run's rows are the leading lanes
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, b = 0.f;
    // eight features per thread; threads that they leave over share the run's rows: group g of G takes rows g, g + G, ..
    // (a row is 0.6 us of one wave: the whole step of 8000 x 64 x 65 took 123 us with G = 1, 88 so)
    constexpr int U = 4;
    const int G = min(256 / width, (n + U - 1) / U);
    for (int j0 = 0; j0 < n; j0 += U * G) {
        uint4 xv[U], xr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long r = __shfl(q, min(j0 + u * G + g, n - 1), 64);
            xv[u] = *(const uint4*)(a.x + r * a.K + (on ? k : 0));
            xr[u] = *(const uint4*)(a.xs + r * a.K + (on ? k : 0));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * G + g, l = min(j, n - 1);
            const float t = __shfl(c.tg, l, 64), h = __shfl(c.hi, l, 64), rest = __shfl(c.rest, l, 64);
            const float tg = j < n ? t : 0.f, hi = j < n ? h : 0.f;
            b += j < n ? rest : 0.f;
            float fv[8], fr[8];
            unpack8(xv[u], fv);
            unpack8(xr[u], fr);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += fmaf(tg, fv[e], -(hi * fr[e]));
        }
    }
    if (G > 1) {                                              // the groups' sums, in order
#pragma unroll
        for (int e = 0; e < 8; ++e) lds.s[tid][e] = s[e];
        lds.b[tid] = b;
        __syncthreads();
        if (g > 0) return;
        for (int o = tid + width; o < G * width; o += width) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += lds.s[o][e];
            b += lds.b[o];
        }
    }
    if (on && g == 0) {
        float* o = a.L + (long)i * a.K + k;
        *(float4*)o = make_float4(s[0], s[1], s[2], s[3]);
        *(float4*)(o + 4) = make_float4(s[4], s[5], s[6], s[7]);
    }
    if (chunk == 0 && tid == 0) {
        if (fresh) a.slot[lab].x = i;
        a.Lb[i] = b;
        if (end >= a.N || a.row[a.order[end]].label != lab) a.slot[lab].y = i;
    }
}
__global__ __launch_bounds__(256) void ce_labels_kernel(const CeLabelsArgs a) {
    __shared__ CeLabelsLds lds;
    ce_labels(a, blockIdx.x, blockIdx.y, lds);
}

// ------------------------------------------------------------------------------------------------ 4. dx
struct CeDxArgs {
    GtOperand w, e;                  // w column order over the classes ([V][K], columns K), E row order [N][Vp]
    int N, V, K;
    int nsplit, per_split;           // classes per split (a multiple of 64)
    const CeRow* row; bf16_t* dx; float* slab;    // slab [nsplit][N][K] when nsplit > 1
    CeLabelsArgs lab; int ntile, nlab_chunks;     // blocks of 256 threads behind the ntile of the tiles do the label terms
    GtMap map;
};

// dx of four features: g (E w) + rest w[label]; exactly 0 in a row without a label
__device__ __forceinline__ void ce_dx_store(const CeRow& c, const bf16_t* w, int K, int k, const f32x4& d, bf16_t* dx) {
    uint2 o = make_uint2(0, 0);
    if (c.label >= 0) {
        const uint2 wl = *(const uint2*)(w + (long)c.label * K + k);
        const float r0 = fmaf(d[0], c.g, c.rest * __uint_as_float(wl.x << 16));
        const float r1 = fmaf(d[1], c.g, c.rest * __uint_as_float(wl.x & 0xffff0000u));
        const float r2 = fmaf(d[2], c.g, c.rest * __uint_as_float(wl.y << 16));
        const float r3 = fmaf(d[3], c.g, c.rest * __uint_as_float(wl.y & 0xffff0000u));
        o = make_uint2(pack2bf(r0, r1), pack2bf(r2, r3));
    }
    *(uint2*)dx = o;
}

template <int BA, int BB, int WA, int WB, int STAGES>
__global__ __launch_bounds__(64 * WA * WB, (BA * BB >= 65536 ? 2 : 1)) void ce_dx_kernel(const CeDxArgs a) {
    using T = GtTile<BA, BB, WA, WB, true, false, STAGES, GT_FENCE>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    if (T::NTHR == 256 && (int)blockIdx.x >= a.ntile) {
        const int b = blockIdx.x - a.ntile, i = b / a.nlab_chunks;
        ce_labels(a.lab, i, b - i * a.nlab_chunks, *(CeLabelsLds*)smem);
        return;
    }
    int ta, tb, split;
    if (!gt_map(a.map, blockIdx.x, ta, tb, split)) return;
    const int k0 = ta * BA, r0 = tb * BB;
    const int v0 = split * a.per_split, v1 = min(v0 + a.per_split, a.V);
    f32x4 acc[T::NA][T::NB];
    T::run(a.w, a.e, k0, r0, v0, v1, smem, acc, [](int, const bf16x8_t (&)[T::NB]) {});
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const int wk = k0 + (wave % WA) * (BA / WA) + 4 * fq, wr = r0 + (wave / WA) * (BB / WB) + fr;
#pragma unroll
    for (int j = 0; j < T::NB; ++j) {
        const int r = wr + 16 * j;
        if (r >= a.N) continue;
        const CeRow c = a.row[r];
#pragma unroll
        for (int i = 0; i < T::NA; ++i) {
            const int k = wk + 16 * i;
            if (k >= a.K) continue;
            const f32x4 d = acc[i][j];
            if (a.slab) {
                *(float4*)(a.slab + ((long)split * a.N + r) * a.K + k) = make_float4(d[0], d[1], d[2], d[3]);
            } else {
                ce_dx_store(c, a.w.p, a.K, k, d, a.dx + (long)r * a.K + k);
            }
        }
    }
}

// block b of nb (256 threads each)
__device__ __forceinline__ void ce_dx_finish(const float* __restrict__ slab, const CeRow* __restrict__ row,
                                             const bf16_t* __restrict__ w, bf16_t* __restrict__ dx, int N, int K, int nsplit,
                                             int b, int nb) {
    const long MK = (long)N * K;
    for (long i = (b * 256L + threadIdx.x) * 4; i < MK; i += nb * 1024L) {
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
        const int r = (int)(i / K);
        const f32x4 d = {s.x, s.y, s.z, s.w};
        ce_dx_store(row[r], w, K, (int)(i - (long)r * K), d, dx + i);
    }
}
__global__ __launch_bounds__(256) void ce_dx_finish_kernel(const float* __restrict__ slab, const CeRow* __restrict__ row,
                                                           const bf16_t* __restrict__ w, bf16_t* __restrict__ dx, int N,
                                                           int K, int nsplit) {
    ce_dx_finish(slab, row, w, dx, N, K, nsplit, blockIdx.x, gridDim.x);
}

// ------------------------------------------------------------------------------------------------ 5. dw, db
struct CeDwArgs {
    GtOperand xs, e;                 // column order over the rows: x' [N][K] (columns K), E [N][Vp] (columns Vp)
    int N, V, K;
    const bf16_t* g2; int g2_pitch;  // zero behind row N up to a multiple of 64
    const int2* slot; const float* L; const float* Lb;       // the label terms' remainders (ce_labels)
    const float* acc_w; const float* acc_b;       // earlier row pieces ([V][K], [V]) or nullptr
    void* dw; void* db; int out_bf16;             // this piece's output: fp32 (possibly the accumulator) or bf16
    // blocks nv, nv + 1, .. (of the first row of the grid; of 256 threads) finish the splits of dx
    const float* slab; const CeRow* row; const bf16_t* w; bf16_t* dx; int nsplit, nv;
    // tile kernels: the rows in rsplit pieces of rper (a multiple of 64) when there are few tiles; their partial sums go to
    // rslab [rsplit][V][K], [rsplit][V] and ce_dw_finish does the rest
    int rsplit, rper; float* rslab;
    GtMap map;
};

// what the label terms add to four features / the bias of a class: its runs in order (x the first, -1: none; y the last)
__device__ __forceinline__ int ce_run_next(int p) { return (p / CE_RUN + 1) * CE_RUN; }
__device__ __forceinline__ void ce_label_add(const CeDwArgs& a, int2 run, int k, f32x4& d) {
    if (run.x < 0) return;
    for (int p = run.x; p <= run.y;) {                        // four loads in flight
        f32x4 v[4];
        bool in[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            in[u] = p <= run.y;
            v[u] = *(const f32x4*)(a.L + (long)min(p, run.y) * a.K + k);
            p = ce_run_next(p);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] += in[u] ? v[u][e] : 0.f;
    }
}
__device__ __forceinline__ float ce_label_bias(const CeDwArgs& a, int2 run) {
    float s = 0.f;
    if (run.x >= 0)
        for (int p = run.x; p <= run.y; p = ce_run_next(p)) s += a.Lb[p];
    return s;
}

template <int BA, int BB, int WA, int WB, int STAGES, int BK>
__global__ __launch_bounds__(64 * WA * WB, (BA * BB >= 65536 ? 2 : 3)) void ce_dw_kernel(const CeDwArgs a) {
    using T = GtTile<BA, BB, WA, WB, true, true, STAGES, GT_PRIO, BK>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    if (T::NTHR == 256 && (int)blockIdx.x >= a.nv) {
        ce_dx_finish(a.slab, a.row, a.w, a.dx, a.N, a.K, a.nsplit, blockIdx.x - a.nv, gridDim.x - a.nv);
        return;
    }
    int ta, tb, split;
    if (!gt_map(a.map, blockIdx.x, ta, tb, split)) return;
    const int k0 = ta * BA, v0 = tb * BB;
    const int n0 = split * a.rper, n1 = min(n0 + a.rper, a.N);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const int wa = wave % WA, wb = wave / WA;
    const bool do_db = ta == 0 && wa == 0;                     // wave-uniform
    f32x4 acc[T::NA][T::NB], bacc = {0.f, 0.f, 0.f, 0.f};
    static_assert(T::NB <= 4, "rows of the bias accumulator");
    int2 slots[T::NB];                                         // the classes' label runs
#pragma unroll
    for (int j = 0; j < T::NB; ++j) {
        const int v = v0 + wb * (BB / WB) + 16 * j + fr;
        slots[j] = v < a.V && !a.rslab ? a.slot[v] : make_int2(-1, -1);
    }
    const int wk = k0 + wa * (BA / WA) + 4 * fq, wv = v0 + wb * (BB / WB) + fr;
    // The sums start from the label terms, loaded while the first steps are on their way: behind the loop the loads of 16
    // classes at a time waited for each other (2048 x 2048 x 32000: 304 us, 276 so; 512 x 1024 x 50021 82 and 77)
    auto labels = [&](f32x4 (&c)[T::NA][T::NB]) {
        int any = -1;
#pragma unroll
        for (int j = 0; j < T::NB; ++j) any = max(any, slots[j].x);
        if (!__any(any >= 0)) return T::clear(c);
        auto at = [&](int sl, int i) { return *(const f32x4*)(a.L + (long)sl * a.K + min(wk + 16 * i, a.K - 4)); };
#pragma unroll
        for (int j = 0; j < T::NB; ++j) {
            const int sl = max(slots[j].x, 0);                // loaded whether there is one or not, and dropped
#pragma unroll
            for (int i = 0; i < T::NA; ++i) c[i][j] = at(sl, i);
        }
#pragma unroll
        for (int j = 0; j < T::NB; ++j) {
#pragma unroll
            for (int i = 0; i < T::NA; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[i][j][e] = slots[j].x >= 0 ? c[i][j][e] : 0.f;
            const int last = slots[j].x >= 0 ? slots[j].y : -1;
            for (int p = ce_run_next(max(slots[j].x, 0)); __any(p <= last); p += CE_RUN)
#pragma unroll
                for (int i = 0; i < T::NA; ++i)
                    if (p <= last) c[i][j] += at(p, i);
        }
    };
    // db = E^T g: one more matrix instruction per B fragment j, against a fragment whose rows 4 j and 4 j + 1 are g's two
    // terms and all others zero: one accumulator holds all of them
    T::template run_from<false>(a.xs, a.e, k0, v0, n0, n1, smem, acc, labels, [&](int k, const bf16x8_t (&bv)[T::NB]) {
        if (do_db) {
            const s16x8 gv = *(const s16x8*)(a.g2 + (fr & 1) * a.g2_pitch + n0 + k + 8 * fq);
            const s16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < T::NB; ++j) {
                const bf16x8_t ga = __builtin_bit_cast(bf16x8_t, (fr & ~1) == 4 * j ? gv : z);
                bacc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ga, bv[j], bacc, 0, 0, 0);
            }
        }
    });
    // bf16 rows leave through the wave's own LDS patch as whole 16-byte groups (8-byte stores of 16 rows at a time: 17 -> 10
    // us of a batch of 32), past the caches: the next reader is the optimiser (the whole step of 1237 x 776 x 30011: 281 ->
    // 270 us, of 96 x 2048 x 60000 256 -> 224, of 512 x 1024 x 50021 228 -> 231)
    constexpr int PITCH = BA / WA * 2 + 16;
    char* patch = smem + wave * (BB / WB) * PITCH;
    if (a.rslab) {
        float* o = a.rslab + (long)split * a.V * a.K;
        float* ob = a.rslab + (long)a.rsplit * a.V * a.K + (long)split * a.V;
#pragma unroll
        for (int j = 0; j < T::NB; ++j) {
            const int v = wv + 16 * j;
            if (v >= a.V) continue;
            if (do_db && fq == j) ob[v] = bacc[0] + bacc[1];
#pragma unroll
            for (int i = 0; i < T::NA; ++i)
                if (wk + 16 * i < a.K) *(f32x4*)(o + (long)v * a.K + wk + 16 * i) = acc[i][j];
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < T::NB; ++j) {
        const int v = wv + 16 * j;
        if (v >= a.V) continue;
        if (do_db && fq == j && a.db) {
            float b = bacc[0] + bacc[1] + ce_label_bias(a, slots[j]);
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
            if (a.out_bf16) *(uint2*)(patch + (16 * j + fr) * PITCH + (16 * i + 4 * fq) * 2) =
                    make_uint2(pack2bf(d[0], d[1]), pack2bf(d[2], d[3]));
            else *(float4*)((float*)a.dw + o) = make_float4(d[0], d[1], d[2], d[3]);
        }
    }
    if (!a.out_bf16) return;
    constexpr int CPR = BA / WA / 8;
#pragma unroll 4
    for (int u = lane; u < (BB / WB) * CPR; u += 64) {
        const int v = v0 + wb * (BB / WB) + u / CPR, k = k0 + wa * (BA / WA) + u % CPR * 8;
        if (v < a.V && k < a.K)
            __builtin_nontemporal_store(*(const gt_u32x4*)(patch + u / CPR * PITCH + u % CPR * 16),
                                        (gt_u32x4*)((bf16_t*)a.dw + (long)v * a.K + k));
    }
}

// the row splits' partial sums (in split order), the label terms and earlier pieces -> dw, db
template <bool BF16>
__global__ __launch_bounds__(256) void ce_dw_finish_kernel(const CeDwArgs a) {
    const long n = (long)a.V * a.K, t0 = blockIdx.x * 256L + threadIdx.x, stride = gridDim.x * 256L;
    for (long i = t0 * 4; i < n; i += stride * 4) {
        const int v = (int)(i / a.K), k = (int)(i - (long)v * a.K);
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        int q = 0;
        for (; q + 7 < a.rsplit; q += 8) {
            f32x4 p[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) p[u] = *(const f32x4*)(a.rslab + (q + u) * n + i);
#pragma unroll
            for (int u = 0; u < 8; ++u) s += p[u];
        }
        for (; q < a.rsplit; ++q) s += *(const f32x4*)(a.rslab + q * n + i);
        ce_label_add(a, a.slot[v], k, s);
        if (a.acc_w) s += *(const f32x4*)(a.acc_w + i);
        if (BF16) *(uint2*)((bf16_t*)a.dw + i) = make_uint2(pack2bf(s[0], s[1]), pack2bf(s[2], s[3]));
        else *(f32x4*)((float*)a.dw + i) = s;
    }
    if (!a.db) return;
    for (long v = t0; v < a.V; v += stride) {
        float s = 0.f;
        for (int q = 0; q < a.rsplit; ++q) s += a.rslab[a.rsplit * n + (long)q * a.V + v];
        s += ce_label_bias(a, a.slot[v]);
        if (a.acc_b) s += a.acc_b[v];
        if (BF16) ((bf16_t*)a.db)[v] = f2bf(s);
        else ((float*)a.db)[v] = s;
    }
}

// dw for at most 64 rows, one step of the reduction: the kernel is its store (2 or 4 K V bytes) and what feeds it.  A wave
// keeps the E fragments of its 32 classes in registers and walks its share of the features (all of them, or fewer when the
// classes alone do not make three blocks per CU) 64 at a time, x' through two LDS buffers (L2 serves it, every block reads
// the same 64 x K).  For up to 1024 features: a chunk of 128 bytes per class every few us spreads over more memory pages the
// wider the rows are (8 x 1024 x 50000, bf16: 26 us, 3.9 TB/s, tiles 29; 64 x 512 x 3000 6.3 and 11; 32 x 1024 x 400000 176 and
// 190; but 32 x 2048 x 65536 85 and 81, 8 x 4096 x 50000 121 and 92; chunks of 128 features 28, 9, 175, 98, 116).
// The store counts as a memory operation like the DMA: waiting for the next chunk leaves the STORES youngest operations,
// this chunk's stores, in flight, which holds because every one of them is issued (out of range: past the descriptor,
// dropped).
template <bool BF16>
__global__ __launch_bounds__(256, 3) void ce_dw_thin_kernel(const CeDwArgs a) {
    constexpr int BV = 128, WV = 32, KC = 64, ES = BF16 ? 2 : 4, PITCH = KC * ES + 16;
    constexpr int STORES = WV * KC * ES / 16 / 64;
    using SE = GtStage<BV, 4, true>;
    using SX = GtStage<KC, 4, true>;
    constexpr int PATCH = 4 * WV * PITCH, E_OR_PATCH = PATCH > SE::BYTES ? PATCH : SE::BYTES;
    extern __shared__ __attribute__((aligned(16))) char smem[];                       // [E, later the patches][x'][x']
    if ((int)blockIdx.x >= a.nv) {
        if (blockIdx.y == 0)
            ce_dx_finish(a.slab, a.row, a.w, a.dx, a.N, a.K, a.nsplit, blockIdx.x - a.nv, gridDim.x - a.nv);
        return;
    }
    const int lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int v0 = blockIdx.x * BV, wv = v0 + wave * WV;
    const unsigned lds0 = (unsigned)(unsigned long)(__attribute__((address_space(3))) char*)smem;
    char* xbuf = smem + E_OR_PATCH;
    SE se;
    se.init(a.e, v0, 0, a.N, wave, lane);
    se.issue(lds0, wave);
    int slots[2];                                             // one window: a class has one run
#pragma unroll
    for (int j = 0; j < 2; ++j) slots[j] = wv + 16 * j + fr < a.V ? a.slot[wv + 16 * j + fr].x : -1;
    auto fetch = [&](int k, int buf) {
        SX sx;
        sx.init(a.xs, k, 0, a.N, wave, lane);
        sx.issue(lds0 + E_OR_PATCH + buf * SX::BYTES, wave);
        asm volatile("" ::: "memory");                       // the stores of this chunk stay behind the DMA of the next
    };
    const int nc = (a.K + KC - 1) / KC, share = (nc + gridDim.y - 1) / gridDim.y;
    const int c0 = blockIdx.y * share, c1 = min(c0 + share, nc);
    fetch(c0 * KC, c0 & 1);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    GtFrag<BV, true> fe;
    GtFrag<KC, true> fx;
    fe.init(wave * WV, lane);
    fx.init(0, lane);
    bf16x8_t ev[2][2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int j = 0; j < 2; ++j) ev[kk][j] = fe.load(smem, j, kk, wave * (WV / 16));
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");                 // E's LDS becomes the patches

    if (a.db && c0 == 0) {
        f32x4 b = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const s16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
            const s16x8 gv = *(const s16x8*)(a.g2 + (fr & 1) * a.g2_pitch + kk * 32 + 8 * fq);
#pragma unroll
            for (int j = 0; j < 2; ++j)
                b = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, (fr & ~1) == 4 * j ? gv : z),
                                                            ev[kk][j], b, 0, 0, 0);
        }
        const int v = wv + 16 * fq + fr;
        if (fq < 2 && v < a.V) {
            const int sl = fq == 0 ? slots[0] : slots[1];
            float t = b[0] + b[1] + (sl >= 0 ? a.Lb[sl] : 0.f);
            if (a.acc_b) t += a.acc_b[v];
            if (BF16) ((bf16_t*)a.db)[v] = f2bf(t);
            else ((float*)a.db)[v] = t;
        }
    }

    char* patch = smem + wave * WV * PITCH;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((char*)a.dw + (long)v0 * a.K * ES, 0, 0x7FFFFFF0,
                                                                        0x00020000);
    for (int c = c0; c < c1; ++c) {
        if (c > c0) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(STORES) : "memory");
        fetch((c + 1) * KC, (c + 1) & 1);                     // past the share unused, past the last feature zeros
        const char* xt = xbuf + (c & 1) * SX::BYTES;
        f32x4 acc[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i][0] = acc[i][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bf16x8_t xv = fx.load(xt, i, kk, 0);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xv, ev[kk][j], acc[i][j], 0, 0, 0);
            }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int v = wv + 16 * j + fr;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = c * KC + 16 * i + 4 * fq;
                f32x4 d = acc[i][j];
                if (k < a.K && slots[j] >= 0) d += *(const f32x4*)(a.L + (long)slots[j] * a.K + k);
                if (a.acc_w && v < a.V && k < a.K) {
                    const float4 p = *(const float4*)(a.acc_w + (long)v * a.K + k);
                    d[0] += p.x; d[1] += p.y; d[2] += p.z; d[3] += p.w;
                }
                char* o = patch + (16 * j + fr) * PITCH + (16 * i + 4 * fq) * ES;
                if (BF16) *(uint2*)o = make_uint2(pack2bf(d[0], d[1]), pack2bf(d[2], d[3]));
                else *(f32x4*)o = d;
            }
        }
        constexpr int CPR = KC * ES / 16;                     // 16-byte groups per class
        typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int t = 0; t < STORES; ++t) {
            const int u = t * 64 + lane, row = u / CPR, g = u % CPR;
            const int k = c * KC + g * (16 / ES);
            const unsigned off = (wv + row < a.V && k < a.K) ? (unsigned)(((wave * WV + row) * a.K + k) * ES) : GT_OOB;
            __builtin_amdgcn_raw_buffer_store_b128(*(const u32x4_t*)(patch + row * PITCH + g * 16), rs, off, 0, CE_NT);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // the last fetch has landed before the LDS is given back
}

// Probabilities of wide rows (prediction): logits [B][Cs] bf16 of which N classes are real -> probs [B][N] fp32.  One block per
// row: a pass for the running maximum and sum, a second one for the result.  4096 x 1000 10.6 us, 4096 x 10007 54.5 (each logit
// counted once: 2.3 and 4.5 TB/s), 512 x 50021 83.5 and 4096 x 50021 467 (1.8 and 2.6; the second pass loads two bytes a lane).
__global__ __launch_bounds__(256) void softmax_wide_kernel(const bf16_t* __restrict__ logits, float* __restrict__ probs, int Cs,
                                                           int N) {
    __shared__ float red[4][2];
    const bf16_t* l = logits + (long)blockIdx.x * Cs;
    float* o = probs + (long)blockIdx.x * N;
    const int tid = threadIdx.x;
    float m = -INFINITY, s = 0.f;
    auto add = [&](float om, float os) {                      // m = -inf: nothing seen but masked classes (or NaN: s is NaN)
        const float t = fmaxf(m, om);
        s = (m == t ? s : s * __expf(m - t)) + (om == t ? os : os * __expf(om - t));
        m = t;
    };
    for (int c = tid * 8; c < N; c += 2048) {                 // Cs is a multiple of 8: the loads stay inside the row
        float f[8];
        unpack8(*(const uint4*)(l + c), f);
        float t = -INFINITY, u = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) t = c + e < N ? fmaxf(t, f[e]) : t;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < N) u += f[e] == -INFINITY ? 0.f : __expf(f[e] - t);
        add(t, u);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) add(__shfl_xor(m, d, 64), __shfl_xor(s, d, 64));
    if ((tid & 63) == 0) { red[tid >> 6][0] = m; red[tid >> 6][1] = s; }
    __syncthreads();
    m = red[0][0]; s = red[0][1];
    for (int w = 1; w < 4; ++w) add(red[w][0], red[w][1]);
    const float inv = 1.f / s;
    for (int c = tid; c < N; c += 256) {
        const float f = bf2f(l[c]);
        o[c] = (f == -INFINITY ? 0.f : __expf(f - m)) * inv;  // every class masked: 0 / 0
    }
}

DDL_API int ddl_softmax_wide(const void* logits, float* probs, int B, int Cs, int N, hipStream_t s) {
    if (B <= 0 || N <= 0 || N > Cs || (Cs & 7)) return -1;
    constexpr int ROWS = 1 << 20;                             // per launch: the runtime takes a grid's threads modulo 2^32
    for (long r = 0; r < B; r += ROWS)
        softmax_wide_kernel<<<(int)(B - r < ROWS ? B - r : ROWS), 256, 0, s>>>((const bf16_t*)logits + r * Cs,
                                                                        probs + r * N, Cs, N);
    return gt_launched();
}

// ------------------------------------------------------------------------------------------------ host side
#define CE_MAX_ROWS 8192      // rows of a piece (their labels are ranked in 32 KiB of LDS)
// A scoring piece: a launch holds less than 2^32 threads (the runtime takes more modulo 2^32, without an error); ce_rows
// takes 256 of them per row, ce_logits 256 per 128 statistics
#define CE_SCORE_ROWS (1 << 20)
constexpr long CE_SCORE_STATS = 4L << 30;  // bytes, 8 per row and wave tile

// Everything a call decides from its sizes alone.
struct CePlan {
    int R;                           // rows per piece
    int Vp, lt, nst, wave_cols;      // logits: tile, stats entries per row, classes per entry
    int xt, ns, per;                 // dx: tile, splits over the classes, classes per split
    int wt, rs, rper;                // dw: tile, splits over the rows, rows per split
    long o_count, o_zt, o_stats, o_row, o_order, o_slot, o_g2, o_xs, o_L, o_Lb, o_E, o_slab, o_rslab, o_accw, o_accb, bytes;
    int g2_pitch;
};

static int ce_cdiv(long a, long b) { return (int)((a + b - 1) / b); }

// force_tile: -1, or decimal digits (dw, dx, logits) of the tiles to take, 9 = by the sizes
static CePlan ce_plan(int N, int V, int K, bool train, bool acc, long budget, int force_tile) {
    CePlan p;
    p.Vp = ce_cdiv(V, 64) * 64;
    p.R = N;
    if (train) {
        long r = budget / (p.Vp * 2L);
        r = r >= 256 ? r / 256 * 256 : 64;
        if (r > CE_MAX_ROWS) r = CE_MAX_ROWS;
        if (p.R > r) p.R = (int)r;
    } else {
        if (p.R > CE_SCORE_ROWS) p.R = CE_SCORE_ROWS;
        if (budget > CE_SCORE_STATS) budget = CE_SCORE_STATS;
    }
    // logits: up to 32 rows the tiles that pad them least, the small ones for enough blocks; else by the estimated time, 64-deep
    // steps plus a block's ends in rounds of one 256 x 256 block or two of 128 x 128 or 128 x 32 per CU (the large and the
    // middle ones: 700 x 2400 x 20000 67 and 91 us, 256 x 2048 x 50000 57 and 75, 256 x 1024 x 30000 33 and 26, 300 x 512 x
    // 20000 23 and 17; the middle and the small ones: 64 x 1024 x 10007 18 and 9, 64 x 2048 x 30000 34 and 22, 96 x 2048 x
    // 60000 48 and 58)
    if (p.R <= 32) {
        p.lt = V < 256 * 128 ? 3 : 2;
    } else {
        const int steps = ce_cdiv(K, 64);
        const double two = ce_cdiv((long)ce_cdiv(V, 128) * ce_cdiv(p.R, 128), 256) * 0.5;
        const double us0 = ce_cdiv((long)ce_cdiv(V, 256) * ce_cdiv(p.R, 256), 256) * (steps * 1.6 + 6.0);
        const double us1 = (two > 0.75 ? two : 0.75) * (steps * 1.1 + 5.0);
        const int small = ce_cdiv((long)ce_cdiv(V, 128) * ce_cdiv(p.R, 32), 256);
        const double us2 = small > 1 ? small * 0.5 * (steps * 0.6 + 2.5) : steps * 0.27 + 2.5;
        p.lt = us2 < us0 && us2 < us1 ? 2 : us0 < us1 ? 0 : 1;
    }
    if (force_tile >= 0 && force_tile % 10 < 4) p.lt = force_tile % 10;
    static const int ba[4] = {256, 128, 128, 32}, cols[4] = {128, 64, 32, 16};
    p.wave_cols = cols[p.lt];
    p.nst = ce_cdiv(p.Vp, ba[p.lt]) * (ba[p.lt] / p.wave_cols);      // the tiles cover E's zero columns too
    if (!train && 8L * p.R * p.nst > budget) {                       // scoring keeps 8 bytes per row and wave tile
        const long r = budget / (8L * p.nst) / 256 * 256;
        p.R = (int)(r > 256 ? r : 256);
        if (p.R > N) p.R = N;
    }
    // dx: the tile and the number of splits over the classes by their estimated time: blocks per CU (one of 256 x 256 at
    // a time or two of the others, which are slower each and faster alone) of 64-deep steps plus a block's start and end, and
    // the splits' fp32 partial sums written and read once (in whole rounds of two: 1000 x 512 x 10000 83 us, 76 so; 32 x 2048
    // x 65536 190 and 182).  128 x 128 and 128 x 32: 64 x 2048 x 30000 25 and 21 us, 64 x 4096 x 50000 66 - 80 and 100 - 106
    {
        static const int xa[3] = {256, 128, 128}, xb[3] = {256, 128, 32};
        const double block_us[3] = {1.75, 0.525, p.R <= 32 ? 0.3 : 0.34}, least_us[3] = {1.75, 0.79, 0.35}, ends = 4.0;
        const int steps = ce_cdiv(V, 64), forced = force_tile >= 0 ? force_tile / 10 % 10 : 9;
        double best = 0;
        for (int t = 0; t < 3; ++t) {
            if (forced < 3 ? t != forced : t < 2 && p.R <= 32) continue;
            const long tiles = (long)ce_cdiv(K, xa[t]) * ce_cdiv(p.R, xb[t]);
            for (int ns = 1; ns <= 64 && (ns == 1 || ns <= steps / 4); ++ns) {
                const int per = ce_cdiv(steps, ns), n = ce_cdiv(steps, per);
                const double share = ce_cdiv(tiles * n, 256) * block_us[t];
                const double us = (share > least_us[t] ? share : least_us[t]) * (per + ends) + (n > 1 ? 4.0 + n * 8.0 * p.R * K / 4.5e6 : 0.0);
                if (best == 0 || us < best) { best = us; p.xt = t; p.ns = n; p.per = per * 64; }
            }
        }
    }
    // dw: the streaming kernel for one step and rows that are not too wide (both sides beside it; with two steps of rows, 100 x
    // 1024 x 20000, 23 us and the tiles 21), else tiles
    // The tiles by their estimated time: a CU holds one 256 x 256 block or three of 128 x 128, which are out of step with one
    // another, so one's store runs under the others' products (stages of 32 rows: three blocks' LDS fits.  512 x 1024 x 50021:
    // 82 us, 256 x 256 tiles 96; 256 x 2048 x 50000: 110 and 132; 4096 x 2048 x 32768: 618 and 555; 8192 x 4096 x 131072: 10.8
    // and 7.4 ms.  Two blocks with stages of 64 rows took 106 on the first, two of 256 x 128 88).  The rows are split when the
    // tiles are few (8000 rows x 64 x 65 classes, one tile: 161 us in one piece)
    {
        static const int edge[2] = {256, 128}, fit[2] = {1, 3};
        static const double round_us[2] = {1.75, 1.64}, one_us[2] = {1.75, 1.3}, ends[2] = {8.0, 3.5};
        const int steps = ce_cdiv(p.R, 64), forced = force_tile >= 0 ? force_tile / 100 % 10 : 9;
        const bool thin = p.R <= 64 && K <= 1024;
        p.wt = 2; p.rs = 1; p.rper = steps * 64;
        double best = 0;
        for (int t = 0; t < 2; ++t) {
            if (forced < 2 ? t != forced : thin) continue;
            const long tiles = (long)ce_cdiv(K, edge[t]) * ce_cdiv(V, edge[t]);
            for (int want = 1; want <= 32 && (want == 1 || want <= steps / 4); ++want) {
                const int per = ce_cdiv(steps, want), n = ce_cdiv(steps, per);
                const double share = (double)ce_cdiv(tiles * n, 256) / fit[t] * round_us[t];
                const double us = (share > one_us[t] ? share : one_us[t]) * (per + ends[t]) +
                                  (n > 1 ? 3.0 + 0.15 * n + n * 8.0 * V * K / 4.5e6 : 0.0);
                if (best == 0 || us < best) { best = us; p.wt = t; p.rs = n; p.rper = per * 64; }
            }
        }
    }
    p.g2_pitch = ce_cdiv(p.R, 64) * 64;
    long o = 0;
    auto take = [&](long bytes) { const long at = o; o += (bytes + 255) / 256 * 256; return at; };
    p.o_count = take(4); p.o_zt = take(4L * p.R); p.o_stats = take(8L * p.R * p.nst);
    p.o_row = p.o_order = p.o_slot = p.o_g2 = p.o_xs = p.o_L = p.o_Lb = p.o_E = p.o_slab = p.o_rslab = p.o_accw = p.o_accb = 0;
    if (train) {
        p.o_row = take(32L * p.R); p.o_order = take(4L * p.R); p.o_slot = take(8L * V); p.o_g2 = take(4L * p.g2_pitch);
        p.o_xs = take(2L * p.R * K); p.o_L = take(4L * p.R * K); p.o_Lb = take(4L * p.R); p.o_E = take(2L * p.R * p.Vp);
        if (p.ns > 1) p.o_slab = take(4L * p.ns * p.R * K);
        if (p.rs > 1) p.o_rslab = take(4L * p.rs * V * (K + 1L));
        if (acc && p.R < N) { p.o_accw = take(4L * V * K); p.o_accb = take(4L * V); }
    }
    p.bytes = o;
    return p;
}

template <int BA, int BB, int WA, int WB, int STAGES, bool STORE>
static int launch_logits(CeLogitsArgs& a, hipStream_t s) {
    using T = GtTile<BA, BB, WA, WB, false, false, STAGES, GT_PLAIN>;
    const size_t out = (STORE ? BB * (BA * 2 + 16) : 0) + (BA + BB) * 4;
    size_t lds = out > T::LDS_BYTES ? out : T::LDS_BYTES;
    if (a.order && 4L * a.N > (long)lds) lds = 4L * a.N;
    constexpr auto kern = ce_logits_kernel<BA, BB, WA, WB, STAGES, STORE>;
    if (int rc = gt_lds<kern>(lds)) return rc;
    a.map = gt_make_map((a.Vp + BA - 1) / BA, (a.N + BB - 1) / BB, 1, 8);
    a.nrank = a.order ? (ce_cdiv(a.N, CE_RANK_ROWS) + 7) / 8 * 8 : 8;
    if (!gt_map_ok(a.map, T::NTHR, a.nrank)) return -1;
    kern<<<a.nrank + gt_grid(a.map), T::NTHR, lds, s>>>(a);
    return gt_launched();
}

template <bool STORE>
static int ce_logits(CeLogitsArgs& a, int tile, hipStream_t s) {
    switch (tile) {
        case 0: return launch_logits<256, 256, 2, 4, 2, STORE>(a, s);
        case 1: return launch_logits<128, 128, 2, 2, 2, STORE>(a, s);
        case 2: return launch_logits<128, 32, 4, 1, 4, STORE>(a, s);
        default: return launch_logits<32, 32, 2, 1, 4, STORE>(a, s);
    }
}

template <int BA, int BB, int WA, int WB, int STAGES>
static int launch_dx(CeDxArgs& a, hipStream_t s) {
    using T = GtTile<BA, BB, WA, WB, true, false, STAGES, GT_FENCE>;
    constexpr auto kern = ce_dx_kernel<BA, BB, WA, WB, STAGES>;
    if (int rc = gt_lds<kern>(T::LDS_BYTES)) return rc;
    a.map = gt_make_map((a.K + BA - 1) / BA, (a.N + BB - 1) / BB, a.nsplit, 8);
    if (!gt_map_ok(a.map, T::NTHR, 2048)) return -1;
    a.nlab_chunks = ce_cdiv(a.K, 2048);
    a.ntile = gt_grid(a.map);
    // The label blocks fill what the last round of tiles leaves (a launch of their own costs 5 us; the large tiles have other
    // blocks and do not notice).  They hold a tile's LDS, so not when they are many (8000 x 64 x 65: 162 us, 125 on their own)
    const int nlab = a.nlab_chunks * (a.N + 1);
    const bool ride = T::NTHR == 256 && nlab <= 2048;
    if (!ride) ce_labels_kernel<<<dim3(a.N + 1, a.nlab_chunks), 256, 0, s>>>(a.lab);
    kern<<<a.ntile + (ride ? nlab : 0), T::NTHR, T::LDS_BYTES, s>>>(a);
    return gt_launched();
}

// blocks that finish the splits of dx: four features per thread, and strides of them in a piece of 2^30 features and more
static int ce_finish_blocks(const CeDwArgs& a) {
    const long n = a.slab ? ((long)a.N * a.K + 1023) / 1024 : 0;
    return n < (1 << 20) ? (int)n : 1 << 20;
}

template <int BA, int BB, int WA, int WB, int STAGES, int BK>
static int launch_dw(CeDwArgs& a, hipStream_t s) {
    using T = GtTile<BA, BB, WA, WB, true, true, STAGES, GT_PRIO, BK>;
    constexpr auto kern = ce_dw_kernel<BA, BB, WA, WB, STAGES, BK>;
    const size_t out = (size_t)T::NW * (BB / WB) * (BA / WA * 2 + 16);
    const size_t lds = a.out_bf16 && out > T::LDS_BYTES ? out : T::LDS_BYTES;
    if (int rc = gt_lds<kern>(lds)) return rc;
    a.map = gt_make_map((a.K + BA - 1) / BA, (a.V + BB - 1) / BB, a.rsplit, 4);
    // the splits of dx are finished in what the last round of tiles leaves, or by a launch of their own (7 us)
    a.nv = gt_grid(a.map);
    const int nfin = ce_finish_blocks(a);
    if (!gt_map_ok(a.map, T::NTHR, nfin)) return -1;
    if (T::NTHR != 256 && nfin) ce_dx_finish_kernel<<<nfin, 256, 0, s>>>(a.slab, a.row, a.w, a.dx, a.N, a.K, a.nsplit);
    kern<<<a.nv + (T::NTHR == 256 ? nfin : 0), T::NTHR, lds, s>>>(a);
    if (a.rsplit > 1) {
        const long nb = ((long)a.V * a.K + 1023) / 1024;
        const int g = (int)(nb > 2048 ? 2048 : nb);
        if (a.out_bf16) ce_dw_finish_kernel<true><<<g, 256, 0, s>>>(a);
        else ce_dw_finish_kernel<false><<<g, 256, 0, s>>>(a);
    }
    return gt_launched();
}

template <bool BF16>
static int launch_dw_thin(CeDwArgs& a, hipStream_t s) {
    const size_t patch = 4 * 32 * (64 * (BF16 ? 2 : 4) + 16), e = 128 * 64 * 2, lds = (patch > e ? patch : e) + 2 * 64 * 64 * 2;
    constexpr auto kern = ce_dw_thin_kernel<BF16>;
    if (int rc = gt_lds<kern>(lds)) return rc;
    const int nc = (a.K + 63) / 64;
    a.nv = (a.V + 127) / 128;
    const int want = (768 + a.nv - 1) / a.nv, nfin = ce_finish_blocks(a);
    kern<<<dim3(a.nv + nfin, want < nc ? want : nc), 256, lds, s>>>(a);
    return gt_launched();
}

static bool ce_range_ok(int N, int V, int K) {
    // 64 k rows or 256 rows of any operand within 31 bits of byte offset
    return N > 0 && V > 0 && K > 0 && (K & 7) == 0 && (long)K * 512 < (1L << 31) && ((long)V + 64) * 512 < (1L << 31) &&
           N < (1 << 28);
}

// Workspace of one call in bytes (negative: sizes outside the kernels' range)
DDL_API long ddl_dense_ce_workspace(int N, int V, int K, int train, int out_bf16, long budget, int force_tile) {
    if (!ce_range_ok(N, V, K) || force_tile > 999) return -1;
    return ce_plan(N, V, K, train, out_bf16, budget, force_tile).bytes;
}

// x [N][K], w [V][K] bf16; bias [V] fp32 or null; labels [N]; dx == null: scoring.  dw / db (db may be null) fp32 or bf16.
DDL_API int ddl_dense_ce(const void* x_, const void* w_, const float* bias, const long* labels, int N, int V, int K,
                         float* loss, float* rows, void* dx, void* dw, void* db, int out_bf16, void* ws_, long ws_bytes,
                         long budget, int force_tile, hipStream_t s) {
    if (!ce_range_ok(N, V, K) || force_tile > 999) return -1;
    const bool train = dx != nullptr;
    const CePlan p = ce_plan(N, V, K, train, out_bf16, budget, force_tile);
    if (ws_bytes < p.bytes || (train && !dw)) return -3;
    const bf16_t* x = (const bf16_t*)x_;
    const bf16_t* w = (const bf16_t*)w_;
    char* ws = (char*)ws_;
    float* count = (float*)(ws + p.o_count);
    float* zt = (float*)(ws + p.o_zt);
    CeRow* row = (CeRow*)(ws + p.o_row);
    bf16_t* E = (bf16_t*)(ws + p.o_E);
    bf16_t* xs = (bf16_t*)(ws + p.o_xs);
    bf16_t* g2 = (bf16_t*)(ws + p.o_g2);
    // The weights are read past the caches where one row tile is all there is and nobody reads them again soon: when scoring
    // (32 x 2048 x 65536: 67 -> 60 us) and in a step whose dx would not find them there either (32 x 4096 x 100000: 642 -> 575
    // us; 64 x 2048 x 30000, whose weights stay: 116 -> 124, so there not)
    static const int l_rows[4] = {256, 128, 32, 32}, x_rows[3] = {256, 128, 32};
    for (int r0 = 0; r0 < N; r0 += p.R) {
        const int n = N - r0 < p.R ? N - r0 : p.R;
        const bool last = r0 + n >= N;
        CeLogitsArgs a;
        a.w = {w, K, V, n <= l_rows[p.lt] && (!train || 2L * V * K > CE_CACHE)}; a.x = {x + (long)r0 * K, K, n};
        a.bias = bias; a.labels = labels + r0; a.N = n; a.V = V; a.K = K; a.Vp = p.Vp;
        a.E = train ? E : nullptr; a.stats = (float2*)(ws + p.o_stats); a.nst = p.nst; a.zt = zt;
        a.labels_all = labels; a.n_all = N; a.count = r0 == 0 ? count : nullptr;
        a.order = train ? (int*)(ws + p.o_order) : nullptr; a.slot = (int2*)(ws + p.o_slot);
        int rc = train ? ce_logits<true>(a, p.lt, s) : ce_logits<false>(a, p.lt, s);
        if (rc) return rc;

        CeRowsArgs b;
        b.stats = a.stats; b.nst = p.nst; b.wave_cols = p.wave_cols; b.zt = zt; b.labels = a.labels; b.count = count;
        b.w = w; b.bias = bias;
        b.N = n; b.V = V; b.K = K; b.Vp = p.Vp; b.E = E; b.x = a.x.p; b.xs = xs; b.rows = rows + r0;
        b.row = row; b.g2 = g2; b.g2_pitch = p.g2_pitch; b.loss = nullptr;
        // few long rows: 1024 threads each (16 -> 6 us at 4096 entries); many short ones: a wave (8000 x 64 x 65: 80 -> 72 us)
        const bool wide = n <= 256 && p.nst > 512, narrow = n > 256 && K <= 512 && p.nst <= 128;
        if (!train) {
            if (N <= CE_FEW_ROWS && p.nst <= CE_FEW_STATS) {
                ce_score_few_kernel<<<1, 1024, 0, s>>>(b, loss);
                return gt_launched();
            }
            if (N == 1) b.loss = loss;
            if (wide) ce_rows_kernel<false, 1024><<<n, 1024, 0, s>>>(b);
            else if (narrow) ce_rows_kernel<false, 64><<<n, 64, 0, s>>>(b);
            else ce_rows_kernel<false, 256><<<n, 256, 0, s>>>(b);
            if (last && N > 1) ce_mean_kernel<<<1, 1024, 0, s>>>(rows, count, N, loss);
            if (int e = gt_launched()) return e;
            continue;
        }
        if (wide) ce_rows_kernel<true, 1024><<<n, 1024, 0, s>>>(b);
        else if (narrow) ce_rows_kernel<true, 64><<<n, 64, 0, s>>>(b);
        else ce_rows_kernel<true, 256><<<n, 256, 0, s>>>(b);

        CeLabelsArgs l;
        l.row = row; l.order = a.order; l.x = a.x.p; l.xs = xs; l.N = n; l.K = K; l.slot = a.slot;
        l.L = (float*)(ws + p.o_L); l.Lb = (float*)(ws + p.o_Lb);
        l.rows_all = rows; l.count = count; l.n_all = N; l.loss = last ? loss : nullptr;
        if (int e = gt_launched()) return e;

        CeDxArgs d;
        d.lab = l;
        d.w = {w, K, K, n <= x_rows[p.xt] && 2L * V * K > CE_CACHE}; d.e = {E, p.Vp, n};
        d.N = n; d.V = V; d.K = K; d.nsplit = p.ns; d.per_split = p.per; d.row = row; d.dx = (bf16_t*)dx + (long)r0 * K;
        d.slab = p.ns > 1 ? (float*)(ws + p.o_slab) : nullptr;
        switch (p.xt) {
            case 0: rc = launch_dx<256, 256, 2, 4, 2>(d, s); break;
            case 1: rc = launch_dx<128, 128, 2, 2, 2>(d, s); break;
            default: rc = launch_dx<128, 32, 4, 1, 4>(d, s);
        }
        if (rc) return rc;

        CeDwArgs c;
        c.xs = {xs, K, K}; c.e = {E, p.Vp, p.Vp};
        c.rsplit = ce_cdiv(n, p.rper); c.rper = p.rper;     // a shorter last piece has fewer splits
        c.rslab = c.rsplit > 1 ? (float*)(ws + p.o_rslab) : nullptr;
        c.slab = d.slab; c.row = row; c.w = w; c.dx = d.dx; c.nsplit = p.ns; c.nv = 0;
        c.N = n; c.V = V; c.K = K; c.g2 = g2; c.g2_pitch = p.g2_pitch; c.slot = a.slot; c.L = l.L; c.Lb = l.Lb;
        // several pieces add up in fp32: in the output itself, or in the workspace until the last piece rounds
        float* aw = out_bf16 ? (float*)(ws + p.o_accw) : (float*)dw;
        float* ab = out_bf16 ? (float*)(ws + p.o_accb) : (float*)db;
        c.acc_w = r0 ? aw : nullptr;
        c.acc_b = r0 && db ? ab : nullptr;
        c.out_bf16 = out_bf16 && last;
        c.dw = last ? dw : (void*)aw;
        c.db = db ? (last ? db : (void*)ab) : nullptr;
        switch (p.wt) {
            case 0: rc = launch_dw<256, 256, 2, 4, 2, 64>(c, s); break;
            case 1: rc = launch_dw<128, 128, 2, 2, 3, 32>(c, s); break;
            default: rc = c.out_bf16 ? launch_dw_thin<true>(c, s) : launch_dw_thin<false>(c, s);
        }
        if (rc) return rc;
    }
    return gt_launched();
}
