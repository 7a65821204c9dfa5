// kernels_ln.hip -- layer normalisation over the rows of a [B][D] activation, forward and backward (gfx950).
//
//   forward   mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps),  y = (x - mean) * rstd * gamma + beta
//   backward  h = (x - mean) * rstd,  p = dy * gamma,
//             dx = skip + rstd * (p - mean(p) - h * mean(p * h)),   dgamma = sum_rows dy * h,   dbeta = sum_rows dy
//
// Both are bound by memory: a row is read once, lies in registers (as it came: 16 bits stay 16 bits) while its sums are formed in two
// passes over them -- the variance from differences to the mean, never from sum x^2 -- and is written once; the next row's loads are in
// flight meanwhile.  The arithmetic is f32 but for the mean, which is the exact sum's rounded once where the values are near each other: a
// mean one step of f32 off is far off where the spread is small (constant rows of 1e5 came out up to 1.7 beside beta).  So f32 is summed
// in f64; 8192 values of at most 11 bits are exact in f32 (bf16, 65536 x 429: 26.3 us in f64, 23.5 so).  A row belongs to TPR lanes (4, 16
// or 64 of one wave, or a workgroup of 256 or 512) that hold up to 16 elements each: a narrow row does not idle a wave, a wide one does
// not spill.  Rows wider than 8192 take the kernels that walk the row again (from L2).  EDGE: the width is no multiple of a 16-byte
// piece, so the last piece is cut off; without it a lane behind the row's end reads the row's first piece and counts it as zeros, and no
// load hides behind a branch.
// Measured: bf16, 65536 x 1024 forward 51 us (5.3 TB/s; a copy of 1 GiB runs at 5.1), backward with skip 108 us (5.0 TB/s), 65536 x 1001
// 115; f32, 4096 x 429 forward 5 us; one row 1.9 us on the device, and 7 with the call's host side.
#include <type_traits>

#include "kernels_tower.h"

namespace {

constexpr int kMaxEpl = 16;            // elements of a row per lane

// N sums over the TPR lanes of a row at once; slot: alternating, so that one barrier is enough
template <int TPR, int N, typename V, int W> __device__ __forceinline__ void row_sums(V (&v)[N], V (*lds)[16][W], int &slot) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o);
    if constexpr (TPR > 64) {          // the waves of the workgroup, in wave order
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) lds[slot][threadIdx.x >> 6][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = lds[slot][0][i];
#pragma unroll
            for (int w = 1; w < TPR / 64; ++w) v[i] += lds[slot][w][i];
        }
        slot ^= 1;
    }
}
template <int TPR, typename V, int W> __device__ __forceinline__ V row_sum(V v, V (*lds)[16][W], int &slot) {
    V s[1] = {v};
    row_sums<TPR>(s, lds, slot);
    return s[0];
}

// EDGE: the piece that the width cuts off runs on into the next row -- what it finds there is masked -- except in the last row, which reads
// it further to the left and shifts it into place before its use (settle): no load hides behind a branch, and no other row pays.  (Shifted
// in every row: bf16, 65536 x 1001 backward 180 us; element by element 156.)
template <typename T, int TPR, int NV, bool EDGE> struct RowPieces {
    static constexpr int VEC = Chunk<T>::N;
    Chunk<T> c[NV];
    __device__ __forceinline__ void load(const T *row, int t, int D, bool last) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (t + i * TPR) * VEC;
            if (EDGE && D < VEC) { c[i].load(row, e, D); continue; }         // (narrower than a piece: it could run past more than one row)
            int at = e < D ? e : 0;
            if (EDGE && last && at + VEC > D) at = D - VEC;
            c[i].u = *reinterpret_cast<const typename Chunk<T>::unaligned_t *>(row + at);
        }
    }
    __device__ __forceinline__ void settle(int t, int D) {                   // of the last row
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (t + i * TPR) * VEC;
            if (D >= VEC && e < D && e + VEC > D) c[i].shift_down(e + VEC - D);
        }
    }
    __device__ __forceinline__ void store(T *row, int t, int D) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (t + i * TPR) * VEC;
            if constexpr (EDGE) c[i].store(row, e, D);
            else if (e < D) *reinterpret_cast<typename Chunk<T>::unaligned_t *>(row + e) = c[i].u;
        }
    }
};
// does element j of piece i lie in the row?
template <int TPR, int VEC, bool EDGE> __device__ __forceinline__ bool inside(int t, int i, int j, int D) {
    return (t + i * TPR) * VEC + (EDGE ? j : 0) < D;
}
// gamma or beta: rows of the store's, 16-byte aligned and padded to a multiple of 16.  Four at a time: one by one they cost a workgroup as
// much as eight of its rows (f16, 16384 x 1024 forward: 37 us, 12.4 so).
template <typename T, int TPR, int NV, bool EDGE> __device__ __forceinline__ void load_params(float (&p)[NV * Chunk<T>::N], const float *src, int t, int D) {
    constexpr int VEC = Chunk<T>::N;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * VEC;
#pragma unroll
        for (int h = 0; h < VEC; h += 4) {
            const f32x4 v = *reinterpret_cast<const f32x4 *>(src + (c < D ? c : 0) + h);
#pragma unroll
            for (int j = 0; j < 4; ++j) p[i * VEC + h + j] = EDGE && c + h + j >= D ? 0.f : v[j];
        }
    }
}

template <typename T> using RowSum = std::conditional_t<sizeof(T) == 4, double, float>;          // of up to 8192 values that are near each other: exact

template <typename T, int TPR, int NV, bool EDGE>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_ln_fwd(LnFwdArgs a) {
    constexpr int VEC = Chunk<T>::N, RPB = TPR > 256 ? 1 : 256 / TPR;
    __shared__ float lds[2][16][1];
    __shared__ RowSum<T> ldsx[2][16][1];
    int slot = 0, slotx = 0;
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float inv_d = 1.f / (float)a.D;
    const double inv_d64 = 1. / a.D;
    const int64_t stride = (int64_t)gridDim.x * RPB;
    int64_t r = (int64_t)blockIdx.x * RPB + sub;
    // a lane group behind the last row repeats it and writes nothing
    RowPieces<T, TPR, NV, EDGE> v, next;
    next.load((const T *)a.x + (r < a.B ? r : a.B - 1) * a.ldx, t, a.D, r >= a.B - 1);
    float g[NV * VEC], b[NV * VEC];
    load_params<T, TPR, NV, EDGE>(g, a.gamma, t, a.D);
    load_params<T, TPR, NV, EDGE>(b, a.beta, t, a.D);
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.B; r0 += stride, r += stride) {
        v = next;
        if (EDGE && r >= a.B - 1) v.settle(t, a.D);
        if (r0 + stride < a.B) next.load((const T *)a.x + (r + stride < a.B ? r + stride : a.B - 1) * a.ldx, t, a.D, r + stride >= a.B - 1);
        RowSum<T> sx = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) sx += inside<TPR, VEC, EDGE>(t, i, j, a.D) ? (float)v.c[i].e[j] : 0.f;
        const float mean = (float)(row_sum<TPR>(sx, ldsx, slotx) * inv_d64);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = inside<TPR, VEC, EDGE>(t, i, j, a.D) ? (float)v.c[i].e[j] - mean : 0.f;
                s = fmaf(d, d, s);
            }
        const float rstd = 1.f / sqrtf(row_sum<TPR>(s, lds, slot) * inv_d + a.eps);
        if (r >= a.B) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) v.c[i].e[j] = (T)fmaf(((float)v.c[i].e[j] - mean) * rstd, g[i * VEC + j], b[i * VEC + j]);
        v.store((T *)a.y + r * a.ldy, t, a.D);
        if (a.stats && t == 0) { a.stats[2 * r] = mean; a.stats[2 * r + 1] = rstd; }
    }
}

// rows of any width: one workgroup per row walks it three times, the second and third from L2 (bf16, 4096 x 16384 78 us, 3.4 TB/s)
template <typename T>
__global__ __launch_bounds__(256) void k_ln_fwd_wide(LnFwdArgs a) {
    constexpr int VEC = Chunk<T>::N;
    __shared__ float lds[2][16][1];
    __shared__ double lds64[2][16][1];
    int slot = 0, slot64 = 0;
    const float inv_d = 1.f / (float)a.D;
    const double inv_d64 = 1. / a.D;
    for (int64_t r = blockIdx.x; r < a.B; r += gridDim.x) {
        const T *x = (const T *)a.x + r * a.ldx;
        T *y = (T *)a.y + r * a.ldy;
        Chunk<T> v;
        double s64 = 0.;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
            v.load(x, (int)c, a.D);
            RowSum<T> sx = 0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) sx += (float)v.e[j];
            s64 += sx;
        }
        const float mean = (float)(row_sum<256>(s64, lds64, slot64) * inv_d64);
        float s = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
            v.load(x, (int)c, a.D);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = c + j < a.D ? (float)v.e[j] - mean : 0.f;
                s = fmaf(d, d, s);
            }
        }
        const float rstd = 1.f / sqrtf(row_sum<256>(s, lds, slot) * inv_d + a.eps);
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
            float g[VEC], b[VEC];
            load_params<T, 256, 1, true>(g, a.gamma, (int)(c / VEC), a.D);
            load_params<T, 256, 1, true>(b, a.beta, (int)(c / VEC), a.D);
            v.load(x, (int)c, a.D);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v.e[j] = (T)fmaf(((float)v.e[j] - mean) * rstd, g[j], b[j]);
            v.store(y, (int)c, a.D);
        }
        if (a.stats && threadIdx.x == 0) { a.stats[2 * r] = mean; a.stats[2 * r + 1] = rstd; }
    }
}

// Every lane keeps the column sums of its own columns over all the rows it sees; a workgroup folds its RPB row groups through LDS and
// writes one slab: no atomics, the same order in every run.
template <typename T, int TPR, int NV, bool EDGE>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_ln_bwd(LnBwdArgs a) {
    constexpr int VEC = Chunk<T>::N, RPB = TPR > 256 ? 1 : 256 / TPR, E = NV * VEC;
    __shared__ float lds[2][16][2];
    __shared__ float fold[TPR < 256 ? 4 * (TPR < 64 ? TPR : 64) * VEC : 1];
    int slot = 0;
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float inv_d = 1.f / (float)a.D;
    const int64_t stride = (int64_t)gridDim.x * RPB;
    int64_t r = (int64_t)blockIdx.x * RPB + sub;
    RowPieces<T, TPR, NV, EDGE> x, dy, k, nx, ndy, nk;
    float mean, rstd, nmean, nrstd;
    auto fetch = [&](int64_t q) {
        const bool last = q >= a.B - 1;
        if (last) q = a.B - 1;
        nx.load((const T *)a.x + q * a.ldx, t, a.D, last);
        ndy.load((const T *)a.dy + q * a.lddy, t, a.D, last);
        if (a.skip) nk.load((const T *)a.skip + q * a.ldskip, t, a.D, last);
        nmean = a.stats[2 * q]; nrstd = a.stats[2 * q + 1];
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) nk.c[i].zero();
    fetch(r);
    float g[E], sg[E], sb[E];
    load_params<T, TPR, NV, EDGE>(g, a.gamma, t, a.D);
#pragma unroll
    for (int i = 0; i < E; ++i) { sg[i] = 0.f; sb[i] = 0.f; }
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.B; r0 += stride, r += stride) {
        const bool live = r < a.B;
        x = nx; dy = ndy; k = nk; mean = nmean; rstd = nrstd;
        if (EDGE && r >= a.B - 1) {
            x.settle(t, a.D); dy.settle(t, a.D);
            if (a.skip) k.settle(t, a.D);
        }
        if (r0 + stride < a.B) fetch(r + stride);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const bool in = live && inside<TPR, VEC, EDGE>(t, i, j, a.D);
                const float h = in ? ((float)x.c[i].e[j] - mean) * rstd : 0.f, d = in ? (float)dy.c[i].e[j] : 0.f, p = d * g[i * VEC + j];
                s[0] += p; s[1] = fmaf(p, h, s[1]);
                sg[i * VEC + j] = fmaf(d, h, sg[i * VEC + j]); sb[i * VEC + j] += d;
            }
        if (!a.dx) continue;
        row_sums<TPR>(s, lds, slot);
        if (!live) continue;
        const float m1 = s[0] * inv_d, m2 = s[1] * inv_d;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float h = ((float)x.c[i].e[j] - mean) * rstd, p = (float)dy.c[i].e[j] * g[i * VEC + j];
                k.c[i].e[j] = (T)((float)k.c[i].e[j] + rstd * (p - m1 - h * m2));
            }
        k.store((T *)a.dx + r * a.lddx, t, a.D);
    }
    float *out = a.part + (size_t)blockIdx.x * 2 * a.D;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        float *acc = w ? sb : sg;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (TPR < 256) {           // the row groups of a wave lane by lane, then the four waves through LDS
                constexpr int L = TPR < 64 ? TPR : 64;
#pragma unroll
                for (int j = 0; j < VEC; ++j)
#pragma unroll
                    for (int o = TPR; o < 64; o <<= 1) acc[i * VEC + j] += __shfl_xor(acc[i * VEC + j], o);
                __syncthreads();
                if ((threadIdx.x & 63) < L)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) fold[((threadIdx.x >> 6) * L + t) * VEC + j] = acc[i * VEC + j];
                __syncthreads();
                if (sub == 0)
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        acc[i * VEC + j] = (fold[t * VEC + j] + fold[(L + t) * VEC + j]) + (fold[(2 * L + t) * VEC + j] + fold[(3 * L + t) * VEC + j]);
            }
            if (sub == 0) {
                float *row = out + (size_t)w * a.D;
#pragma unroll
                for (int h = 0; h < VEC; h += 4) {
                    const int c = (t + i * TPR) * VEC + h;
                    Quad<float> q;
#pragma unroll
                    for (int j = 0; j < 4; ++j) q.e[j] = acc[i * VEC + h + j];
                    if (c < a.D) q.store(row, c, a.D);
                }
            }
        }
    }
}

// wide rows: the column sums live in the workgroup's slab (its own columns, its own lane: plain adds), which is most of the traffic: 16 bytes
// a value (bf16, 4096 x 16384 300 us, 1.3 TB/s of x, dy and dx)
template <typename T>
__global__ __launch_bounds__(256) void k_ln_bwd_wide(LnBwdArgs a) {
    constexpr int VEC = Chunk<T>::N;
    __shared__ float lds[2][16][2];
    int slot = 0;
    const float inv_d = 1.f / (float)a.D;
    float *sg = a.part + (size_t)blockIdx.x * 2 * a.D, *sb = sg + a.D;
    for (int64_t r = blockIdx.x; r < a.B; r += gridDim.x) {
        const bool first = r == blockIdx.x;
        const T *x = (const T *)a.x + r * a.ldx, *dy = (const T *)a.dy + r * a.lddy, *sk = (const T *)a.skip + r * a.ldskip;
        const float mean = a.stats[2 * r], rstd = a.stats[2 * r + 1];
        Chunk<T> v, w, k;
        float s1 = 0.f, s2 = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
            float g[VEC];
            load_params<T, 256, 1, true>(g, a.gamma, (int)(c / VEC), a.D);
            v.load(x, (int)c, a.D); w.load(dy, (int)c, a.D);
            Quad<float> pg[VEC / 4], pb[VEC / 4];
#pragma unroll
            for (int q = 0; q < VEC / 4; ++q) {
#pragma unroll
                for (int j = 0; j < 4; ++j) { pg[q].e[j] = 0.f; pb[q].e[j] = 0.f; }
                if (!first) { pg[q].load(sg, (int)c + 4 * q, a.D); pb[q].load(sb, (int)c + 4 * q, a.D); }
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = (float)w.e[j], h = c + j < a.D ? ((float)v.e[j] - mean) * rstd : 0.f, p = d * g[j];      // (d and g are 0 behind the row)
                s1 += p; s2 = fmaf(p, h, s2);
                pg[j / 4].e[j % 4] = fmaf(d, h, pg[j / 4].e[j % 4]);
                pb[j / 4].e[j % 4] += d;
            }
#pragma unroll
            for (int q = 0; q < VEC / 4; ++q)
                if (c + 4 * q < a.D) { pg[q].store(sg, (int)c + 4 * q, a.D); pb[q].store(sb, (int)c + 4 * q, a.D); }
        }
        if (!a.dx) continue;
        const float m1 = row_sum<256>(s1, lds, slot) * inv_d, m2 = row_sum<256>(s2, lds, slot) * inv_d;
        T *dx = (T *)a.dx + r * a.lddx;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
            float g[VEC];
            load_params<T, 256, 1, true>(g, a.gamma, (int)(c / VEC), a.D);
            v.load(x, (int)c, a.D); w.load(dy, (int)c, a.D);
            k.zero();
            if (a.skip) k.load(sk, (int)c, a.D);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float h = ((float)v.e[j] - mean) * rstd, p = (float)w.e[j] * g[j];
                k.e[j] = (T)((float)k.e[j] + rstd * (p - m1 - h * m2));
            }
            k.store(dx, (int)c, a.D);
        }
    }
}

// 64 columns a workgroup; its 16 waves take the slabs in turn, 8 loads in flight each, and are added in wave order
__global__ __launch_bounds__(1024) void k_grad_reduce(const float *__restrict__ part, int nslab, int64_t n, int B, float *__restrict__ dst, int accum) {
    __shared__ float sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t i = (int64_t)blockIdx.x * 64 + lane, ic = i < n ? i : n - 1;
    float s = 0.f;
    for (int z0 = wave; z0 < nslab; z0 += 128) {
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = z0 + q * 16 < nslab ? part[(int64_t)(z0 + q * 16) * n + ic] : 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) s += v[q];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave || i >= n) return;
#pragma unroll
    for (int w = 1; w < 16; ++w) s += sums[w][lane];
    s /= (float)B;
    dst[i] = accum ? dst[i] + s : s;
}

// the row layout of a width: lanes per row and pieces per lane (0 lanes: the walking kernel)
struct Layout { int tpr, nv; };
Layout layout_of(int vec, int D) {
    const int chunks = (D + vec - 1) / vec;
    for (int tpr : {4, 16, 64, 256, 512}) {
        if (chunks > tpr * (kMaxEpl / vec)) continue;
        int nv = 1;
        while (tpr * nv < chunks) nv *= 2;
        return {tpr, nv};
    }
    return {0, 0};
}

template <typename T, int TPR, int NV>
int fwd_go(const LnFwdArgs &a, hipStream_t st) {
    constexpr int RPB = TPR > 256 ? 1 : 256 / TPR;
    const int64_t need = ((int64_t)a.B + RPB - 1) / RPB, most = TPR > 256 ? 512 : 2048;
    const dim3 grid((unsigned)(need < most ? need : most)), block(TPR > 256 ? TPR : 256);
    if (a.D % Chunk<T>::N) hipLaunchKernelGGL((k_ln_fwd<T, TPR, NV, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_ln_fwd<T, TPR, NV, false>), grid, block, 0, st, a);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
template <typename T, int TPR, int NV>
int bwd_go(const LnBwdArgs &a, int nblk, hipStream_t st) {
    const dim3 grid((unsigned)nblk), block(TPR > 256 ? TPR : 256);
    if (a.D % Chunk<T>::N) hipLaunchKernelGGL((k_ln_bwd<T, TPR, NV, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_ln_bwd<T, TPR, NV, false>), grid, block, 0, st, a);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
// every (lanes, pieces) that layout_of can return for the type: a wider group takes over where two pieces (f32: four) do not do
#define LN_ROW(TPR, GO, ...)                                                                                   \
    if (l.tpr == TPR) {                                                                                        \
        if (l.nv == 1) return GO<T, TPR, 1>(__VA_ARGS__);                                                      \
        if (l.nv == 2) return GO<T, TPR, 2>(__VA_ARGS__);                                                      \
        if constexpr (sizeof(T) == 4) return GO<T, TPR, 4>(__VA_ARGS__);                                       \
    }
#define LN_DISPATCH(GO, ...)                                                                                   \
    LN_ROW(4, GO, __VA_ARGS__)                                                                                 \
    LN_ROW(16, GO, __VA_ARGS__)                                                                                \
    LN_ROW(64, GO, __VA_ARGS__)                                                                                \
    LN_ROW(256, GO, __VA_ARGS__)                                                                               \
    LN_ROW(512, GO, __VA_ARGS__)

template <typename T> int fwd_t(const LnFwdArgs &a, hipStream_t st) {
    const Layout l = layout_of(Chunk<T>::N, a.D);
    LN_DISPATCH(fwd_go, a, st)
    hipLaunchKernelGGL((k_ln_fwd_wide<T>), dim3((unsigned)(a.B < 4096 ? a.B : 4096)), dim3(256), 0, st, a);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
template <typename T> int bwd_t(const LnBwdArgs &a, int nblk, hipStream_t st) {
    const Layout l = layout_of(Chunk<T>::N, a.D);
    LN_DISPATCH(bwd_go, a, nblk, st)
    hipLaunchKernelGGL((k_ln_bwd_wide<T>), dim3((unsigned)nblk), dim3(256), 0, st, a);
    HIPCHK(hipGetLastError());
    return PS_OK;
}

}  // namespace

int launch_ln_fwd(int type, const LnFwdArgs &a, hipStream_t st) {
    return type == PS_T_F32 ? fwd_t<float>(a, st) : type == PS_T_BF16 ? fwd_t<__bf16>(a, st) : fwd_t<_Float16>(a, st);
}
// Two workgroups a CU: with prefetched rows that is bytes enough in flight, and every further workgroup is a slab more to fold, write and
// add up (bf16, 65536 x 1024: 111 us with 512 workgroups, 130 with 768, 119 with 1024, 128 with 1536; f32, 65536 x 256: 56 / 75 / 77 / 95).
// One a CU where the rows are few: up to 8 row groups a workgroup the slabs cost more than the rows (512 / 256: bf16, 4096 x 512 12.3 / 11.0,
// f16, 4096 x 1024 17.9 / 14.6, f32, 8192 x 256 13.1 / 11.4, bf16, 8192 x 512 14.3 / 14.5; beyond: 16384 x 512 18.3 / 21.2, 32768 x 512
// 25.9 / 35.8); and for rows of 512 lanes, which fill a CU by themselves.
int ln_bwd_blocks(int type, int B, int D) {
    const Layout l = layout_of(type == PS_T_F32 ? 4 : 8, D);
    const int rpb = l.tpr && l.tpr < 256 ? 256 / l.tpr : 1;
    const int64_t need = ((int64_t)B + rpb - 1) / rpb, most = l.tpr > 256 || need <= 2048 ? 256 : 512;
    return (int)(need < most ? need : most);
}
int launch_ln_bwd(int type, const LnBwdArgs &a, int nblk, hipStream_t st) {
    return type == PS_T_F32 ? bwd_t<float>(a, nblk, st) : type == PS_T_BF16 ? bwd_t<__bf16>(a, nblk, st) : bwd_t<_Float16>(a, nblk, st);
}
int launch_grad_reduce(const float *part, int nslab, int64_t n, int B, float *dst, int accum, hipStream_t st) {
    hipLaunchKernelGGL(k_grad_reduce, dim3((unsigned)((n + 63) / 64)), dim3(1024), 0, st, part, nslab, n, B, dst, accum);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
