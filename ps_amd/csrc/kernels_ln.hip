// kernels_ln.hip -- layer normalisation over the rows of a [B][D] activation, forward and backward (gfx950).
//
//   forward   mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps),  y = (x - mean) * rstd * gamma + beta
//   backward  h = (x - mean) * rstd,  p = dy * gamma,
//             dx = skip + rstd * (p - mean(p) - h * mean(p * h)),   dgamma = sum_rows dy * h,   dbeta = sum_rows dy
//
// Both are bound by memory: a row is read once, lies in registers (as it came: 16 bits stay 16 bits) while its sums are formed in two
// passes over them -- the variance from differences to the mean, never from sum x^2 -- and is written once.  All arithmetic is f32.
// A row belongs to TPR lanes (4, 16, 64 of one wave, or a workgroup of 256) that hold NV 16-byte pieces each: a narrow row does not
// idle a wave, a wide one does not spill.  Rows wider than 256 lanes x 32 elements take the kernels that walk the row again (from L2).
#include "kernels_tower.h"

namespace {

constexpr int kMaxEpl = 32;            // elements of a row per lane

template <int TPR> __device__ __forceinline__ float row_sum(float v, float *lds) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if (TPR > 64) {                    // the four waves of the workgroup, in wave order
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    }
    return v;
}

template <typename T, int TPR, int NV>
__global__ __launch_bounds__(256) void k_ln_fwd(LnFwdArgs a) {
    constexpr int VEC = Chunk<T>::N, RPB = 256 / TPR;
    __shared__ float lds[4];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float inv_d = 1.f / (float)a.D;
    float g[NV * VEC], b[NV * VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int c = (t + i * TPR) * VEC + j;
            g[i * VEC + j] = c < a.D ? a.gamma[c] : 0.f;
            b[i * VEC + j] = c < a.D ? a.beta[c] : 0.f;
        }
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.B; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + sub < a.B ? r0 + sub : a.B - 1;      // a lane group behind the last row repeats it and writes nothing
        const T *x = (const T *)a.x + r * a.ldx;
        Chunk<T> v[NV];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i].load(x, (t + i * TPR) * VEC, a.D);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) s += (float)v[i].e[j];
        const float mean = row_sum<TPR>(s, lds) * inv_d;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = (t + i * TPR) * VEC + j < a.D ? (float)v[i].e[j] - mean : 0.f;
                s = fmaf(d, d, s);
            }
        const float rstd = 1.f / sqrtf(row_sum<TPR>(s, lds) * inv_d + a.eps);
        if (r0 + sub >= a.B) continue;
        T *y = (T *)a.y + r * a.ldy;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i].e[j] = (T)fmaf(((float)v[i].e[j] - mean) * rstd, g[i * VEC + j], b[i * VEC + j]);
            v[i].store(y, (t + i * TPR) * VEC, a.D);
        }
        if (a.stats && t == 0) { a.stats[2 * r] = mean; a.stats[2 * r + 1] = rstd; }
    }
}

// rows of any width: one workgroup per row walks it three times
template <typename T>
__global__ __launch_bounds__(256) void k_ln_fwd_wide(LnFwdArgs a) {
    constexpr int VEC = Chunk<T>::N;
    __shared__ float lds[4];
    const float inv_d = 1.f / (float)a.D;
    for (int64_t r = blockIdx.x; r < a.B; r += gridDim.x) {
        const T *x = (const T *)a.x + r * a.ldx;
        T *y = (T *)a.y + r * a.ldy;
        Chunk<T> v;
        float s = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
            v.load(x, (int)c, a.D);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s += (float)v.e[j];
        }
        const float mean = row_sum<256>(s, lds) * inv_d;
        s = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
            v.load(x, (int)c, a.D);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = c + j < a.D ? (float)v.e[j] - mean : 0.f;
                s = fmaf(d, d, s);
            }
        }
        const float rstd = 1.f / sqrtf(row_sum<256>(s, lds) * inv_d + a.eps);
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
            v.load(x, (int)c, a.D);
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (c + j < a.D) v.e[j] = (T)fmaf(((float)v.e[j] - mean) * rstd, a.gamma[c + j], a.beta[c + j]);
            v.store(y, (int)c, a.D);
        }
        if (a.stats && threadIdx.x == 0) { a.stats[2 * r] = mean; a.stats[2 * r + 1] = rstd; }
    }
}

// Every lane keeps the column sums of its own columns over all the rows it sees; a workgroup folds its RPB row groups through LDS and
// writes one slab: no atomics, the same order in every run.
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(256) void k_ln_bwd(LnBwdArgs a) {
    constexpr int VEC = Chunk<T>::N, RPB = 256 / TPR, E = NV * VEC;
    __shared__ float lds[4];
    __shared__ float fold[RPB > 1 ? 256 * VEC : 1];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float inv_d = 1.f / (float)a.D;
    float g[E], sg[E], sb[E];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int c = (t + i * TPR) * VEC + j;
            g[i * VEC + j] = c < a.D ? a.gamma[c] : 0.f;
            sg[i * VEC + j] = 0.f; sb[i * VEC + j] = 0.f;
        }
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.B; r0 += (int64_t)gridDim.x * RPB) {
        const bool live = r0 + sub < a.B;
        const int64_t r = live ? r0 + sub : a.B - 1;
        const T *x = (const T *)a.x + r * a.ldx, *dy = (const T *)a.dy + r * a.lddy;
        Chunk<T> v[NV], w[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) { v[i].load(x, (t + i * TPR) * VEC, a.D); w[i].load(dy, (t + i * TPR) * VEC, a.D); }
        const float mean = a.stats[2 * r], rstd = a.stats[2 * r + 1];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const bool in = live && (t + i * TPR) * VEC + j < a.D;
                const float h = in ? ((float)v[i].e[j] - mean) * rstd : 0.f, d = in ? (float)w[i].e[j] : 0.f, p = d * g[i * VEC + j];
                s1 += p; s2 = fmaf(p, h, s2);
                sg[i * VEC + j] = fmaf(d, h, sg[i * VEC + j]); sb[i * VEC + j] += d;
            }
        if (!a.dx) continue;
        const float m1 = row_sum<TPR>(s1, lds) * inv_d, m2 = row_sum<TPR>(s2, lds) * inv_d;
        if (!live) continue;
        T *dx = (T *)a.dx + r * a.lddx;
        const T *sk = (const T *)a.skip + r * a.ldskip;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * VEC;
            Chunk<T> k;
            k.zero();
            if (a.skip) k.load(sk, c, a.D);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float h = ((float)v[i].e[j] - mean) * rstd, p = (float)w[i].e[j] * g[i * VEC + j];
                k.e[j] = (T)((float)k.e[j] + rstd * (p - m1 - h * m2));
            }
            k.store(dx, c, a.D);
        }
    }
    float *out = a.part + (size_t)blockIdx.x * 2 * a.D;
    for (int w = 0; w < 2; ++w) {
        float *acc = w ? sb : sg;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (RPB > 1) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < VEC; ++j) fold[threadIdx.x * VEC + j] = acc[i * VEC + j];
                __syncthreads();
                if (sub == 0) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        float s = fold[t * VEC + j];
#pragma unroll 1
                        for (int q = 1; q < RPB; ++q) s += fold[(q * TPR + t) * VEC + j];
                        acc[i * VEC + j] = s;
                    }
                }
            }
            if (sub == 0) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const int c = (t + i * TPR) * VEC + j;
                    if (c < a.D) out[(size_t)w * a.D + c] = acc[i * VEC + j];
                }
            }
        }
    }
}

// wide rows: the column sums live in the workgroup's slab (its own columns, its own lane: plain adds)
template <typename T>
__global__ __launch_bounds__(256) void k_ln_bwd_wide(LnBwdArgs a) {
    constexpr int VEC = Chunk<T>::N;
    __shared__ float lds[4];
    const float inv_d = 1.f / (float)a.D;
    float *sg = a.part + (size_t)blockIdx.x * 2 * a.D, *sb = sg + a.D;
    for (int64_t r = blockIdx.x; r < a.B; r += gridDim.x) {
        const bool first = r == blockIdx.x;
        const T *x = (const T *)a.x + r * a.ldx, *dy = (const T *)a.dy + r * a.lddy, *sk = (const T *)a.skip + r * a.ldskip;
        const float mean = a.stats[2 * r], rstd = a.stats[2 * r + 1];
        Chunk<T> v, w, k;
        float s1 = 0.f, s2 = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
            v.load(x, (int)c, a.D); w.load(dy, (int)c, a.D);
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (c + j < a.D) {
                    const float h = ((float)v.e[j] - mean) * rstd, d = (float)w.e[j], p = d * a.gamma[c + j];
                    s1 += p; s2 = fmaf(p, h, s2);
                    sg[c + j] = first ? d * h : fmaf(d, h, sg[c + j]);
                    sb[c + j] = first ? d : sb[c + j] + d;
                }
        }
        if (!a.dx) continue;
        const float m1 = row_sum<256>(s1, lds) * inv_d, m2 = row_sum<256>(s2, lds) * inv_d;
        T *dx = (T *)a.dx + r * a.lddx;
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < a.D; c += 256 * VEC) {
            v.load(x, (int)c, a.D); w.load(dy, (int)c, a.D);
            k.zero();
            if (a.skip) k.load(sk, (int)c, a.D);
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (c + j < a.D) {
                    const float h = ((float)v.e[j] - mean) * rstd, p = (float)w.e[j] * a.gamma[c + j];
                    k.e[j] = (T)((float)k.e[j] + rstd * (p - m1 - h * m2));
                }
            k.store(dx, (int)c, a.D);
        }
    }
}

__global__ __launch_bounds__(256) void k_grad_reduce(const float *__restrict__ part, int nslab, int64_t stride, int64_t n, int B,
                                                     float *__restrict__ dst, int accum) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float s = 0.f;
    for (int z = 0; z < nslab; ++z) s += part[(size_t)z * stride + i];
    s /= (float)B;
    dst[i] = accum ? dst[i] + s : s;
}

// the row layout of a width: lanes per row and pieces per lane (0 lanes: the walking kernel)
struct Layout { int tpr, nv; };
Layout layout_of(int vec, int D) {
    const int chunks = (D + vec - 1) / vec;
    const int tprs[4] = {4, 16, 64, 256};
    for (int i = 0; i < 4; ++i) {
        const int cap = tprs[i] < 64 ? 2 : kMaxEpl / vec;
        if (chunks > tprs[i] * cap) continue;
        int nv = 1;
        while (tprs[i] * nv < chunks) nv *= 2;
        return {tprs[i], nv};
    }
    return {0, 0};
}

template <typename T, int TPR, int NV>
int fwd_go(const LnFwdArgs &a, hipStream_t st) {
    const int64_t need = ((int64_t)a.B + 256 / TPR - 1) / (256 / TPR);
    hipLaunchKernelGGL((k_ln_fwd<T, TPR, NV>), dim3((unsigned)(need < 4096 ? need : 4096)), dim3(256), 0, st, a);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
template <typename T, int TPR, int NV>
int bwd_go(const LnBwdArgs &a, int nblk, hipStream_t st) {
    hipLaunchKernelGGL((k_ln_bwd<T, TPR, NV>), dim3((unsigned)nblk), dim3(256), 0, st, a);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
// every (lanes, pieces) that layout_of can return for the type; NV 8 holds 32 elements only for f32
#define LN_DISPATCH(GO, ...)                                                                                   \
    switch (l.tpr * 16 + l.nv) {                                                                               \
    case 4 * 16 + 1: return GO<T, 4, 1>(__VA_ARGS__);                                                          \
    case 4 * 16 + 2: return GO<T, 4, 2>(__VA_ARGS__);                                                          \
    case 16 * 16 + 1: return GO<T, 16, 1>(__VA_ARGS__);                                                        \
    case 16 * 16 + 2: return GO<T, 16, 2>(__VA_ARGS__);                                                        \
    case 64 * 16 + 1: return GO<T, 64, 1>(__VA_ARGS__);                                                        \
    case 64 * 16 + 2: return GO<T, 64, 2>(__VA_ARGS__);                                                        \
    case 64 * 16 + 4: return GO<T, 64, 4>(__VA_ARGS__);                                                        \
    case 256 * 16 + 2: return GO<T, 256, 2>(__VA_ARGS__);                                                      \
    case 256 * 16 + 4: return GO<T, 256, 4>(__VA_ARGS__);                                                      \
    }                                                                                                          \
    if constexpr (sizeof(T) == 4) {                                                                            \
        if (l.tpr == 64 && l.nv == 8) return GO<T, 64, 8>(__VA_ARGS__);                                        \
        if (l.tpr == 256 && l.nv == 8) return GO<T, 256, 8>(__VA_ARGS__);                                      \
    }

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
int ln_bwd_blocks(int type, int B, int D) {
    const Layout l = layout_of(type == PS_T_F32 ? 4 : 8, D);
    const int rpb = l.tpr ? 256 / l.tpr : 1;
    const int64_t need = ((int64_t)B + rpb - 1) / rpb;
    return (int)(need < 512 ? need : 512);
}
int launch_ln_bwd(int type, const LnBwdArgs &a, int nblk, hipStream_t st) {
    return type == PS_T_F32 ? bwd_t<float>(a, nblk, st) : type == PS_T_BF16 ? bwd_t<__bf16>(a, nblk, st) : bwd_t<_Float16>(a, nblk, st);
}
int launch_grad_reduce(const float *part, int nslab, int64_t stride, int64_t n, int B, float *dst, int accum, hipStream_t st) {
    hipLaunchKernelGGL(k_grad_reduce, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, part, nslab, stride, n, B, dst, accum);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
