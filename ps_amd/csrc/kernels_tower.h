// kernels_tower.h -- the residual tower's operators (layer normalisation; FC with bias, activation and residual): argument structs and
// launchers (kernels_ln.hip, kernels_fcres.hip) behind the entry points of ps_tower.hip, and the typed loads and stores they share.
#pragma once
#include "ps_common.h"

struct LnFwdArgs {
    const void *x; int64_t ldx;
    void *y; int64_t ldy;
    const float *gamma, *beta;         // [D] each (rows 0 and 1 of the layer's W')
    float *stats;                      // [B][2] mean, 1 / sqrt(var + eps), or NULL
    int B, D;
    float eps;
};
struct LnBwdArgs {
    const void *x; int64_t ldx;
    const void *dy; int64_t lddy;
    const void *skip; int64_t ldskip;  // NULL: none
    void *dx; int64_t lddx;            // NULL: parameter gradients only
    const float *gamma, *stats;
    float *part;                       // [nblk][2][D]: every workgroup's column sums of dy * h and dy
    int B, D;
};
int launch_ln_fwd(int type, const LnFwdArgs &a, hipStream_t st);
int ln_bwd_blocks(int type, int B, int D);             // workgroups (= slabs of part) of launch_ln_bwd
int launch_ln_bwd(int type, const LnBwdArgs &a, int nblk, hipStream_t st);

// dst[i] = (accum ? dst[i] : 0) + (sum over z of part[z * n + i]) / B        (fixed order of z)
int launch_grad_reduce(const float *part, int nslab, int64_t n, int B, float *dst, int accum, hipStream_t st);

// Y[m][n] = act(sum_k A[m][k] * Wr[n][k] + bias[n]) + R[m][n], Z = the pre-activation; Wr f32, rounded to the activations' type on the way
struct FcNtArgs {
    const void *A; int64_t lda;
    const float *W; int ldw;           // [N][ldw], rows padded to a multiple of 16, 16-byte aligned
    const float *bias;                 // [N] or NULL
    const void *R; int64_t ldr;        // NULL: none
    void *Z; int64_t ldz;              // NULL: none
    void *Y; int64_t ldy;
    int M, N, K, act;
};
size_t fc_nt_workspace(int type, const FcNtArgs &a);                        // bytes of ws that launch_fc_nt needs, 256-byte aligned
int launch_fc_nt(int type, const FcNtArgs &a, char *ws, hipStream_t st);
// dz = dy * act'(z), rounded to the type (act NONE: a copy); rows of lddz elements, a multiple of 8, 16-byte aligned, zeros behind N
int launch_act_grad(int type, int act, const void *dy, int64_t lddy, const void *z, int64_t ldz, void *dz, int64_t lddz, int M, int N, hipStream_t st);
// dst[k][n] = (accum ? dst[k][n] : 0) + (sum over m of X[m][k] * D[m][n]) / M, k < K; row K: of D[m][n].  Through slabs of parts of m,
// part[nsplit][K + nbias][N], the nbias rows behind: shares of the sum of D[m][n].
struct FcTnArgs {
    const void *X; int64_t ldx;
    const void *D; int64_t ldd;        // D NULL before the plan: rows in 16-byte pieces, ldd a multiple of 8, zeros behind N
    int M, K, N;
    int tile, nsplit, nbias;           // filled by fc_tn_plan, and ...
    int pack_x, pack_d, Kload, Nload;  // ... X / D have to be replaced by a copy in rows of Kload / Nload elements (launch_act_grad, act NONE)
    float *part, *dst;
    int accum;
};
void fc_tn_plan(int type, FcTnArgs &a);
int launch_fc_tn(int type, const FcTnArgs &a, hipStream_t st);
// both products of a backward pass in one launch, where both are of few tiles
bool fc_both_ok(int type, const FcNtArgs &a, const FcTnArgs &t);
int launch_fc_both(int type, const FcNtArgs &a, const FcTnArgs &t, hipStream_t st);

#ifdef __HIPCC__
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));
template <int SIZE> struct AtElem { typedef u32x4_at2 v; };
template <> struct AtElem<4> { typedef u32x4_at4 v; };
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_at2 __attribute__((aligned(2)));
template <int SIZE> struct AtElem4 { typedef u32x2_at2 v; };      // 4 elements
template <> struct AtElem4<4> { typedef u32x4_at4 v; };

// 16 bytes of one row in registers: 4 f32 or 8 16-bit values.  A row may start at any multiple of its element's size (odd row strides,
// views into wider rows): the type's alignment says so and the memory unit takes such a load whole.
template <typename T> struct Chunk {
    static constexpr int N = 16 / (int)sizeof(T);
    typedef typename AtElem<(int)sizeof(T)>::v unaligned_t;
    union { u32x4 u; T e[N]; };
    __device__ __forceinline__ void zero() { u = u32x4{0u, 0u, 0u, 0u}; }
    // elements [c, c + N) of a row of n elements; zeros behind its end
    __device__ __forceinline__ void load(const T *row, int c, int n) {
        if (c + N <= n) { u = *reinterpret_cast<const unaligned_t *>(row + c); return; }
        zero();
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c + j < n) e[j] = row[c + j];
    }
    // the same without a branch, for n >= N: the piece that the row's end cuts off is read further to the left and shifted down (a load
    // behind a branch waits by itself, and these are often a call's first)
    __device__ __forceinline__ void load_cut(const T *row, int c, int n) {
        const int at = c < n - N ? c : n - N;
        u = *reinterpret_cast<const unaligned_t *>(row + at);
        shift_down(c - at);
    }
    // element s comes first, zeros last
    __device__ __forceinline__ void shift_down(int s) {
        constexpr int ODD = sizeof(T) == 2 ? 1 : 0;                          // log2 of the elements in a word
        if constexpr (ODD)
            u = s & 1 ? u32x4{__builtin_amdgcn_alignbit(u[1], u[0], 16), __builtin_amdgcn_alignbit(u[2], u[1], 16), __builtin_amdgcn_alignbit(u[3], u[2], 16), u[3] >> 16} : u;
        u = (s >> ODD) & 1 ? u32x4{u[1], u[2], u[3], 0u} : u;
        u = (s >> ODD) & 2 ? u32x4{u[2], u[3], 0u, 0u} : u;
        u = s >= N ? u32x4{0u, 0u, 0u, 0u} : u;
    }
    __device__ __forceinline__ void store(T *row, int c, int n) const {
        if (c + N <= n) { *reinterpret_cast<unaligned_t *>(row + c) = u; return; }
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c + j < n) row[c + j] = e[j];
    }
};
// 4 values of one row, at any alignment of theirs
template <typename T> struct Quad {
    typedef typename AtElem4<(int)sizeof(T)>::v bits_t;
    T e[4];
    __device__ __forceinline__ void load(const T *p) { const bits_t b = *reinterpret_cast<const bits_t *>(p); __builtin_memcpy(e, &b, 4 * sizeof(T)); }
    __device__ __forceinline__ void load(const T *row, int c, int n) {
        if (c + 4 <= n) { const bits_t b = *reinterpret_cast<const bits_t *>(row + c); __builtin_memcpy(e, &b, 4 * sizeof(T)); return; }
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = c + j < n ? row[c + j] : (T)0.f;
    }
    __device__ __forceinline__ void store(T *row, int c, int n) const {
        if (c + 4 <= n) { bits_t b; __builtin_memcpy(&b, e, 4 * sizeof(T)); *reinterpret_cast<bits_t *>(row + c) = b; return; }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < n) row[c + j] = e[j];
    }
};
#endif
