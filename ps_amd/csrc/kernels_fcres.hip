// kernels_fcres.hip -- the FC layer with bias, activation and residual in its epilogue, and its gradients (gfx950 matrix cores).
//
//   forward    z = x W + b,  y = act(z) + r
//   backward   dz = dy act'(z),  dx = skip + dz W^T,  dW = x^T dz / B,  db = sum dz / B
//
// Three products: x W and dz W^T are both "NT" (rows of activations times rows of a weight matrix, both contiguous along the sum: the
// store keeps W and its transpose), x^T dz is "TN" (the sum runs over the batch, across the rows of both).  Activations are f32, bf16
// or f16; weights are f32 in the store and are rounded to the activations' type on their way into LDS; sums are f32.
#include "kernels_tower.h"

namespace {

template <typename T> struct Mma;      // one matrix instruction: NI x MI results, KS of the sum
template <> struct Mma<__bf16> {
    typedef bf16x8 frag; typedef f32x4 acc;
    static constexpr int TILE = 16, BK = 64;
    static __device__ __forceinline__ acc mma(frag a, frag b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<_Float16> {
    typedef f16x8 frag; typedef f32x4 acc;
    static constexpr int TILE = 16, BK = 64;
    static __device__ __forceinline__ acc mma(frag a, frag b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<float> {        // a fragment holds 4 steps of 2: the lanes' halves take k = 8 i + 4 h + j, the same for both operands
    typedef f32x4 frag; typedef f32x16 acc;
    static constexpr int TILE = 32, BK = 32;
    static __device__ __forceinline__ acc mma(frag a, frag b, acc c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

// The normal law's tail Q(|z|) = erfc(|z| / sqrt 2) / 2 as 2 to a polynomial of |z|: log2 Q is nearly a parabola, and the polynomial is the
// one of degree 10 whose greatest error of Q on [0, 8], measured against the smaller of 2e-8 and Q / 1024, is least (0.3 of that); it
// falls from there on.  In f32: |error| < 5e-8, the rounding of numbers near 1/2, and below 4e-4 of Q up to 8 (1e-6 up to 2, 6e-6 up to 3,
// 4e-5 up to 4): a 16-bit GELU is its value rounded once down to -8, where it is 5e-15, and an ever smaller number below.  10
// multiply-adds and one exponential: in the epilogue of a product nothing hides them.
__device__ __forceinline__ float normal_tail(float z) {
    const float x = fabsf(z);
    float p = fmaf(-1.76279684e-08f, x, 6.04504919e-07f);
    p = fmaf(p, x, -8.63394234e-06f);
    p = fmaf(p, x, 6.51972878e-05f);
    p = fmaf(p, x, -0.00024829671f);
    p = fmaf(p, x, -5.21555776e-05f);
    p = fmaf(p, x, 0.00699824048f);
    p = fmaf(p, x, -0.0524695776f);
    p = fmaf(p, x, -0.459213197f);
    p = fmaf(p, x, -1.15110493f);
    return __builtin_amdgcn_exp2f(fmaf(p, x, -1.f));
}
// e^-x for 0 <= x <= 128 as 2^t (1 + what t's rounding and log2 e's leave)
__device__ __forceinline__ float exp_minus(float x) {
    const float t = -1.44269504f * x, p = __builtin_amdgcn_exp2f(t);
    return fmaf(p, 0.69314718f * fmaf(-1.92596299e-8f, x, fmaf(-1.44269504f, x, -t)), p);
}
// z / (1 + e^-z) to f32's last bits: with e = e^-|z|, z / (1 + e) above 0 and z e / (1 + e) below, so that nothing overflows, and 1 / (1 + e)
// refined once.  The short form that 16 bits take is off by more the farther z is below 0: 5.5e-7 of the value at -10, 3.9e-6 beyond -40,
// 65 of f32's roundings.  (f32, 32768 x 256 -> 256: 49.5 us by the short form, 51.9 so, 53.0 by expf and a division; 4096 x 429 -> 512
// 23.3 / 24.0 / 24.4.)
__device__ __forceinline__ float silu_f32(float z) {
    const float x = fminf(fabsf(z), 128.f), e = exp_minus(x), d = 1.f + e, r = __builtin_amdgcn_rcpf(d);
    return (z < 0.f ? -x * e : z) * fmaf(r, fmaf(-d, r, 1.f), r);
}
// a product in which 0 times infinity is 0 (a NaN stays one): one instruction, like any product
extern "C" __device__ float mul_zero_wins(float, float) __asm("llvm.amdgcn.fmul.legacy");
template <typename T, int NV> __device__ __forceinline__ void act_apply(float (&v)[NV], int act) {
    if (act == PS_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];        // (a NaN stays one)
    } else if (act == PS_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < NV; ++j)             // z Phi(z) = max(z, 0) - |z| Q(|z|), the first as whole numbers (fmaxf is two instructions)
            v[j] = __int_as_float(max(__float_as_int(v[j]), 0)) - mul_zero_wins(fabsf(v[j]), normal_tail(v[j]));
    } else if (act == PS_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if constexpr (sizeof(T) == 4) v[j] = silu_f32(v[j]);
            else v[j] = mul_zero_wins(v[j], __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * v[j])));      // (0 at -infinity)
    }
}
// dy times GELU' = Phi(z) + z phi(z) or SILU' = s (1 + z (1 - s)), s = 1 / (1 + e^-z).  Both slopes are w(|z|) below 0 and 1 - w(|z|) above:
// the 1 goes into the product's own rounding.  dz is rounded to 16 bits, and every value that a slope's error sends to the other
// neighbour is a whole step in dW's sums.  (With a slope 1e-7 off, dW of 32768 x 1024 -> 4096 with GELU was 6.3e-6 off; so 0.6e-6, where
// f32 formulas with a library's erf leave 3.7e-6.)
__device__ __forceinline__ float slope_below(float z, int act) {             // w; 0 to the last bit beyond 128, where infinity times 0 is not
    if (act == PS_ACT_GELU) return fmaf(fminf(fabsf(z), 128.f) * -0.39894228f, __builtin_amdgcn_exp2f(-0.72134752f * z * z), normal_tail(z));
    // 1 / (1 + e) as r + c, so that 1 - x / (1 + e) is exact at its zero
    const float x = fabsf(z) > 128.f ? 128.f : fabsf(z), e = exp_minus(x), d = 1.f + e;
    const float r = __builtin_amdgcn_rcpf(d), c = r * fmaf(-r, e - (d - 1.f), fmaf(-d, r, 1.f));
    return e * (r + c) * fmaf(-x, c, fmaf(-x, r, 1.f));
}

// workgroup -> tile so that an XCD (workgroup id mod 8) owns a contiguous range of tiles: its L2 then serves the tiles' shared rows
__device__ __forceinline__ int xcd_tile(int id, int n) {
    const int q = n >> 3, r = n & 7, x = id & 7, i = id >> 3;
    return x * q + (x < r ? x : r) + i;
}

// 8 (4) weights of one row as 16 bytes of the activations' type
template <typename T> __device__ __forceinline__ void load_w(Chunk<T> &o, const float *row, int c, int n) {
    if constexpr (sizeof(T) == 4) {
        o.load(row, c, n);
    } else {
        float w[8];
        if (c + 8 <= n) {
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(row + c), hi = *reinterpret_cast<const f32x4 *>(row + c + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) { w[j] = lo[j]; w[4 + j] = hi[j]; }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = c + j < n ? row[c + j] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) o.e[j] = (T)w[j];
    }
}

// ... as they come, and rounded when they go into LDS
template <typename T> struct Weights {
    f32x4 lo, hi;
    __device__ __forceinline__ void load(const float *p) { lo = reinterpret_cast<const f32x4 *>(p)[0]; hi = reinterpret_cast<const f32x4 *>(p)[1]; }
    // zeros behind n; the store's rows are padded to multiples of 16, so a piece that begins in one lies in it
    __device__ __forceinline__ void load_cut(const float *row, int c, int n) {
        load(row + (c < n ? c : 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) { lo[j] = c + j < n ? lo[j] : 0.f; hi[j] = c + 4 + j < n ? hi[j] : 0.f; }
    }
    __device__ __forceinline__ Chunk<T> rounded() const {
        Chunk<T> o;
#pragma unroll
        for (int j = 0; j < 4; ++j) { o.e[j] = (T)lo[j]; o.e[4 + j] = (T)hi[j]; }
        return o;
    }
};
template <> struct Weights<float> {
    Chunk<float> w;
    __device__ __forceinline__ void load(const float *p) { w.u = *reinterpret_cast<const u32x4 *>(p); }
    __device__ __forceinline__ void load_cut(const float *row, int c, int n) {
        load(row + (c < n ? c : 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) w.e[j] = c + j < n ? w.e[j] : 0.f;
    }
    __device__ __forceinline__ Chunk<float> rounded() const { return w; }
};

// A barrier that waits for this wave's LDS traffic and lets its memory loads fly on (the builtin, which the compiler's own wait counting
// sees: behind waits written in assembly it took finished loads for pending ones and waited again where it hurt)
#define PS_WAIT_COUNTS(vm) __builtin_amdgcn_s_waitcnt(((vm) & 15) | 0x70 | (((vm) >> 4) << 14))
#define PS_ORDERED(x)                  \
    do {                               \
        asm volatile("" ::: "memory"); \
        x;                             \
        asm volatile("" ::: "memory"); \
    } while (0)
#define PS_WAIT_LDS() PS_ORDERED(PS_WAIT_COUNTS(63))
#define PS_WAIT_LOADS(n) PS_ORDERED(PS_WAIT_COUNTS(n))      // all but the last n loads have landed, too
#define PS_BARRIER() PS_ORDERED(__builtin_amdgcn_s_barrier())

// One BM x BN tile of the output per workgroup of G groups of 4 waves (2 x 2 each).  LDS rows are 128 bytes of the sum's axis (BK elements), 16-byte
// pieces exchanged by the row's low bits so that the fragment reads of 8 neighbouring rows touch all banks once.  The pieces of the
// next AHEAD steps travel in registers while this step multiplies; two LDS buffers, one barrier a step (which waits for LDS alone, not for
// the loads).
// G > 1: the groups share the sum out -- for outputs of few tiles, whose chain of steps is what a call costs -- and add up through LDS, in
// group order.
// The product is formed transposed (weights as the first operand): a lane then holds 4 neighbouring columns of one row of y.
// Measured: f32, 4096 x 429 -> 512, relu, z kept 21 us (84 TF; matrix units busy 0.64 of the launch, the rest is its start, first loads
// and end; the order and number of accumulators makes no difference), 8192 x 2048 -> 2048 550 us (125 TF, 0.85 of a library's bare
// product); bf16, 4096 x 429 -> 512 10 us.
template <typename T, int BM, int BN, int AHEAD, int G>
__device__ __forceinline__ void fc_nt_tile(const FcNtArgs &a, int tiles_n, int tile, u32x4 *lds) {
    typedef Mma<T> X;
    typedef typename X::frag frag;
    constexpr int CN = Chunk<T>::N, BK = X::BK, TILE = X::TILE, FM = BM / 2 / TILE, FN = BN / 2 / TILE, PA = BM * 8 / 256, PB = BN * 8 / 256;
    const int64_t m0 = (int64_t)(tile / tiles_n) * BM;
    const int n0 = (tile % tiles_n) * BN;
    const int tid = threadIdx.x & 255, grp = G > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
    u32x4 *own = lds + grp * 2 * (BM + BN) * 8;
    u32x4(*sA)[BM * 8] = reinterpret_cast<u32x4(*)[BM * 8]>(own), (*sB)[BN * 8] = reinterpret_cast<u32x4(*)[BN * 8]>(own + 2 * BM * 8);
    const T *pa[PA];
    const float *pb[PB];
    int dst_a[PA], dst_b[PB];
    const int ch = tid & 7;
#pragma unroll
    for (int i = 0; i < PA; ++i) {
        const int row = (tid >> 3) + i * 32;
        const int64_t m = m0 + row < a.M ? m0 + row : a.M - 1;      // rows behind the last: any row, their results go nowhere
        pa[i] = (const T *)a.A + m * a.lda;
        dst_a[i] = row * 8 + (ch ^ (row & 7));
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
        const int row = (tid >> 3) + i * 32, n = n0 + row < a.N ? n0 + row : a.N - 1;
        pb[i] = a.W + (size_t)n * a.ldw;
        dst_b[i] = row * 8 + (ch ^ (row & 7));
    }
    Chunk<T> ra[AHEAD][PA];
    Weights<T> rb[AHEAD][PB];
    auto fetch = [&](int set, int k0) {
        const int k = k0 + ch * CN;
#pragma unroll
        for (int i = 0; i < PA; ++i) ra[set][i].u = *reinterpret_cast<const typename Chunk<T>::unaligned_t *>(pa[i] + k);
#pragma unroll
        for (int i = 0; i < PB; ++i) rb[set][i].load(pb[i] + k);
    };
    auto fetch_cut = [&](int k0) {               // (a.K >= CN)
        const int k = k0 + ch * CN;
#pragma unroll
        for (int i = 0; i < PA; ++i) ra[0][i].load_cut(pa[i], k, a.K);
#pragma unroll
        for (int i = 0; i < PB; ++i) rb[0][i].load_cut(pb[i], k, a.K);
    };
    auto put = [&](int set, int buf) {
#pragma unroll
        for (int i = 0; i < PA; ++i) sA[buf][dst_a[i]] = ra[set][i].u;
#pragma unroll
        for (int i = 0; i < PB; ++i) sB[buf][dst_b[i]] = rb[set][i].rounded().u;
    };
    typename X::acc acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
            for (int e = 0; e < (int)(sizeof(acc[0][0]) / 4); ++e) acc[i][j][e] = 0.f;
    const int lr = lane % TILE, lg = lane / TILE;
    constexpr int GR = (int)(sizeof(acc[0][0]) / 16);            // a lane's results: GR groups of 4 neighbouring columns of one row
    f32x4 bias[FN][GR];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int q = 0; q < GR; ++q) {
            const int n = n0 + wn + i * TILE + q * 8 + lg * 4;
            bias[i][q] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (a.bias) bias[i][q] = *reinterpret_cast<const f32x4 *>(a.bias + (n < a.N ? n : 0));      // (its row is padded to a multiple of 16)
        }
    constexpr int KS = 8 / (64 / TILE);          // fragment steps per LDS row
    auto multiply = [&](int buf) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            frag fa[FM], fb[FN];
            const int c = ks * (64 / TILE) + lg;
#pragma unroll
            for (int j = 0; j < FM; ++j) { const int r = wm + j * TILE + lr; fa[j] = *reinterpret_cast<const frag *>(&sA[buf][r * 8 + (c ^ (r & 7))]); }
#pragma unroll
            for (int i = 0; i < FN; ++i) { const int r = wn + i * TILE + lr; fb[i] = *reinterpret_cast<const frag *>(&sB[buf][r * 8 + (c ^ (r & 7))]); }
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FM; ++j) acc[i][j] = X::mma(fb[i], fa[j], acc[i][j]);
        }
    };
    // the step that K cuts off, if there is one, goes first: behind it no load hides behind a branch
    const int full = a.K / BK, cut = a.K % BK ? 1 : 0, total = full + cut;
    const int lo = total * grp / G, mine = total * (grp + 1) / G - lo, steps = (total + G - 1) / G;      // (with G > 1 every group has a step)
    if (!full) {                                 // nothing but the cut step
        if (a.K >= CN) {
            fetch_cut(0);
        } else {
#pragma unroll
            for (int i = 0; i < PA; ++i) ra[0][i].load(pa[i], ch * CN, a.K);
#pragma unroll
            for (int i = 0; i < PB; ++i) rb[0][i].load_cut(pb[i], ch * CN, a.K);
        }
        put(0, 0);
        PS_WAIT_LDS(); PS_BARRIER();
        multiply(0);
    } else {
        // step s + p lies in buffer p and the next ones in registers or on their way.  The last steps ask again for what is there: the
        // loads are never behind a branch, so the waits know how many of them are younger than those they wait for.
        auto ask = [&](int set, int s) { const int q = lo + (s < mine ? s : mine - 1); fetch(set, (q > cut ? q - cut : 0) * BK); };
        auto half = [&](int s, int p) {
            if (AHEAD > 1) ask(p, s + p + 2); else ask(0, s + p + 1);
            if (G == 1 || s + p < mine) multiply(p);
            put(AHEAD > 1 ? p ^ 1 : 0, p ^ 1);
            PS_WAIT_LDS(); PS_BARRIER();
        };
        if (cut && grp == 0) fetch_cut(full * BK); else ask(0, 0);
        if (AHEAD > 1) ask(1, 1);
        put(0, 0);
        PS_WAIT_LDS(); PS_BARRIER();
        int s = 0;
        for (; s + 2 <= steps; s += 2) { half(s, 0); half(s, 1); }
        if (s < steps) half(s, 0);
    }
    if constexpr (G > 1) {
        constexpr int AE = (int)(sizeof(acc[0][0]) / 4);
        float *sums = reinterpret_cast<float *>(lds) + (wave * 64 + lane);
        if (grp) {
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FM; ++j)
#pragma unroll
                    for (int e = 0; e < AE; ++e) sums[(((grp - 1) * FN + i) * FM + j) * AE * 256 + e * 256] = acc[i][j][e];
        }
        PS_WAIT_LDS(); PS_BARRIER();
        if (grp) return;
#pragma unroll
        for (int g = 0; g < G - 1; ++g)
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FM; ++j)
#pragma unroll
                    for (int e = 0; e < AE; ++e) acc[i][j][e] += sums[((g * FN + i) * FM + j) * AE * 256 + e * 256];
    }
    // epilogue: the residual first -- a load behind a store waits for the store, too
    Quad<T> res[FM][FN][GR];
    if (a.R) {
        const bool whole = n0 + BN <= a.N;
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int64_t m = m0 + wm + j * TILE + lr;
            const T *rr = (const T *)a.R + (m < a.M ? m : a.M - 1) * a.ldr;
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int q = 0; q < GR; ++q) {
                    const int n = n0 + wn + i * TILE + q * 8 + lg * 4;
                    if (whole) res[j][i][q].load(rr + n); else res[j][i][q].load(rr, n, a.N);
                }
        }
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const int64_t m = m0 + wm + j * TILE + lr;
        if (m >= a.M) continue;
        T *y = (T *)a.Y + m * a.ldy, *zr = (T *)a.Z + m * a.ldz;
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int q = 0; q < GR; ++q) {
                const int n = n0 + wn + i * TILE + q * 8 + lg * 4;
                if (n >= a.N) continue;
                float v[4];
                Quad<T> o;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][q * 4 + e] + bias[i][q][e];
                if (a.Z) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) o.e[e] = (T)v[e];
                    o.store(zr, n, a.N);
                }
                act_apply<T>(v, a.act);
                if (a.R)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += (float)res[j][i][q].e[e];
#pragma unroll
                for (int e = 0; e < 4; ++e) o.e[e] = (T)v[e];
                o.store(y, n, a.N);
            }
    }
}
template <typename T, int BM, int BN, int AHEAD, int G>
__global__ __launch_bounds__(256 * G, BM == 64 ? 4 : 2) void k_fc_nt(FcNtArgs a, int tiles_n) {
    __shared__ u32x4 lds[G * 2 * (BM + BN) * 8];
    fc_nt_tile<T, BM, BN, AHEAD, G>(a, tiles_n, xcd_tile(blockIdx.x, gridDim.x), lds);
}

// Few rows (or few tiles): one workgroup of 16 waves per 16 columns and 16 FM rows.  The waves share out the sum in steps and take their
// fragments straight from memory -- the weights in f32, rounded in registers, each read once per row of tiles -- so that a call is two
// dependent trips to memory and not a chain of staged steps; their sums meet in LDS and are added in wave order.
// Bound by latency: 3.3 us on the device for one row of 429 -> 512, 6.6 us for bf16, 16 x 2048 -> 2048 (16.8 MB of weights, 2.5 TB/s).
template <typename T> struct MmaFew {
    static constexpr int KS = 32;
    static __device__ __forceinline__ f32x4 mma(const Chunk<T> &a, const Chunk<T> &b, f32x4 c) {
        typedef typename Mma<T>::frag frag;
        return Mma<T>::mma(__builtin_bit_cast(frag, a.u), __builtin_bit_cast(frag, b.u), c);
    }
};
template <> struct MmaFew<float> {
    static constexpr int KS = 16;
    static __device__ __forceinline__ f32x4 mma(const Chunk<float> &a, const Chunk<float> &b, f32x4 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.e[j], b.e[j], c, 0, 0, 0);
        return c;
    }
};
template <typename T, int FM>
__global__ __launch_bounds__(1024) void k_fc_few(FcNtArgs a, int tiles_n) {
    typedef MmaFew<T> X;
    constexpr int W = 16;
    __shared__ float sums[W][FM * 256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
    const int64_t m0 = (int64_t)(blockIdx.x / tiles_n) * (FM * 16);
    const int n0 = (int)(blockIdx.x % tiles_n) * 16;
    const float *w = a.W + (size_t)(n0 + lr < a.N ? n0 + lr : a.N - 1) * a.ldw;      // (rows behind the last: any row, their results go nowhere)
    const T *x[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const int64_t m = m0 + j * 16 + lr;
        x[j] = (const T *)a.A + (m < a.M ? m : a.M - 1) * a.lda;
    }
    // the thread's result, and what is added to it: asked for first, there when the sums are
    const int64_t m = m0 + (threadIdx.x >> 4);
    const int n = n0 + (threadIdx.x & 15);
    const bool mine = (int)threadIdx.x < FM * 256 && m < a.M && n < a.N;
    float bias = 0.f;
    T res = (T)0.f;
    if (mine && a.bias) bias = a.bias[n];
    if (mine && a.R) res = ((const T *)a.R)[m * a.ldr + n];
    f32x4 acc[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int full = a.K / X::KS, c = lg * Chunk<T>::N;
#pragma unroll 4
    for (int s = wave; s < full; s += W) {
        Chunk<T> fw, fx;
        load_w<T>(fw, w, s * X::KS + c, 0x7fffffff);
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            fx.u = *reinterpret_cast<const typename Chunk<T>::unaligned_t *>(x[j] + s * X::KS + c);
            acc[j] = X::mma(fw, fx, acc[j]);
        }
    }
    if (a.K % X::KS && full % W == wave) {
        Chunk<T> fx[FM];
        Weights<T> fw;
        fw.load_cut(w, full * X::KS + c, a.K);
        if (a.K >= Chunk<T>::N) {
#pragma unroll
            for (int j = 0; j < FM; ++j) fx[j].load_cut(x[j], full * X::KS + c, a.K);
        } else {
#pragma unroll
            for (int j = 0; j < FM; ++j) fx[j].load(x[j], c, a.K);
        }
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[j] = X::mma(fw.rounded(), fx[j], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) *reinterpret_cast<f32x4 *>(&sums[wave][(j * 16 + lr) * 16 + lg * 4]) = acc[j];
    __syncthreads();
    if (!mine) return;
    float v[1] = {0.f};
#pragma unroll
    for (int q = 0; q < W; ++q) v[0] += sums[q][threadIdx.x];
    v[0] += bias;
    if (a.Z) ((T *)a.Z)[m * a.ldz + n] = (T)v[0];
    act_apply<T>(v, a.act);
    if (a.R) v[0] += (float)res;
    ((T *)a.Y)[m * a.ldy + n] = (T)v[0];
}

// The weights of a product in the activations' type, laid out for k_fc_nt_big: rows padded with zeros to a multiple of BK and of BN.  In
// every call -- a copy kept from one call to the next would have to learn of every update: 6 to 8 us for 4.2 M weights (3.5 TB/s).
template <typename T> __global__ __launch_bounds__(256) void k_cast_w(const float *__restrict__ W, int ldw, int N, int K, T *__restrict__ out, int Kp, int Np) {
    const int per = Kp / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)per * Np) return;
    const int n = (int)(i / per), c = (int)(i % per) * 8;
    Chunk<T> o;
    o.zero();
    if (n < N && c < K) load_w<T>(o, W + (size_t)n * ldw, c, K);
    *reinterpret_cast<u32x4 *>(out + (size_t)n * Kp + c) = o.u;
}

constexpr int BIG_M = 256, BIG_K = 64, BIG_GROUP = 8;
typedef __attribute__((address_space(3))) void lds_void;

// 16-bit operands, a 256 x BN tile per workgroup of 8 waves, one workgroup a CU.  BN = 256 (waves
// 2 x 4, 128 x 64 each) asks least of L2 and of LDS per product; BN = 128 (waves 4 x 2, 64 x 64 each) is for outputs of so few tiles
// that half the chip would idle.
// Both operands go straight from memory into LDS (no registers, no conversion: the weights were cast once).
// LDS holds two steps of 64 along the sum, each in four quarters (x's rows by their wave's upper and lower half, the weights' by their
// wave's half too), and a step is four phases, each over a quarter of the wave's tile (16 or 8 matrix instructions):
//      phase 0: read x0, w0 -- x0 w0      1: read w1 -- x0 w1      2: read x1 -- x1 w1      3: x1 w0
// A quarter is free once its phase has read it, and is asked for again -- two steps ahead -- in the phase after that: one quarter per
// phase, five quarters in flight; what a phase reads was asked for five phases ago (the waits count the loads since).
// The two waves of a SIMD work in turn: one reads and asks for memory while the other multiplies; a barrier ends every half phase and
// the second four waves run one half phase behind.
// (A workgroup that walked several tiles, asking for the next one's first quarters before storing, lost: its load counts wait for its
// stores, a new workgroup's do not -- 347 against 326 us for 32768 x 1024 -> 4096 with GELU.)
// LDS rows are 128 bytes, 16-byte pieces exchanged by a row key so that 8 neighbouring lanes of a fragment read touch different banks;
// the exchange is made in the loads' addresses, LDS itself is written in lane order.  A wave's weight rows are dealt to its four
// fragments in groups of 4, so that a lane ends with 16 neighbouring columns of a row of y: whole 128-byte lines per row and wave (1-3 %
// faster than 64 bytes of four lanes per store).
// Rows of x behind the last read as zeros through the buffer's bound; a last step that K does not fill goes through registers, where
// its tail is cut off.
// Measured: bf16, 8192 x 8192 -> 8192 1320 TF, 32768 x 4096 -> 1024 1190 (a library's bare products 1330 and 1240): the clock that the power
// limit leaves bounds these.  32768 x 1024 -> 4096 with GELU and z kept 318 us (865 TF): 16 steps of 64 are 20 us of a tile's 38, its first
// loads, GELU's arithmetic and the stores the rest, and nothing overlaps them: two workgroups a CU of 256 x 128 tiles in steps of 32 do,
// but their loop runs at 990 TF where this one has 1320, and lose (377 us).
template <typename T, int BN>
__global__ __launch_bounds__(512, 2) void k_fc_nt_big(FcNtArgs a, const T *Wc, int Kp, int tiles_m, int tiles_n) {
    typedef Mma<T> X;
    typedef typename X::frag frag;
    constexpr int WN = BN / 64, WM = 8 / WN, HX = BIG_M / WM / 2, FJ = HX / 16;      // waves along n and m; rows and fragments of half a wave's x
    constexpr int QX = 128 * 8, QW = BN / 2 * 8, LX = 2, LW = QW / 512;              // pieces of a quarter, loads of a lane for it
    constexpr int OX[2] = {0, QX + 2 * QW}, OW[2] = {QX, QX + QW};
    // (one array for everything: with several the compiler tells their loads apart and waits for all of them before a read of any)
    __shared__ u32x4 lds[2][2 * QX + 2 * QW];    // [step][x0 | w0 | w1 | x1]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
    const bool second = wave >= 4;
    const int sb = Kp * 2;
    // row q of a quarter: x's row (q / HX) * 2 HX + half * HX + q % HX, the weights' row (q / 32) * 64 + (q / 8 % 4) * 16 + half * 8 + q % 8
    const int q = tid >> 3, pc = tid & 7, ca = (pc ^ (q & 7)) * 16, cb = (pc ^ ((q & 3) | ((q >> 1) & 4))) * 16;
    const int rx = (q / HX) * 2 * HX + q % HX;                                       // x's row of the lane's first piece; the second one's is 128 on
    int va[2][2];                                                                    // in the lane's offset, which the bound is checked with
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) va[h][i] = (int)((rx + i * 128 + h * HX) * a.lda * 2) + ca;
    const int vb = ((q >> 5) * 64 + ((q >> 3) & 3) * 16 + (q & 7)) * sb + cb;
    // an XCD's tiles in groups of BIG_GROUP rows of tiles: what runs on it at one time shares rows of x and of the weights in its L2
    const int tile = xcd_tile(blockIdx.x, gridDim.x), per = BIG_GROUP * tiles_n, g = tile / per, left = tiles_m - g * BIG_GROUP;
    const int gm = left < BIG_GROUP ? left : BIG_GROUP;
    const int64_t m0 = (int64_t)(g * BIG_GROUP + (tile % per) % gm) * BIG_M;
    const int n0 = (tile % per) / gm * BN;
    const T *A0 = (const T *)a.A + m0 * a.lda;
    const int64_t rows = a.M - m0 < BIG_M ? a.M - m0 : BIG_M;
    const auto rsA = __builtin_amdgcn_make_buffer_rsrc((void *)A0, 0, (int)(((rows - 1) * a.lda + a.K) * 2), 0x00020000);
    const auto rsB = __builtin_amdgcn_make_buffer_rsrc((void *)(Wc + (size_t)n0 * Kp), 0, BN * sb, 0x00020000);
    auto ask_x = [&](int t, int half) {
#pragma unroll
        for (int i = 0; i < LX; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsA, (lds_void *)&lds[t & 1][OX[half] + i * 512 + wave * 64], 16, va[half][i], t * 128, 0, 0);
    };
    auto ask_w = [&](int t, int half) {
#pragma unroll
        for (int i = 0; i < LW; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsB, (lds_void *)&lds[t & 1][OW[half] + i * 512 + wave * 64], 16, vb, t * 128 + (i * 128 + half * 8) * sb, 0, 0);
    };
    f32x4 acc[4][2 * FJ];
    const int lr = lane & 15, lg = lane >> 4;
    frag fx[2][FJ], fw[2][4];                    // [step of 32][fragment]
    int ox[2], ow[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        ox[k] = (wm * HX + lr) * 8 + ((k * 4 + lg) ^ (lr & 7));
        const int r = wn * 32 + (lr >> 2) * 8 + (lr & 3);
        ow[k] = r * 8 + ((k * 4 + lg) ^ ((r & 3) | ((r >> 1) & 4)));
    }
    auto read_x = [&](int t, int half) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < FJ; ++j) fx[k][j] = *reinterpret_cast<const frag *>(&lds[t & 1][OX[half] + ox[k] + j * 128]);
    };
    auto read_w = [&](int t, int half) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) fw[k][half * 2 + i] = *reinterpret_cast<const frag *>(&lds[t & 1][OW[half] + ow[k] + i * 32]);
    };
    auto multiply = [&](int hx, int hw) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < FJ; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) acc[hw * 2 + i][hx * FJ + j] = X::mma(fw[k][hw * 2 + i], fx[k][j], acc[hw * 2 + i][hx * FJ + j]);
        __builtin_amdgcn_s_setprio(0);
    };
    auto turn = [&]() { __builtin_amdgcn_sched_barrier(0); __builtin_amdgcn_s_barrier(); __builtin_amdgcn_sched_barrier(0); };
    const int steps = a.K / BIG_K;
    if (steps > 0) { ask_x(0, 0); ask_w(0, 0); ask_w(0, 1); ask_x(0, 1); }
    if (steps > 1) {
        ask_x(1, 0); ask_w(1, 0); ask_w(1, 1);
        PS_WAIT_LOADS(2 * LX + 3 * LW);
    } else {
        PS_WAIT_LOADS(0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2 * FJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    turn();
    if (second) turn();                          // half a phase behind from here on
    int t = 0;
    for (; t < steps - 2; ++t) {
        read_x(t, 0); read_w(t, 0); ask_x(t + 1, 1);
        PS_WAIT_LOADS(3 * LX + 2 * LW); turn(); multiply(0, 0); turn();
        read_w(t, 1); ask_x(t + 2, 0);
        PS_WAIT_LOADS(3 * LX + 2 * LW); turn(); multiply(0, 1); turn();
        read_x(t, 1); ask_w(t + 2, 0);
        PS_WAIT_LOADS(2 * LX + 3 * LW); turn(); multiply(1, 1); turn();
        ask_w(t + 2, 1);
        PS_WAIT_LOADS(2 * LX + 3 * LW); turn(); multiply(1, 0); turn();
    }
    const int n = n0 + wn * 64 + lg * 16;
    f32x4 bias[4];                               // (its row is padded to a multiple of 16)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bias[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (a.bias) bias[e] = reinterpret_cast<const f32x4 *>(a.bias + (n < a.N ? n : 0))[e];
    }
    for (; t < steps; ++t) {                     // the last two: nothing but x1 is left to ask for
        read_x(t, 0); read_w(t, 0);
        if (t + 1 < steps) ask_x(t + 1, 1);
        PS_WAIT_LOADS(0); turn(); multiply(0, 0); turn();
        read_w(t, 1);
        PS_WAIT_LOADS(0); turn(); multiply(0, 1); turn();
        read_x(t, 1);
        PS_WAIT_LOADS(0); turn(); multiply(1, 1); turn();
        turn(); multiply(1, 0); turn();
    }
    if (!second) turn();
    if (a.K % BIG_K) {                           // every wave has read all there was; all eight in step from here on
        ask_w(steps, 0); ask_w(steps, 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = rx + (i & 1) * 128 + (i >> 1) * HX;
            const T *row = A0 + (r < rows ? r : rows - 1) * a.lda;                   // (rows behind the last: their results go nowhere)
            Chunk<T> c;
            if (a.K >= Chunk<T>::N) c.load_cut(row, steps * BIG_K + ca / 2, a.K);
            else c.load(row, ca / 2, a.K);
            lds[steps & 1][OX[i >> 1] + (i & 1) * 512 + tid] = c.u;
        }
        PS_WAIT_LOADS(0);
        turn();
        read_x(steps, 0); read_w(steps, 0); read_w(steps, 1);
        multiply(0, 0); multiply(0, 1);
        read_x(steps, 1);
        multiply(1, 1); multiply(1, 0);
    }
    if (n >= a.N) return;
    Chunk<T> res[2 * FJ][2];                     // the residual first: a load behind a store waits for the store, too
    if (a.R) {
        const bool whole = n0 + BN <= a.N;
#pragma unroll
        for (int j = 0; j < 2 * FJ; ++j) {
            const int64_t m = m0 + wm * 2 * HX + j * 16 + lr;
            const T *row = (const T *)a.R + (m < a.M ? m : a.M - 1) * a.ldr;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (whole) res[j][h].u = *reinterpret_cast<const typename Chunk<T>::unaligned_t *>(row + n + h * 8);
                else if (a.N >= Chunk<T>::N) res[j][h].load_cut(row, n + h * 8, a.N);
                else res[j][h].load(row, n + h * 8, a.N);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 2 * FJ; ++j) {
        const int64_t m = m0 + wm * 2 * HX + j * 16 + lr;
        if (m >= a.M) continue;
        float v[16];
        Chunk<T> o;
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = acc[e >> 2][j][e & 3] + bias[e >> 2][e & 3];
        if (a.Z) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int e = 0; e < 8; ++e) o.e[e] = (T)v[h * 8 + e];
                o.store((T *)a.Z + m * a.ldz, n + h * 8, a.N);
            }
        }
        act_apply<T>(v, a.act);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (a.R)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[h * 8 + e] += (float)res[j][h].e[e];
#pragma unroll
            for (int e = 0; e < 8; ++e) o.e[e] = (T)v[h * 8 + e];
            o.store((T *)a.Y + m * a.ldy, n + h * 8, a.N);
        }
    }
}

// dz = dy act'(z), rounded to the type; z NULL: a copy.  dz's rows are 16-byte pieces, zeros behind the width.  Bound by memory: bf16,
// 32768 x 4096 147 us, 5.5 TB/s.  (dz is read by both products of the pass, many times over: forming it on the way into each of them
// would cost its arithmetic once per tile.)
template <typename T> __global__ __launch_bounds__(256) void k_act_grad(const T *dy, int64_t lddy, const T *z, int64_t ldz, T *dz, int64_t lddz, int M, int N, int act) {
    const int64_t per = lddz / Chunk<T>::N, total = per * M;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / per;
        const int c = (int)(i % per) * Chunk<T>::N;
        Chunk<T> d, v;
        d.zero();
        if (c < N) {
            if (!z && N >= Chunk<T>::N) d.load_cut(dy + m * lddy, c, N); else d.load(dy + m * lddy, c, N);
            if (z) {
                v.load(z + m * ldz, c, N);
                if (act == PS_ACT_RELU) {
#pragma unroll
                    for (int j = 0; j < Chunk<T>::N; ++j) d.e[j] = (float)v.e[j] > 0.f ? d.e[j] : (T)0.f;
                } else {
                    float o[Chunk<T>::N], any = 0.f;
#pragma unroll
                    for (int j = 0; j < Chunk<T>::N; ++j) {
                        const float g = (float)d.e[j], zz = (float)v.e[j], w = slope_below(zz, act);
                        o[j] = zz < 0.f ? g * w : fmaf(-g, w, g);
                        any += o[j];
                    }
                    if (any != any)                  // an infinite dy is one behind a slope, too: inf - inf w is not
#pragma unroll
                        for (int j = 0; j < Chunk<T>::N; ++j) {
                            const float g = (float)d.e[j], zz = (float)v.e[j], w = slope_below(zz, act);
                            o[j] = g * (zz < 0.f ? w : 1.f - w);
                        }
#pragma unroll
                    for (int j = 0; j < Chunk<T>::N; ++j) d.e[j] = (T)o[j];
                }
            }
        }
        *reinterpret_cast<u32x4 *>(dz + m * lddz + c) = d.u;
    }
}

// One BT x BT tile of x^T dz over one part of the batch.  LDS holds the rows as they lie in memory; 16-bit fragments need 8 values
// down a column, which the transposing LDS read delivers (16 lanes read 4 rows x 16 columns and get a column's 4 rows each).  The order
// of the sum inside a step is the same for both operands and otherwise free.  32-byte pieces are exchanged by a row key: the 8 rows
// that 32 lanes of a transposing read touch lie in different banks.  The workgroups of the first row of tiles also multiply dz by a
// fragment of ones: db, row K of the slab.
// Two steps ahead in registers, as in k_fc_nt: the step that M cuts off goes first, its pieces cut off in registers.  Columns behind K and
// N are any values, their results go nowhere: whole pieces of them are read from the row's start, and a piece that the width cuts off
// (edge) runs on into the next row -- so the step with the last row counts as cut off too.  NARROW: widths below a piece, whose pieces
// could run past more than one row: every load element by element.
template <typename T, int BT, bool NARROW>
__device__ __forceinline__ void fc_tn_tile(const FcTnArgs &a, int tiles_n, int split, int tile, bool edge, u32x4 *lds) {
    typedef Mma<T> X;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int CN = Chunk<T>::N, ROWS = F32 ? 32 : 64, PER = BT / CN, P = ROWS * PER / 256, TILE = X::TILE, FK = BT / 2 / TILE, FN = BT / 2 / TILE;
    constexpr int BUF = ROWS * PER;              // pieces of one operand's step; lds: [step][x | dz]
    const int k0 = (tile / tiles_n) * BT, n0 = (tile % tiles_n) * BT;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wk = (wave >> 1) * (BT / 2), wn = (wave & 1) * (BT / 2);
    auto key = [](int row) { return F32 ? 0 : BT == 128 ? row & 7 : (row >> 1) & 3; };
    // this part's rows: whole steps, dealt evenly
    const int64_t all = ((int64_t)a.M + ROWS - 1) / ROWS, s_lo = all * split / a.nsplit, s_hi = all * (split + 1) / a.nsplit;
    const int cut = s_hi * ROWS > a.M || (edge && s_hi == all) ? 1 : 0, steps = (int)(s_hi - s_lo), full = steps - cut;
    Chunk<T> rx[2][P], rd[2][P];
    int dst[P], cx[P], cd[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int q = tid + i * 256, row = q / PER, c = q % PER;
        dst[i] = row * PER + (c ^ (key(row) << 1));
        cx[i] = k0 + c * CN; cd[i] = n0 + c * CN;
        if (!NARROW) { cx[i] = cx[i] < a.K ? cx[i] : 0; cd[i] = cd[i] < a.N ? cd[i] : 0; }
    }
    auto fetch = [&](int set, int64_t step) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int64_t m = (s_lo + step) * ROWS + (tid + i * 256) / PER;
            const T *px = (const T *)a.X + m * a.ldx, *pd = (const T *)a.D + m * a.ldd;
            if constexpr (NARROW) { rx[set][i].load(px, cx[i], a.K); rd[set][i].load(pd, cd[i], a.N); }
            else {
                rx[set][i].u = *reinterpret_cast<const typename Chunk<T>::unaligned_t *>(px + cx[i]);
                rd[set][i].u = *reinterpret_cast<const typename Chunk<T>::unaligned_t *>(pd + cd[i]);
            }
        }
    };
    auto fetch_cut = [&]() {                     // rows behind the last are zeros
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int64_t m = (s_hi - 1) * ROWS + (tid + i * 256) / PER;
            if constexpr (NARROW) {
                rx[0][i].zero(); rd[0][i].zero();
                if (m < a.M) { rx[0][i].load((const T *)a.X + m * a.ldx, cx[i], a.K); rd[0][i].load((const T *)a.D + m * a.ldd, cd[i], a.N); }
            } else {
                const int64_t r = m < a.M ? m : a.M - 1;
                rx[0][i].load_cut((const T *)a.X + r * a.ldx, cx[i], a.K); rd[0][i].load_cut((const T *)a.D + r * a.ldd, cd[i], a.N);
                const u32x4 none = {0u, 0u, 0u, 0u};
                rx[0][i].u = m < a.M ? rx[0][i].u : none; rd[0][i].u = m < a.M ? rd[0][i].u : none;
            }
        }
    };
    auto put = [&](int set, int buf) {
#pragma unroll
        for (int i = 0; i < P; ++i) { lds[buf * 2 * BUF + dst[i]] = rx[set][i].u; lds[(buf * 2 + 1) * BUF + dst[i]] = rd[set][i].u; }
    };
    typename X::acc acc[FK][FN], accb[FN];
    constexpr int AE = (int)(sizeof(accb[0]) / 4);
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < AE; ++e) {
            accb[j][e] = 0.f;
#pragma unroll
            for (int i = 0; i < FK; ++i) acc[i][j][e] = 0.f;
        }
    typename X::frag ones;
#pragma unroll
    for (int j = 0; j < CN; ++j) ones[j] = (T)1.f;
    const bool do_bias = k0 == 0 && wk == 0;
    const int lr = lane % TILE, lg = lane / TILE;
    auto multiply = [&](int buf) {
        const u32x4 *sx = lds + buf * 2 * BUF, *sd = sx + BUF;
#pragma unroll
        for (int ks = 0; ks < (F32 ? 4 : 2); ++ks) {
            typename X::frag fk[FK], fn[FN];
            if constexpr (F32) {
                const float *lx = reinterpret_cast<const float *>(sx), *ld = reinterpret_cast<const float *>(sd);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = ks * 8 + e * 2 + lg;
#pragma unroll
                    for (int i = 0; i < FK; ++i) fk[i][e] = lx[row * BT + wk + i * TILE + lr];
#pragma unroll
                    for (int j = 0; j < FN; ++j) fn[j][e] = ld[row * BT + wn + j * TILE + lr];
                }
            } else {
                typedef __attribute__((address_space(3))) s16x4 lds4;
                union { typename X::frag f; s16x4 h[2]; } u;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const short *base = reinterpret_cast<const short *>(w ? sd : sx);
#pragma unroll
                    for (int i = 0; i < FK; ++i) {
                        const int piece = ((w ? wn : wk) >> 4) + i;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int row = ks * 32 + h * 16 + lg * 4 + (lr >> 2);
                            u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(base + row * BT + (piece ^ key(row)) * 16 + (lr & 3) * 4));
                        }
                        if (w) fn[i] = u.f; else fk[i] = u.f;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < FK; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = X::mma(fk[i], fn[j], acc[i][j]);
            if (do_bias) {
                if constexpr (F32) {             // (f32 matrix instructions are the slow ones: plain adds, a lane's own rows)
#pragma unroll
                    for (int j = 0; j < FN; ++j) accb[j][0] += (fn[j][0] + fn[j][1]) + (fn[j][2] + fn[j][3]);
                } else {
#pragma unroll
                    for (int j = 0; j < FN; ++j) accb[j] = X::mma(ones, fn[j], accb[j]);
                }
            }
        }
    };
    if (cut) fetch_cut(); else fetch(0, 0);
    if (!full) {                                 // (a part has at least one step)
        put(0, 0);
        PS_WAIT_LDS(); PS_BARRIER();
        multiply(0);
    } else {
        auto ask = [&](int set, int step) { fetch(set, step < steps ? step - cut : full - 1); };
        auto half = [&](int s, int p) {
            ask(p, s + p + 2);
            multiply(p);
            put(p ^ 1, p ^ 1);
            PS_WAIT_LDS(); PS_BARRIER();
        };
        ask(1, 1);
        put(0, 0);
        PS_WAIT_LDS(); PS_BARRIER();
        int s = 0;
        for (; s + 2 <= steps; s += 2) { half(s, 0); half(s, 1); }
        if (s < steps) half(s, 0);
    }
    // one part: the result itself
    float *part = a.nsplit == 1 ? a.dst : a.part + (size_t)split * (size_t)(a.K + a.nbias) * a.N;
    auto leave = [&](size_t i, float v) {
        if (a.nsplit == 1) { v /= (float)a.M; if (a.accum) v = part[i] + v; }
        part[i] = v;
    };
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        if constexpr (F32) accb[j][0] += __shfl_xor(accb[j][0], 32);
        const int n = n0 + wn + j * TILE + lr;
        if (n >= a.N) continue;
#pragma unroll
        for (int i = 0; i < FK; ++i)
#pragma unroll
            for (int e = 0; e < AE; ++e) {
                const int k = k0 + wk + i * TILE + (e >> 2) * 8 + lg * 4 + (e & 3);
                if (k < a.K) leave((size_t)k * a.N + n, acc[i][j][e]);
            }
        if (do_bias && lg == 0) leave((size_t)a.K * a.N + n, accb[j][0]);
    }
}
template <typename T, int BT> constexpr int kTnLds = 4 * (sizeof(T) == 4 ? 32 : 64) * BT / Chunk<T>::N;
template <typename T, int BT> __device__ __forceinline__ void fc_tn_part(const FcTnArgs &a, int tiles_n, int tiles, int id, u32x4 *lds) {
    constexpr int CN = Chunk<T>::N;
    const int split = id / tiles, tile = id % tiles;
    const bool edge = (a.K % CN && (tile / tiles_n + 1) * BT > a.K) || (a.N % CN && (tile % tiles_n + 1) * BT > a.N);
    if (a.K < CN || a.N < CN) fc_tn_tile<T, BT, true>(a, tiles_n, split, tile, edge, lds);
    else fc_tn_tile<T, BT, false>(a, tiles_n, split, tile, edge, lds);
}
template <typename T, int BT>
__global__ __launch_bounds__(256, BT == 64 ? 3 : 2) void k_fc_tn(FcTnArgs a, int tiles_n, int tiles) {
    __shared__ u32x4 lds[kTnLds<T, BT>];
    fc_tn_part<T, BT>(a, tiles_n, tiles, xcd_tile(blockIdx.x, gridDim.x), lds);
}
// Measured (k_fc_tn with k_fc_grad_reduce): f32, 8192 x 1024 -> 1024, both gradients 313 us (110 TF).
// dW's tiles and, behind them, dx's, in one launch: where neither fills the chip they run side by side, and there is one start and one end
// less (two launches / one: bf16, 4096 x 512 -> 256 with relu 24.7 / 21.5 us, 4096 x 429 -> 512 with GELU 30.2 / 25.4; f32 40.8 / 35.4 and
// 57.2 / 52.0; where the chip is full no difference: f32, 16384 x 429 -> 512 169.7 / 168.2, bf16, 100000 x 64 -> 64 38.2 / 38.5).
template <typename T>
__global__ __launch_bounds__(256, 3) void k_fc_both(FcTnArgs t, int t_tiles_n, int t_tiles, int t_blocks, FcNtArgs a, int tiles_n) {
    __shared__ u32x4 lds[kTnLds<T, 64> > 2 * 128 * 8 ? kTnLds<T, 64> : 2 * 128 * 8];
    const int id = blockIdx.x;
    if (id < t_blocks) fc_tn_part<T, 64>(t, t_tiles_n, t_tiles, xcd_tile(id, t_blocks), lds);
    else fc_nt_tile<T, 64, 64, 2, 1>(a, tiles_n, xcd_tile(id - t_blocks, gridDim.x - t_blocks), lds);
}

// The transposing LDS read.  As a function of a restrict pointer: the compiler then knows what it reads, and does not wait for every load
// on its way into LDS in front of it (which made every phase of k_fc_tn_big a round trip to memory).
__device__ __forceinline__ s16x4 read_transposed(const short *__restrict__ p) {
    typedef __attribute__((address_space(3))) s16x4 lds4;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)p);
}

// x^T dz, 16-bit: the same machine as k_fc_nt_big with the batch as the sum's axis, 256 x 256 of dW per workgroup over one part of the
// batch.  A step is 64 rows of both operands; a quarter holds their columns 128 h .. 128 h + 127, so its rows are 256 contiguous bytes.
// Fragments need 8 values down a column: two transposing LDS reads (16 lanes read 4 rows x 16 columns and get a column's 4 rows each;
// both operands take the batch in the same order, which is all the sum needs).  32-byte pieces are exchanged by the row's low 3 bits,
// which are the lane's own, the same in every read.
// db is dz times a fragment of ones: every workgroup of a row of tiles, and of it one of the two wave rows, takes its share of the
// steps, so that no workgroup is the slow one; each leaves its own row behind dW's in the slab.
// Columns behind K and N, and rows behind the part's last, are sent out of the buffer's bounds: zeros.
// Measured: bf16, 32768 x 1024 -> 4096 248 us with its reduction (1107 TF; a library's bare product 346 us), matrix units busy 0.63, LDS 0.23.
template <typename T>
__global__ __launch_bounds__(512, 2) void k_fc_tn_big(FcTnArgs a, int tiles_k, int tiles_n) {
    typedef Mma<T> X;
    typedef typename X::frag frag;
    constexpr int Q = 64 * 16;
    constexpr int OX[2] = {0, 3 * Q}, OW[2] = {Q, 2 * Q};
    __shared__ u32x4 lds[2][4 * Q];              // [step][x0 | w0 | w1 | x1] (w: dz)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 2, wn = wave & 3;
    const bool second = wave >= 4;
    const int tiles = tiles_k * tiles_n, id = xcd_tile(blockIdx.x, gridDim.x), split = id / tiles, tile = id % tiles;
    // (the shorter side first: what an XCD runs at one time is nearer a square and shares more of both operands in its L2)
    const int kt = tiles_k < tiles_n ? tile % tiles_k : tile / tiles_n, k0 = kt * 256, n0 = (tiles_k < tiles_n ? tile / tiles_k : tile % tiles_n) * 256;
    const int64_t all = ((int64_t)a.M + 63) / 64, s_lo = all * split / a.nsplit, s_hi = all * (split + 1) / a.nsplit;
    const int64_t m_lo = s_lo * 64, m_hi = s_hi * 64 < a.M ? s_hi * 64 : a.M;
    const int steps = (int)(s_hi - s_lo), tail = (int)(m_hi - m_lo) - (steps - 1) * 64;      // rows of the last step
    const auto rsX = __builtin_amdgcn_make_buffer_rsrc((void *)((const T *)a.X + m_lo * a.ldx), 0, (int)(((m_hi - m_lo - 1) * a.ldx + a.Kload) * 2), 0x00020000);
    const auto rsW = __builtin_amdgcn_make_buffer_rsrc((void *)((const T *)a.D + m_lo * a.ldd), 0, (int)(((m_hi - m_lo - 1) * a.ldd + a.Nload) * 2), 0x00020000);
    // piece tid of the first 32 rows of a quarter and of the second: row tid / 16 (+ 32), its 16 bytes exchanged within the row
    const int row = tid >> 4, col = ((((tid & 15) >> 1) ^ (row & 7)) * 2 + (tid & 1)) * 8;
    constexpr int OUT = 0x7ffffff0;
    int vx[2], vw[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        vx[h] = k0 + h * 128 + col < a.Kload ? (int)(row * a.ldx + k0 + h * 128 + col) * 2 : OUT;
        vw[h] = n0 + h * 128 + col < a.Nload ? (int)(row * a.ldd + n0 + h * 128 + col) * 2 : OUT;
    }
    const int sx = (int)a.ldx * 64, sw = (int)a.ldd * 64;                    // bytes of 32 rows
    auto ask = [&](int t, const __amdgpu_buffer_rsrc_t &rs, int v, int s32, int at) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int vv = t == steps - 1 && row + i * 32 >= tail ? OUT : v;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void *)&lds[t & 1][at + i * 512 + wave * 64], 16, vv, (2 * t + i) * s32, 0, 0);
        }
    };
    auto ask_x = [&](int t, int half) { ask(t, rsX, vx[half], sx, OX[half]); };
    auto ask_w = [&](int t, int half) { ask(t, rsW, vw[half], sw, OW[half]); };
    f32x4 acc[4][8], accb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        accb[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int lr = lane & 15, lg = lane >> 4, key = (lg & 1) * 4 + (lr >> 2), lo = (lg * 4 + (lr >> 2)) * 128 + (lr & 3) * 4;
    int ox[4], ow[2];                            // in 16-bit values
#pragma unroll
    for (int j = 0; j < 4; ++j) ox[j] = lo + ((wm * 4 + j) ^ key) * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) ow[i] = lo + ((wn * 2 + i) ^ key) * 16;
    frag fx[2][4], fw[2][4], fv[2][2], ones;     // [half step][fragment]; fv: the next step's w0, read ahead of its step
#pragma unroll
    for (int e = 0; e < 8; ++e) ones[e] = (T)1.f;
    auto column = [&](const short *base, int k) {
        union { frag f; s16x4 h[2]; } u;
#pragma unroll
        for (int h = 0; h < 2; ++h) u.h[h] = read_transposed(base + (k * 32 + h * 16) * 128);
        return u.f;
    };
    auto read_x = [&](int t, int half) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) fx[k][j] = column((const short *)&lds[t & 1][OX[half]] + ox[j], k);
    };
    auto read_w1 = [&](int t) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) fw[k][2 + i] = column((const short *)&lds[t & 1][OW[1]] + ow[i], k);
    };
    auto read_w0 = [&](int t) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) fv[k][i] = column((const short *)&lds[t & 1][OW[0]] + ow[i], k);
    };
    auto take_w0 = [&]() {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) fw[k][i] = fv[k][i];
    };
    auto multiply = [&](int hx, int hw) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) acc[hw * 2 + i][hx * 4 + j] = X::mma(fw[k][hw * 2 + i], fx[k][j], acc[hw * 2 + i][hx * 4 + j]);
        __builtin_amdgcn_s_setprio(0);
    };
    auto turn = [&]() { __builtin_amdgcn_sched_barrier(0); __builtin_amdgcn_s_barrier(); __builtin_amdgcn_sched_barrier(0); };
    int next_b = kt * 2 + wm;                    // the next step whose dz this wave adds up
    auto add_up = [&](int t, int hw) {
        if (t != next_b) return;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) accb[hw * 2 + i] = X::mma(fw[k][hw * 2 + i], ones, accb[hw * 2 + i]);
        if (hw == 1) next_b += 2 * tiles_k;
    };
    // The transposing reads are twice as many as k_fc_nt_big's plain ones, and a phase should not hold more of them than the other waves'
    // matrix instructions cover: w0 is read in the phase before its step (16, 8, 16, 8 reads a phase instead of 24, 8, 16, 0).
    ask_w(0, 0); ask_x(0, 0); ask_w(0, 1); ask_x(0, 1);
    if (steps > 1) {
        ask_w(1, 0); ask_x(1, 0); ask_w(1, 1);
        PS_WAIT_LOADS(10);
    } else {
        PS_WAIT_LOADS(0);
    }
    turn();
    if (second) turn();
    read_w0(0);
    int t = 0;
    for (; t < steps - 2; ++t) {
        read_x(t, 0); ask_x(t + 1, 1);
        PS_WAIT_LOADS(10); turn(); take_w0(); multiply(0, 0); add_up(t, 0); turn();
        read_w1(t); ask_w(t + 2, 0);
        PS_WAIT_LOADS(10); turn(); multiply(0, 1); add_up(t, 1); turn();
        read_x(t, 1); ask_x(t + 2, 0);
        PS_WAIT_LOADS(10); turn(); multiply(1, 1); turn();
        read_w0(t + 1); ask_w(t + 2, 1);
        PS_WAIT_LOADS(10); turn(); multiply(1, 0); turn();
    }
    for (; t < steps; ++t) {
        read_x(t, 0);
        if (t + 1 < steps) ask_x(t + 1, 1);
        PS_WAIT_LOADS(0); turn(); take_w0(); multiply(0, 0); add_up(t, 0); turn();
        read_w1(t);
        PS_WAIT_LOADS(0); turn(); multiply(0, 1); add_up(t, 1); turn();
        read_x(t, 1);
        PS_WAIT_LOADS(0); turn(); multiply(1, 1); turn();
        if (t + 1 < steps) read_w0(t + 1);
        PS_WAIT_LOADS(0); turn(); multiply(1, 0); turn();
    }
    if (!second) turn();
    float *part = a.part + (size_t)split * (size_t)(a.K + a.nbias) * a.N;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = n0 + (i >> 1) * 128 + wn * 32 + (i & 1) * 16 + lg * 4;
        if (n >= a.N) continue;
        auto row = [&](int k, const f32x4 &v) {
            Quad<float> o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o.e[e] = v[e];
            o.store(part + (size_t)k * a.N, n, a.N);
        };
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int k = k0 + (j >> 2) * 128 + wm * 64 + (j & 3) * 16 + lr;
            if (k < a.K) row(k, acc[i][j]);
        }
        if (lr == 0) row(a.K + kt * 2 + wm, accb[i]);
    }
}

// The slabs' sum and mean: dW over the parts, db over the parts and their rows.  A wave takes 256 neighbouring elements (4 a lane) and 8
// slabs at a time: 15 us for 4 slabs of 1024 x 4096 (5.6 TB/s, from the Infinity Cache).  W = 1: every wave its own elements; W = 4
// and 16, many slabs: the waves of a workgroup share them out and are added in wave order.  The workgroups behind dW's do db, 64 columns each.
template <int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void k_fc_grad_reduce(FcTnArgs a, int dw_blocks) {
    typedef f32x4 f32x4_at4 __attribute__((aligned(4)));
    __shared__ f32x4 sums[W == 1 ? 4 : W][64];
    const int64_t n = (int64_t)a.K * a.N, slab = (int64_t)(a.K + a.nbias) * a.N;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int WAVES = W == 1 ? 4 : W;
    auto finish = [&](int64_t i, float s) { s /= (float)a.M; a.dst[i] = a.accum ? a.dst[i] + s : s; };
    if ((int)blockIdx.x < dw_blocks) {
        const int64_t i = (W == 1 ? ((int64_t)blockIdx.x * 4 + wave) : (int64_t)blockIdx.x) * 256 + lane * 4;
        const int64_t ic = i + 4 <= n ? i : n >= 4 ? n - 4 : 0;              // (n < 4: the elements behind dW are db's, in bounds)
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        for (int z0 = W == 1 ? 0 : wave; z0 < a.nsplit; z0 += 8 * W) {
            f32x4 v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = *reinterpret_cast<const f32x4_at4 *>(a.part + (z0 + q * W < a.nsplit ? z0 + q * W : a.nsplit - 1) * slab + ic);
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (z0 + q * W < a.nsplit) s += v[q];
        }
        if constexpr (W > 1) {
            sums[wave][lane] = s;
            __syncthreads();
            if (wave) return;
#pragma unroll
            for (int w = 1; w < W; ++w) s += sums[w][lane];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)              // (a lane at dW's end read from n - 4 on and keeps what is its own)
            if (ic + e >= i && ic + e < n) finish(ic + e, s[e]);
        return;
    }
    const int col = ((int)blockIdx.x - dw_blocks) * 64 + lane, cc = col < a.N ? col : a.N - 1, rows = a.nsplit * a.nbias;
    float s = 0.f;
    for (int z0 = wave; z0 < rows; z0 += 8 * WAVES) {
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int z = z0 + q * WAVES < rows ? z0 + q * WAVES : rows - 1;
            v[q] = a.part[(z / a.nbias) * slab + n + (int64_t)(z % a.nbias) * a.N + cc];
        }
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (z0 + q * WAVES < rows) s += v[q];
    }
    sums[wave][lane][0] = s;
    __syncthreads();
    if (wave || col >= a.N) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += sums[w][lane][0];
    finish(n + col, s);
}

int grid_ok(int64_t blocks) {
    return blocks * 256 < (1ll << 32) ? PS_OK : ps_set_err(PS_E_UNSUPPORTED, "the batch needs more workgroups than one launch has");
}

template <typename T, int BM, int BN, int AHEAD, int G> int nt_go(const FcNtArgs &a, hipStream_t st) {
    const int tiles_n = cdiv(a.N, BN);
    const int64_t blocks = (int64_t)tiles_n * cdiv(a.M, BM);
    PSCHK(grid_ok(blocks));
    hipLaunchKernelGGL((k_fc_nt<T, BM, BN, AHEAD, G>), dim3((unsigned)blocks), dim3(256 * G), 0, st, a, tiles_n);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
template <typename T>
int ag_t(int act, const void *dy, int64_t lddy, const void *z, int64_t ldz, void *dz, int64_t lddz, int M, int N, hipStream_t st) {
    const int64_t blocks = (lddz / Chunk<T>::N * M + 255) / 256;
    hipLaunchKernelGGL((k_act_grad<T>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st, (const T *)dy, lddy, (const T *)z, ldz,
                       (T *)dz, lddz, M, N, act);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
// Whether and how a product takes k_fc_nt_big.  Its loads want 16-byte pieces and its offsets 31 bits; rows that start elsewhere are
// copied first, which a product of 256 columns or more pays for (bf16, 20000 x 1001 -> 1001 relu: 118 us without, 79 with).
// 128 columns cost 0.6 of 256 (measured on full chips), so they win where they halve the rounds of the 256 CUs; below half a round of
// 128 columns the small tiles win (4096 x 1024 -> 512, 64 tiles: 20 us by 256 x 128, 14 by 64 x 64), below a quarter for long sums
// (500 x 4096 -> 4096, 64 tiles: 64 / 132; 1000 x 4096 -> 1024, 32 tiles: 53 / 31).
struct NtPlan { int bn = 0; bool pack = false; };
NtPlan nt_plan(int type, const FcNtArgs &a) {
    NtPlan p;
    if (type == PS_T_F32 || a.K > (1 << 21)) return p;
    p.pack = (uintptr_t)a.A % 16 || a.lda % 8 || a.lda > (1 << 21);
    const int64_t tm = cdiv(a.M, BIG_M), t2 = tm * cdiv(a.N, 256), t1 = tm * cdiv(a.N, 128);
    if (t1 < (a.K >= 4096 ? 64 : 128) || t1 >= (1 << 30) || (p.pack && a.N < 256)) return p;
    p.bn = 10 * cdiv(t2, 256) <= 6 * cdiv(t1, 256) ? 256 : 128;
    return p;
}
template <typename T, int BN> int nt_big(FcNtArgs a, bool pack, char *ws, hipStream_t st) {
    const int Kp = (int)round_up(a.K, BIG_K), Np = (int)round_up(a.N, BN), tiles_n = Np / BN, tiles_m = cdiv(a.M, BIG_M);
    const int64_t pieces = (int64_t)Kp / 8 * Np;
    PSCHK(grid_ok(cdiv(pieces, 256)));
    PSCHK(grid_ok(2ll * tiles_m * tiles_n));
    hipLaunchKernelGGL((k_cast_w<T>), dim3((unsigned)cdiv(pieces, 256)), dim3(256), 0, st, a.W, a.ldw, a.N, a.K, (T *)ws, Kp, Np);
    if (pack) {
        char *x = ws + round_up((int64_t)Kp * Np * 2, 256);
        PSCHK((ag_t<T>(PS_ACT_NONE, a.A, a.lda, nullptr, 0, x, Kp, a.M, a.K, st)));
        a.A = x; a.lda = a.K = Kp;
    }
    hipLaunchKernelGGL((k_fc_nt_big<T, BN>), dim3((unsigned)(tiles_m * tiles_n)), dim3(512), 0, st, a, (const T *)ws, Kp, tiles_m, tiles_n);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
template <typename T, int FM> int few_go(const FcNtArgs &a, hipStream_t st) {
    const int tiles_n = cdiv(a.N, 16);
    const int64_t blocks = (int64_t)tiles_n * cdiv(a.M, FM * 16);
    PSCHK(grid_ok(4 * blocks));
    hipLaunchKernelGGL((k_fc_few<T, FM>), dim3((unsigned)blocks), dim3(1024), 0, st, a, tiles_n);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
// Which kernel takes a product that k_fc_nt_big does not (us, few rows' kernel / 64 x 64 tiles).  Too few tiles for the chip leave the
// tiles' chain of staged steps bare: bf16, 64 tiles, 128 x 2048 -> 2048: 11 / 18; 128 tiles, 1000 x 1000 -> 500: 12 / 10; f32, whose steps
// are four times as long, 128 tiles, 2000 x 2000 -> 200: 35 / 42; 234 tiles, 2442 x 3688 -> 324: 116 / 76.
// 128 x 128 tiles only where they fill the two a CU twice (f32: 8192 x 2048 -> 2048 592 by 64, 533 by 128; 20000 x 300 -> 300 46 / 53;
// 2442 x 324 -> 3688 78 / 92).
// One tile a CU and a long sum, 16-bit: four groups of waves share it (1000 x 4096 -> 1024: 47 us by one group, 31 by four; with 512 tiles
// 55 / 57; with a sum of 2048 21 / 20, of 1024 11 / 12; f32, bound by its matrix instructions, only loses: 26 / 34 for 4096 x 429 -> 512).
enum NtKind { NT_FEW, NT_128, NT_64_SPLIT, NT_64 };
template <typename T> NtKind nt_kind(const FcNtArgs &a) {
    const int64_t t128 = (int64_t)cdiv(a.M, 128) * cdiv(a.N, 128), t64 = (int64_t)cdiv(a.M, 64) * cdiv(a.N, 64);
    if (a.M <= 64 || t64 < (sizeof(T) == 4 ? 200 : 100)) return NT_FEW;
    if (t128 >= 1024) return NT_128;
    return sizeof(T) == 2 && t64 <= 256 && a.K >= 2048 ? NT_64_SPLIT : NT_64;
}
template <typename T> int nt_t(const FcNtArgs &a, hipStream_t st) {
    const NtKind k = nt_kind<T>(a);
    if (k == NT_FEW) {
        // more rows a workgroup read the weights less often, fewer fill the chip: as many as leave 160 workgroups (us by 64 / 32 / 16 rows
        // and how many workgroups: bf16, 64 x 2048 -> 2048 11.2 (128) / 7.6 (256); f32, 146 x 1979 -> 246 17.1 (48) / 9.8 (80) / 7.5 (160),
        // 128 x 1024 -> 512 10.8 (64) / 6.9 (128) / 5.0 (256); f16, 2000 x 2000 -> 40 10.0 (96) / 7.3 (189) / 10.0 (375))
        const int64_t tn = cdiv(a.N, 16);
        if (a.M > 32 && tn * cdiv(a.M, 64) >= 160) return few_go<T, 4>(a, st);
        if (a.M > 16 && tn * cdiv(a.M, 32) >= 160) return few_go<T, 2>(a, st);
        return few_go<T, 1>(a, st);
    }
    if (k == NT_128) return nt_go<T, 128, 128, sizeof(T) == 4 ? 2 : 1, 1>(a, st);
    if constexpr (sizeof(T) == 2) {
        if (k == NT_64_SPLIT) return nt_go<T, 64, 64, 2, 4>(a, st);
    }
    return nt_go<T, 64, 64, 2, 1>(a, st);
}
template <typename T, int BT> int tn_go(const FcTnArgs &a, hipStream_t st) {
    const int tiles_n = cdiv(a.N, BT), tiles = tiles_n * cdiv(a.K, BT);
    const int64_t blocks = (int64_t)tiles * a.nsplit;
    PSCHK(grid_ok(blocks));
    hipLaunchKernelGGL((k_fc_tn<T, BT>), dim3((unsigned)blocks), dim3(256), 0, st, a, tiles_n, tiles);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
template <typename T> int tn_t(const FcTnArgs &a, hipStream_t st) { return a.tile == 128 ? tn_go<T, 128>(a, st) : tn_go<T, 64>(a, st); }
template <typename T> int tn_big(const FcTnArgs &a, hipStream_t st) {
    const int tiles_n = cdiv(a.N, 256), tiles_k = cdiv(a.K, 256);
    const int64_t blocks = (int64_t)tiles_n * tiles_k * a.nsplit;
    PSCHK(grid_ok(2 * blocks));
    hipLaunchKernelGGL((k_fc_tn_big<T>), dim3((unsigned)blocks), dim3(512), 0, st, a, tiles_k, tiles_n);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
}  // namespace

size_t fc_nt_workspace(int type, const FcNtArgs &a) {
    const NtPlan p = nt_plan(type, a);
    if (!p.bn) return 0;
    const int64_t Kp = round_up(a.K, BIG_K), w = round_up(Kp * round_up(a.N, p.bn) * 2, 256);
    return (size_t)(w + (p.pack ? Kp * a.M * 2 : 0));
}
int launch_fc_nt(int type, const FcNtArgs &a, char *ws, hipStream_t st) {
    const NtPlan p = nt_plan(type, a);
    if (p.bn == 256) return type == PS_T_BF16 ? nt_big<__bf16, 256>(a, p.pack, ws, st) : nt_big<_Float16, 256>(a, p.pack, ws, st);
    if (p.bn == 128) return type == PS_T_BF16 ? nt_big<__bf16, 128>(a, p.pack, ws, st) : nt_big<_Float16, 128>(a, p.pack, ws, st);
    return type == PS_T_F32 ? nt_t<float>(a, st) : type == PS_T_BF16 ? nt_t<__bf16>(a, st) : nt_t<_Float16>(a, st);
}
int launch_act_grad(int type, int act, const void *dy, int64_t lddy, const void *z, int64_t ldz, void *dz, int64_t lddz, int M, int N, hipStream_t st) {
    return type == PS_T_F32    ? ag_t<float>(act, dy, lddy, z, ldz, dz, lddz, M, N, st)
           : type == PS_T_BF16 ? ag_t<__bf16>(act, dy, lddy, z, ldz, dz, lddz, M, N, st)
                               : ag_t<_Float16>(act, dy, lddy, z, ldz, dz, lddz, M, N, st);
}
// How dW is taken apart: a.tile, a.nsplit, a.nbias, and what has to be copied into 16-byte pieces first (pack_x, pack_d: the caller lays
// rows of 8-element multiples out and tells where).  The 256 tiles: such pieces, offsets of 31 bits inside a part, parts of at least 16
// steps, one workgroup for each of the 256 CUs; a copy is paid for from 256 columns of the other operand on.  The smaller ones: two
// workgroups a CU, no part shorter than four steps, and 128 only where parts stay eight steps long -- shorter ones are all start and end
// (bf16, 4096 x 429 -> 512: 34 us in parts of 4 steps of 128, 24 by 64; 16384 x 1001 -> 1001 in parts of 32: 159 / 343).  16-bit parts below 12
// steps: one workgroup a CU, whose slabs are half as many (two / one: bf16, both gradients of 4096 x 512 -> 256 19.2 / 16.5 us, of
// 4096 x 429 -> 512 24.0 / 21.5, dW alone 16.1 / 14.4 and 19.5 / 18.5; f32, whose steps are long, 49.8 / 59.6).
void fc_tn_plan(int type, FcTnArgs &a) {
    const bool f32 = type == PS_T_F32;
    const int64_t big = (int64_t)cdiv(a.N, 256) * cdiv(a.K, 256), steps = cdiv(a.M, 64);
    a.pack_x = (uintptr_t)a.X % 16 || a.ldx % 8 || a.K % 8;
    a.pack_d = (uintptr_t)a.D % 16 || a.ldd % 8 || (a.D && a.N % 8);         // (D NULL: dz, which will lie in pieces in any case)
    a.Kload = (int)round_up(a.K, 8); a.Nload = (int)round_up(a.N, 8);
    if (!f32 && big * steps >= 2048 && !(a.pack_x && a.N < 256) && !(a.pack_d && a.K < 256)) {
        int64_t s = big >= 256 ? 1 : 256 / big;
        if (s > steps / 16) s = steps / 16 > 0 ? steps / 16 : 1;
        const int64_t lx = a.pack_x ? a.Kload : a.ldx, ld = a.pack_d ? a.Nload : a.ldd;
        if ((cdiv(steps, s) + 1) * 64 * (lx > ld ? lx : ld) * 2 < (1ll << 31) - 64) { a.tile = 256; a.nsplit = (int)s; a.nbias = 2 * cdiv(a.K, 256); return; }
    }
    a.pack_x = a.pack_d = 0;
    const int64_t st = cdiv(a.M, f32 ? 32 : 64);
    a.nbias = 1;
    for (a.tile = 128;; a.tile = 64) {
        const int64_t tiles = (int64_t)cdiv(a.N, a.tile) * cdiv(a.K, a.tile);
        int64_t s = 512 / tiles;                 // (rounded down: one workgroup too many is a round too many)
        if (!f32 && a.tile == 64 && st < 12 * s && tiles < 256) s = 256 / tiles;
        if (s > st / 4) s = st / 4;
        a.nsplit = (int)(s < 1 ? 1 : s);
        if (a.tile == 64 || st >= 8 * a.nsplit) return;
    }
}
namespace {
int tn_reduce(const FcTnArgs &a, hipStream_t st) {
    if (a.nsplit * a.nbias == 1) return PS_OK;               // (the kernel has left the result itself)
    const int64_t n = (int64_t)a.K * a.N;
    const int db = cdiv(a.N, 64);
    if (a.nsplit >= 16 && n < 256 * 1024) {                  // (from one workgroup of four waves for each CU on they need not share)
        // up to 32 slabs are one trip of four waves (16 slabs, 512 x 256: the whole pass 19.3 us, 22.3 by sixteen), more want sixteen
        // (390 slabs, 64 x 64: 40.2 / 37.2)
        const int64_t dw = (n + 255) / 256;
        PSCHK(grid_ok(4 * (dw + db)));
        if (a.nsplit <= 32) hipLaunchKernelGGL(k_fc_grad_reduce<4>, dim3((unsigned)(dw + db)), dim3(256), 0, st, a, (int)dw);
        else hipLaunchKernelGGL(k_fc_grad_reduce<16>, dim3((unsigned)(dw + db)), dim3(1024), 0, st, a, (int)dw);
    } else {
        const int64_t dw = (n + 1023) / 1024;
        PSCHK(grid_ok(dw + db));
        hipLaunchKernelGGL(k_fc_grad_reduce<1>, dim3((unsigned)(dw + db)), dim3(256), 0, st, a, (int)dw);
    }
    HIPCHK(hipGetLastError());
    return PS_OK;
}
template <typename T> int both_go(const FcNtArgs &a, const FcTnArgs &t, hipStream_t st) {
    const int tn = cdiv(t.N, 64), tt = tn * cdiv(t.K, 64), tiles_n = cdiv(a.N, 64);
    const int64_t tb = (int64_t)tt * t.nsplit, blocks = tb + (int64_t)tiles_n * cdiv(a.M, 64);
    PSCHK(grid_ok(blocks));
    hipLaunchKernelGGL((k_fc_both<T>), dim3((unsigned)blocks), dim3(256), 0, st, t, tn, tt, (int)tb, a, tiles_n);
    HIPCHK(hipGetLastError());
    return PS_OK;
}
}  // namespace

int launch_fc_tn(int type, const FcTnArgs &a, hipStream_t st) {
    if (a.tile == 256) PSCHK(type == PS_T_BF16 ? tn_big<__bf16>(a, st) : tn_big<_Float16>(a, st));
    else PSCHK(type == PS_T_F32 ? tn_t<float>(a, st) : type == PS_T_BF16 ? tn_t<__bf16>(a, st) : tn_t<_Float16>(a, st));
    return tn_reduce(a, st);
}
bool fc_both_ok(int type, const FcNtArgs &a, const FcTnArgs &t) {
    return t.tile == 64 && !nt_plan(type, a).bn && (type == PS_T_F32 ? nt_kind<float>(a) : nt_kind<__bf16>(a)) == NT_64;
}
int launch_fc_both(int type, const FcNtArgs &a, const FcTnArgs &t, hipStream_t st) {
    PSCHK(type == PS_T_F32 ? both_go<float>(a, t, st) : type == PS_T_BF16 ? both_go<__bf16>(a, t, st) : both_go<_Float16>(a, t, st));
    return tn_reduce(t, st);
}
