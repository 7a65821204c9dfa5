// ps_tower.hip -- the residual tower's operators of the C ABI (ps_ln_*, ps_fc_res_*): argument checks, the store's parameters and
// workspace, and the launches.  Kernels: kernels_ln.hip, kernels_fcres.hip.
#include <string.h>

#include "kernels_tower.h"
#include "ps_store.h"

namespace {

int type_size(int type) { return type == PS_T_F32 ? 4 : 2; }

// a [B][w] operand of the call: its device pointer, row stride and width in elements
struct Mat { const char *name; const void *p; int64_t ld; int64_t w; };

// does any element of a lie where one of b does?  Two views into the same wide rows interleave without touching: equal strides are
// compared by their columns, everything else by its range.
bool overlap(const Mat &a, const Mat &b, int64_t B, int es) {
    if (!a.p || !b.p) return false;
    const uint64_t pa = (uint64_t)(uintptr_t)a.p, pb = (uint64_t)(uintptr_t)b.p;
    const uint64_t ea = pa + (uint64_t)((B - 1) * a.ld + a.w) * es, eb = pb + (uint64_t)((B - 1) * b.ld + b.w) * es;
    if (ea <= pb || eb <= pa) return false;
    if (a.ld != b.ld || B == 1) return true;
    const uint64_t pitch = (uint64_t)a.ld * es, off = pb >= pa ? (pb - pa) % pitch : (pitch - (pa - pb) % pitch) % pitch;      // b's first column, from a's
    return off < (uint64_t)a.w * es || off + (uint64_t)b.w * es > pitch;
}
bool same(const Mat &a, const Mat &b) { return a.p == b.p && a.ld == b.ld; }

int check_mat(const Mat &m, int64_t B, int es) {
    if (!m.p) return PS_OK;
    if (m.ld < m.w) return ps_set_err(PS_E_BAD_ARG, "%s: row stride %lld < width %lld", m.name, (long long)m.ld, (long long)m.w);
    if (m.ld > (1ll << 40) / B) return ps_set_err(PS_E_BAD_ARG, "%s: %lld rows of stride %lld are beyond the device's memory", m.name, (long long)B, (long long)m.ld);
    if ((uintptr_t)m.p % es) return ps_set_err(PS_E_BAD_ARG, "%s is not aligned to its elements", m.name);
    return PS_OK;
}
int check_out(const Mat &out, const Mat &in, int64_t B, int es, bool may_be_same = false) {
    if (!overlap(out, in, B, es) || (may_be_same && same(out, in))) return PS_OK;
    return ps_set_err(PS_E_BAD_ARG, "%s overlaps %s", out.name, in.name);
}
// an f32 output of n contiguous values beside [B][w] operands
int check_f32(const char *name, const float *p, int64_t n, std::initializer_list<Mat> others, int64_t B, int es) {
    if (!p) return PS_OK;
    if ((uintptr_t)p % 4) return ps_set_err(PS_E_BAD_ARG, "%s is not aligned to its elements", name);
    for (const Mat &m : others) {
        if (!m.p) continue;
        const uint64_t pa = (uint64_t)(uintptr_t)p, pm = (uint64_t)(uintptr_t)m.p;
        if (pa + (uint64_t)n * 4 > pm && pm + (uint64_t)((B - 1) * m.ld + m.w) * es > pa) return ps_set_err(PS_E_BAD_ARG, "%s overlaps %s", name, m.name);
    }
    return PS_OK;
}

int check_call(ps_store *s, int type, int B) {
    if (!s) return ps_set_err(PS_E_BAD_ARG, "store is NULL");
    if (type != PS_T_F32 && type != PS_T_BF16 && type != PS_T_F16) return ps_set_err(PS_E_BAD_ARG, "unknown type %d", type);
    if (B <= 0) return ps_set_err(PS_E_BAD_ARG, "bad batch %d", B);
    return PS_OK;
}
int find_ln(ps_store *s, int layer, FcParams **out) {
    if (layer < 0 || layer >= (int)s->ln.size() || !s->ln[layer].present) return ps_set_err(PS_MISSING, "ln%d absent", layer);
    *out = &s->ln[layer];
    return PS_OK;
}
int find_fc(ps_store *s, int layer, FcParams **out) {
    if (layer < 0 || layer >= (int)s->fc.size() || !s->fc[layer].present) return ps_set_err(PS_MISSING, "fc%d absent", layer);
    *out = &s->fc[layer];
    return PS_OK;
}
int check_act(int act) {
    if (act == PS_ACT_SIGMOID) return ps_set_err(PS_E_UNSUPPORTED, "the clipped sigmoid is the head's activation (ps_fc_forward)");
    if (act != PS_ACT_NONE && act != PS_ACT_RELU && act != PS_ACT_GELU && act != PS_ACT_SILU) return ps_set_err(PS_E_BAD_ARG, "unknown activation %d", act);
    return PS_OK;
}

// store_enter; a fused step's last join cannot be recorded (its event lies outside the graph) and must not be lost either
int tower_enter(ps_store *s) {
    if (s->pending_ev && stream_is_capturing(s->stream))
        return ps_set_err(PS_E_STATE, "a training step is still to be joined: call ps_store_sync before a graph is recorded");
    return store_enter(s);
}

// `need` bytes of workspace for one call; its contents are dead when the call's launches are done
int workspace(ps_store *s, size_t need, char **out) {
    ps_store::TowerWs &w = s->tower;
    const bool rec = stream_is_capturing(s->stream);
    if (need > w.cap) {
        if (rec) return ps_set_err(PS_E_STATE, "the workspace would have to grow while a graph is recorded: run the call once eagerly first");
        RtGuard rt_guard;
        const size_t cap = (need + need / 4 + 4095) & ~(size_t)4095;
        if (w.p && w.recorded) {                 // a recorded graph points to it: it stays until the store goes
            try { w.retired.push_back(w.p); } catch (...) { return ps_set_err(PS_E_HIP, "out of host memory"); }
        } else if (w.p) {
            HIPCHK(hipStreamSynchronize(s->stream));
            (void)hipFree(w.p);
            s->bytes -= (int64_t)w.cap;
        }
        w.p = nullptr; w.cap = 0; w.recorded = false;
        HIPCHK(hipMalloc((void **)&w.p, cap));
        w.cap = cap;
        s->bytes += (int64_t)cap;
    }
    w.recorded = w.recorded || rec;
    *out = w.p;
    return PS_OK;
}

// where a parameter gradient goes: the caller's buffer (overwritten) or the layer's pending sum
int grad_target(ps_store *s, FcParams &p, float *grad_dev, float **dst, int *accum) {
    if (grad_dev) { *dst = grad_dev; *accum = 0; return PS_OK; }
    if (stream_is_capturing(s->stream))
        return ps_set_err(PS_E_UNSUPPORTED, "the pending gradient's count lives on the host: give grad_dev while a graph is recorded");
    if (!p.pending) PSCHK(store_dev_alloc(s, (void **)&p.pending, sizeof(float) * (size_t)(p.K + 1) * p.N, true));
    *dst = p.pending; *accum = p.pending_cnt > 0 ? 1 : 0;
    return PS_OK;
}

}  // namespace

extern "C" int ps_ln_forward(ps_store_t *s, int layer, int type, const void *x_dev, int64_t ldx, int B, float eps, void *y_dev, int64_t ldy,
                             float *stats_dev) {
    RoctxRange roctx_range("ps_ln_forward");
    PSCHK(check_call(s, type, B));
    if (!x_dev || !y_dev) return ps_set_err(PS_E_BAD_ARG, "null argument");
    if (!(eps >= 0.f)) return ps_set_err(PS_E_BAD_ARG, "eps must not be negative");
    FcParams *p;
    PSCHK(find_ln(s, layer, &p));
    const int es = type_size(type);
    const Mat x = {"x_dev", x_dev, ldx, p->N}, y = {"y_dev", y_dev, ldy, p->N};
    PSCHK(check_mat(x, B, es));
    PSCHK(check_mat(y, B, es));
    PSCHK(check_out(y, x, B, es, true));
    PSCHK(check_f32("stats_dev", stats_dev, 2ll * B, {x, y}, B, es));
    PSCHK(tower_enter(s));
    LnFwdArgs a;
    a.x = x_dev; a.ldx = ldx; a.y = y_dev; a.ldy = ldy; a.gamma = p->W; a.beta = p->W + p->ldw; a.stats = stats_dev;
    a.B = B; a.D = p->N; a.eps = eps;
    return launch_ln_fwd(type, a, s->stream);
}

extern "C" int ps_ln_backward(ps_store_t *s, int layer, int type, const void *x_dev, int64_t ldx, const float *stats_dev, const void *dy_dev,
                              int64_t lddy, int B, const void *skip_dev, int64_t ldskip, void *dx_dev, int64_t lddx, float *grad_dev) {
    RoctxRange roctx_range("ps_ln_backward");
    PSCHK(check_call(s, type, B));
    if (!x_dev || !stats_dev || !dy_dev) return ps_set_err(PS_E_BAD_ARG, "null argument");
    FcParams *p;
    PSCHK(find_ln(s, layer, &p));
    const int es = type_size(type), D = p->N;
    const Mat x = {"x_dev", x_dev, ldx, D}, dy = {"dy_dev", dy_dev, lddy, D}, sk = {"skip_dev", skip_dev, ldskip, D}, dx = {"dx_dev", dx_dev, lddx, D};
    for (const Mat *m : {&x, &dy, &sk, &dx}) PSCHK(check_mat(*m, B, es));
    if (skip_dev && !dx_dev) return ps_set_err(PS_E_BAD_ARG, "skip_dev without dx_dev");
    PSCHK(check_out(dx, x, B, es));
    PSCHK(check_out(dx, dy, B, es, true));
    PSCHK(check_out(dx, sk, B, es, true));
    PSCHK(check_f32("grad_dev", grad_dev, 2ll * D, {x, dy, sk, dx}, B, es));
    PSCHK(check_f32("stats_dev", stats_dev, 2ll * B, {dx}, B, es));
    if (grad_dev && stats_dev + 2ll * B > grad_dev && grad_dev + 2ll * D > stats_dev) return ps_set_err(PS_E_BAD_ARG, "grad_dev overlaps stats_dev");
    PSCHK(tower_enter(s));
    float *dst;
    int accum;
    PSCHK(grad_target(s, *p, grad_dev, &dst, &accum));
    const int nblk = ln_bwd_blocks(type, B, D);
    char *ws;
    PSCHK(workspace(s, sizeof(float) * 2 * (size_t)D * nblk, &ws));
    LnBwdArgs a;
    a.x = x_dev; a.ldx = ldx; a.dy = dy_dev; a.lddy = lddy; a.skip = skip_dev; a.ldskip = skip_dev ? ldskip : 0; a.dx = dx_dev; a.lddx = lddx;
    a.gamma = p->W; a.stats = stats_dev; a.part = (float *)ws; a.B = B; a.D = D;
    PSCHK(launch_ln_bwd(type, a, nblk, s->stream));
    PSCHK(launch_grad_reduce(a.part, nblk, 2ll * D, B, dst, accum, s->stream));
    if (!grad_dev) p->pending_cnt++;
    return PS_OK;
}

extern "C" int ps_ln_pending_grad(ps_store_t *s, int layer, int bias, float *out, int cap, int *count) {
    if (!s || !out) return ps_set_err(PS_E_BAD_ARG, "null argument");
    FcParams *p;
    PSCHK(find_ln(s, layer, &p));
    if (count) *count = p->pending_cnt;
    if (p->pending_cnt == 0) return ps_set_err(PS_MISSING, "ln%d has no pending gradient", layer);
    if (cap < p->N) return ps_set_err(PS_E_BAD_ARG, "buffer too small");
    PSCHK(store_enter(s));
    HIPCHK(hipMemcpyAsync(out, p->pending + (bias ? p->N : 0), sizeof(float) * (size_t)p->N, hipMemcpyDeviceToHost, s->stream));
    HIPCHK(hipStreamSynchronize(s->stream));
    return PS_OK;
}

extern "C" int ps_ln_update(ps_store_t *s, int layer) {
    RoctxRange roctx_range("ps_ln_update");
    if (!s) return ps_set_err(PS_E_BAD_ARG, "store is NULL");
    FcParams *p;
    PSCHK(find_ln(s, layer, &p));
    if (p->pending_cnt > 0) PSCHK(store_check_ln_update(s));
    PSCHK(store_enter(s));
    bool done = false;
    PSCHK(store_apply_pending(s, *p, "ln", layer, &done));
    if (!done) return ps_set_err(PS_MISSING, "ln%d has no pending gradient", layer);
    s->global_step++;
    return PS_OK;
}

extern "C" int ps_fc_res_forward(ps_store_t *s, int layer, int type, int act, const void *x_dev, int64_t ldx, int B, const void *r_dev, int64_t ldr,
                                 void *z_dev, int64_t ldz, void *y_dev, int64_t ldy) {
    RoctxRange roctx_range("ps_fc_res_forward");
    PSCHK(check_call(s, type, B));
    if (!x_dev || !y_dev) return ps_set_err(PS_E_BAD_ARG, "null argument");
    PSCHK(check_act(act));
    FcParams *p;
    PSCHK(find_fc(s, layer, &p));
    const int es = type_size(type);
    const Mat x = {"x_dev", x_dev, ldx, p->K}, r = {"r_dev", r_dev, ldr, p->N}, z = {"z_dev", z_dev, ldz, p->N}, y = {"y_dev", y_dev, ldy, p->N};
    for (const Mat *m : {&x, &r, &z, &y}) PSCHK(check_mat(*m, B, es));
    PSCHK(check_out(y, x, B, es));
    PSCHK(check_out(y, r, B, es, true));
    PSCHK(check_out(y, z, B, es));
    PSCHK(check_out(z, x, B, es));
    PSCHK(check_out(z, r, B, es));
    PSCHK(tower_enter(s));
    FcNtArgs a;
    a.A = x_dev; a.lda = ldx; a.W = p->Wt; a.ldw = p->Kpad; a.bias = p->W + (size_t)p->K * p->ldw; a.R = r_dev; a.ldr = r_dev ? ldr : 0;
    a.Z = z_dev; a.ldz = z_dev ? ldz : 0; a.Y = y_dev; a.ldy = ldy; a.M = B; a.N = p->N; a.K = p->K; a.act = act;
    const size_t need = fc_nt_workspace(type, a);
    char *ws = nullptr;
    if (need) PSCHK(workspace(s, need, &ws));
    return launch_fc_nt(type, a, ws, s->stream);
}

extern "C" int ps_fc_res_backward(ps_store_t *s, int layer, int type, int act, const void *x_dev, int64_t ldx, const void *z_dev, int64_t ldz,
                                  const void *dy_dev, int64_t lddy, int B, const void *skip_dev, int64_t ldskip, void *dx_dev, int64_t lddx,
                                  float *grad_dev) {
    RoctxRange roctx_range("ps_fc_res_backward");
    PSCHK(check_call(s, type, B));
    if (!x_dev || !dy_dev) return ps_set_err(PS_E_BAD_ARG, "null argument");
    PSCHK(check_act(act));
    if (act != PS_ACT_NONE && !z_dev) return ps_set_err(PS_E_BAD_ARG, "act' needs the pre-activation z_dev");
    if (skip_dev && !dx_dev) return ps_set_err(PS_E_BAD_ARG, "skip_dev without dx_dev");
    FcParams *p;
    PSCHK(find_fc(s, layer, &p));
    const int es = type_size(type), K = p->K, N = p->N;
    if (act == PS_ACT_NONE) z_dev = nullptr;
    const Mat x = {"x_dev", x_dev, ldx, K}, z = {"z_dev", z_dev, ldz, N}, dy = {"dy_dev", dy_dev, lddy, N}, sk = {"skip_dev", skip_dev, ldskip, K},
              dx = {"dx_dev", dx_dev, lddx, K};
    for (const Mat *m : {&x, &z, &dy, &sk, &dx}) PSCHK(check_mat(*m, B, es));
    for (const Mat *m : {&x, &z, &dy}) PSCHK(check_out(dx, *m, B, es));
    PSCHK(check_out(dx, sk, B, es, true));
    PSCHK(check_f32("grad_dev", grad_dev, (int64_t)(K + 1) * N, {x, z, dy, sk, dx}, B, es));
    PSCHK(tower_enter(s));
    hipStream_t st = s->stream;
    float *dst;
    int accum;
    PSCHK(grad_target(s, *p, grad_dev, &dst, &accum));
    FcTnArgs t;
    t.X = x_dev; t.ldx = ldx; t.D = z_dev ? nullptr : dy_dev; t.ldd = z_dev ? round_up(N, 8) : lddy; t.M = B; t.K = K; t.N = N;
    t.dst = dst; t.accum = accum;
    fc_tn_plan(type, t);
    FcNtArgs a;
    a.A = t.D; a.lda = t.ldd; a.W = p->W; a.ldw = p->ldw; a.bias = nullptr; a.R = skip_dev; a.ldr = skip_dev ? ldskip : 0; a.Z = nullptr; a.ldz = 0;
    a.Y = dx_dev; a.ldy = lddx; a.M = B; a.N = K; a.K = N; a.act = PS_ACT_NONE;
    const bool own_dz = z_dev || t.pack_d;       // dz in the workspace: behind an activation, or dy's copy in 16-byte pieces
    if (own_dz) { t.D = a.A = nullptr; t.ldd = a.lda = round_up(N, 8); }
    // workspace: [slabs of dW | db][dz][x in pieces][what the product for dx needs], each 256-byte aligned
    const size_t slabs = t.nsplit * t.nbias == 1 ? 0 : (size_t)round_up((int64_t)sizeof(float) * (K + t.nbias) * N * t.nsplit, 256);
    const size_t dzs = own_dz ? (size_t)round_up(es * t.ldd * B, 256) : 0, xs = t.pack_x ? (size_t)round_up((int64_t)es * t.Kload * B, 256) : 0;
    const size_t need = slabs + dzs + xs + (dx_dev ? fc_nt_workspace(type, a) : 0);
    char *ws = nullptr;
    if (need) PSCHK(workspace(s, need, &ws));
    t.part = (float *)ws;
    if (own_dz) {
        t.D = a.A = ws + slabs;
        PSCHK(launch_act_grad(type, act, dy_dev, lddy, z_dev, ldz, ws + slabs, t.ldd, B, N, st));
    }
    if (dx_dev && fc_both_ok(type, a, t)) {
        PSCHK(launch_fc_both(type, a, t, st));
    } else {
        if (dx_dev) PSCHK(launch_fc_nt(type, a, ws + slabs + dzs + xs, st));
        if (t.pack_x) {
            PSCHK(launch_act_grad(type, PS_ACT_NONE, x_dev, ldx, nullptr, 0, ws + slabs + dzs, t.Kload, B, K, st));
            t.X = ws + slabs + dzs; t.ldx = t.Kload;
        }
        PSCHK(launch_fc_tn(type, t, st));
    }
    if (!grad_dev) p->pending_cnt++;
    return PS_OK;
}
