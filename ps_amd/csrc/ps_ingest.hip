// ps_ingest.hip -- the step in front of the hot path: libsvm text ->
// the arrays Model.train consumes, resident in HBM.
//
//   data/LibsvmParser.java:13-25   line.split(" "): cols[0] = label (Float.parseFloat),
//                                  cols[i] = "<Long.parseLong idx>:<Float.parseFloat value>"
//   CTR.java:47-68 parseFeature    Y = cols[0]; E[f] = idx of col 1+f (f < F, the long goes
//                                  through a float); X[j] = value of col 1+F+j (j < X);
//                                  W = MatrixUtil.hash(E, wideSize) = fmodf(E, wideSize)
//   data/DataSource.java:25-46     worker sharding: this reader takes lines offset, offset+step, ...
//   data/DataSet.java              reader threads fill a queue of parsed batches
//
// Here: the text is mapped once, the line index of this worker's lines is built once, and a
// pool of host threads parses one batch at a time straight into PINNED buffers (int64 ids,
// f32 dense / labels, int64 wide ids) while the previous batch trains; the H2D copies run on
// their own stream into one of two device slots (double buffering), and ps_ingest_next hands
// out a ps_batch_t whose pointers are device pointers.  ps_libsvm_parse is the same parser as
// a plain host function (no GPU) -- what the CPU tests pin against the restated reference.
#include <fcntl.h>
#include <pthread.h>
#include <sched.h>
#include <math.h>
#include <stdlib.h>
#include <string.h>
#include <sys/mman.h>
#include <sys/stat.h>
#include <unistd.h>

#include <algorithm>
#include <atomic>
#include <chrono>
#include <condition_variable>
#include <functional>
#include <mutex>
#include <thread>
#include <vector>

#include "ps_store.h"

namespace {

// ---- numbers ------------------------------------------------------------------
const float kPow10f[11] = {1e0f, 1e1f, 1e2f, 1e3f, 1e4f, 1e5f, 1e6f, 1e7f, 1e8f, 1e9f, 1e10f};

// Float.parseFloat: the decimal string rounded once to the nearest float.  Fast path: a
// mantissa below 2^24 and a power of ten up to 10^10 are both exact floats, so ONE IEEE
// multiply/divide is the correctly rounded result.  Everything else (long mantissas, large
// exponents, nan/inf, hex) goes to strtof, which glibc rounds correctly as well.
bool parse_float_tok(const char *p, const char *e, float *out) {
    const char *q = p;
    bool neg = false;
    if (q < e && (*q == '-' || *q == '+')) { neg = *q == '-'; ++q; }
    uint64_t m = 0;
    int exp10 = 0;
    bool any = false, slow = false;
    while (q < e && *q >= '0' && *q <= '9') {
        if (m < (1ull << 24)) m = m * 10 + (uint64_t)(*q - '0');
        else slow = true;
        any = true; ++q;
    }
    if (q < e && *q == '.') {
        ++q;
        while (q < e && *q >= '0' && *q <= '9') {
            if (m < (1ull << 24)) { m = m * 10 + (uint64_t)(*q - '0'); --exp10; }
            else slow = true;
            any = true; ++q;
        }
    }
    if (!any) slow = true;
    if (!slow && q < e && (*q == 'e' || *q == 'E')) {
        const char *r = q + 1;
        bool eneg = false;
        if (r < e && (*r == '-' || *r == '+')) { eneg = *r == '-'; ++r; }
        int ev = 0;
        bool edig = false;
        while (r < e && *r >= '0' && *r <= '9' && ev < 1000) { ev = ev * 10 + (*r - '0'); ++r; edig = true; }
        if (!edig) slow = true;
        exp10 += eneg ? -ev : ev;
        q = r;
    }
    if (!slow && q == e && m < (1ull << 24) && exp10 >= -10 && exp10 <= 10) {
        float v = (float)m;
        if (exp10 < 0) v = v / kPow10f[-exp10];
        else if (exp10 > 0) v = v * kPow10f[exp10];
        *out = neg ? -v : v;
        return true;
    }
    char buf[64];
    const size_t n = (size_t)(e - p);
    if (n == 0 || n >= sizeof buf) return false;
    memcpy(buf, p, n);
    buf[n] = 0;
    if (buf[n - 1] == 'f' || buf[n - 1] == 'F' || buf[n - 1] == 'd' || buf[n - 1] == 'D') buf[n - 1] = 0;   // Java accepts a type suffix
    char *end = nullptr;
    const float v = strtof(buf, &end);
    if (end == buf || *end != 0) return false;
    *out = v;
    return true;
}

bool parse_long_tok(const char *p, const char *e, int64_t *out) {
    bool neg = false;
    if (p < e && (*p == '-' || *p == '+')) { neg = *p == '-'; ++p; }
    if (p == e) return false;
    uint64_t v = 0;
    for (; p < e; ++p) {
        if (*p < '0' || *p > '9') return false;
        if (v > (uint64_t)INT64_MAX / 10) return false;
        v = v * 10 + (uint64_t)(*p - '0');
        if (v > (uint64_t)INT64_MAX) return false;
    }
    *out = neg ? -(int64_t)v : (int64_t)v;
    return true;
}

// MatrixUtil.hash (util/MatrixUtil.java:27-33): fmodf(fe, (float)wideSize) on an id that went through a float.  fe is integral (a long cast
// to float) and so is (float)wideSize: the float remainder of two integers IS the integer remainder, sign of the dividend -- C's % on the
// two values as int64 -- and needs no libm call (fmodf was most of a line's parse time: 26 calls of ~30 ns).  Beyond 2^62 the cast would
// overflow: fmodf itself.
static inline int64_t wide_of(float fe, int64_t wide_size) {
    const float ws = (float)wide_size;
    if (fe > -4.0e18f && fe < 4.0e18f && ws < 4.0e18f) return (int64_t)fe % (int64_t)ws;
    return (int64_t)fmodf(fe, ws);
}
struct LineOut { int64_t *ids; float *dense; float *label; int64_t *wide; };

// one line -> one sample.  0 ok, else the 1-based column that failed (1 = label), -1 = too few columns
int parse_line_general(const char *p, const char *e, const ps_ingest_config_t &c, const LineOut &o) {
    while (e > p && (e[-1] == '\r' || e[-1] == ' ' || e[-1] == '\t')) --e;
    int col = 0;
    const int need = 1 + c.F + c.X;
    while (p < e && col < need) {
        while (p < e && *p == ' ') ++p;
        const char *t = p;
        while (p < e && *p != ' ') ++p;
        if (t == p) break;
        if (col == 0) {
            if (!parse_float_tok(t, p, o.label)) return 1;
        } else {
            const char *colon = (const char *)memchr(t, ':', (size_t)(p - t));
            if (!colon) return col + 1;
            if (col <= c.F) {
                int64_t idx;
                if (!parse_long_tok(t, colon, &idx)) return col + 1;
                float junk;
                if (!parse_float_tok(colon + 1, p, &junk)) return col + 1;     // LibsvmParser parses (and boxes) it anyway
                int64_t id = idx, w = 0;
                if (c.ids_via_float) {
                    const float fe = (float)idx;                               // E[j-1][i] = cols.get(j).getIdx()  (long -> float)
                    id = (int64_t)fe;
                    if (c.wide_size > 0) w = wide_of(fe, c.wide_size);   // MatrixUtil.hash (util/MatrixUtil.java:27-33)
                } else if (c.wide_size > 0) {
                    w = idx % c.wide_size;
                }
                o.ids[col - 1] = id;
                if (o.wide) o.wide[col - 1] = w;
            } else {
                int64_t idx;
                if (!parse_long_tok(t, colon, &idx)) return col + 1;
                if (!parse_float_tok(colon + 1, p, &o.dense[col - 1 - c.F])) return col + 1;
            }
        }
        ++col;
    }
    return col == need ? 0 : -1;
}


// ---- the common line, in one pass ------------------------------------------------------------------------------------
// Round 6: the pipeline needs ~22 parser threads at 0.7 us per line to feed a 135 us step, and that many busy host threads slow the
// step's launches (profiles/r06_ingest_probes.txt).  A CTR line is 40 tokens of three shapes -- `label`, `idx:1`, `idx:-0.123456` --
// so one forward scan handles it: digits into an integer, ':', an optional sign, digits, an optional fraction, a space.  The values
// computed are parse_line_general's, operation for operation (same mantissa < 2^24 rule, same one IEEE division by a power of ten,
// the same long -> float -> id path).  Anything else on the line -- an exponent, a ninth significant digit, a suffix, a tab, a
// missing column, an index beyond 18 digits -- and the line is handed to parse_line_general untouched: errors keep their column numbers.
// Returns 0 (parsed) or -2 (not this shape).
#define PS_FAST_FLOAT(V)                                                                                   \
    do {                                                                                                   \
        bool neg_ = false;                                                                                 \
        if (p < e && (*p == '-' || *p == '+')) { neg_ = *p == '-'; ++p; }                                  \
        uint32_t m_ = 0; int nd_ = 0, fr_ = 0;                                                             \
        while (p < e && (unsigned)(*p - '0') <= 9u) { m_ = m_ * 10u + (uint32_t)(*p - '0'); ++nd_; ++p; }  \
        if (p < e && *p == '.') {                                                                          \
            ++p;                                                                                           \
            while (p < e && (unsigned)(*p - '0') <= 9u) { m_ = m_ * 10u + (uint32_t)(*p - '0'); ++nd_; ++fr_; ++p; } \
        }                                                                                                  \
        /* 8 digits: m_ < 10^8 fits; the general rule stops accumulating once m >= 2^24 BEFORE a digit: with <= 7 digits m stays below */ \
        if (nd_ == 0 || nd_ > 7 || (p < e && *p != ' ')) return -2;                                        \
        float v_ = (float)m_;                                                                              \
        if (fr_ > 0) v_ = v_ / kPow10f[fr_];                                                               \
        (V) = neg_ ? -v_ : v_;                                                                             \
    } while (0)
int parse_line_fast(const char *p, const char *e, const ps_ingest_config_t &c, const LineOut &o) {
    float label;
    PS_FAST_FLOAT(label);
    const int ncol = c.F + c.X;
    for (int col = 0; col < ncol; ++col) {
        if (p >= e || *p != ' ') return -2;
        while (p < e && *p == ' ') ++p;
        bool ineg = false;
        if (p < e && (*p == '-' || *p == '+')) { ineg = *p == '-'; ++p; }
        uint64_t v = 0; int nd = 0;
        while (p < e && (unsigned)(*p - '0') <= 9u) { v = v * 10u + (uint64_t)(*p - '0'); ++nd; ++p; }
        if (nd == 0 || nd > 18 || p >= e || *p != ':') return -2;
        ++p;
        float val;
        PS_FAST_FLOAT(val);
        if (col < c.F) {
            const int64_t idx = ineg ? -(int64_t)v : (int64_t)v;
            int64_t id = idx, w = 0;
            if (c.ids_via_float) {
                const float fe = (float)idx;
                id = (int64_t)fe;
                if (c.wide_size > 0) w = wide_of(fe, c.wide_size);
            } else if (c.wide_size > 0) {
                w = idx % c.wide_size;
            }
            o.ids[col] = id;
            if (o.wide) o.wide[col] = w;
        } else {
            o.dense[col - c.F] = val;
        }
    }
    // (columns beyond 1 + F + X are ignored by the general parser too; trailing blanks were trimmed by the caller)
    *o.label = label;
    return 0;
}
#undef PS_FAST_FLOAT

int g_ingest_fast = getenv("PS_INGEST_FAST") ? atoi(getenv("PS_INGEST_FAST")) : 1;     // 0: every line through parse_line_general (rounds 2-5)
int parse_line(const char *p, const char *e, const ps_ingest_config_t &c, const LineOut &o) {
    if (g_ingest_fast) {
        const char *e2 = e;
        while (e2 > p && (e2[-1] == '\r' || e2[-1] == ' ' || e2[-1] == '\t')) --e2;
        if (parse_line_fast(p, e2, c, o) == 0) return 0;
    }
    return parse_line_general(p, e, c, o);
}

// ---- a small pool: run fn(i) for i in [0,n) on the pool's threads + the caller ----
class Pool {
  public:
    explicit Pool(int nthreads) {
        for (int i = 1; i < nthreads; ++i) th_.emplace_back([this] { loop(); });
    }
    ~Pool() {
        { std::lock_guard<std::mutex> l(mu_); stop_ = true; }
        cv_.notify_all();
        for (auto &t : th_) t.join();
    }
    void run(int64_t n, int64_t grain, const std::function<void(int64_t, int64_t)> &fn) {
        if (n <= 0) return;
        {
            std::lock_guard<std::mutex> l(mu_);
            fn_ = &fn; n_ = n; grain_ = grain < 1 ? 1 : grain; next_.store(0); pending_ = (int)th_.size(); ++gen_;
        }
        cv_.notify_all();
        work();
        std::unique_lock<std::mutex> l(mu_);
        done_.wait(l, [this] { return pending_ == 0; });
        fn_ = nullptr;
    }

  private:
    void work() {
        for (;;) {
            const int64_t b = next_.fetch_add(grain_);
            if (b >= n_) return;
            (*fn_)(b, b + grain_ < n_ ? b + grain_ : n_);
        }
    }
    void loop() {
        uint64_t seen = 0;
        for (;;) {
            {
                std::unique_lock<std::mutex> l(mu_);
                cv_.wait(l, [&] { return stop_ || gen_ != seen; });
                if (stop_) return;
                seen = gen_;
            }
            work();
            {
                std::lock_guard<std::mutex> l(mu_);
                --pending_;
            }
            done_.notify_one();
        }
    }
    std::vector<std::thread> th_;
    std::mutex mu_;
    std::condition_variable cv_, done_;
    const std::function<void(int64_t, int64_t)> *fn_ = nullptr;
    int64_t n_ = 0, grain_ = 1;
    std::atomic<int64_t> next_{0};
    int pending_ = 0;
    uint64_t gen_ = 0;
    bool stop_ = false;
};

// start offsets of this worker's lines.  DataSource.readLine (data/DataSource.java:25-46) counts RAW lines, blank ones
// included: raw line g is this reader's iff g >= offset and (g - offset) % step == 0; a selected line that is blank
// then yields an empty feature list (LibsvmParser.parse, StringUtils.isBlank) and is dropped.
void index_lines(const char *d, size_t len, int offset, int step, std::vector<size_t> *starts, std::vector<size_t> *ends) {
    size_t pos = 0;
    int64_t g = 0;
    while (pos < len) {
        const char *nl = (const char *)memchr(d + pos, '\n', len - pos);
        const size_t end = nl ? (size_t)(nl - d) : len;
        if (g >= offset && (g - offset) % step == 0) {
            bool blank = true;
            for (size_t i = pos; i < end; ++i)
                if (d[i] != ' ' && d[i] != '\t' && d[i] != '\r') { blank = false; break; }
            if (!blank) { starts->push_back(pos); ends->push_back(end); }
        }
        ++g;
        pos = end + 1;
    }
}

// The same index by chunks of the text (round 6: the serial walk was what bounded the host parser at 64 threads -- 131 072 lines,
// 52 MB: 6 ms of memchr in front of 4 ms of parsing).  A chunk owns the lines that START inside it; the raw number of a chunk's
// first line is the number of newlines in front of the chunk -- a prefix over per-chunk counts -- so offset / step select the same
// raw lines as the serial walk, and the chunks' lists concatenate in order.
void index_lines_parallel(const char *d, size_t len, int offset, int step, std::vector<size_t> *starts, std::vector<size_t> *ends, Pool *pool) {
    const size_t CH = (size_t)4 << 20;
    const int64_t nch = (int64_t)((len + CH - 1) / CH);
    if (!pool || nch < 4) { index_lines(d, len, offset, step, starts, ends); return; }
    std::vector<int64_t> nl((size_t)nch + 1, 0);
    pool->run(nch, 1, [&](int64_t b, int64_t e) {
        for (int64_t c = b; c < e; ++c) {
            const size_t lo = (size_t)c * CH, hi = std::min(len, lo + CH);
            int64_t k = 0;
            for (const char *q = d + lo; (q = (const char *)memchr(q, '\n', (size_t)(d + hi - q))) != nullptr; ++q) ++k;
            nl[(size_t)c + 1] = k;
        }
    });
    for (int64_t c = 0; c < nch; ++c) nl[(size_t)c + 1] += nl[(size_t)c];
    std::vector<std::vector<size_t>> st((size_t)nch), en((size_t)nch);
    pool->run(nch, 1, [&](int64_t b, int64_t e) {
        for (int64_t c = b; c < e; ++c) {
            const size_t lo = (size_t)c * CH, hi = std::min(len, lo + CH);
            size_t pos = lo;
            int64_t g = nl[(size_t)c];                       // raw number of the line that contains byte lo
            if (lo > 0 && d[lo - 1] != '\n') {               // ... which started in an earlier chunk: skip to the first start in here
                const char *q = (const char *)memchr(d + lo, '\n', hi - lo);
                if (!q) continue;                            // (no line starts in this chunk)
                pos = (size_t)(q - d) + 1; ++g;
            }
            while (pos < hi) {                               // lines that START in [lo, hi); they may end beyond hi
                const char *q = (const char *)memchr(d + pos, '\n', len - pos);
                const size_t end = q ? (size_t)(q - d) : len;
                if (g >= offset && (g - offset) % step == 0) {
                    bool blank = true;
                    for (size_t i = pos; i < end; ++i)
                        if (d[i] != ' ' && d[i] != '\t' && d[i] != '\r') { blank = false; break; }
                    if (!blank) { st[(size_t)c].push_back(pos); en[(size_t)c].push_back(end); }
                }
                ++g;
                pos = end + 1;
            }
        }
    });
    size_t tot = 0;
    for (auto &v : st) tot += v.size();
    starts->reserve(tot); ends->reserve(tot);
    for (int64_t c = 0; c < nch; ++c) {
        starts->insert(starts->end(), st[(size_t)c].begin(), st[(size_t)c].end());
        ends->insert(ends->end(), en[(size_t)c].begin(), en[(size_t)c].end());
    }
}

int check_cfg(const ps_ingest_config_t *c) {
    if (!c || c->F < 0 || c->X < 0 || c->F + c->X <= 0 || c->batch <= 0 || c->offset < 0 || c->step < 1 || c->wide_size < 0)
        return ps_set_err(PS_E_BAD_ARG, "bad ingest config");
    return PS_OK;
}

int parse_range(const char *d, const std::vector<size_t> &st, const std::vector<size_t> &en, int64_t first, int64_t n,
                const ps_ingest_config_t &c, int64_t *ids, float *dense, float *labels, int64_t *wide, Pool *pool) {
    std::atomic<int64_t> bad_line{-1};
    std::atomic<int> bad_col{0};
    auto body = [&](int64_t b, int64_t e) {
        for (int64_t i = b; i < e; ++i) {
            LineOut o{ids + i * c.F, dense + i * c.X, labels + i, (wide && c.wide_size > 0) ? wide + i * c.F : nullptr};
            const int rc = parse_line(d + st[first + i], d + en[first + i], c, o);
            if (rc != 0) {
                int64_t exp = -1;
                if (bad_line.compare_exchange_strong(exp, first + i)) bad_col.store(rc);
            }
        }
    };
    if (pool) pool->run(n, 64, body);
    else body(0, n);
    if (bad_line.load() >= 0) {
        if (bad_col.load() < 0)
            return ps_set_err(PS_E_BAD_ARG, "libsvm line %lld of this reader: fewer than %d columns", (long long)bad_line.load(), 1 + c.F + c.X);
        return ps_set_err(PS_E_BAD_ARG, "libsvm line %lld of this reader: column %d does not parse", (long long)bad_line.load(), bad_col.load());
    }
    return PS_OK;
}

}  // namespace

// ---------------------------------------------------------------------------
// host-only parser
// ---------------------------------------------------------------------------
extern "C" int ps_libsvm_count(const char *text, size_t len, int offset, int step, int64_t *n_lines) {
    if (!text || !n_lines || offset < 0 || step < 1) return ps_set_err(PS_E_BAD_ARG, "bad argument");
    std::vector<size_t> st, en;
    index_lines(text, len, offset, step, &st, &en);
    *n_lines = (int64_t)st.size();
    return PS_OK;
}

extern "C" int ps_libsvm_parse(const char *text, size_t len, const ps_ingest_config_t *cfg, int64_t first_line, int64_t max_lines,
                               int64_t *ids, float *dense, float *labels, int64_t *wide_ids, int64_t *n_parsed) {
    PSCHK(check_cfg(cfg));
    if (!text || !n_parsed || first_line < 0 || max_lines < 0 || (cfg->F > 0 && !ids) || (cfg->X > 0 && !dense) || !labels)
        return ps_set_err(PS_E_BAD_ARG, "null argument");
    std::vector<size_t> st, en;
    const int nt = cfg->threads > 1 ? cfg->threads : 1;
    Pool *pool = nt > 1 ? new Pool(nt) : nullptr;
    index_lines_parallel(text, len, cfg->offset, cfg->step, &st, &en, pool);
    int64_t n = (int64_t)st.size() - first_line;
    if (n < 0) n = 0;
    if (n > max_lines) n = max_lines;
    *n_parsed = n;
    int rc = PS_OK;
    if (n > 0) rc = parse_range(text, st, en, first_line, n, *cfg, ids, dense, labels, wide_ids, pool);
    delete pool;
    return rc;
}

// ---------------------------------------------------------------------------
// the pipeline: a RING of batches between the text and the training stream
// ---------------------------------------------------------------------------
// Round 6.  Rounds 2-5 filled ONE batch at a time: a pool parsed its 4096 lines 64 at a chunk, then four H2D copies, then a
// stream wait -- wake-up of the pool, parse, copies and wait in series per batch: 12.7 M lines/s on 64 threads while the
// resident step consumes 30 M examples/s.  Now the unit of parallel work is a BATCH:
//   * `threads` parser threads each take the next unparsed batch and parse all of it into that batch's slot of a ring of
//     pinned blocks [ids | wide ids | dense | labels] -- no HIP call, no shared state but two counters;
//   * a COPIER thread takes the parsed batches in order: waits until the kernels that read the slot's previous batch are done (an
//     event the training thread recorded), ONE hipMemcpyAsync of the whole block, an event behind it -- and goes on to the next
//     batch; a COMPLETER thread waits for those events in order and marks the batches ready.  (One thread that copied AND waited
//     was the pipeline's limit: 167 us per batch, 24 M lines/s, with the parsers at 138 M when it was.)
//   * ps_ingest_next hands out batch b when it is ready and gives batch b - 2's slot back to the parsers (its consumers were
//     enqueued before this call: "valid until the call after the next one").
// The ring holds RING batches (2 x threads, 4..64): that many batches may be in flight between the parsers and the step.
int g_ingest_compact = getenv("PS_INGEST_COMPACT") ? atoi(getenv("PS_INGEST_COMPACT")) : 1;      // 0: every batch crosses the link as int64 arrays (rounds 2-5)
namespace {
// ids[i] = ids32[i] (sign-extended), wide[i] = what the parser computes from the same id (parse_line: MatrixUtil.hash through a float when
// ids_via_float -- (float)id is the parser's own float, the id came out of it -- else id % wide_size; fmodf is exact on both sides)
// (blockIdx.y: the slot inside a group of neighbouring blocks, `pitch` bytes apart)
__global__ __launch_bounds__(256) void k_ingest_expand(const int32_t *__restrict__ ids32, int64_t n, int64_t wide_size, int via_float, int64_t *__restrict__ ids, int64_t *__restrict__ wide, size_t pitch) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    ids32 = reinterpret_cast<const int32_t *>(reinterpret_cast<const char *>(ids32) + blockIdx.y * pitch);
    ids = reinterpret_cast<int64_t *>(reinterpret_cast<char *>(ids) + blockIdx.y * pitch);
    if (wide_size > 0) wide = reinterpret_cast<int64_t *>(reinterpret_cast<char *>(wide) + blockIdx.y * pitch);
    const int64_t id = (int64_t)ids32[i];
    ids[i] = id;
    if (wide_size > 0) wide[i] = via_float ? (int64_t)fmodf((float)id, (float)wide_size) : id % wide_size;
}
}  // namespace

struct ps_ingest {
    ps_store *s = nullptr;
    ps_ingest_config_t cfg{};
    const char *data = nullptr;
    size_t len = 0;
    void *map = nullptr; size_t map_len = 0;          // mmap of a file
    std::vector<char> copy;                           // or a private copy of the caller's memory
    std::vector<size_t> st, en;
    hipStream_t copy_stream = nullptr;
    size_t off_ids = 0, off_wide = 0, off_dense = 0, off_labels = 0, off_ids32 = 0, block = 0;     // layout of a slot's block: [ids | wide ids | dense | labels | ids as int32]
    struct Slot {
        char *host = nullptr, *dev = nullptr;         // pinned | HBM
        hipEvent_t consumed = nullptr;                // the kernels that read the slot were enqueued before this (store stream)
        hipEvent_t consumed_wait = nullptr;           // ... as recorded for the group of slots released together (the last one's `consumed`)
        hipEvent_t copied = nullptr;                  // the slot's H2D copy has landed (copy stream)
        hipEvent_t wait_ev = nullptr;                 // ... as recorded for the GROUP this batch crossed the link in (its last slot's `copied`)
        bool consumed_recorded = false;
        int B = 0;
        int rc = PS_OK;
        bool skipped = false;                         // (measurement knobs: this batch's copy was left out)
        bool compact = false;                         // every id of the batch fits an int32: only [dense | labels | ids32] crosses the link
        char err[256] = "";
    };
    std::vector<Slot> slot;
    char *host_all = nullptr, *dev_all = nullptr;     // the ring's blocks, slot after slot
    int ring = 0, release_every = 1;                 // slots go back to the parsers this many at a time (one event on the training stream per group)
    int64_t nbatches = 0;
    // progress, all under mu: batch b may be PARSED into its slot once free_upto > b; it is parsed when parsed[b % ring] == b,
    // in HBM when ready_upto > b
    std::mutex mu;
    std::condition_variable cv_free, cv_parsed, cv_issued, cv_ready;
    int64_t next_parse = 0, free_upto = 0, issued_upto = 0, ready_upto = 0, cur = 0;
    std::vector<int64_t> parsed;
    std::vector<std::thread> parsers;
    std::thread copier, completer;
    bool running = false, stop = false;
    bool inline_copy = true;          // the TRAINING thread issues the copies itself (ps_ingest_next): no second thread talks to HIP while the step is enqueued
    double parse_s = 0; int64_t parsed_lines = 0, parsed_bytes = 0;
};

namespace {

// PS_INGEST_PIN=1: the parser threads keep to the upper half of the CPUs this process may use (measured: 96 busy host threads slow
// the fused step's launches on the GPU from 0.137 to 0.20-0.24 ms per step; kept away from the launching thread's half: 0.147 with 48 --
// tools/r06_host_load_probe2.py, profiles/r06_host_load_probe.txt)
void pin_parser_thread() {
    static const bool pin = getenv("PS_INGEST_PIN") != nullptr;
    if (!pin) return;
    cpu_set_t have, want;
    CPU_ZERO(&have); CPU_ZERO(&want);
    if (sched_getaffinity(0, sizeof have, &have) != 0) return;
    const int n = CPU_COUNT(&have);
    int k = 0;
    for (int c = 0; c < CPU_SETSIZE; ++c)
        if (CPU_ISSET(c, &have)) { if (k >= n / 2) CPU_SET(c, &want); ++k; }
    if (CPU_COUNT(&want) > 0) (void)pthread_setaffinity_np(pthread_self(), sizeof want, &want);
}

void parser_loop(ps_ingest *g) {
    const ps_ingest_config_t &c = g->cfg;
    pin_parser_thread();
    for (;;) {
        int64_t b;
        bool last;
        {
            // a thread takes a batch only once that batch's slot is free: a freed slot then wakes ONE sleeper (taking first and waiting
            // afterwards had all 96 threads wake at every release -- the training thread shares the mutex and the cores with them)
            std::unique_lock<std::mutex> l(g->mu);
            g->cv_free.wait(l, [&] { return g->stop || g->next_parse >= g->nbatches || g->free_upto > g->next_parse; });
            if (g->stop || g->next_parse >= g->nbatches) return;
            b = g->next_parse++;
            last = g->next_parse >= g->nbatches;
        }
        if (last) g->cv_free.notify_all();             // (nothing left to take: the sleepers leave)
        ps_ingest::Slot &S = g->slot[(size_t)(b % g->ring)];
        const int64_t first = b * c.batch;
        int64_t n = (int64_t)g->st.size() - first;
        if (n > c.batch) n = c.batch;
        const auto t0 = std::chrono::steady_clock::now();
        S.B = (int)n;
        S.rc = parse_range(g->data, g->st, g->en, first, n, c, (int64_t *)(S.host + g->off_ids), (float *)(S.host + g->off_dense),
                           (float *)(S.host + g->off_labels), c.wide_size > 0 ? (int64_t *)(S.host + g->off_wide) : nullptr, nullptr);
        if (S.rc != PS_OK) snprintf(S.err, sizeof S.err, "%s", ps_last_error());
        // Two thirds of a batch's bytes are its ids as int64, twice (ids and wide ids = a function of the ids): when every id fits
        // an int32 only [dense | labels | ids32] is copied (0.65 instead of 1.93 MB at configs[1]) and a kernel on the copy stream
        // writes the two int64 arrays the step reads (k_ingest_expand).  H2D moved 22 GB/s alone and 10 GB/s beside a training step:
        // it, not the parsers, bounded the pipeline (profiles/r06_ingest_*).
        S.compact = false;
        if (S.rc == PS_OK && c.F > 0 && g_ingest_compact) {
            const int64_t *src = (const int64_t *)(S.host + g->off_ids);
            int32_t *dst = (int32_t *)(S.host + g->off_ids32);
            const int64_t cnt = n * c.F;
            bool fits = true;
            for (int64_t i = 0; i < cnt; ++i) { const int64_t v = src[i]; dst[i] = (int32_t)v; fits = fits && v == (int64_t)(int32_t)v; }
            S.compact = fits;
        }
        const double dt = std::chrono::duration<double>(std::chrono::steady_clock::now() - t0).count();
        {
            std::lock_guard<std::mutex> l(g->mu);
            g->parsed[(size_t)(b % g->ring)] = b;
            g->parse_s += dt; g->parsed_lines += n; g->parsed_bytes += (int64_t)(g->en[(size_t)(first + n - 1)] - g->st[(size_t)first]);
        }
        g->cv_parsed.notify_all();
    }
}

// the H2D copies of one parsed batch (+ the kernel that rebuilds the int64 arrays of a compact one), enqueued on the copy stream
hipError_t issue_copy(ps_ingest *g, ps_ingest::Slot &S, hipError_t e) {
    // (a short last batch: the arrays keep their full-batch offsets inside the block, the tail of each is not copied)
    const ps_ingest_config_t &c = g->cfg;
    if (S.compact) {
        const size_t n = (size_t)S.B;
        if (S.B == c.batch) {           // [dense | labels | ids32] lie back to back: one copy
            if (e == hipSuccess) e = hipMemcpyAsync(S.dev + g->off_dense, S.host + g->off_dense, g->off_ids32 + sizeof(int32_t) * n * c.F - g->off_dense, hipMemcpyHostToDevice, g->copy_stream);
        } else {
            if (e == hipSuccess && c.X > 0) e = hipMemcpyAsync(S.dev + g->off_dense, S.host + g->off_dense, sizeof(float) * n * c.X, hipMemcpyHostToDevice, g->copy_stream);
            if (e == hipSuccess) e = hipMemcpyAsync(S.dev + g->off_labels, S.host + g->off_labels, sizeof(float) * n, hipMemcpyHostToDevice, g->copy_stream);
            if (e == hipSuccess) e = hipMemcpyAsync(S.dev + g->off_ids32, S.host + g->off_ids32, sizeof(int32_t) * n * c.F, hipMemcpyHostToDevice, g->copy_stream);
        }
        if (e == hipSuccess) {
            const int64_t cnt = (int64_t)n * c.F;
            hipLaunchKernelGGL(k_ingest_expand, dim3((unsigned int)((cnt + 255) / 256)), dim3(256), 0, g->copy_stream, (const int32_t *)(S.dev + g->off_ids32), cnt,
                               c.wide_size, c.ids_via_float, (int64_t *)(S.dev + g->off_ids), (int64_t *)(S.dev + g->off_wide), (size_t)0);
            e = hipGetLastError();
        }
    } else if (S.B == c.batch) {
        if (e == hipSuccess) e = hipMemcpyAsync(S.dev, S.host, g->off_ids32, hipMemcpyHostToDevice, g->copy_stream);
    } else {
        const size_t n = (size_t)S.B;
        if (e == hipSuccess && c.F > 0) e = hipMemcpyAsync(S.dev + g->off_ids, S.host + g->off_ids, sizeof(int64_t) * n * c.F, hipMemcpyHostToDevice, g->copy_stream);
        if (e == hipSuccess && c.F > 0 && c.wide_size > 0) e = hipMemcpyAsync(S.dev + g->off_wide, S.host + g->off_wide, sizeof(int64_t) * n * c.F, hipMemcpyHostToDevice, g->copy_stream);
        if (e == hipSuccess && c.X > 0) e = hipMemcpyAsync(S.dev + g->off_dense, S.host + g->off_dense, sizeof(float) * n * c.X, hipMemcpyHostToDevice, g->copy_stream);
        if (e == hipSuccess) e = hipMemcpyAsync(S.dev + g->off_labels, S.host + g->off_labels, sizeof(float) * n, hipMemcpyHostToDevice, g->copy_stream);
    }
    return e;
}

static double ing_now() { return std::chrono::duration<double, std::micro>(std::chrono::steady_clock::now().time_since_epoch()).count(); }
void copier_loop(ps_ingest *g) {
    (void)hipSetDevice(g->s->device);
    static const bool timing = getenv("PS_INGEST_TIMING") != nullptr;
    double t_wait = 0, t_sync = 0, t_issue = 0;
    const int group_max = getenv("PS_INGEST_GROUP") ? atoi(getenv("PS_INGEST_GROUP")) : std::max(1, g->ring / 2);      // batches per H2D call at most (1: one call per batch)
    const int64_t low_water = getenv("PS_INGEST_LOW") ? atoi(getenv("PS_INGEST_LOW")) : std::max(1, g->ring / 4);        // ... gathered while the consumer has this many batches ahead of it
    for (int64_t b = 0; b < g->nbatches; ++b) {
        ps_ingest::Slot &S = g->slot[(size_t)(b % g->ring)];
        const double c0 = timing ? ing_now() : 0;
        {
            // wait for batch b -- and, while the consumer still has `low_water` batches in HBM ahead of it, for a whole group behind b: in the
            // steady state batches are parsed one by one at the consumer's pace, and a copier that sends each as it appears sends groups of one
            std::unique_lock<std::mutex> l(g->mu);
            g->cv_parsed.wait(l, [&] {
                if (g->stop) return true;
                if (g->parsed[(size_t)(b % g->ring)] != b) return false;
                if (group_max <= 1 || b - g->cur < low_water) return true;
                int have = 1;
                while (have < group_max && b + have < g->nbatches && (b + have) % g->ring != 0 && g->parsed[(size_t)((b + have) % g->ring)] == b + have) ++have;
                return have >= group_max || b + have >= g->nbatches || (b + have) % g->ring == 0;
            });
            if (g->stop) return;
        }
        const double c1 = timing ? ing_now() : 0;
        t_wait += c1 - c0;
        static const bool nocopy_all = getenv("PS_INGEST_NOCOPY") != nullptr;        // (measurement only: the batches in HBM are not refreshed)
        static const int copy_every = getenv("PS_INGEST_COPY_EVERY") ? atoi(getenv("PS_INGEST_COPY_EVERY")) : 1;      // (measurement only)
        const bool nocopy = nocopy_all || (copy_every > 1 && b % copy_every != 0);
        S.skipped = nocopy;
        S.wait_ev = S.copied;
        // A GROUP: the batches behind b that are parsed already, full-size, of b's kind (compact or not) and in neighbouring blocks cross the
        // link in ONE call and are rebuilt by ONE kernel launch.  What a copy costs the training step is its HIP calls, not its bytes: one copy per
        // batch 0.1953 ms per step, every 4th batch copied 0.1518, every 16th 0.1428, none 0.1442 (16 parser threads; profiles/r06_ingest_probes.txt).
        int group = 1;
        if (S.rc == PS_OK && S.B == g->cfg.batch && !nocopy && group_max > 1) {
            std::lock_guard<std::mutex> l(g->mu);
            while (group < group_max && b + group < g->nbatches && (b + group) % g->ring != 0) {
                const ps_ingest::Slot &T = g->slot[(size_t)((b + group) % g->ring)];
                if (g->parsed[(size_t)((b + group) % g->ring)] != b + group || T.rc != PS_OK || T.B != g->cfg.batch || T.compact != S.compact) break;
                ++group;
            }
        }
        if (group > 1) {
            const ps_ingest_config_t &c = g->cfg;
            hipError_t e = hipSuccess;
            for (int k = 0; k < group && e == hipSuccess; ++k) {
                ps_ingest::Slot &T = g->slot[(size_t)((b + k) % g->ring)];
                if (T.consumed_recorded) e = hipEventSynchronize(T.consumed_wait);
            }
            if (S.compact) {
                const size_t w = g->block - g->off_dense;          // [dense | labels | ids32] to the end of the block
                if (e == hipSuccess) e = hipMemcpy2DAsync(S.dev + g->off_dense, g->block, S.host + g->off_dense, g->block, w, (size_t)group, hipMemcpyHostToDevice, g->copy_stream);
                if (e == hipSuccess) {
                    const int64_t cnt = (int64_t)c.batch * c.F;
                    hipLaunchKernelGGL(k_ingest_expand, dim3((unsigned int)((cnt + 255) / 256), (unsigned int)group), dim3(256), 0, g->copy_stream, (const int32_t *)(S.dev + g->off_ids32), cnt,
                                       c.wide_size, c.ids_via_float, (int64_t *)(S.dev + g->off_ids), (int64_t *)(S.dev + g->off_wide), g->block);
                    e = hipGetLastError();
                }
            } else if (e == hipSuccess) {
                e = hipMemcpyAsync(S.dev, S.host, g->block * (size_t)group, hipMemcpyHostToDevice, g->copy_stream);
            }
            ps_ingest::Slot &Last = g->slot[(size_t)((b + group - 1) % g->ring)];
            if (e == hipSuccess) e = hipEventRecord(Last.copied, g->copy_stream);
            for (int k = 0; k < group; ++k) {
                ps_ingest::Slot &T = g->slot[(size_t)((b + k) % g->ring)];
                T.skipped = false; T.wait_ev = Last.copied;
                if (e != hipSuccess) { T.rc = PS_E_HIP; snprintf(T.err, sizeof T.err, "ingest H2D: %s", hipGetErrorString(e)); }
            }
            if (timing) t_issue += ing_now() - c1;
            {
                std::lock_guard<std::mutex> l(g->mu);
                g->issued_upto = b + group;
            }
            g->cv_issued.notify_all();
            b += group - 1;
            continue;
        }
        if (S.rc == PS_OK && S.B > 0 && !nocopy) {
            // host-synchronised HERE, in the background: the kernels that read this slot's previous batch are done, the block is
            // copied, the copy has landed -- the training thread needs no cross-stream event (cross-thread event WAITS proved
            // unreliable in round 2: occasional stale batches)
            hipError_t e = hipSuccess;
            if (S.consumed_recorded) e = hipEventSynchronize(S.consumed_wait);
            if (timing) t_sync += ing_now() - c1;
            e = issue_copy(g, S, e);
            if (e == hipSuccess) e = hipEventRecord(S.copied, g->copy_stream);
            if (e != hipSuccess) { S.rc = PS_E_HIP; snprintf(S.err, sizeof S.err, "ingest H2D: %s", hipGetErrorString(e)); }
        }
        if (timing) t_issue += ing_now() - c1;
        {
            std::lock_guard<std::mutex> l(g->mu);
            g->issued_upto = b + 1;
        }
        g->cv_issued.notify_all();
    }
    if (timing && g->nbatches > 0) fprintf(stderr, "[ingest copier] per batch: %.1f us waiting for the parsers, %.1f us in HIP calls (of which %.1f waiting for the slot's consumers)\n",
                                          t_wait / g->nbatches, t_issue / g->nbatches, t_sync / g->nbatches);
}

void completer_loop(ps_ingest *g) {
    (void)hipSetDevice(g->s->device);
    for (int64_t b = 0; b < g->nbatches; ++b) {
        ps_ingest::Slot &S = g->slot[(size_t)(b % g->ring)];
        {
            std::unique_lock<std::mutex> l(g->mu);
            g->cv_issued.wait(l, [&] { return g->stop || g->issued_upto > b; });
            if (g->stop) return;
        }
        if (S.rc == PS_OK && S.B > 0 && !S.skipped) {
            // (polled: a blocking hipEventSynchronize here and the copier's calls share the runtime's locks with the training
            //  thread's launches -- PS_INGEST_SYNC=1 is the blocking form, for the A/B)
            static const bool blocking = getenv("PS_INGEST_SYNC") != nullptr;
            hipError_t e = hipSuccess;
            if (blocking) e = hipEventSynchronize(S.wait_ev);
            else {
                while ((e = hipEventQuery(S.wait_ev)) == hipErrorNotReady) std::this_thread::sleep_for(std::chrono::microseconds(15));
            }
            if (e != hipSuccess) { S.rc = PS_E_HIP; snprintf(S.err, sizeof S.err, "ingest H2D: %s", hipGetErrorString(e)); }
        }
        {
            std::lock_guard<std::mutex> l(g->mu);
            g->ready_upto = b + 1;
        }
        g->cv_ready.notify_all();
    }
}

void ingest_stop(ps_ingest *g) {                      // join every thread of the running epoch (open / reset / destroy)
    {
        std::lock_guard<std::mutex> l(g->mu);
        g->stop = true;
    }
    g->cv_free.notify_all(); g->cv_parsed.notify_all(); g->cv_issued.notify_all(); g->cv_ready.notify_all();
    for (auto &t : g->parsers) if (t.joinable()) t.join();
    g->parsers.clear();
    if (g->copier.joinable()) g->copier.join();
    if (g->completer.joinable()) g->completer.join();
    if (g->copy_stream) (void)hipStreamSynchronize(g->copy_stream);
    g->running = false; g->stop = false;
}

void ingest_rewind(ps_ingest *g) {
    ingest_stop(g);
    g->next_parse = 0; g->free_upto = g->ring; g->issued_upto = 0; g->ready_upto = 0; g->cur = 0;
    for (auto &v : g->parsed) v = -1;
    g->nbatches = ((int64_t)g->st.size() + g->cfg.batch - 1) / g->cfg.batch;
}

void ingest_start(ps_ingest *g) {
    if (g->running) return;
    g->running = true;
    const int nt = g->cfg.threads > 1 ? g->cfg.threads : 1;
    for (int i = 0; i < nt; ++i) g->parsers.emplace_back(parser_loop, g);
    static const bool inline_copy = getenv("PS_INGEST_INLINE") != nullptr;      // (measured: the training thread issuing the copies itself, 0.38 ms per step -- not the default)
    g->inline_copy = inline_copy;
    if (!g->inline_copy) {
        g->copier = std::thread(copier_loop, g);
        g->completer = std::thread(completer_loop, g);
    }
}

int ingest_alloc(ps_ingest *g) {
    const ps_ingest_config_t &c = g->cfg;
    const size_t nb = (size_t)c.batch;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    g->off_ids = 0;
    g->off_wide = up(g->off_ids + sizeof(int64_t) * nb * (c.F > 0 ? c.F : 1));
    g->off_dense = up(g->off_wide + sizeof(int64_t) * nb * (c.F > 0 ? c.F : 1));
    g->off_labels = up(g->off_dense + sizeof(float) * nb * (c.X > 0 ? c.X : 1));
    g->off_ids32 = up(g->off_labels + sizeof(float) * nb);
    g->block = up(g->off_ids32 + sizeof(int32_t) * nb * (c.F > 0 ? c.F : 1));
    const int nt = c.threads > 1 ? c.threads : 1;
    g->ring = std::max(4, std::min(128, 2 * nt));
    g->release_every = getenv("PS_INGEST_REL") ? std::max(1, atoi(getenv("PS_INGEST_REL"))) : (g->ring >= 32 ? 4 : 1);
    if (g->release_every > g->ring / 4) g->release_every = std::max(1, g->ring / 4);
    g->slot.resize((size_t)g->ring);
    g->parsed.assign((size_t)g->ring, -1);
    // ONE pinned and ONE device allocation for the whole ring: neighbouring slots are neighbouring blocks, so a GROUP of parsed batches
    // crosses the link in one call (copier_loop)
    HIPCHK(hipHostMalloc((void **)&g->host_all, g->block * (size_t)g->ring, hipHostMallocDefault));
    HIPCHK(hipMalloc((void **)&g->dev_all, g->block * (size_t)g->ring));
    for (size_t k = 0; k < g->slot.size(); ++k) {
        ps_ingest::Slot &S = g->slot[k];
        S.host = g->host_all + k * g->block; S.dev = g->dev_all + k * g->block;
        HIPCHK(hipEventCreateWithFlags(&S.consumed, hipEventDisableTiming));
        HIPCHK(hipEventCreateWithFlags(&S.copied, hipEventDisableTiming));
        S.wait_ev = S.copied; S.consumed_wait = S.consumed;
    }
    HIPCHK(hipStreamCreateWithFlags(&g->copy_stream, hipStreamNonBlocking));
    return PS_OK;
}

int ingest_open(ps_ingest *g) {
    g->st.clear(); g->en.clear();
    if (g->cfg.threads > 1) {
        Pool pool(std::min(g->cfg.threads, 16));
        index_lines_parallel(g->data, g->len, g->cfg.offset, g->cfg.step, &g->st, &g->en, &pool);
    } else {
        index_lines(g->data, g->len, g->cfg.offset, g->cfg.step, &g->st, &g->en);
    }
    ingest_rewind(g);
    return PS_OK;
}

}  // namespace

extern "C" int ps_ingest_create(ps_store_t *s, const ps_ingest_config_t *cfg, ps_ingest_t **out) {
    if (!s || !out) return ps_set_err(PS_E_BAD_ARG, "null argument");
    *out = nullptr;
    PSCHK(check_cfg(cfg));
    PSCHK(store_enter(s));
    ps_ingest *g = new ps_ingest();
    g->s = s; g->cfg = *cfg;
    const int rc = ingest_alloc(g);
    if (rc != PS_OK) { ps_ingest_destroy(g); return rc; }
    *out = g;
    return PS_OK;
}

extern "C" int ps_ingest_destroy(ps_ingest_t *g) {
    if (!g) return PS_OK;
    (void)hipSetDevice(g->s->device);
    ingest_stop(g);
    for (auto &S : g->slot) {
        if (S.consumed) (void)hipEventDestroy(S.consumed);
        if (S.copied) (void)hipEventDestroy(S.copied);
    }
    if (g->host_all) (void)hipHostFree(g->host_all);
    if (g->dev_all) (void)hipFree(g->dev_all);
    if (g->copy_stream) (void)hipStreamDestroy(g->copy_stream);
    if (g->map) munmap(g->map, g->map_len);
    delete g;
    return PS_OK;
}

extern "C" int ps_ingest_open_file(ps_ingest_t *g, const char *path) {
    if (!g || !path) return ps_set_err(PS_E_BAD_ARG, "null argument");
    ingest_stop(g);
    if (g->map) { munmap(g->map, g->map_len); g->map = nullptr; }
    const int fd = open(path, O_RDONLY);
    if (fd < 0) return ps_set_err(PS_MISSING, "cannot open %s", path);
    struct stat sb;
    if (fstat(fd, &sb) != 0) { close(fd); return ps_set_err(PS_MISSING, "cannot stat %s", path); }
    g->map_len = (size_t)sb.st_size;
    if (g->map_len > 0) {
        g->map = mmap(nullptr, g->map_len, PROT_READ, MAP_PRIVATE, fd, 0);
        if (g->map == MAP_FAILED) { g->map = nullptr; close(fd); return ps_set_err(PS_E_HIP, "mmap of %s failed", path); }
        (void)madvise(g->map, g->map_len, MADV_SEQUENTIAL);
    }
    close(fd);
    g->data = (const char *)g->map; g->len = g->map_len;
    return ingest_open(g);
}

extern "C" int ps_ingest_open_memory(ps_ingest_t *g, const char *text, size_t len) {
    if (!g || (!text && len)) return ps_set_err(PS_E_BAD_ARG, "null argument");
    ingest_stop(g);
    g->copy.assign(text, text + len);
    g->data = g->copy.data(); g->len = len;
    return ingest_open(g);
}

extern "C" int ps_ingest_lines(ps_ingest_t *g, int64_t *n_lines) {
    if (!g || !n_lines) return ps_set_err(PS_E_BAD_ARG, "null argument");
    *n_lines = (int64_t)g->st.size();
    return PS_OK;
}

// The next batch (B <= cfg.batch samples) as device pointers, valid until the call after the next one.
// PS_MISSING at the end of the data (FileSource returns null -> DataSet ends the epoch); ps_ingest_reset rewinds.
extern "C" int ps_ingest_next(ps_ingest_t *g, ps_batch_t *out) {
    if (!g || !out) return ps_set_err(PS_E_BAD_ARG, "null argument");
    if (!g->data && g->len == 0 && g->st.empty()) return ps_set_err(PS_E_STATE, "ps_ingest_open_* first");
    HIPCHK(hipSetDevice(g->s->device));
    const int64_t b = g->cur;
    if (b >= g->nbatches) return ps_set_err(PS_MISSING, "end of data");
    ingest_start(g);
    // batch b - 2 goes back to the parsers: its consumers were enqueued on the store's stream before this call; the copier waits
    // (host side) for this event before it overwrites the slot's HBM block
    // (... `rel` batches at a time: every event recorded on the training stream is a barrier packet between two of its kernels, 3-4 us of the
    //  step; one event stands for the slots of the `rel` batches handed out before it)
    const int rel = g->release_every;
    if (b >= 2 && (b - 1) % rel == 0) {
        const int64_t last = b - 2, first = std::max<int64_t>(0, last - rel + 1);
        ps_ingest::Slot &R = g->slot[(size_t)(last % g->ring)];
        static const bool noevent = getenv("PS_INGEST_NOEVENT") != nullptr;      // (measurement only: unsafe)
        if (!noevent) {
            HIPCHK(hipEventRecord(R.consumed, g->s->stream));
            for (int64_t q = first; q <= last; ++q) { ps_ingest::Slot &Q = g->slot[(size_t)(q % g->ring)]; Q.consumed_wait = R.consumed; Q.consumed_recorded = true; }
        }
        {
            std::lock_guard<std::mutex> l(g->mu);
            g->free_upto = last + g->ring + 1;
        }
        g->cv_free.notify_all();
    }
    if (g->inline_copy) {
        // Every parsed batch that has not been sent yet is sent NOW, by this thread (the one that enqueues the step): a copier thread's HIP
        // calls beside the step's launches cost the step 45 us of 135 -- 0.1885 against 0.1442 ms per step with the copies switched off, 12
        // parser threads, whatever the bytes (profiles/r06_ingest_probes.txt).  The slot's previous consumers are waited for ON THE COPY
        // STREAM (same thread: no host wait), the batch handed out is waited for on the host (sent batches ago: normally long done).
        static const bool nocopy = getenv("PS_INGEST_NOCOPY") != nullptr;
        for (;;) {
            const int64_t nb = g->issued_upto;
            if (nb >= g->nbatches) break;
            {
                std::unique_lock<std::mutex> l(g->mu);
                if (g->parsed[(size_t)(nb % g->ring)] != nb) {
                    if (nb > b) break;                      // not needed yet: next call
                    g->cv_parsed.wait(l, [&] { return g->parsed[(size_t)(nb % g->ring)] == nb; });
                }
            }
            ps_ingest::Slot &N = g->slot[(size_t)(nb % g->ring)];
            if (N.rc == PS_OK && N.B > 0 && !nocopy) {
                hipError_t e = hipSuccess;
                if (N.consumed_recorded) e = hipStreamWaitEvent(g->copy_stream, N.consumed_wait, 0);
                e = issue_copy(g, N, e);
                if (e == hipSuccess) e = hipEventRecord(N.copied, g->copy_stream);
                if (e != hipSuccess) { N.rc = PS_E_HIP; snprintf(N.err, sizeof N.err, "ingest H2D: %s", hipGetErrorString(e)); }
            }
            g->issued_upto = nb + 1;
        }
        ps_ingest::Slot &W = g->slot[(size_t)(b % g->ring)];
        if (W.rc == PS_OK && W.B > 0 && !nocopy) HIPCHK(hipEventSynchronize(W.copied));
    } else {
        std::unique_lock<std::mutex> l(g->mu);
        g->cv_ready.wait(l, [&] { return g->ready_upto > b; });
    }
    ps_ingest::Slot &S = g->slot[(size_t)(b % g->ring)];
    if (S.rc != PS_OK) return ps_set_err(S.rc, "%s", S.err);
    memset(out, 0, sizeof *out);
    out->B = S.B;
    out->ids = (int64_t *)(S.dev + g->off_ids); out->offsets = nullptr; out->dense = g->cfg.X > 0 ? (float *)(S.dev + g->off_dense) : nullptr;
    out->labels = (float *)(S.dev + g->off_labels); out->wide_ids = g->cfg.wide_size > 0 ? (int64_t *)(S.dev + g->off_wide) : nullptr;
    out->on_device = 1;
    {
        std::lock_guard<std::mutex> l(g->mu);
        g->cur = b + 1;
    }
    g->cv_parsed.notify_all();          // (the copier gathers groups while the consumer is far enough behind it: tell it where the consumer is)
    return PS_OK;
}

extern "C" int ps_ingest_reset(ps_ingest_t *g) {
    if (!g) return ps_set_err(PS_E_BAD_ARG, "null argument");
    // (the blocks handed out last may still be read by kernels in flight: the next epoch's copies into them wait for the store's stream)
    HIPCHK(hipSetDevice(g->s->device));
    ingest_rewind(g);
    for (auto &S : g->slot) { HIPCHK(hipEventRecord(S.consumed, g->s->stream)); S.consumed_wait = S.consumed; S.consumed_recorded = true; }
    return PS_OK;
}

// parse_seconds: THREAD-seconds the parser threads spent parsing (divide by the threads for wall time); lines and text bytes parsed
extern "C" int ps_ingest_stats(ps_ingest_t *g, double *parse_seconds, int64_t *lines, int64_t *bytes) {
    if (!g) return ps_set_err(PS_E_BAD_ARG, "null argument");
    std::lock_guard<std::mutex> l(g->mu);
    if (parse_seconds) *parse_seconds = g->parse_s;
    if (lines) *lines = g->parsed_lines;
    if (bytes) *bytes = g->parsed_bytes;
    return PS_OK;
}

// CTR.java:84-100's epoch loop (dataSet.next -> trainer.train until the source is dry) for one reader and one model, in C: up to
// max_batches batches (< 0: to the end of the data) of the pipeline trained without a host wait in between (ps_model_train
// with loss = NULL); *trained receives their number.  PS_OK at the end of the data too (ps_ingest_reset rewinds).
extern "C" int ps_ingest_train(ps_ingest_t *g, ps_model_t *m, int64_t max_batches, int64_t *trained) {
    if (!g || !m) return ps_set_err(PS_E_BAD_ARG, "null argument");
    int64_t k = 0;
    int rc = PS_OK;
    // PS_INGEST_TIMING=1 (measurement): where the training thread's time goes, per batch: taking the batch | enqueueing the step
    static const bool timing = getenv("PS_INGEST_TIMING") != nullptr;
    static const int lead = getenv("PS_INGEST_LEAD") ? atoi(getenv("PS_INGEST_LEAD")) : 0;
    double t_next = 0, t_train = 0, t_sync = 0, gpu_ms = 0;
    hipEvent_t ev0 = nullptr, ev1 = nullptr;
    if (timing && lead > 0) { (void)hipEventCreate(&ev0); (void)hipEventCreate(&ev1); (void)hipEventRecord(ev0, g->s->stream); }
    auto now = [] { return std::chrono::duration<double, std::micro>(std::chrono::steady_clock::now().time_since_epoch()).count(); };
    while (max_batches < 0 || k < max_batches) {
        ps_batch_t b;
        const double t0 = timing ? now() : 0;
        rc = ps_ingest_next(g, &b);
        if (rc == PS_MISSING) { rc = PS_OK; break; }
        if (rc != PS_OK) break;
        const double t1 = timing ? now() : 0;
        rc = ps_model_train(m, &b, nullptr);
        if (rc != PS_OK) break;
        if (timing) { t_next += t1 - t0; t_train += now() - t1; }
        ++k;
        if (lead > 0 && k % lead == 0) {       // (measurement: the host at most `lead` steps ahead of the GPU; GPU time of every group of `lead` steps)
            if (timing && ev0) {
                (void)hipEventRecord(ev1, g->s->stream);
                const double ts0 = now();
                (void)hipEventSynchronize(ev1);
                t_sync += now() - ts0;
                float ms = 0.f;
                if (hipEventElapsedTime(&ms, ev0, ev1) == hipSuccess) gpu_ms += ms;
                (void)hipEventRecord(ev0, g->s->stream);
            } else (void)hipStreamSynchronize(g->s->stream);
        }
    }
    if (timing && k > 0) fprintf(stderr, "[ps_ingest_train] %lld batches: %.1f us per batch taking it from the ring, %.1f us enqueueing its step; groups of %d steps: GPU %.1f us per step between the group's events, host %.1f us per step waiting for the group\n",
                                 (long long)k, t_next / k, t_train / k, lead, 1e3 * gpu_ms / k, t_sync / k);
    if (ev0) { (void)hipEventDestroy(ev0); (void)hipEventDestroy(ev1); }
    if (trained) *trained = k;
    return rc;
}
