// Entry points of the layer operators: argument checks, the attention plan, launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <initializer_list>
#include <new>
#include <string>
#include <vector>

#include "../../include/dptm.h"
#include "dptm_layers.h"

using namespace dptm;

namespace {

thread_local std::string g_lerr;

int fail(int code, const std::string& msg) {
    g_lerr = msg;
    return code;
}

// An exception must not leave an extern "C" function: the handlers of the entry points land here.
int on_exception(const char* where) noexcept {
    int code = DPTM_EHIP;
    try {
        try {
            throw;
        } catch (const std::bad_alloc&) {
            code = DPTM_ENOMEM;
            g_lerr = std::string(where) + ": out of host memory";
        } catch (const std::exception& e) {
            g_lerr = std::string(where) + ": " + e.what();
        } catch (...) {
            g_lerr = std::string(where) + ": unknown C++ exception";
        }
    } catch (...) {
    }
    return code;
}

// the caller's current device comes back when the call returns
struct OnDevice {
    int before = -1;
    bool ok = false;
    explicit OnDevice(int device) {
        if (hipGetDevice(&before) != hipSuccess) before = -1;
        ok = (before >= 0 && before == device) || hipSetDevice(device) == hipSuccess;
        if (!ok) (void)hipGetLastError();      // the refusal is the call's result and nobody else's
    }
    ~OnDevice() {
        int now = -1;
        if (before >= 0 && hipGetDevice(&now) == hipSuccess && now != before) (void)hipSetDevice(before);
    }
};

bool good_dim(int d) { return d == 16 || d == 32 || d == 64 || d == 128; }
int size_of(int dtype) { return dtype == DPTM_PREC_F32 ? 4 : 2; }
bool good_type(int t) { return t == DPTM_PREC_F32 || t == DPTM_PREC_BF16 || t == DPTM_PREC_F16; }

// A tensor [rows][heads][dim] whose kernels fetch 16-byte vectors; `written`: rows and heads may not overlap.
int check_rows(const char* who, const char* name, const dptm_rows& t, int64_t rows, int heads, int dim, int dtype, bool written,
               Strided* out) {
    auto at = [&] { return std::string(who) + ": " + name; };
    if (rows == 0) {
        *out = Strided{nullptr, 0, 0};
        return DPTM_OK;
    }
    const int size = size_of(dtype);
    if (!t.data) return fail(DPTM_EINVAL, at() + ": NULL buffer");
    if (t.rows < rows) return fail(DPTM_EINVAL, at() + " has " + std::to_string(t.rows) + " rows, the call needs " + std::to_string(rows));
    if (t.row_stride < 0 || t.head_stride < 0) return fail(DPTM_EINVAL, at() + ": negative stride");
    // a tile's rows are reached by 32-bit offsets from the first
    if (t.row_stride >= (int64_t(1) << 25) / size || t.head_stride > (int64_t(1) << 40))
        return fail(DPTM_EINVAL, at() + ": row stride of 32 MiB or more");
    if ((reinterpret_cast<uintptr_t>(t.data) & 15) || (t.row_stride * size) % 16 || (t.head_stride * size) % 16)
        return fail(DPTM_EINVAL, at() + ": address and strides must be multiples of 16 bytes");
    if (written) {
        const bool rows_outside = (heads == 1 || t.head_stride >= dim) && (rows == 1 || t.row_stride >= (heads - 1) * t.head_stride + dim);
        const bool heads_outside = (rows == 1 || t.row_stride >= dim) && (heads == 1 || t.head_stride >= (rows - 1) * t.row_stride + dim);
        if (!rows_outside && !heads_outside) return fail(DPTM_EINVAL, at() + ": rows or heads of a written tensor overlap");
    }
    *out = Strided{t.data, t.row_stride, t.head_stride};
    return DPTM_OK;
}

// The memory of a tensor of a call, for check_apart: runs of `run` bytes at at + i * step[0] + j * step[1], i < n[0], j < n[1].
struct Place {
    const char* name;
    uintptr_t at;
    int64_t n[2], step[2], run;

    Place(const char* name, const Strided& t, int64_t rows, int heads, int dim, int size)
        : name(name), at(reinterpret_cast<uintptr_t>(t.p)), n{rows, heads}, step{t.row * size, t.head * size}, run((int64_t)dim * size) {
        tidy();
    }
    Place(const char* name, const void* p, int64_t bytes) : name(name), at(reinterpret_cast<uintptr_t>(p)), n{1, 1}, step{0, 0}, run(p ? bytes : 0) {}

    bool empty() const { return !at || n[0] <= 0 || n[1] <= 0 || run <= 0; }
    int64_t bytes() const { return (n[0] - 1) * step[0] + (n[1] - 1) * step[1] + run; }
    // the larger step first, repeated memory once, steps that leave no gap as one run
    void tidy() {
        if (empty()) return;
        for (int d = 0; d < 2; ++d)
            if (n[d] == 1 || step[d] == 0) n[d] = 1, step[d] = 0;
        if (step[0] < step[1]) std::swap(step[0], step[1]), std::swap(n[0], n[1]);
        for (int d = 1; d >= 0; --d)
            if (n[d] > 1 && step[d] <= run && (d || n[1] == 1)) run += (n[d] - 1) * step[d], n[d] = 1, step[d] = 0;
    }
    // whether [from, from + len), counted from `at`, meets a run.  For what is written: there the inner runs of an outer
    // step end before the next one begins (check_rows)
    bool meets(int64_t from, int64_t len) const {
        // the outer steps whose span [i step0, i step0 + span) the bytes touch
        const int64_t span = (n[1] - 1) * step[1] + run;
        auto first_not_before = [](int64_t x, int64_t step, int64_t width) {      // smallest i >= 0 with i step + width > x
            return x < width || step == 0 ? 0 : (x - width) / step + 1;
        };
        for (int64_t i = first_not_before(from, step[0], span); i < n[0] && i * step[0] < from + len; ++i) {
            const int64_t x = from - i * step[0], j = first_not_before(x, step[1], run);
            if (j < n[1] && j * step[1] < x + len && j * step[1] + run > x) return true;
        }
        return false;
    }
};

// Whether two tensors share memory; `a` is written.  Exact: where both go by the same steps -- views of one packed tensor -- from the
// difference of their addresses, otherwise by the runs of `b`, one by one.  Tensors beside each other are told by their bounds.
bool overlap(const Place& a, const Place& b) {
    if (a.empty() || b.empty() || a.at + a.bytes() <= b.at || b.at + b.bytes() <= a.at) return false;
    const int64_t off = (int64_t)(b.at - a.at);
    int64_t step[2];
    bool alike = true;
    for (int d = 0; d < 2; ++d) {
        step[d] = b.n[d] == 1 ? a.step[d] : b.step[d];
        alike &= a.n[d] == 1 || a.step[d] == step[d];
    }
    if (!alike) {
        for (int64_t i = 0; i < b.n[0]; ++i)
            for (int64_t j = 0; j < b.n[1]; ++j)
                if (a.meets(off + i * b.step[0] + j * b.step[1], b.run)) return true;
        return false;
    }
    // runs that are di and dj steps apart meet if -b.run < off + di step + dj step' < a.run: every dj of the shorter direction, and the
    // largest di that satisfies the right side
    const int s = a.n[0] + b.n[0] < a.n[1] + b.n[1] ? 0 : 1, l = 1 - s;
    for (int64_t dj = 1 - a.n[s]; dj < b.n[s]; ++dj) {
        const int64_t x = off + dj * step[s], room = a.run - 1 - x;
        int64_t di = 0;
        if (step[l]) di = std::min(room >= 0 ? room / step[l] : -((-room + step[l] - 1) / step[l]), b.n[l] - 1);
        if (di > -a.n[l] && x + di * step[l] < a.run && x + di * step[l] > -b.run) return true;
    }
    return false;
}

// What a call writes lies apart from what it reads and from what else it writes.
int check_apart(const char* who, const Place& written, std::initializer_list<const Place*> others) {
    for (const Place* o : others)
        if (overlap(written, *o)) return fail(DPTM_EINVAL, std::string(who) + ": " + written.name + " shares memory with " + o->name);
    return DPTM_OK;
}

// The same for the small buffers of a call: the first pair that shares memory.  Reported with the device, which is the last check: a call
// refused for its device says so first.
struct Shared {
    const char *written = nullptr, *with = nullptr;
    void look(const Place& w, std::initializer_list<const Place*> others) {
        for (const Place* o : others)
            if (!written && overlap(w, *o)) written = w.name, with = o->name;
    }
    int check(const char* who, bool device) const {
        if (device && !written) return DPTM_OK;
        std::string msg = std::string(who) + (device ? "" : ": no such device");
        if (written) msg += std::string(device ? ": " : "; ") + written + " shares memory with " + with;
        return fail(DPTM_EINVAL, msg);
    }
};

constexpr int kGroups = 768;   // workgroups that keys are cut for: three a processor

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

uint32_t header_sum(const int32_t* p) {
    uint32_t h = 2166136261u;
    for (int i = 0; i < kPlanHeader; ++i)
        if (i != kPlanCheck) h = (h ^ (uint32_t)p[i]) * 16777619u;
    return h;
}

struct Seq { int q0, nq, k0, nk, pos0, tile0; };

struct PlanMaker {
    int left, right, sinks;
    const int32_t* pos;      // packed, NULL: row i of a sequence stands at i + nk - nq
    std::vector<Seq> seqs;
    std::vector<int> bounds;   // smallest and largest position of every 32 rows, where `pos` is given

    void span(const Seq& s, int first, int n, int* lo, int* hi) const {
        if (!pos) {
            *lo = s.pos0 + first;
            *hi = s.pos0 + first + n - 1;
            return;
        }
        *lo = kFar, *hi = -kFar;
        for (int i = 0; i < n; ++i) {
            const int p = pos[s.q0 + first + i];
            *lo = std::min(*lo, p), *hi = std::max(*hi, p);
        }
    }
    // rows [first, first + n) of a sequence and the keys some of them see
    QItem q_item(const Seq& s, int first, int n) const {
        int lo, hi;
        span(s, first, n, &lo, &hi);
        QItem it{s.q0 + first, n, s.k0, s.pos0 + first, 0, 0, 0, -1};
        it.ke = (int)std::max<int64_t>(0, std::min<int64_t>(s.nk, (int64_t)hi + right + 1));
        it.kb = (int)std::min<int64_t>(it.ke, std::max<int64_t>(0, (int64_t)lo - left));
        it.sink_end = std::min(std::min(sinks, it.kb), it.ke);
        return it;
    }
    static int64_t keys(const QItem& it) { return (int64_t)it.ke - it.kb + it.sink_end; }
    std::vector<QItem> q_items(int tile) const {
        std::vector<QItem> all;
        for (const Seq& s : seqs)
            for (int i = 0; i < s.nq; i += tile) all.push_back(q_item(s, i, std::min(tile, s.nq - i)));
        return all;
    }
    // the rows [qb, qe) that see some of the keys [j0, j1)
    void q_range(const Seq& s, int j0, int j1, int* qb, int* qe) const {
        auto sees = [&](int lo, int hi) {
            return (int64_t)hi + right >= j0 && ((int64_t)lo - left <= j1 - 1 || j0 < sinks);
        };
        *qb = *qe = 0;
        if (!pos) {
            // positions grow with the row: rows from the first whose window reaches j0 to the last whose window still holds j1 - 1
            const int64_t b = std::max<int64_t>(0, (int64_t)j0 - right - s.pos0);
            const int64_t e = j0 < sinks ? s.nq : std::min<int64_t>(s.nq, (int64_t)j1 + left - s.pos0);
            if (b < e) *qb = (int)(b / 32 * 32), *qe = (int)e;
            return;
        }
        bool any = false;
        for (int i = 0; i < s.nq; i += 32)
            if (sees(bounds[2 * (s.tile0 + i / 32)], bounds[2 * (s.tile0 + i / 32) + 1])) {
                if (!any) *qb = i;
                any = true;
                *qe = std::min(i + 32, s.nq);
            }
    }
};

int make_plan(const dptm_attention_desc& d, const int32_t* q_len, const int32_t* k_len, const int32_t* q_pos, int64_t n_seqs,
              std::vector<int32_t>& words) {
    const char* who = "dptm_attention_plan: ";
    PlanMaker m;
    m.left = d.window_left < 0 ? kFar : std::min(d.window_left, kFar);
    m.right = d.window_right < 0 ? kFar : std::min(d.window_right, kFar);
    m.sinks = std::min(d.sinks, kFar);
    m.pos = q_pos;
    int64_t q0 = 0, k0 = 0;
    for (int64_t b = 0; b < n_seqs; ++b) {
        const int nq = q_len[b], nk = k_len ? k_len[b] : q_len[b];
        if (nq < 0 || nk < 0 || nq >= kFar || nk >= kFar)
            return fail(DPTM_EINVAL, std::string(who) + "length of sequence " + std::to_string(b) + " is outside 0..2^29-1");
        m.seqs.push_back(Seq{(int)q0, nq, (int)k0, nk, nk - nq, (int)(m.bounds.size() / 2)});
        int nearest = q_pos ? kFar : nk - nq;
        if (q_pos)
            for (int i = 0; i < nq; i += 32) {
                int lo = kFar, hi = -kFar;
                for (int r = i; r < std::min(i + 32, nq); ++r) {
                    const int p = q_pos[q0 + r];
                    if (p <= -kFar || p >= kFar) return fail(DPTM_EINVAL, std::string(who) + "a position is outside -2^29..2^29");
                    lo = std::min(lo, p), hi = std::max(hi, p);
                }
                m.bounds.push_back(lo);
                m.bounds.push_back(hi);
                nearest = std::min(nearest, lo);
            }
        // a side without limit is one of 2^29
        if (m.right == kFar && nq && nk && (int64_t)nk - 1 - nearest > kFar)
            return fail(DPTM_EINVAL, std::string(who) + "a key lies more than 2^29 positions ahead of a row of a window without a right limit");
        q0 += nq, k0 += nk;
        if (q0 > INT32_MAX || k0 > INT32_MAX) return fail(DPTM_EINVAL, std::string(who) + "more than 2^31-1 rows");
    }
    int64_t t32 = 0, t64 = 0, t128 = 0;
    for (const Seq& s : m.seqs) t32 += up(s.nq, 32) / 32, t64 += up(s.nq, 64) / 64, t128 += up(s.nq, 128) / 128;

    // Forward.  Tiles of 128 rows while they fill the card twice and waste little; of 64 below; workgroups that split the
    // keys of 32 rows where even those leave processors idle, or no sequence has more rows than one wavefront takes.
    int mode = kWide128;
    if (t64 * d.heads < 256 || t32 == t64) mode = kSplitKeys;
    else if (t128 * d.heads < 512 || t64 * 64 * 5 < t128 * 128 * 4) mode = kWide64;
    // Where keys are split, a tile's 32 rows are queries of up to eight heads that read the same keys (their bias tables
    // have to fit LDS together), as many as the longest sequence leaves room for.
    int pack = 1;
    if (mode == kSplitKeys) {
        int longest = 1;
        for (const Seq& s : m.seqs) longest = std::max(longest, s.nq);
        for (int p = 2; p <= 8; ++p)
            if (d.heads / d.kv_heads % p == 0 && p * std::min(longest, 32) <= 32) pack = p;
    }
    std::vector<QItem> fwd = m.q_items(mode == kWide128 ? 128 : mode == kWide64 ? 64 : 32 / pack);
    std::vector<Join> joins;
    int slots = 0;
    if (mode == kSplitKeys) {
        int64_t total = 0;
        for (const QItem& it : fwd) total += m.keys(it);
        // keys of a workgroup: at least four tiles of each of its four wavefronts (joining parts takes a launch of 4 us), and no
        // more parts than fill the card
        const int64_t chunk = std::max<int64_t>(512, up((total * (d.heads / pack) + kGroups - 1) / kGroups, 128));
        std::vector<QItem> cut;
        for (const QItem& it : fwd) {
            const int64_t n = it.ke - it.kb, parts = std::max<int64_t>(1, (n + chunk - 1) / chunk);
            if (parts == 1) {
                cut.push_back(it);
                continue;
            }
            const int64_t each = up((n + parts - 1) / parts, 32);
            Join j{it.q0, it.nq, slots, 0};
            for (int64_t b = it.kb; b < it.ke; b += each) {
                QItem p = it;
                p.kb = (int)b, p.ke = (int)std::min<int64_t>(it.ke, b + each);
                if (b != it.kb) p.sink_end = 0;
                p.slot = slots++;
                ++j.slots;
                cut.push_back(p);
            }
            joins.push_back(j);
        }
        fwd.swap(cut);
        // tiles that read the same keys one behind the other, so that they meet in an L2 (53 rows over 34,003 keys, 20 heads:
        // 181 MB from memory instead of 250; the time stays, 57 us, it waits for tiles one by one)
        std::stable_sort(fwd.begin(), fwd.end(), [](const QItem& a, const QItem& b) { return a.k0 != b.k0 ? a.k0 < b.k0 : a.kb < b.kb; });
    }
    auto heavy = [](const QItem& a, const QItem& b) { return PlanMaker::keys(a) > PlanMaker::keys(b); };
    std::stable_sort(fwd.begin(), fwd.end(), heavy);

    // Backward.  Batches of short sequences: both in one kernel.  Otherwise dq as the forward pass without splitting; dk, dv by tiles of keys, the range of rows cut where there
    // are few tiles, or where a tile (the first keys of a window with sinks) sees far more rows than the others.
    std::vector<QItem> dq;
    std::vector<KItem> dkv;
    std::vector<Join> dkv_joins;
    int dq_waves = 4, dkv_waves = 4, dkv_slots = 0;
    int longest = 0;
    for (const Seq& s : m.seqs) longest = std::max(longest, std::max(s.nq, s.nk));
    if (d.training && !q_pos && d.heads == d.kv_heads && d.head_dim <= kShortDim && longest <= 64) {
        dq_waves = kTogether, dkv_waves = longest <= 32 ? 1 : 2;
        for (const Seq& s : m.seqs) {
            if (s.nq + s.nk == 0) continue;
            dq.push_back(m.q_item(s, 0, s.nq));
            KItem it{s.k0, s.nk, 0, s.q0, 0, 0, s.pos0, -1, s.tile0, s.nq, {0, 0}};
            m.q_range(s, 0, s.nk, &it.qb, &it.qe);
            dkv.push_back(it);
        }
    } else if (d.training) {
        if (t128 * d.heads < 512 || t64 * 64 * 5 < t128 * 128 * 4) dq_waves = 2;
        dq = m.q_items(32 * dq_waves);
        std::stable_sort(dq.begin(), dq.end(), heavy);
        int64_t k64 = 0, k128 = 0;
        for (const Seq& s : m.seqs) k64 += up(s.nk, 64) / 64, k128 += up(s.nk, 128) / 128;
        if (k128 * d.kv_heads < 512 || k64 * 64 * 5 < k128 * 128 * 4) dkv_waves = 2;
        const int tile = 32 * dkv_waves;
        int64_t total = 0;
        for (const Seq& s : m.seqs)
            for (int j = 0; j < s.nk; j += tile) {
                KItem it{s.k0 + j, std::min(tile, s.nk - j), j, s.q0, 0, 0, s.pos0, -1, s.tile0, s.nq, {0, 0}};
                m.q_range(s, j, j + it.nk, &it.qb, &it.qe);
                dkv.push_back(it);
                total += it.qe - it.qb;
            }
        const int64_t n = (int64_t)dkv.size();
        if (n) {
            const int64_t chunk = n * d.kv_heads >= kGroups ? std::max<int64_t>(1024, up(2 * total / n, 64))
                                                            : std::max<int64_t>(128, up((total * d.kv_heads + kGroups - 1) / kGroups, 64));
            std::vector<KItem> cut;
            for (const KItem& it : dkv) {
                const int64_t rows = it.qe - it.qb, parts = std::max<int64_t>(1, (rows + chunk - 1) / chunk);
                if (parts == 1) {
                    cut.push_back(it);
                    continue;
                }
                const int64_t each = up((rows + parts - 1) / parts, 64);
                Join j{it.k0, it.nk, dkv_slots, 0};
                for (int64_t b = it.qb; b < it.qe; b += each) {
                    KItem p = it;
                    p.qb = (int)b, p.qe = (int)std::min<int64_t>(it.qe, b + each);
                    p.slot = dkv_slots++;
                    ++j.slots;
                    cut.push_back(p);
                }
                dkv_joins.push_back(j);
            }
            dkv.swap(cut);
            std::stable_sort(dkv.begin(), dkv.end(), [](const KItem& a, const KItem& b) { return a.qe - a.qb > b.qe - b.qb; });
        }
    }
    // threads of a launch are counted in 32 bits
    const int64_t most = (int64_t(1) << 32) / 256 - 1;
    if ((int64_t)fwd.size() * d.heads > most || (int64_t)dq.size() * d.heads > most || (int64_t)dkv.size() * d.kv_heads > most)
        return fail(DPTM_EINVAL, std::string(who) + "too many tiles for one launch");

    words.assign(kPlanHeader, 0);
    auto append = [&](const void* p, size_t bytes) {
        const int at = (int)words.size();
        words.resize(words.size() + bytes / 4);
        if (bytes) memcpy(words.data() + at, p, bytes);
        return at;
    };
    const int fwd_at = append(fwd.data(), fwd.size() * sizeof(QItem));
    const int join_at = append(joins.data(), joins.size() * sizeof(Join));
    const int dq_at = append(dq.data(), dq.size() * sizeof(QItem));
    const int dkv_at = append(dkv.data(), dkv.size() * sizeof(KItem));
    const int dkv_join_at = append(dkv_joins.data(), dkv_joins.size() * sizeof(Join));
    const int pos_at = append(q_pos, q_pos ? (size_t)q0 * 4 : 0);
    const int tiles_at = append(m.bounds.data(), m.bounds.size() * 4);
    if (words.size() > (size_t)INT32_MAX) return fail(DPTM_EINVAL, std::string(who) + "plan too large");
    int32_t* p = words.data();
    p[kPlanMagicAt] = kPlanMagic, p[kPlanWords] = (int32_t)words.size();
    p[kPlanHeads] = d.heads, p[kPlanKvHeads] = d.kv_heads, p[kPlanHeadDim] = d.head_dim;
    p[kPlanLeft] = m.left, p[kPlanRight] = m.right, p[kPlanSinks] = m.sinks;
    p[kPlanSeqs] = (int32_t)n_seqs, p[kPlanQRows] = (int32_t)q0, p[kPlanKRows] = (int32_t)k0;
    p[kPlanMode] = mode, p[kPlanFwd] = (int32_t)fwd.size(), p[kPlanFwdAt] = fwd_at, p[kPlanSlots] = slots;
    p[kPlanJoin] = (int32_t)joins.size(), p[kPlanJoinAt] = join_at;
    p[kPlanDq] = (int32_t)dq.size(), p[kPlanDqAt] = dq_at, p[kPlanDqWaves] = d.training ? dq_waves : 0;
    p[kPlanDkv] = (int32_t)dkv.size(), p[kPlanDkvAt] = dkv_at, p[kPlanDkvWaves] = dkv_waves, p[kPlanDkvSlots] = dkv_slots;
    p[kPlanDkvJoin] = (int32_t)dkv_joins.size(), p[kPlanDkvJoinAt] = dkv_join_at;
    p[kPlanHasPos] = q_pos ? 1 : 0, p[kPlanPosAt] = pos_at;
    p[kPlanTiles] = (int32_t)(m.bounds.size() / 2), p[kPlanTilesAt] = tiles_at;
    p[kPlanPack] = pack;
    p[kPlanCheck] = (int32_t)header_sum(p);
    return DPTM_OK;
}

int check_plan(const char* who, const int32_t* plan, const int32_t* plan_dev) {
    if (!plan || !plan_dev) return fail(DPTM_EINVAL, std::string(who) + ": NULL plan");
    if ((reinterpret_cast<uintptr_t>(plan) | reinterpret_cast<uintptr_t>(plan_dev)) & 3) return fail(DPTM_EINVAL, std::string(who) + ": plan must be 4-byte aligned");
    if (plan[kPlanMagicAt] != kPlanMagic || plan[kPlanCheck] != (int32_t)header_sum(plan))
        return fail(DPTM_EINVAL, std::string(who) + ": not a plan of dptm_attention_plan");
    return DPTM_OK;
}

// byte sizes of the workspace's parts, each rounded up to 256
struct Work { size_t fwd_o, fwd_ml, delta, dkv, bias, groups; };
// the tiles whose sums make the bias gradient: of keys, or of rows where the plan lists positions
int bias_items(const int32_t* p) { return p[p[kPlanHasPos] ? kPlanDq : kPlanDkv]; }
Work work_of(const int32_t* p, int n_buckets, int reach) {
    Work w;
    const size_t dim = p[kPlanHeadDim], heads = p[kPlanHeads], kv = p[kPlanKvHeads];
    w.fwd_o = up((size_t)p[kPlanSlots] * (heads / p[kPlanPack]) * 32 * dim * 4, 256);
    w.fwd_ml = up((size_t)p[kPlanSlots] * (heads / p[kPlanPack]) * 32 * 2 * 4, 256);
    w.delta = up(heads * (size_t)p[kPlanQRows] * 4, 256);
    w.dkv = up((size_t)p[kPlanDkvSlots] * kv * 2 * 32 * (size_t)p[kPlanDkvWaves] * dim * 4, 256);
    w.bias = up(heads * (size_t)bias_items(p) * (size_t)(n_buckets ? dtable_words(p[kPlanHasPos], n_buckets, reach) : 0) * 4, 256);
    w.groups = n_buckets ? up(heads * (size_t)dtable_groups(bias_items(p)) * (size_t)dtable_words(p[kPlanHasPos], n_buckets, reach) * 8, 256) : 0;
    return w;
}

constexpr int kMaxBuckets = 64, kMaxReach = 1024;

int check_bias(const char* who, const dptm_attention_args& x, BiasArgs* out) {
    *out = BiasArgs{nullptr, nullptr, 0, 0};
    if (!x.table && !x.buckets) return DPTM_OK;
    if (!x.table || !x.buckets) return fail(DPTM_EINVAL, std::string(who) + ": table and buckets go together");
    if (x.n_buckets < 1 || x.n_buckets > kMaxBuckets) return fail(DPTM_EINVAL, std::string(who) + ": 1 to 64 buckets are supported");
    if (x.max_distance < 0 || x.max_distance > kMaxReach)
        return fail(DPTM_EINVAL, std::string(who) + ": a largest distance of 0 to 1024 is supported");
    if ((reinterpret_cast<uintptr_t>(x.buckets) & 3) || (reinterpret_cast<uintptr_t>(x.table) & 3 & (size_of(x.dtype) - 1)))
        return fail(DPTM_EINVAL, std::string(who) + ": table and buckets must be aligned to their elements");
    *out = BiasArgs{x.table, x.buckets, x.n_buckets, x.max_distance};
    return DPTM_OK;
}

int check_common(const char* who, const dptm_attention_args& x, size_t need) {
    const float scale = x.scale;
    const void* ws = x.workspace;
    const size_t have = x.workspace_bytes;
    if (!good_type(x.dtype)) return fail(DPTM_EINVAL, std::string(who) + ": dtype must be DPTM_PREC_F32, _BF16 or _F16");
    // the kernels start the score products from lse and bias over the scale
    if (!(scale >= 0x1p-64f && scale <= 0x1p64f)) return fail(DPTM_EINVAL, std::string(who) + ": scale must be in 2^-64..2^64");
    if (need && (!ws || have < need))
        return fail(DPTM_EINVAL, std::string(who) + ": workspace of " + std::to_string(need) + " bytes needed, " + std::to_string(ws ? have : 0) + " given");
    if (need && (reinterpret_cast<uintptr_t>(ws) & 255)) return fail(DPTM_EINVAL, std::string(who) + ": workspace must be 256-byte aligned");
    return DPTM_OK;
}

AttnArgs common_args(const int32_t* p, const int32_t* dev, float scale) {
    AttnArgs a{};
    a.plan = dev;
    a.scale = scale;
    a.heads = p[kPlanHeads];
    a.group = p[kPlanHeads] / p[kPlanKvHeads];
    a.left = p[kPlanLeft], a.right = p[kPlanRight], a.sinks = p[kPlanSinks];
    a.q_rows = p[kPlanQRows];
    a.pack = p[kPlanPack];
    a.has_pos = p[kPlanHasPos], a.pos_at = p[kPlanPosAt], a.tiles_at = p[kPlanTilesAt];
    return a;
}

int hip_result(const char* who, hipError_t e) {
    return e == hipSuccess ? DPTM_OK : fail(DPTM_EHIP, std::string(who) + ": " + hipGetErrorString(e));
}

#define BY_TYPE(F, ...) (dtype == DPTM_PREC_BF16 ? F##_bf16(__VA_ARGS__) : dtype == DPTM_PREC_F16 ? F##_f16(__VA_ARGS__) : F##_f32(__VA_ARGS__))
#define OK_OR_RETURN(x)            \
    do {                           \
        const int rc_ = (x);       \
        if (rc_) return rc_;       \
    } while (0)

}  // namespace

extern "C" {

const char* dptm_layer_last_error(void) { return g_lerr.c_str(); }

int64_t dptm_attention_plan(const dptm_attention_desc* d, const int32_t* q_len, const int32_t* k_len, const int32_t* q_pos,
                            int64_t n_seqs, int32_t* plan, int64_t capacity) try {
    const char* who = "dptm_attention_plan: ";
    if (!d) return fail(DPTM_EINVAL, std::string(who) + "NULL description");
    if (d->heads < 1 || d->kv_heads < 1 || d->heads > 4096 || d->heads % d->kv_heads)
        return fail(DPTM_EINVAL, std::string(who) + "heads must be 1..4096 and a multiple of kv_heads");
    if (!good_dim(d->head_dim)) return fail(DPTM_EINVAL, std::string(who) + "head_dim must be 16, 32, 64 or 128");
    if (d->sinks < 0) return fail(DPTM_EINVAL, std::string(who) + "negative number of first tokens");
    if (n_seqs < 0 || n_seqs > INT32_MAX || (n_seqs > 0 && !q_len)) return fail(DPTM_EINVAL, std::string(who) + "bad sequence lengths");
    if (capacity < 0 || (capacity > 0 && !plan)) return fail(DPTM_EINVAL, std::string(who) + "NULL plan");
    std::vector<int32_t> words;
    OK_OR_RETURN(make_plan(*d, q_len, k_len, q_pos, n_seqs, words));
    if ((int64_t)words.size() <= capacity) memcpy(plan, words.data(), words.size() * 4);
    return (int64_t)words.size();
} catch (...) {
    return on_exception("dptm_attention_plan");
}

int64_t dptm_attention_workspace(const int32_t* plan, int32_t n_buckets, int32_t max_distance, int32_t backward) try {
    OK_OR_RETURN(check_plan("dptm_attention_workspace", plan, plan));
    if (n_buckets < 0 || n_buckets > kMaxBuckets) return fail(DPTM_EINVAL, "dptm_attention_workspace: 0 to 64 buckets are supported");
    if (max_distance < 0 || max_distance > kMaxReach)
        return fail(DPTM_EINVAL, "dptm_attention_workspace: a largest distance of 0 to 1024 is supported");
    const Work w = work_of(plan, n_buckets, max_distance);
    return (int64_t)(backward ? w.delta + w.dkv + w.bias + w.groups : w.fwd_o + w.fwd_ml);
} catch (...) {
    return on_exception("dptm_attention_workspace");
}

int dptm_attention_forward(const dptm_attention_args* args) try {
    const char* who = "dptm_attention_forward";
    if (!args) return fail(DPTM_EINVAL, std::string(who) + ": NULL arguments");
    const dptm_attention_args& x = *args;
    const int32_t* plan = x.plan;
    OK_OR_RETURN(check_plan(who, plan, x.plan_dev));
    const Work w = work_of(plan, 0, 0);
    OK_OR_RETURN(check_common(who, x, w.fwd_o + w.fwd_ml));
    const int heads = plan[kPlanHeads], kv = plan[kPlanKvHeads], dim = plan[kPlanHeadDim], dtype = x.dtype;
    const int64_t nq = plan[kPlanQRows], nk = plan[kPlanKRows];
    AttnArgs a = common_args(plan, x.plan_dev, x.scale);
    OK_OR_RETURN(check_rows(who, "q", x.q, nq, heads, dim, dtype, false, &a.q));
    OK_OR_RETURN(check_rows(who, "k", x.k, nk, kv, dim, dtype, false, &a.k));
    OK_OR_RETURN(check_rows(who, "v", x.v, nk, kv, dim, dtype, false, &a.v));
    OK_OR_RETURN(check_rows(who, "out", x.out, nq, heads, dim, dtype, true, &a.out));
    OK_OR_RETURN(check_bias(who, x, &a.bias));
    if (nq == 0) return DPTM_OK;
    if (!x.lse || (reinterpret_cast<uintptr_t>(x.lse) & 3)) return fail(DPTM_EINVAL, std::string(who) + ": lse is NULL or misaligned");
    const int size = size_of(dtype);
    const Place pq{"q", a.q, nq, heads, dim, size}, pk{"k", a.k, nk, kv, dim, size}, pv{"v", a.v, nk, kv, dim, size};
    const Place po{"out", a.out, nq, heads, dim, size}, pl{"lse", x.lse, 4 * heads * nq}, pw{"workspace", x.workspace, (int64_t)(w.fwd_o + w.fwd_ml)};
    const Place pt{"table", a.bias.table, (int64_t)a.bias.n_buckets * heads * size}, pb{"buckets", a.bias.buckets, 4 * (2 * (int64_t)a.bias.reach + 1)};
    const Place pp{"plan", x.plan_dev, 4 * (int64_t)plan[kPlanWords]};
    OK_OR_RETURN(check_apart(who, po, {&pq, &pk, &pv}));
    Shared shared;
    shared.look(po, {&pl, &pw, &pt, &pb, &pp});
    shared.look(pl, {&pq, &pk, &pv, &pw, &pt, &pb, &pp});
    shared.look(pw, {&pq, &pk, &pv, &pt, &pb, &pp});
    a.lse = x.lse;
    a.part_o = static_cast<float*>(x.workspace);
    a.part_ml = reinterpret_cast<float*>(static_cast<char*>(x.workspace) + w.fwd_o);
    a.n_items = plan[kPlanFwd], a.items_at = plan[kPlanFwdAt];
    // tiles that share no keys: better the heads' parts of the same cache lines together (heads of 64 bytes: 58 -> 54 us)
    a.by_sequence = plan[kPlanFwd] <= plan[kPlanSeqs];
    const OnDevice on(x.device);
    OK_OR_RETURN(shared.check(who, on.ok));
    const hipStream_t s = static_cast<hipStream_t>(x.stream);
    OK_OR_RETURN(hip_result(who, BY_TYPE(attn_forward, a, dim, plan[kPlanMode], s)));
    return hip_result(who, BY_TYPE(attn_join, a, dim, plan[kPlanJoin], plan[kPlanJoinAt], s));
} catch (...) {
    return on_exception("dptm_attention_forward");
}

int dptm_attention_backward(const dptm_attention_args* args) try {
    const char* who = "dptm_attention_backward";
    if (!args) return fail(DPTM_EINVAL, std::string(who) + ": NULL arguments");
    const dptm_attention_args& x = *args;
    const int32_t* plan = x.plan;
    OK_OR_RETURN(check_plan(who, plan, x.plan_dev));
    if (!plan[kPlanDqWaves]) return fail(DPTM_EINVAL, std::string(who) + ": the plan was made without training");
    AttnArgs a = common_args(plan, x.plan_dev, x.scale);
    OK_OR_RETURN(check_bias(who, x, &a.bias));
    const Work w = work_of(plan, a.bias.n_buckets, a.bias.reach);
    OK_OR_RETURN(check_common(who, x, w.delta + w.dkv + w.bias + w.groups));
    const int heads = plan[kPlanHeads], kv = plan[kPlanKvHeads], dim = plan[kPlanHeadDim], dtype = x.dtype;
    const int64_t nq = plan[kPlanQRows], nk = plan[kPlanKRows];
    OK_OR_RETURN(check_rows(who, "dout", x.dout, nq, heads, dim, dtype, false, &a.dout));
    OK_OR_RETURN(check_rows(who, "q", x.q, nq, heads, dim, dtype, false, &a.q));
    OK_OR_RETURN(check_rows(who, "k", x.k, nk, kv, dim, dtype, false, &a.k));
    OK_OR_RETURN(check_rows(who, "v", x.v, nk, kv, dim, dtype, false, &a.v));
    OK_OR_RETURN(check_rows(who, "out", x.out, nq, heads, dim, dtype, false, &a.out));
    OK_OR_RETURN(check_rows(who, "dq", x.dq, nq, heads, dim, dtype, true, &a.dq));
    OK_OR_RETURN(check_rows(who, "dk", x.dk, nk, kv, dim, dtype, true, &a.dk));
    OK_OR_RETURN(check_rows(who, "dv", x.dv, nk, kv, dim, dtype, true, &a.dv));
    if (nq && (!x.lse || (reinterpret_cast<uintptr_t>(x.lse) & 3))) return fail(DPTM_EINVAL, std::string(who) + ": lse is NULL or misaligned");
    if (a.bias.table && (!x.dtable || (reinterpret_cast<uintptr_t>(x.dtable) & 3 & (size_of(dtype) - 1))))
        return fail(DPTM_EINVAL, std::string(who) + ": bias without an aligned buffer for its gradient");
    const int size = size_of(dtype);
    const Place pq{"q", a.q, nq, heads, dim, size}, pk{"k", a.k, nk, kv, dim, size}, pv{"v", a.v, nk, kv, dim, size};
    const Place po{"out", a.out, nq, heads, dim, size}, pg{"dout", a.dout, nq, heads, dim, size};
    const Place pdq{"dq", a.dq, nq, heads, dim, size}, pdk{"dk", a.dk, nk, kv, dim, size}, pdv{"dv", a.dv, nk, kv, dim, size};
    const Place pl{"lse", x.lse, 4 * heads * nq}, pw{"workspace", x.workspace, (int64_t)(w.delta + w.dkv + w.bias + w.groups)};
    const int64_t entries = (int64_t)a.bias.n_buckets * heads * size;
    const Place pt{"table", a.bias.table, entries}, pb{"buckets", a.bias.buckets, 4 * (2 * (int64_t)a.bias.reach + 1)}, pdt{"dtable", x.dtable, entries};
    const Place pp{"plan", x.plan_dev, 4 * (int64_t)plan[kPlanWords]};
    OK_OR_RETURN(check_apart(who, pdq, {&pq, &pk, &pv, &po, &pg, &pdk, &pdv}));
    OK_OR_RETURN(check_apart(who, pdk, {&pq, &pk, &pv, &po, &pg, &pdv}));
    OK_OR_RETURN(check_apart(who, pdv, {&pq, &pk, &pv, &po, &pg}));
    Shared shared;
    for (const Place* p : {&pdq, &pdk, &pdv}) shared.look(*p, {&pl, &pt, &pb, &pp, &pdt, &pw});
    shared.look(pdt, {&pq, &pk, &pv, &po, &pg, &pl, &pt, &pb, &pp, &pw});
    shared.look(pw, {&pq, &pk, &pv, &po, &pg, &pl, &pt, &pb, &pp});
    a.lse = x.lse;
    a.delta = static_cast<float*>(x.workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(x.workspace) + w.delta);
    a.part_bias = reinterpret_cast<float*>(static_cast<char*>(x.workspace) + w.delta + w.dkv);
    a.part_groups = reinterpret_cast<double*>(static_cast<char*>(x.workspace) + w.delta + w.dkv + w.bias);
    a.dtable = x.dtable;
    const OnDevice on(x.device);
    OK_OR_RETURN(shared.check(who, on.ok));
    const hipStream_t s = static_cast<hipStream_t>(x.stream);
    a.n_items = plan[kPlanDq], a.items_at = plan[kPlanDqAt];
    if (plan[kPlanDqWaves] == kTogether) {
        OK_OR_RETURN(hip_result(who, BY_TYPE(attn_short_grad, a, dim, plan[kPlanDkvWaves], plan[kPlanDkvAt], s)));
        return a.bias.table ? hip_result(who, BY_TYPE(attn_dtable, a, plan[kPlanDq], s)) : DPTM_OK;
    }
    OK_OR_RETURN(hip_result(who, BY_TYPE(attn_dq, a, dim, plan[kPlanDqWaves], s)));
    a.n_items = plan[kPlanDkv], a.items_at = plan[kPlanDkvAt];
    OK_OR_RETURN(hip_result(who, BY_TYPE(attn_dkv, a, dim, plan[kPlanDkvWaves], s)));
    if (a.bias.table) OK_OR_RETURN(hip_result(who, BY_TYPE(attn_dtable, a, bias_items(plan), s)));
    return hip_result(who, BY_TYPE(attn_dkv_join, a, dim, plan[kPlanDkvJoin], plan[kPlanDkvJoinAt], 32 * plan[kPlanDkvWaves], s));
} catch (...) {
    return on_exception("dptm_attention_backward");
}

static int norm_rope_args(const char* who, const dptm_norm_rope_args* x, NormRopeArgs* a) {
    if (!x) return fail(DPTM_EINVAL, std::string(who) + ": NULL arguments");
    if (!good_type(x->dtype)) return fail(DPTM_EINVAL, std::string(who) + ": dtype must be DPTM_PREC_F32, _BF16 or _F16");
    if (!good_dim(x->head_dim)) return fail(DPTM_EINVAL, std::string(who) + ": head_dim must be 16, 32, 64 or 128");
    if (x->heads < 0 || x->kv_heads < 0 || x->heads + x->kv_heads < 1 || x->heads > 4096 || x->kv_heads > 4096)
        return fail(DPTM_EINVAL, std::string(who) + ": 0 to 4096 heads each, at least one in all");
    if (x->rows < 0 || x->rows > (int64_t(1) << 31) - 1) return fail(DPTM_EINVAL, std::string(who) + ": bad row count");
    if (!(x->eps >= 0.f) || !std::isfinite(x->eps)) return fail(DPTM_EINVAL, std::string(who) + ": eps must be finite and not negative");
    if (x->n_positions < 0) return fail(DPTM_EINVAL, std::string(who) + ": negative number of positions");
    // every row's heads, D / 16 lanes each: threads of a launch are counted in 32 bits
    if (x->rows * (x->heads + x->kv_heads) * (x->head_dim / 16) >= (int64_t(1) << 32) - 256)
        return fail(DPTM_EINVAL, std::string(who) + ": too many rows for one launch");
    if (x->rows && (!x->cosv || !x->sinv || (reinterpret_cast<uintptr_t>(x->cosv) & 15) || (reinterpret_cast<uintptr_t>(x->sinv) & 15)))
        return fail(DPTM_EINVAL, std::string(who) + ": cos / sin are NULL or not 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(x->positions) & 3) || (reinterpret_cast<uintptr_t>(x->q_gain) & 15) || (reinterpret_cast<uintptr_t>(x->k_gain) & 15))
        return fail(DPTM_EINVAL, std::string(who) + ": positions must be 4-byte and gains 16-byte aligned");
    *a = NormRopeArgs{};
    OK_OR_RETURN(check_rows(who, "q", x->q, x->heads ? x->rows : 0, x->heads, x->head_dim, x->dtype, false, &a->x[0]));
    OK_OR_RETURN(check_rows(who, "k", x->k, x->kv_heads ? x->rows : 0, x->kv_heads, x->head_dim, x->dtype, false, &a->x[1]));
    a->heads[0] = x->heads, a->heads[1] = x->kv_heads;
    a->gain[0] = x->q_gain, a->gain[1] = x->k_gain;
    a->cosv = x->cosv, a->sinv = x->sinv, a->positions = x->positions;
    a->rows = x->rows, a->n_pos = x->n_positions, a->dim = x->head_dim, a->interleaved = x->interleaved ? 1 : 0, a->eps = x->eps;
    return DPTM_OK;
}

// A head's result may take the place of what it is made from, element for element, and lies apart from the rest.
static int norm_rope_apart(const char* who, const dptm_norm_rope_args& x, const Strided (&from)[2], const Strided (&to)[2], const char* const (&name)[4],
                           Shared* shared) {
    const int size = size_of(x.dtype), n[2] = {x.heads, x.kv_heads};
    const Place f0{name[0], from[0], x.rows, n[0], x.head_dim, size}, f1{name[1], from[1], x.rows, n[1], x.head_dim, size};
    const Place t0{name[2], to[0], x.rows, n[0], x.head_dim, size}, t1{name[3], to[1], x.rows, n[1], x.head_dim, size};
    auto same = [&](int i) {
        return from[i].p == to[i].p && (x.rows == 1 || from[i].row == to[i].row) && (n[i] == 1 || from[i].head == to[i].head);
    };
    OK_OR_RETURN(check_apart(who, t0, {&f1, &t1}));
    OK_OR_RETURN(check_apart(who, t1, {&f0}));
    if (!same(0)) OK_OR_RETURN(check_apart(who, t0, {&f0}));
    if (!same(1)) OK_OR_RETURN(check_apart(who, t1, {&f1}));
    const int64_t table = (int64_t)x.n_positions * (x.head_dim / 2) * 4, gain = (int64_t)x.head_dim * 4;
    const Place c{"cos", x.cosv, table}, s{"sin", x.sinv, table}, p{"positions", x.positions, x.rows * 4};
    const Place g0{"q_gain", x.q_gain, gain}, g1{"k_gain", x.k_gain, gain};
    for (const Place* t : {&t0, &t1}) shared->look(*t, {&c, &s, &p, &g0, &g1});
    return DPTM_OK;
}

int dptm_qk_norm_rope_forward(const dptm_norm_rope_args* x) try {
    const char* who = "dptm_qk_norm_rope_forward";
    NormRopeArgs a;
    OK_OR_RETURN(norm_rope_args(who, x, &a));
    OK_OR_RETURN(check_rows(who, "q_out", x->q_out, x->heads ? x->rows : 0, x->heads, x->head_dim, x->dtype, true, &a.y[0]));
    OK_OR_RETURN(check_rows(who, "k_out", x->k_out, x->kv_heads ? x->rows : 0, x->kv_heads, x->head_dim, x->dtype, true, &a.y[1]));
    Shared shared;
    OK_OR_RETURN(norm_rope_apart(who, *x, a.x, a.y, {"q", "k", "q_out", "k_out"}, &shared));
    if (x->rows == 0) return DPTM_OK;
    const OnDevice on(x->device);
    OK_OR_RETURN(shared.check(who, on.ok));
    return hip_result(who, norm_rope_forward(a, x->dtype, static_cast<hipStream_t>(x->stream)));
} catch (...) {
    return on_exception("dptm_qk_norm_rope_forward");
}

int64_t dptm_qk_norm_rope_workspace(const dptm_norm_rope_args* x) try {
    if (!x || !good_dim(x->head_dim) || x->rows < 0 || x->rows > INT32_MAX || x->heads < 0 || x->heads > 4096 || x->kv_heads < 0 || x->kv_heads > 4096)
        return fail(DPTM_EINVAL, "dptm_qk_norm_rope_workspace: bad sizes");
    return (int64_t)norm_rope_blocks(x->rows, x->heads + x->kv_heads, x->head_dim) * x->head_dim * 2 * 4;
} catch (...) {
    return on_exception("dptm_qk_norm_rope_workspace");
}

int dptm_qk_norm_rope_backward(const dptm_norm_rope_args* x) try {
    const char* who = "dptm_qk_norm_rope_backward";
    NormRopeArgs a;
    OK_OR_RETURN(norm_rope_args(who, x, &a));
    const int64_t rq = x->heads ? x->rows : 0, rk = x->kv_heads ? x->rows : 0;
    OK_OR_RETURN(check_rows(who, "dq_out", x->dq_out, rq, x->heads, x->head_dim, x->dtype, false, &a.dy[0]));
    OK_OR_RETURN(check_rows(who, "dk_out", x->dk_out, rk, x->kv_heads, x->head_dim, x->dtype, false, &a.dy[1]));
    OK_OR_RETURN(check_rows(who, "dq", x->dq, rq, x->heads, x->head_dim, x->dtype, true, &a.dx[0]));
    OK_OR_RETURN(check_rows(who, "dk", x->dk, rk, x->kv_heads, x->head_dim, x->dtype, true, &a.dx[1]));
    if ((x->q_gain && !x->dq_gain) || (x->k_gain && !x->dk_gain))
        return fail(DPTM_EINVAL, std::string(who) + ": gain without a buffer for its gradient");
    if ((reinterpret_cast<uintptr_t>(x->dq_gain) & 3) || (reinterpret_cast<uintptr_t>(x->dk_gain) & 3))
        return fail(DPTM_EINVAL, std::string(who) + ": gradients of gains must be aligned to their elements");
    const int64_t half = dptm_qk_norm_rope_workspace(x) / 2;
    if ((x->q_gain || x->k_gain) && (!x->workspace || x->workspace_bytes < (size_t)half * 2 || (reinterpret_cast<uintptr_t>(x->workspace) & 255)))
        return fail(DPTM_EINVAL, std::string(who) + ": workspace of " + std::to_string(half * 2) + " bytes, 256-byte aligned, needed");
    Shared shared;
    OK_OR_RETURN(norm_rope_apart(who, *x, a.dy, a.dx, {"dq_out", "dk_out", "dq", "dk"}, &shared));
    OK_OR_RETURN(norm_rope_apart(who, *x, a.x, a.dx, {"q", "k", "dq", "dk"}, &shared));
    if (x->q_gain || x->k_gain) {
        const int size = size_of(x->dtype), dim = x->head_dim;
        const int64_t table = (int64_t)x->n_positions * (dim / 2) * 4;
        const Place q{"q", a.x[0], x->rows, x->heads, dim, size}, k{"k", a.x[1], x->rows, x->kv_heads, dim, size};
        const Place gq{"dq_out", a.dy[0], x->rows, x->heads, dim, size}, gk{"dk_out", a.dy[1], x->rows, x->kv_heads, dim, size};
        const Place dq{"dq", a.dx[0], x->rows, x->heads, dim, size}, dk{"dk", a.dx[1], x->rows, x->kv_heads, dim, size};
        const Place c{"cos", x->cosv, table}, s{"sin", x->sinv, table}, p{"positions", x->positions, x->rows * 4};
        const Place g0{"q_gain", x->q_gain, dim * 4}, g1{"k_gain", x->k_gain, dim * 4}, w{"workspace", x->workspace, half * 2};
        const Place d0{"dq_gain", x->q_gain ? x->dq_gain : nullptr, dim * 4}, d1{"dk_gain", x->k_gain ? x->dk_gain : nullptr, dim * 4};
        shared.look(d0, {&q, &k, &gq, &gk, &dq, &dk, &c, &s, &p, &g0, &g1, &d1, &w});
        shared.look(d1, {&q, &k, &gq, &gk, &dq, &dk, &c, &s, &p, &g0, &g1, &w});
        shared.look(w, {&q, &k, &gq, &gk, &dq, &dk, &c, &s, &p, &g0, &g1});
    }
    a.part[0] = static_cast<float*>(x->workspace);
    a.part[1] = x->workspace ? reinterpret_cast<float*>(static_cast<char*>(x->workspace) + half) : nullptr;
    a.dgain[0] = x->dq_gain, a.dgain[1] = x->dk_gain;
    const OnDevice on(x->device);
    OK_OR_RETURN(shared.check(who, on.ok));
    return hip_result(who, norm_rope_backward(a, x->dtype, static_cast<hipStream_t>(x->stream)));
} catch (...) {
    return on_exception("dptm_qk_norm_rope_backward");
}

}  // extern "C"
