// kr_kv.cpp -- entry points of the operators over a caller's paged cache: checks of arguments, the plan of a step, the division of attention into workgroups.
#include <math.h>

#include <algorithm>
#include <vector>

#include "kr_engine_internal.h"
#include "kr_kv.h"

namespace {
constexpr int KV_CUS = 256;
// header of a plan; the arrays follow: row0 [batch + 1], lens [batch], page0 [batch], pages [entries], slots [rows]
enum { H_BATCH, H_ROWS, H_ENTRIES, H_PAGE_TOKENS, H_PAGES, H_OWN, H_SIZE = 8 };

struct Plan {
    int batch, rows, entries;
    const int *row0, *lens, *page0, *pages, *slots;
    explicit Plan(const int* p) : batch(p[H_BATCH]), rows(p[H_ROWS]), entries(p[H_ENTRIES]) {
        row0 = p + H_SIZE; lens = row0 + batch + 1; page0 = lens + batch; pages = page0 + batch; slots = pages + entries;
    }
};
int bits_of(int format) { return format == KR_KV_BF16 || format == KR_KV_F16 ? 16 : format == KR_KV_E4M3 || format == KR_KV_MX8 ? 8 : 4; }
int fmt_of(int format) { return bits_of(format) == 16 ? 0 : bits_of(format) == 8 ? 1 : 2; }
bool scaled(int format) { return format == KR_KV_MX8 || format == KR_KV_MX4; }
bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }

int check_pages(const kr_kv_pages* p, const int* plan, KvPages& o) {
    if (!p || !plan) return kr_fail(KR_ERR_VALUE, "kr_kv: pages and plan must not be null");
    if (p->format < KR_KV_BF16 || p->format > KR_KV_MX4) return kr_fail(KR_ERR_VALUE, "kr_kv: unknown page format %d", p->format);
    if (p->kv_heads < 1 || p->dim < 32 || p->dim > 256 || p->dim % 32) return kr_fail(KR_ERR_VALUE, "kr_kv: %d heads of %d channels (a multiple of 32 up to 256)", p->kv_heads, p->dim);
    if (p->kv_heads > 4096) return kr_fail(KR_ERR_VALUE, "kr_kv: %d heads", p->kv_heads);
    if (p->page_tokens < 1 || p->n_pages < 1 || (int64_t)p->page_tokens * p->n_pages > INT32_MAX) return kr_fail(KR_ERR_VALUE, "kr_kv: %d pages of %d tokens", p->n_pages, p->page_tokens);
    if (plan[H_PAGE_TOKENS] != p->page_tokens || plan[H_PAGES] != p->n_pages)
        return kr_fail(KR_ERR_VALUE, "kr_kv: the plan is for %d pages of %d tokens, the cache has %d of %d", plan[H_PAGES], plan[H_PAGE_TOKENS], p->n_pages, p->page_tokens);
    if (!p->k || !p->v || misaligned(p->k) || misaligned(p->v)) return kr_fail(KR_ERR_VALUE, "kr_kv: pages must be aligned to 16 bytes");
    if (scaled(p->format) != (p->k_scale != nullptr) || scaled(p->format) != (p->v_scale != nullptr)) return kr_fail(KR_ERR_VALUE, "kr_kv: scales belong to the microscaled formats, and only to them");
    o.k = (uint8_t*)p->k; o.v = (uint8_t*)p->v; o.ks = (uint8_t*)p->k_scale; o.vs = (uint8_t*)p->v_scale;
    o.head_bytes = p->dim * bits_of(p->format) / 8; o.row_bytes = o.head_bytes * p->kv_heads;
    o.shead_bytes = scaled(p->format) ? p->dim / 32 : 0; o.srow_bytes = o.shead_bytes * p->kv_heads;
    if (p->format == KR_KV_E4M3) { o.ks = o.k; o.vs = o.v; o.shead_bytes = o.head_bytes; o.srow_bytes = o.row_bytes; }      // read, and replaced by 127
    if ((int64_t)p->page_tokens * p->n_pages * (o.row_bytes / 16) > UINT32_MAX) return kr_fail(KR_ERR_VALUE, "kr_kv: %d pages of %d tokens are more than 64 GiB", p->n_pages, p->page_tokens);
    o.row16 = (uint32_t)o.row_bytes / 16; o.scale_and = scaled(p->format) ? 0xFFu : 0u; o.scale_or = scaled(p->format) ? 0u : 127u;
    o.scale_shift = p->format == KR_KV_MX8 ? 1 : 0;
    o.page = kv_divisor((uint32_t)p->page_tokens);
    return KR_OK;
}
KvSeqs seqs_of(const int* plan, const int* dev) {
    const Plan h(plan);
    KvSeqs s;
    s.batch = h.batch; s.rows = h.rows;
    s.row0 = dev + (h.row0 - plan); s.lens = dev + (h.lens - plan); s.page0 = dev + (h.page0 - plan); s.pages = dev + (h.pages - plan); s.slots = dev + (h.slots - plan);
    return s;
}
hipStream_t stream_of(void* s) { return s == (void*)1 ? nullptr : (hipStream_t)s; }
int launched(const char* what, int rc) {
    if (rc) return kr_fail(KR_ERR_HIP, "%s: the launch was refused", what);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KR_OK : kr_fail(KR_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

int rows_call(const char* what, const kr_kv_pages* p, const int* plan, const int* dev, const void* k, const void* v, const int64_t* strides, int dtype, void* stream, bool write) {
    KvRowsArgs a{};
    if (int rc = check_pages(p, plan, a.p)) return rc;
    if (dtype != KR_KV_BF16 && dtype != KR_KV_F16) return kr_fail(KR_ERR_VALUE, "%s: rows are bf16 or f16", what);
    if (write && !plan[H_OWN]) return kr_fail(KR_ERR_VALUE, "%s: two of the step's rows lie in one slot", what);
    const KvSeqs s = seqs_of(plan, dev);
    if (!s.rows) return KR_OK;
    if (!dev || !k || !v || !strides || misaligned(k) || misaligned(v)) return kr_fail(KR_ERR_VALUE, "%s: rows must be aligned to 16 bytes", what);
    for (int i = 0; i < 4; i++) if (strides[i] % 8) return kr_fail(KR_ERR_VALUE, "%s: strides must be multiples of 8 elements", what);
    if ((int64_t)s.rows * (p->kv_heads * p->dim / 8) > INT32_MAX - 4096) return kr_fail(KR_ERR_VALUE, "%s: %d rows are too many for one call", what, s.rows);
    a.slots = s.slots; a.rows = s.rows; a.k = (void*)k; a.v = (void*)v;
    a.k_tok = strides[0]; a.k_head = strides[1]; a.v_tok = strides[2]; a.v_head = strides[3];
    a.per_row = kv_divisor((uint32_t)(p->kv_heads * p->dim / 8)); a.per_head = kv_divisor((uint32_t)(p->dim / 8)); a.format = p->format; a.half = dtype == KR_KV_F16;
    return launched(what, write ? kr_launch_kv_write(a, stream_of(stream)) : kr_launch_kv_read(a, stream_of(stream)));
}

// one launch's share of a call: the sequences whose rows (new tokens x heads of a group) lie in a range
struct Part { int min_rows, max_rows, bm, kt, tps; int64_t items, units; int shares; bool split, few, one; };
// How many key tiles a workgroup takes.  A workgroup works on `side` tiles side by side, `deep` workgroups share a CU's time.  With k workgroups a CU a launch lasts k tiles' time for every
// `side` tiles of a share, what it takes to begin and to end (`extra`) for every `deep` workgroups, and `join` more when shares have to be joined (all in the time of a tile): the cheapest
// number up to 4 * deep is taken.  More row tiles than that fill the chip evenly by themselves.  Measured around the choice, us at shares of so many tiles: a dozen drafts of eight chats
// 2: 23.9, 3 (taken): 21.0, 4: 21.6, 6: 23.4; 64 drafts late in four documents 32: 146, 54 (taken): 120, 64: 130; nine sequences of 496 tokens, 33 drafts each, 2: 37.7, 3 (taken): 25.1,
// 4: 27.5, all 8: 29.8; 32 single tokens of up to 8192 96: 35.4, the choice 34.5, 128: 40.6.
void divide(const Plan& h, int kv_heads, int G, int window, int first, bool tree, int deep, int side, int extra, int join, Part& p) {
    constexpr int hold = KV_CUS;
    struct Seq { int tiles; int64_t row_tiles; };
    std::vector<Seq> seqs;
    int64_t total = 0, whole = 0; int longest = 0;
    for (int b = 0; b < h.batch; b++) {
        const int cnt = h.row0[b + 1] - h.row0[b]; const int64_t rows = (int64_t)cnt * G;
        if (rows < p.min_rows || rows > p.max_rows) continue;
        const int n = kv_tiles_ub(h.lens[b], cnt, kv_divisor((uint32_t)G), window, first, tree, p.bm, p.kt);
        const int64_t rt = (int64_t)kv_row_tiles(cnt, G, p.bm) * kv_heads;
        seqs.push_back({n, rt}); total += rt * n; whole += rt; longest = n > longest ? n : longest;
    }
    p.items = whole; p.units = 0; p.split = p.few = false; p.tps = longest > 0 ? longest : 1;
    if (seqs.empty()) return;
    auto items = [&](int tps) { int64_t n = 0; for (const Seq& s : seqs) n += s.row_tiles * ((s.tiles + tps - 1) / tps); return n; };
    auto cost = [&](int64_t k, int tiles) { return k * ((tiles + side - 1) / side) + (k + deep - 1) / deep * extra; };
    if (whole < 4ll * deep * hold) {
        const int least = std::max(side, (longest + KV_MAX_SHARES - 1) / KV_MAX_SHARES);
        int64_t k = (whole + hold - 1) / hold, best = cost(k, longest);
        for (; k <= 4 * deep; k++) {
            int lo = std::max(least, (int)(total / (k * hold))), hi = longest;      // the smallest share whose items fit
            while (lo < hi) { const int mid = lo + (hi - lo) / 2; if (items(mid) <= k * hold) hi = mid; else lo = mid + 1; }
            if (lo < longest && cost(k, lo) + join < best) { best = cost(k, lo) + join; p.tps = lo; }
        }
    }
    int most = 1;
    p.items = 0;
    for (const Seq& s : seqs) {
        const int ns = (s.tiles + p.tps - 1) / p.tps;
        p.items += s.row_tiles * ns;
        if (ns > 1) p.split = true;
        most = ns > most ? ns : most;
    }
    p.shares = most;
    // Up to 16 shares are joined 16 rows a workgroup, which reads them one after the other, more of them a row a workgroup (kr_kv_join.hip).  From 9 shares on the former needs a workgroup
    // for every CU: 13 shares of 700 such workgroups 43.5 -> 33 us, of 320 21.4 -> 18.9, but 16 shares of 128 21.6 -> 25.8, 13 of 8 14.1 -> 15.2 us.
    int64_t units = 0, rows = 0;
    for (const Seq& s : seqs) if (s.tiles > p.tps) { units += s.row_tiles * (p.bm / 16); rows += s.row_tiles * p.bm; }
    p.few = most <= 8 || (most <= 16 && (p.bm == KV_STEP_BM || units >= KV_CUS));
    p.units = p.few ? units : rows;
}
void parts_of(const Plan& h, int kv_heads, int heads, int dim, int fmt, bool half, int window, int first, bool tree, Part* p) {
    const int G = heads / kv_heads;
    p[0] = Part{1, KV_STEP_BM, KV_STEP_BM, KV_STEP_KT, 0, 0, 0, 1, false, false, false};
    // Eight waves share what brings a tile to LDS where two of them fit on a SIMD and some sequence has rows for more than four: two prompts of up to 8192 tokens 1289 -> 1217 us,
    // 64 drafts late in four documents 145 -> 133.
    int64_t most = 0;
    for (int b = 0; b < h.batch; b++) most = std::max(most, (int64_t)(h.row0[b + 1] - h.row0[b]) * G);
    const int waves = (dim == 96 || dim == 128) && most > 128 ? 8 : 4;
    p[1] = Part{KV_STEP_BM + 1, INT32_MAX, 32 * waves, KV_TILE_KT, 0, 0, 0, 1, false, false, false};
    bool one = !tree;
    for (int b = 0; b < h.batch && one; b++) { const int64_t cnt = h.row0[b + 1] - h.row0[b]; one = cnt <= 1 || cnt * G > KV_STEP_BM; }
    p[0].one = one;
    divide(h, kv_heads, G, window, first, tree, 1, kv_step_waves(dim, fmt, half, one), 3, 3, p[0]);
    divide(h, kv_heads, G, window, first, tree, waves == 8 ? 1 : kv_tile_waves(dim, fmt, half), 1, 6, 4, p[1]);
}
size_t part_bytes(const Part& p, int dim) { return p.split ? (size_t)p.items * p.bm * (dim + 2) * sizeof(float) : 0; }

int check_attend(const kr_kv_pages* p, const int* plan, int heads, int window, int keep_first, bool tree, KvPages& o) {
    if (int rc = check_pages(p, plan, o)) return rc;
    if (p->dim != 64 && p->dim != 96 && p->dim != 128 && p->dim != 192 && p->dim != 256) return kr_fail(KR_ERR_VALUE, "kr_kv_attend: heads of %d channels (64, 96, 128, 192 or 256)", p->dim);
    if (heads < 1 || heads % p->kv_heads) return kr_fail(KR_ERR_VALUE, "kr_kv_attend: %d heads do not divide among %d key / value heads", heads, p->kv_heads);
    if (window < 0 || keep_first < 0) return kr_fail(KR_ERR_VALUE, "kr_kv_attend: window %d, keep_first %d", window, keep_first);
    const Plan h(plan);
    for (int b = 0; b < h.batch; b++) {
        const int64_t cnt = h.row0[b + 1] - h.row0[b];
        if (cnt * (heads / p->kv_heads) > INT32_MAX / 2) return kr_fail(KR_ERR_VALUE, "kr_kv_attend: %lld new tokens of sequence %d are too many for one call", (long long)cnt, b);
        if (tree && cnt > KV_MAX_TREE) return kr_fail(KR_ERR_VALUE, "kr_kv_attend: %lld drafts of sequence %d, at most %d", (long long)cnt, b, KV_MAX_TREE);
    }
    return KR_OK;
}
int clamp_first(const Plan& h, int window, int keep_first) {      // more first tokens than any sequence has are all of them
    int longest = 0;
    for (int b = 0; b < h.batch; b++) longest = h.lens[b] > longest ? h.lens[b] : longest;
    return window ? (keep_first < longest ? keep_first : longest) : 0;
}
}  // namespace

extern "C" int kr_kv_plan(int n_pages, int page_tokens, int batch, const int* lens, const int* counts, const int* tables, const int* table_lens, int* plan, size_t ints, size_t* need) {
    if (batch < 0 || page_tokens < 1 || n_pages < 1 || (int64_t)n_pages * page_tokens > INT32_MAX) return kr_fail(KR_ERR_VALUE, "kr_kv_plan: %d sequences, %d pages of %d tokens", batch, n_pages, page_tokens);
    if ((batch && (!lens || !counts || !tables || !table_lens)) || !need) return kr_fail(KR_ERR_VALUE, "kr_kv_plan: null argument");
    int64_t rows = 0, entries = 0;
    for (int b = 0; b < batch; b++) {
        if (counts[b] < 0 || lens[b] < counts[b]) return kr_fail(KR_ERR_VALUE, "kr_kv_plan: sequence %d has %d tokens, %d of them new", b, lens[b], counts[b]);
        if (table_lens[b] < 0 || (int64_t)table_lens[b] * page_tokens < lens[b]) return kr_fail(KR_ERR_VALUE, "kr_kv_plan: sequence %d has %d tokens in %d pages of %d", b, lens[b], table_lens[b], page_tokens);
        if (lens[b] > INT32_MAX - 4096) return kr_fail(KR_ERR_VALUE, "kr_kv_plan: sequence %d has %d tokens", b, lens[b]);      // positions are 32-bit, tiles of them end past the last
        rows += counts[b]; entries += ((int64_t)lens[b] + page_tokens - 1) / page_tokens;
    }
    if (rows > INT32_MAX || entries > INT32_MAX || H_SIZE + 3ll * batch + 1 + rows + entries > INT32_MAX) return kr_fail(KR_ERR_VALUE, "kr_kv_plan: %lld new rows, %lld pages are too many for one step", (long long)rows, (long long)entries);
    *need = (size_t)(H_SIZE + 3 * (int64_t)batch + 1 + rows + entries);
    if (!plan) return KR_OK;
    if (ints < *need) return kr_fail(KR_ERR_VALUE, "kr_kv_plan: %zu integers for a plan of %zu", ints, *need);
    try {
        int* row0 = plan + H_SIZE; int* ln = row0 + batch + 1; int* page0 = ln + batch; int* pages = page0 + batch; int* slots = pages + entries;
        std::vector<uint8_t> written((size_t)n_pages, 0);
        bool own = true;                                      // no slot twice: a page that gets rows twice may still hold them apart
        int r = 0, e = 0; int64_t t0 = 0;
        for (int b = 0; b < batch; b++) {
            row0[b] = r; ln[b] = lens[b]; page0[b] = e;
            const int n = (int)(((int64_t)lens[b] + page_tokens - 1) / page_tokens), before = lens[b] - counts[b];
            for (int i = 0; i < n; i++) {
                const int id = tables[t0 + i];
                if (id < 0 || id >= n_pages) return kr_fail(KR_ERR_VALUE, "kr_kv_plan: sequence %d lists page %d of %d", b, id, n_pages);
                pages[e + i] = id;
            }
            for (int j = before; j < lens[b];) {
                const int pg = j / page_tokens, id = pages[e + pg];
                if (written[id]) own = false;
                written[id] = 1;
                const int64_t stop = ((int64_t)pg + 1) * page_tokens;
                for (; j < lens[b] && j < stop; j++) slots[r++] = id * page_tokens + (j - pg * page_tokens);
            }
            e += n; t0 += table_lens[b];
        }
        row0[batch] = r;
        if (!own) {
            std::vector<int> sorted(slots, slots + r);
            std::sort(sorted.begin(), sorted.end());
            own = std::adjacent_find(sorted.begin(), sorted.end()) == sorted.end();
        }
        for (int i = 0; i < H_SIZE; i++) plan[i] = 0;
        plan[H_BATCH] = batch; plan[H_ROWS] = r; plan[H_ENTRIES] = e; plan[H_PAGE_TOKENS] = page_tokens; plan[H_PAGES] = n_pages; plan[H_OWN] = own;
    } catch (const std::exception& x) { return kr_fail(KR_ERR_STATE, "kr_kv_plan: %s", x.what()); }
    return KR_OK;
}

extern "C" int kr_kv_write(const kr_kv_pages* p, const int* plan, const int* dev_plan, const void* k, const void* v, const int64_t* strides, int dtype, void* stream) {
    return rows_call("kr_kv_write", p, plan, dev_plan, k, v, strides, dtype, stream, true);
}
extern "C" int kr_kv_read(const kr_kv_pages* p, const int* plan, const int* dev_plan, void* k, void* v, const int64_t* strides, int dtype, void* stream) {
    return rows_call("kr_kv_read", p, plan, dev_plan, k, v, strides, dtype, stream, false);
}

static int attend_workspace(const kr_kv_pages* p, const int* plan, int heads, int dtype, int window, int keep_first, int tree, size_t* bytes) {
    KvPages o;
    if (int rc = check_attend(p, plan, heads, window, keep_first, tree != 0, o)) return rc;
    if (!bytes) return kr_fail(KR_ERR_VALUE, "kr_kv_attend_workspace: null argument");
    const Plan h(plan);
    Part part[2];
    parts_of(h, p->kv_heads, heads, p->dim, fmt_of(p->format), dtype == KR_KV_F16, window, clamp_first(h, window, keep_first), tree != 0, part);
    *bytes = part_bytes(part[0], p->dim) + part_bytes(part[1], p->dim);
    return KR_OK;
}

static int attend(const kr_kv_pages* p, const int* plan, const int* dev_plan, const void* q, int64_t q_token_stride, int64_t q_head_stride, void* out, int dtype, int heads, float scale,
                            int window, int keep_first, const int* parents, void* workspace, size_t workspace_bytes, void* stream) {
    KvAttnArgs a{};
    if (int rc = check_attend(p, plan, heads, window, keep_first, parents != nullptr, a.p)) return rc;
    if (dtype != KR_KV_BF16 && dtype != KR_KV_F16) return kr_fail(KR_ERR_VALUE, "kr_kv_attend: queries are bf16 or f16");
    if (bits_of(p->format) == 16 && p->format != dtype) return kr_fail(KR_ERR_VALUE, "kr_kv_attend: queries of another 16-bit type than the pages");
    const float scale_log2 = scale * 1.44269504088896340736f;
    if (!isfinite(scale_log2)) return kr_fail(KR_ERR_VALUE, "kr_kv_attend: scale %g", scale);
    const Plan h(plan);
    if (!h.rows) return KR_OK;
    if (!dev_plan || !q || !out || misaligned(q) || misaligned(out)) return kr_fail(KR_ERR_VALUE, "kr_kv_attend: queries and output must be aligned to 16 bytes");
    if (q_token_stride % 8 || q_head_stride % 8) return kr_fail(KR_ERR_VALUE, "kr_kv_attend: strides must be multiples of 8 elements");
    a.s = seqs_of(plan, dev_plan);
    a.q = (const uint16_t*)q; a.out = (uint16_t*)out; a.q_tok = q_token_stride; a.q_head = q_head_stride; a.parents = parents;
    a.heads = heads; a.kv_heads = kv_divisor((uint32_t)p->kv_heads); a.G = kv_divisor((uint32_t)(heads / p->kv_heads));
    a.window = window; a.first = clamp_first(h, window, keep_first);
    a.scale_log2 = scale_log2;
    Part part[2];
    parts_of(h, p->kv_heads, heads, p->dim, fmt_of(p->format), dtype == KR_KV_F16, window, a.first, parents != nullptr, part);
    const size_t b0 = part_bytes(part[0], p->dim), b1 = part_bytes(part[1], p->dim);
    if (workspace_bytes < b0 + b1 || ((b0 + b1) && (!workspace || misaligned(workspace)))) return kr_fail(KR_ERR_VALUE, "kr_kv_attend: a workspace of %zu bytes for %zu", workspace_bytes, b0 + b1);
    if (part[0].items > INT32_MAX || part[1].items > INT32_MAX || part[0].units > INT32_MAX || part[0].shares > KV_MAX_SHARES || part[1].shares > KV_MAX_SHARES || part[1].units > INT32_MAX) return kr_fail(KR_ERR_VALUE, "kr_kv_attend: %d rows are too many for one call", h.rows);
    const int fmt = fmt_of(p->format), half = dtype == KR_KV_F16;
    hipStream_t st = stream_of(stream);
    static int (*const step[3])(const KvAttnArgs&, int, int, hipStream_t) = {kr_launch_kv_step_16, kr_launch_kv_step_8, kr_launch_kv_step_4};
    static int (*const tile[3])(const KvAttnArgs&, int, int, int, hipStream_t) = {kr_launch_kv_tile_16, kr_launch_kv_tile_8, kr_launch_kv_tile_4};
    for (int i = 1; i >= 0; i--) {                            // prompts first, they take longest
        if (!part[i].items) continue;
        a.min_rows = part[i].min_rows; a.max_rows = part[i].max_rows; a.tps = kv_divisor((uint32_t)part[i].tps); a.items = (int)part[i].items; a.whole = a.items / (8 * p->kv_heads) * (8 * p->kv_heads); a.one = part[i].one;
        a.ws = (float*)((char*)workspace + (i ? b0 : 0));
        if (int rc = launched("kr_kv_attend", i ? tile[fmt](a, p->dim, half, part[i].bm / 32, st) : step[fmt](a, p->dim, half, st))) return rc;
        if (part[i].split)
            if (int rc = launched("kr_kv_attend", kr_launch_kv_join(a, p->dim, part[i].bm, part[i].kt, (int)part[i].units, part[i].few, half, st))) return rc;
    }
    return KR_OK;
}

// no exception leaves a C entry: the division of a call keeps a list of its sequences
extern "C" int kr_kv_attend_workspace(const kr_kv_pages* p, const int* plan, int heads, int dtype, int window, int keep_first, int tree, size_t* bytes) {
    try { return attend_workspace(p, plan, heads, dtype, window, keep_first, tree, bytes); }
    catch (const std::exception& x) { return kr_fail(KR_ERR_STATE, "kr_kv_attend_workspace: %s", x.what()); }
}
extern "C" int kr_kv_attend(const kr_kv_pages* p, const int* plan, const int* dev_plan, const void* q, int64_t q_token_stride, int64_t q_head_stride, void* out, int dtype, int heads, float scale,
                            int window, int keep_first, const int* parents, void* workspace, size_t workspace_bytes, void* stream) {
    try { return attend(p, plan, dev_plan, q, q_token_stride, q_head_stride, out, dtype, heads, scale, window, keep_first, parents, workspace, workspace_bytes, stream); }
    catch (const std::exception& x) { return kr_fail(KR_ERR_STATE, "kr_kv_attend: %s", x.what()); }
}

extern "C" int kr_kv_move(const kr_kv_pages* p, int layers, int n_seq, const int* dev_start, const int* dev_src, const int* dev_dst, void* stream) {
    const int like[H_SIZE] = {0, 0, 0, p ? p->page_tokens : 0, p ? p->n_pages : 0, 1, 0, 0};
    KvPages o;
    if (int rc = check_pages(p, like, o)) return rc;
    if (layers < 0 || n_seq < 0 || n_seq > 65535 || layers > 16383) return kr_fail(KR_ERR_VALUE, "kr_kv_move: %d layers, %d sequences", layers, n_seq);
    if (!layers || !n_seq) return KR_OK;
    if (!dev_start || !dev_src || !dev_dst) return kr_fail(KR_ERR_VALUE, "kr_kv_move: null argument");
    KvMoveArgs a{};
    const int64_t slots = (int64_t)p->n_pages * p->page_tokens;
    a.base[0] = o.k; a.base[1] = o.v; a.base[2] = (uint8_t*)p->k_scale; a.base[3] = (uint8_t*)p->v_scale;
    for (int i = 0; i < 4; i++) { a.row_bytes[i] = i < 2 ? o.row_bytes : scaled(p->format) ? o.srow_bytes : 0; a.layer_bytes[i] = slots * a.row_bytes[i]; }
    a.start = dev_start; a.src = dev_src; a.dst = dev_dst; a.n_seq = n_seq; a.layers = layers;
    return launched("kr_kv_move", kr_launch_kv_move(a, stream_of(stream)));
}
