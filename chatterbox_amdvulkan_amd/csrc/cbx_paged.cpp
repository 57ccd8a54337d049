// cbx_paged.cpp -- the C ABI of decoding many streams over a paged key-value
// cache: argument checks in front of k_paged_plan.hip, k_qk.hip,
// k_paged_attn.hip and k_logprob.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "cbx_internal.h"

namespace cbx {
namespace {

constexpr int64_t k2G = int64_t{1} << 31;
// Workgroups of 256 threads stay below this many: a launch has fewer than 2^32 threads.
constexpr int64_t kMostGroups = int64_t{1} << 24;

int fail(int code, const char* what, const char* msg) { return set_error(code, std::string(what) + ": " + msg); }
int bad(const char* what, const char* msg) { return fail(CBX_ERR_INVALID_ARG, what, msg); }

// Whether an element of a and one of b share a byte.  Views that interleave
// in one buffer (q and k of one projection, K and V of one allocation) have
// overlapping byte ranges but equal strides: the index difference t of each
// stride, from the largest on, is then tried where the rest can still meet.
// Different strides: the ranges decide.
struct Dim { int64_t stride, na, nb; };

bool lattice_meets(const Dim* d, int n, int64_t delta, int64_t es) {
    if (n == 0) return delta < es && -delta < es;
    int64_t span_a = es, span_b = es;          // of the dims after this one
    for (int i = 1; i < n; i++) {
        span_a += (d[i].na - 1) * d[i].stride;
        span_b += (d[i].nb - 1) * d[i].stride;
    }
    // b's rest starts at delta + t * stride: it can meet a's for
    // -span_b < delta + t * stride < span_a
    const int64_t s = d[0].stride;
    auto floor_div = [](int64_t x, int64_t y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
    const int64_t lo = std::max(-(d[0].na - 1), floor_div(-span_b - delta, s) + 1);
    const int64_t hi = std::min(d[0].nb - 1, floor_div(span_a - 1 - delta, s));
    if (hi - lo >= 8) return true;             // rows that run into each other: taken as one
    for (int64_t t = lo; t <= hi; t++) {
        if (lattice_meets(d + 1, n - 1, delta + t * s, es)) return true;
    }
    return false;
}

bool meets(const cbx_tensor* a, const cbx_tensor* b) {
    if (nelements(a) == 0 || nelements(b) == 0 || !bytes_overlap(a, b)) return false;
    if (type_size(a->type) != type_size(b->type)) return true;
    Dim d[4];
    int n = 0;
    for (int i = 0; i < 4; i++) {
        if (a->ne[i] == 1 && b->ne[i] == 1) continue;
        if (a->ne[i] > 1 && b->ne[i] > 1 && a->nb[i] != b->nb[i]) return true;
        const int64_t s = static_cast<int64_t>(a->ne[i] > 1 ? a->nb[i] : b->nb[i]);
        if (s == 0) return true;
        int k = n++;
        for (; k > 0 && d[k - 1].stride < s; k--) d[k] = d[k - 1];
        d[k] = Dim{s, a->ne[i], b->ne[i]};
    }
    return lattice_meets(d, n, reinterpret_cast<intptr_t>(b->data) - reinterpret_cast<intptr_t>(a->data),
                         static_cast<int64_t>(type_size(a->type)));
}

// An output written by many workgroups: no element stands for two.
bool repeats(const cbx_tensor* t) {
    if (nelements(t) == 0) return false;
    for (int i = 0; i < 4; i++) if (t->ne[i] > 1 && t->nb[i] == 0) return true;
    return false;
}

bool is_itself(const cbx_tensor* a, const cbx_tensor* b) {
    if (a->data != b->data || a->type != b->type || !same_shape(a, b)) return false;
    for (int i = 0; i < 4; i++) if (a->ne[i] > 1 && a->nb[i] != b->nb[i]) return false;
    return true;
}

// A 1-D I32 tensor of n elements.
int check_ints(const cbx_tensor* t, int64_t n, const char* what, const char* name) {
    int rc = validate(t, what, name);
    if (rc) return rc;
    if (t->type != CBX_TYPE_I32 || t->ne[1] != 1 || t->ne[2] != 1 || t->ne[3] != 1 || (n >= 0 && t->ne[0] != n)) {
        return set_error(CBX_ERR_INVALID_ARG, std::string(what) + ": " + name + " must be 1-D I32" +
                                                  (n >= 0 ? " with " + std::to_string(n) + " elements" : ""));
    }
    return CBX_OK;
}

int check_floats(const cbx_tensor* t, const char* what, const char* name) {
    int rc = validate(t, what, name);
    if (rc) return rc;
    if (t->type != CBX_TYPE_F32 && t->type != CBX_TYPE_F16) {
        return set_error(CBX_ERR_UNSUPPORTED, std::string(what) + ": " + name + " must be F32 or F16");
    }
    return CBX_OK;
}

int check_tables(const cbx_tensor* t, int64_t n_seq, int64_t page, const char* what) {
    int rc = validate(t, what, "block_tables");
    if (rc) return rc;
    if (t->type != CBX_TYPE_I32 || t->ne[1] != n_seq || t->ne[2] != 1 || t->ne[3] != 1) {
        return bad(what, "block_tables must be I32 with ne = (max_pages, n_seq, 1, 1)");
    }
    if (t->ne[1] > 1 && (t->nb[1] % 4 != 0)) return bad(what, "block_tables rows must be 4-byte aligned");
    if (t->ne[0] >= k2G || t->ne[0] * page >= k2G) {
        return fail(CBX_ERR_UNSUPPORTED, what, "max_pages * page_size must be below 2^31");
    }
    return CBX_OK;
}

// K and V pages: one float type and one shape, (head_dim, page_size, n_head_kv, n_pages).
int check_cache(const cbx_tensor* k, const cbx_tensor* v, const char* what) {
    int rc;
    if ((rc = check_floats(k, what, "k_cache")) || (rc = check_floats(v, what, "v_cache"))) return rc;
    if (k->type != v->type) return fail(CBX_ERR_UNSUPPORTED, what, "k_cache and v_cache types differ");
    if (!same_shape(k, v)) return bad(what, "k_cache and v_cache shapes differ");
    const size_t es = type_size(k->type);
    for (const cbx_tensor* t : {k, v}) {
        for (int i = 1; i < 4; i++) {
            if (t->ne[i] > 1 && t->nb[i] % es) return bad(what, "cache strides must be whole elements");
        }
        if (reinterpret_cast<uintptr_t>(t->data) % es) return bad(what, "cache pages must be aligned to their elements");
    }
    if (k->ne[1] >= k2G || k->ne[3] >= k2G || k->ne[1] * k->ne[3] >= k2G) {
        return fail(CBX_ERR_UNSUPPORTED, what, "page_size * n_pages must be below 2^31");
    }
    return CBX_OK;
}

int overlap_error(const char* what, const char* out, const char* other) {
    return set_error(CBX_ERR_INVALID_ARG, std::string(what) + ": " + out + " must not overlap " + other);
}

// n outputs, each whole, apart from each other and from the m inputs.
int check_apart(const char* what, const cbx_tensor* const* outs, const char* const* names, int n,
                const cbx_tensor* const* ins, int m) {
    for (int i = 0; i < n; i++) {
        if (repeats(outs[i])) {
            return set_error(CBX_ERR_INVALID_ARG, std::string(what) + ": " + names[i] + " has a stride of 0");
        }
        for (int j = 0; j < m; j++) {
            if (ins[j] && meets(outs[i], ins[j])) return overlap_error(what, names[i], "an input");
        }
        for (int j = i + 1; j < n; j++) {
            if (meets(outs[i], outs[j])) return overlap_error(what, names[i], names[j]);
        }
    }
    return CBX_OK;
}

// Scratch of at least `need` bytes, apart from the call's n tensors.
int check_scratch(const char* what, const void* ws, size_t ws_bytes, size_t need, const cbx_tensor* const* ts, int n) {
    if (ws_bytes < need || (need && !ws)) {
        return set_error(CBX_ERR_INVALID_ARG, std::string(what) + ": ws needs " + std::to_string(need) + " bytes");
    }
    if (reinterpret_cast<uintptr_t>(ws) % 16) return bad(what, "ws must be 16-byte aligned");
    if (need == 0) return CBX_OK;
    cbx_tensor w{};
    w.data = const_cast<void*>(ws);
    w.type = CBX_TYPE_F32;
    const int64_t words = cdiv(static_cast<int64_t>(need), 4);
    for (int i = 0; i < 4; i++) {
        w.ne[i] = i == 0 ? words : 1;
        w.nb[i] = i == 0 ? 4 : 4 * static_cast<size_t>(words);
    }
    for (int i = 0; i < n; i++) {
        if (ts[i] && nelements(ts[i]) > 0 && bytes_overlap(&w, ts[i])) return overlap_error(what, "ws", "a tensor of the call");
    }
    return CBX_OK;
}

const int32_t* ints_of(const cbx_tensor* t) { return static_cast<const int32_t*>(t->data); }
int32_t* ints_of(cbx_tensor* t) { return static_cast<int32_t*>(t->data); }

}  // namespace
}  // namespace cbx

using namespace cbx;

extern "C" {

int cbx_paged_append(const cbx_tensor* n_past, const cbx_tensor* n_new, const cbx_tensor* free_pages,
                     const cbx_tensor* n_free, cbx_tensor* block_tables, int32_t page_size, cbx_tensor* seq_lens,
                     cbx_tensor* n_free_out, cbx_tensor* tok_start, cbx_tensor* slots, cbx_tensor* positions,
                     cbx_stream stream) {
    const char* what = "cbx_paged_append";
    clear_error();
    int rc;
    if ((rc = check_ints(n_past, -1, what, "n_past"))) return rc;
    const int64_t n = n_past->ne[0];
    if (page_size <= 0) return bad(what, "page_size must be > 0");
    if ((rc = check_ints(n_new, n, what, "n_new")) || (rc = check_ints(free_pages, -1, what, "free_pages")) ||
        (rc = check_ints(n_free, 1, what, "n_free")) || (rc = check_tables(block_tables, n, page_size, what)) ||
        (rc = check_ints(seq_lens, n, what, "seq_lens")) || (rc = check_ints(n_free_out, 1, what, "n_free_out")) ||
        (rc = check_ints(tok_start, n + 1, what, "tok_start")) || (rc = check_ints(slots, -1, what, "slots")) ||
        (rc = check_ints(positions, slots->ne[0], what, "positions"))) return rc;
    if (n > kPagedMaxSeq) return fail(CBX_ERR_UNSUPPORTED, what, "more than 4096 requests");
    if (free_pages->ne[0] >= k2G || slots->ne[0] >= k2G) return fail(CBX_ERR_UNSUPPORTED, what, "2^31 elements or more");
    const cbx_tensor* outs[] = {block_tables, seq_lens, n_free_out, tok_start, slots, positions};
    const char* names[] = {"block_tables", "seq_lens", "n_free_out", "tok_start", "slots", "positions"};
    const cbx_tensor* ins[] = {n_past, n_new, free_pages, n_free};
    if ((rc = check_apart(what, outs, names, 6, ins, 4))) return rc;
    DeviceState* st = current_state(&rc);
    if (!st) return rc;
    AppendArgs a{};
    a.n_past = ints_of(n_past);
    a.n_new = ints_of(n_new);
    a.free_pages = ints_of(free_pages);
    a.n_free = ints_of(n_free);
    a.seq_lens = ints_of(seq_lens);
    a.n_free_out = ints_of(n_free_out);
    a.tok_start = ints_of(tok_start);
    a.slots = ints_of(slots);
    a.positions = ints_of(positions);
    a.tables = static_cast<char*>(block_tables->data);
    a.tables_nb1 = static_cast<int64_t>(block_tables->nb[1]);
    a.n_seq = static_cast<int32_t>(n);
    a.max_pages = static_cast<int32_t>(block_tables->ne[0]);
    a.page = page_size;
    a.pool = static_cast<int32_t>(free_pages->ne[0]);
    a.n_slots = static_cast<int32_t>(slots->ne[0]);
    return launch_paged_append(a, st, reinterpret_cast<hipStream_t>(stream));
}

int cbx_paged_release(const cbx_tensor* seq_lens, const cbx_tensor* release, cbx_tensor* block_tables,
                      int32_t page_size, cbx_tensor* free_pages, const cbx_tensor* n_free, cbx_tensor* seq_lens_out,
                      cbx_tensor* n_free_out, cbx_stream stream) {
    const char* what = "cbx_paged_release";
    clear_error();
    int rc;
    if ((rc = check_ints(seq_lens, -1, what, "seq_lens"))) return rc;
    const int64_t n = seq_lens->ne[0];
    if (page_size <= 0) return bad(what, "page_size must be > 0");
    if ((rc = check_ints(release, n, what, "release")) || (rc = check_tables(block_tables, n, page_size, what)) ||
        (rc = check_ints(free_pages, -1, what, "free_pages")) || (rc = check_ints(n_free, 1, what, "n_free")) ||
        (rc = check_ints(seq_lens_out, n, what, "seq_lens_out")) ||
        (rc = check_ints(n_free_out, 1, what, "n_free_out"))) return rc;
    if (n > kPagedMaxSeq) return fail(CBX_ERR_UNSUPPORTED, what, "more than 4096 requests");
    if (free_pages->ne[0] >= k2G) return fail(CBX_ERR_UNSUPPORTED, what, "2^31 elements or more");
    const cbx_tensor* outs[] = {block_tables, free_pages, seq_lens_out, n_free_out};
    const char* names[] = {"block_tables", "free_pages", "seq_lens_out", "n_free_out"};
    const cbx_tensor* ins[] = {seq_lens, release, n_free};
    if ((rc = check_apart(what, outs, names, 4, ins, 3))) return rc;
    DeviceState* st = current_state(&rc);
    if (!st) return rc;
    ReleaseArgs a{};
    a.seq_lens = ints_of(seq_lens);
    a.release = ints_of(release);
    a.n_free = ints_of(n_free);
    a.free_pages = ints_of(free_pages);
    a.seq_lens_out = ints_of(seq_lens_out);
    a.n_free_out = ints_of(n_free_out);
    a.tables = static_cast<char*>(block_tables->data);
    a.tables_nb1 = static_cast<int64_t>(block_tables->nb[1]);
    a.n_seq = static_cast<int32_t>(n);
    a.max_pages = static_cast<int32_t>(block_tables->ne[0]);
    a.page = page_size;
    a.pool = static_cast<int32_t>(free_pages->ne[0]);
    return launch_paged_release(a, st, reinterpret_cast<hipStream_t>(stream));
}

// Shared by the calls over q, k and v rows: shapes and types of the rows,
// the cache and its slots.
static int check_kv_rows(const cbx_tensor* k, const cbx_tensor* v, const cbx_tensor* slots, const cbx_tensor* k_cache,
                         const cbx_tensor* v_cache, const char* what) {
    int rc;
    if ((rc = check_floats(k, what, "k")) || (rc = check_floats(v, what, "v"))) return rc;
    if (k->type != v->type) return fail(CBX_ERR_UNSUPPORTED, what, "k and v types differ");
    if (!same_shape(k, v) || k->ne[3] != 1) return bad(what, "k and v must both be (head_dim, n_head_kv, n_tok, 1)");
    if ((rc = check_cache(k_cache, v_cache, what))) return rc;
    if (k_cache->ne[0] != k->ne[0] || k_cache->ne[2] != k->ne[1]) {
        return bad(what, "the cache must be (head_dim, page_size, n_head_kv, n_pages) with k's head_dim and n_head_kv");
    }
    return check_ints(slots, k->ne[2], what, "slots");
}

static int check_row_count(const char* what, int64_t tok, int64_t heads, int64_t d) {
    if (tok >= kMostGroups || heads >= k2G || tok * heads >= k2G || d > 512) {
        return fail(CBX_ERR_UNSUPPORTED, what, "head_dim up to 512, fewer than 2^24 tokens and 2^31 rows");
    }
    return CBX_OK;
}

int cbx_paged_store(const cbx_tensor* k, const cbx_tensor* v, const cbx_tensor* slots, cbx_tensor* k_cache,
                    cbx_tensor* v_cache, cbx_stream stream) {
    const char* what = "cbx_paged_store";
    clear_error();
    int rc;
    if ((rc = check_kv_rows(k, v, slots, k_cache, v_cache, what))) return rc;
    if ((rc = check_row_count(what, k->ne[2], 2 * k->ne[1], k->ne[0]))) return rc;
    const cbx_tensor* outs[] = {k_cache, v_cache};
    const char* names[] = {"k_cache", "v_cache"};
    const cbx_tensor* ins[] = {k, v, slots};
    if ((rc = check_apart(what, outs, names, 2, ins, 3))) return rc;
    DeviceState* st = current_state(&rc);
    if (!st) return rc;
    if (nelements(k) == 0) return CBX_OK;
    QkCall c{};
    c.k = k;
    c.v = v;
    c.slots = slots;
    c.k_cache = k_cache;
    c.v_cache = v_cache;
    return launch_qk(c, st, reinterpret_cast<hipStream_t>(stream));
}

static int check_gain(const cbx_tensor* g, int64_t d, const char* what, const char* name) {
    if (!g) return CBX_OK;
    int rc = validate(g, what, name);
    if (rc) return rc;
    if (g->type != CBX_TYPE_F32 || g->ne[0] != d || g->ne[1] != 1 || g->ne[2] != 1 || g->ne[3] != 1) {
        return set_error(CBX_ERR_INVALID_ARG, std::string(what) + ": " + name + " must be F32 with head_dim elements");
    }
    return CBX_OK;
}

static int check_qk(const char* what, const cbx_tensor* q, const cbx_tensor* gq, const cbx_tensor* k,
                    const cbx_tensor* gk, float eps, const cbx_tensor* pos, const cbx_rope_cache* rope,
                    const cbx_tensor* yq) {
    int rc;
    if ((rc = check_floats(q, what, "q")) || (rc = check_floats(k, what, "k")) || (rc = check_floats(yq, what, "yq"))) return rc;
    if (q->type != k->type || yq->type != q->type) return fail(CBX_ERR_UNSUPPORTED, what, "q, k and yq types differ");
    const int64_t d = q->ne[0];
    if (q->ne[3] != 1 || k->ne[3] != 1 || k->ne[0] != d || k->ne[2] != q->ne[2]) {
        return bad(what, "q must be (head_dim, n_head, n_tok, 1) and k (head_dim, n_head_kv, n_tok, 1)");
    }
    if (!same_shape(q, yq)) return bad(what, "q and yq shapes differ");
    if (d % 8) return fail(CBX_ERR_UNSUPPORTED, what, "head_dim must be a multiple of 8");
    if (!(eps >= 0.0f) || std::isinf(eps)) return bad(what, "eps must be finite and >= 0");
    if ((rc = check_gain(gq, d, what, "gq")) || (rc = check_gain(gk, d, what, "gk")) ||
        (rc = check_ints(pos, q->ne[2], what, "pos"))) return rc;
    if (!rope) return bad(what, "rope is NULL");
    return CBX_OK;
}

static int check_rope(const char* what, const cbx_rope_cache* rope, int64_t d, const DeviceState* st) {
    const RopeTable t = rope_table(rope);
    if (t.device != st->device) return bad(what, "rope belongs to another device");
    if (t.p.n_dims > d) return bad(what, "n_dims > head_dim");
    if (t.p.n_dims % 8) return fail(CBX_ERR_UNSUPPORTED, what, "n_dims must be a multiple of 8");
    return CBX_OK;
}

int cbx_qk_norm_rope(const cbx_tensor* q, const cbx_tensor* gq, const cbx_tensor* k, const cbx_tensor* gk, float eps,
                     const cbx_tensor* pos, const cbx_rope_cache* rope, cbx_tensor* yq, cbx_tensor* yk,
                     cbx_stream stream) {
    const char* what = "cbx_qk_norm_rope";
    clear_error();
    int rc;
    if ((rc = check_qk(what, q, gq, k, gk, eps, pos, rope, yq)) || (rc = check_floats(yk, what, "yk"))) return rc;
    if (yk->type != k->type) return fail(CBX_ERR_UNSUPPORTED, what, "k and yk types differ");
    if (!same_shape(k, yk)) return bad(what, "k and yk shapes differ");
    if ((rc = check_row_count(what, q->ne[2], q->ne[1] + k->ne[1], q->ne[0]))) return rc;
    const cbx_tensor* outs[] = {yq, yk};
    const char* names[] = {"yq", "yk"};
    const cbx_tensor* ins_q[] = {k, gq, gk, pos, is_itself(yq, q) ? nullptr : q};
    const cbx_tensor* ins_k[] = {q, gq, gk, pos, is_itself(yk, k) ? nullptr : k};
    if ((rc = check_apart(what, outs, names, 2, nullptr, 0)) || (rc = check_apart(what, outs, names, 1, ins_q, 5)) ||
        (rc = check_apart(what, outs + 1, names + 1, 1, ins_k, 5))) return rc;
    DeviceState* st = current_state(&rc);
    if (!st || (rc = check_rope(what, rope, q->ne[0], st))) return rc;
    if (nelements(q) + nelements(k) == 0) return CBX_OK;
    QkCall c{};
    c.q = q;
    c.gq = gq;
    c.k = k;
    c.gk = gk;
    c.pos = pos;
    c.yq = yq;
    c.yk = yk;
    c.eps = eps;
    c.rope = rope_table(rope);
    c.norm = true;
    return launch_qk(c, st, reinterpret_cast<hipStream_t>(stream));
}

int cbx_qk_norm_rope_store(const cbx_tensor* q, const cbx_tensor* gq, const cbx_tensor* k, const cbx_tensor* gk,
                           const cbx_tensor* v, float eps, const cbx_tensor* pos, const cbx_rope_cache* rope,
                           const cbx_tensor* slots, cbx_tensor* yq, cbx_tensor* k_cache, cbx_tensor* v_cache,
                           cbx_stream stream) {
    const char* what = "cbx_qk_norm_rope_store";
    clear_error();
    int rc;
    if ((rc = check_qk(what, q, gq, k, gk, eps, pos, rope, yq)) ||
        (rc = check_kv_rows(k, v, slots, k_cache, v_cache, what)) ||
        (rc = check_row_count(what, q->ne[2], q->ne[1] + 2 * k->ne[1], q->ne[0]))) return rc;
    const cbx_tensor* outs[] = {k_cache, v_cache, yq};
    const char* names[] = {"k_cache", "v_cache", "yq"};
    const cbx_tensor* ins[] = {k, v, gq, gk, pos, slots, q};
    if ((rc = check_apart(what, outs, names, 3, ins, 6)) || (rc = check_apart(what, outs, names, 2, ins + 6, 1))) return rc;
    if (!is_itself(yq, q) && meets(yq, q)) return overlap_error(what, "yq", "an input");
    DeviceState* st = current_state(&rc);
    if (!st || (rc = check_rope(what, rope, q->ne[0], st))) return rc;
    if (nelements(q) + nelements(k) == 0) return CBX_OK;
    QkCall c{};
    c.q = q;
    c.gq = gq;
    c.k = k;
    c.gk = gk;
    c.v = v;
    c.pos = pos;
    c.slots = slots;
    c.yq = yq;
    c.k_cache = k_cache;
    c.v_cache = v_cache;
    c.eps = eps;
    c.rope = rope_table(rope);
    c.norm = true;
    return launch_qk(c, st, reinterpret_cast<hipStream_t>(stream));
}

static int check_attention(const char* what, const cbx_tensor* q, const cbx_tensor* k_cache, const cbx_tensor* tables) {
    int rc;
    if ((rc = check_floats(q, what, "q")) || (rc = check_floats(k_cache, what, "k_cache")) ||
        (rc = check_tables(tables, q->ne[2], k_cache->ne[1], what))) return rc;
    if (q->ne[3] != 1) return bad(what, "q must be (head_dim, n_head, n_seq, 1)");
    if (k_cache->ne[0] != q->ne[0]) return bad(what, "q and the cache differ in head_dim");
    const int64_t hkv = k_cache->ne[2];
    if (hkv == 0 ? q->ne[1] != 0 : q->ne[1] % hkv != 0) return bad(what, "n_head must be a multiple of n_head_kv");
    const int64_t keys = tables->ne[0] * k_cache->ne[1];
    if (q->ne[0] > 512 || q->ne[1] >= k2G || q->ne[2] >= k2G || q->ne[1] * q->ne[2] >= kMostGroups ||
        (keys / 32 + 1) * q->ne[1] * q->ne[2] >= (int64_t{1} << 40)) {
        return fail(CBX_ERR_UNSUPPORTED, what, "head_dim up to 512, n_head * n_seq below 2^24");
    }
    return CBX_OK;
}

int cbx_paged_attention_workspace(const cbx_tensor* q, const cbx_tensor* k_cache, const cbx_tensor* block_tables,
                                  size_t* bytes) {
    const char* what = "cbx_paged_attention_workspace";
    clear_error();
    int rc;
    if (!bytes) return bad(what, "bytes is NULL");
    *bytes = 0;
    if ((rc = check_attention(what, q, k_cache, block_tables))) return rc;
    DeviceState* st = current_state(&rc);
    if (!st) return rc;
    if (nelements(q) > 0) *bytes = paged_attention_workspace(q, k_cache, block_tables, st);
    return CBX_OK;
}

int cbx_paged_attention(const cbx_tensor* q, const cbx_tensor* k_cache, const cbx_tensor* v_cache,
                        const cbx_tensor* block_tables, const cbx_tensor* seq_lens, float scale, float softcap,
                        int32_t window, cbx_tensor* y, void* ws, size_t ws_bytes, cbx_stream stream) {
    const char* what = "cbx_paged_attention";
    clear_error();
    int rc;
    if ((rc = check_cache(k_cache, v_cache, what)) || (rc = check_attention(what, q, k_cache, block_tables)) ||
        (rc = check_ints(seq_lens, q->ne[2], what, "seq_lens")) || (rc = check_floats(y, what, "y"))) return rc;
    if (y->type != q->type) return fail(CBX_ERR_UNSUPPORTED, what, "q and y types differ");
    if (!same_shape(q, y)) return bad(what, "q and y shapes differ");
    if (!std::isfinite(scale)) return bad(what, "scale must be finite");
    if (!(softcap >= 0.0f) || std::isinf(softcap)) return bad(what, "softcap must be finite and >= 0");
    if (window < 0) return bad(what, "window must be >= 0");
    const cbx_tensor* outs[] = {y};
    const char* names[] = {"y"};
    const cbx_tensor* ins[] = {q, k_cache, v_cache, block_tables, seq_lens};
    if ((rc = check_apart(what, outs, names, 1, ins, 5))) return rc;
    DeviceState* st = current_state(&rc);
    if (!st) return rc;
    if (nelements(q) == 0) return CBX_OK;
    const size_t need = paged_attention_workspace(q, k_cache, block_tables, st);
    const cbx_tensor* all[] = {q, k_cache, v_cache, block_tables, seq_lens, y};
    if ((rc = check_scratch(what, ws, ws_bytes, need, all, 6))) return rc;
    PagedAttnCall c{q, k_cache, v_cache, block_tables, seq_lens, y, scale, softcap, window, ws};
    return launch_paged_attention(c, st, reinterpret_cast<hipStream_t>(stream));
}

static int check_logits(const char* what, const cbx_tensor* x, int64_t n_top) {
    int rc = check_floats(x, what, "logits");
    if (rc) return rc;
    if (x->ne[2] != 1 || x->ne[3] != 1) return bad(what, "logits must be (n_vocab, n_tok, 1, 1)");
    if (n_top < 0 || n_top > kLogProbTop) return fail(CBX_ERR_UNSUPPORTED, what, "n_top must be 0 to 64");
    if (x->ne[1] > 0 && (x->ne[0] == 0 || n_top > x->ne[0])) return bad(what, "n_vocab must be at least 1 and n_top");
    if (x->ne[0] >= k2G - 65536 || x->ne[1] >= kMostGroups) return fail(CBX_ERR_UNSUPPORTED, what, "n_vocab or n_tok too large");
    return CBX_OK;
}

int cbx_token_log_probs_workspace(const cbx_tensor* logits, int32_t n_top, size_t* bytes) {
    const char* what = "cbx_token_log_probs_workspace";
    clear_error();
    int rc;
    if (!bytes) return bad(what, "bytes is NULL");
    *bytes = 0;
    if ((rc = check_logits(what, logits, n_top))) return rc;
    DeviceState* st = current_state(&rc);
    if (!st) return rc;
    if (nelements(logits) > 0) *bytes = token_log_probs_workspace(logits, n_top, st);
    return CBX_OK;
}

int cbx_token_log_probs(const cbx_tensor* logits, const cbx_tensor* ids, float scale, cbx_tensor* logp,
                        cbx_tensor* entropy, cbx_tensor* top_ids, cbx_tensor* top_logp, void* ws, size_t ws_bytes,
                        cbx_stream stream) {
    const char* what = "cbx_token_log_probs";
    clear_error();
    int rc;
    if ((ids == nullptr) != (logp == nullptr)) return bad(what, "ids and logp go together");
    if ((top_ids == nullptr) != (top_logp == nullptr)) return bad(what, "top_ids and top_logp go together");
    if (!logp && !entropy && !top_ids) return bad(what, "no output is asked for");
    if (top_ids && (rc = validate(top_ids, what, "top_ids"))) return rc;
    const int64_t n_top = top_ids ? top_ids->ne[0] : 0;
    if ((rc = check_logits(what, logits, n_top))) return rc;
    const int64_t rows = logits->ne[1];
    auto row_out = [&](const cbx_tensor* t, const char* name, int type, int64_t ne0, int64_t ne1) -> int {
        int r = validate(t, what, name);
        if (r) return r;
        if (t->type != type || t->ne[0] != ne0 || t->ne[1] != ne1 || t->ne[2] != 1 || t->ne[3] != 1) {
            return set_error(CBX_ERR_INVALID_ARG, std::string(what) + ": " + name + " has a wrong shape or type");
        }
        return CBX_OK;
    };
    if (logp && ((rc = check_ints(ids, rows, what, "ids")) || (rc = row_out(logp, "logp", CBX_TYPE_F32, rows, 1)))) return rc;
    if (entropy && (rc = row_out(entropy, "entropy", CBX_TYPE_F32, rows, 1))) return rc;
    if (top_ids && ((rc = row_out(top_ids, "top_ids", CBX_TYPE_I32, n_top, rows)) ||
                    (rc = row_out(top_logp, "top_logp", CBX_TYPE_F32, n_top, rows)))) return rc;
    if (!(scale > 0.0f) || std::isinf(scale)) return bad(what, "scale must be finite and > 0");
    // twice the scale times log2(e) is a factor of the kernels
    if (scale >= 0x1p126f) return fail(CBX_ERR_UNSUPPORTED, what, "scale must be below 2^126");
    const cbx_tensor* outs[4];
    const char* names[4];
    int n = 0;
    auto out = [&](const cbx_tensor* t, const char* name) { if (t) { outs[n] = t; names[n++] = name; } };
    out(logp, "logp");
    out(entropy, "entropy");
    out(top_ids, "top_ids");
    out(top_logp, "top_logp");
    const cbx_tensor* ins[] = {logits, ids};
    if ((rc = check_apart(what, outs, names, n, ins, 2))) return rc;
    DeviceState* st = current_state(&rc);
    if (!st) return rc;
    if (rows == 0) return CBX_OK;
    const size_t need = token_log_probs_workspace(logits, static_cast<int>(n_top), st);
    const cbx_tensor* all[] = {logits, ids, logp, entropy, top_ids, top_logp};
    if ((rc = check_scratch(what, ws, ws_bytes, need, all, 6))) return rc;
    LogProbCall c{logits, ids, logp, entropy, n_top ? top_ids : nullptr, n_top ? top_logp : nullptr, scale,
                  static_cast<int>(n_top), ws};
    return launch_token_log_probs(c, st, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
