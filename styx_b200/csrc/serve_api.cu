// serve_api.cu -- the C entry points of include/styx_serve.h: validation,
// workspaces and launches; the kernels are in paged.cu, paged_attn.cu and
// sample.cu.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include <cuda_runtime.h>

#include "../../include/styx_serve.h"
#include "kernels.h"

namespace {

int fail(int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return styx::set_error(code, buf);
}

#define CK(call)                                                                                   \
    do {                                                                                           \
        cudaError_t e_ = (call);                                                                   \
        if (e_ != cudaSuccess) return fail(STYX_ECUDA, "%s: %s", #call, cudaGetErrorString(e_));   \
    } while (0)

#define NEED(cond, ...)                                                                            \
    do {                                                                                           \
        if (!(cond)) return fail(STYX_EINVAL, __VA_ARGS__);                                        \
    } while (0)

inline cudaStream_t S(styx_stream s) { return static_cast<cudaStream_t>(s); }
bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
uint64_t a256(uint64_t v) { return (v + 255) & ~uint64_t(255); }

// n elements of `size` bytes each, `rows` times, `stride` elements apart
bool rows_ok(const void *p, uint64_t rows, uint64_t stride, uint64_t n, uint64_t size) {
    return rows == 0 || styx::range_ok(p, ((rows - 1) * stride + n) * size);
}

// the bytes of such rows, [begin, end), for checks of overlaps
struct Span {
    const char *begin, *end;
    Span(const void *p, uint64_t bytes) : begin(static_cast<const char *>(p)), end(begin + (p ? bytes : 0)) {}
    Span(const void *p, uint64_t rows, uint64_t stride, uint64_t n, uint64_t size) : Span(p, ((rows - 1) * stride + n) * size) {}
    bool apart(const Span &o) const { return end <= o.begin || o.end <= begin; }
};

int check_kv(const styx_paged_kv *kv, bool with_buffers, styx::PagedKv &o) {
    NEED(kv, "null styx_paged_kv");
    NEED(kv->dtype == STYX_F32 || kv->dtype == STYX_F16 || kv->dtype == STYX_BF16,
         "cache type %d: f32 (0), f16 (1) or bf16 (30)", kv->dtype);
    const int size = kv->dtype == STYX_F32 ? 4 : 2;
    NEED(kv->head_dim > 0 && kv->head_dim <= 256 && kv->head_dim * size % 16 == 0,
         "head_dim %d: rows of 16 bytes' multiples, <= 256 elements, needed", kv->head_dim);
    NEED(kv->page_size > 0 && kv->page_size <= 4096 && (kv->page_size & (kv->page_size - 1)) == 0,
         "page_size %d: a power of two, <= 4096, needed", kv->page_size);
    NEED(kv->n_kv_heads > 0 && kv->n_kv_heads <= 1024, "n_kv_heads %d", kv->n_kv_heads);
    NEED(kv->n_seqs > 0 && kv->n_seqs <= 65535, "n_seqs %d: 1 to 65535", kv->n_seqs);
    NEED(kv->n_pages > 0 && kv->max_pages > 0 && kv->table_stride >= kv->max_pages, "n_pages %d, max_pages %d, table_stride %d",
         kv->n_pages, kv->max_pages, kv->table_stride);
    NEED(static_cast<int64_t>(kv->max_pages) * kv->page_size < (int64_t(1) << 31) - 4096,
         "max_pages %d x page_size %d: fewer than 2^31 rows needed", kv->max_pages, kv->page_size);
    const int64_t page = static_cast<int64_t>(kv->n_kv_heads) * kv->page_size * kv->head_dim;
    NEED(page < (int64_t(1) << 31), "a page of %lld elements", static_cast<long long>(page));
    NEED(kv->page_stride >= page && kv->page_stride * size % 16 == 0,
         "page_stride %lld: at least n_kv_heads x page_size x head_dim, 16-byte multiples", static_cast<long long>(kv->page_stride));
    if (with_buffers) {
        NEED(kv->k && kv->v && kv->table && kv->lens, "null cache, table or lens");
        NEED(aligned(kv->k, 16) && aligned(kv->v, 16), "k and v must be 16-byte aligned");
        NEED(rows_ok(kv->k, kv->n_pages, kv->page_stride, page, size) && rows_ok(kv->v, kv->n_pages, kv->page_stride, page, size),
             "k / v smaller than n_pages pages");
        NEED(rows_ok(kv->table, kv->n_seqs, kv->table_stride, kv->max_pages, 4) && styx::range_ok(kv->lens, kv->n_seqs * 4ull),
             "table / lens smaller than n_seqs rows");
    }
    o.k = kv->k;
    o.v = kv->v;
    o.page_stride = kv->page_stride;
    o.table = kv->table;
    o.lens = kv->lens;
    o.dtype = kv->dtype;
    o.n_pages = kv->n_pages;
    o.page_shift = __builtin_ctz(static_cast<unsigned>(kv->page_size));
    o.n_kv = kv->n_kv_heads;
    o.hd = kv->head_dim;
    o.n_seqs = kv->n_seqs;
    o.max_pages = kv->max_pages;
    o.table_stride = kv->table_stride;
    return STYX_OK;
}
// warps find their work from lens and the table, each for itself: one that changed in between would part them at a barrier
bool clear_of_lengths(const styx_paged_kv *kv, const Span &o) {
    return o.apart(Span(kv->lens, kv->n_seqs * 4ull)) &&
           o.apart(Span(kv->table, kv->n_seqs, kv->table_stride, kv->max_pages, 4));
}
uint64_t max_rows(const styx_paged_kv *kv) { return static_cast<uint64_t>(kv->max_pages) * kv->page_size; }

// attend's workspace: the finished portions of every (sequence, kv head,
// group of 8 or more heads), two partial results per worker; with weights,
// every head's maximum and sum, and every row's scores
struct AttendWs {
    uint64_t cnt, part, ml, scores, total;
};
// the tensor cores take 16-bit rows of up to 128 elements in pages of 16 rows
// or more (a warp's 16 rows then lie together; its ring, and q and O in its
// registers, are laid out for rows of up to 256 bytes); everything else runs on
// the FMA units.  Where both could (32 / 4 heads of 128): 37 rows 6.4 us against
// 9.7, one sequence of 131071 f16 rows 50 against 117, 32 ragged bf16 ones 34
// against 75, 64 of 64 / 4 heads 117 against 448
bool on_tensor_cores(const styx_paged_kv *kv) {
    return kv->dtype != STYX_F32 && kv->head_dim <= 128 && kv->page_size >= 16;
}
AttendWs attend_ws(const styx_paged_kv *kv, int n_heads, bool with_acc, int sms) {
    AttendWs w{};
    uint64_t o = 0;
    const uint64_t heads = static_cast<uint64_t>(kv->n_seqs) * n_heads;
    w.cnt = o;
    o += a256(heads * 4);
    w.part = o;
    o += a256(on_tensor_cores(kv) ? styx::attend_mma_parts(n_heads / kv->n_kv_heads, sms) : styx::attend_fma_parts(sms));
    w.ml = o;
    if (with_acc) o += a256(heads * 8);
    w.scores = o;
    if (with_acc) o += a256(heads * max_rows(kv) * 4);
    w.total = o;
    return w;
}

// evict's workspace: the moves' sources, places and number; the keys of long lines.  A line moves no more rows than
// the budget, nor than it has (room for those in whole slices of 4096)
struct EvictWs {
    uint64_t places, moves, keys, total;
};
EvictWs evict_ws(const styx_paged_kv *kv, int budget) {
    EvictWs w{};
    const uint64_t lines = static_cast<uint64_t>(kv->n_seqs) * kv->n_kv_heads;
    w.places = a256(lines * std::min<uint64_t>(static_cast<uint64_t>(budget), (max_rows(kv) + 4095) & ~uint64_t(4095)) * 4);
    w.moves = w.places * 2;
    w.keys = w.moves + a256(lines * 4);
    w.total = w.keys + (styx::evict_staged(static_cast<long long>(max_rows(kv))) ? 0 : a256(lines * max_rows(kv) * 4));
    return w;
}

#define CHECK(call)                                                                                \
    do {                                                                                           \
        int rc_ = (call);                                                                          \
        if (rc_) return rc_;                                                                       \
    } while (0)

}  // namespace

extern "C" {

int styx_paged_append(styx_ctx *ctx, styx_stream stream, const styx_paged_kv *kv, int n_tokens, int n_heads,
                      const float *q, int64_t q_stride, const float *k, int64_t k_stride, const float *v,
                      int64_t v_stride, const float *q_norm, const float *k_norm, float eps, float freq_base,
                      const int32_t *pos, const int32_t *seq, const int32_t *row, float *q_out) {
    styx::PagedAppendArgs a{};
    int sms = 0;
    CHECK(styx::ctx_enter(ctx, &sms, &a.kv.err));
    CHECK(check_kv(kv, true, a.kv));
    NEED(n_tokens > 0 && n_heads >= 0 && static_cast<int64_t>(n_tokens) * (n_heads + kv->n_kv_heads) < (int64_t(1) << 31),
         "n_tokens %d, n_heads %d", n_tokens, n_heads);
    NEED(seq || n_tokens <= kv->n_seqs, "%d tokens without seq for %d sequences", n_tokens, kv->n_seqs);
    NEED(aligned(q_out, 16), "q_out must be 16-byte aligned");
    const int64_t qd = static_cast<int64_t>(n_heads) * kv->head_dim, kd = static_cast<int64_t>(kv->n_kv_heads) * kv->head_dim;
    NEED(k && v && pos && (n_heads == 0 || (q && q_out)), "null pointer");
    NEED((n_heads == 0 || q_stride >= qd) && k_stride >= kd && v_stride >= kd, "a token stride smaller than its heads");
    NEED(freq_base > 0.f, "freq_base must be positive");
    NEED((n_heads == 0 || (rows_ok(q, n_tokens, q_stride, qd, 4) && rows_ok(q_out, n_tokens, qd, qd, 4))) &&
             rows_ok(k, n_tokens, k_stride, kd, 4) && rows_ok(v, n_tokens, v_stride, kd, 4),
         "q / k / v / q_out smaller than n_tokens");
    NEED(styx::range_ok(pos, n_tokens * 4ull) && styx::range_ok(seq, seq ? n_tokens * 4ull : 0) &&
             styx::range_ok(row, row ? n_tokens * 4ull : 0) && styx::range_ok(q_norm, q_norm ? kv->head_dim * 4ull : 0) &&
             styx::range_ok(k_norm, k_norm ? kv->head_dim * 4ull : 0),
         "pos / seq / row / norms too small");
    if (n_heads) {
        const Span to(q_out, n_tokens, qd, qd, 4);
        NEED(to.apart(Span(q, n_tokens, q_stride, qd, 4)), "q_out overlaps q");
        NEED(to.apart(Span(k, n_tokens, k_stride, kd, 4)) && to.apart(Span(v, n_tokens, v_stride, kd, 4)), "q_out overlaps k or v");
    }
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    a.log2_base = -2.0 / static_cast<double>(kv->head_dim) * std::log2(static_cast<double>(freq_base));
    a.step = std::exp2(a.log2_base);
    a.pos = pos;
    a.seq = seq;
    a.row = row;
    a.q_out = q_out;
    a.n_tokens = n_tokens;
    a.n_heads = n_heads;
    CK(styx::launch_paged_append(a, sms, S(stream)));
    return STYX_OK;
}

int styx_paged_attend_workspace_bytes(styx_ctx *ctx, const styx_paged_kv *kv, int n_heads, int with_acc, uint64_t *out) {
    styx::PagedKv o{};
    int sms = 0;
    CHECK(styx::ctx_enter(ctx, &sms, nullptr));
    CHECK(check_kv(kv, false, o));
    NEED(out && n_heads > 0 && n_heads % kv->n_kv_heads == 0, "n_heads %d must be a multiple of n_kv_heads %d", n_heads,
         kv->n_kv_heads);
    *out = attend_ws(kv, n_heads, with_acc != 0, sms).total;
    return STYX_OK;
}

int styx_paged_attend_workspace_init(styx_ctx *ctx, styx_stream stream, void *workspace, uint64_t workspace_bytes) {
    CHECK(styx::ctx_enter(ctx, nullptr, nullptr));
    NEED(workspace && styx::range_ok(workspace, workspace_bytes), "bad workspace");
    CK(cudaMemsetAsync(workspace, 0, workspace_bytes, S(stream)));
    return STYX_OK;
}

int styx_paged_attend(styx_ctx *ctx, styx_stream stream, const styx_paged_kv *kv, int n_heads, const float *q,
                      float scale, int window, float *out, float *lse, const float *acc, float *acc_out,
                      int64_t acc_stride, void *workspace, uint64_t workspace_bytes) {
    styx::PagedAttendArgs a{};
    int sms = 0;
    CHECK(styx::ctx_enter(ctx, &sms, &a.kv.err));
    CHECK(check_kv(kv, true, a.kv));
    NEED(n_heads > 0 && n_heads <= 65535 && n_heads % kv->n_kv_heads == 0, "n_heads %d must be a multiple of n_kv_heads %d",
         n_heads, kv->n_kv_heads);
    NEED(q && out && workspace, "null pointer");
    NEED(aligned(q, 16) && aligned(out, 16) && aligned(workspace, 256),
         "q and out must be 16-byte aligned, the workspace 256-byte");
    NEED(window >= 0, "window %d", window);
    NEED(std::isfinite(scale), "scale must be finite");
    NEED(!acc_out || acc, "acc_out without acc");
    NEED(!acc_out || acc_stride >= static_cast<int64_t>(max_rows(kv)), "acc_stride %lld: at least max_pages x page_size",
         static_cast<long long>(acc_stride));
    const uint64_t heads = static_cast<uint64_t>(kv->n_seqs) * n_heads;
    NEED(styx::range_ok(q, heads * kv->head_dim * 4) && styx::range_ok(out, heads * kv->head_dim * 4) &&
             styx::range_ok(lse, lse ? heads * 4 : 0),
         "q / out / lse smaller than n_seqs x n_heads");
    NEED(out == q || Span(q, heads * kv->head_dim * 4).apart(Span(out, heads * kv->head_dim * 4)), "out overlaps q in part");
    if (acc_out) {
        const uint64_t lines = static_cast<uint64_t>(kv->n_seqs) * kv->n_kv_heads * acc_stride * 4;
        NEED(kv->n_seqs * static_cast<int64_t>(kv->n_kv_heads) <= 65535, "accumulation: n_seqs x n_kv_heads <= 65535");   // lines x row blocks: a grid's x
        NEED(styx::range_ok(acc, lines) && styx::range_ok(acc_out, lines), "acc / acc_out smaller than n_seqs x n_kv_heads lines");
        NEED(acc == acc_out || Span(acc, lines).apart(Span(acc_out, lines)), "acc_out overlaps acc in part");
    }
    const AttendWs w = attend_ws(kv, n_heads, acc_out != nullptr, sms);
    NEED(workspace_bytes >= w.total && styx::range_ok(workspace, w.total), "workspace: %llu bytes needed",
         static_cast<unsigned long long>(w.total));
    NEED(clear_of_lengths(kv, Span(out, heads * kv->head_dim * 4)) && clear_of_lengths(kv, Span(lse, heads * 4)) &&
             clear_of_lengths(kv, Span(acc_out, static_cast<uint64_t>(kv->n_seqs) * kv->n_kv_heads * acc_stride * 4)) &&
             clear_of_lengths(kv, Span(workspace, w.total)),
         "an output or the workspace overlaps lens or the table");
    char *ws = static_cast<char *>(workspace);
    a.q = q;
    a.out = out;
    a.lse = lse;
    a.acc = acc;
    a.acc_out = acc_out;
    a.acc_stride = acc_stride;
    a.scale = scale;
    a.window = window;
    a.n_heads = n_heads;
    a.gqa = n_heads / kv->n_kv_heads;
    a.ml = reinterpret_cast<float *>(ws + w.ml);
    a.scores = reinterpret_cast<float *>(ws + w.scores);
    a.part = reinterpret_cast<float *>(ws + w.part);
    a.cnt = reinterpret_cast<unsigned *>(ws + w.cnt);
    if (on_tensor_cores(kv))
        CK(styx::launch_attend_mma(a, sms, S(stream)));
    else
        CK(styx::launch_attend_fma(a, sms, S(stream)));
    return STYX_OK;
}

int styx_paged_evict_workspace_bytes(const styx_paged_kv *kv, int budget, uint64_t *out) {
    styx::PagedKv o{};
    CHECK(check_kv(kv, false, o));
    NEED(out && budget > 0, "budget %d", budget);
    *out = evict_ws(kv, budget).total;
    return STYX_OK;
}

int styx_paged_evict(styx_ctx *ctx, styx_stream stream, const styx_paged_kv *kv, const float *acc, const int32_t *pos,
                     const int32_t *next_pos, int64_t stride, int budget, int n_recent, int n_sink, float *acc_out,
                     int32_t *pos_out, int32_t *lens_out, void *workspace, uint64_t workspace_bytes) {
    styx::PagedEvictArgs a{};
    int sms = 0;
    CHECK(styx::ctx_enter(ctx, &sms, &a.kv.err));
    CHECK(check_kv(kv, true, a.kv));
    NEED(acc && pos && next_pos && acc_out && pos_out && lens_out && workspace, "null pointer");
    NEED(budget > 0 && n_recent >= 0 && n_sink >= 0 && static_cast<int64_t>(n_recent) + n_sink <= budget,
         "budget %d, n_recent %d, n_sink %d: n_recent + n_sink <= budget needed", budget, n_recent, n_sink);
    NEED(stride >= static_cast<int64_t>(max_rows(kv)), "stride %lld: at least max_pages x page_size",
         static_cast<long long>(stride));
    const int64_t heads = static_cast<int64_t>(kv->n_seqs) * kv->n_kv_heads;
    const uint64_t lines = static_cast<uint64_t>(heads) * stride * 4;
    NEED(styx::range_ok(acc, lines) && styx::range_ok(pos, lines) && styx::range_ok(acc_out, lines) &&
             styx::range_ok(pos_out, lines) && styx::range_ok(next_pos, kv->n_seqs * 4ull) &&
             styx::range_ok(lens_out, kv->n_seqs * 4ull),
         "weights / positions / lengths smaller than n_seqs x n_kv_heads lines");
    const Span outs[3] = {Span(acc_out, lines), Span(pos_out, lines), Span(lens_out, kv->n_seqs * 4ull)};
    const Span ins[4] = {Span(acc, lines), Span(pos, lines), Span(next_pos, kv->n_seqs * 4ull), Span(kv->lens, kv->n_seqs * 4ull)};
    for (int o = 0; o < 3; o++) {
        for (const Span &i : ins) NEED(outs[o].apart(i), "acc_out, pos_out and lens_out must be other arrays than the inputs");
        for (int p = 0; p < o; p++) NEED(outs[o].apart(outs[p]), "acc_out, pos_out and lens_out must be other arrays than each other");
    }
    const EvictWs w = evict_ws(kv, budget);
    NEED(workspace_bytes >= w.total && aligned(workspace, 256) && styx::range_ok(workspace, w.total),
         "workspace: %llu bytes, 256-byte aligned, needed", static_cast<unsigned long long>(w.total));
    NEED(clear_of_lengths(kv, outs[0]) && clear_of_lengths(kv, outs[1]) && clear_of_lengths(kv, outs[2]) &&
             clear_of_lengths(kv, Span(workspace, w.total)),
         "an output or the workspace overlaps lens or the table");
    char *ws = static_cast<char *>(workspace);
    a.acc = acc;
    a.pos = pos;
    a.next_pos = next_pos;
    a.stride = stride;
    a.budget = static_cast<int>(std::min<uint64_t>(static_cast<uint64_t>(budget), max_rows(kv)));
    a.n_recent = n_recent;
    a.n_sink = n_sink;
    a.acc_out = acc_out;
    a.pos_out = pos_out;
    a.lens_out = lens_out;
    a.src = reinterpret_cast<int32_t *>(ws);
    a.places = reinterpret_cast<int32_t *>(ws + w.places);
    a.moves = reinterpret_cast<int32_t *>(ws + w.moves);
    a.keys = reinterpret_cast<uint32_t *>(ws + w.keys);
    CK(styx::launch_paged_evict(a, sms, S(stream)));
    return STYX_OK;
}

int styx_sample(styx_ctx *ctx, styx_stream stream, const float *logits, int64_t row_stride, int n_rows, int n_vocab,
                const float *u, const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                int32_t *token, float *logprob) {
    styx::SampleArgs a{};
    CHECK(styx::ctx_enter(ctx, nullptr, &a.err));
    NEED(logits && u && token, "null pointer");
    NEED(n_rows > 0 && n_vocab > 0 && n_vocab <= (1 << 22) && row_stride >= n_vocab, "n_rows %d, n_vocab %d, row_stride %lld",
         n_rows, n_vocab, static_cast<long long>(row_stride));
    const uint64_t n4 = static_cast<uint64_t>(n_rows) * 4;
    auto opt = [&](const void *p) { return styx::range_ok(p, p ? n4 : 0); };
    NEED(rows_ok(logits, n_rows, row_stride, n_vocab, 4) && opt(u) && opt(temperature) && opt(top_k) && opt(top_p) &&
             opt(min_p) && opt(token) && opt(logprob),
         "logits or a per-row array smaller than n_rows");
    // rows are ordered by all rows' settings: one that a finished row overwrites could order them differently for another
    // (each row's u is read by that row alone, before its outputs are written)
    const Span ins[5] = {Span(logits, n_rows, row_stride, n_vocab, 4), Span(temperature, n4), Span(top_k, n4), Span(top_p, n4),
                         Span(min_p, n4)};
    const Span outs[2] = {Span(token, n4), Span(logprob, n4)}, us(u, n4);
    for (const Span &o : outs) {
        for (const Span &i : ins) NEED(o.apart(i), "token or logprob overlaps an input");
        NEED(o.begin == us.begin || o.apart(us), "token or logprob overlaps u in part");
    }
    NEED(outs[0].apart(outs[1]), "token overlaps logprob");
    a.logits = logits;
    a.row_stride = row_stride;
    a.n_rows = n_rows;
    a.n_vocab = n_vocab;
    a.u = u;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.token = token;
    a.logprob = logprob;
    CK(styx::launch_sample(a, S(stream)));
    return STYX_OK;
}

}  // extern "C"
