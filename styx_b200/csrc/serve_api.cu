// serve_api.cu -- the C entry points of include/styx_serve.h: validation,
// workspaces and launches; the kernels are in paged.cu, paged_attn.cu,
// sample.cu, paged_plan.cu, paged_rope.cu, paged_chunk.cu
// and paged_chunk_tc.cu.
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

// what styx_paged_append and its rotary form have in common; q_size: bytes of an element of q_out
int append_args(styx_ctx *ctx, const styx_paged_kv *kv, int n_tokens, int n_heads, const float *q, int64_t q_stride, const float *k,
                int64_t k_stride, const float *v, int64_t v_stride, const float *q_norm, const float *k_norm, float eps,
                const int32_t *pos, const int32_t *seq, const int32_t *row, const void *q_out, uint64_t q_size,
                styx::PagedAppendArgs &a, int &sms) {
    CHECK(styx::ctx_enter(ctx, &sms, &a.kv.err));
    CHECK(check_kv(kv, true, a.kv));
    NEED(n_tokens > 0 && n_heads >= 0 && static_cast<int64_t>(n_tokens) * (n_heads + kv->n_kv_heads) < (int64_t(1) << 31),
         "n_tokens %d, n_heads %d", n_tokens, n_heads);
    NEED(seq || n_tokens <= kv->n_seqs, "%d tokens without seq for %d sequences", n_tokens, kv->n_seqs);
    NEED(aligned(q_out, 16), "q_out must be 16-byte aligned");
    const int64_t qd = static_cast<int64_t>(n_heads) * kv->head_dim, kd = static_cast<int64_t>(kv->n_kv_heads) * kv->head_dim;
    NEED(k && v && pos && (n_heads == 0 || (q && q_out)), "null pointer");
    NEED((n_heads == 0 || q_stride >= qd) && k_stride >= kd && v_stride >= kd, "a token stride smaller than its heads");
    NEED((n_heads == 0 || (rows_ok(q, n_tokens, q_stride, qd, 4) && rows_ok(q_out, n_tokens, qd, qd, q_size))) &&
             rows_ok(k, n_tokens, k_stride, kd, 4) && rows_ok(v, n_tokens, v_stride, kd, 4),
         "q / k / v / q_out smaller than n_tokens");
    NEED(styx::range_ok(pos, n_tokens * 4ull) && styx::range_ok(seq, seq ? n_tokens * 4ull : 0) &&
             styx::range_ok(row, row ? n_tokens * 4ull : 0) && styx::range_ok(q_norm, q_norm ? kv->head_dim * 4ull : 0) &&
             styx::range_ok(k_norm, k_norm ? kv->head_dim * 4ull : 0),
         "pos / seq / row / norms too small");
    if (n_heads) {
        const Span to(q_out, n_tokens, qd, qd, q_size);
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
    a.pos = pos;
    a.seq = seq;
    a.row = row;
    a.n_tokens = n_tokens;
    a.n_heads = n_heads;
    return STYX_OK;
}

// attend_chunk's workspace: two partial results per worker, and what has to be joined
struct ChunkWs {
    uint64_t joins, total;
};
ChunkWs chunk_ws(const styx::PagedKv &kv, int sms) {
    ChunkWs w{};
    w.joins = a256(std::max(styx::chunk_mma_parts(kv, sms), kv.dtype == STYX_F32 ? 0 : styx::chunk_tc_parts(sms)));
    w.total = w.joins + a256(sms * 16ull);
    return w;
}

}  // namespace

extern "C" {

int styx_paged_append(styx_ctx *ctx, styx_stream stream, const styx_paged_kv *kv, int n_tokens, int n_heads,
                      const float *q, int64_t q_stride, const float *k, int64_t k_stride, const float *v,
                      int64_t v_stride, const float *q_norm, const float *k_norm, float eps, float freq_base,
                      const int32_t *pos, const int32_t *seq, const int32_t *row, float *q_out) {
    styx::PagedAppendArgs a{};
    int sms = 0;
    CHECK(append_args(ctx, kv, n_tokens, n_heads, q, q_stride, k, k_stride, v, v_stride, q_norm, k_norm, eps, pos, seq, row,
                      q_out, 4, a, sms));
    NEED(freq_base > 0.f, "freq_base must be positive");
    a.log2_base = -2.0 / static_cast<double>(kv->head_dim) * std::log2(static_cast<double>(freq_base));
    a.step = std::exp2(a.log2_base);
    a.q_out = q_out;
    CK(styx::launch_paged_append(a, sms, S(stream)));
    return STYX_OK;
}

int styx_paged_append_rope(styx_ctx *ctx, styx_stream stream, const styx_paged_kv *kv, int n_tokens, int n_heads,
                           const float *q, int64_t q_stride, const float *k, int64_t k_stride, const float *v,
                           int64_t v_stride, const float *q_norm, const float *k_norm, float eps,
                           const styx_rope *rope, const int32_t *pos, const int32_t *seq, const int32_t *row,
                           int q_type, void *q_out) {
    styx::PagedAppendArgs a{};
    int sms = 0;
    NEED(kv, "null styx_paged_kv");
    NEED(q_type == STYX_F32 || q_type == kv->dtype, "q_type %d: f32 (0) or the cache's type", q_type);
    CHECK(append_args(ctx, kv, n_tokens, n_heads, q, q_stride, k, k_stride, v, v_stride, q_norm, k_norm, eps, pos, seq, row,
                      q_out, q_type == STYX_F32 ? 4 : 2, a, sms));
    NEED(rope && rope->freq, "null rope");
    NEED(rope->n_dims > 0 && rope->n_dims % 2 == 0 && rope->n_dims <= kv->head_dim, "n_dims %d: even, <= head_dim %d", rope->n_dims,
         kv->head_dim);
    NEED(aligned(rope->freq, 8) && styx::range_ok(rope->freq, rope->n_dims * 4ull), "freq smaller than n_dims / 2");
    if (n_heads) {
        const int64_t qd = static_cast<int64_t>(n_heads) * kv->head_dim;
        NEED(Span(q_out, n_tokens, qd, qd, q_type == STYX_F32 ? 4 : 2).apart(Span(rope->freq, rope->n_dims * 4ull)), "q_out overlaps freq");
    }
    const styx::PagedRope r{rope->freq, rope->n_dims, rope->interleaved != 0, rope->magnitude};
    CK(styx::launch_paged_append_rope(a, r, q_out, q_type != STYX_F32, sms, S(stream)));
    return STYX_OK;
}

int styx_rope_freqs(const styx_rope_params *p, const float *factors, double *freq, float *magnitude) {
    NEED(p && freq && magnitude, "null pointer");
    NEED(p->n_dims > 0 && p->n_dims % 2 == 0 && p->n_dims <= 4096, "n_dims %d: even, <= 4096", p->n_dims);
    NEED(p->base > 1.0 && std::isfinite(p->base), "base %g: above 1", p->base);
    NEED(p->scaling == STYX_ROPE_NONE || p->scaling == STYX_ROPE_LINEAR || p->scaling == STYX_ROPE_YARN, "scaling %d", p->scaling);
    const bool yarn = p->scaling == STYX_ROPE_YARN;
    NEED(p->scaling == STYX_ROPE_NONE || (p->factor >= 1.0 && std::isfinite(p->factor)), "factor %g: at least 1", p->factor);
    NEED(!yarn || (p->orig_ctx > 0 && std::isfinite(p->orig_ctx) && p->beta_fast > 0 && p->beta_slow > 0 &&
                   std::isfinite(p->beta_fast) && std::isfinite(p->beta_slow)),
         "yarn: orig_ctx %g, beta_fast %g, beta_slow %g must be positive", p->orig_ctx, p->beta_fast, p->beta_slow);
    const int n = p->n_dims;
    for (int i = 0; factors && i < n / 2; i++) NEED(factors[i] > 0.f && std::isfinite(factors[i]), "factors[%d] must be positive", i);
    auto dim = [&](double turns) {
        return n * std::log(p->orig_ctx / (2 * 3.14159265358979323846 * turns)) / (2 * std::log(p->base));
    };
    const double lo = yarn ? std::max(0.0, std::floor(dim(p->beta_fast))) : 0.0;
    const double hi = yarn ? std::min(n - 1.0, std::ceil(dim(p->beta_slow))) : 0.0;
    for (int i = 0; i < n / 2; i++) {
        double f = std::pow(p->base, -2.0 * i / n);
        if (factors) f /= static_cast<double>(factors[i]);
        const double r = yarn ? std::min(1.0, std::max(0.0, (i - lo) / std::max(hi - lo, 0.001))) : 0.0;
        freq[i] = p->scaling == STYX_ROPE_LINEAR ? f / p->factor : yarn ? f * (1.0 - r) + f / p->factor * r : f;
    }
    *magnitude = yarn ? static_cast<float>(1.0 + 0.1 * std::log(p->factor)) : 1.f;
    return STYX_OK;
}

int styx_paged_plan(styx_ctx *ctx, styx_stream stream, const styx_page_table *pt, const int32_t *want, int n_tokens,
                    const int32_t *next_pos, int32_t *start, int32_t *seq, int32_t *row, int32_t *pos,
                    int32_t *lens_out, int32_t *held_out, int32_t *n_free_out, int32_t *next_pos_out) {
    styx::PagedPlanArgs a{};
    CHECK(styx::ctx_enter(ctx, nullptr, &a.err));
    NEED(pt, "null styx_page_table");
    NEED(pt->page_size > 0 && pt->page_size <= 4096 && (pt->page_size & (pt->page_size - 1)) == 0,
         "page_size %d: a power of two, <= 4096, needed", pt->page_size);
    NEED(pt->n_seqs > 0 && pt->n_seqs <= 65535, "n_seqs %d: 1 to 65535", pt->n_seqs);
    NEED(pt->n_pages > 0 && pt->max_pages > 0 && pt->table_stride >= pt->max_pages, "n_pages %d, max_pages %d, table_stride %d",
         pt->n_pages, pt->max_pages, pt->table_stride);
    NEED(static_cast<int64_t>(pt->max_pages) * pt->page_size < (int64_t(1) << 31) - 4096,
         "max_pages %d x page_size %d: fewer than 2^31 rows needed", pt->max_pages, pt->page_size);
    NEED(n_tokens > 0 && n_tokens <= (1 << 30), "n_tokens %d", n_tokens);
    NEED(pt->table && pt->free && pt->n_free && pt->lens && pt->held && want && start && seq && row && pos && lens_out &&
             held_out && n_free_out,
         "null pointer");
    NEED((next_pos != nullptr) == (next_pos_out != nullptr), "next_pos and next_pos_out: both or neither");
    const uint64_t n4 = pt->n_seqs * 4ull, t4 = n_tokens * 4ull;
    // outputs first; of the inputs the last four may each be the output of the same number
    const Span outs[10] = {{lens_out, n4}, {held_out, n4}, {n_free_out, 4}, {next_pos_out, n4}, {start, n4 + 4}, {seq, t4},
                           {row, t4}, {pos, t4}, {pt->free, pt->n_pages * 4ull},
                           Span(pt->table, pt->n_seqs, pt->table_stride, pt->max_pages, 4)};
    const Span ins[5] = {{pt->lens, n4}, {pt->held, n4}, {pt->n_free, 4}, {next_pos, n4}, {want, n4}};
    for (const Span &o : outs) NEED(styx::range_ok(o.begin, static_cast<uint64_t>(o.end - o.begin)), "an output smaller than needed");
    for (const Span &i : ins) NEED(styx::range_ok(i.begin, static_cast<uint64_t>(i.end - i.begin)), "an input smaller than n_seqs");
    for (int o = 0; o < 10; o++) {
        for (int i = 0; i < 5; i++)
            NEED(outs[o].apart(ins[i]) || (o == i && o < 4 && outs[o].begin == ins[i].begin), "an output overlaps an input that is not its own");
        for (int p = 0; p < o; p++) NEED(outs[o].apart(outs[p]), "outputs overlap");
    }
    a.table = pt->table;
    a.free = pt->free;
    a.want = want;
    a.lens = pt->lens;
    a.held = pt->held;
    a.n_free = pt->n_free;
    a.next_pos = next_pos;
    a.start = start;
    a.seq = seq;
    a.row = row;
    a.pos = pos;
    a.lens_out = lens_out;
    a.held_out = held_out;
    a.n_free_out = n_free_out;
    a.next_pos_out = next_pos_out;
    a.table_stride = pt->table_stride;
    a.n_seqs = pt->n_seqs;
    a.max_pages = pt->max_pages;
    a.page_shift = __builtin_ctz(static_cast<unsigned>(pt->page_size));
    a.n_pages = pt->n_pages;
    a.n_tokens = n_tokens;
    CK(styx::launch_paged_plan(a, S(stream)));
    return STYX_OK;
}

int styx_paged_chunk_workspace_bytes(styx_ctx *ctx, const styx_paged_kv *kv, int n_heads, int q_type, uint64_t *out) {
    styx::PagedKv o{};
    int sms = 0;
    CHECK(styx::ctx_enter(ctx, &sms, nullptr));
    CHECK(check_kv(kv, false, o));
    NEED(out && n_heads > 0 && n_heads % kv->n_kv_heads == 0, "n_heads %d must be a multiple of n_kv_heads %d", n_heads,
         kv->n_kv_heads);
    NEED(q_type == STYX_F32 || q_type == kv->dtype, "q_type %d: f32 (0) or the cache's type", q_type);
    *out = chunk_ws(o, sms).total;
    return STYX_OK;
}

int styx_paged_attend_chunk(styx_ctx *ctx, styx_stream stream, const styx_paged_kv *kv, int n_tokens, int n_heads,
                            int q_type, const void *q, int64_t q_stride, const int32_t *start, float scale, int window,
                            void *out, float *lse, void *workspace, uint64_t workspace_bytes) {
    styx::PagedChunkArgs a{};
    int sms = 0;
    CHECK(styx::ctx_enter(ctx, &sms, &a.kv.err));
    CHECK(check_kv(kv, true, a.kv));
    NEED(n_heads > 0 && n_heads <= 65535 && n_heads % kv->n_kv_heads == 0, "n_heads %d must be a multiple of n_kv_heads %d",
         n_heads, kv->n_kv_heads);
    NEED(n_tokens > 0 && static_cast<int64_t>(n_tokens) * n_heads < (int64_t(1) << 31), "n_tokens %d, n_heads %d", n_tokens, n_heads);
    NEED(q_type == STYX_F32 || q_type == kv->dtype, "q_type %d: f32 (0) or the cache's type", q_type);
    const uint64_t size = q_type == STYX_F32 ? 4 : 2;
    const int64_t qd = static_cast<int64_t>(n_heads) * kv->head_dim;
    NEED(q && out && start && workspace, "null pointer");
    NEED(aligned(q, 16) && aligned(out, 16) && aligned(workspace, 256),
         "q and out must be 16-byte aligned, the workspace 256-byte");
    NEED(q_stride >= qd && q_stride * size % 16 == 0, "q_stride %lld: at least n_heads x head_dim, 16-byte multiples",
         static_cast<long long>(q_stride));
    NEED(window >= 0, "window %d", window);
    NEED(std::isfinite(scale), "scale must be finite");
    const Span outs[3] = {Span(out, n_tokens, qd, qd, size), Span(lse, lse ? static_cast<uint64_t>(n_tokens) * n_heads * 4 : 0),
                          Span(workspace, workspace_bytes)};
    const Span ins[2] = {Span(q, n_tokens, q_stride, qd, size), Span(start, kv->n_seqs * 4ull + 4)};
    NEED(rows_ok(q, n_tokens, q_stride, qd, size) && rows_ok(out, n_tokens, qd, qd, size) &&
             styx::range_ok(lse, lse ? static_cast<uint64_t>(n_tokens) * n_heads * 4 : 0) && styx::range_ok(start, kv->n_seqs * 4ull + 4),
         "q / out / lse / start smaller than n_tokens, n_seqs + 1");
    const ChunkWs w = chunk_ws(a.kv, sms);
    NEED(workspace_bytes >= w.total && styx::range_ok(workspace, w.total), "workspace: %llu bytes needed",
         static_cast<unsigned long long>(w.total));
    for (int o = 0; o < 3; o++) {
        NEED(outs[o].apart(ins[0]) && outs[o].apart(ins[1]) && clear_of_lengths(kv, outs[o]),
             "an output or the workspace overlaps q, start, lens or the table");
        for (int p = 0; p < o; p++) NEED(outs[o].apart(outs[p]), "outputs or the workspace overlap each other");
    }
    char *ws = static_cast<char *>(workspace);
    a.q = q;
    a.out = out;
    a.lse = lse;
    a.start = start;
    a.q_stride = q_stride;
    a.scale = scale;
    a.window = window;
    a.n_tokens = n_tokens;
    a.n_heads = n_heads;
    a.gqa = n_heads / kv->n_kv_heads;
    a.q16 = q_type != STYX_F32;
    a.part = reinterpret_cast<float *>(ws);
    a.joins = ws + w.joins;
    if (styx::chunk_on_tc(a)) CK(styx::launch_chunk_tc(a, sms, S(stream)));
    else CK(styx::launch_chunk_mma(a, sms, S(stream)));
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
