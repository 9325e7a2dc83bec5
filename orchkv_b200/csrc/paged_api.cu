// paged_api.cu — the paged operators' C entries: argument checks, the choice
// of kernels, workspace layout.
#include <algorithm>

#include "kernels.h"
#include "paged.cuh"
#include "paged_overlap.h"

using namespace okv;

namespace {

constexpr uint32_t kMaxHeadDim = 256;
constexpr uint64_t kMaxTokens = 1ull << 30;      // of one sequence's table

bool aligned(const void *p, int64_t s0, int64_t s1, size_t e)
{
    return p && (uintptr_t)p % 16 == 0 && s0 >= 0 && s1 >= 0 && (s0 * (int64_t)e) % 16 == 0 &&
           (s1 * (int64_t)e) % 16 == 0;
}

bool rows_ok(const orchkv_rows_t &r, size_t e) { return aligned(r.p, r.row_stride, r.head_stride, e); }

bool shapes_ok(const orchkv_pages_t *p, const orchkv_batch_t *b, bool need_v)
{
    if (!p || !b) return false;
    if (p->dtype != DTYPE_FP16 && p->dtype != DTYPE_BF16 && p->dtype != DTYPE_FP32) return false;
    const size_t e = dtype_size((DataType)p->dtype);
    if (p->d_head == 0 || p->d_head > kMaxHeadDim || p->d_head * e % 16) return false;
    if (p->page_tokens == 0 || p->n_kv_heads == 0 || p->n_kv_heads > 65535 || p->n_pages == 0 ||
        p->n_pages > 0x7FFFFFFFu)
        return false;
    if (!aligned(p->k, p->page_stride, p->head_stride, e) || p->token_stride < 0 ||
        (p->token_stride * (int64_t)e) % 16)
        return false;
    if (need_v && !aligned(p->v, 0, 0, e)) return false;
    if (b->n_seqs && (!b->table || !b->lens || !b->starts)) return false;
    if (b->table_width == 0) return false;
    if ((uint64_t)b->table_width * p->page_tokens > kMaxTokens) return false;
    if (b->n_seqs > 0x7FFFFFFEu || b->n_rows > 0x7FFFFFFFu) return false;
    return true;
}

// Whether the places that an append writes differ: no zero stride over several
// pages, tokens or (in one page for all heads) heads.
bool places_ok(const orchkv_pages_t *p, const orchkv_batch_t *b)
{
    return (p->page_stride || p->n_pages == 1) && (p->token_stride || p->page_tokens == 1) &&
           (p->head_stride || b->table_head_stride || p->n_kv_heads == 1);
}

bool heads_ok(const orchkv_pages_t *p, const orchkv_batch_t *b, uint32_t hq)
{
    return hq != 0 && hq % p->n_kv_heads == 0 && (uint64_t)hq * b->n_rows < 0x7FFFFFFFull;
}

PagesDev pages_dev(const orchkv_pages_t *p)
{
    const long long e = (long long)dtype_size((DataType)p->dtype);
    PagesDev d;
    d.k = (char *)p->k;
    d.v = (char *)p->v;
    d.page_b = p->page_stride * e;
    d.head_b = p->head_stride * e;
    d.tok_b = p->token_stride * e;
    d.n_pages = p->n_pages;
    d.H = p->n_kv_heads;
    d.D = p->d_head;
    d.bs = fast_div(p->page_tokens);
    return d;
}

BatchDev batch_dev(const orchkv_batch_t *b)
{
    BatchDev d;
    d.table = b->table;
    d.ts_seq = b->table_seq_stride;
    d.ts_head = b->table_head_stride;
    d.width = b->table_width;
    d.n = b->n_seqs;
    d.rows = b->n_rows;
    d.lens = b->lens;
    d.starts = b->starts;
    return d;
}

RowsDev rows_dev(const orchkv_rows_t &r, size_t e)
{
    return RowsDev{(char *)r.p, r.row_stride * (long long)e, r.head_stride * (long long)e};
}

// Which sequences go to the attention's tile kernel: none in calls whose row
// tiles (16 packed rows) times key tiles (64 keys) are at most kSmall for each
// of the few-row kernel's 296 places, where the second pair of launches costs
// more than the tensor cores gain; else those with more than kFewRows packed
// rows.  One request of 48 tokens over 500, 32/8 heads: 13.8 us against 26.1 by
// the tile kernel; 8 requests of 12 over 500, 28/4 heads: 15.4 against 33.4; one
// of 48 over 4000 (19 a place): 44.3 against 59.3; 8 of 12 over 4000 (41): 68.3
// against 46.8.
constexpr uint32_t kFewRows = 32;
constexpr uint64_t kSmall = 24;
// The masses' tile kernel has one product to do and two small launches: it takes
// every sequence of more rows than this.  48 rows over 500: 8.7 us against 13.5
// by the tile kernel; 96 rows: 15.2 against 14.3; 400 rows: 56.7 against 15.4.
constexpr uint32_t kFewMassRows = 64;

bool small_call(const orchkv_pages_t *p, const orchkv_batch_t *b, uint64_t G, uint64_t keys)
{
    const uint64_t units = p->n_kv_heads * (b->n_rows * G / 16 + b->n_seqs);
    return units * ((keys + 63) / 64) <= kSmall * 296;
}

// No sequence is longer than 2^30: a larger window is no window.
uint32_t window_of(uint32_t w) { return w > (1u << 30) ? 0 : w; }

// What one attend call launches, from what the host knows of it.
struct AttendPlan {
    SplitDev rows, tile;     // ctas 0: not launched
    ClassDev few, many;
    bool no_rows;
    size_t bytes;
};

AttendPlan plan_attend(const orchkv_pages_t *p, const orchkv_batch_t *b, const orchkv_attend_args_t *args)
{
    AttendPlan pl = {};
    const uint64_t G = args->n_q_heads / p->n_kv_heads, H = p->n_kv_heads;
    const uint64_t keys = (uint64_t)b->table_width * p->page_tokens;
    const uint64_t most = (uint64_t)(b->max_new < b->n_rows ? b->max_new : b->n_rows) * G;
    const bool tile = most > kFewRows && !small_call(p, b, G, keys) &&
                      attend_tile_takes(pages_dev(p), p->dtype, args->scale);
    const uint32_t R = p->dtype == DTYPE_FP32 ? kSimtRows : kRowsRows;
    uint64_t units = H * (b->n_rows * G / R + b->n_seqs);
    if (tile) units = std::min(units, H * b->n_seqs * (kFewRows / R));
    pl.few = ClassDev{0, tile ? kFewRows : 0xFFFFFFFFu};
    pl.many = ClassDev{kFewRows, 0xFFFFFFFFu};
    pl.no_rows = tile && b->n_seqs == 1;     // one sequence is of one kind: one pair of launches
    if (pl.no_rows)
        pl.many.min_rows = 0;
    else if (p->dtype == DTYPE_FP32)
        pl.rows.ctas = attend_simt_ctas(units, keys);
    else
        pl.rows = attend_rows_split(p->d_head, b->n_seqs, p->n_kv_heads,
                                    std::max<uint32_t>(1, (std::min<uint64_t>(most, pl.few.max_rows) + R - 1) / R),
                                    units, keys);
    if (tile) pl.tile.ctas = attend_tile_ctas(H * (b->n_rows * G / kTileRows + b->n_seqs), keys);
    // both may use the same memory: the tile kernel starts when the rows are joined
    const size_t row = (p->d_head + 2) * sizeof(float) * 2;
    pl.bytes = std::max(pl.rows.ctas * R, pl.tile.ctas * kTileRows) * row;
    pl.bytes = (pl.bytes + 255) & ~size_t(255);
    return pl;
}

struct MassPlan {
    SplitDev tile;           // ctas 0: not launched
    ClassDev few, many;
    size_t bytes;
};

MassPlan plan_mass(const orchkv_pages_t *p, const orchkv_batch_t *b, const orchkv_mass_args_t *args)
{
    MassPlan pl = {};
    const size_t e = dtype_size((DataType)p->dtype);
    const uint32_t G = args->n_q_heads / p->n_kv_heads;
    const uint64_t keys = (uint64_t)b->table_width * p->page_tokens;
    const uint64_t new_rows = b->max_new < b->n_rows ? b->max_new : b->n_rows;
    const bool tile = new_rows * G > kFewMassRows &&
                      mass_tile_takes(pages_dev(p), p->dtype, args->scale, rows_dev(args->q, e), G);
    pl.few = ClassDev{0, tile ? kFewMassRows : 0xFFFFFFFFu};
    pl.many = ClassDev{kFewMassRows, 0xFFFFFFFFu};
    if (tile)
        pl.tile.ctas = mass_tile_ctas((uint64_t)p->n_kv_heads * b->n_seqs * ((keys + 255) / 256), new_rows * G);
    pl.bytes = ((size_t)2 * pl.tile.ctas * kMassSlot * sizeof(float) + 255) & ~size_t(255);
    return pl;
}

}  // namespace

extern "C" {

int orchkv_paged_append(const orchkv_pages_t *pages, const orchkv_batch_t *batch,
                        const orchkv_append_args_t *args, void *stream)
{
    OKV_RANGE("orchkv_paged_append");
    if (!args || !shapes_ok(pages, batch, true)) return ORCHKV_ERR_INVALID;
    const size_t e = dtype_size((DataType)pages->dtype);
    if (args->rot_dim % 2 || args->rot_dim > pages->d_head) return ORCHKV_ERR_INVALID;
    if (args->rot_dim && !args->turns) return ORCHKV_ERR_INVALID;
    if (batch->n_rows == 0 || batch->n_seqs == 0) return ORCHKV_OK;
    if (!rows_ok(args->k, e) || !rows_ok(args->v, e) || !places_ok(pages, batch)) return ORCHKV_ERR_INVALID;
    if (args->n_q_heads && (!rows_ok(args->q, e) || !rows_ok(args->q_out, e))) return ORCHKV_ERR_INVALID;
    const auto span = [&](const orchkv_rows_t &r, uint32_t heads) {
        return row_span(r, batch->n_rows, heads, (int64_t)(pages->d_head * e), (int64_t)e);
    };
    if (args->n_q_heads) {
        // (other CTAs read what one of them writes)
        const RowSpan q = span(args->q, args->n_q_heads), o = span(args->q_out, args->n_q_heads);
        if (overlaps_itself(o) || (!same_rows(q, o) && overlap(q, o)) ||
            overlap(o, span(args->k, pages->n_kv_heads)) || overlap(o, span(args->v, pages->n_kv_heads)))
            return ORCHKV_ERR_INVALID;
    }
    if (args->n_q_heads > 65535 ||
        (uint64_t)batch->n_rows * (args->n_q_heads + 2ull * pages->n_kv_heads) > 0x7FFFFFFFull)
        return ORCHKV_ERR_INVALID;
    AppendDev a;
    a.q = rows_dev(args->q, e);
    a.q_out = rows_dev(args->q_out, e);
    a.k = rows_dev(args->k, e);
    a.v = rows_dev(args->v, e);
    a.Hq = args->n_q_heads;
    a.rot = args->rot_dim;
    a.inter = args->interleaved != 0;
    a.pos64 = args->positions_64 != 0;
    a.scale = args->scale;
    a.eps = args->eps;
    a.turns = args->turns;
    a.pos = args->positions;
    a.q_norm = args->q_norm;
    a.k_norm = args->k_norm;
    return launch_paged_append(pages->dtype, pages_dev(pages), batch_dev(batch), a,
                               (cudaStream_t)stream);
}

size_t orchkv_paged_attend_workspace(const orchkv_pages_t *pages, const orchkv_batch_t *batch,
                                     const orchkv_attend_args_t *args)
{
    if (!args || !shapes_ok(pages, batch, false) || !heads_ok(pages, batch, args->n_q_heads)) return 0;
    if (batch->n_rows == 0 || batch->n_seqs == 0) return 0;
    return plan_attend(pages, batch, args).bytes;
}

int orchkv_paged_attend(const orchkv_pages_t *pages, const orchkv_batch_t *batch,
                        const orchkv_attend_args_t *args, void *workspace, size_t bytes, void *stream)
{
    OKV_RANGE("orchkv_paged_attend");
    if (!args || !shapes_ok(pages, batch, true) || !heads_ok(pages, batch, args->n_q_heads))
        return ORCHKV_ERR_INVALID;
    if (batch->n_rows == 0 || batch->n_seqs == 0) return ORCHKV_OK;
    const size_t e = dtype_size((DataType)pages->dtype);
    if (!rows_ok(args->q, e) || !rows_ok(args->out, e)) return ORCHKV_ERR_INVALID;
    // (several CTAs read a row of q that one of them writes the result of)
    const RowSpan qs = row_span(args->q, batch->n_rows, args->n_q_heads, (int64_t)(pages->d_head * e), (int64_t)e);
    const RowSpan os = row_span(args->out, batch->n_rows, args->n_q_heads, (int64_t)(pages->d_head * e), (int64_t)e);
    if (overlap(qs, os) || overlaps_itself(os)) return ORCHKV_ERR_INVALID;
    AttendPlan pl = plan_attend(pages, batch, args);
    if (pl.bytes && (!workspace || (uintptr_t)workspace % 256 || bytes < pl.bytes)) return ORCHKV_ERR_INVALID;
    AttendDev a;
    a.q = rows_dev(args->q, e);
    a.out = rows_dev(args->out, e);
    a.lse = args->lse;
    a.Hq = args->n_q_heads;
    a.G = args->n_q_heads / pages->n_kv_heads;
    a.window = window_of(args->window);
    a.sl2 = args->scale * 1.4426950408889634f;
    const PagesDev p = pages_dev(pages);
    const BatchDev b = batch_dev(batch);
    pl.rows.ws = pl.tile.ws = (float *)workspace;
    const cudaStream_t st = (cudaStream_t)stream;
    if (pages->dtype == DTYPE_FP32) return launch_attend_simt(p, b, a, pl.few, pl.rows, st);
    int rc = ORCHKV_OK;
    if (!pl.no_rows) rc = launch_attend_rows(pages->dtype, p, b, a, pl.few, pl.rows, st);
    if (rc || pl.tile.ctas == 0) return rc;
    return launch_attend_tile(pages->dtype, p, b, a, pl.many, pl.tile, st);
}

size_t orchkv_paged_block_mass_workspace(const orchkv_pages_t *pages, const orchkv_batch_t *batch,
                                         const orchkv_mass_args_t *args)
{
    if (!args || !shapes_ok(pages, batch, false) || !heads_ok(pages, batch, args->n_q_heads)) return 0;
    if (batch->n_seqs == 0) return 0;
    return plan_mass(pages, batch, args).bytes;
}

int orchkv_paged_block_mass(const orchkv_pages_t *pages, const orchkv_batch_t *batch,
                            const orchkv_mass_args_t *args, void *workspace, size_t bytes, void *stream)
{
    OKV_RANGE("orchkv_paged_block_mass");
    if (!args || !shapes_ok(pages, batch, false) || !heads_ok(pages, batch, args->n_q_heads))
        return ORCHKV_ERR_INVALID;
    if (batch->n_seqs == 0) return ORCHKV_OK;
    const size_t e = dtype_size((DataType)pages->dtype);
    if (!args->mass || (batch->n_rows && (!rows_ok(args->q, e) || !args->lse))) return ORCHKV_ERR_INVALID;
    if (batch->n_rows) {
        const RowSpan q = row_span(args->q, batch->n_rows, args->n_q_heads, (int64_t)(pages->d_head * e), (int64_t)e);
        if (mass_overlaps(args->mass, batch->n_seqs, pages->n_kv_heads, batch->table_width, q, args->lse))
            return ORCHKV_ERR_INVALID;
    }
    MassPlan pl = plan_mass(pages, batch, args);
    if (pl.bytes && (!workspace || (uintptr_t)workspace % 256 || bytes < pl.bytes)) return ORCHKV_ERR_INVALID;
    MassDev a;
    a.q = rows_dev(args->q, e);
    a.lse = args->lse;
    a.mass = args->mass;
    a.Hq = args->n_q_heads;
    a.G = args->n_q_heads / pages->n_kv_heads;
    a.window = window_of(args->window);
    a.sl2 = args->scale * 1.4426950408889634f;
    const PagesDev p = pages_dev(pages);
    const BatchDev b = batch_dev(batch);
    const cudaStream_t st = (cudaStream_t)stream;
    if (pages->dtype == DTYPE_FP32) return launch_mass_simt(p, b, a, pl.few, st);
    const int rc = launch_mass_rows(pages->dtype, p, b, a, pl.few, st);
    if (rc || pl.tile.ctas == 0) return rc;
    pl.tile.ws = (float *)workspace;
    return launch_mass_tile(pages->dtype, p, b, a, pl.many, pl.tile, st);
}

}  // extern "C"
