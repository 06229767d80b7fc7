// The operators of a serving step over a paged cache: attention_paged, kv_append_paged and qk_norm_rope.  They have no
// counterpart in the reference crate, whose cache is one buffer per sequence (attention_kv_cached/args.rs:8-30) and whose
// operators take one sequence at a time; names, layouts, verbs and errors follow the crate's operators.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>

#include "../kernels/params.h"
#include "handle.hpp"

using namespace ophip;

namespace {

void expect_index_type(uint64_t dt, const char *name) {
    if (dt != OPHIP_DT_U32 && dt != OPHIP_DT_I32) throw type_not_support(std::string(name) + " must be 32-bit integers");
}
void expect_position_type(uint64_t dt) {
    if (dt != OPHIP_DT_U32 && dt != OPHIP_DT_U64 && dt != OPHIP_DT_I32 && dt != OPHIP_DT_I64) throw type_not_support("p must be 32 or 64-bit integers");
}
void expect_element_type(uint64_t dt) {
    if (dt != OPHIP_DT_F16 && dt != OPHIP_DT_BF16 && dt != OPHIP_DT_F32) throw type_not_support("f16, bf16 and f32 are supported");
}
int type_index(uint64_t dt) { return dt == OPHIP_DT_F16 ? 0 : dt == OPHIP_DT_BF16 ? 1 : 2; }

// every size and stride known, strides and address whole elements
void expect_static(const ophip_tensor_layout &l, const void *base, const char *name) {
    const ptrdiff_t unit = (ptrdiff_t)ophip_dtype_nbytes(l.dt);
    for (uint64_t i = 0; i < l.ndim; ++i) {
        (void)static_of(l.shape[i]);
        if (static_of(l.strides[i]) % unit != 0) throw strides_not_support(std::string("misaligned strides of ") + name);
    }
    if (reinterpret_cast<uintptr_t>(base) % (size_t)unit != 0) throw args_not_support(std::string("misaligned base of ") + name);
}
// elements adjacent, everything else on 16-byte boundaries
bool vector_rows(const ophip_tensor_layout &l, const void *base) {
    if (!aligned16(base) || l.strides[l.ndim - 1] != (ptrdiff_t)ophip_dtype_nbytes(l.dt)) return false;
    for (uint64_t i = 0; i + 1 < l.ndim; ++i)
        if (!mult16(l.strides[i])) return false;
    return true;
}

// Whether the address ranges two views reach do not meet (an empty view reaches nothing).
bool apart(const ophip_tensor_layout &a, const void *a_base, const ophip_tensor_layout &b, const void *b_base) {
    auto span = [](const ophip_tensor_layout &l, const void *base) {
        const char *lo = static_cast<const char *>(base), *hi = lo + ophip_dtype_nbytes(l.dt);
        for (uint64_t i = 0; i < l.ndim; ++i) {
            if (l.shape[i] == 0) return std::pair<const char *, const char *>(nullptr, nullptr);
            const ptrdiff_t reach = (ptrdiff_t)((l.shape[i] - 1) * (size_t)l.strides[i]);
            (reach < 0 ? lo : hi) += reach;
        }
        return std::pair<const char *, const char *>(lo, hi);
    };
    const auto x = span(a, a_base), y = span(b, b_base);
    return x.first == x.second || y.first == y.second || x.second <= y.first || y.second <= x.first;
}
bool same_view(const ophip_tensor_layout &a, const void *a_base, const ophip_tensor_layout &b, const void *b_base) {
    if (a_base != b_base) return false;
    for (uint64_t i = 0; i < a.ndim; ++i)
        if (a.shape[i] > 1 && a.strides[i] != b.strides[i]) return false;
    return true;
}

// theta as rope has it; 0: no rotation
bool rotation(float theta, size_t dh, double *freq_step) {
    const float t = static_of(theta);
    if (!(t >= 0.f)) throw args_not_support("theta must not be negative");
    if (t == 0.f) return false;
    if (dh % 2) throw shape_not_support("rotation needs an even head dimension");
    *freq_step = std::log2((double)t) / (double)(dh / 2);
    return true;
}

constexpr size_t MAX_HEAD = 512;         // elements of a head
constexpr size_t MAX_INDEX = 0x7fffffffu;
constexpr size_t MAX_TOKENS = 0xffffffu;  // a workgroup of 256 each: a launch has fewer than 2^32 work-items
constexpr size_t MAX_KEYS = 0x40000000u;  // of a sequence: key numbers and the ends of their tiles fit 31 bits

// ---- the batch: page table [nseq, cols], first tokens [nseq + 1], lengths [nseq], cache [pages, nkvh, page, dh]
struct BatchMeta {
    size_t nseq, cols, npages, nkvh, page;
};
BatchMeta batch_meta(const ophip_tensor_layout &k_cache, const ophip_tensor_layout &v_cache, const ophip_tensor_layout &table,
                     const ophip_tensor_layout &q_start, const ophip_tensor_layout &kv_len) {
    expect_rank(k_cache, "k_cache", 4);
    expect_rank(v_cache, "v_cache", 4);
    expect_rank(table, "page_table", 2);
    expect_rank(q_start, "q_start", 1);
    expect_rank(kv_len, "kv_len", 1);
    expect_index_type(table.dt, "page_table");
    expect_index_type(q_start.dt, "q_start");
    expect_index_type(kv_len.dt, "kv_len");
    BatchMeta m;
    const size_t starts = q_start.shape[0];
    if (starts == 0) throw shape_mismatch("q_start has one value more than there are sequences");
    m.nseq = dim_distinct({table.shape[0], kv_len.shape[0], is_dyn(starts) ? starts : starts - 1});
    m.cols = table.shape[1];
    m.npages = dim_distinct({k_cache.shape[0], v_cache.shape[0]});
    m.nkvh = dim_distinct({k_cache.shape[1], v_cache.shape[1]});
    m.page = dim_distinct({k_cache.shape[2], v_cache.shape[2]});
    return m;
}
PagedBatch batch_params(const BatchMeta &m, size_t nt, const ophip_tensor_layout &table, const void *table_base, const ophip_tensor_layout &q_start,
                        const void *q_start_base, const ophip_tensor_layout &kv_len, const void *kv_len_base) {
    const size_t page = static_of(m.page), npages = static_of(m.npages), nseq = static_of(m.nseq);
    if (page == 0) throw shape_not_support("a page of no tokens");
    const size_t cols = npages ? static_of(m.cols) : 0;  // (no pages: no keys)
    if (nt > MAX_TOKENS || nseq >= MAX_INDEX || npages > MAX_INDEX || page > MAX_KEYS || (cols && page > MAX_KEYS / cols))
        throw shape_not_support("batch or cache too large");
    expect_static(table, table_base, "page_table");
    expect_static(q_start, q_start_base, "q_start");
    expect_static(kv_len, kv_len_base, "kv_len");
    if (!q_start_base || !kv_len_base || (cols && !table_base)) throw args_not_support("null base address");
    PagedBatch b{};
    b.table = table_base;
    b.q_start = q_start_base;
    b.kv_len = kv_len_base;
    b.t_row = table.strides[0], b.t_col = table.strides[1], b.s_step = q_start.strides[0], b.l_step = kv_len.strides[0];
    b.nseq = (uint32_t)nseq, b.nt = (uint32_t)nt, b.cols = (uint32_t)cols, b.npages = (uint32_t)npages;
    b.page = make_fastdiv((uint32_t)page);
    return b;
}

}  // namespace

// ============================================================== attention_paged ===

struct ophip_attention_paged : OpBase {
    hipFunction_t f32[3];        // [dh up to 64, 128, 256]: tiles of 64 rows
    hipFunction_t any[3][4][2];  // [type][dh up to 64, 128, 256, 512][4 / 16 waves]
    // [f16 / bf16][tiles of 16 / 128 / 256 / 128 rows for two groups][dh 64, 128, below 64, below 128, up to 256]; 256 rows for dh 128
    // only, two groups for 64 and 128
    hipFunction_t rows[2][4][5], join[2][4][5];
    // read once, here (tests, sweeps): OPHIP_ATTN_PAGED_SLOTS=<n> key ranges to cut a launch into, OPHIP_ATTN_PAGED_TILE=0|1|2|3
    // one kind of tile (1 where there is no other for the head dimension)
    int slots = 0, tile = -1;
    explicit ophip_attention_paged(ophip_device *d) : OpBase(d) {
        for (int n = 0; n < 3; ++n) f32[n] = d->kernel("attention_paged_f32", ("attn_paged_f32_d" + std::to_string(64 << n)).c_str());
        static const char *const tag[3] = {"f16", "bf16", "f32"};
        for (int t = 0; t < 3; ++t)
            for (int n = 0; n < 4; ++n)
                for (int w = 0; w < 2; ++w) any[t][n][w] = d->kernel("attention_paged_any", (std::string("attn_paged_any_") + tag[t] + "_n" + std::to_string(1 << n) + (w ? "_w16" : "")).c_str());
        for (int e = 0; e < 2; ++e)
            for (int r = 0; r < 4; ++r)
                for (int h = 0; h < 5; ++h) {
                    if ((r == 2 && h != 1) || (r == 3 && h > 1)) continue;
                    static const char *const head[5] = {"d64", "d128", "d64_pad", "d128_pad", "d256_pad"};
                    const char *mod = e ? "attention_paged_bf16" : "attention_paged";
                    const std::string tail = std::string(head[h]) + (e ? "_bf16" : "");
                    static const char *const of[4] = {"few_", "many_", "wide_", "pair_"};
                    rows[e][r][h] = d->kernel(mod, ("attn_paged_" + (of[r] + tail)).c_str());
                    join[e][r][h] = d->kernel(mod, ("attn_paged_join_" + (of[r == 3 ? 1 : r] + tail)).c_str());
                }
        if (const char *e = std::getenv("OPHIP_ATTN_PAGED_SLOTS")) slots = std::atoi(e);
        if (const char *e = std::getenv("OPHIP_ATTN_PAGED_TILE")) tile = std::atoi(e);
    }
};

namespace {

struct AttnPagedMeta : BatchMeta {
    uint64_t dt;
    size_t nh, nt, dh;
};
AttnPagedMeta attention_paged_meta(const ophip_attention_paged_args &a) {
    expect_rank(a.q_layout, "q", 3);
    expect_rank(a.o_layout, "o", 3);
    AttnPagedMeta m;
    static_cast<BatchMeta &>(m) = batch_meta(a.k_cache_layout, a.v_cache_layout, a.page_table_layout, a.q_start_layout, a.kv_len_layout);
    m.dt = type_distinct({a.q_layout.dt, a.k_cache_layout.dt, a.v_cache_layout.dt, a.o_layout.dt});
    expect_element_type(m.dt);
    m.nh = dim_distinct({a.q_layout.shape[0], a.o_layout.shape[0]});
    m.nt = dim_distinct({a.q_layout.shape[1], a.o_layout.shape[1]});
    m.dh = dim_distinct({a.q_layout.shape[2], a.o_layout.shape[2], a.k_cache_layout.shape[3], a.v_cache_layout.shape[3]});
    if (a.mask != OPHIP_MASK_NONE && a.mask != OPHIP_MASK_CAUSAL) throw args_not_support("unknown mask");
    if (!is_dyn(m.nh) && !is_dyn(m.nkvh) && (m.nkvh == 0 ? m.nh != 0 : m.nh % m.nkvh != 0)) throw shape_mismatch("nh must be a multiple of nkvh");
    if (!is_dyn(m.dh) && m.dh > MAX_HEAD) throw shape_not_support("head dimension too large");
    return m;
}

// How the matrix kernels take a call (attention_paged.hip), from its sizes alone.
struct AttnPagedPlan {
    bool matrix;                    // they serve these types and sizes
    int tile, head;                 // tiles of 16, 128 or 256 rows, or of 128 for two groups of waves: 0, 1, 2, 3; of the kernels' head dimensions
    size_t grid, slots;  // workgroups; key ranges the workspace holds (0: no tile can be cut)
    size_t workspace;
};
AttnPagedPlan attention_paged_plan(const ophip_attention_paged *op, const AttnPagedMeta &m) {
    AttnPagedPlan a{};
    for (size_t v : {m.nh, m.nt, m.dh, m.nkvh, m.nseq, m.page, m.cols})
        if (is_dyn(v) || v == 0) return a;
    if ((m.dt != OPHIP_DT_F16 && m.dt != OPHIP_DT_BF16) || m.dh % 8 || m.dh > 256 || m.nh % m.nkvh) return a;
    if (m.nh > MAX_INDEX / m.nt || m.page > MAX_KEYS / m.cols) return a;
    a.matrix = true;
    a.head = m.dh == 64 ? 0 : m.dh == 128 ? 1 : m.dh < 64 ? 2 : m.dh < 128 ? 3 : 4;
    const size_t dh = m.dh <= 64 ? 64 : m.dh <= 128 ? 128 : 256;  // columns that they work on
    const size_t cus = (size_t)(op ? op->dev->props.multiProcessorCount : 256);
    // Tiles of 16 rows where nearly all sequences have no more, and where there is little to do: a tile of 128 rows then takes
    // its keys with fewer workgroups than there are CUs (403 tokens of 12 sequences, 4 heads over 2, up to 2035 keys: 14.0
    // against 17.5 us; 127 tokens of 2 sequences, 16 heads over 8, 5479 keys, over twice the bound: 57 against 26.5; 280 tokens
    // of 2 sequences, 64 heads over 32, 161 keys, twice the bound of rows: 11.5 against 8.5).
    // Tiles of 256, which load once for twice the rows, where a sequence fills several and the work is long (8192 tokens,
    // 32 heads over 8: 558 against 585 us, 511 tokens over 32511 keys 299 against 318; shorter than the bound, 7 prompts of up
    // to 546 tokens 36.8 against 32.6; dh 64 never gains by them).
    const size_t group = m.nh / m.nkvh, rows = m.nt * group, products = m.nkvh * rows * (m.page * m.cols);  // (below 2^61)
    // Tiles of 128 that two groups of waves share, half of the keys each, where there is about one for each CU or fewer and no
    // ranges are cut (70 batches of up to 768 keys, up to 1024 with three quarters of the CUs, 6 to 17 % faster, the worst 5 %
    // slower).  With more tiles the second workgroup of a CU serves better than the second group (some 450 rows to a
    // sequence, 32 kv heads of 64, up to 600 keys: 47 against 28 us), with more keys ranges do, as often as not (133 batches
    // of up to 4096 keys between 0.74 and 1.38 times as long).
    const size_t len = m.cols * m.page, tiles128 = m.nkvh * (rows + std::min(m.nseq, m.nt) * 127);  // times 128, at the most
    if ((products <= cus << 14 && m.nkvh * rows <= cus << 5) || (group <= 16 && m.nt <= 2 * m.nseq)) a.tile = 0;
    else if (m.dh == 128 && rows >= 1024 * m.nseq && products >= cus << 20) a.tile = 2;
    else a.tile = a.head <= 1 && tiles128 <= 154 * cus && rows >= 64 * m.nseq && len <= (tiles128 >= 96 * cus ? 1024u : 768u) ? 3 : 1;
    if (op && op->tile >= 0 && op->tile <= 3) a.tile = op->tile;
    if ((a.tile == 2 && m.dh != 128) || (a.tile == 3 && a.head > 1)) a.tile = 1;
    const size_t tile = a.tile == 0 ? 16 : a.tile == 2 ? 256 : 128;
    // the most tiles there can be, whatever the lengths: each sequence that has a token may have one that is not full
    const size_t units = m.nkvh * ((rows + std::min(m.nseq, m.nt) * (tile - 1)) / tile);
    const size_t steps = (m.cols * m.page + 31) / 32;
    const size_t most = std::max<size_t>(1, steps / 4);  // (a key range has four steps of 32 keys at least)
    // Key ranges for all tiles together: as many as workgroups of 128 or 256 rows run at a time (two or one per CU, one for
    // heads above 128; 511 tokens over 32511 keys, 32 heads over 8, on tiles of 128: 420 us with half as many, 321, 338 with twice
    // as many), and four per CU for 16 rows, where a range costs little and the rates of memory even out (50 decode steps
    // over 165008 keys: 134 us with 512, 122 with 1024, 124 with 1536).  The device makes fewer of them for short batches
    // (paged_per_step).
    const size_t want = op && op->slots > 0 ? (size_t)op->slots : (a.tile == 0 ? 4 : a.tile == 1 && dh <= 128 ? 2 : 1) * cus;
    a.grid = units;
    // No ranges, and no second launch, where a tile takes its keys in less time than cutting and joining would cost: short ones, and
    // longer ones where the tiles fill the machine as it is (615 tokens of 2 sequences, 64 heads over 4, up to 597 keys: 25.1 us
    // against 37.1 with ranges; 4097 tokens of 17 sequences, 16 heads over 1, 923 keys: 35.6 against 41.1; on tiles of 16 rows,
    // up to 384 keys: 8.4 against 10.0; past the bounds, a quarter of the machine and 1024 keys: 22.1 against 20.3, an
    // eighth, on tiles of 16 rows: 15.9 against 14.8).
    const size_t have = m.nkvh * rows, fill = want * tile;
    const bool whole = a.tile == 0 ? len <= 512 || (len <= 1024 && have >= fill / 8) : len <= 768 || (len <= 1024 && have >= fill / 4) || (len <= 2048 && have >= fill);
    if (most > 1 && !whole) {
        a.slots = std::min((4 * want + 2) / 3, units * most);
        a.grid = std::min(units * most, units + (4 * want + 2) / 3);
        a.workspace = 64 + a.slots * (32 + tile * (dh + 2) * sizeof(float));
    }
    return a;
}

void attention_paged_launch(const ophip_attention_paged *op, const ophip_attention_paged_args &a, void *workspace, size_t workspace_len,
                            const ophip_queue_alloc *qa) {
    const AttnPagedMeta m = attention_paged_meta(a);
    const size_t nh = static_of(m.nh), nt = static_of(m.nt), dh = static_of(m.dh), nkvh = static_of(m.nkvh), nseq = static_of(m.nseq);
    const float scale = static_of(a.scale);
    if (std::isnan(scale) || std::isinf(scale)) throw args_not_support("scale must be a number");
    expect_static(a.q_layout, a.q_base, "q");
    expect_static(a.o_layout, a.o_base, "o");
    expect_static(a.k_cache_layout, a.k_cache_base, "k_cache");
    expect_static(a.v_cache_layout, a.v_cache_base, "v_cache");
    if (nh == 0 || nt == 0 || dh == 0 || nseq == 0) return;
    AttnPagedParams p{};
    p.b = batch_params(m, nt, a.page_table_layout, a.page_table_base, a.q_start_layout, a.q_start_base, a.kv_len_layout, a.kv_len_base);
    if (nh > 0xffffu || nh > MAX_INDEX / nt) throw shape_not_support("too many rows");
    if (!a.q_base || !a.o_base || (p.b.cols && (!a.k_cache_base || !a.v_cache_base))) throw args_not_support("null base address");
    // a workgroup writes rows of o while others still read: o lies apart from what is read, or is q itself, row by row
    if (!same_view(a.o_layout, a.o_base, a.q_layout, a.q_base) && !apart(a.o_layout, a.o_base, a.q_layout, a.q_base))
        throw args_not_support("o overlaps q");
    if (!apart(a.o_layout, a.o_base, a.k_cache_layout, a.k_cache_base) || !apart(a.o_layout, a.o_base, a.v_cache_layout, a.v_cache_base))
        throw args_not_support("o overlaps the cache");
    if (!apart(a.o_layout, a.o_base, a.page_table_layout, a.page_table_base) || !apart(a.o_layout, a.o_base, a.q_start_layout, a.q_start_base) ||
        !apart(a.o_layout, a.o_base, a.kv_len_layout, a.kv_len_base))
        throw args_not_support("o overlaps the page table, q_start or kv_len");
    p.q = a.q_base, p.o = a.o_base, p.k = a.k_cache_base, p.v = a.v_cache_base;
    const ptrdiff_t *s = a.q_layout.strides;
    p.q_sh = s[0], p.q_st = s[1], p.q_sd = s[2];
    s = a.o_layout.strides;
    p.o_sh = s[0], p.o_st = s[1], p.o_sd = s[2];
    s = a.k_cache_layout.strides;
    p.k_sp = s[0], p.k_sh = s[1], p.k_sr = s[2], p.k_sd = s[3];
    s = a.v_cache_layout.strides;
    p.v_sp = s[0], p.v_sh = s[1], p.v_sr = s[2], p.v_sd = s[3];
    p.group = make_fastdiv((uint32_t)(nh / nkvh));
    p.nkvh = (uint32_t)nkvh, p.dh = (uint32_t)dh, p.causal = a.mask == OPHIP_MASK_CAUSAL;
    p.scale = scale;
    const bool vec = vector_rows(a.q_layout, a.q_base) && vector_rows(a.o_layout, a.o_base) && vector_rows(a.k_cache_layout, a.k_cache_base) &&
                     vector_rows(a.v_cache_layout, a.v_cache_base);
    const AttnPagedPlan plan = attention_paged_plan(op, m);
    // (a scale that is not positive: the matrix kernels take the maximum before they scale)
    if (plan.matrix && p.b.cols && scale > 0.f && plan.grid <= 0xffffffffu / 512 && vec) {
        Workspace ws(qa, workspace, workspace_len, plan.workspace);
        p.work = ws.ptr();
        p.slots = (uint32_t)plan.slots;
        p.cus = (uint32_t)(op->slots > 0 ? op->slots : op->dev->props.multiProcessorCount);
        const ptrdiff_t far = (ptrdiff_t)1 << 31;
        p.narrow = p.k_sp == p.v_sp && p.k_sr == p.v_sr && p.k_sp >= 0 && p.k_sp < far && p.k_sr >= 0 && p.k_sr < far / (ptrdiff_t)p.b.page.d &&
                   p.b.t_col >= 0 && p.b.t_col < far / (ptrdiff_t)p.b.cols;
        const int e = m.dt == OPHIP_DT_BF16, h = plan.head;
        op->dev->make_current();
        launch(op->rows[e][plan.tile][h], Dim3{(unsigned)plan.grid}, Dim3{plan.tile >= 2 ? 512u : 256u}, 0, stream_of(qa), p);
        if (plan.slots) launch(op->join[e][plan.tile][h], Dim3{(unsigned)plan.slots}, Dim3{plan.tile ? 512u : 256u}, 0, stream_of(qa), p);
        return;
    }
    op->dev->make_current();
    // f32: tiles of 64 rows on the matrix cores where they are less work than a row at a time.  A tile's keys are never cut into
    // ranges, so it takes its place on a CU (two at dh up to 128, one above) as long as `worth` rows, of which as many run at a
    // time as there are CUs; fewer tiles than places take no less time for that.  Over 2117 batches of 1 to 256 sequences and tokens, of
    // like and unlike lengths up to 32768, 1 to 32 query heads to a kv head, 1 to 2 % from the faster one, the worst 1.17, 1.26, 1.49 times as
    // long at dh 64, 128, 256.  Tiles against rows, dh 128: a step of 16 heads over 1 and 4096 keys 379 us, 109; 32 steps of 32
    // over 8, 2000 to 4000 keys 455, 421; 16 tokens, 32 heads over 8, 32768 keys 3.42 ms, 1.76; 64 tokens 3.45, 5.88; 256
    // tokens, 4096 keys 0.41, 2.59.
    const size_t cus = (size_t)op->dev->props.multiProcessorCount, rows = nt * (nh / nkvh), units = nkvh * ((rows + std::min(nseq, nt) * 63) / 64);
    const double worth = dh <= 64 ? 2 : dh <= 128 ? 4.5 : 6;
    const bool tiles = op->tile >= 0 ? op->tile > 0 : (double)(nt * nh) >= worth * (double)std::max(dh <= 128 ? units / 2 : units, cus);
    if (m.dt == OPHIP_DT_F32 && dh % 4 == 0 && dh <= 256 && p.b.cols && vec && units <= 0xffffffffu / 256 && tiles) {
        launch(op->f32[dh <= 64 ? 0 : dh <= 128 ? 1 : 2], Dim3{(unsigned)units}, Dim3{256}, 0, stream_of(qa), p);
        return;
    }
    // sixteen waves to a row where there are no more than two rows to a CU
    const int n = dh <= 64 ? 0 : dh <= 128 ? 1 : dh <= 256 ? 2 : 3, w = nt * nh <= 2 * cus;
    launch(op->any[type_index(m.dt)][n][w], Dim3{(unsigned)nt, (unsigned)nh}, Dim3{w ? 1024u : 256u}, 0, stream_of(qa), p);
}

}  // namespace

extern "C" {

int ophip_attention_paged_create(ophip_device *dev, ophip_attention_paged **out) {
    return guard([&] {
        if (!dev || !out) throw args_not_support("null argument");
        *out = new ophip_attention_paged(dev);
    });
}
void ophip_attention_paged_destroy(ophip_attention_paged *op) { delete op; }

int ophip_attention_paged_scheme(ophip_attention_paged *op, const ophip_attention_paged_args *args, size_t max_ws, size_t *ws) {
    return guard([&] {
        if (ws) *ws = 0;
        if (!args) throw args_not_support("null argument");
        const AttnPagedMeta m = attention_paged_meta(*args);
        const size_t need = attention_paged_plan(op, m).workspace;
        if (ws && need <= max_ws) *ws = need;  // (with less, launch takes it from the queue's allocator)
    });
}

int ophip_attention_paged_launch(const ophip_attention_paged *op, const ophip_attention_paged_args *args, void *workspace, size_t workspace_len,
                                 const ophip_queue_alloc *qa) {
    return guard([&] {
        if (!op || !args) throw args_not_support("null argument");
        attention_paged_launch(op, *args, workspace, workspace_len, qa);
    });
}

}  // extern "C"

// ============================================================== kv_append_paged ===

struct ophip_kv_append_paged : OpBase {
    hipFunction_t vec[3][2], pairs[3];  // vec: plain and non-temporal stores
    explicit ophip_kv_append_paged(ophip_device *d) : OpBase(d) {
        static const char *tag[3] = {"f16", "bf16", "f32"};
        for (int t = 0; t < 3; ++t) {
            for (int nt = 0; nt < 2; ++nt) vec[t][nt] = d->kernel("kv_append_paged", (std::string("kv_append_") + tag[t] + (nt ? "_vec_nt" : "_vec")).c_str());
            pairs[t] = d->kernel("kv_append_paged", (std::string("kv_append_") + tag[t] + "_pairs").c_str());
        }
    }
};

namespace {

struct KvAppendMeta : BatchMeta {
    uint64_t dt;
    size_t nt, dh;
};
KvAppendMeta kv_append_paged_meta(const ophip_kv_append_paged_args &a) {
    expect_rank(a.k_layout, "k", 3);
    expect_rank(a.v_layout, "v", 3);
    expect_rank(a.p_layout, "p", 1);
    expect_position_type(a.p_layout.dt);
    KvAppendMeta m;
    static_cast<BatchMeta &>(m) = batch_meta(a.k_cache_layout, a.v_cache_layout, a.page_table_layout, a.q_start_layout, a.kv_len_layout);
    m.dt = type_distinct({a.k_layout.dt, a.v_layout.dt, a.k_cache_layout.dt, a.v_cache_layout.dt});
    expect_element_type(m.dt);
    m.nkvh = dim_distinct({m.nkvh, a.k_layout.shape[0], a.v_layout.shape[0]});
    m.nt = dim_distinct({a.k_layout.shape[1], a.v_layout.shape[1], a.p_layout.shape[0]});
    m.dh = dim_distinct({a.k_layout.shape[2], a.v_layout.shape[2], a.k_cache_layout.shape[3], a.v_cache_layout.shape[3]});
    if (!is_dyn(m.dh) && m.dh > MAX_HEAD) throw shape_not_support("head dimension too large");
    return m;
}

void kv_append_paged_launch(const ophip_kv_append_paged *op, const ophip_kv_append_paged_args &a, const ophip_queue_alloc *qa) {
    const KvAppendMeta m = kv_append_paged_meta(a);
    const size_t nt = static_of(m.nt), dh = static_of(m.dh), nkvh = static_of(m.nkvh), nseq = static_of(m.nseq);
    KvAppendPagedParams p{};
    p.rotate = rotation(a.theta, dh, &p.freq_step);
    expect_static(a.k_layout, a.k_base, "k");
    expect_static(a.v_layout, a.v_base, "v");
    expect_static(a.p_layout, a.p_base, "p");
    expect_static(a.k_cache_layout, a.k_cache_base, "k_cache");
    expect_static(a.v_cache_layout, a.v_cache_base, "v_cache");
    if (nt == 0 || dh == 0 || nkvh == 0 || nseq == 0) return;
    p.b = batch_params(m, nt, a.page_table_layout, a.page_table_base, a.q_start_layout, a.q_start_base, a.kv_len_layout, a.kv_len_base);
    if (p.b.cols == 0) return;  // no place for any key
    if (nkvh > MAX_INDEX / MAX_HEAD) throw shape_not_support("too many heads");
    if (!a.k_base || !a.v_base || !a.k_cache_base || !a.v_cache_base || (p.rotate && !a.p_base)) throw args_not_support("null base address");
    // a workgroup writes the caches while others still read everything else
    const struct {
        const ophip_tensor_layout &l;
        const void *base;
    } from[6] = {{a.k_layout, a.k_base}, {a.v_layout, a.v_base}, {a.page_table_layout, a.page_table_base}, {a.q_start_layout, a.q_start_base},
                 {a.kv_len_layout, a.kv_len_base}, {a.p_layout, a.p_base}};
    for (int i = 0; i < (p.rotate ? 6 : 5); ++i)
        if (!apart(from[i].l, from[i].base, a.k_cache_layout, a.k_cache_base) || !apart(from[i].l, from[i].base, a.v_cache_layout, a.v_cache_base))
            throw args_not_support(i < 2 ? "k or v overlaps the cache" : "the page table, q_start, kv_len or p overlaps the cache");
    // (the caches' address ranges may meet, as those of two halves of one buffer do, their elements not)
    if (a.k_cache_base == a.v_cache_base) throw args_not_support("k_cache and v_cache are one");
    p.k = a.k_base, p.v = a.v_base, p.pos = a.p_base, p.k_cache = a.k_cache_base, p.v_cache = a.v_cache_base;
    const ptrdiff_t *s = a.k_layout.strides;
    p.k_sh = s[0], p.k_st = s[1], p.k_sd = s[2];
    s = a.v_layout.strides;
    p.v_sh = s[0], p.v_st = s[1], p.v_sd = s[2];
    s = a.k_cache_layout.strides;
    p.kc_sp = s[0], p.kc_sh = s[1], p.kc_sr = s[2], p.kc_sd = s[3];
    s = a.v_cache_layout.strides;
    p.vc_sp = s[0], p.vc_sh = s[1], p.vc_sr = s[2], p.vc_sd = s[3];
    p.p_step = a.p_layout.strides[0];
    p.pos_is_u64 = ophip_dtype_nbytes(a.p_layout.dt) == 8;
    p.nkvh = (uint32_t)nkvh, p.dh = (uint32_t)dh;
    const bool vec = dh * ophip_dtype_nbytes(m.dt) % 16 == 0 && vector_rows(a.k_layout, a.k_base) && vector_rows(a.v_layout, a.v_base) &&
                     vector_rows(a.k_cache_layout, a.k_cache_base) && vector_rows(a.v_cache_layout, a.v_cache_base);
    op->dev->make_current();
    // (more than the L2 caches hold together, 8 x 4 MiB: whoever reads it next does not find it there)
    const bool stream_out = 2 * nt * nkvh * dh * ophip_dtype_nbytes(m.dt) > (size_t)32 << 20;
    const int t = type_index(m.dt);
    launch(vec ? op->vec[t][stream_out] : op->pairs[t], Dim3{(unsigned)nt}, Dim3{256}, p.rotate ? dh / 2 * 8 : 0, stream_of(qa), p);
}

}  // namespace

extern "C" {

int ophip_kv_append_paged_create(ophip_device *dev, ophip_kv_append_paged **out) {
    return guard([&] {
        if (!dev || !out) throw args_not_support("null argument");
        *out = new ophip_kv_append_paged(dev);
    });
}
void ophip_kv_append_paged_destroy(ophip_kv_append_paged *op) { delete op; }

int ophip_kv_append_paged_scheme(ophip_kv_append_paged *, const ophip_kv_append_paged_args *args, size_t, size_t *ws) {
    return guard([&] {
        if (ws) *ws = 0;
        if (!args) throw args_not_support("null argument");
        (void)kv_append_paged_meta(*args);
    });
}

int ophip_kv_append_paged_launch(const ophip_kv_append_paged *op, const ophip_kv_append_paged_args *args, void *, size_t, const ophip_queue_alloc *qa) {
    return guard([&] {
        if (!op || !args) throw args_not_support("null argument");
        kv_append_paged_launch(op, *args, qa);
    });
}

}  // extern "C"

// ================================================================= qk_norm_rope ===

struct ophip_qk_norm_rope : OpBase {
    hipFunction_t vec[3][4][3], pairs[3];  // vec: rows of 8, 16, 32, 64 lanes; one row per thread, several, several with non-temporal stores
    explicit ophip_qk_norm_rope(ophip_device *d) : OpBase(d) {
        static const char *tag[3] = {"f16", "bf16", "f32"}, *lanes[4] = {"_l8", "_l16", "_l32", "_l64"}, *form[3] = {"", "_multi", "_multi_nt"};
        for (int t = 0; t < 3; ++t) {
            const std::string name = std::string("qk_norm_rope_") + tag[t];
            for (int l = 0; l < 4; ++l)
                for (int f = 0; f < 3; ++f) vec[t][l][f] = d->kernel("qk_norm_rope", (name + lanes[l] + form[f]).c_str());
            pairs[t] = d->kernel("qk_norm_rope", (name + "_pairs").c_str());
        }
    }
};

namespace {

struct QkNormRopeMeta {
    uint64_t dt, dt_w;
    size_t nt, nh, nkh, dh;
};
QkNormRopeMeta qk_norm_rope_meta(const ophip_qk_norm_rope_args &a) {
    expect_rank(a.qy_layout, "qy", 3);
    expect_rank(a.q_layout, "q", 3);
    expect_rank(a.qw_layout, "qw", 1);
    expect_rank(a.ky_layout, "ky", 3);
    expect_rank(a.k_layout, "k", 3);
    expect_rank(a.kw_layout, "kw", 1);
    expect_rank(a.p_layout, "p", 1);
    QkNormRopeMeta m;
    m.dt = type_distinct({a.qy_layout.dt, a.q_layout.dt, a.ky_layout.dt, a.k_layout.dt});
    m.dt_w = type_distinct({a.qw_layout.dt, a.kw_layout.dt});
    expect_element_type(m.dt);
    if (m.dt_w != m.dt && m.dt_w != OPHIP_DT_F32) throw type_not_support("the weights have the rows' type or f32");
    expect_position_type(a.p_layout.dt);
    m.nt = dim_distinct({a.qy_layout.shape[0], a.q_layout.shape[0], a.ky_layout.shape[0], a.k_layout.shape[0], a.p_layout.shape[0]});
    m.nh = dim_distinct({a.qy_layout.shape[1], a.q_layout.shape[1]});
    m.nkh = dim_distinct({a.ky_layout.shape[1], a.k_layout.shape[1]});
    m.dh = dim_distinct({a.qy_layout.shape[2], a.q_layout.shape[2], a.ky_layout.shape[2], a.k_layout.shape[2], a.qw_layout.shape[0], a.kw_layout.shape[0]});
    if (!is_dyn(m.dh) && (m.dh > MAX_HEAD || m.dh % 2)) throw shape_not_support("head dimension odd or too large");
    return m;
}

void qk_norm_rope_launch(const ophip_qk_norm_rope *op, const ophip_qk_norm_rope_args &a, const ophip_queue_alloc *qa) {
    const QkNormRopeMeta m = qk_norm_rope_meta(a);
    const size_t nt = static_of(m.nt), nh = static_of(m.nh), nkh = static_of(m.nkh), dh = static_of(m.dh), heads = nh + nkh;
    QkNormRopeParams p{};
    p.rotate = rotation(a.theta, dh, &p.freq_step);
    p.epsilon = static_of(a.epsilon);
    const ptrdiff_t unit = (ptrdiff_t)ophip_dtype_nbytes(m.dt), wunit = (ptrdiff_t)ophip_dtype_nbytes(m.dt_w);
    expect_static(a.p_layout, a.p_base, "p");
    const struct {
        const ophip_tensor_layout &y, &x, &w;
        void *y_base;
        const void *x_base, *w_base;
        size_t nh;
    } half[2] = {{a.qy_layout, a.q_layout, a.qw_layout, a.qy_base, a.q_base, a.qw_base, nh}, {a.ky_layout, a.k_layout, a.kw_layout, a.ky_base, a.k_base, a.kw_base, nkh}};
    bool vec = dh * unit % 16 == 0;
    for (int i = 0; i < 2; ++i) {
        expect_static(half[i].y, half[i].y_base, "y");
        expect_static(half[i].x, half[i].x_base, "x");
        expect_static(half[i].w, half[i].w_base, "w");
        if (dh && (half[i].y.strides[2] != unit || half[i].x.strides[2] != unit || half[i].w.strides[0] != wunit))
            throw strides_not_support("qk_norm_rope needs a contiguous head dimension");
        p.x[i] = half[i].x_base, p.y[i] = half[i].y_base, p.w[i] = half[i].w_base;
        p.x_st[i] = half[i].x.strides[0], p.x_sh[i] = half[i].x.strides[1], p.y_st[i] = half[i].y.strides[0], p.y_sh[i] = half[i].y.strides[1];
        p.nh[i] = (uint32_t)half[i].nh;
    }
    if (nt == 0 || heads == 0 || dh == 0) return;
    if (nt > MAX_TOKENS || nh > 0xffffu || nkh > 0xffffu) throw shape_not_support("too many tokens or heads");
    for (int i = 0; i < 2; ++i) {
        const auto &h = half[i];
        if (h.nh == 0) continue;
        if (!h.y_base || !h.x_base || !h.w_base) throw args_not_support("null base address");
        if (!same_view(h.y, h.y_base, h.x, h.x_base) && !apart(h.y, h.y_base, h.x, h.x_base)) throw args_not_support("y overlaps its x");
        vec = vec && vector_rows(h.y, h.y_base) && vector_rows(h.x, h.x_base);
    }
    if (p.rotate && !a.p_base) throw args_not_support("null base address");
    // a workgroup writes its rows while others still read weights, positions and the other rows
    for (int i = 0; i < 2; ++i) {
        const auto &h = half[i], &other = half[1 - i];
        if (h.nh == 0) continue;
        if (!apart(h.y, h.y_base, h.w, h.w_base) || (other.nh && !apart(h.y, h.y_base, other.w, other.w_base)) || (p.rotate && !apart(h.y, h.y_base, a.p_layout, a.p_base)))
            throw args_not_support("y overlaps weights or positions");
        // (the ranges of q's and k's rows may meet, as those of one projection's parts do, their elements not)
        if (other.nh && (h.y_base == other.y_base || h.y_base == other.x_base)) throw args_not_support("qy shares elements with k or ky, or ky with q");
    }
    p.pos = a.p_base;
    p.p_step = a.p_layout.strides[0];
    p.pos_is_u64 = ophip_dtype_nbytes(a.p_layout.dt) == 8;
    p.nt = (uint32_t)nt, p.dh = (uint32_t)dh;
    p.w_is_f32 = m.dt_w == OPHIP_DT_F32;
    const size_t vectors = dh * unit / 16;
    vec = vec && vectors <= 64;
    const int li = vectors <= 8 ? 0 : vectors <= 16 ? 1 : vectors <= 32 ? 2 : 3;
    // Few tokens: a token's heads over several workgroups, down to one row for each group of lanes.  More: up to eight tokens to
    // a workgroup, so that its 256 threads share the sines and cosines, two pairs for each at the most; as many as its four
    // rows per thread hold, or more where that still leaves two workgroups per CU (16 + 2 heads of 128, tokens with 1 / 2 / 4 / 8
    // to a workgroup: 512 10.1 / 6.9 / 7.8 / 9.9 us, 2048 19.3 / 12.7 / 10.7 / 11.3, 4095 34.1 / 21.1 / 16.5 / 15.6;
    // 36 + 12 heads, 2048 21.7 / 17.3 / 17.3 / 20.9; 4 + 1 heads, 2048 17.1 / 10.1 / 7.8 / 6.5).  Stores are non-temporal where
    // the result is larger than the L2 caches together (8 x 4 MiB): whoever reads it next does not find it there.
    const size_t rows = vec ? 32u >> li : 4, fit = nt < 256 ? 1 : 4 * rows / heads, full = nt < 512 ? 1 : nt < 2048 ? 2 : nt < 4096 ? 4 : 8;
    const size_t tokens = vec ? std::max<size_t>(1, std::min({std::max(fit, full), (size_t)8, 1024 / dh})) : 1;
    const size_t by = tokens > 1 ? 1 : std::min((heads + rows - 1) / rows, std::max<size_t>(1, 1024 / nt)), per = (heads + by - 1) / by;
    p.heads_per_block = make_fastdiv((uint32_t)per);
    p.tokens_per_block = (uint32_t)tokens;
    op->dev->make_current();
    const int t = type_index(m.dt), form = tokens * per <= rows ? 0 : nt * heads * dh * unit <= (size_t)32 << 20 ? 1 : 2;
    launch(vec ? op->vec[t][li][form] : op->pairs[t], Dim3{(unsigned)((nt + tokens - 1) / tokens), (unsigned)((heads + per - 1) / per)}, Dim3{256},
           p.rotate ? tokens * (dh / 2) * 8 : 0, stream_of(qa), p);
}

}  // namespace

extern "C" {

int ophip_qk_norm_rope_create(ophip_device *dev, ophip_qk_norm_rope **out) {
    return guard([&] {
        if (!dev || !out) throw args_not_support("null argument");
        *out = new ophip_qk_norm_rope(dev);
    });
}
void ophip_qk_norm_rope_destroy(ophip_qk_norm_rope *op) { delete op; }

int ophip_qk_norm_rope_scheme(ophip_qk_norm_rope *, const ophip_qk_norm_rope_args *args, size_t, size_t *ws) {
    return guard([&] {
        if (ws) *ws = 0;
        if (!args) throw args_not_support("null argument");
        (void)qk_norm_rope_meta(*args);
    });
}

int ophip_qk_norm_rope_launch(const ophip_qk_norm_rope *op, const ophip_qk_norm_rope_args *args, void *, size_t, const ophip_queue_alloc *qa) {
    return guard([&] {
        if (!op || !args) throw args_not_support("null argument");
        qk_norm_rope_launch(op, *args, qa);
    });
}

}  // extern "C"
