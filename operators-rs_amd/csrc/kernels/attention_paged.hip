// attention over a paged cache on the matrix cores: o = softmax(scale q . k^T) . v for a packed batch of sequences of
// unlike lengths, f16 / bf16, head dimensions of a multiple of 8 up to 256 (kernels for 64, 128 and 256 columns).
//
// Work units.  The query rows of one kv head and sequence are its new tokens times the `group` query heads that share
// the kv head, row = token * group + head-in-group.  A sequence of up to 16 rows (a decode step) is one tile that
// paged_few works on: the caches are all the traffic.  One of more rows (prompts, chunks) is cut into tiles of 128 or 256 rows
// for paged_many: the products are the work.  So keys and values are read once per tile whatever the group, and a short
// group fills the rows with further tokens.  Four kernels: attn_paged_few, on tiles of 16 rows only, for batches that are
// nearly all decode steps and for little work; attn_paged_many, which has both inside and gives each sequence its own (24 decode
// steps and a chunk of 333 tokens over 56185 keys in all, dh 64: 35 us; on tiles of 16 rows alone 59); attn_paged_wide, the same
// on tiles of 256 rows, for long sequences; attn_paged_pair, the same on tiles of 128 rows whose keys two groups of waves
// take in turn, for so few tiles that a CU has one at the most.  The host chooses by sizes (attention_paged_plan).
//
// Plan.  The host knows the number of tokens and sequences, not the lengths, and must not wait for them; so every
// workgroup works its own unit out from the lengths on the device (paged_item: a prefix sum over the sequences, 2.5 to 3.5 us).
// The tiles of a sequence with more keys than 1 / slots of all tiles' keys are cut into that many more key ranges, one workgroup
// each, so that a launch has about `slots` equal pieces of work whatever the mix of lengths.  Ranges of a cut tile leave
// their maximum, sum and output in the workspace and attn_paged_join merges them in a fixed order: results do not
// depend on which workgroup ends first.  (Joining in the first launch, by the workgroup that finds all ranges of its tile
// there, spares a launch of 3 us but makes every workgroup wait for its stores: a decode step over 2048 keys 12.1 us against
// 11.3, 47 of them 127 against 118.)
//
// Compiled twice, like the other MFMA kernels (gemm_elem.h).
#include "gemm_elem.h"
#include "paged_plan.h"

constexpr float PA_LOG2E = 1.4426950408889634f;
// The softmax is taken against a reference that trails the running maximum by at most 2^PA_LAG: sums and output are
// rescaled only when a row's maximum has outgrown its reference by more, which after the first tiles is next to never (the
// largest score of a row of random ones grows by its logarithm), instead of in most tiles (any of 32 rows will do).
constexpr float PA_LAG = 8.f;
// Probabilities are kept times 2^PA_BIAS (as are their sums), up to 2^15 with the lag: in f16, steps of 2^-24 below 2^-14
// would cost the many small ones of a long row their bits.
#ifdef GEMM_ELEM_BF16
constexpr float PA_BIAS = 0.f;
#else
constexpr float PA_BIAS = 7.f;
#endif

// Whether any of a vector's elements is infinite or NaN: its exponent is all ones
__device__ __forceinline__ uint32_t exponents(uint32_t most, uint32_t pair) {  // the larger of each half, signs aside
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, most), __builtin_bit_cast(u16x2, pair & 0x7fff7fffu)));
}
__device__ __forceinline__ bool not_finite(uint32_t most) {
#ifdef GEMM_ELEM_BF16
    constexpr uint32_t ONES = 0x7f80u;
#else
    constexpr uint32_t ONES = 0x7c00u;
#endif
    return (most & 0xffffu) >= ONES || (most >> 16) >= ONES;
}

// sum + the pair's two elements (v_dot2c: subnormal ones count, f32 rounding)
__device__ __forceinline__ float add_pair(float sum, uint32_t pair) {
    typedef elem elem2 __attribute__((ext_vector_type(2)));
    const elem2 x = __builtin_bit_cast(elem2, pair), one = {(elem)1.f, (elem)1.f};
#ifdef GEMM_ELEM_BF16
    return __builtin_amdgcn_fdot2_f32_bf16(x, one, sum, false);
#else
    return __builtin_amdgcn_fdot2(x, one, sum, false);
#endif
}

// The matrix kernels multiply the values of a tile's keys with a probability of zero where a row does not keep them, and
// zero times infinity or NaN is NaN.  Where paged_many has met values that are not finite in a tile that some row keeps in part
// (the last ones under a causal mask), and where paged_few's sums are not finite, they come here for the whole range instead
// of handing out their result: a wave to a row, key by key, as in attention_paged_any.hip.  What a row does not keep then
// does not touch it, whatever it is.  Right, but slow, a row and key at a time: an infinite value at the end of one of 47 decode
// steps 530 us against 122 for all of them, of a prompt of 546 tokens among seven 0.9 ms against 29 us, of 511 tokens over 32511
// keys 121 ms against 0.34.
template <int DH, int ROWS, bool PAD>
__device__ __forceinline__ void paged_exactly(const AttnPagedParams &p, const PagedItem &it, uint32_t key0, uint32_t key1, uint32_t waves) {
    constexpr int W = DH / WAVE;  // columns per lane
    const uint32_t lane = threadIdx.x % WAVE;
    const bool live = !PAD || W * lane < p.dh;  // (the others: column 0 again, of no weight and not stored)
    const uint32_t c0 = live ? W * lane : 0;
    const char *kb = reinterpret_cast<const char *>(p.k) + (int64_t)it.kvh * p.k_sh + 2 * c0;
    const char *vb = reinterpret_cast<const char *>(p.v) + (int64_t)it.kvh * p.v_sh + 2 * c0;
    for (uint32_t r = threadIdx.x / WAVE; r < it.nrows; r += waves) {
        const uint32_t row = it.row0 + r, token = fastdiv(row, p.group), head = it.kvh * p.group.d + (row - token * p.group.d);
        const elem *qr = reinterpret_cast<const elem *>(reinterpret_cast<const char *>(p.q) + (int64_t)head * p.q_sh + (int64_t)(it.s.start + token) * p.q_st) + c0;
        const uint32_t keep = min(key1, paged_keep(p, it, token));
        float m = -INFINITY, l = 0.f, o[W] = {};
        for (uint32_t key = key0; key < keep; ++key) {
            const uint32_t col = fastdiv(key, p.b.page), line = key - col * p.b.page.d, page = min(paged_page(p.b, it.seq, col), p.b.npages - 1);
            const elem *kr = reinterpret_cast<const elem *>(kb + (int64_t)page * p.k_sp + (int64_t)line * p.k_sr);
            const elem *vr = reinterpret_cast<const elem *>(vb + (int64_t)page * p.v_sp + (int64_t)line * p.v_sr);
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < W; ++i) dot += live ? e2f(qr[i]) * e2f(kr[i]) : 0.f;
            const float x = wave_sum_dpp(dot) * (p.scale * PA_LOG2E), top = fmaxf(m, x);
            const float old = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top), e = x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x - top + PA_BIAS);
            l = l * old + e;
#pragma unroll
            for (int i = 0; i < W; ++i) o[i] = o[i] * old + e * e2f(vr[i]);
            m = top;
        }
        if (!live) continue;
        if (it.pieces > 1) {
            float *dst = paged_partial(p, ROWS) + ((size_t)it.slot * ROWS + r) * DH + c0;
#pragma unroll
            for (int i = 0; i < W; ++i) dst[i] = o[i];
            if (lane == 0) *reinterpret_cast<f32x2 *>(paged_stats(p) + ((size_t)it.slot * ROWS + r) * 2) = f32x2{m, l};
        } else {
            elem *dst = reinterpret_cast<elem *>(reinterpret_cast<char *>(p.o) + (int64_t)head * p.o_sh + (int64_t)(it.s.start + token) * p.o_st) + c0;
            const float inv = keep ? 1.0f / l : 0.f;  // (no key: zeros; no score above -inf: 0 / 0, as the definition has it)
#pragma unroll
            for (int i = 0; i < W; ++i) dst[i] = f2e(o[i] * inv);
        }
    }
}

// ---- up to 16 rows: one pass over the keys at the rate of memory
//
// A workgroup of four waves takes a key range in steps of 32 keys, a step per wave; nothing is shared between the waves
// until the end.  Keys and values go from memory straight into the lanes' registers, the next step's on their way while one
// is multiplied, and the page numbers one step ahead of those.
//   S^T = K . Q^T (v_mfma 16x16x32): A is 16 keys, 16 bytes per lane as they lie in memory; lane (j, g) of the result has
//   query j and the keys 4 g + i of the 16.  So a query's maximum and sum are eight registers of four lanes, its
//   factors are scalars of the lane, and the probabilities are, as they lie, B operands of
//   O^T = V^T . P^T, contraction slot 8 g + 4 c + i being key 16 c + 4 g + i.  A is then the values of those eight keys, of
//   which the lane reads DH / 16 adjacent columns each and transposes them in registers.
// The matrix cores are idle most of the time: 16 KB of keys and values take about 500 cycles of one wave, a CU's share of
// the memory's rate delivers them in 1300.  Memory bounds it: 50 decode steps over 165008 keys, 8 kv heads of 128, 676 MB,
// 116 us, 5.8 TB/s (a pure read of that size with the non-temporal hint 6.46, a copy 4.89); below some 50 MB the latencies of the
// launches, the plan and a range's first loads do (one step over 2047 keys, 8 MB: 11 us, of which 9 are the two launches).
template <int CW>
struct FewTile {  // 32 keys
    u32x4 k[2][CW / 2];
    uint32_t v[8][CW / 2];
};

template <int DH>
struct FewLds {
    float m[4][16], l[4][16], o[4][DH / 4][WAVE];
    uint32_t bad[4];  // by wave: sums of values that are not finite, of a row whose probabilities are
};

// ROWS: of the tiles whose partial results the workspace holds
template <int DH, int ROWS, bool PAD>
__device__ __forceinline__ void paged_few(const AttnPagedParams &p, const PagedItem &it, FewLds<DH> &lds) {
    constexpr int CW = DH / 16, KS = DH / 32;  // columns of v per lane, contraction steps of q . k
    const uint32_t wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, j = lane % 16, g = lane / 16;
    const uint32_t row = it.row0 + min(j, it.nrows - 1), token = fastdiv(row, p.group), head = it.kvh * p.group.d + (row - token * p.group.d);
    const uint32_t keep = paged_keep(p, it, token), keys = paged_keep(p, it, fastdiv(it.row0 + it.nrows - 1, p.group));
    const uint32_t steps = (keys + 31) / 32, per = (steps + it.pieces - 1) / it.pieces;
    const uint32_t first = it.piece * per + wave, last = min(steps, it.piece * per + per);

    u32x4 q[KS];
    {
        const char *src = reinterpret_cast<const char *>(p.q) + (int64_t)head * p.q_sh + (int64_t)(it.s.start + token) * p.q_st + 16 * g;
#pragma unroll
        for (int s = 0; s < KS; ++s) q[s] = !PAD || 32 * s + 8 * g < p.dh ? ld128(src + 64 * s) : u32x4{0, 0, 0, 0};
    }
    const char *kb = reinterpret_cast<const char *>(p.k) + (int64_t)it.kvh * p.k_sh + 16 * g;
    const char *vb = reinterpret_cast<const char *>(p.v) + (int64_t)it.kvh * p.v_sh + 2 * CW * j;
    // the lane's two keys of a step (16 c + j), bounded by the sequence's last
    uint32_t col[2], line[2], page[2];
    auto look_up = [&](uint32_t step) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t key = min(step * 32 + 16 * c + j, it.s.len - 1);
            col[c] = fastdiv(key, p.b.page);
            line[c] = key - col[c] * p.b.page.d;
            page[c] = paged_page(p.b, it.seq, col[c]);
        }
    };
    auto fetch = [&](FewTile<CW> &t) {
        uint32_t pg[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            pg[c] = min(page[c], p.b.npages - 1);
            const char *src = kb + (int64_t)pg[c] * p.k_sp + (int64_t)line[c] * p.k_sr;
#pragma unroll
            for (int s = 0; s < KS; ++s) t.k[c][s] = !PAD || 32 * s + 8 * g < p.dh ? ld128_nt(src + 64 * s) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t vp = __shfl(pg[c], 4 * g + i, WAVE), vl = __shfl(line[c], 4 * g + i, WAVE);
                const char *src = vb + (int64_t)vp * p.v_sp + (int64_t)vl * p.v_sr;
                if constexpr (CW == 4) {
                    *reinterpret_cast<u32x2 *>(t.v[4 * c + i]) = !PAD || CW * j < p.dh ? __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(src)) : u32x2{0, 0};
                } else {
#pragma unroll
                    for (int w = 0; w < CW; w += 8)
                        *reinterpret_cast<u32x4 *>(t.v[4 * c + i] + w / 2) = !PAD || CW * j + w < p.dh ? ld128_nt(src + 2 * w) : u32x4{0, 0, 0, 0};
                }
            }
    };
    const float scale2 = p.scale * PA_LOG2E;
    float m = -INFINITY, l = 0.f;
    f32x4 o[CW];
#pragma unroll
    for (int t = 0; t < CW; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](FewTile<CW> &t, uint32_t step) {
        if (step * 32 + 32 > it.s.len) {  // (behind the last key: that key again)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int d = 0; d < CW / 2; ++d)
                    if (step * 32 + 16 * (i / 4) + 4 * g + i % 4 >= it.s.len) t.v[i][d] = 0;
        }
        float x[8], mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                PackE a, b;
                a.u = t.k[c][k];
                b.u = q[k];
                s = mfma_16x16x32(a.h, b.h, s);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[4 * c + i] = step * 32 + 16 * c + 4 * g + i < keep ? s[i] * scale2 : -INFINITY;
                mx = fmaxf(mx, x[4 * c + i]);
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16, WAVE));
        mx = fmaxf(mx, __shfl_xor(mx, 32, WAVE));
        if (__builtin_amdgcn_ballot_w64(mx > m + PA_LAG) != 0) {
            const float now = fmaxf(m, mx), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - now);
            l *= f;
#pragma unroll
            for (int c = 0; c < CW; ++c) o[c] *= f;
            m = now;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        // A probability goes in as two elements, its rounding and what that left out: the matrix cores have the time, and the
        // result then is as exact as with f32 probabilities.
        PackE pr, rest;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float e = __builtin_amdgcn_exp2f(x[i] - ref + PA_BIAS);
            l += e;
            pr.e[i] = f2e(e);
            rest.e[i] = f2e(e - e2f(pr.e[i]));
        }
#pragma unroll
        for (int c = 0; c < CW; ++c) {
            PackE a;
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const uint32_t lo = t.v[2 * d][c / 2], hi = t.v[2 * d + 1][c / 2];
                a.u[d] = (c & 1) ? ((lo >> 16) | (hi & 0xffff0000u)) : ((lo & 0xffffu) | (hi << 16));
            }
            o[c] = mfma_16x16x32(a.h, pr.h, o[c]);
            o[c] = mfma_16x16x32(a.h, rest.h, o[c]);
        }
    };
    if (first < last) {
        FewTile<CW> a, b;
        look_up(first);
        fetch(a);
        look_up(first + 4);
#pragma unroll
        for (int s = 0; s < KS; ++s) OPHIP_ARRIVED(q[s]);
        for (uint32_t step = first; step < last; step += 8) {
            if (step + 4 < last) {
                fetch(b);
                look_up(step + 8);
            }
            multiply(a, step);
            if (step + 4 < last) {
                if (step + 8 < last) {
                    fetch(a);
                    look_up(step + 12);
                }
                multiply(b, step + 4);
            }
        }
    }
    l += __shfl_xor(l, 16, WAVE);
    l += __shfl_xor(l, 32, WAVE);
    // A value that is not finite has made NaN of its column here even in rows that do not keep it (zero times infinity), and in those that do,
    // where a probability's rest is zero or negative.  (A sum that is NaN makes the whole row NaN: nothing to mend.)
    bool bad = false;
#pragma unroll
    for (int c = 0; c < CW; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad = bad || !(fabsf(o[c][i]) < INFINITY);
    const bool spoiled = __builtin_amdgcn_ballot_w64(bad && l < INFINITY) != 0;

    // the four waves' results, on one maximum
    if (g == 0) lds.m[wave][j] = m, lds.l[wave][j] = l;
    if (lane == 0) lds.bad[wave] = spoiled;
    __syncthreads();
    if (lds.bad[0] | lds.bad[1] | lds.bad[2] | lds.bad[3]) return paged_exactly<DH, ROWS, PAD>(p, it, it.piece * per * 32, last * 32, 4);
    float top = lds.m[0][j];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, lds.m[w][j]);
    const float ref = top == -INFINITY ? 0.f : top, f = __builtin_amdgcn_exp2f(m - ref);
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) total += lds.l[w][j] * __builtin_amdgcn_exp2f(lds.m[w][j] - ref);
#pragma unroll
    for (int t = 0; t < CW; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) lds.o[wave][4 * t + i][lane] = o[t][i] * f;
    __syncthreads();
    // lane (j, g) of wave i: query j, columns CW (4 g + i) .. + CW - 1
    if (j >= it.nrows) return;
    float out[CW];
#pragma unroll
    for (int t = 0; t < CW; ++t) {
        out[t] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) out[t] += lds.o[w][4 * t + wave][lane];
    }
    const uint32_t column = CW * (4 * g + wave);
    if (it.pieces > 1) {
        float *dst = paged_partial(p, ROWS) + ((size_t)it.slot * ROWS + j) * DH + column;
#pragma unroll
        for (int t = 0; t < CW; t += 4) *reinterpret_cast<f32x4 *>(dst + t) = f32x4{out[t], out[t + 1], out[t + 2], out[t + 3]};
        if (column == 0) *reinterpret_cast<f32x2 *>(paged_stats(p) + ((size_t)it.slot * ROWS + j) * 2) = f32x2{top, total};
        return;
    }
    const float inv = keep ? 1.0f / total : 0.f;  // (no key: zeros; no score above -inf: 0 / 0)
    union {
        elem e[CW];
        uint32_t u[CW / 2];
    } y;
#pragma unroll
    for (int t = 0; t < CW; ++t) y.e[t] = f2e(out[t] * inv);
    char *dst = reinterpret_cast<char *>(p.o) + (int64_t)head * p.o_sh + (int64_t)(it.s.start + token) * p.o_st + 2 * column;
    if constexpr (CW == 4) {
        if (!PAD || column < p.dh) *reinterpret_cast<u32x2 *>(dst) = u32x2{y.u[0], y.u[1]};
    } else {
#pragma unroll
        for (int w = 0; w < CW; w += 8)
            if (!PAD || column + w < p.dh) st128(dst + 2 * w, u32x4{y.u[w / 2], y.u[w / 2 + 1], y.u[w / 2 + 2], y.u[w / 2 + 3]});
    }
}

// ---- up to 128 rows: the products are the work
//
// Pages of a whole number of the rows that the workgroup loads at a time (RS) leave those rows in one page, so that the
// page and the address are scalars and a thread adds an offset that never changes; in vector registers the same
// arithmetic (products of 64 bits at a quarter of the rate) takes as long as the exponentials.  Other pages, caches that are
// not alike and a tile that reaches past the last key take it row by row.
//
// A workgroup of four waves, 32 rows each, walks its key range in tiles of 64 keys that go through registers into LDS,
// double-buffered, one barrier a tile; two workgroups share a CU.  S^T = K . Q^T with v_mfma 32x32x16: a lane holds one
// query and half the tile's keys, so maxima, sums and factors are scalars of the lane; the probabilities are packed in
// registers into B operands of O^T = V^T . P^T, whose A operands come from the row-major tile through the transposing
// LDS read.  A wave without rows, or whose rows all end before a tile, only helps to load.
// What bounds it is the matrix cores' rate together with the exponentials that their order leaves between the products: 8192
// tokens, 32 heads over 8 of 128, causal, 0.55 Tflop kept: 552 us, 1.0 PF (a plain product of 8192^3 reaches 1.26) with eight
// waves that share a tile's loads (565 against 602 with four on one machine); 511 tokens over 32511 keys 275 us, 0.98 PF (machines
// differ by a tenth).  In the order that the compiler gives them, products, LDS reads and the second half's exponentials took 633 us where the one
// below took 593; a raised priority of the wave around its products changed nothing.  Short prompts are bound by a unit's
// fixed time, some 6 us, and by the longest tiles, two of which share a CU: 7 prompts of 104 to 546 tokens, 32 heads of 128: 26 us.
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int DH>
struct ManyLds {
    static constexpr int BN = 64;                    // keys of a tile
    static constexpr int KP = DH + 8, VP = DH + 32;  // pitches of a row: reads of consecutive rows spread over the banks
    elem k[2][BN * KP], v[2][BN * VP];
    uint32_t bad[8];  // by wave: values that are not finite, in a tile that some row keeps in part
};

// G groups of W waves share the rows; each takes every G-th tile of keys into LDS of its own, and the second hands its maxima,
// sums and outputs to the first through LDS.
template <int DH, int W, int G, bool PAD>
__device__ __forceinline__ void paged_many(const AttnPagedParams &p, const PagedItem &it, ManyLds<DH> (&both)[G]) {
    constexpr int BN = ManyLds<DH>::BN, KP = ManyLds<DH>::KP, VP = ManyLds<DH>::VP;
    constexpr int CPR = DH / 8, ROWS = 32 * W, NCH = BN * CPR / (W * WAVE), RS = W * WAVE / CPR;  // 16-byte chunks per row, per thread; rows between a thread's chunks
    constexpr int DS = DH / 16, DB = DH / 32;
    const uint32_t group = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / (W * WAVE)), tid = threadIdx.x - group * (W * WAVE), wave = tid / WAVE, lane = tid % WAVE;
    ManyLds<DH> &lds = both[group];
    const uint32_t n32 = lane % 32, h = lane / 32, s16 = lane % 16, b16 = (lane / 16) % 2;
    const uint32_t wrow = wave * 32, at = min(wrow + n32, it.nrows - 1);
    const uint32_t row = it.row0 + at, token = fastdiv(row, p.group), head = it.kvh * p.group.d + (row - token * p.group.d);
    const uint32_t keys = paged_keep(p, it, fastdiv(it.row0 + it.nrows - 1, p.group));
    const int32_t lim = (int32_t)paged_keep(p, it, token);  // the lane's row keeps keys below it ...
    const int32_t lim_first = __builtin_amdgcn_readfirstlane(lim);  // ... the wave's first row, which keeps the fewest ...
    const int32_t lim_last = wrow < it.nrows ? (int32_t)paged_keep(p, it, fastdiv(it.row0 + min(wrow + 31, it.nrows - 1), p.group)) : 0;  // ... its last
    const uint32_t tiles = (keys + BN - 1) / BN, per = (tiles + it.pieces - 1) / it.pieces;
    const uint32_t first = it.piece * per, last = min(tiles, first + per);

    PackE qf[DS];
    {
        const char *src = reinterpret_cast<const char *>(p.q) + (int64_t)head * p.q_sh + (int64_t)(it.s.start + token) * p.q_st + 16 * h;
#pragma unroll
        for (int d = 0; d < DS; ++d) qf[d].u = !PAD || 16 * d + 8 * h < p.dh ? ld128(src + 32 * d) : u32x4{0, 0, 0, 0};
    }
    const uint32_t cc = tid % CPR, cr = tid / CPR;
    const bool live = !PAD || 8 * cc < p.dh;
    const char *kb = reinterpret_cast<const char *>(p.k) + (int64_t)it.kvh * p.k_sh + 16 * cc;
    const char *vb = reinterpret_cast<const char *>(p.v) + (int64_t)it.kvh * p.v_sh + 16 * cc;
    uint32_t page[NCH], line[NCH];  // of the next tile's rows: scalars when `aligned`
    u32x4 kreg[NCH], vreg[NCH];
    const bool aligned = p.narrow && p.b.page.d % RS == 0;
    const uint32_t off = cr * (uint32_t)p.k_sr + 16 * cc;
    const char *kh = reinterpret_cast<const char *>(p.k) + (int64_t)it.kvh * p.k_sh, *vh = reinterpret_cast<const char *>(p.v) + (int64_t)it.kvh * p.v_sh;
    const char *table = reinterpret_cast<const char *>(p.b.table) + (int64_t)it.seq * p.b.t_row;
    auto look_up = [&](uint32_t t) {
        if (aligned) {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const uint32_t key = min(t * BN + RS * i, it.s.len - 1), col = fastdiv(key, p.b.page);
                line[i] = key - col * p.b.page.d;
                page[i] = *reinterpret_cast<const uint32_t *>(table + col * (uint32_t)p.b.t_col);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const uint32_t key = min(t * BN + cr + RS * i, it.s.len - 1), col = fastdiv(key, p.b.page);
                line[i] = key - col * p.b.page.d;
                page[i] = *reinterpret_cast<const uint32_t *>(table + (int64_t)col * p.b.t_col);
            }
        }
    };
    auto fetch = [&](uint32_t t) {
        if (aligned && t * BN + BN <= it.s.len) {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const uint32_t pg = __builtin_amdgcn_readfirstlane(min(page[i], p.b.npages - 1)), ln = __builtin_amdgcn_readfirstlane(line[i]);
                const uint64_t at = (uint64_t)pg * (uint32_t)p.k_sp + ln * (uint32_t)p.k_sr;
                kreg[i] = live ? ld128(kh + at + off) : u32x4{0, 0, 0, 0};
                vreg[i] = live ? ld128(vh + at + off) : u32x4{0, 0, 0, 0};
            }
        } else {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const uint32_t pg = min(page[i], p.b.npages - 1);
                uint32_t ln = line[i];
                if (aligned) {  // the first of the RS rows, or the last key
                    const uint32_t key = t * BN + RS * i;
                    if (key < it.s.len) ln += min(cr, it.s.len - 1 - key);
                }
                kreg[i] = live ? ld128(kb + (int64_t)pg * p.k_sp + (int64_t)ln * p.k_sr) : u32x4{0, 0, 0, 0};
                vreg[i] = live ? ld128(vb + (int64_t)pg * p.v_sp + (int64_t)ln * p.v_sr) : u32x4{0, 0, 0, 0};
            }
        }
    };
    const int32_t keep_first = (int32_t)paged_keep(p, it, fastdiv(it.row0, p.group));  // the tile's first row keeps the fewest
    bool spoiled = false;
    auto commit = [&](int buf, uint32_t t) {
        if ((int32_t)(t * BN + BN) > keep_first) {  // some rows do not keep some keys
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    if (t * BN + cr + RS * i >= it.s.len) vreg[i][d] = 0;  // (the last key again)
                    most = exponents(most, vreg[i][d]);
                }
            spoiled |= __builtin_amdgcn_ballot_w64(not_finite(most)) != 0;
        }
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            st128(&lds.k[buf][(cr + RS * i) * KP + 8 * cc], kreg[i]);
            st128(&lds.v[buf][(cr + RS * i) * VP + 8 * cc], vreg[i]);
        }
    };
    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float scale2 = p.scale * PA_LOG2E;  // (positive: maxima commute with it)

    if (first + group < last) {
        look_up(first + group);
        fetch(first + group);
        commit(0, first + group);
        if (first + group + G < last) look_up(first + group + G);
    }
#pragma unroll
    for (int d = 0; d < DS; ++d) OPHIP_ARRIVED(qf[d].u);
    __syncthreads();
    for (uint32_t t0 = first; t0 < last; t0 += G) {
        const uint32_t t = t0 + group;
        const int buf = (t0 - first) / G & 1;
        const bool more = t + G < last;
        if (more) {
            fetch(t + G);
            look_up(t + 2 * G);
        }
        if ((int32_t)(t * BN) < lim_last && (G == 1 || t < last)) {
            const elem *kt = lds.k[buf], *vt = lds.v[buf];
            // sacc[b][e]: key 32 b + 8 (e / 4) + 4 h + e % 4 of the tile, query n32
            f32x16 sacc[2];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) sacc[b][e] = 0.f;
            {
                constexpr int N = 2 * DS, AHEAD = 8;
                PackE a[N];
                auto load = [&](int i) { a[i].u = ld128(kt + (32 * (i % 2) + n32) * KP + 16 * (i / 2) + 8 * h); };
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) load(i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    sacc[i % 2] = mfma_32x32x16(a[i].h, qf[i / 2].h, sacc[i % 2]);
                    if (i + AHEAD < N) load(i + AHEAD);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if ((int32_t)(t * BN + BN) > lim_first) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if ((int32_t)(t * BN + 32 * b + 8 * (e / 4) + 4 * h + e % 4) >= lim) sacc[b][e] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sacc[b][e]);
            mx = fmaxf(mx, __shfl_xor(mx, 32, WAVE));
            const float top = mx * scale2;
            if (__builtin_amdgcn_ballot_w64(top > m + PA_LAG) != 0) {
                const float now = fmaxf(m, top), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - now);
                l *= f;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[d][e] *= f;
                m = now;
            }
            const float shift = PA_BIAS - (m == -INFINITY ? 0.f : m);  // (a row that has kept nothing so far: every term is 0)
            PackE pb[4];  // MFMA n: the tile's keys 16 n .. + 15, slots 8 h .. 8 h + 7 keys 16 n + 4 h + {0..3}, 16 n + 8 + 4 h + {0..3}
            // Rounded to the type for the product: a second product for the rest, as in paged_few, would be half as much again of the matrix
            // cores' work, which bounds the kernel; errors against 64 bits are 1.2 to 1.4 times those of f32 probabilities.  The sum is of the
            // rounded ones, so that a row stays a mean of its values (with the sum of the others rows of f16's largest value came out
            // infinite); the pair's sum is one instruction (8192 tokens 556 us; a conversion and an addition for each 595).
            auto power = [&](int b, int e) {
                PackE &eight = pb[2 * b + e / 8];
                eight.e[e % 8] = f2e(__builtin_amdgcn_exp2f(__builtin_fmaf(sacc[b][e], scale2, shift)));
                if (e % 2) l = add_pair(l, eight.u[e % 8 / 2]);
            };
            typedef __attribute__((address_space(3))) s16x4 *lds_s16x4;
            {
                constexpr int N = 4 * DB, AHEAD = 4, EACH = 32 / N;  // powers of the second half with each of the first half's products
                union Frag {
                    s16x4 half[2];
                    elem8 hv;
                } a[N];
                auto load = [&](int i) {
                    const int n = i / DB, d = i % DB;
                    const elem *src = vt + (16 * n + 4 * h + s16 / 4) * VP + 32 * d + 16 * b16 + 4 * (s16 % 4);
                    a[i].half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)src);
                    a[i].half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(src + 8 * VP));
                };
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) load(i);
#pragma unroll
                for (int e = 0; e < 16; ++e) power(0, e);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    o[i % DB] = mfma_32x32x16(a[i].hv, pb[i / DB].h, o[i % DB]);
                    if (i + AHEAD < N) load(i + AHEAD);
                    if (i < N / 2)
#pragma unroll
                        for (int e = EACH * i; e < EACH * (i + 1); ++e) power(1, e);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        if (more) commit(buf ^ 1, t + G);
        __syncthreads();
    }
    if (lane == 0) lds.bad[wave] = spoiled;
    __syncthreads();
    uint32_t bad = 0;
#pragma unroll
    for (int w = 0; w < W * G; ++w) bad |= both[w / W].bad[w % W];
    if (bad) return paged_exactly<DH, ROWS, PAD>(p, it, first * BN, last * BN, W * G);
    float total = l + __shfl_xor(l, 32, WAVE);
    if constexpr (G == 2) {  // the second group's results, where its tiles were
        static_assert(sizeof(ManyLds<DH>) - sizeof lds.bad >= (size_t)W * WAVE * (DB * 16 + 2) * sizeof(float));
        f32x4 *out = reinterpret_cast<f32x4 *>(both[1].k) + tid;
        f32x2 *stats = reinterpret_cast<f32x2 *>(reinterpret_cast<f32x4 *>(both[1].k) + DB * 4 * W * WAVE) + tid;
        __syncthreads();
        if (group == 1) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q) out[(4 * d + q) * W * WAVE] = f32x4{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
            *stats = f32x2{m, total};
        }
        __syncthreads();
        if (group == 1) return;
        const f32x2 other = *stats;
        const float now = fmaxf(m, other[0]), ref = now == -INFINITY ? 0.f : now;
        const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(other[0] - ref);
        total = total * f0 + other[1] * f1;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 x = out[(4 * d + q) * W * WAVE];
#pragma unroll
                for (int r = 0; r < 4; ++r) o[d][4 * q + r] = o[d][4 * q + r] * f0 + x[r] * f1;
            }
        m = now;
    }
    if (wrow + n32 >= it.nrows) return;
    // o[d][4 q + r]: column 32 d + 8 q + 4 h + r of the lane's query
    if (it.pieces > 1) {
        float *dst = paged_partial(p, ROWS) + ((size_t)it.slot * ROWS + at) * DH + 4 * h;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q) *reinterpret_cast<f32x4 *>(dst + 32 * d + 8 * q) = f32x4{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
        if (h == 0) *reinterpret_cast<f32x2 *>(paged_stats(p) + ((size_t)it.slot * ROWS + at) * 2) = f32x2{m, total};
        return;
    }
    // two quads of a query are adjacent in lanes l and l + 32: one of each pair goes over, so that a lane stores 16 bytes
    const float inv = lim ? 1.0f / total : 0.f;  // (no key: zeros; no score above -inf: 0 / 0)
    char *dst = reinterpret_cast<char *>(p.o) + (int64_t)head * p.o_sh + (int64_t)(it.s.start + token) * p.o_st + 16 * h;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
            union {
                elem e[8];
                uint32_t u[4];
            } y;
#pragma unroll
            for (int r = 0; r < 8; ++r) y.e[r] = f2e(o[d][4 * q + r] * inv);
            const uint32_t s0 = __shfl_xor(h ? y.u[0] : y.u[2], 32, WAVE), s1 = __shfl_xor(h ? y.u[1] : y.u[3], 32, WAVE);
            if (!PAD || 32 * d + 8 * (q + h) < p.dh) st128(dst + 64 * d + 16 * q, h ? u32x4{s0, s1, y.u[2], y.u[3]} : u32x4{y.u[0], y.u[1], s0, s1});
        }
}

// ---- the ranges of a cut tile: o = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c
//
// The rows of a tile are dealt out to the workgroups of its ranges, DH / 4 threads to a row; four ranges' loads are on their
// way at a time, and the ranges are folded in one pass with a running maximum.  2.5 to 5 us, nearly all latency; 8 for the
// 256-row tiles of 511 tokens over 32511 keys, 34 MB.  Large tiles have eight waves (of four, eight and sixteen: 298 / 296 /
// 299 us for those tokens, 0.6 % between the first two over 250 drawn batches).
template <int DH, int ROWS, bool PAD>
__device__ __forceinline__ void attn_paged_join(const AttnPagedParams &p) {
    constexpr int TPR = DH / 4, RPP = (ROWS == FEW ? 256 : 512) / TPR;  // threads per row, rows per pass
    const uint32_t slot = blockIdx.x, col = 4 * (threadIdx.x % TPR);
    const PagedDesc d = paged_desc(p)[slot];
    // Slots behind the count hold no descriptor; nor do those of a batch whose sequences overlap, when it has more tiles than
    // the grid allows for: what lies there must not lead outside the workspace or o.
    if (slot >= *reinterpret_cast<const uint32_t *>(p.work) || d.pieces < 2 || d.pieces > p.slots || d.piece >= d.pieces || d.kvh >= p.nkvh || d.nrows > ROWS) return;
    const uint64_t before = (uint64_t)d.piece * p.nkvh, behind = (uint64_t)(d.pieces - 1 - d.piece) * p.nkvh;
    if (before > slot || slot + behind >= p.slots || (PAD && col >= p.dh)) return;
    const uint32_t slot0 = slot - (uint32_t)before;
    const size_t step = (size_t)p.nkvh * ROWS;
    for (uint32_t r = d.piece * RPP + threadIdx.x / TPR; r < d.nrows; r += d.pieces * RPP) {
        const float *st = paged_stats(p) + ((size_t)slot0 * ROWS + r) * 2, *po = paged_partial(p, ROWS) + ((size_t)slot0 * ROWS + r) * DH + col;
        float top = -INFINITY, total = 0.f;
        f32x4 out = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t c0 = 0; c0 < d.pieces; c0 += 4) {
            f32x2 ml[4];
            f32x4 o[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t c = min(c0 + i, d.pieces - 1);
                ml[i] = *reinterpret_cast<const f32x2 *>(st + 2 * step * c);
                o[i] = *reinterpret_cast<const f32x4 *>(po + step * DH * c);
            }
            float now = top;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                if (c0 + i >= d.pieces) ml[i] = f32x2{-INFINITY, 0.f};
                now = fmaxf(now, ml[i][0]);
            }
            const float ref = now == -INFINITY ? 0.f : now, old = __builtin_amdgcn_exp2f(top - ref);
            total *= old;
            out *= old;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const float f = __builtin_amdgcn_exp2f(ml[i][0] - ref);
                total += f * ml[i][1];
                if (c0 + i < d.pieces) out += f * o[i];
            }
            top = now;
        }
        const uint32_t row = d.row0 + r, token = fastdiv(row, p.group), head = d.kvh * p.group.d + (row - token * p.group.d);
        const float inv = token < d.blind ? 0.f : 1.0f / total;
        if (d.start >= p.b.nt || token >= p.b.nt - d.start) return;
        union {
            elem e[4];
            u32x2 u;
        } y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.e[i] = f2e(out[i] * inv);
        *reinterpret_cast<u32x2 *>(reinterpret_cast<char *>(p.o) + (int64_t)head * p.o_sh + (int64_t)(d.start + token) * p.o_st + 2 * col) = y.u;
    }
}

// PAD: a head dimension of fewer columns than DH, a multiple of 8; the others are zero and not stored
template <int DH, bool PAD>
__device__ __forceinline__ void attn_paged_few(const AttnPagedParams &p) {
    __shared__ __attribute__((aligned(16))) FewLds<DH> lds;
    PagedItem it;
    if (paged_item<16, 4>(p, it)) paged_few<DH, 16, PAD>(p, it, lds);
}
// G groups of W waves of 32 rows: 4, two workgroups to a CU, or 8 in one or two groups, one
template <int DH, int W, int G, bool PAD>
__device__ __forceinline__ void attn_paged_many(const AttnPagedParams &p) {
    __shared__ __attribute__((aligned(16))) union {
        FewLds<DH> few;
        ManyLds<DH> many[G];
    } lds;
    PagedItem it;
    if (!paged_item<32 * W, W * G>(p, it)) return;
    if (it.s.n * p.group.d <= FEW) {
        if (threadIdx.x < 4 * WAVE) paged_few<DH, 32 * W, PAD>(p, it, lds.few);  // (waves that have ended are not waited for)
    } else paged_many<DH, W, G, PAD>(p, it, lds.many);
}

#define ATTN_PAGED(name, DH, PAD, PER_CU)                                                                                                                 \
    extern "C" __global__ void __launch_bounds__(256, PER_CU) GEMM_KERNEL(attn_paged_few_##name)(AttnPagedParams p) { attn_paged_few<DH, PAD>(p); }        \
    extern "C" __global__ void __launch_bounds__(256, PER_CU) GEMM_KERNEL(attn_paged_many_##name)(AttnPagedParams p) { attn_paged_many<DH, 4, 1, PAD>(p); }   \
    extern "C" __global__ void __launch_bounds__(256) GEMM_KERNEL(attn_paged_join_few_##name)(AttnPagedParams p) { attn_paged_join<DH, 16, PAD>(p); }      \
    extern "C" __global__ void __launch_bounds__(512) GEMM_KERNEL(attn_paged_join_many_##name)(AttnPagedParams p) { attn_paged_join<DH, 128, PAD>(p); }
ATTN_PAGED(d64, 64, false, 2)
ATTN_PAGED(d128, 128, false, 2)
ATTN_PAGED(d64_pad, 64, true, 2)
ATTN_PAGED(d128_pad, 128, true, 2)
ATTN_PAGED(d256_pad, 256, true, 1)
// (dh 64 gains nothing by tiles of 256: 8192 tokens, 32 heads over 8, 391 against 363 us)
extern "C" __global__ void __launch_bounds__(512, 2) GEMM_KERNEL(attn_paged_wide_d128)(AttnPagedParams p) { attn_paged_many<128, 8, 1, false>(p); }
extern "C" __global__ void __launch_bounds__(512) GEMM_KERNEL(attn_paged_join_wide_d128)(AttnPagedParams p) { attn_paged_join<128, 256, false>(p); }
extern "C" __global__ void __launch_bounds__(512, 2) GEMM_KERNEL(attn_paged_pair_d64)(AttnPagedParams p) { attn_paged_many<64, 4, 2, false>(p); }
extern "C" __global__ void __launch_bounds__(512, 2) GEMM_KERNEL(attn_paged_pair_d128)(AttnPagedParams p) { attn_paged_many<128, 4, 2, false>(p); }
