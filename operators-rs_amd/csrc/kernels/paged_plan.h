// Which tile of which sequence, and which of its keys, a workgroup of attention over a paged cache works on, and where the
// results of key ranges go in the workspace.  The lengths are device data: every workgroup finds its place in prefix sums over
// all sequences (attention_paged.hip says why).
#pragma once
#include "paged.h"

// ---- the workspace: a count, a descriptor per slot (32 bytes), then per slot ROWS pairs (maximum, sum), then per slot
// ROWS rows of DH floats
struct PagedDesc {
    uint32_t piece, pieces, kvh, row0, nrows, start, blind, _pad;  // blind: the sequence's first tokens, that see no key
};
__device__ __forceinline__ PagedDesc *paged_desc(const AttnPagedParams &p) { return reinterpret_cast<PagedDesc *>(reinterpret_cast<char *>(p.work) + 64); }
__device__ __forceinline__ float *paged_stats(const AttnPagedParams &p) { return reinterpret_cast<float *>(reinterpret_cast<char *>(p.work) + 64 + 32 * (size_t)p.slots); }
__device__ __forceinline__ float *paged_partial(const AttnPagedParams &p, int rows) { return paged_stats(p) + 2 * (size_t)rows * p.slots; }

struct PagedItem {
    PagedSeq s;
    uint32_t seq, kvh, piece, pieces, slot;  // slot: where the range's result goes, when pieces > 1
    uint32_t row0, nrows;                     // rows of the sequence and kv head
};

constexpr uint32_t FEW = 16;
template <int ROWS>
__device__ __forceinline__ uint32_t paged_tiles(const AttnPagedParams &p, const PagedSeq &s) {
    const uint64_t rows = (uint64_t)s.n * p.group.d;
    return rows <= FEW ? (rows ? 1 : 0) : (uint32_t)((rows + ROWS - 1) / ROWS);
}
__device__ __forceinline__ uint32_t paged_steps(const PagedSeq &s) { return (s.len + 31) / 32; }
// What a step of 32 keys costs a workgroup, roughly: twice as much where a tile's rows fill the matrix cores
__device__ __forceinline__ float paged_weight(const AttnPagedParams &p, const PagedSeq &s) {
    return (uint64_t)s.n * p.group.d <= FEW ? (float)paged_steps(s) : 2.f * (float)paged_steps(s);
}
// Key ranges that a sequence's tiles are cut into, from the ranges that a unit of weight is worth
template <int ROWS>
__device__ __forceinline__ uint32_t paged_pieces(const AttnPagedParams &p, const PagedSeq &s, float per_step) {
    const uint32_t least = (uint64_t)s.n * p.group.d <= FEW ? 4 : 8;  // steps in a range: one for each wave, four tiles of 64 keys
    const uint32_t most = paged_steps(s) / least;
    return p.slots && most > 1 ? min(most, max(1u, (uint32_t)(paged_weight(p, s) * per_step + 0.5f))) : 1;
}
// Ranges per unit of weight.  `work`: tiles times weight of all sequences.  As many as there are slots (three quarters: a count
// rounded to two or more is at most four thirds of what it was) for long batches, but beyond one per CU only while each has
// 24 steps of its own (12 of heads above 128), or 8 of a tile that weighs twice: the plan, the first loads and the join cost as much as several
// steps (31 decode steps over 57 MB in 1024 / 512 / 256 ranges: 27.9 / 19.4 / 17.5 us).
template <int ROWS>
__device__ __forceinline__ float paged_per_step(const AttnPagedParams &p, float work) {
    if (!(work > 0.f)) return 0.f;
    const float all = work * (float)p.nkvh;
    return fminf(0.74999f * (float)p.slots, fmaxf((float)p.cus, all * (1.f / (ROWS == FEW && p.dh <= 128 ? 24.f : ROWS == FEW ? 12.f : 16.f)))) / all;
}

// What workgroup blockIdx.x does; false: nothing.  Every thread calls it and gets the same.
template <int ROWS, int WAVES>
__device__ __forceinline__ bool paged_item(const AttnPagedParams &p, PagedItem &it) {
    const uint32_t tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE, w = blockIdx.x;
    uint32_t local, first_slot;
    if (p.b.nseq <= WAVE) {
        // A sequence per lane, and the longest first: the units that end last should not also begin last.  So what comes before
        // a sequence is a sum over all others, of which each wave takes its share.
        __shared__ uint32_t s_before[2][WAVES][WAVE], s_all[WAVES];
        const bool on = lane < p.b.nseq;
        PagedSeq s{0, 0, 0};
        if (on) s = paged_seq(p.b, lane);
        const uint32_t tiles = paged_tiles<ROWS>(p, s);
        const float work = p.slots ? wave_sum_dpp((float)tiles * paged_weight(p, s)) : 0.f;
        const uint32_t pieces = paged_pieces<ROWS>(p, s, paged_per_step<ROWS>(p, work));
        const uint32_t items = tiles * p.nkvh * pieces, slots = pieces > 1 ? items : 0;
        uint32_t items0 = 0, slots0 = 0, all_slots = 0;
        for (uint32_t k = wave; k < p.b.nseq; k += WAVES) {
            const uint32_t len = __builtin_amdgcn_readlane(s.len, k), ni = __builtin_amdgcn_readlane(items, k), ns = __builtin_amdgcn_readlane(slots, k);
            const bool before = len > s.len || (len == s.len && k < lane);
            items0 += before ? ni : 0;
            slots0 += before ? ns : 0;
            all_slots += ns;
        }
        s_before[0][wave][lane] = items0, s_before[1][wave][lane] = slots0;
        if (lane == 0) s_all[wave] = all_slots;
        __syncthreads();
        items0 = slots0 = all_slots = 0;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) items0 += s_before[0][v][lane], slots0 += s_before[1][v][lane], all_slots += s_all[v];
        if (w == 0 && tid == 0 && p.slots) *reinterpret_cast<uint32_t *>(p.work) = min(all_slots, p.slots);
        const uint64_t mine = __builtin_amdgcn_ballot_w64(w - items0 < items);
        if (mine == 0) return false;
        const uint32_t at = (uint32_t)__ffsll((long long)mine) - 1;
        it.seq = at;
        it.s = PagedSeq{(uint32_t)__builtin_amdgcn_readlane(s.start, at), (uint32_t)__builtin_amdgcn_readlane(s.n, at), (uint32_t)__builtin_amdgcn_readlane(s.len, at)};
        it.pieces = __builtin_amdgcn_readlane(pieces, at);
        local = w - __builtin_amdgcn_readlane(items0, at);
        first_slot = __builtin_amdgcn_readlane(slots0, at);
    } else {
        constexpr uint32_t THREADS = WAVES * WAVE;
        __shared__ float s_work[WAVES];
        __shared__ uint32_t s_scan[2][WAVES], s_found[4];
        float per_step = 0.f;
        if (tid == 0) s_found[0] = 0xffffffffu;
        if (p.slots) {
            float work = 0.f;
            for (uint32_t i = tid; i < p.b.nseq; i += THREADS) {
                const PagedSeq s = paged_seq(p.b, i);
                work += (float)paged_tiles<ROWS>(p, s) * paged_weight(p, s);
            }
            work = wave_sum_dpp(work);
            if (lane == 0) s_work[wave] = work;
        }
        __syncthreads();
        if (p.slots) {
            float work = 0.f;
#pragma unroll
            for (int v = 0; v < WAVES; ++v) work += s_work[v];
            per_step = paged_per_step<ROWS>(p, work);
        }
        uint32_t items0 = 0, slots0 = 0;
        for (uint32_t i0 = 0; i0 < p.b.nseq; i0 += THREADS) {
            uint32_t items = 0, slots = 0, pieces = 1;
            if (i0 + tid < p.b.nseq) {
                const PagedSeq s = paged_seq(p.b, i0 + tid);
                pieces = paged_pieces<ROWS>(p, s, per_step);
                items = paged_tiles<ROWS>(p, s) * p.nkvh * pieces;
                slots = pieces > 1 ? items : 0;
            }
            uint32_t a = items, b = slots;
#pragma unroll
            for (int o = 1; o < WAVE; o <<= 1) {
                const uint32_t ua = __shfl_up(a, o, WAVE), ub = __shfl_up(b, o, WAVE);
                if (lane >= (uint32_t)o) a += ua, b += ub;
            }
            if (lane == WAVE - 1) s_scan[0][wave] = a, s_scan[1][wave] = b;
            __syncthreads();
            uint32_t ta = 0, tb = 0;
#pragma unroll
            for (uint32_t v = 0; v < WAVES; ++v) {
                if (v < wave) a += s_scan[0][v], b += s_scan[1][v];
                ta += s_scan[0][v], tb += s_scan[1][v];
            }
            const uint32_t before = items0 + a - items;
            if (w - before < items) s_found[0] = i0 + tid, s_found[1] = w - before, s_found[2] = pieces, s_found[3] = slots0 + b - slots;
            items0 += ta, slots0 += tb;
            __syncthreads();
            if (w < items0 && w != 0) break;  // (workgroup 0 counts all slots)
        }
        if (w == 0 && tid == 0 && p.slots) *reinterpret_cast<uint32_t *>(p.work) = min(slots0, p.slots);
        if (s_found[0] == 0xffffffffu) return false;
        it.seq = __builtin_amdgcn_readfirstlane(s_found[0]);
        local = __builtin_amdgcn_readfirstlane(s_found[1]);
        it.pieces = __builtin_amdgcn_readfirstlane(s_found[2]);
        first_slot = __builtin_amdgcn_readfirstlane(s_found[3]);
        it.s = paged_seq(p.b, it.seq);
    }
    it.slot = first_slot + local;
    if (it.pieces > 1 && it.slot >= p.slots) return false;
    // kv heads next to each other (consecutive workgroups go to different XCDs, so a kv head's tiles meet in one L2), a
    // tile's ranges next, the tiles last to first: the last has the most keys under a causal mask
    it.kvh = local % p.nkvh;
    const uint32_t rest = local / p.nkvh, rows = it.s.n * p.group.d, back = rest / it.pieces, tiles = paged_tiles<ROWS>(p, it.s);
    it.piece = rest - back * it.pieces;
    it.row0 = (tiles - 1 - back) * ROWS;
    it.nrows = min((uint32_t)ROWS, rows - it.row0);
    if (it.pieces > 1 && tid == 0) {
        const uint32_t blind = p.causal && it.s.n > it.s.len ? it.s.n - it.s.len : 0;
        paged_desc(p)[it.slot] = PagedDesc{it.piece, it.pieces, it.kvh, it.row0, it.nrows, it.s.start, blind, 0};
    }
    return true;
}

// Keys that a row (of the sequence and kv head) keeps
__device__ __forceinline__ uint32_t paged_keep(const AttnPagedParams &p, const PagedItem &it, uint32_t token) {
    if (!p.causal) return it.s.len;
    const int64_t keep = (int64_t)it.s.len - it.s.n + token + 1;
    return keep < 0 ? 0 : (uint32_t)keep;
}
