// What the kernels over a paged cache share: reading the batch's description, and the rotation's angles.
//
// The description (page table, first token and length of each sequence) is device data that the host never sees, so the
// kernels bound every index they take from it: token ranges by the number of tokens, lengths by the table's width, page
// numbers by the number of pages.  Wrong data can give wrong results, not accesses outside the operands.
#pragma once
#include "device_util.h"

__device__ __forceinline__ uint32_t paged_u32(const void *base, int64_t offset) {
    return *reinterpret_cast<const uint32_t *>(reinterpret_cast<const char *>(base) + offset);
}

struct PagedSeq {
    uint32_t start, n, len;  // first token, new tokens, keys
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch &b, uint32_t s) {
    const uint32_t a = min(paged_u32(b.q_start, (int64_t)s * b.s_step), b.nt), e = min(paged_u32(b.q_start, (int64_t)(s + 1) * b.s_step), b.nt);
    // (the host checked that cols * page tokens fit 31 bits)
    return PagedSeq{a, e > a ? e - a : 0, min(paged_u32(b.kv_len, (int64_t)s * b.l_step), b.cols * b.page.d)};
}

// The sequence that token t belongs to, found by each wave for itself: as many as end at or before t come before it.
// nseq: it belongs to none.
__device__ __forceinline__ uint32_t paged_seq_of(const PagedBatch &b, uint32_t t) {
    const uint32_t lane = threadIdx.x % WAVE;
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < b.nseq; s0 += WAVE) {
        const bool ended = s0 + lane < b.nseq && paged_u32(b.q_start, (int64_t)(s0 + lane + 1) * b.s_step) <= t;
        before += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(ended));
    }
    return before;
}

// Page number of key `key` of sequence `seq` (key / page < cols)
__device__ __forceinline__ uint32_t paged_page(const PagedBatch &b, uint32_t seq, uint32_t column) {
    return paged_u32(b.table, (int64_t)seq * b.t_row + (int64_t)column * b.t_col);
}

// (sin, cos) of position * theta^(-k / half), theta^(-1 / half) = 2^-freq_step.  The angle is a product of up to 10^5 and
// more radians: in f32 it would be off by its 24th bit, hundredths of a radian.  It is taken in f64 and in turns
// (2 pi radians), reduced to half a turn either way, where f32 is exact to 2^-25 of a turn.
__device__ __forceinline__ double rope_turns(double freq_step, uint32_t k) {
    return exp2(-freq_step * (double)k) * 0.15915494309189533577;
}
__device__ __forceinline__ float2 rope_sin_cos(double pos, double turns_per_position) {
    const double turns = pos * turns_per_position;
    float2 sc;
    sincospif(2.0f * (float)(turns - rint(turns)), &sc.x, &sc.y);
    return sc;
}
__device__ __forceinline__ double rope_position(const void *pos, int64_t offset, uint32_t is_u64) {
    if (is_u64) return (double)*reinterpret_cast<const uint64_t *>(reinterpret_cast<const char *>(pos) + offset);
    return (double)paged_u32(pos, offset);
}
