// attention over a paged cache in f32 on the matrix cores, for enough rows to fill the machine with tiles (the host chooses): o = softmax(scale q . k^T) . v,
// head dimensions of a multiple of 4 up to 256 (kernels for 64, 128 and 256 columns, the missing ones zero).
//
// A workgroup takes 64 rows of a sequence and kv head (row = token * group + head-in-group), 16 to each of its four waves, and
// walks the keys in tiles of 32 that go through registers into LDS, double-buffered, one barrier a tile.
//   S^T = K . Q^T (v_mfma 16x16x4 f32): the order of the contraction is free, so slot g of step 4 s + e is column 16 s + 4 g + e, and
//   a lane reads 16 bytes of its key for four steps.  Lane (j, g) of the result has query j and the keys 4 g + i of the 16,
//   which are, as they lie, the B operand of step i of
//   O^T = V^T . P^T.  Its rows are free as well: row r of block d is column 64 (d / 4) + 4 r + d % 4, so that a lane reads 16 bytes of
//   a value for four blocks, and stores 16 bytes of the result.
// The matrix cores bound it: 157 Tflop/s in f32, a sixteenth of what they do in f16.  2048 tokens, 32 heads over 8 of 128, causal,
// 34 Gflop kept: 396 us, 0.09 Pflop/s (a row at a time, attention_paged_any.hip, 5.3 ms); 512 tokens 59 us.  A tile's keys are
// not cut into ranges: 256 tokens over 8256 keys are 128 workgroups on 256 CUs, 839 us.
#include "paged_plan.h"

template <int DH>
struct F32Lds {
    static constexpr int BN = 32, PITCH = DH + 4;
    float k[2][BN * PITCH], v[2][BN * PITCH];
    uint32_t bad[4];  // by wave: values that are not finite, in a tile that some row keeps in part
};

// As paged_exactly in attention_paged.hip: row by row and key by key, where such values were met
template <int DH>
__device__ __forceinline__ void f32_exactly(const AttnPagedParams &p, const PagedItem &it) {
    constexpr int N = DH / WAVE;
    const uint32_t lane = threadIdx.x % WAVE;
    const char *kb = reinterpret_cast<const char *>(p.k) + (int64_t)it.kvh * p.k_sh, *vb = reinterpret_cast<const char *>(p.v) + (int64_t)it.kvh * p.v_sh;
    for (uint32_t r = threadIdx.x / WAVE; r < it.nrows; r += 4) {
        const uint32_t row = it.row0 + r, token = fastdiv(row, p.group), head = it.kvh * p.group.d + (row - token * p.group.d);
        const float *q = reinterpret_cast<const float *>(reinterpret_cast<const char *>(p.q) + (int64_t)head * p.q_sh + (int64_t)(it.s.start + token) * p.q_st);
        float *dst = reinterpret_cast<float *>(reinterpret_cast<char *>(p.o) + (int64_t)head * p.o_sh + (int64_t)(it.s.start + token) * p.o_st);
        const uint32_t keep = paged_keep(p, it, token);
        float m = -INFINITY, l = 0.f, o[N] = {};
        for (uint32_t key = 0; key < keep; ++key) {
            const uint32_t col = fastdiv(key, p.b.page), line = key - col * p.b.page.d, page = min(paged_page(p.b, it.seq, col), p.b.npages - 1);
            const float *kr = reinterpret_cast<const float *>(kb + (int64_t)page * p.k_sp + (int64_t)line * p.k_sr);
            const float *vr = reinterpret_cast<const float *>(vb + (int64_t)page * p.v_sp + (int64_t)line * p.v_sr);
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (lane + WAVE * i < p.dh) dot += q[lane + WAVE * i] * kr[lane + WAVE * i];
            const float x = wave_sum_dpp(dot) * p.scale, top = fmaxf(m, x);
            const float old = m == -INFINITY ? 0.f : expf(m - top), e = x == -INFINITY ? 0.f : expf(x - top);
            l = l * old + e;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (lane + WAVE * i < p.dh) o[i] = o[i] * old + e * vr[lane + WAVE * i];
            m = top;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lane + WAVE * i < p.dh) dst[lane + WAVE * i] = keep ? o[i] / l : 0.f;
    }
}

template <int DH>
__device__ __forceinline__ void attn_paged_f32(const AttnPagedParams &p) {
    constexpr int BN = F32Lds<DH>::BN, PITCH = F32Lds<DH>::PITCH;
    constexpr int CPR = DH / 4, RS = 256 / CPR, NCH = BN / RS;  // 16-byte chunks per row; rows of a pass of all threads; chunks per thread
    constexpr int QS = DH / 16, DB = DH / 16;                    // quads of q per lane, blocks of 16 columns
    __shared__ __attribute__((aligned(16))) F32Lds<DH> lds;
    PagedItem it;
    if (!paged_item<64, 4>(p, it)) return;
    const uint32_t tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE, j = lane % 16, g = lane / 16;
    const uint32_t wrow = 16 * wave, at = min(wrow + j, it.nrows - 1);
    const uint32_t row = it.row0 + at, token = fastdiv(row, p.group), head = it.kvh * p.group.d + (row - token * p.group.d);
    const uint32_t keys = paged_keep(p, it, fastdiv(it.row0 + it.nrows - 1, p.group)), tiles = (keys + BN - 1) / BN;
    const uint32_t keep_first = paged_keep(p, it, fastdiv(it.row0, p.group));  // the tile's first row keeps the fewest
    const uint32_t lim = paged_keep(p, it, token), lim_last = wrow < it.nrows ? paged_keep(p, it, fastdiv(it.row0 + min(wrow + 15, it.nrows - 1), p.group)) : 0;

    f32x4 q[QS];
    {
        const char *src = reinterpret_cast<const char *>(p.q) + (int64_t)head * p.q_sh + (int64_t)(it.s.start + token) * p.q_st + 16 * g;
#pragma unroll
        for (int s = 0; s < QS; ++s) q[s] = 16 * s + 4 * g < p.dh ? *reinterpret_cast<const f32x4 *>(src + 64 * s) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const uint32_t cc = tid % CPR, cr = tid / CPR;
    const bool live = 4 * cc < p.dh;
    const char *kb = reinterpret_cast<const char *>(p.k) + (int64_t)it.kvh * p.k_sh + 16 * cc;
    const char *vb = reinterpret_cast<const char *>(p.v) + (int64_t)it.kvh * p.v_sh + 16 * cc;
    uint32_t page[NCH], line[NCH];
    u32x4 kreg[NCH], vreg[NCH];
    auto look_up = [&](uint32_t t) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const uint32_t key = min(t * BN + cr + RS * i, it.s.len - 1), col = fastdiv(key, p.b.page);
            line[i] = key - col * p.b.page.d;
            page[i] = paged_page(p.b, it.seq, col);
        }
    };
    auto fetch = [&]() {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const uint32_t pg = min(page[i], p.b.npages - 1);
            kreg[i] = live ? ld128(kb + (int64_t)pg * p.k_sp + (int64_t)line[i] * p.k_sr) : u32x4{0, 0, 0, 0};
            vreg[i] = live ? ld128(vb + (int64_t)pg * p.v_sp + (int64_t)line[i] * p.v_sr) : u32x4{0, 0, 0, 0};
        }
    };
    bool spoiled = false;
    auto commit = [&](int buf, uint32_t t) {
        if (t * BN + BN > keep_first) {  // some rows do not keep some keys
            bool bad = false;
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    if (t * BN + cr + RS * i >= it.s.len) vreg[i][d] = 0;  // (the last key again)
                    bad = bad || (vreg[i][d] & 0x7f800000u) == 0x7f800000u;
                }
            spoiled |= __builtin_amdgcn_ballot_w64(bad) != 0;
        }
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            st128(&lds.k[buf][(cr + RS * i) * PITCH + 4 * cc], kreg[i]);
            st128(&lds.v[buf][(cr + RS * i) * PITCH + 4 * cc], vreg[i]);
        }
    };
    const float scale2 = p.scale * 1.4426950408889634f;
    float m = -INFINITY, l = 0.f;
    f32x4 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};

    if (tiles) {
        look_up(0);
        fetch();
        commit(0, 0);
        if (1 < tiles) look_up(1);
    }
#pragma unroll
    for (int s = 0; s < QS; ++s) OPHIP_ARRIVED(q[s]);
    __syncthreads();
    for (uint32_t t = 0; t < tiles; ++t) {
        const int buf = t & 1;
        const bool more = t + 1 < tiles;
        if (more) {
            fetch();
            look_up(t + 2);
        }
        if (t * BN < lim_last) {
            const float *kt = lds.k[buf] + j * PITCH + 4 * g, *vt = lds.v[buf] + 4 * g * PITCH + 4 * j;
            f32x4 s[2] = {};
#pragma unroll
            for (int c = 0; c < QS; ++c) {
                const f32x4 a0 = *reinterpret_cast<const f32x4 *>(kt + 16 * c), a1 = *reinterpret_cast<const f32x4 *>(kt + 16 * PITCH + 16 * c);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(a0[e], q[c][e], s[0], 0, 0, 0);
                    s[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(a1[e], q[c][e], s[1], 0, 0, 0);
                }
            }
            float x[2][4], mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[c][i] = t * BN + 16 * c + 4 * g + i < lim ? s[c][i] * scale2 : -INFINITY;
                    mx = fmaxf(mx, x[c][i]);
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16, WAVE));
            mx = fmaxf(mx, __shfl_xor(mx, 32, WAVE));
            if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {
                const float now = fmaxf(m, mx), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - now);
                l *= f;
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] *= f;
                m = now;
            }
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[c][i] = __builtin_amdgcn_exp2f(x[c][i] - ref);
                    l += x[c][i];
                }
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int d = 0; d < DB; d += 4) {
                        const f32x4 a = *reinterpret_cast<const f32x4 *>(vt + (16 * c + i) * PITCH + 16 * d);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[d + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], x[c][i], o[d + e], 0, 0, 0);
                    }
        }
        if (more) commit(buf ^ 1, t + 1);
        __syncthreads();
    }
    if (lane == 0) lds.bad[wave] = spoiled;
    __syncthreads();
    if (lds.bad[0] | lds.bad[1] | lds.bad[2] | lds.bad[3]) return f32_exactly<DH>(p, it);
    l += __shfl_xor(l, 16, WAVE);
    l += __shfl_xor(l, 32, WAVE);
    if (wrow + j >= it.nrows) return;
    const float inv = lim ? 1.0f / l : 0.f;  // (no key: zeros; no score above -inf: 0 / 0)
    char *dst = reinterpret_cast<char *>(p.o) + (int64_t)head * p.o_sh + (int64_t)(it.s.start + token) * p.o_st + 64 * g;
#pragma unroll
    for (int d = 0; d < DB; d += 4)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (16 * d + 16 * g + 4 * i < p.dh)
                *reinterpret_cast<f32x4 *>(dst + 64 * d + 16 * i) = f32x4{o[d][i], o[d + 1][i], o[d + 2][i], o[d + 3][i]} * inv;
}

extern "C" __global__ void __launch_bounds__(256, 2) attn_paged_f32_d64(AttnPagedParams p) { attn_paged_f32<64>(p); }
extern "C" __global__ void __launch_bounds__(256, 2) attn_paged_f32_d128(AttnPagedParams p) { attn_paged_f32<128>(p); }
extern "C" __global__ void __launch_bounds__(256, 1) attn_paged_f32_d256(AttnPagedParams p) { attn_paged_f32<256>(p); }
