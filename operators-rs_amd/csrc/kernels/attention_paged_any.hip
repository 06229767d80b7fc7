// attention over a paged cache for what the matrix kernels (attention_paged.hip) do not take: f32, head dimensions other
// than theirs, elements that are not adjacent, addresses that are not 16-byte aligned.
//
// One workgroup of four waves per token and query head.  A wave takes every fourth key: its lanes hold the elements of q
// (element e in lane e % 64), the dot product is a sum over the wave, and the wave keeps the running maximum, sum and
// output of the softmax; the four are joined in LDS.  Every key is read once per query head and token: this kernel is for
// being right wherever the others do not reach, not for speed.
#include "paged.h"

constexpr int PA_MAX = 512 / WAVE;  // elements of a head per lane

template <typename T>
__device__ __forceinline__ void attn_paged_any(const AttnPagedParams &p) {
    __shared__ float s_m[4], s_l[4], s_o[4][512];
    const uint32_t wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
    const uint32_t token = blockIdx.x, head = blockIdx.y, kvh = fastdiv(head, p.group);
    const uint32_t seq = paged_seq_of(p.b, token);
    if (seq >= p.b.nseq) return;
    const PagedSeq s = paged_seq(p.b, seq);
    if (token < s.start || token >= s.start + s.n) return;
    // keys that the token keeps
    int64_t keep = s.len;
    if (p.causal) keep = min(keep, max((int64_t)0, (int64_t)s.len - s.n + (token - s.start) + 1));

    const char *qr = reinterpret_cast<const char *>(p.q) + (int64_t)head * p.q_sh + (int64_t)token * p.q_st;
    const char *kb = reinterpret_cast<const char *>(p.k) + (int64_t)kvh * p.k_sh, *vb = reinterpret_cast<const char *>(p.v) + (int64_t)kvh * p.v_sh;
    float q[PA_MAX], acc[PA_MAX];
#pragma unroll
    for (int i = 0; i < PA_MAX; ++i) {
        const uint32_t e = lane + WAVE * i;
        q[i] = e < p.dh ? (float)*reinterpret_cast<const T *>(qr + (int64_t)e * p.q_sd) : 0.f;
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (uint32_t key = wave; key < keep; key += 4) {
        const uint32_t col = fastdiv(key, p.b.page), row = key - col * p.b.page.d;
        const uint32_t page = min(paged_page(p.b, seq, col), p.b.npages - 1);
        const char *kr = kb + (int64_t)page * p.k_sp + (int64_t)row * p.k_sr, *vr = vb + (int64_t)page * p.v_sp + (int64_t)row * p.v_sr;
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < PA_MAX; ++i) {
            const uint32_t e = lane + WAVE * i;
            if (e < p.dh) dot += q[i] * (float)*reinterpret_cast<const T *>(kr + (int64_t)e * p.k_sd);
        }
        const float x = wave_sum(dot) * p.scale, top = fmaxf(m, x);
        // (a key of score -inf before any other: nothing yet, and nothing added)
        const float old = m == -INFINITY ? 0.f : expf(m - top), add = x == -INFINITY ? 0.f : expf(x - top);
        l = l * old + add;
#pragma unroll
        for (int i = 0; i < PA_MAX; ++i) {
            const uint32_t e = lane + WAVE * i;
            if (e < p.dh) acc[i] = acc[i] * old + add * (float)*reinterpret_cast<const T *>(vr + (int64_t)e * p.v_sd);
        }
        m = top;
    }
    if (lane == 0) s_m[wave] = m, s_l[wave] = l;
#pragma unroll
    for (int i = 0; i < PA_MAX; ++i) s_o[wave][lane + WAVE * i] = acc[i];
    __syncthreads();
    float top = s_m[0];
    for (int w = 1; w < 4; ++w) top = fmaxf(top, s_m[w]);
    float f[4], total = 0.f;
    for (int w = 0; w < 4; ++w) {
        f[w] = s_m[w] == -INFINITY ? 0.f : expf(s_m[w] - top);
        total += f[w] * s_l[w];
    }
    char *orow = reinterpret_cast<char *>(p.o) + (int64_t)head * p.o_sh + (int64_t)token * p.o_st;
    for (uint32_t e = threadIdx.x; e < p.dh; e += WG_THREADS) {
        float x = 0.f;
        for (int w = 0; w < 4; ++w) x += f[w] * s_o[w][e];
        // a row that keeps no key is zero
        *reinterpret_cast<T *>(orow + (int64_t)e * p.o_sd) = (T)(keep ? x / total : 0.f);
    }
}

extern "C" __global__ void __launch_bounds__(256) attn_paged_any_f16(AttnPagedParams p) { attn_paged_any<f16>(p); }
extern "C" __global__ void __launch_bounds__(256) attn_paged_any_bf16(AttnPagedParams p) { attn_paged_any<bf16>(p); }
extern "C" __global__ void __launch_bounds__(256) attn_paged_any_f32(AttnPagedParams p) { attn_paged_any<float>(p); }
