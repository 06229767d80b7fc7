// attention over a paged cache for what the matrix kernels (attention_paged.hip, attention_paged_f32.hip) do not take: few rows in
// f32, head dimensions other than theirs, elements that are not adjacent, addresses that are not 16-byte aligned.
//
// One workgroup per token and query head.  A wave takes U keys at a time, every WAVES-th such group, and requests all their
// elements at once (element e in lane e % 64), the page numbers one group ahead.  The U dot products are summed over the
// lanes together: each exchange halves the number of values a lane holds, until it holds one key's sum; the
// softmax's maximum is then taken, and its powers, once for every key and not in every lane.  The waves' maxima, sums
// and outputs are joined in LDS.  Every key is read once per query head and token, from the caches where it
// was read before; what bounds the kernel is instructions for many tokens and latency for few, which then get sixteen waves.
// f32, 32 heads over 8 of 128 columns: a decode step over 2048 keys 61 us, 32 of them over 2000 to 4000 keys 422 us (790 MB,
// 1.9 TB/s), 2048 tokens with rows off 16 bytes 5.3 ms (with one key at a time 839 us, 2.3 ms, 11.6 ms).
#include "paged.h"

// x[u], u < U: the sum over the wave of x[lane % U]
template <int U>
__device__ __forceinline__ float sum_of_each(float (&x)[U]) {
    const uint32_t lane = threadIdx.x % WAVE;
#pragma unroll
    for (int n = U, bit = 1; n > 1; n /= 2, bit *= 2)
#pragma unroll
        for (int i = 0; i < n / 2; ++i) {
            const float keep = lane & bit ? x[2 * i + 1] : x[2 * i], give = lane & bit ? x[2 * i] : x[2 * i + 1];
            x[i] = keep + __shfl_xor(give, bit, WAVE);
        }
    float sum = x[0];
#pragma unroll
    for (int o = U; o < WAVE; o *= 2) sum += __shfl_xor(sum, o, WAVE);
    return sum;
}

// N: elements of a head per lane
template <typename T, int N, int WAVES>
__device__ __forceinline__ void attn_paged_any(const AttnPagedParams &p) {
    constexpr int U = N == 1 ? 8 : 16 / N;
    __shared__ float s_m[WAVES], s_l[WAVES], s_o[WAVES][N * WAVE];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const uint32_t token = blockIdx.x, head = blockIdx.y, kvh = fastdiv(head, p.group);
    const uint32_t seq = paged_seq_of(p.b, token);
    if (seq >= p.b.nseq) return;
    const PagedSeq s = paged_seq(p.b, seq);
    if (token < s.start || token >= s.start + s.n) return;
    // keys that the token keeps
    uint32_t keep = s.len;
    if (p.causal) keep = (uint32_t)min((int64_t)keep, max((int64_t)0, (int64_t)s.len - s.n + (token - s.start) + 1));

    const char *qr = reinterpret_cast<const char *>(p.q) + (int64_t)head * p.q_sh + (int64_t)token * p.q_st;
    const char *kb = reinterpret_cast<const char *>(p.k) + (int64_t)kvh * p.k_sh, *vb = reinterpret_cast<const char *>(p.v) + (int64_t)kvh * p.v_sh;
    float q[N], acc[N];
    int64_t ke[N], ve[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t e = lane + WAVE * i;
        q[i] = e < p.dh ? (float)*reinterpret_cast<const T *>(qr + (int64_t)e * p.q_sd) : 0.f;
        ke[i] = e < p.dh ? (int64_t)e * p.k_sd : 0, ve[i] = e < p.dh ? (int64_t)e * p.v_sd : 0;  // (beyond dh: element 0, not used)
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    uint32_t page[U], line[U];
    auto look_up = [&](uint32_t key0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t key = min(key0 + u, keep - 1), col = fastdiv(key, p.b.page);
            line[u] = key - col * p.b.page.d;
            page[u] = paged_page(p.b, seq, col);
        }
    };
    if (wave * U < keep) look_up(wave * U);
    for (uint32_t key0 = wave * U; key0 < keep; key0 += WAVES * U) {
        T k[U][N], v[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t pg = min(page[u], p.b.npages - 1);
            const char *kr = kb + (int64_t)pg * p.k_sp + (int64_t)line[u] * p.k_sr, *vr = vb + (int64_t)pg * p.v_sp + (int64_t)line[u] * p.v_sr;
#pragma unroll
            for (int i = 0; i < N; ++i) k[u][i] = *reinterpret_cast<const T *>(kr + ke[i]), v[u][i] = *reinterpret_cast<const T *>(vr + ve[i]);
        }
        look_up(key0 + WAVES * U < keep ? key0 + WAVES * U : key0);
        float dot[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            dot[u] = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) dot[u] += lane + WAVE * i < p.dh ? q[i] * (float)k[u][i] : 0.f;
        }
        // the lane's key: key0 + lane % U
        const float sum = sum_of_each<U>(dot), x = key0 + lane % U < keep ? sum * p.scale : -INFINITY;
        float top = fmaxf(m, x);
#pragma unroll
        for (int o = 1; o < U; o *= 2) top = fmaxf(top, __shfl_xor(top, o, WAVE));
        // (keys of score -inf before any other: nothing yet, and nothing added)
        const float old = m == -INFINITY ? 0.f : expf(m - top), add = x == -INFINITY ? 0.f : expf(x - top);
        l = l * old + add;  // of the lane's keys: lanes that differ by a multiple of U have the same
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] *= old;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float w = __shfl(add, u, WAVE);
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] += key0 + u < keep ? w * (float)v[u][i] : 0.f;
        }
        m = top;
    }
#pragma unroll
    for (int o = 1; o < U; o *= 2) l += __shfl_xor(l, o, WAVE);
    if (lane == 0) s_m[wave] = m, s_l[wave] = l;
#pragma unroll
    for (int i = 0; i < N; ++i) s_o[wave][lane + WAVE * i] = acc[i];
    __syncthreads();
    float top = s_m[0];
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, s_m[w]);
    // (a wave without keys has a maximum of -inf, zeros beside it and no weight; one whose scores are all NaN has NaN beside it, which stays)
    const float ref = top == -INFINITY ? 0.f : top;
    float total = 0.f;
    for (int w = 0; w < WAVES; ++w) total += expf(s_m[w] - ref) * s_l[w];
    char *orow = reinterpret_cast<char *>(p.o) + (int64_t)head * p.o_sh + (int64_t)token * p.o_st;
    for (uint32_t e = threadIdx.x; e < p.dh; e += WAVES * WAVE) {
        float x = 0.f;
        for (int w = 0; w < WAVES; ++w) x += expf(s_m[w] - ref) * s_o[w][e];
        // a row that keeps no key is zero
        *reinterpret_cast<T *>(orow + (int64_t)e * p.o_sd) = (T)(keep ? x / total : 0.f);
    }
}

#define ATTN_ANY_N(name, T, N)                                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256) attn_paged_any_##name##_n##N(AttnPagedParams p) { attn_paged_any<T, N, 4>(p); }              \
    extern "C" __global__ void __launch_bounds__(1024) attn_paged_any_##name##_n##N##_w16(AttnPagedParams p) { attn_paged_any<T, N, 16>(p); }
#define ATTN_ANY(name, T) ATTN_ANY_N(name, T, 1) ATTN_ANY_N(name, T, 2) ATTN_ANY_N(name, T, 4) ATTN_ANY_N(name, T, 8)
ATTN_ANY(f16, f16)
ATTN_ANY(bf16, bf16)
ATTN_ANY(f32, float)
