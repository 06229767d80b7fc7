// qk_norm_rope: y = rope(x / sqrt(mean(x^2) + epsilon) * w, p) for every head of q and of k, in one pass and one launch.
//
// A workgroup serves up to eight consecutive tokens, or one slice of one token's nh + nkh heads when there are few.  A row (one
// head) is 16 bytes in each of L consecutive lanes, so its sum of squares is a sum over L lanes and everything else stays
// in the lane: each byte is read once and written once, and what bounds the kernel is memory.  The tokens' sines and
// cosines are evaluated once into LDS, a pair of a token per thread, while the first rows travel (an evaluation is some fifty
// f64 instructions behind the load of a position), and four rows per thread are on their way at a time (one where a few tokens
// leave a thread no more).  8191 tokens of 40
// heads of 128 (168 MB moved), on one machine: 73 us with a token per workgroup, 59 with two, 49 with four, 45.5 with eight,
// 48 with sixteen; with non-temporal stores 41 (4.1 TB/s; a plain copy of 4 GiB 4.9), with the next rows requested before
// the present ones are worked on 40.4: not worth the registers.
#include "paged.h"

extern __shared__ float2 qk_sc[];  // [token][dh / 2] of (sin, cos)

__device__ __forceinline__ void qk_fill_table(const QkNormRopeParams &p, uint32_t token0, uint32_t tokens) {
    const uint32_t half = p.dh / 2;
    for (uint32_t e = threadIdx.x; e < tokens * half; e += WG_THREADS) {
        const uint32_t t = e / half;
        qk_sc[e] = rope_sin_cos(rope_position(p.pos, (int64_t)(token0 + t) * p.p_step, p.pos_is_u64), rope_turns(p.freq_step, e - t * half));
    }
    __syncthreads();
}

// Rows of whole 16-byte vectors, aligned; L = the power of two of lanes that holds one (lanes past dh idle)
// U: rows of a thread on their way at a time; NT: with the non-temporal hint on the stores
template <typename T, int L, int U, bool NT>
__device__ __forceinline__ void qk_norm_rope_vec(const QkNormRopeParams &p) {
    constexpr int E = 16 / sizeof(T), G = WG_THREADS / L;
    const uint32_t token0 = blockIdx.x * p.tokens_per_block, tokens = min(p.tokens_per_block, p.nt - token0), lane = threadIdx.x % L;
    const uint32_t heads = p.heads_per_block.d, h0 = blockIdx.y * heads, h1 = p.nh[0] + p.nh[1], rows = tokens * heads;
    const bool live = lane * E < p.dh;
    float w[2][E];
#pragma unroll
    for (int i = 0; i < E; ++i) w[0][i] = w[1][i] = 0.f;
    auto weights = [&]() {
        if (!live) return;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (p.nh[k] == 0) continue;
#pragma unroll
            for (int i = 0; i < E; ++i)
                w[k][i] = p.w_is_f32 ? reinterpret_cast<const float *>(p.w[k])[lane * E + i] : (float)reinterpret_cast<const T *>(p.w[k])[lane * E + i];
        }
    };
    bool first = true;
    for (uint32_t r0 = threadIdx.x / L; first || r0 < rows; r0 += U * G) {
        PackOf<T> x[U];
        uint32_t tok[U], which[U], head[U];
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t r = r0 + u * G;
            tok[u] = fastdiv(r, p.heads_per_block);
            const uint32_t h = h0 + r - tok[u] * heads;
            on[u] = live && r < rows && h < h1;
            which[u] = h >= p.nh[0];
            head[u] = which[u] ? h - p.nh[0] : h;
            x[u].u = u32x4{0, 0, 0, 0};
            if (on[u]) x[u].u = ld128(reinterpret_cast<const char *>(p.x[which[u]]) + (int64_t)(token0 + tok[u]) * p.x_st[which[u]] + (int64_t)head[u] * p.x_sh[which[u]] + 16 * lane);
        }
        if (first) {  // (the same for the whole workgroup)
            weights();
            if (p.rotate) qk_fill_table(p, token0, tokens);
            first = false;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[E], sum = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                f[i] = (float)x[u].e[i];
                sum += f[i] * f[i];
            }
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, WAVE);
            if (!on[u]) continue;
            const float r = rsqrtf(sum / (float)p.dh + p.epsilon);
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] *= r * (which[u] ? w[1][i] : w[0][i]);
            if (p.rotate) {
                const float2 *sc = qk_sc + tok[u] * (p.dh / 2) + lane * (E / 2);
#pragma unroll
                for (int i = 0; i < E / 2; ++i) {
                    const float a = f[2 * i], b = f[2 * i + 1];
                    f[2 * i] = a * sc[i].y - b * sc[i].x;
                    f[2 * i + 1] = a * sc[i].x + b * sc[i].y;
                }
            }
#pragma unroll
            for (int i = 0; i < E; ++i) x[u].e[i] = (T)f[i];
            char *dst = reinterpret_cast<char *>(p.y[which[u]]) + (int64_t)(token0 + tok[u]) * p.y_st[which[u]] + (int64_t)head[u] * p.y_sh[which[u]] + 16 * lane;
            if constexpr (NT) st128_nt(dst, x[u].u);
            else st128(dst, x[u].u);
        }
    }
}

// Any alignment and any even dh: a wave per row, a pair of elements per lane and step; the row is read twice
template <typename T>
__device__ __forceinline__ void qk_norm_rope_pairs(const QkNormRopeParams &p) {
    const uint32_t token = blockIdx.x, lane = threadIdx.x % WAVE;
    const uint32_t h0 = blockIdx.y * p.heads_per_block.d, h1 = min(h0 + p.heads_per_block.d, p.nh[0] + p.nh[1]);
    if (p.rotate) qk_fill_table(p, token, 1);
    for (uint32_t h = h0 + threadIdx.x / WAVE; h < h1; h += WG_THREADS / WAVE) {
        const uint32_t which = h >= p.nh[0], hh = which ? h - p.nh[0] : h;
        const T *x = reinterpret_cast<const T *>(reinterpret_cast<const char *>(p.x[which]) + (int64_t)token * p.x_st[which] + (int64_t)hh * p.x_sh[which]);
        T *y = reinterpret_cast<T *>(reinterpret_cast<char *>(p.y[which]) + (int64_t)token * p.y_st[which] + (int64_t)hh * p.y_sh[which]);
        float sum = 0.f;
        for (uint32_t k = lane; k < p.dh / 2; k += WAVE) {
            const float a = (float)x[2 * k], b = (float)x[2 * k + 1];
            sum += a * a + b * b;
        }
        const float r = rsqrtf(wave_sum(sum) / (float)p.dh + p.epsilon);
        for (uint32_t k = lane; k < p.dh / 2; k += WAVE) {
            float w0, w1;
            if (p.w_is_f32) w0 = reinterpret_cast<const float *>(p.w[which])[2 * k], w1 = reinterpret_cast<const float *>(p.w[which])[2 * k + 1];
            else w0 = (float)reinterpret_cast<const T *>(p.w[which])[2 * k], w1 = (float)reinterpret_cast<const T *>(p.w[which])[2 * k + 1];
            const float a = (float)x[2 * k] * (r * w0), b = (float)x[2 * k + 1] * (r * w1);
            const float2 sc = p.rotate ? qk_sc[k] : float2{0.f, 1.f};
            y[2 * k] = (T)(a * sc.y - b * sc.x);
            y[2 * k + 1] = (T)(a * sc.x + b * sc.y);
        }
    }
}

#define QK_NORM_ROPE_L(name, T, L)                                                                                                                       \
    extern "C" __global__ void __launch_bounds__(256) qk_norm_rope_##name##_l##L(QkNormRopeParams p) { qk_norm_rope_vec<T, L, 1, false>(p); }            \
    extern "C" __global__ void __launch_bounds__(256) qk_norm_rope_##name##_l##L##_multi(QkNormRopeParams p) { qk_norm_rope_vec<T, L, 4, false>(p); }    \
    extern "C" __global__ void __launch_bounds__(256) qk_norm_rope_##name##_l##L##_multi_nt(QkNormRopeParams p) { qk_norm_rope_vec<T, L, 4, true>(p); }
#define QK_NORM_ROPE(name, T)                                                                                                                     \
    QK_NORM_ROPE_L(name, T, 8)                                                                                                                    \
    QK_NORM_ROPE_L(name, T, 16)                                                                                                                   \
    QK_NORM_ROPE_L(name, T, 32)                                                                                                                   \
    QK_NORM_ROPE_L(name, T, 64)                                                                                                                   \
    extern "C" __global__ void __launch_bounds__(256) qk_norm_rope_##name##_pairs(QkNormRopeParams p) { qk_norm_rope_pairs<T>(p); }
QK_NORM_ROPE(f16, f16)
QK_NORM_ROPE(bf16, bf16)
QK_NORM_ROPE(f32, float)
