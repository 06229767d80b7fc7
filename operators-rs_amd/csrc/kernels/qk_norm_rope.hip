// qk_norm_rope: y = rope(x / sqrt(mean(x^2) + epsilon) * w, p) for every head of q and of k, in one pass and one launch.
//
// A workgroup serves one token, or one slice of its nh + nkh heads: its sines and cosines are evaluated once into LDS
// while the first rows travel.  A row (one head) is 16 bytes in each of L consecutive lanes, so its sum of squares is a
// sum over L lanes and everything else stays in the lane: each byte is read once and written once.
#include "paged.h"

extern __shared__ float2 qk_sc[];  // dh / 2 entries of (sin, cos)

__device__ __forceinline__ void qk_fill_table(const QkNormRopeParams &p, uint32_t token) {
    const double pos = rope_position(p.pos, (int64_t)token * p.p_step, p.pos_is_u64);
    for (uint32_t k = threadIdx.x; k < p.dh / 2; k += WG_THREADS) qk_sc[k] = rope_sin_cos(pos, rope_turns(p.freq_step, k));
}

// Rows of whole 16-byte vectors, aligned; L = the power of two of lanes that holds one (lanes past dh idle)
template <typename T, int L>
__device__ __forceinline__ void qk_norm_rope_vec(const QkNormRopeParams &p) {
    constexpr int E = 16 / sizeof(T);
    const uint32_t token = blockIdx.x, lane = threadIdx.x % L;
    const uint32_t h0 = blockIdx.y * p.heads_per_block, h1 = min(h0 + p.heads_per_block, p.nh[0] + p.nh[1]);
    const bool live = lane * E < p.dh;
    if (p.rotate) {
        qk_fill_table(p, token);
        __syncthreads();
    }
    for (uint32_t h = h0 + threadIdx.x / L; h < h1; h += WG_THREADS / L) {
        const uint32_t which = h >= p.nh[0], hh = which ? h - p.nh[0] : h;
        PackOf<T> x;
        x.u = u32x4{0, 0, 0, 0};
        if (live) x.u = ld128(reinterpret_cast<const char *>(p.x[which]) + (int64_t)token * p.x_st[which] + (int64_t)hh * p.x_sh[which] + 16 * lane);
        float f[E], sum = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            f[i] = (float)x.e[i];
            sum += f[i] * f[i];
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, WAVE);
        const float r = rsqrtf(sum / (float)p.dh + p.epsilon);
        if (live) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const uint32_t e = lane * E + i;
                f[i] *= r * (p.w_is_f32 ? reinterpret_cast<const float *>(p.w[which])[e] : (float)reinterpret_cast<const T *>(p.w[which])[e]);
            }
            if (p.rotate) {
#pragma unroll
                for (int i = 0; i < E / 2; ++i) {
                    const float2 sc = qk_sc[lane * (E / 2) + i];
                    const float a = f[2 * i], b = f[2 * i + 1];
                    f[2 * i] = a * sc.y - b * sc.x;
                    f[2 * i + 1] = a * sc.x + b * sc.y;
                }
            }
#pragma unroll
            for (int i = 0; i < E; ++i) x.e[i] = (T)f[i];
            st128(reinterpret_cast<char *>(p.y[which]) + (int64_t)token * p.y_st[which] + (int64_t)hh * p.y_sh[which] + 16 * lane, x.u);
        }
    }
}

// Any alignment and any even dh: a wave per row, a pair of elements per lane and step; the row is read twice
template <typename T>
__device__ __forceinline__ void qk_norm_rope_pairs(const QkNormRopeParams &p) {
    const uint32_t token = blockIdx.x, lane = threadIdx.x % WAVE;
    const uint32_t h0 = blockIdx.y * p.heads_per_block, h1 = min(h0 + p.heads_per_block, p.nh[0] + p.nh[1]);
    if (p.rotate) {
        qk_fill_table(p, token);
        __syncthreads();
    }
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

#define QK_NORM_ROPE(name, T)                                                                                                        \
    extern "C" __global__ void __launch_bounds__(256) qk_norm_rope_##name##_l8(QkNormRopeParams p) { qk_norm_rope_vec<T, 8>(p); }    \
    extern "C" __global__ void __launch_bounds__(256) qk_norm_rope_##name##_l16(QkNormRopeParams p) { qk_norm_rope_vec<T, 16>(p); }  \
    extern "C" __global__ void __launch_bounds__(256) qk_norm_rope_##name##_l32(QkNormRopeParams p) { qk_norm_rope_vec<T, 32>(p); }  \
    extern "C" __global__ void __launch_bounds__(256) qk_norm_rope_##name##_l64(QkNormRopeParams p) { qk_norm_rope_vec<T, 64>(p); }  \
    extern "C" __global__ void __launch_bounds__(256) qk_norm_rope_##name##_pairs(QkNormRopeParams p) { qk_norm_rope_pairs<T>(p); }
QK_NORM_ROPE(f16, f16)
QK_NORM_ROPE(bf16, bf16)
QK_NORM_ROPE(f32, float)
