// kv_append_paged: the new rows of k and v into a paged cache, k rotated on the way.
//
// Token i of a sequence with n new tokens and len keys is key len - n + i: row key % page of page table[key / page].  One
// workgroup per token finds the sequence (a ballot over the sequences' ends), evaluates the token's dh / 2 sines and
// cosines once into LDS for all heads, and moves the token's heads 16 bytes per thread and step: k and v are read once and
// written once, and nothing else of the cache is touched.  Memory bounds it: 8118 tokens of 32 heads of 128 (259 MB moved) take
// 52.8 us, 50.1 with non-temporal stores (5.2 TB/s; a plain copy of 4 GiB 4.9).  A few tokens are a chain of five loads, each
// waiting for the one before (starts, length, table, row): 3 us.
#include "paged.h"

extern __shared__ float2 append_sc[];  // dh / 2 entries of (sin, cos)

// Where the token's rows go: false when it belongs to no sequence, or its key has no column of the table, or its page is none of the
// cache's.  The key comes from the description as it stands: bounded by the table first, a length beyond it would move the
// last tokens over keys that are there.
__device__ __forceinline__ bool append_place(const KvAppendPagedParams &p, uint32_t token, uint32_t &page, uint32_t &row) {
    const uint32_t seq = paged_seq_of(p.b, token);
    if (seq >= p.b.nseq) return false;
    const uint32_t start = paged_u32(p.b.q_start, (int64_t)seq * p.b.s_step), end = paged_u32(p.b.q_start, (int64_t)(seq + 1) * p.b.s_step);
    const int64_t key = (int64_t)paged_u32(p.b.kv_len, (int64_t)seq * p.b.l_step) - end + token;  // len - (end - start) + (token - start)
    if (token < start || token >= end || key < 0 || key >= (int64_t)(p.b.cols * p.b.page.d)) return false;
    const uint32_t col = fastdiv((uint32_t)key, p.b.page);
    page = paged_page(p.b, seq, col);
    row = (uint32_t)key - col * p.b.page.d;
    return page < p.b.npages;
}

__device__ __forceinline__ void append_fill_table(const KvAppendPagedParams &p, uint32_t token) {
    const double pos = rope_position(p.pos, (int64_t)token * p.p_step, p.pos_is_u64);
    for (uint32_t k = threadIdx.x; k < p.dh / 2; k += WG_THREADS) append_sc[k] = rope_sin_cos(pos, rope_turns(p.freq_step, k));
    __syncthreads();
}

// elements adjacent, rows on 16-byte boundaries, whole 16-byte vectors (NT: with the non-temporal hint on the stores)
template <typename T, bool NT>
__device__ __forceinline__ void kv_append_vec(const KvAppendPagedParams &p) {
    constexpr int E = 16 / sizeof(T);
    const uint32_t token = blockIdx.x;
    uint32_t page = 0, row = 0;
    if (!append_place(p, token, page, row)) return;  // (the same for the whole workgroup)
    if (p.rotate) append_fill_table(p, token);
    const uint32_t per_head = p.dh / E, half = p.nkvh * per_head;
    auto store = [](char *dst, u32x4 v) {
        if constexpr (NT) st128_nt(dst, v);
        else st128(dst, v);
    };
    for (uint32_t v = threadIdx.x; v < 2 * half; v += WG_THREADS) {
        const bool is_v = v >= half;
        const uint32_t r = is_v ? v - half : v, h = r / per_head, c = r - h * per_head;
        PackOf<T> x;
        if (is_v) {
            x.u = ld128(reinterpret_cast<const char *>(p.v) + (int64_t)h * p.v_sh + (int64_t)token * p.v_st + 16 * c);
            store(reinterpret_cast<char *>(p.v_cache) + (int64_t)page * p.vc_sp + (int64_t)h * p.vc_sh + (int64_t)row * p.vc_sr + 16 * c, x.u);
        } else {
            x.u = ld128(reinterpret_cast<const char *>(p.k) + (int64_t)h * p.k_sh + (int64_t)token * p.k_st + 16 * c);
            if (p.rotate) {
#pragma unroll
                for (int i = 0; i < E / 2; ++i) {
                    const float2 sc = append_sc[c * (E / 2) + i];
                    const float a = (float)x.e[2 * i], b = (float)x.e[2 * i + 1];
                    x.e[2 * i] = (T)(a * sc.y - b * sc.x);
                    x.e[2 * i + 1] = (T)(a * sc.x + b * sc.y);
                }
            }
            store(reinterpret_cast<char *>(p.k_cache) + (int64_t)page * p.kc_sp + (int64_t)h * p.kc_sh + (int64_t)row * p.kc_sr + 16 * c, x.u);
        }
    }
}

// any strides: a pair of adjacent elements per thread and step (a last single one where dh is odd, without rotation)
template <typename T>
__device__ __forceinline__ void kv_append_pairs(const KvAppendPagedParams &p) {
    const uint32_t token = blockIdx.x;
    uint32_t page = 0, row = 0;
    if (!append_place(p, token, page, row)) return;
    if (p.rotate) append_fill_table(p, token);
    const uint32_t per_head = (p.dh + 1) / 2;
    for (uint32_t v = threadIdx.x; v < p.nkvh * per_head; v += WG_THREADS) {
        const uint32_t h = v / per_head, k = v - h * per_head;
        const bool two = 2 * k + 1 < p.dh;
        const char *ks = reinterpret_cast<const char *>(p.k) + (int64_t)h * p.k_sh + (int64_t)token * p.k_st + (int64_t)(2 * k) * p.k_sd;
        const char *vs = reinterpret_cast<const char *>(p.v) + (int64_t)h * p.v_sh + (int64_t)token * p.v_st + (int64_t)(2 * k) * p.v_sd;
        char *kd = reinterpret_cast<char *>(p.k_cache) + (int64_t)page * p.kc_sp + (int64_t)h * p.kc_sh + (int64_t)row * p.kc_sr + (int64_t)(2 * k) * p.kc_sd;
        char *vd = reinterpret_cast<char *>(p.v_cache) + (int64_t)page * p.vc_sp + (int64_t)h * p.vc_sh + (int64_t)row * p.vc_sr + (int64_t)(2 * k) * p.vc_sd;
        *reinterpret_cast<T *>(vd) = *reinterpret_cast<const T *>(vs);
        if (two) *reinterpret_cast<T *>(vd + p.vc_sd) = *reinterpret_cast<const T *>(vs + p.v_sd);
        T a = *reinterpret_cast<const T *>(ks), b = two ? *reinterpret_cast<const T *>(ks + p.k_sd) : a;
        if (p.rotate) {
            const float2 sc = append_sc[k];
            const float x = (float)a, y = (float)b;
            a = (T)(x * sc.y - y * sc.x);
            b = (T)(x * sc.x + y * sc.y);
        }
        *reinterpret_cast<T *>(kd) = a;
        if (two) *reinterpret_cast<T *>(kd + p.kc_sd) = b;
    }
}

#define KV_APPEND(name, T)                                                                                                                    \
    extern "C" __global__ void __launch_bounds__(256) kv_append_##name##_vec(KvAppendPagedParams p) { kv_append_vec<T, false>(p); }           \
    extern "C" __global__ void __launch_bounds__(256) kv_append_##name##_vec_nt(KvAppendPagedParams p) { kv_append_vec<T, true>(p); }         \
    extern "C" __global__ void __launch_bounds__(256) kv_append_##name##_pairs(KvAppendPagedParams p) { kv_append_pairs<T>(p); }
KV_APPEND(f16, f16)
KV_APPEND(bf16, bf16)
KV_APPEND(f32, float)
