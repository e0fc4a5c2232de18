// cbq_paged_append.cu -- keys and values of new tokens into a paged cache,
// with the per-head RMSNorm and the rotary embedding of queries and keys
// applied on the way (sm_100a).
//
// For the head vector x [D] of a token at position p, w the norm weight:
//   y_i = w_i x_i rsqrt(mean(x^2) + eps),  h = D / 2,
//   o_i = y_i cos[p, i] - y_{i+h} sin[p, i],  o_{i+h} = y_{i+h} cos[p, i+h] + y_i sin[p, i+h].
// All of it in fp32 with one rounding at the end, so the row in the cache is
// the fp32 result rounded once whatever the activation type.
#include <algorithm>

#include "cbq_paged.cuh"

namespace {

using namespace cbq;

struct AppendArgs {
    const void *q, *kn, *vn;
    int64_t qs, ks, vs;                // token strides, elements
    int hq;
    float eps;
    const float *qw, *kw, *cosT, *sinT;
    int64_t rope_len;
    void *q_out;
};

template <typename T> struct Vec16;    // 16 bytes of T as floats
template <> struct Vec16<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void ld(const float *p, float (&x)[4]) {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    }
    static __device__ __forceinline__ void st(float *p, const float (&x)[4]) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    }
};
template <> struct Vec16<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void ld(const __nv_bfloat16 *p, float (&x)[8]) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void st(__nv_bfloat16 *p, const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// One CTA per token.  LPH = D / (2 N) neighbouring lanes hold a head: lane l
// the elements [l N, l N + N) of each half, so a rotation pair sits in one
// lane, loads and stores are 16 bytes, and the sum of squares is a shuffle
// over LPH lanes.
template <typename T, int D>
__global__ void __launch_bounds__(512) k_paged_append(const PagedView pv, const AppendArgs a) {
    constexpr int N = Vec16<T>::N, LPH = D / (2 * N), H = D / 2;
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x;
    // the token's sequence, row, position and page
    int s = t, row;
    if (pv.cu) {
        s = warp_upper(pv.cu, pv.seqs, t);
        row = pv.lens[s] - pv.cu[s + 1] + t;
    } else {
        row = pv.lens[s] - 1;
    }
    int64_t pos = row;
    if (pv.groups) pos += pv.plens[warp_upper(pv.gs, pv.groups, s)];
    int page = -1;
    bool ok = row >= 0 && row < pv.cap && pos >= 0 && pos < a.rope_len;
    if (ok) {
        page = pv.table[s * pv.table_stride + (row >> pv.ps_shift)];
        ok = page >= 0 && page < pv.pages;
    }
    if (!ok && row >= 0 && threadIdx.x == 0) report(pv.status, CBQ_FLAG_CORRUPT, (uint32_t)t);
    const int line = row & ((1 << pv.ps_shift) - 1);
    const int64_t at = page * pv.page_stride + line * pv.row_stride;
    const int sub = threadIdx.x % LPH;
    const int heads = a.hq + 2 * pv.kv_heads;
    float c0[N], c1[N], s0[N], s1[N];
    if (ok) {
        const float *cr = a.cosT + pos * D + sub * N, *sr = a.sinT + pos * D + sub * N;
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 x0 = *reinterpret_cast<const float4 *>(cr + i), x1 = *reinterpret_cast<const float4 *>(cr + H + i);
            const float4 y0 = *reinterpret_cast<const float4 *>(sr + i), y1 = *reinterpret_cast<const float4 *>(sr + H + i);
            c0[i] = x0.x; c0[i + 1] = x0.y; c0[i + 2] = x0.z; c0[i + 3] = x0.w;
            c1[i] = x1.x; c1[i + 1] = x1.y; c1[i + 2] = x1.z; c1[i + 3] = x1.w;
            s0[i] = y0.x; s0[i + 1] = y0.y; s0[i + 2] = y0.z; s0[i + 3] = y0.w;
            s1[i] = y1.x; s1[i + 1] = y1.y; s1[i + 2] = y1.z; s1[i + 3] = y1.w;
        }
    }
    // every lane of a warp runs every pass, so the shuffles are whole
    for (int h0 = 0; h0 < heads; h0 += blockDim.x / LPH) {
        const int h = h0 + threadIdx.x / LPH;
        const bool live = h < heads;
        const int kind = h < a.hq ? 0 : (h < a.hq + pv.kv_heads ? 1 : 2);
        const int hh = kind == 0 ? h : (kind == 1 ? h - a.hq : h - a.hq - pv.kv_heads);
        float x0[N], x1[N];
        float ss = 0.f;
        if (live && ok) {
            const T *src = kind == 0 ? static_cast<const T *>(a.q) + t * a.qs
                                     : (kind == 1 ? static_cast<const T *>(a.kn) + t * a.ks
                                                  : static_cast<const T *>(a.vn) + t * a.vs);
            src += hh * D + sub * N;
            Vec16<T>::ld(src, x0);
            Vec16<T>::ld(src + H, x1);
#pragma unroll
            for (int i = 0; i < N; ++i) ss += x0[i] * x0[i] + x1[i] * x1[i];
        }
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (!live) continue;
        T *dst;
        if (kind == 0) {
            dst = static_cast<T *>(a.q_out) + ((int64_t)t * a.hq + hh) * D + sub * N;
            if (!ok) {
#pragma unroll
                for (int i = 0; i < N; ++i) x0[i] = 0.f;
                Vec16<T>::st(dst, x0);
                Vec16<T>::st(dst + H, x0);
                continue;
            }
        } else {
            if (!ok) continue;
            dst = const_cast<T *>(static_cast<const T *>(kind == 1 ? pv.k : pv.v)) + at + hh * pv.head_stride + sub * N;
        }
        if (kind != 2) {
            const float scale = a.eps >= 0.f ? rsqrtf(ss / (float)D + a.eps) : 1.f;
            const float *w = kind == 0 ? a.qw : a.kw;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float y0 = x0[i] * scale, y1 = x1[i] * scale;
                if (w && a.eps >= 0.f) {
                    y0 *= w[sub * N + i];
                    y1 *= w[H + sub * N + i];
                }
                x0[i] = y0 * c0[i] - y1 * s0[i];
                x1[i] = y1 * c1[i] + y0 * s1[i];
            }
        }
        Vec16<T>::st(dst, x0);
        Vec16<T>::st(dst + H, x1);
    }
}

template <typename T, int D>
int launch_append(const PagedView &pv, const AppendArgs &a, cudaStream_t s) {
    constexpr int LPH = D / (2 * Vec16<T>::N);
    const int lanes = (a.hq + 2 * pv.kv_heads) * LPH;
    const int threads = std::min(512, (lanes + 31) / 32 * 32);
    CBQ_CUDA_TRY(cbq_host::launch_pdl(k_paged_append<T, D>, dim3((unsigned)pv.tokens), dim3(threads), 0, s, pv, a));
    return CBQ_OK;
}

}  // namespace

extern "C" int cbq_paged_append_rope(const cbq_paged_cache *cache, const cbq_paged_batch *batch, int64_t tokens,
                                     const void *q_dev, int64_t q_stride, const void *k_dev, int64_t k_stride,
                                     const void *v_dev, int64_t v_stride, int64_t q_heads, float eps,
                                     const float *q_weight_dev, const float *k_weight_dev, const float *cos_dev,
                                     const float *sin_dev, int64_t rope_len, void *q_out_dev, void *stream) {
    PagedView pv;
    const int rc = cbq_host::paged_view(cache, batch, tokens, q_heads, &pv);
    if (rc != CBQ_OK) return rc;
    if (tokens == 0 || batch->seqs == 0) return tokens ? CBQ_ERR_ARG : CBQ_OK;
    if (!q_dev || !k_dev || !v_dev || !cos_dev || !sin_dev || !q_out_dev || rope_len < 0) return CBQ_ERR_ARG;
    const int64_t unit = cache->dtype == CBQ_BF16 ? 8 : 4, d = cache->head_dim;
    if (q_stride < q_heads * d || k_stride < cache->kv_heads * d || v_stride < cache->kv_heads * d || q_stride % unit ||
        k_stride % unit || v_stride % unit)
        return CBQ_ERR_ARG;
    for (const void *p : {q_dev, k_dev, v_dev, (const void *)cos_dev, (const void *)sin_dev, (const void *)q_out_dev})
        if (reinterpret_cast<uintptr_t>(p) & 15) return CBQ_ERR_ARG;
    const AppendArgs a{q_dev, k_dev, v_dev, q_stride, k_stride, v_stride, (int)q_heads, eps, q_weight_dev,
                       k_weight_dev, cos_dev, sin_dev, rope_len, q_out_dev};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (cache->dtype == CBQ_F32)
        return d == 64 ? launch_append<float, 64>(pv, a, s)
                       : (d == 128 ? launch_append<float, 128>(pv, a, s) : launch_append<float, 256>(pv, a, s));
    return d == 64 ? launch_append<__nv_bfloat16, 64>(pv, a, s)
                   : (d == 128 ? launch_append<__nv_bfloat16, 128>(pv, a, s)
                               : launch_append<__nv_bfloat16, 256>(pv, a, s));
}
