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

#include "cbq_paged_line.cuh"

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
    static __device__ __forceinline__ void get(const uint4 &v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y);
        x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 put(const float (&x)[4]) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
};
template <> struct Vec16<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4 &v, float (&x)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 put(const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// One CTA per token.  LPH = D / (2 N) neighbouring lanes hold a head: lane l
// the elements [l N, l N + N) of each half, so a rotation pair sits in one
// lane, loads and stores are 16 bytes, and the sum of squares is a shuffle
// over LPH lanes.  A thread takes kHeads heads at a time: their loads go out
// before the chain of small loads that finds the token's row and table entries,
// and the cos / sin values serve all of them.  HBM bounds it: 16384 tokens of 48
// heads of 128 (419 MB) take 84 us = 5.0 TB/s (147 us with one head a thread and
// the table chain first); one token 3.5 us, a launch and five dependent loads.
//
// Two shapes: 128 threads with 3 heads at a time, and 64 with 6, whose tables
// serve twice the heads and of which more fit an SM (bf16: 8 to 5, fp32: 10 to 7),
// but whose waves take longer.  The one whose waves add up to less is taken, a wave
// of the second counted as 1.25 of the first.  Measured with 4 + 2 to 64 + 16 heads
// of 64 to 256, in units of the first's time: one wave each 1.05 to 1.35; two waves to
// one (bf16 780 to 1100 tokens, fp32 1100 to 1470) 0.75 to 0.9 (fp32 heads of 128 and
// 256: 0.95 to 1.0); two each 1.0 to 1.27; 16384 tokens bf16 0.77 to 0.94, fp32 0.95 to
// 1.02.
template <typename T, int D, int kThreads, int kHeads>
__global__ void __launch_bounds__(kThreads) k_paged_append(const PagedView pv, const AppendArgs a) {
    constexpr int N = Vec16<T>::N, LPH = D / (2 * N), H = D / 2, HPP = kThreads / LPH;   // heads per pass
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x;
    const int sub = threadIdx.x % LPH, hd = threadIdx.x / LPH;
    const int heads = a.hq + 2 * pv.kv_heads;
    uint4 raw[kHeads][2];
    auto fetch = [&](int h0) {
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const int h = h0 + i * HPP + hd;
            if (h >= heads) continue;
            const T *src = h < a.hq ? static_cast<const T *>(a.q) + t * a.qs + h * D
                                    : (h < a.hq + pv.kv_heads ? static_cast<const T *>(a.kn) + t * a.ks + (h - a.hq) * D
                                                              : static_cast<const T *>(a.vn) + t * a.vs +
                                                                    (h - a.hq - pv.kv_heads) * D);
            raw[i][0] = __ldcs(reinterpret_cast<const uint4 *>(src + sub * N));
            raw[i][1] = __ldcs(reinterpret_cast<const uint4 *>(src + sub * N + H));
        }
    };
    fetch(0);
    // the token's sequence, row, position and page; a token outside cu[0] .. cu[seqs] - 1
    // (a captured step with fewer tokens than it was captured for) has no row
    int s = t, row;
    if (pv.cu) {
        s = warp_upper(pv.cu, pv.seqs, t);
        const int first = pv.cu[s], end = pv.cu[s + 1];
        row = t >= first && t < end ? pv.lens[s] - end + t : -1;
    } else {
        row = pv.lens[s] - 1;
    }
    int page = -1;
    bool ok = row >= 0 && row < pv.cap;
    if (ok) page = pv.table[s * pv.table_stride + (row >> pv.ps_shift)];
    int64_t pos = row;
    if (pv.groups) {
        const int g = warp_upper(pv.gs, pv.groups, s), plen = pv.plens[g];
        if (s >= pv.gs[g] && s < pv.gs[g + 1]) pos += plen;            // else in no group
    }
    ok = ok && pos >= 0 && pos < a.rope_len && page >= 0 && page < pv.pages;
    if (!ok && row >= 0 && threadIdx.x == 0) report(pv.status, CBQ_FLAG_CORRUPT, (uint32_t)t);
    const int line = row & ((1 << pv.ps_shift) - 1);
    const int64_t at = page * pv.page_stride + line * pv.row_stride;
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
    for (int h0 = 0; h0 < heads; h0 += kHeads * HPP) {
        if (h0) fetch(h0);
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const int h = h0 + i * HPP + hd;
            const bool live = h < heads;
            float x0[N], x1[N];
            Vec16<T>::get(raw[i][0], x0);
            Vec16<T>::get(raw[i][1], x1);
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < N; ++j) ss += x0[j] * x0[j] + x1[j] * x1[j];
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (!live) continue;
            const bool isq = h < a.hq, isv = h >= a.hq + pv.kv_heads;
            if (!ok && !isq) continue;
            T *dst = isq ? static_cast<T *>(a.q_out) + ((int64_t)t * a.hq + h) * D
                         : const_cast<T *>(static_cast<const T *>(isv ? pv.v : pv.k)) + at +
                               (h - a.hq - (isv ? pv.kv_heads : 0)) * pv.head_stride;
            uint4 *d0 = reinterpret_cast<uint4 *>(dst + sub * N), *d1 = reinterpret_cast<uint4 *>(dst + sub * N + H);
            if (!ok) {
                *d0 = *d1 = make_uint4(0u, 0u, 0u, 0u);
                continue;
            }
            if (isv) {
                *d0 = raw[i][0];
                *d1 = raw[i][1];
                continue;
            }
            const float scale = a.eps >= 0.f ? rsqrtf(ss / (float)D + a.eps) : 1.f;
            const float *w = a.eps >= 0.f ? (isq ? a.qw : a.kw) : nullptr;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float y0 = x0[j] * scale, y1 = x1[j] * scale;
                if (w) {
                    y0 *= w[sub * N + j];
                    y1 *= w[H + sub * N + j];
                }
                x0[j] = y0 * c0[j] - y1 * s0[j];
                x1[j] = y1 * c1[j] + y0 * s1[j];
            }
            *d0 = Vec16<T>::put(x0);
            *d1 = Vec16<T>::put(x1);
        }
    }
}

template <typename T, int D>
int launch_append(const PagedView &pv, const AppendArgs &a, cudaStream_t s) {
    const int64_t sms = cbq_host::sm_count();
    bool narrow = false;
    if (pv.tokens > sms) {                             // else one CTA an SM, whatever the shape
        int w = 0, n = 0, rc;
        if ((rc = cbq_host::resident_ctas(reinterpret_cast<const void *>(k_paged_append<T, D, 128, 3>), 128, 0, &w)) != CBQ_OK ||
            (rc = cbq_host::resident_ctas(reinterpret_cast<const void *>(k_paged_append<T, D, 64, 6>), 64, 0, &n)) != CBQ_OK)
            return rc;
        narrow = 5 * ((pv.tokens + n * sms - 1) / (n * sms)) < 4 * ((pv.tokens + w * sms - 1) / (w * sms));
    }
    if (!narrow)
        CBQ_CUDA_TRY(cbq_host::launch_pdl(k_paged_append<T, D, 128, 3>, dim3((unsigned)pv.tokens), dim3(128), 0, s, pv, a));
    else
        CBQ_CUDA_TRY(cbq_host::launch_pdl(k_paged_append<T, D, 64, 6>, dim3((unsigned)pv.tokens), dim3(64), 0, s, pv, a));
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
