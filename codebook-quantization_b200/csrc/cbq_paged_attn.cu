// cbq_paged_attn.cu -- attention over a paged key/value cache: one new token
// per sequence with prefixes shared by groups of sequences (decode), and any
// number of new tokens per sequence, causally (extend) (sm_100a).
//
// For a query row q and its visible keys j: x_j = scale log2(e) q.k_j,
// m = max x_j, l = sum 2^(x_j - m), o = sum 2^(x_j - m) v_j / l.  A part of the
// keys gives (m, l, unnormalised o), both sums smaller by 2^kHead; parts join as
// M = max m, each l and o scaled by 2^(m - M) and added.  m, l and o are fp32 everywhere.
//
// k_paged_stream is the kernel for few query rows per kv head: the cache is
// read once and its bytes bound it.  A CTA whose part of the line (see
// cbq_paged_line.cuh) holds all of a unit writes the result; other units leave
// one (m, l, o) per part in the workspace, joined in part order: by the CTA that
// arrives last at a cut unit, or, where a prefix adds its parts to every unit,
// by k_join_rows.
#include <mutex>

#include "cbq_paged_line.cuh"

namespace {

using namespace cbq;

constexpr int kKeys = 16;              // keys of a stage (one warp's unit of loads); page_size is a multiple

// ---------------------------------------------------------------- small PTX
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// fp32 products on the tensor cores: each factor as the sum of two tf32 values
// (hi: rounded to 11 bits, lo: the rest, cut to as many by the instruction),
// x y = hi hi + hi lo + lo hi.  What is left out is 2^-21 of a product, against
// 2^-24 for an fp32 multiplication.
__device__ __forceinline__ uint32_t tf32_hi(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t tf32_lo(float x, uint32_t hi) { return __float_as_uint(x - __uint_as_float(hi)); }
__device__ __forceinline__ void mma1688(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// c += a b for NB right-hand sides given as (hi, lo) pairs of b0 and b1; the
// small terms go to a sum of their own (shorter chains of dependent products).
template <int NB>
__device__ __forceinline__ void mma_f32(float (*c)[4], float (*small)[4], const float (&a)[4], const uint32_t (*b)[4]) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = tf32_hi(a[i]);
        l[i] = tf32_lo(a[i], h[i]);
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        mma1688(small[nb], l, b[nb][0], b[nb][1]);
        mma1688(small[nb], h, b[nb][2], b[nb][3]);
        mma1688(c[nb], h, b[nb][0], b[nb][1]);
    }
}

// ------------------------------------------------------------ configuration
template <typename T, int D, int NB> struct StreamCfg {
    static constexpr bool kF32 = sizeof(T) == 4;
    static constexpr int R = 8 * NB;                                   // query rows of a unit
    static constexpr int NW = kF32 && D == 256 ? 2 : 4;                 // warps; a key tile is NW stages
    static constexpr int NT = 32 * NW;
    static constexpr int kRowB = D * (int)sizeof(T);
    static constexpr int kHalf = kKeys * kRowB;                         // K (or V) of a stage
    static constexpr int kStage = 2 * kHalf;
    static constexpr int S = kF32 ? (D == 64 ? 2 : 3) : (D == 64 ? 4 : (D == 256 && NB > 1 ? 2 : 3));   // ring stages of a warp
    static constexpr int kPitch = D + 4;                                // merge rows, padded against bank conflicts
    static constexpr int kMerge = NW * R * (kPitch + 2) * 4;
    static constexpr int kSmem = NW * S * kStage + kMerge;
    static constexpr int kSlot = R * D + 2 * R;                         // floats of a workspace slot
    static constexpr int kCtas = 2 * (kSmem + 1280) <= 228 * 1024 ? 2 : 1;   // an SM's, that registers are planned for
};

// Stages of a unit that any of its rows can see.
__device__ __forceinline__ int unit_stages(const Owner &w, int tt, const LineArgs &a) {
    const int np = (w.plen + kKeys - 1) / kKeys;
    if (a.mode == kPrefix) return np;
    return np + (own_limit(w, min((tt + 1) * a.geo.tq, w.nt) - 1) + kKeys - 1) / kKeys;
}

// A warp's share of a piece once more, row by row by fp32 FMAs on the cached
// values themselves.  The tf32 pair of an infinity, or of a value that rounds to
// one, is NaN or two infinities of opposite sign, and every product it enters
// comes out NaN: a warp that ends a piece with a NaN leaves what this finds
// instead (an infinity or a NaN that remains is the formula's).  Rare and slow;
// checking once a piece costs under 1 us
// a call (two prefixes 26 -> 27 us, 2000 new tokens 2.42 ms as before; a check of every
// product took 10 to 18 %).
struct ExactPiece {
    const float *q, *k, *v;            // of the unit's first row; of its kv head
    const int32_t *ptab, *otab;
    int64_t qs, page_stride, row_stride;
    int pages, ps_shift, plen, olen, np, st0, st1, step;   // stages st0, st0 + step, ..
    int tok0, nt, gb, nrows;
    bool own;                          // whether own rows count
    float sc;
    float *o, *m, *l;                  // of the warp, in shared memory
    int pitch;
};
template <int D> __device__ __noinline__ void exact_piece(const ExactPiece x) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int r = 0; r < x.nrows; ++r) {
        const int tk = r / x.gb;
        const float *q = x.q + tk * x.qs + (int64_t)(r - tk * x.gb) * D;
        const int lim = x.own ? clampi(x.olen - x.nt + x.tok0 + tk + 1, 0, x.olen) : 0;
        float m = -INFINITY, l = 0.f, o[D / 32];
#pragma unroll
        for (int e = 0; e < D / 32; ++e) o[e] = 0.f;
#pragma unroll 1
        for (int st = x.st0; st < x.st1; st += x.step) {
            const bool pre = st < x.np;
            const int key0 = (pre ? st : st - x.np) * kKeys, n = min((pre ? x.plen : lim) - key0, kKeys);
            if (n <= 0) continue;
            const int page = __ldg((pre ? x.ptab : x.otab) + (key0 >> x.ps_shift));
            const bool ok = page >= 0 && page < x.pages;               // else rows of zeros
            const int64_t off = (ok ? page : 0) * x.page_stride + (int64_t)(key0 & ((1 << x.ps_shift) - 1)) * x.row_stride;
            float s = -INFINITY;
            if (lane < n) {
                s = 0.f;
                const float *k = x.k + off + lane * x.row_stride;
#pragma unroll 1
                for (int d = 0; d < D && ok; ++d) s = fmaf(q[d], k[d], s);
                s *= x.sc;
            }
            float mx = s;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.f : mn, f = ex2(m - mu);
            const float w = lane < n ? ex2(s - (mu + kHead)) : 0.f;
            m = mn;
            l = l * f + warp_sum(w);
#pragma unroll
            for (int e = 0; e < D / 32; ++e) o[e] *= f;
#pragma unroll 1
            for (int j = 0; j < n && ok; ++j) {
                const float wj = __shfl_sync(0xffffffffu, w, j), *v = x.v + off + j * x.row_stride + lane;
#pragma unroll
                for (int e = 0; e < D / 32; ++e) o[e] = fmaf(wj, v[e * 32], o[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < D / 32; ++e) x.o[r * x.pitch + e * 32 + lane] = o[e];
        if (lane == 0) {
            x.m[r] = m;
            x.l[r] = l;
        }
    }
}

// One warp's 16 keys starting at `key0` of a table, into its slot: K then V,
// 16-byte chunks exchanged within groups of 8 by the row (no bank conflicts
// for the fragment reads).  Rows at or after `lim` are zero-filled, not read,
// so what they hold cannot reach a result.
template <typename T, int D>
__device__ __forceinline__ void load_stage(const PagedView &pv, int page, int key0, int lim, int h, uint32_t dst) {
    constexpr int kRowB = D * (int)sizeof(T), CH = kRowB / 16, kHalf = kKeys * kRowB;
    const int lane = threadIdx.x & 31;
    const bool ok = page >= 0 && page < pv.pages;
    const int64_t off = (ok ? page : 0) * pv.page_stride + h * pv.head_stride +
                        (int64_t)(key0 & ((1 << pv.ps_shift) - 1)) * pv.row_stride;
    const T *kb = static_cast<const T *>(pv.k) + off, *vb = static_cast<const T *>(pv.v) + off;
    const int valid = ok ? lim - key0 : 0;
#pragma unroll
    for (int i = 0; i < kKeys * CH / 32; ++i) {
        const int f = i * 32 + lane, r = f / CH, c = f % CH;
        const uint32_t d = dst + r * kRowB + ((c ^ (r & 7)) << 4);
        const bool in = r < valid;
        const int64_t so = in ? r * pv.row_stride + c * (16 / (int)sizeof(T)) : 0;
        cp_async16(d, kb + so, in);
        cp_async16(d + kHalf, vb + so, in);
    }
}

// All NT threads of a CTA join the parts of a cut unit of R rows.  Thread t
// holds D / 4 * R / NT float4 of the result; weights pass through shared
// memory in blocks of kWB parts.
constexpr int kWB = 32;
template <typename T, int D, int R, int NT, typename F>
__device__ __forceinline__ void join_unit(const LineArgs &a, const Cut &cut, int nrows, float *sm, F dst_row) {
    constexpr int SL = R * D + 2 * R, V = R * D / 4 / NT, TPR = NT / R;
    static_assert(V >= 1 && TPR >= 1 && (TPR & (TPR - 1)) == 0 && TPR <= 32, "a row's threads are lanes of one warp");
    const int tid = threadIdx.x;
    float *sW = sm, *sI = sm + kWB * R;                // [kWB][R] weights, [R] 1 / l
    // each row's maximum and sum: TPR lanes over its parts
    const int row = tid / TPR, sub = tid % TPR;
    float M = -INFINITY;
    for (int k = sub; k < cut.n; k += TPR) M = fmaxf(M, __ldcg(cut.slot(a, k, SL) + R * D + row));
#pragma unroll
    for (int d = TPR / 2; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    float L = 0.f;
    float4 y[V];
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < cut.n; k0 += kWB) {
        const int nk = min(kWB, cut.n - k0);
        __syncthreads();                               // the weights before
        for (int k = sub; k < nk; k += TPR) {
            const float *b = cut.slot(a, k0 + k, SL) + R * D + row;
            const float m = __ldcg(b), f = m == -INFINITY ? 0.f : ex2(m - M);
            L = fmaf(__ldcg(b + R), f, L);
            sW[k * R + row] = f;
        }
        __syncthreads();
#pragma unroll 4
        for (int k = 0; k < nk; ++k) {
            const float *b = cut.slot(a, k0 + k, SL);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int e = tid + v * NT, r = e / (D / 4);
                if (r >= nrows) continue;
                const float4 x = __ldcg(reinterpret_cast<const float4 *>(b) + e);
                const float f = sW[k * R + r];
                y[v].x = fmaf(x.x, f, y[v].x);
                y[v].y = fmaf(x.y, f, y[v].y);
                y[v].z = fmaf(x.z, f, y[v].z);
                y[v].w = fmaf(x.w, f, y[v].w);
            }
        }
    }
#pragma unroll
    for (int d = TPR / 2; d > 0; d >>= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
    if (sub == 0) sI[row] = L == 0.f ? 0.f : 1.f / L;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = tid + v * NT, r = e / (D / 4);
        if (r >= nrows) continue;
        const float inv = sI[r];
        st4(dst_row(r) + (e - r * (D / 4)) * 4, y[v].x * inv, y[v].y * inv, y[v].z * inv, y[v].w * inv);
    }
}

// The warp computes S^T = K Q^T and O^T = V^T P^T with the row-of-16 matrix
// instructions, keys (then dimensions of V) on the 16-row side and the query
// rows on the 8-column side, so 1..8 query rows waste none of the long side.
// bf16: m16n8k16; P^T turns into the second product's operand with two 8x8
// register transposes, rounded to bf16 like the values it multiplies, while l sums
// it unrounded: against 64 bits the results are off by 2.1e-3 where the rounding of
// an exact one takes 1.66e-3.  A second bf16 term brings that back to 1.66e-3, but
// a value of inf then meets terms of both signs; with those pieces worked out again
// (exact_piece) it costs 64 ragged sequences 169 -> 173 us, 16 of 4 new tokens 102
// -> 108, head_dim 256 86 -> 91.  fp32: m16n8k8 on tf32 pairs (see mma_f32), three
// products each: about 280 instructions for 16 keys and 8 rows where fp32 FMAs
// fed from shared memory took 950.
//
// Each warp copies its own 16 keys of a tile into its own ring (no barrier in the
// loop).  HBM bounds long sequences: 64 ragged ones of up to 8192 keys, 8 kv heads
// of 128 (960 MB), take 170 us = 5.7 TB/s, 0.88 of a copy's rate, with two CTAs an
// SM and 16 KB in flight per warp.  Short work is a chain of latencies: 1000 keys
// of one sequence (4 MB) take 10 us, of which the plan 2, the first loads 3, the
// tile 1, arrival and joining 3.
template <typename T, int D, int NB>
__global__ void __launch_bounds__(StreamCfg<T, D, NB>::NT, StreamCfg<T, D, NB>::kCtas)
    k_paged_stream(const PagedView pv, const LineArgs a) {
    using Cfg = StreamCfg<T, D, NB>;
    constexpr bool kF32 = Cfg::kF32;
    constexpr int R = Cfg::R, NW = Cfg::NW, NT = Cfg::NT, S = Cfg::S, kPitch = Cfg::kPitch;
    extern __shared__ __align__(128) uint8_t smem[];
    float *mO = reinterpret_cast<float *>(smem + NW * S * Cfg::kStage);  // [NW][R][kPitch]
    float *mM = mO + NW * R * kPitch, *mL = mM + NW * R;                 // [NW][R] each
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (a.wait_first) pdl_wait();
    pdl_launch_dependents();

    Cursor cons{};
    uint32_t w1 = 0, per = 1;
    __shared__ int last;
    __shared__ LineStart start;
    const Ends ends = token_ends(pv, a);
    const bool any = plan_line<NT>(pv, a, start, cons, w1, per);
    zero_rest<T, D>(pv, a, ends);
    if (any) {
        Cursor load = cons;
        Piece lp{};
        bool lgo = next_piece(load, pv, a, w1, lp);
        int lt = lp.tb;
        cons = load;                                   // the first piece is found once
        Piece p = lp;
        bool cgo = lgo;
        const uint32_t ring = smem_u32(smem) + warp * S * Cfg::kStage;
        // fills ring slot `slot` with this warp's next stage on the line, or with nothing
        auto issue = [&](int slot) {
            while (lgo && lt == lp.te) {
                lgo = next_piece(load, pv, a, w1, lp);
                lt = lp.tb;
            }
            if (lgo) {
                const int st = lt * NW + warp;
                if (st < unit_stages(load.ow, lp.tt, a)) {
                    const int np = (load.ow.plen + kKeys - 1) / kKeys;
                    const bool pre = st < np;
                    const int key0 = (pre ? st : st - np) * kKeys, lim = pre ? load.ow.plen : load.ow.olen;
                    const int32_t *tab = pre ? pv.ptable + load.ow.group * pv.ptable_stride
                                             : pv.table + load.o * pv.table_stride;
                    const int page = __ldg(tab + (key0 >> pv.ps_shift));
                    if (page < 0 || page >= pv.pages) {
                        if (lane == 0) report(pv.status, CBQ_FLAG_CORRUPT, (uint32_t)load.o);
                    }
                    load_stage<T, D>(pv, page, key0, lim, lp.h, ring + slot * Cfg::kStage);
                }
                ++lt;
            }
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < S - 1; ++i) issue(i);
        int it = 0;                                    // ring uses
        for (; cgo; cgo = next_piece(cons, pv, a, w1, p)) {
            const Owner &ow = cons.ow;
            const int np = (ow.plen + kKeys - 1) / kKeys, nst = unit_stages(ow, p.tt, a);
            // row r of the unit: token tok0 + r / gb, query head head0 + r % gb
            const int gb = min(a.geo.G, R), tok0 = p.tt * a.geo.tq;
            const int hleft = min(a.geo.G - p.hc * R, gb);            // heads of this chunk
            const int head0 = p.h * a.geo.G + p.hc * R;
            const int nrows = hleft < gb ? hleft : min(a.geo.tq, ow.nt - tok0) * gb;
            auto token = [&](int r) { return tok0 + r / gb; };
            auto row_at = [&](int r, int64_t stride) {
                const int tk = r / gb;
                return (int64_t)(ow.t0 + tok0 + tk) * stride + (int64_t)(head0 + r - tk * gb) * D;
            };
            auto q_row = [&](int r) { return static_cast<const T *>(a.q) + row_at(r, a.qs); };
            const int lim_first = a.mode == kPrefix ? 0 : own_limit(ow, tok0);
            {
                constexpr int KK = D / 16, KF = D / 8;   // steps of 16 (bf16) and 8 (fp32) dimensions
                const int rq = lane >> 2, cq = (lane & 3) * 2;
                // the query rows as the first product's right-hand side; fp32: the values, split at use
                uint32_t qf[NB][kF32 ? 1 : KK][2];
                float qv[NB][kF32 ? KF : 1][2];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const int r = nb * 8 + rq;
                    const T *qr = q_row(r < nrows ? r : 0);
                    if constexpr (kF32) {
#pragma unroll
                        for (int kk = 0; kk < KF; ++kk)
#pragma unroll
                            for (int e = 0; e < 2; ++e) qv[nb][kk][e] = r < nrows ? qr[kk * 8 + e * 4 + (lane & 3)] : 0.f;
                    } else
#pragma unroll
                    for (int kk = 0; kk < KK; ++kk) {
                        qf[nb][kk][0] = r < nrows ? *reinterpret_cast<const uint32_t *>(qr + kk * 16 + cq) : 0u;
                        qf[nb][kk][1] = r < nrows ? *reinterpret_cast<const uint32_t *>(qr + kk * 16 + 8 + cq) : 0u;
                    }
                }
                int lim[NB][2];                        // own rows visible to this thread's two query rows
                float m[NB][2], l[NB][2], o[NB][KK][4];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        lim[nb][e] = a.mode == kPrefix ? 0 : own_limit(ow, token(nb * 8 + cq + e));
                        m[nb][e] = -INFINITY;
                        l[nb][e] = 0.f;
#pragma unroll
                        for (int i = 0; i < KK; ++i) o[nb][i][e] = o[nb][i][e + 2] = 0.f;
                    }
                for (int t = p.tb; t < p.te; ++t, ++it) {
                    cp_wait<S - 2>();
                    __syncwarp();
                    issue((it + S - 1) % S);
                    const int st = t * NW + warp;
                    if (st >= nst) continue;
                    const uint32_t kb = ring + (it % S) * Cfg::kStage, vb = kb + Cfg::kHalf;
                    float s[NB][4];
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
                    if constexpr (kF32) {
                        // a 16-byte row of an 8x8 matrix of halves is 4 floats: the same load serves tf32
                        const int r = (lane & 7) + (lane & 8), cx = lane >> 4;
                        float part[3][NB][4] = {};     // odd steps; small terms of even and odd steps
#pragma unroll
                        for (int kk = 0; kk < KF; ++kk) {
                            uint32_t af[4], b[NB][4];
                            ldsm4(kb + r * Cfg::kRowB + (((kk * 2 + cx) ^ (r & 7)) << 4), af);
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    b[nb][e] = tf32_hi(qv[nb][kk][e]);
                                    b[nb][e + 2] = tf32_lo(qv[nb][kk][e], b[nb][e]);
                                }
                            const float av[4] = {__uint_as_float(af[0]), __uint_as_float(af[1]), __uint_as_float(af[2]),
                                                 __uint_as_float(af[3])};
                            mma_f32<NB>(kk & 1 ? part[0] : s, part[1 + (kk & 1)], av, b);
                        }
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                s[nb][e] = (s[nb][e] + part[0][nb][e]) + (part[1][nb][e] + part[2][nb][e]);
                    } else {
                        const int r = (lane & 7) + (lane & 8), cx = lane >> 4;
#pragma unroll
                        for (int kk = 0; kk < KK; ++kk) {
                            uint32_t af[4];
                            ldsm4(kb + r * Cfg::kRowB + (((kk * 2 + cx) ^ (r & 7)) << 4), af);
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) mma16816(s[nb], af, qf[nb][kk][0], qf[nb][kk][1]);
                        }
                    }
                    const bool pre = st < np;
                    const int key0 = (pre ? st : st - np) * kKeys;
                    const bool edge = key0 + kKeys > (pre ? ow.plen : lim_first);
                    const int ka = key0 + (lane >> 2), kc = ka + 8;
                    uint32_t pf[NB][2], pw[2][NB][4];        // P as the second product's right-hand side (fp32: by 8 keys)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        float pr[4];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x0 = s[nb][e] * a.sc, x1 = s[nb][e + 2] * a.sc;
                            if (edge) {
                                const int lm = pre ? ow.plen : lim[nb][e];
                                x0 = ka < lm ? x0 : -INFINITY;
                                x1 = kc < lm ? x1 : -INFINITY;
                            }
                            float mx = fmaxf(x0, x1);
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                            const float mn = fmaxf(m[nb][e], mx);
                            const float mu = mn == -INFINITY ? 0.f : mn;     // no key yet: 2^(-inf - 0) = 0
                            const float f = ex2(m[nb][e] - mu), mk = mu + kHead;
                            m[nb][e] = mn;
                            pr[e] = ex2(x0 - mk);
                            pr[e + 2] = ex2(x1 - mk);
                            l[nb][e] = l[nb][e] * f + (pr[e] + pr[e + 2]);
                            if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
                                for (int i = 0; i < KK; ++i) {
                                    o[nb][i][e] *= f;
                                    o[nb][i][e + 2] *= f;
                                }
                            }
                        }
                        if constexpr (kF32) {
                            // lane (row l / 4, key l % 4 and key + 4) from the lanes that hold the keys
                            const int src = (lane & 3) * 4 + (lane >> 3);
                            const bool odd = lane & 4;
#pragma unroll
                            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const float x0 = __shfl_sync(0xffffffffu, pr[ks * 2], src + e * 16);
                                    const float x1 = __shfl_sync(0xffffffffu, pr[ks * 2 + 1], src + e * 16);
                                    const float x = odd ? x1 : x0;
                                    pw[ks][nb][e] = tf32_hi(x);
                                    pw[ks][nb][e + 2] = tf32_lo(x, pw[ks][nb][e]);
                                }
                        } else {
                            pf[nb][0] = movm(pack_bf16(pr[0], pr[1]));
                            pf[nb][1] = movm(pack_bf16(pr[2], pr[3]));
                        }
                    }
                    if constexpr (kF32) {
                        const uint8_t *vs = smem + (warp * S + it % S) * Cfg::kStage + Cfg::kHalf;
#pragma unroll
                        for (int i = 0; i < KK; ++i) {
                            float c[NB][4], small[NB][4] = {};
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                                for (int e = 0; e < 4; ++e) c[nb][e] = o[nb][i][e];
#pragma unroll
                            for (int ks = 0; ks < 2; ++ks) {
                                float av[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int key = ks * 8 + (lane & 3) + (e >> 1) * 4, d = i * 16 + rq + (e & 1) * 8;
                                    av[e] = *reinterpret_cast<const float *>(vs + key * Cfg::kRowB +
                                                                             (((d >> 2) ^ (key & 7)) << 4) + (d & 3) * 4);
                                }
                                mma_f32<NB>(c, small, av, pw[ks]);
                            }
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[nb][i][e] = c[nb][e] + small[nb][e];
                        }
                    } else {
                        const int r = (lane & 7) + ((lane >> 4) << 3), cx = (lane >> 3) & 1;
#pragma unroll
                        for (int i = 0; i < KK; ++i) {
                            uint32_t af[4];
                            ldsm4t(vb + r * Cfg::kRowB + (((i * 2 + cx) ^ (r & 7)) << 4), af);
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) mma16816(o[nb][i], af, pf[nb][0], pf[nb][1]);
                        }
                    }
                }
                // this warp's (m, l, o) for the merge
                bool odd = false;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float ls = l[nb][e];
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, d);
                        const int r = nb * 8 + cq + e;
                        if (lane < 4) {
                            mM[warp * R + r] = m[nb][e];
                            mL[warp * R + r] = ls;
                        }
                        if constexpr (kF32) odd |= ls != ls;
                        float *dst = mO + (warp * R + r) * kPitch + rq;
#pragma unroll
                        for (int i = 0; i < KK; ++i) {
                            dst[i * 16] = o[nb][i][e];
                            dst[i * 16 + 8] = o[nb][i][e + 2];
                            if constexpr (kF32) odd |= o[nb][i][e] != o[nb][i][e] || o[nb][i][e + 2] != o[nb][i][e + 2];
                        }
                    }
                if constexpr (kF32) {
                    if (__builtin_expect(__any_sync(0xffffffffu, odd), 0)) {
                        ExactPiece x;
                        x.q = q_row(0);
                        x.k = static_cast<const float *>(pv.k) + p.h * pv.head_stride;
                        x.v = static_cast<const float *>(pv.v) + p.h * pv.head_stride;
                        x.ptab = pv.ptable + ow.group * pv.ptable_stride;
                        x.otab = pv.table + cons.o * pv.table_stride;
                        x.qs = a.qs; x.page_stride = pv.page_stride; x.row_stride = pv.row_stride;
                        x.pages = pv.pages; x.ps_shift = pv.ps_shift; x.plen = ow.plen; x.olen = ow.olen; x.np = np;
                        x.st0 = p.tb * NW + warp; x.st1 = min(p.te * NW, nst); x.step = NW;
                        x.tok0 = tok0; x.nt = ow.nt; x.gb = gb; x.nrows = nrows;
                        x.own = a.mode != kPrefix;
                        x.sc = a.sc;
                        x.o = mO + warp * R * kPitch; x.m = mM + warp * R; x.l = mL + warp * R;
                        x.pitch = kPitch;
                        __syncwarp();
                        exact_piece<D>(x);
                    }
                }
            }
            __syncthreads();
            // the NW warps' states joined in warp order; a whole unit is the
            // result, a part of one goes to its slot
            const bool whole = a.direct && p.tb == 0 && p.te == p.tiles;
            const int64_t slot = slot_of(cons, p, a, (int)blockIdx.x);
            float *ps = a.part + slot * Cfg::kSlot;
            for (int e = tid; e < nrows * (D / 4); e += NT) {
                const int r = e / (D / 4), d = (e - r * (D / 4)) * 4;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < NW; ++w) M = fmaxf(M, mM[w * R + r]);
                float L = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const float mw = mM[w * R + r];
                    const float f = mw == -INFINITY ? 0.f : ex2(mw - M);
                    const float4 v = *reinterpret_cast<const float4 *>(mO + (w * R + r) * kPitch + d);
                    L = fmaf(mL[w * R + r], f, L);
                    y[0] = fmaf(v.x, f, y[0]);
                    y[1] = fmaf(v.y, f, y[1]);
                    y[2] = fmaf(v.z, f, y[2]);
                    y[3] = fmaf(v.w, f, y[3]);
                }
                if (whole) {
                    const float inv = L == 0.f ? 0.f : 1.f / L;
                    st4(static_cast<T *>(a.out) + row_at(r, (int64_t)a.hq * D) + d, y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
                } else if (slot < a.slots) {
                    st4(ps + r * D + d, y[0], y[1], y[2], y[3]);
                    if (d == 0) {
                        ps[R * D + r] = M;
                        ps[R * D + R + r] = L;
                    }
                }
            }
            __syncthreads();
            if (a.direct && !whole) {
                // the CTA that arrives last at a cut unit joins its parts
                const Cut cut = cut_of(cons, p, per);
                if (tid == 0) {
                    __threadfence();
                    last = atomicAdd(a.count + cut.i0, 1u) == (uint32_t)(cut.n - 1);
                }
                __syncthreads();
                if (last) {
                    __threadfence();
                    join_unit<T, D, R, NT>(a, cut, nrows, mO, [&](int r) {
                        return static_cast<T *>(a.out) + row_at(r, (int64_t)a.hq * D);
                    });
                    if (tid == 0) a.count[cut.i0] = 0u;
                }
                __syncthreads();
            }
        }
        cp_wait<0>();
    }
    if (!a.wait_first) pdl_wait();                     // this kernel's end tells its successor that the previous one ended too
}

// ------------------------------------------------------------------- joining
// The parts of a line that a launch left.
struct JoinSource {
    const float *part;
    const uint64_t *cum;
    int64_t slots;
    int owners, grid, min_tiles, rows, tile_rows, mode;
    LineGeo geo;
};

// A query row's parts: the slot of the first one and the row's place in each.
struct Parts {
    const JoinSource *s;
    int64_t slot0;
    int n, row;

    __device__ __forceinline__ const float *slot(int k, int d) const {
        return s->part + (slot0 + k) * ((int64_t)s->rows * (d + 2));
    }
};

// Slot row of head gi of a unit's tl-th token (head chunk by head chunk where a token's heads are cut).
__device__ __forceinline__ int slot_row(const JoinSource &s, int tl, int gi) {
    if (s.tile_rows) {
        const int tb = s.tile_rows / s.geo.G;
        return tl / tb * s.tile_rows + tl % tb * s.geo.G + gi;
    }
    return s.geo.G <= s.rows ? tl * s.geo.G + gi : gi % s.rows;
}

// One warp joins one query row over two lists of parts.
template <typename T, int D>
__device__ __forceinline__ void join_row(const Parts &pa, const Parts &pb, T *dst) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31, n = pa.n + pb.n;
    auto stat = [&](int i, float &m, float &l) {
        const Parts &x = i < pa.n ? pa : pb;
        const float *b = x.slot(i < pa.n ? i : i - pa.n, D) + (int64_t)x.s->rows * D;
        m = __ldcg(b + x.row);
        l = __ldcg(b + x.s->rows + x.row);
    };
    float M = -INFINITY;
    for (int i0 = 0; i0 < n; i0 += 32) {
        float m = -INFINITY, l;
        if (i0 + lane < n) stat(i0 + lane, m, l);
        M = fmaxf(M, m);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    float L = 0.f, y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = 0.f;
    for (int i0 = 0; i0 < n; i0 += 32) {
        float m = -INFINITY, l = 0.f;
        if (i0 + lane < n) stat(i0 + lane, m, l);
        const float f = m == -INFINITY ? 0.f : ex2(m - M);
        L = fmaf(l, f, L);
        const int top = min(32, n - i0);
#pragma unroll 8
        for (int i = 0; i < top; ++i) {
            const float fi = __shfl_sync(0xffffffffu, f, i);
            const Parts &x = i0 + i < pa.n ? pa : pb;
            const float *b = x.slot(i0 + i < pa.n ? i0 + i : i0 + i - pa.n, D) + (int64_t)x.row * D + lane * E;
            if constexpr (E == 2) {
                const float2 v = __ldcg(reinterpret_cast<const float2 *>(b));
                y[0] = fmaf(v.x, fi, y[0]);
                y[1] = fmaf(v.y, fi, y[1]);
            } else {
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(b + e));
                    y[e] = fmaf(v.x, fi, y[e]);
                    y[e + 1] = fmaf(v.y, fi, y[e + 1]);
                    y[e + 2] = fmaf(v.z, fi, y[e + 2]);
                    y[e + 3] = fmaf(v.w, fi, y[e + 3]);
                }
            }
        }
    }
    L = warp_sum(L);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    if constexpr (E == 2) {
        dst[lane * 2] = from_f32<T>(y[0] * inv);
        dst[lane * 2 + 1] = from_f32<T>(y[1] * inv);
    } else {
#pragma unroll
        for (int e = 0; e < E; e += 4)
            st4(dst + lane * E + e, y[e] * inv, y[e + 1] * inv, y[e + 2] * inv, y[e + 3] * inv);
    }
}

// Where every unit left parts: those of the row of token tok, head (h, gi), of
// owner o; none where the token is not the owner's.
__device__ __forceinline__ Parts parts_of(const JoinSource &s, int o, const Owner &w, const OwnerTiles &t, int tok, int h,
                                          int gi) {
    Parts p{};
    p.s = &s;
    const uint64_t c0 = s.cum[o], all = s.cum[s.owners];
    const int tl = tok - w.t0, tt = tl / s.geo.tq;
    if (tl < 0 || tl >= w.nt) return p;
    const uint32_t per = tiles_per_cta((uint32_t)all, (uint32_t)s.grid, (uint32_t)s.min_tiles), tiles = t.of(tt);
    const int nhc = s.geo.hc, hc = nhc > 1 ? gi / s.rows : 0;
    const uint32_t u = (uint32_t)((h * t.tt + tt) * nhc + hc);
    const uint32_t w0 = (uint32_t)c0 + ((uint32_t)h * t.all() + t.before(tt)) * (uint32_t)nhc + (uint32_t)hc * tiles;
    const int i0 = (int)(w0 / per);
    p.slot0 = (int64_t)(c0 >> 32) + u + i0;
    p.n = (int)((w0 + tiles - 1) / per) - i0 + 1;
    p.row = slot_row(s, tl - tt * s.geo.tq, gi);
    if (p.slot0 + p.n > s.slots) p.n = 0;
    return p;
}

// One warp per (token, query head).
template <typename T, int D>
__global__ void __launch_bounds__(128) k_join_rows(const PagedView pv, const JoinSource own, const JoinSource pre, int hq,
                                                   void *out) {
    // lengths and tables were there before the launches that this one waits for (they let
    // it start after their own wait): the rows' owners are found meanwhile
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const bool in = row < (int64_t)pv.tokens * hq;
    const int t = in ? (int)(row / hq) : 0, x = in ? (int)(row - (int64_t)t * hq) : 0, h = x / own.geo.G, gi = x - h * own.geo.G;
    const int o = own.mode == kFull && pv.cu ? warp_upper(pv.cu, pv.seqs, t) : t;
    const Owner w = owner_of(pv, own.mode, o);
    const OwnerTiles tw = owner_tiles(w, own.geo, own.mode);
    int g = 0;
    Owner wg{};
    OwnerTiles tg{};
    if (pre.part) {
        g = warp_upper(pv.gs, pv.groups, t);
        wg = owner_of(pv, kPrefix, g);
        tg = owner_tiles(wg, pre.geo, kPrefix);
    }
    pdl_wait();
    pdl_launch_dependents();
    if (!in) return;
    const Parts po = parts_of(own, o, w, tw, t, h, gi);
    Parts pp{};
    if (pre.part) pp = parts_of(pre, g, wg, tg, t, h, gi);
    join_row<T, D>(pp, po, static_cast<T *>(out) + row * D);
}

// ---------------------------------------------------------------- host side

template <typename T, int D, int NB> int stream_grid(cbq_host::LinePlan *p) {
    using Cfg = StreamCfg<T, D, NB>;
    int n = 0;
    const int rc = cbq_host::resident_ctas(reinterpret_cast<const void *>(k_paged_stream<T, D, NB>), Cfg::NT, Cfg::kSmem, &n);
    if (rc != CBQ_OK) return rc;
    p->rows = Cfg::R;
    p->geo.keys = kKeys * Cfg::NW;
    p->grid = n * cbq_host::sm_count();
    return CBQ_OK;
}

template <typename T, int D, int NB>
int stream_launch(const PagedView &pv, const LineArgs &a, int grid, cudaStream_t s) {
    using Cfg = StreamCfg<T, D, NB>;
    CBQ_CUDA_TRY(cbq_host::launch_pdl(k_paged_stream<T, D, NB>, dim3((unsigned)grid), dim3(Cfg::NT), (size_t)Cfg::kSmem,
                                      s, pv, a));
    return CBQ_OK;
}

// f(type, head_dim, row blocks) for the instantiations that exist: fp32 takes
// 8 rows per unit; bf16 8, 16 or 32 (16 at head_dim 256, whose sums take the registers).
#define CBQ_STREAM_DISPATCH(dtype, d, nb, CALL)                                                    \
    if ((dtype) == CBQ_F32) {                                                                      \
        if ((d) == 64) { CALL(float, 64, 1); } else if ((d) == 128) { CALL(float, 128, 1); }         \
        else { CALL(float, 256, 1); }                                                              \
    } else if ((d) == 64) {                                                                        \
        if ((nb) == 1) { CALL(__nv_bfloat16, 64, 1); } else if ((nb) == 2) { CALL(__nv_bfloat16, 64, 2); } \
        else { CALL(__nv_bfloat16, 64, 4); }                                                       \
    } else if ((d) == 128) {                                                                       \
        if ((nb) == 1) { CALL(__nv_bfloat16, 128, 1); } else if ((nb) == 2) { CALL(__nv_bfloat16, 128, 2); } \
        else { CALL(__nv_bfloat16, 128, 4); }                                                      \
    } else {                                                                                       \
        if ((nb) == 1) { CALL(__nv_bfloat16, 256, 1); } else { CALL(__nv_bfloat16, 256, 2); }        \
    }

int row_blocks(int64_t rows) { return rows <= 8 ? 1 : (rows <= 16 ? 2 : 4); }

// Plan of a k_paged_stream launch whose owners have about `rows` query rows
// per kv head: as few blocks of 8 as hold them, at most 32.
int stream_plan(const PagedView &pv, int dtype, int d, int G, int64_t rows, int64_t off, cbq_host::LinePlan *p) {
    int rc = CBQ_OK;
#define CBQ_CALL(T, DD, NN) rc = stream_grid<T, DD, NN>(p)
    CBQ_STREAM_DISPATCH(dtype, d, row_blocks(rows), CBQ_CALL)
#undef CBQ_CALL
    if (rc != CBQ_OK) return rc;
    p->tile_rows = 0;
    p->geo.G = G;
    p->geo.tq = std::max(1, p->rows / G);
    p->geo.hc = (G + p->rows - 1) / p->rows;
    p->geo.join = 1;
    p->min_tiles = 1;
    return cbq_host::line_room(pv, d, off, p) ? CBQ_OK : CBQ_ERR_UNSUPPORTED;
}

// Query rows per kv head up to which k_paged_stream is the faster kernel (row /
// tile kernel, us, 1 to 8 heads a kv head, 2 to 8 kv heads).  Head_dim 128: 8 rows
// of 16 sequences on 4000 keys 63 / 70, of 64 on 2000 127 / 117 (46 / 51 with 4 kv
// heads); 12 rows 113 / 73 and 199 / 121.  Few units leave both kernels to cut the
// keys, and the tile kernel's longer chain shows: 16 rows of one sequence on 2000
// keys 13 / 21, on 20000 37 / 38, 24 rows 18 / 21 and 56 / 39; a prefix of 2000
// rows 24 / 25, of 16000 43 / 37 and (2 kv heads) 35 / 43.  Head_dim 64: 16 rows of 16
// sequences 53 / 53, of 64 103 / 103, 24 rows 73 / 60.
int stream_rows(int d, int64_t units) { return d == 128 && units > 16 ? 8 : 16; }

struct AttnPlan {
    PagedView pv;
    int dtype, d, G;
    bool extend, prefix, own_tile, pre_tile;           // *_tile: the tensor-core kernel takes that line
    cbq_host::LinePlan own, pre;
    int64_t bytes;
};

// The prefix's and the own rows' launches on SMs of their own, where both are
// short: one after the other each pays its launch, plan and first loads (32
// sequences on a prefix of 8192 rows: 50 us in turn, 39 side by side).  Long
// ones gain nothing and would wait for the slower of two guesses (256 of 1024 own
// rows on 32768: 260 in turn, 284 side by side), so they run in turn; so does fp32,
// whose products and not the bytes take the time.  The times are guessed from the
// lengths' bounds, own rows at half of theirs, at the rates measured on long ones.
// Of 36 shapes (4 to 256 sequences, 2 or 8 kv heads, head_dim 64 or 128) the guess
// takes the faster side for 30, loses 2 to 8 % on 5, and 27 % where 256 sequences
// own next to nothing (256 of 100 rows on 32768, 2 kv heads: 75 in turn, 95).
constexpr double kShareUs = 60.0;
void share_sms(const cbq_paged_cache *c, const cbq_paged_batch *b, int64_t group_rows, int sms, AttnPlan *p) {
    const double row = (double)c->kv_heads * c->head_dim * 4;
    const double keys = (double)b->groups * ((group_rows + p->pre.rows - 1) / p->pre.rows) * p->pv.pcap;   // once per row tile
    const double pre = p->pre_tile ? 1.2 * keys * c->kv_heads / p->pre.geo.keys / sms : keys * row / 4e6;
    const double own = 0.5 * (double)b->seqs * p->pv.cap * row / 5e6;
    if (p->dtype == CBQ_F32 || pre + own > kShareUs) return;
    const int mine = std::min(std::max((int)(sms * pre / (pre + own + 1e-9) + 0.5), sms / 12), sms - sms / 12);
    p->pre.grid = std::max(p->pre.grid / sms * mine, 1);
    p->own.grid = std::max(p->own.grid / sms * (sms - mine), 1);
}

int plan_attn(const cbq_paged_cache *c, const cbq_paged_batch *b, int64_t tokens, int64_t q_heads, bool extend,
              AttnPlan *p) {
    *p = AttnPlan{};
    const int rc = cbq_host::paged_view(c, b, tokens, q_heads, &p->pv);
    if (rc != CBQ_OK) return rc;
    if (b->seqs == 0 || tokens == 0) return CBQ_OK;
    if (!extend && tokens != b->seqs) return CBQ_ERR_ARG;
    p->dtype = (int)c->dtype;
    p->d = (int)c->head_dim;
    p->G = (int)(q_heads / c->kv_heads);
    p->extend = extend;
    // the lengths' bounds given by the caller, where they are tighter than the tables
    p->pv.cap = (int)std::min<int64_t>(p->pv.cap, b->max_kv_len);
    p->pv.pcap = (int)std::min<int64_t>(p->pv.pcap, b->groups ? b->max_prefix_len : 0);
    p->prefix = !extend && b->groups && p->pv.pcap > 0;
    const bool tile = cbq_host::tile_takes(c);
    // query rows that share a kv head's keys, on the mean of the owners
    const int64_t own_rows = extend ? (tokens * p->G + b->seqs - 1) / b->seqs : p->G;
    p->own.mode = extend ? kFull : kOwn;
    p->own_tile = tile && extend && own_rows > stream_rows(p->d, b->seqs * c->kv_heads);
    const int sms = cbq_host::sm_count();
    int64_t group_rows = 0;
    if (p->prefix) {
        group_rows = ((int64_t)b->seqs + b->groups - 1) / b->groups * p->G;
        p->pre_tile = tile && group_rows > stream_rows(p->d, b->groups * c->kv_heads);
    }
    p->own.direct = !p->prefix;
    if (p->own_tile) {
        // few units: each is cut into many parts, which k_join_rows joins with a warp for every row
        const bool two = own_rows > 128;
        const int64_t units = (tokens * p->G / (two ? 256 : 128) + b->seqs) * c->kv_heads;
        if (2 * units < sms) p->own.direct = 0;
    }
    int e = p->own_tile ? cbq_host::tile_plan(p->pv, p->d, p->G, kFull, own_rows > 128, cbq_host::kCountBytes, &p->own)
                        : stream_plan(p->pv, p->dtype, p->d, p->G, own_rows, cbq_host::kCountBytes, &p->own);
    if (e != CBQ_OK) return e;
    p->bytes = p->own.end;
    if (p->prefix) {
        p->pre.mode = kPrefix;
        p->pre.direct = 0;
        e = p->pre_tile ? cbq_host::tile_plan(p->pv, p->d, p->G, kPrefix, group_rows > 128, p->bytes, &p->pre)
                        : stream_plan(p->pv, p->dtype, p->d, p->G, group_rows, p->bytes, &p->pre);
        if (e != CBQ_OK) return e;
        p->bytes = p->pre.end;
        share_sms(c, b, group_rows, sms, p);
    }
    return CBQ_OK;
}

LineArgs line_args(const cbq_host::LinePlan &lp, LineArgs a, uint8_t *ws) {
    a.geo = lp.geo;
    a.mode = lp.mode;
    a.owners = lp.owners;
    a.slots = lp.slots;
    a.min_tiles = lp.min_tiles;
    a.direct = lp.direct;
    a.count = reinterpret_cast<uint32_t *>(ws);
    a.cum = reinterpret_cast<uint64_t *>(ws + lp.cum_off);
    a.part = reinterpret_cast<float *>(ws + lp.part_off);
    return a;
}

int run_line(const cbq_paged_cache *c, const AttnPlan &p, const cbq_host::LinePlan &lp, bool tile, const LineArgs &a,
             cudaStream_t s) {
    if (tile) return cbq_host::tile_launch(c, p.pv, lp, a, s);
#define CBQ_CALL(T, DD, NN) return stream_launch<T, DD, NN>(p.pv, a, lp.grid, s)
    CBQ_STREAM_DISPATCH(p.dtype, p.d, lp.rows / 8, CBQ_CALL)
#undef CBQ_CALL
}

template <typename T, int D>
int join_launch(const AttnPlan &p, const LineArgs &own, const JoinSource &so, const JoinSource &sp, cudaStream_t s) {
    const int64_t blocks = ((int64_t)p.pv.tokens * own.hq + 3) / 4;
    CBQ_CUDA_TRY(cbq_host::launch_pdl(k_join_rows<T, D>, dim3((unsigned)blocks), dim3(128), 0, s, p.pv, so, sp, own.hq,
                                      own.out));
    return CBQ_OK;
}

// Held over a call's launches: they pass parts to one another through the
// workspace, which another thread's call on the same stream may share, and in
// stream order that call must come before all of them or behind.
std::mutex &launch_mutex(cudaStream_t s) {
    static std::mutex mu[64];
    const uintptr_t h = reinterpret_cast<uintptr_t>(s);
    return mu[(h ^ h >> 6 ^ h >> 12) & 63];
}

int paged_attn(const cbq_paged_cache *c, const cbq_paged_batch *b, int64_t tokens, const void *q, int64_t q_stride,
               int64_t q_heads, float scale, void *out, void *ws, int64_t ws_bytes, bool extend, cudaStream_t s) {
    AttnPlan p;
    int rc = plan_attn(c, b, tokens, q_heads, extend, &p);
    if (rc != CBQ_OK) return rc;
    if (tokens == 0) return CBQ_OK;
    if (b->seqs == 0) return CBQ_ERR_ARG;
    const int64_t unit = c->dtype == CBQ_BF16 ? 8 : 4;
    if (!q || !out || !ws || ws_bytes < p.bytes || q_stride < q_heads * c->head_dim || q_stride % unit) return CBQ_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(out) & 31) ||
        (reinterpret_cast<uintptr_t>(ws) & 255))
        return CBQ_ERR_ARG;
    uint8_t *w = static_cast<uint8_t *>(ws);
    LineArgs a{};
    a.q = q;
    a.qs = q_stride;
    a.hq = (int)q_heads;
    a.sc = scale * kLog2e;
    a.out = out;
    a.wait_first = 1;
    auto source = [&](const cbq_host::LinePlan &lp) {
        return JoinSource{reinterpret_cast<const float *>(w + lp.part_off),
                          reinterpret_cast<const uint64_t *>(w + lp.cum_off), lp.slots, lp.owners, lp.grid, lp.min_tiles,
                          lp.rows, lp.tile_rows, lp.mode, lp.geo};
    };
    std::lock_guard<std::mutex> guard(launch_mutex(s));
    if (p.prefix) {
        if ((rc = run_line(c, p, p.pre, p.pre_tile, line_args(p.pre, a, w), s)) != CBQ_OK) return rc;
        a.wait_first = 0;                              // the prefix launch passed its wait before this one can start
    }
    const LineArgs own = line_args(p.own, a, w);
    if ((rc = run_line(c, p, p.own, p.own_tile, own, s)) != CBQ_OK) return rc;
    if (p.own.direct) return CBQ_OK;
    const JoinSource so = source(p.own), sp = p.prefix ? source(p.pre) : JoinSource{};
    if (p.dtype == CBQ_F32)
        return p.d == 64 ? join_launch<float, 64>(p, own, so, sp, s)
                         : (p.d == 128 ? join_launch<float, 128>(p, own, so, sp, s)
                                       : join_launch<float, 256>(p, own, so, sp, s));
    return p.d == 64 ? join_launch<__nv_bfloat16, 64>(p, own, so, sp, s)
                     : (p.d == 128 ? join_launch<__nv_bfloat16, 128>(p, own, so, sp, s)
                                   : join_launch<__nv_bfloat16, 256>(p, own, so, sp, s));
}

}  // namespace

namespace cbq_host {

int resident_ctas(const void *kern, int threads, int smem, int *out) {
    static std::mutex mu;
    struct Entry { const void *kern; int dev, n; };
    static Entry seen[256];
    static int nseen = 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return CBQ_ERR_CUDA;
    std::lock_guard<std::mutex> g(mu);
    for (int i = 0; i < nseen; ++i)
        if (seen[i].kern == kern && seen[i].dev == dev) {
            *out = seen[i].n;
            return CBQ_OK;
        }
    CBQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    int n = 0;
    CBQ_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem));
    if (n < 1) return CBQ_ERR_UNSUPPORTED;
    if (nseen < 256) seen[nseen++] = Entry{kern, dev, n};
    *out = n;
    return CBQ_OK;
}

}  // namespace cbq_host

extern "C" int64_t cbq_paged_attn_workspace_bytes(const cbq_paged_cache *cache, const cbq_paged_batch *batch,
                                                  int64_t tokens, int64_t q_heads, int extend) {
    AttnPlan p;
    if (plan_attn(cache, batch, tokens, q_heads, extend != 0, &p) != CBQ_OK) return -1;
    return p.bytes;
}

extern "C" int cbq_paged_attn_decode(const cbq_paged_cache *cache, const cbq_paged_batch *batch, int64_t tokens,
                                     const void *q_dev, int64_t q_stride, int64_t q_heads, float scale, void *out_dev,
                                     void *workspace_dev, int64_t workspace_bytes, void *stream) {
    return paged_attn(cache, batch, tokens, q_dev, q_stride, q_heads, scale, out_dev, workspace_dev, workspace_bytes,
                      false, static_cast<cudaStream_t>(stream));
}

extern "C" int cbq_paged_attn_extend(const cbq_paged_cache *cache, const cbq_paged_batch *batch, int64_t tokens,
                                     const void *q_dev, int64_t q_stride, int64_t q_heads, float scale, void *out_dev,
                                     void *workspace_dev, int64_t workspace_bytes, void *stream) {
    return paged_attn(cache, batch, tokens, q_dev, q_stride, q_heads, scale, out_dev, workspace_dev, workspace_bytes,
                      true, static_cast<cudaStream_t>(stream));
}
