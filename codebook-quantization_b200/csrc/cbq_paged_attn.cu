// cbq_paged_attn.cu -- attention over a paged key/value cache: one new token
// per sequence with prefixes shared by groups of sequences (decode), and any
// number of new tokens per sequence, causally (extend) (sm_100a).
//
// For a query row q and its visible keys j: x_j = scale log2(e) q.k_j,
// m = max x_j, l = sum 2^(x_j - m), o = sum 2^(x_j - m) v_j / l.  A part of the
// keys gives (m, l, unnormalised o); parts join as M = max m, each l and o
// scaled by 2^(m - M) and added.  m, l and o are fp32 everywhere.
//
// k_paged_stream is the kernel for few query rows per kv head: the cache is
// read once and its bytes bound it.  The work is one line of key tiles
// (owner, kv head, row tile, tile): an owner is a sequence (its own rows, or
// for extend its prefix and own rows) or a group (its prefix, the query rows of
// all its sequences).  The line is cut into equal parts, one per resident CTA,
// so ragged lengths balance by themselves and a single long sequence spreads
// over all SMs.  A CTA whose part holds all of a unit writes the result; other
// units leave one (m, l, o) per part in the workspace, joined in part order by
// k_paged_join.  All of it is found from the lengths on the device.
#include <algorithm>
#include <mutex>

#include "cbq_paged.cuh"

namespace {

using namespace cbq;

constexpr int kKeys = 16;              // keys of a stage (one warp's unit of loads); page_size is a multiple
constexpr float kLog2e = 1.4426950408889634f;

enum StreamMode : int {
    kOwn = 0,                          // owner = sequence, keys = its own rows (decode)
    kPrefix = 1,                       // owner = group, keys = its prefix, rows = all its sequences' (decode)
    kFull = 2,                         // owner = sequence, keys = prefix then own rows, causal (extend)
};

struct StreamArgs {
    const void *q;
    int64_t qs;                        // token stride, elements
    int hq, G;
    float sc;                          // scale * log2(e)
    void *out;
    float *part;                       // [slot][R * D + 2 * R] fp32: o, m, l
    uint64_t *cum;                     // [owners + 1] units << 32 | tiles before each owner (for k_paged_join)
    int64_t slots;                     // slots of `part` (starts that are not in order could name more)
    int owners;
    int mode;
    int direct;                        // whole units go to `out`
    int wait_first;                    // wait for the previous kernel before reading (else before the end only)
};

struct Owner {
    int t0, nt;                        // its query tokens
    int plen, olen;                    // prefix and own rows
    int group;
};

// Largest i in [0, n) with a[i] <= x (one thread).
__device__ __forceinline__ int upper(const int32_t *a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

__device__ __forceinline__ Owner owner_of(const PagedView &pv, int mode, int o) {
    Owner w{};
    w.group = -1;
    if (mode == kPrefix) {
        w.t0 = clampi(pv.gs[o], 0, pv.tokens);
        w.nt = clampi(pv.gs[o + 1], w.t0, pv.tokens) - w.t0;
        w.plen = clampi(pv.plens[o], 0, pv.pcap);
        w.group = o;
        return w;
    }
    if (pv.cu && mode == kFull) {
        w.t0 = clampi(pv.cu[o], 0, pv.tokens);
        w.nt = clampi(pv.cu[o + 1], w.t0, pv.tokens) - w.t0;
    } else {
        w.t0 = o;
        w.nt = 1;
    }
    w.olen = clampi(pv.lens[o], 0, pv.cap);
    if (mode == kFull && pv.groups) {
        w.group = upper(pv.gs, pv.groups, o);
        w.plen = clampi(pv.plens[w.group], 0, pv.pcap);
    }
    return w;
}

__device__ __forceinline__ int stages_of(const Owner &w) {
    return (w.plen + kKeys - 1) / kKeys + (w.olen + kKeys - 1) / kKeys;
}

// ---------------------------------------------------------------- small PTX
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
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
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
}
__device__ __forceinline__ void st4(float *p, float a, float b, float c, float d) {
    *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d);
}
__device__ __forceinline__ void st4(__nv_bfloat16 *p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(a, b), pack_bf16(c, d));
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
    static constexpr int S = D == 64 && !kF32 ? 4 : (D == 256 && !kF32 && NB > 1 ? 2 : 3);   // stages in flight per warp
    static constexpr int kPitch = D + 4;                                // merge rows, padded against bank conflicts
    static constexpr int kMerge = NW * R * (kPitch + 2) * 4;
    static constexpr int kQ = kF32 ? R * D * 4 : 0;
    static constexpr int kP = kF32 ? NW * kKeys * R * 4 : 0;
    static constexpr int kSmem = NW * S * kStage + kMerge + kQ + kP;
    static constexpr int kSlot = R * D + 2 * R;                         // floats of a workspace slot
};

// Position on the line of tiles: the unit it is in and where that ends.
struct Cursor {
    uint32_t w;                        // next tile
    uint32_t base;                     // first tile of owner o
    uint32_t ubase;                    // units before owner o
    int o, tiles, rts;                 // tiles of a unit, row tiles of owner o
    Owner ow;
};
struct Piece {
    int h, rt, tb, te;                 // unit (h, rt) of the cursor's owner, its tiles [tb, te)
};

template <int R, int NW>
__device__ __forceinline__ void cursor_owner(Cursor &c, const PagedView &pv, int mode, int G, int o) {
    c.o = o;
    c.ow = owner_of(pv, mode, o);
    c.tiles = (stages_of(c.ow) + NW - 1) / NW;
    c.rts = (c.ow.nt * G + R - 1) / R;
}

// The next piece of [.., w1); false at the end.  Leaves c.w behind it.
template <int R, int NW>
__device__ __forceinline__ bool next_piece(Cursor &c, const PagedView &pv, const StreamArgs &a, uint32_t w1, Piece &p) {
    if (c.w >= w1) return false;
    while (true) {
        const uint32_t units = (uint32_t)(pv.kv_heads * c.rts), n = units * (uint32_t)c.tiles;
        if (c.w < c.base + n) break;
        if (c.o + 1 >= a.owners) return false;
        c.base += n;
        c.ubase += units;
        cursor_owner<R, NW>(c, pv, a.mode, a.G, c.o + 1);
    }
    const uint32_t at = c.w - c.base, u = at / (uint32_t)c.tiles;
    p.h = (int)(u / (uint32_t)c.rts);
    p.rt = (int)(u - (uint32_t)p.h * c.rts);
    p.tb = (int)(at - u * (uint32_t)c.tiles);
    p.te = (int)min((uint32_t)c.tiles, p.tb + (w1 - c.w));
    c.w += (uint32_t)(p.te - p.tb);
    return true;
}

// Own rows visible to query row r of an owner (row r is token r / G).
__device__ __forceinline__ int own_limit(const Owner &w, int r, int G) {
    return clampi(w.olen - w.nt + r / G + 1, 0, w.olen);
}

// Stages of a unit that any of its rows can see.
template <int R>
__device__ __forceinline__ int unit_stages(const Owner &w, int rt, int G, int mode) {
    const int np = (w.plen + kKeys - 1) / kKeys;
    if (mode == kPrefix) return np;
    const int last = min(rt * R + R, w.nt * G) - 1;
    return np + (own_limit(w, last, G) + kKeys - 1) / kKeys;
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

// The tile line: total, this CTA's part [w0, w1) and the owner w0 falls into.
// CTA 0 leaves the sums before each owner in a.cum.
template <int R, int NW>
__device__ __forceinline__ bool plan_line(const PagedView &pv, const StreamArgs &a, Cursor &c, uint32_t &w1) {
    constexpr int NT = 32 * NW;
    __shared__ uint64_t red[NW];
    __shared__ uint64_t found_base;
    __shared__ int found;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto weight = [&](int o) -> uint64_t {
        if (o >= a.owners) return 0;
        const Owner w = owner_of(pv, a.mode, o);
        if (blockIdx.x == 0 && (a.mode == kPrefix ? pv.plens[o] > pv.pcap : pv.lens[o] > pv.cap))
            report(pv.status, CBQ_FLAG_CORRUPT, (uint32_t)o);
        const uint32_t units = (uint32_t)(pv.kv_heads * ((w.nt * a.G + R - 1) / R));
        return (uint64_t)units << 32 | units * (uint32_t)((stages_of(w) + NW - 1) / NW);
    };
    const uint64_t first = weight(tid);
    uint64_t sum = first;
    for (int o = tid + NT; o < a.owners; o += NT) sum += weight(o);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) red[warp] = sum;
    if (tid == 0) found = -1;
    __syncthreads();
    uint64_t total = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) total += red[i];
    const uint32_t W = (uint32_t)total;
    const uint32_t per = (W + gridDim.x - 1) / gridDim.x;
    const uint32_t w0 = min((uint64_t)per * blockIdx.x, (uint64_t)W);
    w1 = min(w0 + per, W);
    const bool writer = blockIdx.x == 0;
    if (writer && tid == 0) a.cum[a.owners] = total;
    if (w0 >= w1 && !writer) return false;
    uint64_t run = 0;
    for (int o0 = 0; o0 < a.owners; o0 += NT) {
        const int o = o0 + tid;
        const uint64_t x = o0 == 0 ? first : weight(o);
        uint64_t inc = x;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += y;
        }
        __syncthreads();                              // red[] of the previous use
        if (lane == 31) red[warp] = inc;
        __syncthreads();
        uint64_t before = run, all = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            if (i < warp) before += red[i];
            all += red[i];
        }
        const uint64_t ex = before + inc - x;
        if (writer && o < a.owners) a.cum[o] = ex;
        if (o < a.owners && (uint32_t)ex <= w0 && w0 < (uint32_t)ex + (uint32_t)x) {
            found = o;
            found_base = ex;
        }
        run += all;
        if (!writer && (uint32_t)run > w0) break;      // the owner is in this block of owners
    }
    __syncthreads();
    if (w0 >= w1 || found < 0) return false;
    c.w = w0;
    c.base = (uint32_t)found_base;
    c.ubase = (uint32_t)(found_base >> 32);
    cursor_owner<R, NW>(c, pv, a.mode, a.G, found);
    return true;
}

// bf16: the warp computes S^T = K Q^T and O^T = V^T P^T with m16n8k16, keys
// (then dimensions of V) on the 16-row side and the query rows on the 8-column
// side, so 1..8 query rows waste none of the long side; P^T turns into the
// second product's operand with two 8x8 register transposes.  fp32: lane l
// takes key l % 16 and half the 8 query rows for the scores, and D / 32
// dimensions of all rows for the sums; fp32 FMAs.
template <typename T, int D, int NB>
__global__ void __launch_bounds__(StreamCfg<T, D, NB>::NT) k_paged_stream(const PagedView pv, const StreamArgs a) {
    using Cfg = StreamCfg<T, D, NB>;
    constexpr bool kF32 = Cfg::kF32;
    constexpr int R = Cfg::R, NW = Cfg::NW, NT = Cfg::NT, S = Cfg::S, kPitch = Cfg::kPitch;
    extern __shared__ __align__(128) uint8_t smem[];
    float *mO = reinterpret_cast<float *>(smem + NW * S * Cfg::kStage);  // [NW][R][kPitch]
    float *mM = mO + NW * R * kPitch, *mL = mM + NW * R;                 // [NW][R] each
    float *sQ = mL + NW * R;                                             // fp32: [R][D]
    float *sP = sQ + (kF32 ? R * D : 0);                                 // fp32: [NW][16][R]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (a.wait_first) pdl_wait();
    pdl_launch_dependents();

    Cursor cons{};
    uint32_t w1 = 0;
    const bool any = plan_line<R, NW>(pv, a, cons, w1);
    if (any) {
        Cursor load = cons;
        Piece lp{};
        bool lgo = next_piece<R, NW>(load, pv, a, w1, lp);
        int lt = lp.tb;
        const uint32_t ring = smem_u32(smem) + warp * S * Cfg::kStage;
        // fills ring slot `slot` with this warp's next stage on the line, or with nothing
        auto issue = [&](int slot) {
            while (lgo && lt == lp.te) {
                lgo = next_piece<R, NW>(load, pv, a, w1, lp);
                lt = lp.tb;
            }
            if (lgo) {
                const int st = lt * NW + warp;
                if (st < unit_stages<R>(load.ow, lp.rt, a.G, a.mode)) {
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
        Piece p;
        while (next_piece<R, NW>(cons, pv, a, w1, p)) {
            const Owner &ow = cons.ow;
            const int r0 = p.rt * R, nrows = min(R, ow.nt * a.G - r0);
            const int np = (ow.plen + kKeys - 1) / kKeys, nst = unit_stages<R>(ow, p.rt, a.G, a.mode);
            // query row r: token t0 + (r0 + r) / G, head h G + (r0 + r) % G
            auto q_row = [&](int r) {
                const int x = r0 + r, tk = x / a.G;
                return static_cast<const T *>(a.q) + (int64_t)(ow.t0 + tk) * a.qs + (p.h * a.G + x - tk * a.G) * D;
            };
            const int lim_first = a.mode == kPrefix ? 0 : own_limit(ow, r0, a.G);
            if constexpr (!kF32) {
                constexpr int KK = D / 16;
                const int rq = lane >> 2, cq = (lane & 3) * 2;
                uint32_t qf[NB][KK][2];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const int r = nb * 8 + rq;
                    const T *qr = q_row(r < nrows ? r : 0);
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
                        lim[nb][e] = a.mode == kPrefix ? 0 : own_limit(ow, r0 + nb * 8 + cq + e, a.G);
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
                    {
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
                    uint32_t pf[NB][2];
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
                            const float f = ex2(m[nb][e] - mu);
                            m[nb][e] = mn;
                            pr[e] = ex2(x0 - mu);
                            pr[e + 2] = ex2(x1 - mu);
                            l[nb][e] = l[nb][e] * f + (pr[e] + pr[e + 2]);
                            if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
                                for (int i = 0; i < KK; ++i) {
                                    o[nb][i][e] *= f;
                                    o[nb][i][e + 2] *= f;
                                }
                            }
                        }
                        pf[nb][0] = movm(pack_bf16(pr[0], pr[1]));
                        pf[nb][1] = movm(pack_bf16(pr[2], pr[3]));
                    }
                    {
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
                        float *dst = mO + (warp * R + r) * kPitch + rq;
#pragma unroll
                        for (int i = 0; i < KK; ++i) {
                            dst[i * 16] = o[nb][i][e];
                            dst[i * 16 + 8] = o[nb][i][e + 2];
                        }
                    }
            } else {
                constexpr int NC = D / 4, E = D / 32;   // 16-byte chunks of a row; dimensions per lane
                constexpr int EV = E < 4 ? E : 4;       // contiguous dimensions per load
                for (int e = tid; e < R * NC; e += NT) {
                    const int r = e / NC, c = e - r * NC;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (r < nrows) v = *reinterpret_cast<const float4 *>(q_row(r) + c * 4);
                    *reinterpret_cast<float4 *>(sQ + e * 4) = v;
                }
                __syncthreads();
                const int key = lane & 15, rh = (lane >> 4) * 4;     // this lane's key of a stage and first query row
                int lim[4];
                float m[4], l[4], o[8][E];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    lim[r] = a.mode == kPrefix ? 0 : own_limit(ow, r0 + rh + r, a.G);
                    m[r] = -INFINITY;
                    l[r] = 0.f;
                }
#pragma unroll
                for (int r = 0; r < 8; ++r)
#pragma unroll
                    for (int e = 0; e < E; ++e) o[r][e] = 0.f;
                float *pw = sP + warp * kKeys * R;
                for (int t = p.tb; t < p.te; ++t, ++it) {
                    cp_wait<S - 2>();
                    __syncwarp();
                    issue((it + S - 1) % S);
                    const int st = t * NW + warp;
                    if (st >= nst) continue;
                    const uint8_t *kb = smem + (warp * S + it % S) * Cfg::kStage, *vb = kb + Cfg::kHalf;
                    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
                    for (int c = 0; c < NC; ++c) {
                        const float4 k4 =
                            *reinterpret_cast<const float4 *>(kb + key * Cfg::kRowB + ((c ^ (key & 7)) << 4));
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float4 q4 = *reinterpret_cast<const float4 *>(sQ + (rh + r) * D + c * 4);
                            s[r] = fmaf(q4.x, k4.x, s[r]);
                            s[r] = fmaf(q4.y, k4.y, s[r]);
                            s[r] = fmaf(q4.z, k4.z, s[r]);
                            s[r] = fmaf(q4.w, k4.w, s[r]);
                        }
                    }
                    const bool pre = st < np;
                    const int kj = (pre ? st : st - np) * kKeys + key;
                    float f[4], pr[4];
                    bool grew = false;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = kj < (pre ? ow.plen : lim[r]) ? s[r] * a.sc : -INFINITY;
                        float mx = x;
#pragma unroll
                        for (int d = 1; d < 16; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                        const float mn = fmaxf(m[r], mx);
                        const float mu = mn == -INFINITY ? 0.f : mn;
                        f[r] = ex2(m[r] - mu);
                        m[r] = mn;
                        pr[r] = ex2(x - mu);
                        l[r] = l[r] * f[r] + pr[r];
                        grew |= f[r] != 1.f;
                    }
                    *reinterpret_cast<float4 *>(pw + key * R + rh) = make_float4(pr[0], pr[1], pr[2], pr[3]);
                    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                        for (int r = 0; r < 8; ++r) {
                            const float fr = __shfl_sync(0xffffffffu, f[r & 3], (r >> 2) * 16);
#pragma unroll
                            for (int e = 0; e < E; ++e) o[r][e] *= fr;
                        }
                    }
                    __syncwarp();
#pragma unroll 4
                    for (int k = 0; k < kKeys; ++k) {
                        float v[E];
#pragma unroll
                        for (int e = 0; e < E; e += EV) {
                            // dimensions lane*EV + (e/EV)*32*EV ..
                            const int d0 = lane * EV + (e / EV) * 32 * EV;
                            const uint8_t *va = vb + k * Cfg::kRowB + (((d0 >> 2) ^ (k & 7)) << 4) + (d0 & 3) * 4;
                            if constexpr (EV == 4) {
                                const float4 x = *reinterpret_cast<const float4 *>(va);
                                v[e] = x.x; v[e + 1] = x.y; v[e + 2] = x.z; v[e + 3] = x.w;
                            } else {
                                const float2 x = *reinterpret_cast<const float2 *>(va);
                                v[e] = x.x; v[e + 1] = x.y;
                            }
                        }
                        const float4 pa = *reinterpret_cast<const float4 *>(pw + k * R);
                        const float4 pb = *reinterpret_cast<const float4 *>(pw + k * R + 4);
                        const float pk[8] = {pa.x, pa.y, pa.z, pa.w, pb.x, pb.y, pb.z, pb.w};
#pragma unroll
                        for (int r = 0; r < 8; ++r)
#pragma unroll
                            for (int e = 0; e < E; ++e) o[r][e] = fmaf(pk[r], v[e], o[r][e]);
                    }
                    __syncwarp();                      // pw is rewritten by the next stage
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float ls = l[r];
#pragma unroll
                    for (int d = 1; d < 16; d <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, d);
                    if (key == 0) {
                        mM[warp * R + rh + r] = m[r];
                        mL[warp * R + rh + r] = ls;
                    }
                }
#pragma unroll
                for (int r = 0; r < 8; ++r)
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        mO[(warp * R + r) * kPitch + lane * EV + (e / EV) * 32 * EV + e % EV] = o[r][e];
            }
            __syncthreads();
            // the NW warps' states joined in warp order; a whole unit is the
            // result, a part of one goes to its slot (units started so far + CTA:
            // one number per piece, in line order)
            const bool whole = a.direct && p.tb == 0 && p.te == cons.tiles;
            const int64_t slot = (int64_t)cons.ubase + p.h * cons.rts + p.rt + blockIdx.x;
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
                    const int x = r0 + r, tk = x / a.G;
                    T *dst = static_cast<T *>(a.out) +
                             ((int64_t)(ow.t0 + tk) * a.hq + p.h * a.G + x - tk * a.G) * D + d;
                    st4(dst, y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
                } else if (slot < a.slots) {
                    st4(ps + r * D + d, y[0], y[1], y[2], y[3]);
                    if (d == 0) {
                        ps[R * D + r] = M;
                        ps[R * D + R + r] = L;
                    }
                }
            }
            __syncthreads();
        }
        cp_wait<0>();
    }
    if (!a.wait_first) pdl_wait();                     // this kernel's end tells its successor that the previous one ended too
}

// ------------------------------------------------------------------- joining
// Where the parts of a query row lie.
struct JoinSource {
    const float *part;
    const uint64_t *cum;
    int64_t slots;
    int owners, grid, R;               // of the k_paged_stream launch that left them
};
struct JoinArgs {
    JoinSource own, pre;               // pre.part null: no prefix parts
    int hq, G, full;                   // full: own parts belong to extend units
    void *out;
};

struct Parts {
    const float *base;                 // first part's slot
    int64_t step;                      // floats to the next
    int n, R, r;                       // parts, rows of a slot, this row
};

template <int D>
__device__ __forceinline__ Parts stream_parts(const JoinSource &s, int kv_heads, int o, int h, int r) {
    Parts p{};
    const uint64_t c0 = s.cum[o], c1 = s.cum[o + 1], all = s.cum[s.owners];
    const int hkv_rts = (int)((c1 >> 32) - (c0 >> 32));
    const uint32_t n = (uint32_t)c1 - (uint32_t)c0;
    p.R = s.R;
    const int rts = hkv_rts / kv_heads, rt = r / s.R;
    if (n == 0 || r < 0 || rt >= rts) return p;
    const uint32_t W = (uint32_t)all, per = (W + s.grid - 1) / s.grid;
    const int tiles = (int)(n / (uint32_t)hkv_rts);
    const int u = h * rts + rt;
    const uint32_t w0 = (uint32_t)c0 + (uint32_t)u * tiles;
    const uint32_t i0 = w0 / per, i1 = (w0 + tiles - 1) / per;
    const int64_t slot = (int64_t)(c0 >> 32) + u + i0;
    if (slot + (i1 - i0) >= s.slots) return p;
    p.step = s.R * D + 2 * s.R;
    p.base = s.part + slot * p.step;
    p.n = (int)(i1 - i0 + 1);
    p.r = r - rt * s.R;
    return p;
}

// One warp per (token, query head): parts of the prefix then of the own rows.
template <typename T, int D>
__global__ void __launch_bounds__(128) k_paged_join(const PagedView pv, const JoinArgs a) {
    constexpr int E = D / 32;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (int64_t)pv.tokens * a.hq) return;
    const int t = (int)(row / a.hq), hq = (int)(row - (int64_t)t * a.hq);
    const int h = hq / a.G, gi = hq - h * a.G;
    int s = t, t0 = t;
    if (a.full && pv.cu) {
        s = warp_upper(pv.cu, pv.seqs, t);
        t0 = pv.cu[s];
    }
    Parts po = stream_parts<D>(a.own, pv.kv_heads, s, h, (t - t0) * a.G + gi), pp{};
    if (a.pre.part) {
        const int g = warp_upper(pv.gs, pv.groups, s);
        pp = stream_parts<D>(a.pre, pv.kv_heads, g, h, (s - pv.gs[g]) * a.G + gi);
    } else if (po.n == 1) {
        return;                                        // a whole unit: written already
    }
    const int n = pp.n + po.n;
    auto part = [&](int i) { return i < pp.n ? pp.base + i * pp.step : po.base + (i - pp.n) * po.step; };
    auto stat = [&](int i, float &m, float &l) {
        const Parts &x = i < pp.n ? pp : po;
        const float *b = part(i) + (int64_t)x.R * D;
        m = __ldcg(b + x.r);
        l = __ldcg(b + x.R + x.r);
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
#pragma unroll 4
        for (int i = 0; i < top; ++i) {
            const float fi = __shfl_sync(0xffffffffu, f, i);
            const Parts &x = i0 + i < pp.n ? pp : po;
            const float *b = part(i0 + i) + (int64_t)x.r * D + lane * E;
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
    T *dst = static_cast<T *>(a.out) + row * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[e] = from_f32<T>(y[e] * inv);
}

// ---------------------------------------------------------------- host side

// CTAs of `kern` that fit an SM (asked once per kernel and device), its
// shared memory limit raised first.
int resident(const void *kern, int threads, int smem, int *out) {
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

// A k_paged_stream launch: its instantiation by row count, and its part of the workspace.
struct StreamPlan {
    int NB, R, NW, grid, slot;         // slot: floats
    int owners;
    int64_t units, cum_off, part_off, end;   // workspace bytes
};

template <typename T, int D, int NB> int stream_grid(StreamPlan *p) {
    using Cfg = StreamCfg<T, D, NB>;
    int n = 0;
    const int rc = resident(reinterpret_cast<const void *>(k_paged_stream<T, D, NB>), Cfg::NT, Cfg::kSmem, &n);
    if (rc != CBQ_OK) return rc;
    p->NB = NB;
    p->R = Cfg::R;
    p->NW = Cfg::NW;
    p->slot = Cfg::kSlot;
    p->grid = n * cbq_host::sm_count();
    return CBQ_OK;
}

template <typename T, int D, int NB>
int stream_launch(const PagedView &pv, const StreamArgs &a, int grid, cudaStream_t s) {
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

// Rows of a unit: as few blocks of 8 as hold an owner's rows (rows <= max_rows), at most 32.
int plan_stream(const PagedView &pv, int dtype, int d, int G, int mode, int64_t max_rows, int64_t off, StreamPlan *p) {
    const int nb = max_rows <= 8 ? 1 : (max_rows <= 16 ? 2 : 4);
    int rc = CBQ_OK;
#define CBQ_CALL(T, DD, NN) rc = stream_grid<T, DD, NN>(p)
    CBQ_STREAM_DISPATCH(dtype, d, nb, CBQ_CALL)
#undef CBQ_CALL
    if (rc != CBQ_OK) return rc;
    p->owners = mode == kPrefix ? pv.groups : pv.seqs;
    // row tiles of all owners: at most one per R rows and one more per owner
    const int64_t rows = (int64_t)pv.tokens * G;
    const int64_t rts = mode == kOwn ? (int64_t)pv.seqs * ((G + p->R - 1) / p->R) : rows / p->R + p->owners;
    p->units = rts * pv.kv_heads;
    const int64_t tile = (int64_t)kKeys * p->NW;
    const int64_t keys = mode == kOwn ? pv.cap : (mode == kPrefix ? pv.pcap : (int64_t)pv.cap + pv.pcap);
    if (p->units * ((keys + 2 * kKeys) / tile + 1) > 0x7fffffffll) return CBQ_ERR_UNSUPPORTED;   // tiles are counted in 32 bits
    p->cum_off = off;
    p->part_off = cbq_host::align_up(off + (p->owners + 1) * 8, 256);
    p->end = cbq_host::align_up(p->part_off + (p->units + p->grid) * (int64_t)p->slot * 4, 256);
    return CBQ_OK;
}

struct AttnPlan {
    PagedView pv;
    int dtype, d, G;
    bool extend, prefix;
    StreamPlan own, pre;
    int64_t bytes;
};

int plan_attn(const cbq_paged_cache *c, const cbq_paged_batch *b, int64_t tokens, int64_t q_heads, bool extend,
              AttnPlan *p) {
    const int rc = cbq_host::paged_view(c, b, tokens, q_heads, &p->pv);
    if (rc != CBQ_OK) return rc;
    p->bytes = 0;
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
    // rows of an owner: the mean, for extend (units of one size serve all owners)
    const int64_t mean = extend ? (tokens * p->G + b->seqs - 1) / b->seqs : p->G;
    int e = plan_stream(p->pv, p->dtype, p->d, p->G, extend ? kFull : kOwn, mean, 0, &p->own);
    if (e != CBQ_OK) return e;
    p->bytes = p->own.end;
    if (p->prefix) {
        const int64_t rows = ((int64_t)b->seqs + b->groups - 1) / b->groups * p->G;
        e = plan_stream(p->pv, p->dtype, p->d, p->G, kPrefix, rows, p->bytes, &p->pre);
        if (e != CBQ_OK) return e;
        p->bytes = p->pre.end;
    }
    return CBQ_OK;
}

int run_stream(const AttnPlan &p, const StreamPlan &sp, StreamArgs a, int mode, uint8_t *ws, cudaStream_t s) {
    a.mode = mode;
    a.owners = sp.owners;
    a.slots = sp.units + sp.grid;
    a.cum = reinterpret_cast<uint64_t *>(ws + sp.cum_off);
    a.part = reinterpret_cast<float *>(ws + sp.part_off);
#define CBQ_CALL(T, DD, NN) return stream_launch<T, DD, NN>(p.pv, a, sp.grid, s)
    CBQ_STREAM_DISPATCH(p.dtype, p.d, sp.NB, CBQ_CALL)
#undef CBQ_CALL
}

template <typename T, int D> int join_launch(const PagedView &pv, const JoinArgs &j, cudaStream_t s) {
    const int64_t blocks = ((int64_t)pv.tokens * j.hq + 3) / 4;
    CBQ_CUDA_TRY(cbq_host::launch_pdl(k_paged_join<T, D>, dim3((unsigned)blocks), dim3(128), 0, s, pv, j));
    return CBQ_OK;
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
    if ((reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(out) & 15) ||
        (reinterpret_cast<uintptr_t>(ws) & 255))
        return CBQ_ERR_ARG;
    uint8_t *w = static_cast<uint8_t *>(ws);
    StreamArgs a{};
    a.q = q;
    a.qs = q_stride;
    a.hq = (int)q_heads;
    a.G = p.G;
    a.sc = scale * kLog2e;
    a.out = out;
    a.wait_first = 1;
    if (p.prefix) {
        if ((rc = run_stream(p, p.pre, a, kPrefix, w, s)) != CBQ_OK) return rc;
        a.wait_first = 0;                              // the prefix launch passed its wait before this one can start
    }
    a.direct = !p.prefix;
    if ((rc = run_stream(p, p.own, a, extend ? kFull : kOwn, w, s)) != CBQ_OK) return rc;
    JoinArgs j{};
    auto source = [&](const StreamPlan &sp) {
        return JoinSource{reinterpret_cast<const float *>(w + sp.part_off), reinterpret_cast<const uint64_t *>(w + sp.cum_off),
                          sp.units + sp.grid, sp.owners, sp.grid, sp.R};
    };
    j.own = source(p.own);
    if (p.prefix) j.pre = source(p.pre);
    j.hq = (int)q_heads;
    j.G = p.G;
    j.full = extend;
    j.out = out;
    if (p.dtype == CBQ_F32)
        return p.d == 64 ? join_launch<float, 64>(p.pv, j, s)
                         : (p.d == 128 ? join_launch<float, 128>(p.pv, j, s) : join_launch<float, 256>(p.pv, j, s));
    return p.d == 64 ? join_launch<__nv_bfloat16, 64>(p.pv, j, s)
                     : (p.d == 128 ? join_launch<__nv_bfloat16, 128>(p.pv, j, s)
                                   : join_launch<__nv_bfloat16, 256>(p.pv, j, s));
}

}  // namespace

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
