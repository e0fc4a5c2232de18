// cbq_paged_tile.cu -- paged attention for many query rows per kv head on the
// 5th-generation tensor cores (sm_100a: tcgen05.mma, TMEM, TMA): prompts
// (extend), and the shared prefix of a group of sequences (decode).
//
// A unit's query rows (whole tokens, the G heads of a kv head side by side) lie
// in NQ blocks of 128.  Per key tile and row block:
//   S = Q K^T          tcgen05.mma, Q and K in shared memory, S fp32 in TMEM
//   P = 2^(sc S - m - kHead)   one thread per row, S from TMEM, P (bf16) to TMEM
//   O += P V           tcgen05.mma with P from TMEM, O fp32 in TMEM
// The running maximum m of a row is only moved when a tile exceeds it by more
// than 2^kGrow: until then the weights are taken relative to the old one (they
// stay below 2^(kGrow - kHead), and sums and O are fp32), so O is rescaled in TMEM a few
// times per unit instead of once per tile.  The result does not depend on m
// beyond rounding: o = (sum 2^(x - m) v) / (sum 2^(x - m)).
//
// P is rounded to bf16, the type of the values it multiplies, while l sums it
// unrounded: against 64 bits the results are off by 2.3e-3 where the rounding of an
// exact one takes 1.66e-3.  The rest as a second bf16 term brings that back to
// 1.66e-3, but takes P's columns and product twice (64 keys a tile): 706 us instead
// of 566 for a prompt of 8192 tokens, 292 instead of 265 for 256 sequences on a
// prefix of 32768 rows.  The usual choice, one term, is kept.
//
// A softmax reads S into registers at once, so the next tile's S can be computed
// while it works; P has columns of its own for that.  TMEM's 512 columns hold,
// per row block, S (one column per key), P (half) and O (one per dimension): at
// head_dim 128 that leaves room for 80 keys a tile, at 64 for 128.
//
// Warp roles: NQ softmax warpgroups (one row block each), a warp for each block's
// products (one thread issues, in code that stays uniform to the compiler: with
// descriptors made in vector registers a product took 90 cycles to issue and
// the tensor pipe waited), a TMA warp (one cp.async.bulk.tensor for 16 rows; K and
// V tiles alternate in a ring), a warp that walks the line ahead of them, leaves
// its pieces in shared memory and fetches Q by TMA.
//
// Measured (B200, bf16, head_dim 128): one prompt of 8192 tokens, 32 heads on 8:
// 564 us = 975 TFLOP/s in a short burst (SM clock 1965 MHz), 0.58 of a plain matrix
// product; 615 us = 894 TFLOP/s repeated for seconds, where the power limit takes the
// clock to about 1815 MHz.  A tile of 80 keys and 256 rows takes 2250 cycles: the
// products 1470 (S at 80 keys is bound by shared memory, 52 cycles instead of 40), both
// softmaxes 1280 of the special-function pipe, plus the latency of a softmax's other
// steps (900), of which two warps a scheduler hide too little.  Tried and slower (when
// this form ran at 995 TFLOP/s): P over S's columns with 128 keys a tile (943); two
// threads a row (950); a part of the exponentials by polynomial on the FMA pipe (950);
// the blocks taking turns at their exponentials (952); tiles copied by 16-byte
// asynchronous copies (618).
// Work is the tile line of cbq_paged_line.cuh, one persistent CTA per part.
// Every mbarrier wait is bounded; a wait that gives up sets CBQ_FLAG_TIMEOUT,
// all roles stop at their next wait, and TMEM is released on the way out.
#include <cuda.h>

#include <mutex>

#include "cbq_paged_line.cuh"

namespace {

using namespace cbq;

constexpr int kBlk = 128;              // rows of a block
constexpr int kBox = 16;               // rows of a copy; page_size is a multiple
constexpr float kGrow = 8.f;           // log2 growth of a row's maximum that moves its reference

template <int D, int NQ> struct TileCfg {
    static constexpr int KT = D == 128 ? 80 : 128;                     // keys of a tile
    static constexpr int kHalves = D / 64;                             // 128-byte wide column blocks
    static constexpr int kQHalfB = kBlk * 128, kQB = kHalves * kQHalfB; // a row block of Q: column block by column block
    static constexpr int kGroupB = kHalves * 1024;                      // 8 rows of K or V, column block by column block
    static constexpr int kTileB = KT / 8 * kGroupB;                     // a K or V tile
    static constexpr int kSlots = 8;                                   // K / V tiles in flight
    static constexpr int kSoft = NQ * 128;
    static constexpr int kThreads = kSoft + 128;                       // + a warpgroup for the other roles
    // registers: NQ = 2 splits the launch's 168 a thread unevenly (NQ = 1 has enough: one CTA on an SM,
    // whose shared memory goes to the ring)
    static constexpr int kSoftRegs = 208, kRestRegs = 88;
    static_assert(NQ == 1 || kSoft * kSoftRegs + 128 * kRestRegs <= kThreads * 168, "registers of the launch");
    static constexpr int kCols = NQ == 2 ? 512 : 256;
    static constexpr int kSmem = 1024 + NQ * kQB + kSlots * kTileB + 768;
    static __host__ __device__ constexpr uint32_t sCol(int b) { return (uint32_t)(b * (KT + KT / 2)); }
    static __host__ __device__ constexpr uint32_t pCol(int b) { return sCol(b) + KT; }
    static __host__ __device__ constexpr uint32_t oCol(int b) { return (uint32_t)(kCols - (NQ - b) * D); }
    static_assert(NQ * (KT + KT / 2 + D) <= kCols, "TMEM columns");
};

// A piece of the line as the roles need it, written by the scheduling warp.
struct Work {
    int o, t0, nt, plen, olen, group;  // owner
    int h, tok, tb, te;                // kv head, first token in the owner, key tiles
    int whole, live;                   // a whole unit of a direct line; 0: the line's end
    Cut cut;
    int64_t slot;
};
constexpr int kWorks = 3;              // the piece in hand, the next one, one ahead

struct Bars {
    uint64_t q_full[2], q_free[2], s_full[2], s_free[2], p_full[2], o_full[2];
    uint64_t kv_full[8], kv_empty[8];
    uint64_t w_full[kWorks], w_empty[kWorks];
    uint64_t drain[2];
    uint32_t tmem;
    int abort_flag;
    Work work[kWorks];
};
static_assert(sizeof(Bars) <= 768, "barriers outgrow their region");

// ---------------------------------------------------------------- PTX helpers
// Shared-memory operand descriptors, 128-byte swizzle.  The low word holds the
// address (in 16-byte units; stepping through an operand adds to it) and the
// leading offset: unused for a K-major operand, the distance of the 64-wide
// column blocks for an MN-major one (rows are K).  The high word: the distance
// of 8-row groups.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lead) { return (addr >> 4) | (lead >> 4) << 16; }
__host__ __device__ constexpr uint32_t desc_hi(uint32_t group) { return (group >> 4) | (1u << 14) | (2u << 29); }
// kind::f16: D fp32, A and B bf16, A K-major, B K-major or (bt) MN-major.
__host__ __device__ constexpr uint32_t idesc(int M, int N, int bt) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)bt << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t ahi, uint32_t b, uint32_t bhi, uint32_t id,
                                       uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %6};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(id), "r"(acc),
        "r"(ahi), "r"(bhi));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t bhi, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(id), "r"(acc),
        "r"(bhi));
}
// One lane of the warp; the code under it stays uniform to the compiler.
__device__ __forceinline__ bool elect() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar)) : "memory");
}
// 32 bytes in one store: a whole sector of each lane's row
__device__ __forceinline__ void st32b(void *p, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void tma_5d(uint32_t dst, const CUtensorMap *map, int c3, int c4, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(0), "r"(c3), "r"(c4), "r"(smem_u32(bar)) : "memory");
}
// 32 columns of this thread's TMEM lane, without waiting for them.
__device__ __forceinline__ void tld32(uint32_t a, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(a));
}
__device__ __forceinline__ void tld16(uint32_t a, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(a));
}
__device__ __forceinline__ void tld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tst16(uint32_t a, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tst8(uint32_t a, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void tst32(uint32_t a, const uint32_t *v) {
    tst16(a, v);
    tst16(a + 16, v + 16);
}
__device__ __forceinline__ void tst_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}

// Bounded wait of a whole warp; false (for all its lanes) once the CTA has
// given up.  The waits of the pipeline end within microseconds: they suspend on
// the barrier and only then look at the clock, whose read is slow.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, Bars *b, uint32_t *status) {
    bool ok = mbar_try_wait(bar, parity);
#pragma unroll 1
    for (int i = 0; i < 4 && !ok; ++i) ok = mbar_try_wait_sleep(bar, parity, 20000u);
    if (!ok) ok = !*(volatile int *)&b->abort_flag && mbar_wait_bounded(bar, parity);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok && (threadIdx.x & 31) == 0 && !*(volatile int *)&b->abort_flag) {
        *(volatile int *)&b->abort_flag = 1;
        report(status, CBQ_FLAG_TIMEOUT, 0u);
    }
    return ok;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A key tile: KT rows of the prefix or of the own rows from row key0 of it.
struct TileAt {
    bool pre;
    int key0, have;                    // rows of the tile that exist (0..KT)
};
template <int KT> __device__ __forceinline__ TileAt tile_at(int plen, int olen, int np, int t) {   // np: tiles of the prefix
    TileAt x;
    x.pre = t < np;
    x.key0 = (x.pre ? t : t - np) * KT;
    x.have = clampi((x.pre ? plen : olen) - x.key0, 0, KT);
    return x;
}

// 32 dimensions of a row of the output.
__device__ __forceinline__ void store_row(__nv_bfloat16 *dst, const uint32_t *o, float f) {
#pragma unroll
    for (int j = 0; j < 32; j += 16) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            w[e] = pack_bf16(__uint_as_float(o[j + 2 * e]) * f, __uint_as_float(o[j + 2 * e + 1]) * f);
        st32b(dst + j, w);
    }
}

// A warp joins its 32 rows of a cut unit (parts dimension by dimension), a
// lane its row `row`.
template <int D, int NQ>
__device__ __forceinline__ void join_block(const LineArgs &a, const Cut &cut, int row, bool live, __nv_bfloat16 *dst) {
    constexpr int RR = NQ * kBlk;
    constexpr int64_t SL = (int64_t)RR * (D + 2);
    float M = -INFINITY, L = 0.f;
    for (int k = 0; k < cut.n; ++k) M = fmaxf(M, __ldcg(cut.slot(a, k, SL) + RR * D + row));
    for (int k = 0; k < cut.n; ++k) {
        const float *b = cut.slot(a, k, SL) + RR * D + row;
        const float m = __ldcg(b);
        if (m != -INFINITY) L = fmaf(__ldcg(b + RR), ex2(m - M), L);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll 1
    for (int i = 0; i < D; i += 32) {
        uint32_t y[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) y[j] = 0u;
        for (int k = 0; k < cut.n; ++k) {
            const float *s = cut.slot(a, k, SL);
            const float m = __ldcg(s + RR * D + row), f = m == -INFINITY ? 0.f : ex2(m - M);
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __ldcg(s + (int64_t)(i + j) * RR + row);
#pragma unroll
            for (int j = 0; j < 32; ++j) y[j] = __float_as_uint(fmaf(v[j], f, __uint_as_float(y[j])));
        }
        if (live) store_row(dst + i, y, inv);
        __syncwarp();
    }
}

// The arrivals that a softmax warp still owes at cut units once a wait has
// given up (it made those of its first `done` pieces), so that the counters are
// zero after such a call too.  Every CTA walks its own part, whatever the
// others did; a unit that is joined from parts nobody wrote is reported.
__device__ __noinline__ void settle(const PagedView &pv, const LineArgs &a, const LineStart &st, uint32_t done) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tb = kBlk / a.geo.G;
    const int q = warp >> 2, rt = ((warp & 3) * 32 + lane) / a.geo.G;
    Cursor c = st.c;
    Piece p{};
    for (uint32_t i = 0; next_piece(c, pv, a, st.w1, p); ++i) {
        const bool live = rt < tb && p.tt * a.geo.tq + q * tb + rt < c.ow.nt;
        if (i < done || (p.tb == 0 && p.te == p.tiles) || !__any_sync(0xffffffffu, live)) continue;
        const Cut cut = cut_of(c, p, st.per);
        uint32_t *cnt = a.count + cut.i0 * 8 + warp;
        if (lane == 0 && atomicAdd(cnt, 1u) == (uint32_t)(cut.n - 1)) *cnt = 0u;
        __syncwarp();
    }
}

template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <int D, int NQ>
__global__ void __launch_bounds__(TileCfg<D, NQ>::kThreads, 1)
    k_paged_tile(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                 const __grid_constant__ CUtensorMap qmap, const __grid_constant__ PagedView pv,
                 const __grid_constant__ LineArgs a) {
    using Cfg = TileCfg<D, NQ>;
    constexpr int kSlots = Cfg::kSlots, kTileB = Cfg::kTileB, KT = Cfg::KT;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sQ = smem, *sKV = smem + NQ * Cfg::kQB;
    Bars *bars = reinterpret_cast<Bars *>(sKV + kSlots * kTileB);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int kTmaWarp = Cfg::kSoft / 32, kWorkWarp = kTmaWarp + 1, kMmaWarp = kTmaWarp + 2;   // kMmaWarp + block

    if (tid == 0) {
        for (int q = 0; q < NQ; ++q) {
            mbar_init(&bars->q_full[q], 1);
            mbar_init(&bars->q_free[q], 1);
            mbar_init(&bars->s_full[q], 1);
            mbar_init(&bars->s_free[q], 128);
            mbar_init(&bars->p_full[q], 128);
            mbar_init(&bars->o_full[q], 1);
        }
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(&bars->kv_full[s], 1);
            mbar_init(&bars->kv_empty[s], NQ);
        }
        for (int i = 0; i < kWorks; ++i) {
            mbar_init(&bars->w_full[i], 1);
            mbar_init(&bars->w_empty[i], kTmaWarp + 1 + NQ);   // one arrival of every warp that reads it
        }
        for (int q = 0; q < NQ; ++q) mbar_init(&bars->drain[q], 1);
        bars->abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem)),
                     "r"(Cfg::kCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (a.wait_first) pdl_wait();
    pdl_launch_dependents();
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem, 0);
    Cursor c{};
    uint32_t w1 = 0, per = 1;
    const Ends ends = token_ends(pv, a);
    __shared__ LineStart start;
    const bool any = plan_line<Cfg::kThreads>(pv, a, start, c, w1, per);
    zero_rest<__nv_bfloat16, D>(pv, a, ends);

    // The i-th piece (0 where the line ends or a wait gave up); done(i) gives its place back.
    auto work = [&](uint32_t i) -> const Work * {
        if (!warp_wait(&bars->w_full[i % kWorks], (i / kWorks) & 1, bars, pv.status)) return nullptr;
        const Work *w = &bars->work[i % kWorks];
        return w->live ? w : nullptr;
    };
    auto done = [&](uint32_t i) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->w_empty[i % kWorks]);
    };
    const int tb = kBlk / a.geo.G;                     // tokens of a row block
    if constexpr (NQ == 2) {
        if (warp < kTmaWarp) regs_up<Cfg::kSoftRegs>(); else regs_down<Cfg::kRestRegs>();
    }
    if (!any) {
        // nothing of the line for this CTA
    } else if (warp < kTmaWarp) {
        // ------------------------------------------- softmax and output: thread = row
        const int q = warp >> 2, r = tid & 127;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t tS = lanes + Cfg::sCol(q), tP = lanes + Cfg::pCol(q), tO = lanes + Cfg::oCol(q);
        const int rt = r / a.geo.G, rg = r - rt * a.geo.G;            // the row's token in the block, head in the group
        // a scale below 0 turns S's sign, a scale of 0 clears it: sc > 0 below
        const float sc = a.sc == 0.f ? 1.f : fabsf(a.sc), turn = a.sc == 0.f ? 0.f : -1.f;
        uint32_t nw = 0, ns = 0;                       // pieces; tiles seen (phases of s_full, p_full and o_full)
        const Work *w = work(0);
        bool go = true;
        while (w) {
            const int tok = w->tok + q * tb + rt;
            const bool live = rt < tb && tok < w->nt;
            const int plen = w->plen, olen = w->olen, np = (plen + KT - 1) / KT, t0 = w->tb, t1 = w->te;
            const int olim = a.mode == kPrefix ? 0 : clampi(olen - w->nt + tok + 1, 0, olen);
            float m = -INFINITY, l = 0.f;
            const bool idle = !__any_sync(0xffffffffu, live);       // a warp whose rows hold no query only keeps step
            bool early = false;                        // S of the tile was there before the last one's end
            for (int t = t0; t < t1; ++t, ++ns) {
                if (!__all_sync(0xffffffffu, early) && !warp_wait(&bars->s_full[q], ns & 1, bars, pv.status)) {
                    go = false;
                    break;
                }
                if (idle) {
                    mbar_arrive(&bars->s_free[q]);
                    // not a P ahead of the others: its arrival would count for theirs
                    if (t > t0 && !warp_wait(&bars->o_full[q], (ns - 1) & 1, bars, pv.status)) { go = false; break; }
                    mbar_arrive(&bars->p_full[q]);
                    early = false;
                    continue;
                }
                tc_after();
                uint32_t s[KT];
#pragma unroll
                for (int i = 0; i + 32 <= KT; i += 32) tld32(tS + i, s + i);
                if constexpr (KT % 32) tld16(tS + KT / 32 * 32, s + KT / 32 * 32);
                tld_wait();
                tc_before();
                mbar_arrive(&bars->s_free[q]);         // the next tile's S may come
                if (a.sc <= 0.f) {
#pragma unroll
                    for (int j = 0; j < KT; ++j) s[j] = __float_as_uint(__uint_as_float(s[j]) * turn);
                }
                const TileAt x = tile_at<KT>(plen, olen, np, t);
                const int vis = x.pre ? x.have : min(x.have, olim - x.key0);   // visible keys of the tile
                // whether the products with the last P are done: asked here, needed after the weights
                bool o_done = t > t0 && mbar_test(&bars->o_full[q], (ns - 1) & 1);
                if (__any_sync(0xffffffffu, vis < KT)) {
#pragma unroll
                    for (int j = 0; j < KT; ++j)
                        if (j >= vis) s[j] = 0xff800000u;                      // -inf
                }
                float mx[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e] = fmaxf(__uint_as_float(s[e]), __uint_as_float(s[e + 4]));
#pragma unroll
                for (int j = 8; j < KT; j += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        mx[e] = max3(mx[e], __uint_as_float(s[j + e]), __uint_as_float(s[j + e + 4]));
                const float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                const bool grow = (mn - m) * sc > kGrow;                       // false where both are -inf
                const float f = grow ? ex2((m - mn) * sc) : 1.f;               // 0 from -inf
                if (grow) m = mn;
                const float mb = m == -INFINITY ? 0.f : fmaf(m, sc, kHead);
                float ls[4] = {0.f, 0.f, 0.f, 0.f};
                uint32_t pk[KT / 2];
#pragma unroll
                for (int j = 0; j < KT; j += 2) {
                    float e[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        e[i] = ex2(fmaf(__uint_as_float(s[j + i]), sc, -mb));
                        ls[(j + i) & 3] += e[i];
                    }
                    pk[j / 2] = pack_bf16(e[0], e[1]);
                }
                l = l * f + ((ls[0] + ls[1]) + (ls[2] + ls[3]));
                if (t > t0) {
                    // the products with the last P are done: P may be written, O scaled
                    if (!__all_sync(0xffffffffu, o_done) && !warp_wait(&bars->o_full[q], (ns - 1) & 1, bars, pv.status)) {
                        go = false;
                        break;
                    }
                    if (__any_sync(0xffffffffu, grow)) {
                        tc_after();
#pragma unroll 1
                        for (int i = 0; i < D; i += 32) {
                            uint32_t o[32];
                            tld32(tO + i, o);
                            tld_wait();
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                            tst32(tO + i, o);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i + 16 <= KT / 2; i += 16) tst16(tP + i, pk + i);
                if constexpr (KT / 2 % 16) tst8(tP + KT / 32 * 16, pk + KT / 32 * 16);
                early = t + 1 < t1 && mbar_test(&bars->s_full[q], (ns + 1) & 1);
                tst_wait();
                tc_before();
                mbar_arrive(&bars->p_full[q]);
            }
            if (!go) break;
            if (!warp_wait(&bars->o_full[q], (ns - 1) & 1, bars, pv.status)) { go = false; break; }
            tc_after();
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const bool fits = w->slot < a.slots, whole = w->whole;
            constexpr int64_t SL = (int64_t)NQ * kBlk * (D + 2);
            float *ps = a.part + w->slot * SL;
            __nv_bfloat16 *dst = static_cast<__nv_bfloat16 *>(a.out) +
                                 ((int64_t)(w->t0 + tok) * a.hq + w->h * a.geo.G + rg) * D;
#pragma unroll 1
            for (int i = 0; i < D && !idle; i += 32) {
                uint32_t o[32];
                tld32(tO + i, o);
                tld_wait();
                if (whole) {
                    if (live) store_row(dst + i, o, inv);
                } else if (fits && a.direct) {
                    // joined by the same rows of another CTA's warps: dimension by dimension, rows side by side
                    float *b = ps + (int64_t)i * (NQ * kBlk) + q * kBlk + r;
#pragma unroll
                    for (int j = 0; j < 32; ++j) __stcg(b + j * (NQ * kBlk), __uint_as_float(o[j]));
                } else if (fits && live) {
                    float *b = ps + (int64_t)(q * kBlk + r) * D + i;
#pragma unroll
                    for (int j = 0; j < 32; j += 8) st32b(b + j, o + j);
                }
                __syncwarp();                          // the next TMEM load is the whole warp's
            }
            tc_before();                               // O's reads before the next unit's first product
            if (!whole && fits && !idle) {
                // joined with parts of either kernel: the maximum in units of log2
                ps[NQ * kBlk * D + q * kBlk + r] = m == -INFINITY ? m : m * sc;
                ps[NQ * kBlk * D + NQ * kBlk + q * kBlk + r] = l;
            }
            if (a.direct && !whole && !idle) {
                // the warp that arrives last at its 32 rows of a cut unit joins
                // their parts (a count for each warp: no barrier that a warp whose
                // wait gave up could leave the others at)
                __threadfence();
                __syncwarp();
                const Cut cut = w->cut;
                uint32_t *cnt = a.count + cut.i0 * 8 + warp;
                uint32_t before = 0;
                if (lane == 0) before = atomicAdd(cnt, 1u);
                before = __shfl_sync(0xffffffffu, before, 0);
                if (before == (uint32_t)(cut.n - 1)) {
                    __threadfence();
                    join_block<D, NQ>(a, cut, q * kBlk + r, live, dst);
                    if (lane == 0) *cnt = 0u;
                }
            }
            __syncwarp();
            done(nw);
            ++nw;
            w = work(nw);
        }
        if (a.direct && *(volatile int *)&bars->abort_flag) settle(pv, a, start, nw);
    } else if (warp == kTmaWarp) {
        // ------------------------------------------------------------- K and V tiles
        uint32_t n = 0, nw = 0;                        // tiles issued (K and V), pieces
        bool go = true;
        const int ps = 1 << pv.ps_shift, ratio = (int)(pv.page_stride / pv.head_stride);
        const int none = (pv.pages - 1) * ratio + pv.kv_heads;
        while (go) {
            const Work *w = work(nw);
            if (!w) break;
            const int plen = w->plen, olen = w->olen, np = (plen + KT - 1) / KT, o = w->o, t1 = w->te, h = w->h;
            const int32_t *ptab = pv.ptable + w->group * pv.ptable_stride, *otab = pv.table + o * pv.table_stride;
            for (int t = w->tb; t < t1 && go; ++t) {
                const TileAt x = tile_at<KT>(plen, olen, np, t);
                const int nbox = __shfl_sync(0xffffffffu, (x.have + kBox - 1) / kBox, 0);
                // lane b: the tile's b-th 16 rows, as a coordinate of (page, head); outside the map: zeros
                int at = none;
                if (lane < nbox) {
                    const int page = __ldg((x.pre ? ptab : otab) + ((x.key0 + lane * kBox) >> pv.ps_shift));
                    if (page >= 0 && page < pv.pages) at = page * ratio + h;
                    else report(pv.status, CBQ_FLAG_CORRUPT, (uint32_t)o);
                }
#pragma unroll
                for (int kv = 0; kv < 2; ++kv, ++n) {
                    const int s = n % kSlots;
                    if (n >= kSlots && !warp_wait(&bars->kv_empty[s], (n / kSlots - 1) & 1, bars, pv.status)) {
                        go = false;
                        break;
                    }
                    const uint32_t dst = smem_u32(sKV) + s * kTileB;
                    uint64_t *full = &bars->kv_full[s];
                    if (elect()) mbar_arrive_expect_tx(full, (uint32_t)(nbox * kBox * D * 2));
                    __syncwarp();
#pragma unroll
                    for (int b = 0; b < KT / kBox; ++b) {
                        if (b >= nbox) break;
                        const int pg = __shfl_sync(0xffffffffu, at, b), grp = ((x.key0 + b * kBox) & (ps - 1)) >> 3;
                        if (elect()) tma_5d(dst + b * 2 * Cfg::kGroupB, kv ? &vmap : &kmap, grp, pg, full);
                        __syncwarp();
                    }
                }
            }
            done(nw++);
        }
        // no copy may still be landing when the CTA ends
        for (uint32_t s = 0; s < kSlots && s < n; ++s) {
            const uint32_t last = n - 1 - (n - 1 - s) % kSlots;
            mbar_wait_bounded(&bars->kv_full[s], (last / kSlots) & 1);
        }
    } else if (warp >= kMmaWarp && warp < kMmaWarp + NQ) {
        // ------------------------------------------------------------------ products of block q
        const int q = warp - kMmaWarp;
        constexpr uint32_t idS = idesc(128, KT, 0), idO = idesc(128, D, 1);
        uint32_t n = 0, ns = 0, nw = 0;                // ring tiles used, tiles of S, pieces
        bool go = true;
        const uint32_t kv0 = desc_lo(smem_u32(sKV), 1024), q0 = desc_lo(smem_u32(sQ + q * Cfg::kQB), 0);
        constexpr uint32_t hiQ = desc_hi(1024), hiKV = desc_hi(Cfg::kGroupB);
        const uint32_t tS = tmem + Cfg::sCol(q), tP = tmem + Cfg::pCol(q), tO = tmem + Cfg::oCol(q);
        auto wait_kv = [&](uint32_t i) {
            return warp_wait(&bars->kv_full[i % kSlots], (i / kSlots) & 1, bars, pv.status);
        };
        // S of the tile whose K is the ring's i-th, once the S before it has been read
        auto scores = [&](uint32_t i, bool last) {
            if (!wait_kv(i) || (ns && !warp_wait(&bars->s_free[q], (ns - 1) & 1, bars, pv.status))) return false;
            tc_after();
            const uint32_t ka = kv0 + (i % kSlots) * (kTileB >> 4);
            if (elect()) {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    mma_ss(tS, q0 + (((kk >> 2) * Cfg::kQHalfB + (kk & 3) * 32) >> 4), hiQ,
                           ka + (((kk >> 2) * 1024 + (kk & 3) * 32) >> 4), hiKV, idS, kk > 0);
                mma_commit(&bars->s_full[q]);
                mma_commit(&bars->kv_empty[i % kSlots]);
                if (last) mma_commit(&bars->q_free[q]);
            }
            __syncwarp();
            ++ns;
            return true;
        };
        while (go) {
            const Work *w = work(nw);
            if (!w) {
                go = !*(volatile int *)&bars->abort_flag;
                break;
            }
            // ring: K of tile t at n + 2 t, V at n + 2 t + 1
            const int plen = w->plen, olen = w->olen, np = (plen + KT - 1) / KT, tb0 = w->tb, nt = __shfl_sync(0xffffffffu, w->te - tb0, 0);
            go = warp_wait(&bars->q_full[q], nw & 1, bars, pv.status) && scores(n, nt == 1);
            for (int t = 0; t < nt && go; ++t) {
                const uint32_t iv = n + 2 * t + 1;
                if (t + 1 < nt && !(go = scores(iv + 1, t + 2 == nt))) break;
                if (!(go = wait_kv(iv))) break;
                const TileAt x = tile_at<KT>(plen, olen, np, tb0 + t);
                if (x.have < KT) {
                    // rows that do not exist (rest of a page, pages not copied) must not meet a weight
                    // of 0; both blocks' warps clear them, each before its own product
                    for (int e = x.have * 8 + lane; e < KT * 8; e += 32) {
                        uint8_t *row = sKV + (iv % kSlots) * kTileB + (e >> 6) * Cfg::kGroupB + (e & 63) * 16;
#pragma unroll
                        for (int hf = 0; hf < Cfg::kHalves; ++hf)
                            *reinterpret_cast<uint4 *>(row + hf * 1024) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                if (!(go = warp_wait(&bars->p_full[q], (ns - (t + 1 < nt ? 2 : 1)) & 1, bars, pv.status))) break;
                tc_after();
                const uint32_t va = kv0 + (iv % kSlots) * (kTileB >> 4);
                if (elect()) {
#pragma unroll
                    for (int kk = 0; kk < KT / 16; ++kk)
                        mma_ts(tO, tP + kk * 8, va + kk * (2 * Cfg::kGroupB >> 4), hiKV, idO, t > 0 || kk > 0);
                    mma_commit(&bars->o_full[q]);
                    mma_commit(&bars->kv_empty[iv % kSlots]);
                }
                __syncwarp();
            }
            if (!go) break;
            n += 2 * nt;
            done(nw++);
        }
        if (!go) {                                     // gave up: products in flight end first
            if (elect()) mma_commit(&bars->drain[q]);
            __syncwarp();
            mbar_wait_bounded(&bars->drain[q], 0);
        }
    } else if (warp == kWorkWarp) {
        // -------------------------------------------------------------- the line ahead
        Piece p{};
        uint32_t nq = 0;                               // pieces whose Q is on its way
        bool more = true;
        for (uint32_t i = 0; more; ++i) {
            if (i >= kWorks && !warp_wait(&bars->w_empty[i % kWorks], (i / kWorks - 1) & 1, bars, pv.status)) break;
            more = next_piece(c, pv, a, w1, p);
            if (lane == 0) {
                Work *w = &bars->work[i % kWorks];
                w->live = more;
                if (more) {
                    w->o = c.o; w->t0 = c.ow.t0; w->nt = c.ow.nt; w->plen = c.ow.plen; w->olen = c.ow.olen;
                    w->group = max(c.ow.group, 0);
                    w->h = p.h; w->tok = p.tt * a.geo.tq; w->tb = p.tb; w->te = p.te;
                    w->whole = a.direct && p.tb == 0 && p.te == p.tiles;
                    w->cut = cut_of(c, p, per);
                    w->slot = slot_of(c, p, a, (int)blockIdx.x);
                }
                mbar_arrive(&bars->w_full[i % kWorks]);
            }
            __syncwarp();
            // Q of the piece, once the products with the last one are done; rows past the
            // tensor's end come as zeros, rows of other tokens are not used
            for (int q = 0; q < NQ && more; ++q) {
                if (i && !(more = warp_wait(&bars->q_free[q], (i - 1) & 1, bars, pv.status))) break;
                if (lane == 0) mbar_arrive_expect_tx(&bars->q_full[q], (uint32_t)(tb * a.geo.G * D * 2));
                __syncwarp();
                if (lane < Cfg::kHalves)
                    tma_3d(smem_u32(sQ + q * Cfg::kQB + lane * Cfg::kQHalfB), &qmap, lane * 64, p.h * a.geo.G,
                           c.ow.t0 + p.tt * a.geo.tq + q * tb, &bars->q_full[q]);
                __syncwarp();
                nq = i + 1;
            }
        }
        // no copy may still be landing when the CTA ends
        for (int q = 0; q < NQ && nq; ++q) mbar_wait_bounded(&bars->q_full[q], (nq - 1) & 1);
    }
    tc_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::kCols) : "memory");
    }
    if (!a.wait_first) pdl_wait();
}

// ---------------------------------------------------------------- host side
using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
    static EncodeFn fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return (EncodeFn) nullptr;
        return reinterpret_cast<EncodeFn>(f);
    }();
    return fn;
}

// The pool as {64 dimensions, 8 rows, column blocks, row groups, (page, head)};
// a box is 16 rows of a page and head, in shared memory 8 rows by 8 rows and
// within them column block by column block, which both products' descriptors
// can step through: 4 KB a copy at head_dim 128 (a copy costs the SM's copy
// engine 46 cycles and 18 a KB).
bool pool_map(const cbq_paged_cache *c, void *pool, CUtensorMap *map) {
    EncodeFn enc = encoder();
    if (!enc) return false;
    const cuuint64_t ratio = (cuuint64_t)(c->page_stride / c->head_stride);
    const cuuint64_t dims[5] = {64, 8, (cuuint64_t)c->head_dim / 64, (cuuint64_t)c->page_size / 8,
                                (cuuint64_t)(c->pages - 1) * ratio + (cuuint64_t)c->kv_heads};
    const cuuint64_t strides[4] = {(cuuint64_t)c->row_stride * 2, 128, (cuuint64_t)c->row_stride * 16,
                                   (cuuint64_t)c->head_stride * 2};
    const cuuint32_t box[5] = {64, 8, (cuuint32_t)c->head_dim / 64, kBox / 8, 1}, es[5] = {1, 1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, pool, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
           CUDA_SUCCESS;
}

// The queries as {dimension, head, token}; a box is the G heads of a row block's tokens by 64 dimensions.
bool query_map(const cbq_paged_cache *c, const cbq::PagedView &pv, const LineArgs &a, CUtensorMap *map) {
    EncodeFn enc = encoder();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)c->head_dim, (cuuint64_t)a.hq, (cuuint64_t)pv.tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)c->head_dim * 2, (cuuint64_t)a.qs * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)a.geo.G, (cuuint32_t)(kBlk / a.geo.G)}, es[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(a.q), dims, strides, box, es,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NQ> int grid_of(int *ctas) {
    using Cfg = TileCfg<D, NQ>;
    return cbq_host::resident_ctas(reinterpret_cast<const void *>(k_paged_tile<D, NQ>), Cfg::kThreads, Cfg::kSmem, ctas);
}

template <int D, int NQ>
int launch_tile(const CUtensorMap &km, const CUtensorMap &vm, const CUtensorMap &qm, const PagedView &pv, const LineArgs &a, int grid,
                cudaStream_t s) {
    using Cfg = TileCfg<D, NQ>;
    CBQ_CUDA_TRY(cbq_host::launch_pdl(k_paged_tile<D, NQ>, dim3((unsigned)grid), dim3(Cfg::kThreads), (size_t)Cfg::kSmem, s,
                                      km, vm, qm, pv, a));
    return CBQ_OK;
}

}  // namespace

namespace cbq_host {

bool tile_takes(const cbq_paged_cache *c) {
    // what the pools' tensor maps hold: pages a whole number of heads apart, strides below 2^40 bytes,
    // (page, head) counted in 32 bits
    const int64_t top = (int64_t)1 << 35;
    return c->dtype == CBQ_BF16 && (c->head_dim == 64 || c->head_dim == 128) && c->pages > 0 && c->head_stride > 0 &&
           c->head_stride < top && c->row_stride < top && c->page_stride % c->head_stride == 0 && c->page_stride > 0 &&
           c->pages < (int64_t)1 << 30 &&
           c->page_stride / c->head_stride < ((int64_t)1 << 31) / (c->pages + 1) - c->kv_heads && encoder() != nullptr;
}

int tile_plan(const cbq::PagedView &pv, int d, int G, int mode, bool two, int64_t off, LinePlan *p) {
    int n = 0;
    const int rc = d == 64 ? (two ? grid_of<64, 2>(&n) : grid_of<64, 1>(&n))
                           : (two ? grid_of<128, 2>(&n) : grid_of<128, 1>(&n));
    if (rc != CBQ_OK) return rc;
    const int nq = two ? 2 : 1;
    p->mode = mode;
    p->rows = nq * kBlk;
    p->tile_rows = kBlk;
    p->geo.G = G;
    p->geo.tq = nq * (kBlk / G);
    p->geo.hc = 1;
    p->geo.keys = d == 64 ? TileCfg<64, 1>::KT : TileCfg<128, 1>::KT;
    p->geo.join = 0;
    p->min_tiles = 2;                  // a part costs its CTA about as much as a tile
    p->grid = n * sm_count();
    return p->grid * 8 <= kCounts && line_room(pv, d, off, p) ? CBQ_OK : CBQ_ERR_UNSUPPORTED;
}

int tile_launch(const cbq_paged_cache *c, const cbq::PagedView &pv, const LinePlan &p, cbq::LineArgs a, cudaStream_t s) {
    CUtensorMap km, vm, qm;
    if (!pool_map(c, c->k_dev, &km) || !pool_map(c, c->v_dev, &vm) || !query_map(c, pv, a, &qm)) return CBQ_ERR_UNSUPPORTED;
    const bool two = p.rows > kBlk;
    if (c->head_dim == 64)
        return two ? launch_tile<64, 2>(km, vm, qm, pv, a, p.grid, s) : launch_tile<64, 1>(km, vm, qm, pv, a, p.grid, s);
    return two ? launch_tile<128, 2>(km, vm, qm, pv, a, p.grid, s) : launch_tile<128, 1>(km, vm, qm, pv, a, p.grid, s);
}

}  // namespace cbq_host
