// cbq_paged_line.cuh -- how the paged attention kernels divide their work.
//
// Work is one line of key tiles.  An owner is a sequence (its own rows, or for
// extend its prefix and own rows) or a group (its prefix, the query rows of all
// its sequences).  A unit is (owner, kv head, token tile, head chunk): the query
// rows that share the keys of one kv head; the line lists every unit's key
// tiles one after the other, under a causal mask only those that some row of
// the unit sees.  The line is cut into equal parts, one for each CTA, so ragged
// lengths and triangles balance by themselves and a single long sequence
// spreads over all SMs.  Everything is found from the lengths on the device:
// owners by a sum over all of them, units inside an owner in closed form.
#pragma once
#include <algorithm>

#include "cbq_paged.cuh"

namespace cbq {

constexpr float kLog2e = 1.4426950408889634f;

// Weights are taken as 2^(x - m - kHead): a sum of up to 2^16 of the largest
// finite values (2^8 in the tile kernel, whose weights run up to 2^8 above a
// reference m) stays finite until l, smaller by the same factor, divides it.
// What is lost lies below 2^-110, of a weight or of a value.
constexpr float kHead = 16.f;

enum LineMode : int {
    kOwn = 0,                          // owner = sequence, keys = its own rows (decode)
    kPrefix = 1,                       // owner = group, keys = its prefix, rows = all its sequences' (decode)
    kFull = 2,                         // owner = sequence, keys = prefix then own rows, causal (extend)
};

// Shape of a unit.  Keys of a unit whose rows see `lim` own rows make
// (prefix tiles) + ceil((carry + lim) / keys) tiles: with `join` the prefix's
// 16-key stages run on into the own rows' tiles (carry), else the prefix ends
// in a tile of its own.
struct LineGeo {
    int G;                             // query heads of a kv head
    int tq, hc;                        // tokens of a unit; chunks that a token's heads are cut into
    int keys;                          // keys of a tile
    int join;
};

struct LineArgs {
    LineGeo geo;
    const void *q;
    int64_t qs;                        // token stride, elements
    int hq;
    float sc;                          // scale * log2(e)
    void *out;
    float *part;                       // slots of [rows * D + 2 * rows] fp32: o (unnormalised), m, l
    uint64_t *cum;                     // [owners + 1] units << 32 | tiles before each owner (not direct)
    uint32_t *count;                   // direct: arrivals at the unit cut at a CTA's end, by CTA (tile kernel: by CTA
                                       // and warp); 0 between calls
    int64_t slots;                     // slots of `part` (starts that are not in order could name more)
    int owners, mode;
    int min_tiles;                     // a CTA's part has at least so many tiles
    int direct;                        // whole units go to `out`; else every unit leaves parts
    int wait_first;                    // wait for the previous kernel before reading (else before the end only)
};

struct Owner {
    int t0, nt;                        // its query tokens
    int plen, olen;                    // prefix and own rows
    int group;
};

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// Largest i in [0, n) with a[i] <= x (one thread).
__device__ __forceinline__ int upper(const int32_t *a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

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
        const int g = upper(pv.gs, pv.groups, o);
        if (o >= pv.gs[g] && o < pv.gs[g + 1]) {       // else in no group
            w.group = g;
            w.plen = clampi(pv.plens[g], 0, pv.pcap);
        }
    }
    return w;
}

// Own rows visible to the owner's token i.
__device__ __forceinline__ int own_limit(const Owner &w, int i) { return clampi(w.olen - w.nt + i + 1, 0, w.olen); }

// sum over i < n of floor((a i + b) / m), by the Euclidean reduction of the
// lattice points under a line.
__device__ __forceinline__ uint32_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
    uint32_t s = 0;
    while (true) {
        if (a >= m) {
            s += n * (n - 1) / 2 * (a / m);
            a %= m;
        }
        if (b >= m) {
            s += n * (b / m);
            b %= m;
        }
        const uint32_t y = a * n + b;
        if (y < m) return s;
        n = y / m;
        b = y % m;
        const uint32_t t = m;
        m = a;
        a = t;
    }
}

// Tiles of an owner's units.
struct OwnerTiles {
    int tt;                            // token tiles
    uint32_t fixed;                    // tiles of every unit before the causal part
    uint32_t b, keys, tq, causal;      // causal part of token tile i: floor((b + i tq) / keys)
    uint32_t last;                     // tiles of the last token tile

    __device__ __forceinline__ uint32_t of(int i) const {
        return i == tt - 1 ? last : fixed + (causal ? (b + (uint32_t)i * tq) / keys : 0u);
    }
    // tiles of the token tiles before i
    __device__ __forceinline__ uint32_t before(int i) const {
        return fixed * (uint32_t)i + (causal && i > 0 ? floor_sum((uint32_t)i, keys, tq, b) : 0u);
    }
    __device__ __forceinline__ uint32_t all() const { return tt > 0 ? before(tt - 1) + last : 0u; }
};

__device__ __forceinline__ OwnerTiles owner_tiles(const Owner &w, const LineGeo &g, int mode) {
    OwnerTiles t{};
    t.tt = (w.nt + g.tq - 1) / g.tq;
    t.keys = (uint32_t)g.keys;
    t.tq = (uint32_t)g.tq;
    const int stages = (w.plen + 15) / 16 * 16;
    const uint32_t carry = g.join ? (uint32_t)stages : 0u;
    const uint32_t pre = g.join ? 0u : (uint32_t)((w.plen + g.keys - 1) / g.keys);
    if (mode == kFull) {
        // a row without own rows of its own (more new tokens than rows) counts as if it had them
        const uint32_t e0 = (uint32_t)max(w.olen - w.nt, 0);
        t.causal = 1;
        t.fixed = pre;
        t.b = carry + e0 + t.tq + t.keys - 1;
        t.last = max(pre + (carry + e0 + (uint32_t)w.nt + t.keys - 1) / t.keys, 1u);
    } else {
        t.fixed = t.last = max(pre + (carry + (uint32_t)w.olen + t.keys - 1) / t.keys, 1u);
    }
    return t;
}

// Extend: the tokens before the first sequence's and behind the last one's
// belong to none; their rows of the result (a.hq * d elements each) are zeros.
// They are asked for before the plan, whose own loads hide theirs.
struct Ends {
    int lo, hi;
};
__device__ __forceinline__ Ends token_ends(const PagedView &pv, const LineArgs &a) {
    Ends e{0, pv.tokens};
    if (a.direct && a.mode == kFull && pv.cu) {
        e.lo = pv.cu[0];
        e.hi = pv.cu[pv.seqs];
    }
    return e;
}
// `row`: 16-byte pieces of a row.
static __device__ __noinline__ void zero_rows(void *out, int lo, int hi, int tokens, int row) {
    lo = clampi(lo, 0, tokens);
    hi = clampi(hi, lo, tokens);
    const int64_t head = (int64_t)lo * row, skip = (int64_t)(hi - lo) * row, n = (int64_t)tokens * row - skip;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
        static_cast<uint4 *>(out)[i < head ? i : i + skip] = make_uint4(0u, 0u, 0u, 0u);
}
template <typename T, int D>
__device__ __forceinline__ void zero_rest(const PagedView &pv, const LineArgs &a, Ends e) {
    if (e.lo > 0 || e.hi < pv.tokens) zero_rows(a.out, e.lo, e.hi, pv.tokens, a.hq * (D * (int)sizeof(T) / 16));
}

struct Piece {
    int h, tt, hc, tiles, tb, te;      // a unit of the cursor's owner, its tiles, the piece [tb, te) of them
};
// Position on the line.
struct Cursor {
    uint32_t w;                        // next tile
    uint32_t base;                     // first tile of owner o
    uint32_t ubase;                    // units before owner o
    uint32_t wh;                       // tiles of one kv head of owner o
    int o;
    Owner ow;
    OwnerTiles tl;
    Piece p;                           // the piece before w (tiles 0: none yet)
};

__device__ __forceinline__ void cursor_owner(Cursor &c, const PagedView &pv, const LineArgs &a, int o) {
    c.o = o;
    c.ow = owner_of(pv, a.mode, o);
    c.tl = owner_tiles(c.ow, a.geo, a.mode);
    c.wh = c.tl.all() * (uint32_t)a.geo.hc;
}

// The unit that holds tile `at` of the cursor's owner.  The whole warp calls it
// (the token tile is found by a 32-way search: a term of the sum is a few
// divisions, and a search by halves took 4 us at 125 token tiles).
__device__ __forceinline__ Piece unit_at(const Cursor &c, const LineGeo &g, uint32_t at) {
    Piece p;
    p.h = (int)(at / c.wh);
    const uint32_t rem = at - (uint32_t)p.h * c.wh, hc = (uint32_t)g.hc;
    int lo = 0, hi = c.tl.tt;
    if (!c.tl.causal) {
        lo = (int)(rem / (c.tl.fixed * hc));
    } else {
        const int lane = threadIdx.x & 31;
        while (hi - lo > 1) {
            const int step = (hi - lo + 31) >> 5, i = lo + (lane + 1) * step;
            const int n = __popc(__ballot_sync(0xffffffffu, i < hi && c.tl.before(i) * hc <= rem));
            lo += n * step;
            hi = min(hi, lo + step);
        }
    }
    p.tt = lo;
    p.tiles = (int)c.tl.of(lo);
    const uint32_t r = rem - c.tl.before(lo) * hc;
    p.hc = (int)(r / (uint32_t)p.tiles);
    p.tb = (int)(r - (uint32_t)p.hc * p.tiles);
    p.te = p.tiles;
    return p;
}

// The next piece of [.., w1); false at the end.  Leaves c.w behind it.
__device__ __forceinline__ bool next_piece(Cursor &c, const PagedView &pv, const LineArgs &a, uint32_t w1, Piece &p) {
    if (c.w >= w1) return false;
    bool step = c.p.tiles > 0;                         // the unit after the last one, if its owner has one
    while (c.w >= c.base + (uint32_t)pv.kv_heads * c.wh) {
        if (c.o + 1 >= a.owners) return false;
        c.base += (uint32_t)pv.kv_heads * c.wh;
        c.ubase += (uint32_t)(pv.kv_heads * c.tl.tt * a.geo.hc);
        cursor_owner(c, pv, a, c.o + 1);
        step = false;
    }
    if (step) {
        p = c.p;
        if (++p.hc == a.geo.hc) {
            p.hc = 0;
            if (++p.tt == c.tl.tt) {
                p.tt = 0;
                ++p.h;
            }
            p.tiles = (int)c.tl.of(p.tt);
        }
        p.tb = 0;
    } else if (c.w == c.base) {
        p = Piece{0, 0, 0, (int)c.tl.of(0), 0, 0};
    } else {
        p = unit_at(c, a.geo, c.w - c.base);
    }
    p.te = (int)min((uint32_t)p.tiles, p.tb + (w1 - c.w));
    c.w += (uint32_t)(p.te - p.tb);
    c.p = p;
    return true;
}

// Slot of a piece.  Where whole units go to `out`, a CTA leaves at most two
// pieces, its first and its last; else one number for every piece in line
// order (units started so far + CTA).
__device__ __forceinline__ int64_t slot_of(const Cursor &c, const Piece &p, const LineArgs &a, int cta) {
    if (a.direct) return 2 * (int64_t)cta + (p.tb == 0 ? 1 : 0);
    return (int64_t)c.ubase + ((int64_t)p.h * c.tl.tt + p.tt) * a.geo.hc + p.hc + cta;
}

__host__ __device__ __forceinline__ uint32_t tiles_per_cta(uint32_t W, uint32_t ctas, uint32_t least) {
    const uint32_t per = (W + ctas - 1) / ctas;
    return per > least ? per : least;
}

// A CTA's part of the line, in shared memory.
struct LineStart {
    Cursor c;
    uint32_t w1, per;
};

// Of this CTA: its part [c.w, w1) of the line and the owner it begins in (left
// in `start` too); false: nothing to do.  Unless direct, CTA 0 leaves the sums
// before each owner in a.cum.  All NT threads call it.
template <int NT>
__device__ __forceinline__ bool plan_line(const PagedView &pv, const LineArgs &a, LineStart &start, Cursor &c, uint32_t &w1,
                                          uint32_t &per) {
    constexpr int NW = NT / 32;
    __shared__ uint64_t red[2 * NW];
    Cursor &at = start.c;                              // written by the thread whose owner holds w0
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool writer = blockIdx.x == 0 && !a.direct;
    const uint32_t per_unit = (uint32_t)(pv.kv_heads * a.geo.hc);
    Owner w{};
    OwnerTiles tl{};
    auto weight = [&](int o) -> uint64_t {
        if (o >= a.owners) return 0;
        w = owner_of(pv, a.mode, o);
        if (blockIdx.x == 0 && (a.mode == kPrefix ? pv.plens[o] > pv.pcap : pv.lens[o] > pv.cap))
            report(pv.status, CBQ_FLAG_CORRUPT, (uint32_t)o);
        tl = owner_tiles(w, a.geo, a.mode);
        return (uint64_t)(per_unit * (uint32_t)tl.tt) << 32 | per_unit * tl.all();
    };
    // prefixes that are cut to their table, where they are not owners (a decode call without
    // room for any prefix has no line of them)
    if (blockIdx.x == 0 && pv.groups && (a.mode == kFull || (a.mode == kOwn && pv.pcap == 0)))
        for (int g = tid; g < pv.groups; g += NT)
            if (pv.plens[g] > pv.pcap) report(pv.status, CBQ_FLAG_CORRUPT, (uint32_t)g);
    // owners beyond the first NT: their sum first, the first NT below in one scan
    uint64_t rest = 0;
    for (int o = tid + NT; o < a.owners; o += NT) rest += weight(o);
    uint64_t x = weight(tid);
    uint64_t inc = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += y;
    }
    if (a.owners > NT)
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, d);
    if (lane == 31) {
        red[warp] = inc;
        red[NW + warp] = rest;
    }
    if (tid == 0) at.o = -1;
    __syncthreads();
    uint64_t before = 0, all = 0, total = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        if (i < warp) before += red[i];
        all += red[i];
        total += red[NW + i];
    }
    total += all;
    const uint32_t W = (uint32_t)total;
    per = tiles_per_cta(W, gridDim.x, (uint32_t)a.min_tiles);
    const uint32_t w0 = (uint32_t)min((uint64_t)per * blockIdx.x, (uint64_t)W);
    w1 = min(w0 + per, W);
    if (writer && tid == 0) a.cum[a.owners] = total;
    if (w0 >= w1 && !writer) return false;
    uint64_t run = 0;
    for (int o0 = 0;; ) {
        const int o = o0 + tid;
        const uint64_t ex = run + before + inc - x;
        if (o < a.owners) {
            if (writer) a.cum[o] = ex;
            if ((uint32_t)ex <= w0 && w0 < (uint32_t)ex + (uint32_t)x) {
                at.w = w0;
                at.base = (uint32_t)ex;
                at.ubase = (uint32_t)(ex >> 32);
                at.wh = tl.all() * (uint32_t)a.geo.hc;
                at.o = o;
                at.ow = w;
                at.tl = tl;
                at.p.tiles = 0;
                start.w1 = w1;
                start.per = per;
            }
        }
        run += all;
        o0 += NT;
        if (o0 >= a.owners || (!writer && (uint32_t)run > w0)) break;   // all seen, or the owner was among these
        x = weight(o0 + tid);
        inc = x;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += y;
        }
        __syncthreads();                              // red[] of the previous block of owners
        if (lane == 31) red[warp] = inc;
        __syncthreads();
        before = all = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            if (i < warp) before += red[i];
            all += red[i];
        }
    }
    __syncthreads();
    if (w0 >= w1 || at.o < 0) return false;
    c = at;
    return true;
}

// A cut unit (direct): the CTA its first piece is in, and how many it spans.
struct Cut {
    int i0, n;
    __device__ __forceinline__ const float *slot(const LineArgs &a, int k, int64_t floats) const {
        return a.part + (2 * (int64_t)(i0 + k) + (k == 0 ? 1 : 0)) * floats;
    }
};
__device__ __forceinline__ Cut cut_of(const Cursor &c, const Piece &p, uint32_t per) {
    const uint32_t w0 = c.w - (uint32_t)p.te;          // the unit's first tile (the cursor stands behind the piece)
    Cut x;
    x.i0 = (int)(w0 / per);
    x.n = (int)((w0 + (uint32_t)p.tiles - 1) / per) - x.i0 + 1;
    return x;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

}  // namespace cbq

namespace cbq_host {

// One launch of a line kernel: its shape, grid and part of the workspace.
struct LinePlan {
    cbq::LineGeo geo;
    int rows;                          // query rows of a slot
    int tile_rows;                     // > 0: tokens are packed in blocks of so many rows (whole tokens each)
    int grid, owners, mode, direct, min_tiles;
    int64_t slots, cum_off, part_off, end;
};

// The workspace begins with the arrival counters of direct lines: a fixed
// place, so calls of any shape may share a workspace.
constexpr int kCounts = 4096;
constexpr int64_t kCountBytes = kCounts * 4;

// Room of a planned line in the workspace from byte `off` on; false: more
// tiles than 32 bits count.
inline bool line_room(const cbq::PagedView &pv, int d, int64_t off, LinePlan *p) {
    p->owners = p->mode == cbq::kPrefix ? pv.groups : pv.seqs;
    const int64_t tt = p->mode == cbq::kOwn ? pv.seqs : pv.tokens / p->geo.tq + p->owners;
    const int64_t units = tt * p->geo.hc * pv.kv_heads;
    const int64_t keys = p->mode == cbq::kOwn ? pv.cap : (p->mode == cbq::kPrefix ? pv.pcap : (int64_t)pv.cap + pv.pcap);
    if (units * ((keys + 32) / p->geo.keys + 2) > 0x7fffffffll || p->grid > kCounts) return false;
    p->slots = p->direct ? 2 * (int64_t)p->grid : units + p->grid;
    p->cum_off = off;
    p->part_off = align_up(off + (p->owners + 1) * 8, 256);
    p->end = align_up(p->part_off + p->slots * ((int64_t)p->rows * (d + 2)) * 4, 256);
    return true;
}

// CTAs of `kern` that fit an SM, its shared memory limit raised first (asked
// of the driver once per kernel and device).
int resident_ctas(const void *kern, int threads, int smem, int *out);

// The tensor-core kernel for many query rows (cbq_paged_tile.cu): whether it
// takes the shape, its plan, and its launch.
bool tile_takes(const cbq_paged_cache *c);
int tile_plan(const cbq::PagedView &pv, int d, int G, int mode, bool two, int64_t off, LinePlan *p);
int tile_launch(const cbq_paged_cache *c, const cbq::PagedView &pv, const LinePlan &p, cbq::LineArgs a, cudaStream_t s);

}  // namespace cbq_host
