// paged_attn.cuh -- attention over a paged cache: the call as its kernels see it and how it is cut into work.
//
// An item is up to MR consecutive query rows of one kv head of one sequence; query row r of a sequence's kv head is q head
// r % group of its token r / group, so the heads that share K and V sit side by side and one pass over the rows serves them.
// A unit is one tile of kPaTile cache rows of an item.  The units of all items in a row -- sequence after sequence -- are cut
// into equal runs, one per block: ragged lengths, single tokens and prompts fill the SMs alike.  An item that lies in several
// runs is put together by a second launch from partials in the workspace.  Everything is found on the device, from the tables,
// so a captured call follows them.
#pragma once

#include "paged.cuh"
#include "tc_tcgen05.cuh"

namespace tc {

constexpr uint32_t kPaTile = 64;  // cache rows of a unit

// A partial: acc [mr][hd], m [mr], l [mr]; out = sum exp2(m - M) acc / sum exp2(m - M) l.  In f32 numbers.
__host__ __device__ constexpr size_t pagedSlot(uint32_t mr, uint32_t hd) { return (static_cast<size_t>(mr) * (hd + 2) + 7) & ~size_t(7); }
// An item that lies in several blocks' runs, as the first of them leaves it for the merge: `count` blocks, the k-th of them block
// (this one + k groups).  The first block's partial is in its second slot -- its run ends with the item -- and the others' in
// their first one.  count 0: nothing to join.
struct PagedJoin {
    uint32_t count, row0, rows, token0, kvHead, mr, groups, pad;  // rows: of the sequence's kv head; row0: the item's first
};

struct PagedAttnParams {
    PagedView c;
    const void *q;   // [tokens][nHeads][hd] f32 / fp16
    void *out;
    const float *ks, *vs;
    float *parts;            // two slots per block
    PagedJoin *joins;        // one per block
    uint32_t nHeads, group, box;  // box: cache rows of one TMA copy
    uint32_t tileTokens;          // tiles kernel: tokens of a query tile
    uint32_t out32;               // out is 32-byte aligned
    uint32_t minRows, maxRows;    // the kernel takes the sequences with so many query rows per kv head (minRows .. maxRows)
    float scaleLog2;
    int half;                // q and out are fp16
    uint32_t zero;           // 0 (releaseStage)
};

#ifdef __CUDACC__
// Quotients of numbers that are small as a rule: a 64-bit division takes some hundred cycles, and a block starts with a chain of them.
__device__ __forceinline__ uint64_t divide(uint64_t a, uint64_t b) {
    return ((a | b) >> 32) == 0u ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}
// sum of (a i + b) / m over i = 0 .. n - 1, rounded down each: term by term while there are few, else by Euclid's steps on (a, m):
// the lattice points under a line, counted by exchanging the axes (the reciprocity of floor sums in Graham, Knuth and Patashnik,
// Concrete Mathematics, 3.5)
__device__ __forceinline__ uint64_t floorSum(uint32_t n, uint32_t m, uint32_t a, uint64_t b0) {
    uint64_t sum = 0;
    if (n <= 24u) {
        const uint64_t q0 = divide(b0, m);
        uint32_t r = static_cast<uint32_t>(b0 - q0 * m), q = 0, part = 0;
        const uint32_t qa = a / m, ra = a - qa * m;
        for (uint32_t i = 0; i < n; ++i) {
            part += q;
            r += ra, q += qa;
            if (r >= m) r -= m, ++q;
        }
        return q0 * n + part;
    }
    uint64_t nn = n, mm = m, aa = a, b = b0;
    for (;;) {
        if (aa >= mm) {
            const uint64_t q = divide(aa, mm);
            sum += nn * (nn - 1) / 2 * q, aa -= q * mm;
        }
        if (b >= mm) {
            const uint64_t q = divide(b, mm);
            sum += nn * q, b -= q * mm;
        }
        const uint64_t top = aa * nn + b;
        if (top < mm) return sum;
        nn = divide(top, mm), b = top - nn * mm;
        const uint64_t x = mm;
        mm = aa, aa = x;
    }
}

// The work of one sequence: query rows per kv head, rows cached, and what its items need.
struct PagedSeq {
    uint32_t rows, len;  // query rows of a kv head (new tokens x group); cache rows
    int32_t before;      // cache rows ahead of the new tokens; negative: the first tokens see nothing
    uint32_t token0;     // first token

    // cache rows that the last of query rows [.., end) sees
    __device__ __forceinline__ uint32_t sees(uint32_t end, uint32_t group) const {
        const int32_t n = before + static_cast<int32_t>((end - 1u) / group) + 1;
        return n > 0 ? static_cast<uint32_t>(n) : 0u;
    }
    __device__ __forceinline__ uint32_t items(uint32_t MR) const { return (rows + MR - 1u) / MR; }
    // tiles of item m: one at least, which writes the zeros of rows that see nothing.  Where `before` is negative every item is
    // counted with the tiles of the whole sequence, so that the sum below keeps its closed form.
    __device__ __forceinline__ uint32_t tiles(uint32_t MR, uint32_t m, uint32_t group) const {
        const uint32_t n = before < 0 ? len : sees(min((m + 1u) * MR, rows), group);
        return max(1u, (n + kPaTile - 1u) / kPaTile);
    }
    // tiles of items 0 .. m - 1
    __device__ __forceinline__ uint64_t tilesBefore(uint32_t MR, uint32_t m, uint32_t group) const {
        if (m == 0u) return 0u;
        if (before < 0) return static_cast<uint64_t>(m) * tiles(MR, 0, group);
        const bool all = m == items(MR);
        const uint32_t n = all ? m - 1u : m;
        uint64_t sum = all ? tiles(MR, m - 1u, group) : 0u;
        // item i sees before + ((i + 1) MR - 1) / group + 1 rows: floor((group (before + kPaTile) + (i + 1) MR - 1) / (kPaTile group)) tiles
        if (n > 0u) sum += floorSum(n, kPaTile * group, MR, static_cast<uint64_t>(group) * (static_cast<uint32_t>(before) + kPaTile) + MR - 1u);
        return sum;
    }
    __device__ __forceinline__ uint64_t tilesAll(uint32_t MR, uint32_t group) const { return rows == 0u ? 0u : tilesBefore(MR, items(MR), group); }
};

// What the tables say of a sequence.  Read through L2: a block may look before the kernels ahead of it are complete (PagedWalk::prepare).
struct PagedRaw {
    uint32_t start, stop, len;
    __device__ __forceinline__ bool operator==(const PagedRaw &o) const { return start == o.start && stop == o.stop && len == o.len; }
};
__device__ __forceinline__ PagedRaw pagedRaw(const PagedAttnParams &p, uint32_t b) {
    PagedRaw r;
    if (p.c.starts != nullptr) r.start = __ldcg(p.c.starts + b), r.stop = __ldcg(p.c.starts + b + 1u);
    else r.start = b * p.c.perSeq, r.stop = r.start + p.c.perSeq;
    r.len = __ldcg(p.c.lens + b);
    return r;
}
// rows that a sequence has pages for
__device__ __forceinline__ uint32_t pagedMost(const PagedAttnParams &p) { return p.c.pagesPerSeq * p.c.pageRows; }
__device__ __forceinline__ PagedSeq pagedSeq(const PagedAttnParams &p, const PagedRaw &r) {
    const uint32_t stop = min(r.stop, p.c.tokens), n = stop > r.start ? stop - r.start : 0u;
    PagedSeq s;
    s.rows = n * p.group;
    if (s.rows < p.minRows || s.rows > p.maxRows) s.rows = 0u;
    s.len = min(r.len, pagedMost(p));
    s.before = static_cast<int32_t>(s.len) - static_cast<int32_t>(n);
    s.token0 = r.start;
    return s;
}

// A walk of a producer warp over its block's run of units, item by item.
struct PagedWalk {
    uint32_t mr, over;        // query rows of an item; units ahead of its tiles that stand for what an item costs beside them
    // Kv heads whose units lie in a row, and groups of blocks (block b: group b % groups).  Either all heads and one group, or a head
    // for each of nKV groups: the blocks of a sequence's heads then pass over the same cache rows at the same time, which are
    // neighbours in memory, and share the scales of an int8 row.
    uint32_t heads, groups, index;  // index: the block's in its group
    static constexpr uint32_t kHeld = 4;
    PagedRaw raw[kHeld];      // sequences lane, 32 + lane, ..
    uint64_t total, at, end;  // units of the group; the block's next and last
    uint32_t blocks;          // ... of the group; its blocks with work
    uint32_t seq, kvHead0, kvHead, item;
    uint64_t item0;           // first unit of the item
    uint32_t tiles;           // its tiles
    PagedSeq s;

    __device__ __forceinline__ uint64_t firstOf(uint32_t block) const { return divide(block * total, blocks); }
    __device__ __forceinline__ uint32_t blockOf(uint64_t unit) const { return static_cast<uint32_t>(divide((unit + 1u) * blocks - 1u, total)); }

    __device__ __forceinline__ uint64_t unitsAll(const PagedSeq &q, uint32_t group) const { return q.tilesAll(mr, group) + static_cast<uint64_t>(over) * q.items(mr); }
    __device__ __forceinline__ uint64_t unitsBefore(uint32_t m, uint32_t group) const { return s.tilesBefore(mr, m, group) + static_cast<uint64_t>(over) * m; }

    // What begin() finds in its first look, before the kernels ahead in the stream are complete: the chain of loads and quotients at a
    // block's start (4 us, most of it instructions that come from far) then passes under them.  As a rule the tables are older than
    // those kernels; start() looks again and begins anew where they were not.
    __device__ __forceinline__ bool prepare(const PagedAttnParams &p, uint32_t itemRows, uint32_t overhead, bool headsApart) {
        headsApart = headsApart && gridDim.x >= p.c.nKV;
        heads = headsApart ? 1u : p.c.nKV, groups = headsApart ? p.c.nKV : 1u;
        index = blockIdx.x / groups, kvHead0 = headsApart ? blockIdx.x - index * groups : 0u;
        look(p, raw);
        return begin(p, itemRows, overhead);
    }
    // Behind the wait for those kernels.  some: what prepare() said; kept: it stands.
    __device__ __forceinline__ bool start(const PagedAttnParams &p, bool some, bool &kept) {
        PagedRaw now[kHeld];
        look(p, now);
        const uint32_t lane = threadIdx.x & 31u;
        if (blockIdx.x == 0)
            for (uint32_t b = lane; b < p.c.batch; b += 32u)
                if (pagedRaw(p, b).len > pagedMost(p)) atomicOr(p.c.err, kDevErrRowBound);  // more rows than the table has pages for
        bool same = p.c.batch <= 32u * kHeld;
#pragma unroll
        for (uint32_t k = 0; k < kHeld; ++k) same = same && now[k] == raw[k], raw[k] = now[k];
        kept = __all_sync(0xffffffffu, same);
        return kept ? some : begin(p, mr, over);
    }
    __device__ __forceinline__ void look(const PagedAttnParams &p, PagedRaw (&r)[kHeld]) const {
        const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
        for (uint32_t k = 0; k < kHeld; ++k) r[k] = 32u * k + lane < p.c.batch ? pagedRaw(p, 32u * k + lane) : PagedRaw{0u, 0u, 0u};
    }

    // All lanes of the warp.  False: nothing to do.
    __device__ __forceinline__ bool begin(const PagedAttnParams &p, uint32_t itemRows, uint32_t overhead) {
        mr = itemRows, over = overhead;
        const uint32_t lane = threadIdx.x & 31u;
        auto unitsOf = [&](uint32_t b, const PagedRaw &r) { return b < p.c.batch ? unitsAll(pagedSeq(p, r), p.group) * heads : 0u; };
        uint64_t held[kHeld], sum = 0;  // units of the first sequences, out of registers; the others are looked up
#pragma unroll
        for (uint32_t k = 0; k < kHeld; ++k) held[k] = unitsOf(32u * k + lane, raw[k]), sum += held[k];
        for (uint32_t b = 32u * kHeld + lane; b < p.c.batch; b += 32u) sum += unitsOf(b, pagedRaw(p, b));
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        total = sum;
        if (total == 0u) return false;
        blocks = static_cast<uint32_t>(min(static_cast<uint64_t>(gridDim.x / groups), total));
        if (index >= blocks) return false;
        at = firstOf(index), end = firstOf(index + 1u);
        // the sequence that holds unit `at`
        uint64_t base = 0;
        bool have = false;
        PagedRaw found{0u, 0u, 0u};
        auto search = [&](uint32_t b0, uint64_t mine, const PagedRaw &r) {
            uint64_t upTo = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t x = __shfl_up_sync(0xffffffffu, upTo, o);
                if (lane >= static_cast<uint32_t>(o)) upTo += x;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, base + upTo > at);
            const int l = past != 0u ? __ffs(past) - 1 : 31;
            if (past != 0u) {
                have = true;
                seq = b0 + l;
                found.start = __shfl_sync(0xffffffffu, r.start, l), found.stop = __shfl_sync(0xffffffffu, r.stop, l), found.len = __shfl_sync(0xffffffffu, r.len, l);
            }
            base += __shfl_sync(0xffffffffu, past != 0u ? upTo - mine : upTo, l);
        };
#pragma unroll
        for (uint32_t k = 0; k < kHeld; ++k)
            if (!have && 32u * k < p.c.batch) search(32u * k, held[k], raw[k]);
        for (uint32_t b0 = 32u * kHeld; !have && b0 < p.c.batch; b0 += 32u) {
            const PagedRaw r = b0 + lane < p.c.batch ? pagedRaw(p, b0 + lane) : PagedRaw{0u, 0u, 0u};
            search(b0, unitsOf(b0 + lane, r), r);
        }
        if (!have) return false;  // (only where the tables changed meanwhile)
        s = pagedSeq(p, found);
        if (s.rows == 0u) return false;  // (only where the tables changed meanwhile)
        uint64_t in = at - base;
        kvHead = kvHead0;
        if (heads > 1u) {
            const uint64_t per = unitsAll(s, p.group);
            kvHead = static_cast<uint32_t>(divide(in, per));
            in -= kvHead * per;
        }
        // the last item that does not begin behind `in`, 32 candidates at a time
        uint32_t lo = 0, n = s.items(mr);
        while (n > 1u) {
            const uint32_t step = (n + 31u) / 32u, try_ = lo + lane * step;
            const uint32_t hits = __popc(__ballot_sync(0xffffffffu, lane * step < n && unitsBefore(try_, p.group) <= in));
            lo += (hits - 1u) * step;
            n = min(step, n - (hits - 1u) * step);
        }
        item = lo;
        item0 = at - in + unitsBefore(item, p.group);
        tiles = s.tiles(mr, item, p.group);
        return end - item0 > over;
    }
    // Tiles [first, last) of the item are the block's; the group's block that has its last one.
    __device__ __forceinline__ uint32_t first() const { return at - item0 > over ? static_cast<uint32_t>(at - item0 - over) : 0u; }
    __device__ __forceinline__ uint32_t last() const { return static_cast<uint32_t>(min(end - item0, static_cast<uint64_t>(tiles) + over)) - over; }
    __device__ __forceinline__ uint32_t lastBlock() const { return blockOf(item0 + over + tiles - 1u); }
    // On to the next item; false: the run is done.
    __device__ __forceinline__ bool next(const PagedAttnParams &p) {
        item0 += tiles + over;
        at = item0;
        if (at + over >= end) return false;  // (a run that ends in front of an item's tiles leaves it to the next block)
        if (++item == s.items(mr)) {
            item = 0;
            if (++kvHead == kvHead0 + heads) {
                kvHead = kvHead0;
                do {
                    if (++seq >= p.c.batch) return false;  // (not reached: the run is not done)
                    s = pagedSeq(p, pagedRaw(p, seq));
                } while (s.rows == 0u);
            }
        }
        tiles = s.tiles(mr, item, p.group);
        return true;
    }
};
__device__ __forceinline__ uint4 ldShared4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint32_t sub1152(uint32_t x) {
    const __half2 b = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    __half2 h = __hsub2(*reinterpret_cast<__half2 *>(&x), b);
    return *reinterpret_cast<uint32_t *>(&h);
}
// bytes 0, 1 (2, 3) of w, each xor-ed with 0x80, as fp16 pairs
__device__ __forceinline__ uint32_t bytesLo(uint32_t w) { return sub1152(__byte_perm(w, 0x64646464u, 0x4140)); }
__device__ __forceinline__ uint32_t bytesHi(uint32_t w) { return sub1152(__byte_perm(w, 0x64646464u, 0x4342)); }

// The block's entry for the merge; one thread, whether the block has work or not.
__device__ __forceinline__ void pagedLeaveJoin(const PagedAttnParams &p, const PagedWalk *w, uint32_t count) {
    PagedJoin j;
    j.count = count;
    if (count != 0u) j.row0 = w->item * w->mr, j.rows = w->s.rows, j.token0 = w->s.token0, j.kvHead = w->kvHead, j.mr = w->mr, j.groups = w->groups;
    p.joins[blockIdx.x] = j;
}
// What a block has of an item, as its producer hands it to the consumers: tiles t0 .. t0 + nTiles - 1 of it (nTiles 0: the run is
// done), query rows m0 .. of `rows`.
struct PaItem {
    uint32_t nTiles, t0, m0, rows, token0, kvHead, len, whole, part;
    int32_t before;
};
constexpr uint32_t kPaItems = 8;  // the ring's stages and two: a consumer may still write the results of an item whose tiles are all released

__device__ __forceinline__ void pagedStore(const PagedAttnParams &p, uint32_t hd, uint32_t token0, uint32_t kvHead, uint32_t r, uint32_t dim, const float4 &x) {
    const uint32_t tok = token0 + r / p.group, head = kvHead * p.group + r % p.group;
    const size_t at = (static_cast<size_t>(tok) * p.nHeads + head) * hd + dim;
    if (p.half) *reinterpret_cast<uint2 *>(static_cast<__half *>(p.out) + at) = make_uint2(packHalf2(x.x, x.y), packHalf2(x.z, x.w));
    else *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at) = x;
}

// A query row of f32 as fp16 pairs, four dims of it a step, dim(st) ..: put(st, {hi 0 1, hi 2 3, lo 0 1, lo 2 3}); the four lanes of a row work together.
// The row's largest goes to [2^10, 2^11), so that what the upper half leaves is a normal fp16 number.  Returns what undoes that.
template <int NS, typename D, typename P>
__device__ __forceinline__ float pagedQuery(const PagedAttnParams &p, const PaItem &it, uint32_t rr, bool valid, uint32_t hd, D &&dim, P &&put) {
    const uint32_t tok = it.token0 + rr / p.group, head = it.kvHead * p.group + rr % p.group;
    const float *src = static_cast<const float *>(p.q) + (static_cast<size_t>(tok) * p.nHeads + head) * hd;
    float4 x[NS];
    float top = 0.0f;
#pragma unroll
    for (int st = 0; st < NS; ++st) {
        x[st] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (valid) x[st] = __ldg(reinterpret_cast<const float4 *>(src + dim(st)));
        top = fmaxf(top, fmaxf(fmaxf(fabsf(x[st].x), fabsf(x[st].y)), fmaxf(fabsf(x[st].z), fabsf(x[st].w))));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float up = 1.0f, back = 1.0f;
    if (top > 0.0f && top < INFINITY) {
        const int e = min(126, max(-116, static_cast<int>(__float_as_uint(top) >> 23) - 127));
        up = __uint_as_float(static_cast<uint32_t>(127 + 10 - e) << 23);
        back = __uint_as_float(static_cast<uint32_t>(127 - 10 + e) << 23);
    }
#pragma unroll
    for (int st = 0; st < NS; ++st) {
        float h[4], l[4];
        splitHalf(x[st].x * up, h[0], l[0]);
        splitHalf(x[st].y * up, h[1], l[1]);
        splitHalf(x[st].z * up, h[2], l[2]);
        splitHalf(x[st].w * up, h[3], l[3]);
        const uint32_t w[4] = {packHalf2(h[0], h[1]), packHalf2(h[2], h[3]), packHalf2(l[0], l[1]), packHalf2(l[2], l[3])};
        put(st, w);
    }
    return back;
}

// The producer warp of the kernels whose consumers share a tile's rows (paged_rows.cu, paged_steps.cu): hands on the items of the block's run
// and requests their tiles into the ring, K and V and an int8 store's scales.  L: the kernel's layout.
template <typename L>
__device__ __forceinline__ void pagedProduce(const PagedAttnParams &p, const CUtensorMap &tmK, const CUtensorMap &tmV, uint8_t *smem, uint64_t *full,
                                             uint64_t *empty, uint64_t *itemFull, PaItem *items) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t g = 0;  // tiles so far
    const uint32_t boxes = kPaTile / p.box, boxBytes = p.box * 128u;
    PagedWalk w;
    uint32_t handed = 0;  // items
    bool ok = true;
    const bool some = w.prepare(p, L::MR, 0u, true);
    gridDepWait();
    gridDepLaunch();
    if (lane == 0) pagedLeaveJoin(p, nullptr, 0u);
    // Where this lane's box of a tile lies: looked up a tile ahead, and the first one's entry on its way beside the second look at the
    // tables.
    struct At {
        uint32_t have, in;
        int32_t page;
    };
    auto look = [&](uint32_t t) {
        const uint32_t row0 = t * kPaTile;
        At at{w.s.len > row0 ? min(boxes, (w.s.len - row0 + p.box - 1u) / p.box) : 0u, 0u, 0};
        if (lane < at.have) {
            const uint32_t row = row0 + lane * p.box, slot = row / p.c.pageRows;
            at.in = row - slot * p.c.pageRows;
            at.page = __ldg(p.c.pages + static_cast<size_t>(w.seq) * p.c.pagesPerSeq + slot);
        }
        return at;
    };
    At next{0u, 0u, 0};
    if (some) next = look(w.first());
    bool kept;
    const bool work = w.start(p, some, kept);
    if (work && !kept) next = look(w.first());
    if (work) do {
        const uint32_t t1 = w.last();
        if (lane == 0) {
            PaItem it;
            it.t0 = w.first(), it.nTiles = t1 - it.t0, it.m0 = w.item * L::MR, it.rows = w.s.rows, it.token0 = w.s.token0;
            it.kvHead = w.kvHead, it.len = w.s.len, it.before = w.s.before;
            it.whole = it.t0 == 0u && t1 == w.tiles, it.part = it.t0 == 0u ? 1u : 0u;  // (the item's first block uses its second slot)
            items[handed % kPaItems] = it;
            mbarArrive(&itemFull[handed % kPaItems]);
        }
        ++handed;
        if (handed > 1u) next = look(w.first());
        for (uint32_t t = w.first(); t < t1; ++t, ++g) {
            const uint32_t n = next.have, in = next.in;
            uint32_t page = static_cast<uint32_t>(next.page);
            next = look(t + 1u);
            if (lane < n && page >= p.c.numPages) {  // no such page: reported, page 0 stands in
                atomicOr(p.c.err, kDevErrRowBound);
                page = 0;
            }
            const uint32_t st = g % uint32_t(L::NST);
            if (g >= uint32_t(L::NST)) ok = pfWait<true>(&empty[st], ((g / uint32_t(L::NST)) - 1u) & 1u, p.c.err, kDevErrEmptyWait);
            if (!ok) break;
            if (lane == 0) mbarExpectTx(&full[st], n * boxBytes * 2u * L::kPanels);
            __syncwarp();
            uint8_t *stage = smem + st * L::kStage;
            if (lane < n) {
#pragma unroll
                for (int h = 0; h < L::kPanels; ++h) {
                    tmaLoad4D(stage + h * L::kPanel + lane * boxBytes, &tmK, &full[st], h * (L::kI8 ? 128 : 64), w.kvHead, in, page);
                    tmaLoad4D(stage + L::kMat + h * L::kPanel + lane * boxBytes, &tmV, &full[st], h * (L::kI8 ? 128 : 64), w.kvHead, in, page);
                }
            }
            if constexpr (L::kI8) {
                float *sc = reinterpret_cast<float *>(smem + L::kScales) + st * 128u;
#pragma unroll
                for (uint32_t u = 0; u < 2; ++u) {
                    const uint32_t key = lane + 32u * u, from = key / p.box;
                    const uint32_t pg = __shfl_sync(0xffffffffu, page, from), r = __shfl_sync(0xffffffffu, in, from) + key - from * p.box;
                    if (from < n) {
                        const size_t at = (static_cast<size_t>(pg) * p.c.pageRows + r) * p.c.nKV + w.kvHead;
                        cpAsync4(sc + key, p.ks + at);
                        cpAsync4(sc + 64u + key, p.vs + at);
                    }
                }
                cpAsyncMbarArriveNoinc(&full[st]);
            }
        }
        // (the quotient waits until the tiles are on their way)
        if (lane == 0 && w.first() == 0u && t1 != w.tiles) pagedLeaveJoin(p, &w, w.lastBlock() - w.index + 1u);
    } while (ok && w.next(p));
    if (lane == 0) {
        items[handed % kPaItems].nTiles = 0u;
        mbarArrive(&itemFull[handed % kPaItems]);
    }
    // no copy is under way any more when the block leaves
    for (uint32_t back = 1; back <= uint32_t(L::NST) && back <= g; ++back)
        if (!pfWait<true>(&full[(g - back) % uint32_t(L::NST)], ((g - back) / uint32_t(L::NST)) & 1u, p.c.err, kDevErrFullWait)) break;
}
#endif

// paged_tiles.cu: the sequences of minRows query rows per kv head and more, fp16 queries, on tcgen05
int pagedAttnTiles(const tc_paged_kv *c, const PagedAttnParams &p, cudaStream_t st, uint32_t *blocks);
// paged_rows.cu: the same for f32 queries over fp16 pages of head_dim 64 and 128
int pagedAttnRows(const tc_paged_kv *c, const PagedAttnParams &p, cudaStream_t st, uint32_t *blocks);
constexpr int kPagedSMs = 148;      // blocks that the workspace has room for, per block of an SM
constexpr uint32_t kPagedTile = 128;  // query rows of a tile of the tiles kernel

// The workspace: two partials per block of the two kernels' widest grids, then what the merge finds per block.
constexpr size_t kStepsParts = size_t(2) * kPagedSMs * 3 * pagedSlot(16, 128);  // f32
constexpr size_t kTilesParts = size_t(2) * kPagedSMs * pagedSlot(2 * kPagedTile, 128);
static_assert(pagedSlot(2 * kPagedTile, 128) >= pagedSlot(kPagedTile, 256), "one query tile at head_dim 256");
constexpr size_t kPagedWorkspace = (kStepsParts + kTilesParts) * 4 + size_t(kPagedSMs) * 5 * sizeof(PagedJoin) + 32;

// paged_steps.cu: any sequences, best for few query rows; rows: how many a sequence brings as a rule, for the choice of a form
int pagedAttnSteps(const tc_paged_kv *c, const PagedAttnParams &p, uint32_t rows, cudaStream_t st, uint32_t *blocks);

int pagedMaps(const tc_paged_kv *c, uint32_t box, CUtensorMap *k, CUtensorMap *v);  // maps of the pools, `box` rows a copy

}  // namespace tc
