// paged_tiles.cu -- attention of many query rows per kv head over a paged cache on tcgen05 (fp16 queries and results, f32
// accumulation in TMEM): chunks of prompts and whole prompts.
//
// The block is prefill_f16.cu's: two 128-row query tiles A and B share a ring of 64-row K and V tiles, warps 0-3 / 4-7 hold the softmax of
// A / B a thread per row, warp 8 requests (fp16 V: warp 13), warps 9, 10 issue S = Q K^T and warps 11, 12 O += P V with P in TMEM over the
// scores' buffer.
// What differs is what a tile is and where it comes from:
//   * a query tile holds tileTokens tokens x the q heads of one kv head (row = token x group + head; one TMA box), so a
//     pass over the cache serves all of them and the causal edge is tileTokens rows wide instead of 128;
//   * K and V tiles are gathered page by page, a TMA copy per `box` rows, issued by the lanes of the producer warp side by side;
//   * the work is the runs of paged_attn.cuh: a block's run of tiles may begin and end inside an item, whose partials the
//     merge launch joins.  An item of one query tile gives its KV tiles to the two halves in turn (even / odd);
//   * an int8 store's tiles go through three converter warps (13 - 15) to fp16 integers, exactly; a row's K scale comes to its
//     scores and its V scale to its probabilities in f32.  The running maximum is then one of score + log2 of the largest V
//     scale of the tile, so that what P holds stays in range;
//   * rows past the sequence may hold anything: scores there are masked by selects, and the warp that issues P V writes zeros
//     over V's.
// What bounds it is the loop through the score buffer that prefill_f16.cu describes: a step of 64 cache rows and 256 query rows takes
// 1.03 us (512 tokens of 28 / 4 / 128 behind 14336 - 28672 rows), over int8 pages 1.6 with the two multiplications by scales
// per score and the conversions.  Four whole prompts of 28 / 4 / 128 run at 0.57 of the bf16 burst rate, 512 tokens behind
// 28672 rows at 0.6.
#include <algorithm>
#include <cstring>

#include "paged_attn.cuh"
#include "tc_tcgen05.cuh"

namespace tc {

constexpr int kPtScales = 132;          // f32 of a scale slot: K's 64, V's 64, the power of two above V's; padding
constexpr uint32_t kPtScaleSlots = 16;
// What an item costs beside its tiles, in tiles: four whole prompts take 371 us with 0, 340 with 2, 347 with 3 and 358 with 6.
constexpr uint32_t kPtOver = 2;
constexpr int kPtBN = int(kPaTile);
constexpr float kPtLazyLog2 = 8.0f;  // O is rescaled when the row's maximum ran ahead by 2^8
constexpr float kPtOff = 6.0f;       // probabilities are held as 2^6 p, at most 2^14: what fp16 has above them goes to the small ones
// int8: the running maximum counts a tile's V scales as 2^-60 at least.  Scales of 0 would take 2^126 into the probabilities, which f32 does not
// hold: inf in the row's sum, inf x 0 in P.  At 2^-60 probabilities stay below 2^(60 + 14), what P holds stays below 2^14 as
// with any larger scale, and what smaller scales add (V below 127 x 2^-60) is 0 in an fp16 result.
constexpr int kPtLeastScale = -60;

// What a block has of an item, as its producer hands it to the other warps (in shared memory: the walk's state would cost the softmax
// threads registers that they spill for).  Tiles j = 0 .. nTiles - 1 are cache rows 64 (t0 + j) ..; query tile X takes tile j if
// mine(X, j).  nTiles 0: the run is done.
struct PtItem {
    uint32_t nTiles, t0, nA, nB;
    uint32_t m0, rowsA, rowsB;                // first row; rows of A and B
    uint32_t split, whole;                    // one query tile for both halves; the item is the block's alone
    uint32_t seq, kvHead, token0, len, part;  // part: the partial's slot
    int32_t before;
    uint32_t pad;
    __device__ __forceinline__ bool mine(uint32_t x, uint32_t j) const { return split ? (j & 1u) == x : j < (x == 0u ? nA : nB); }
};
constexpr uint32_t kPtItems = 8;  // (the producer is two items ahead of the score products, which are at most two tiles ahead of the softmax)
template <bool ONE>
__device__ __forceinline__ PtItem ptItem(const PagedAttnParams &p, const PagedWalk &w, uint32_t &joins) {
    PtItem it;
    const uint32_t tile = p.tileTokens * p.group;
    it.m0 = w.item * w.mr;
    const uint32_t rows = min(w.mr, w.s.rows - it.m0);
    it.rowsA = min(rows, tile), it.rowsB = rows - it.rowsA;
    it.t0 = w.first();
    const uint32_t t1 = w.last();
    it.nTiles = t1 - it.t0;
    it.whole = it.t0 == 0u && t1 == w.tiles;
    it.split = !ONE && it.rowsB == 0u;
    if (it.split) {
        it.nB = it.nTiles / 2u, it.nA = it.nTiles - it.nB;
    } else {
        // A's rows end before B's
        const uint32_t tilesA = it.rowsB == 0u ? w.tiles : min(w.tiles, max(1u, (w.s.sees(it.m0 + it.rowsA, p.group) + kPaTile - 1u) / kPaTile));
        it.nA = min(t1, tilesA) > it.t0 ? min(t1, tilesA) - it.t0 : 0u;
        it.nB = it.rowsB != 0u ? it.nTiles : 0u;
    }
    it.seq = w.seq, it.kvHead = w.kvHead, it.token0 = w.s.token0, it.len = w.s.len, it.before = w.s.before;
    it.part = it.t0 == 0u ? 1u : 0u, it.pad = 0;  // (the item's first block uses its second slot)
    joins = it.part && !it.whole ? w.lastBlock() - w.index + 1u : 0u;
    return it;
}

template <int HD, bool I8>
struct PtL {
    static constexpr int kThreads = I8 ? 512 : 448;
    static constexpr int kHalves = HD / 64;
    static constexpr int kQTiles = HD > 128 ? 1 : 2;
    static constexpr int NK = HD > 128 ? 2 : I8 ? 3 : 6, NV = HD > 128 ? 2 : I8 ? 3 : 4;
    static constexpr int NS = !I8 ? 0 : HD > 128 ? 3 : 6;      // int8: 64 x 128 byte panels on their way to the converters
    static constexpr int kPanels = I8 ? HD / 128 : 1;          // ... of a tile
    static constexpr int kQHalf = int(kPagedTile) * 128;
    static constexpr int kKvHalf = kPtBN * 128;
    static constexpr int kQTile = kHalves * kQHalf;
    static constexpr int kKvTile = kHalves * kKvHalf;
    static constexpr int kQ = 0;
    static constexpr int kK = kQTiles * kQTile;
    static constexpr int kV = kK + NK * kKvTile;
    static constexpr int kStaging = kV + NV * kKvTile;
    static constexpr int kScale = kStaging + NS * kKvHalf;
    static constexpr int kExch = kScale + (I8 ? int(kPtScaleSlots) * kPtScales * 4 : 0);  // [half][row] (m, l) of items of one tile
    static constexpr int kBars = kExch + (HD > 128 ? 0 : 2 * int(kPagedTile) * 8);
    // qFull, kFull + kEmpty, vFull + vEmpty, sFull[2][2], pFull[2][2], pvDone[2], pvBuf[2][2], qFree[2], exFull, exRead, sFree[2],
    // stFull + stEmpty, itemFull
    static constexpr int kNumBars = 1 + 2 * NK + 2 * NV + 4 + 4 + 2 + 4 + 2 + 2 + 2 + 2 * NS + int(kPtItems);
    static constexpr int kTmemSlot = kBars + kNumBars * 8;
    static constexpr int kItems = (kTmemSlot + 16 + 15) / 16 * 16;
    static constexpr int kTotal = kItems + int(kPtItems) * int(sizeof(PtItem));
    static_assert(kTotal <= 227 * 1024, "shared memory of an SM");
};

template <int HD, bool I8>
__global__ void __launch_bounds__((PtL<HD, I8>::kThreads), 1)
pagedTilesKernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ PagedAttnParams p) {
    using L = PtL<HD, I8>;
    constexpr int NC = kPtBN / 32;  // 32-column chunks of a score row
    constexpr uint32_t NK = L::NK, NV = L::NV, NS = L::NS, BN = kPtBN;
    constexpr bool kCall = HD < 256;
    constexpr bool kOne = L::kQTiles == 1;
    constexpr bool kAhead = kOne;   // one score buffer and two for probabilities (prefill_f16.cu)
    extern __shared__ __align__(1024) uint8_t smem[];  // (head_dim 128 has no room to round the address up)
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBars);
    uint64_t *qFull = bars, *kFull = bars + 1, *kEmpty = kFull + NK, *vFull = kEmpty + NK, *vEmpty = vFull + NV, *sFull = vEmpty + NV /* [x][b] */,
             *pFull = sFull + 4 /* [x][b] */, *pvDone = pFull + 4 /* [x] */, *pvBuf = pvDone + 2 /* [x][b] */, *qFree = pvBuf + 4 /* [x] */,
             *exFull = qFree + 2, *exRead = exFull + 1, *sFree = exRead + 1 /* [x] */, *stFull = sFree + 2, *stEmpty = stFull + NS, *itemFull = stEmpty + NS;
    PtItem *items = reinterpret_cast<PtItem *>(smem + L::kItems);
    uint32_t *tmemSlot = reinterpret_cast<uint32_t *>(smem + L::kTmemSlot);
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u;
    unsigned int *const err = p.c.err;

    if ((smemAddr(smem) & 1023u) != 0u) {  // the swizzle needs it; reported like the other resource that a block may not get
        if (threadIdx.x == 0) {
            gridDepWait();
            pagedLeaveJoin(p, nullptr, 0u);
            atomicOr(err, kDevErrTmemAlloc);
        }
        return;
    }
    if (threadIdx.x == 0) {
        mbarInit(qFull, 1);
        const uint32_t users = kOne ? 1u : 2u;  // a K (V) tile is released by the score (P.V) warps of both query tiles
        for (uint32_t s = 0; s < NK; ++s) mbarInit(&kFull[s], L::kPanels), mbarInit(&kEmpty[s], users);
        for (uint32_t s = 0; s < NV; ++s) mbarInit(&vFull[s], L::kPanels), mbarInit(&vEmpty[s], users);
        for (uint32_t s = 0; s < NS; ++s) mbarInit(&stFull[s], 1), mbarInit(&stEmpty[s], 1);
        for (int i = 0; i < 4; ++i) {
            mbarInit(&sFull[i], 1);
            mbarInit(&pFull[i], 4);  // one arrival per warp
            mbarInit(&pvBuf[i], 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbarInit(&sFree[x], 4);
            mbarInit(&pvDone[x], 1);
            mbarInit(&qFree[x], 1);
        }
        for (uint32_t i = 0; i < kPtItems; ++i) mbarInit(&itemFull[i], 1);
        mbarInit(exFull, 2 * kPagedTile);
        mbarInit(exRead, 2 * kPagedTile);
        fenceBarrierInit();
        tmaPrefetchDesc(&tmQ);
        tmaPrefetchDesc(&tmK);
        tmaPrefetchDesc(&tmV);
    }
    if (warp == 0) {
        tmemAlloc(tmemSlot, 512);
        tmemRelinquish();
        tcFenceBefore();
    }
    __syncthreads();
    tcFenceAfter();
    const uint32_t tmemBase = *reinterpret_cast<volatile uint32_t *>(tmemSlot);
    const uint32_t tileRows = p.tileTokens * p.group;
    if (warp != 8) {
        gridDepWait();
        gridDepLaunch();
    }
    // The n-th item of the block, once the producer has put it down; false: there is none any more.
    auto takeItem = [&](uint32_t n, const PtItem *&it) {
        it = &items[n % kPtItems];
        return pfWait<kCall>(&itemFull[n % kPtItems], (n / kPtItems) & 1u, err, kDevErrFullWait) && it->nTiles != 0u;
    };

    // ---- requests: a copy per box of a tile, by the lanes side by side ----
    // Where this lane's box of tile j lies.  Looked up a tile ahead of its first use: a request that waits for its table entry falls
    // behind the products.
    struct At {
        uint32_t have, in;
        int32_t page;
    };
    const uint32_t boxes = BN / p.box, boxBytes = p.box * 128u;
    auto tableOf = [&](const PtItem &it) { return p.c.pages + static_cast<size_t>(it.seq) * p.c.pagesPerSeq; };
    auto look = [&](const PtItem &it, const int32_t *table, uint32_t j) {
        const uint32_t row0 = (it.t0 + j) * BN;
        At at{it.len > row0 ? min(boxes, (it.len - row0 + p.box - 1u) / p.box) : 0u, 0u, 0};
        if (lane < at.have) {
            const uint32_t row = row0 + lane * p.box, slot = row / p.c.pageRows;
            at.in = row - slot * p.c.pageRows;
            at.page = __ldg(table + slot);
        }
        return at;
    };
    auto pageOf = [&](const At &at) {
        uint32_t page = static_cast<uint32_t>(at.page);
        if (lane < at.have && page >= p.c.numPages) {  // no such page: reported, page 0 stands in
            atomicOr(err, kDevErrRowBound);
            page = 0;
        }
        return page;
    };
    // an item's tiles of K or V, fp16
    auto requestTiles = [&](const PtItem &it, const CUtensorMap *map, uint32_t base, uint64_t *full, uint64_t *empty, uint32_t &g, uint32_t N) {
        const int32_t *table = tableOf(it);
        At next = look(it, table, 0);
        for (uint32_t j = 0; j < it.nTiles; ++j, ++g) {
            const At at = next;
            next = look(it, table, j + 1u);
            const uint32_t page = pageOf(at), s = g % N;
            if (g >= N && !pfWait<kCall>(&empty[s], ((g / N) - 1u) & 1u, err, kDevErrEmptyWait)) return false;
            if (lane == 0) mbarExpectTx(&full[s], at.have * boxBytes * L::kHalves);
            __syncwarp();
            if (lane < at.have) {
#pragma unroll
                for (int h = 0; h < L::kHalves; ++h)
                    tmaLoad4D(smem + base + s * L::kKvTile + h * L::kKvHalf + lane * boxBytes, map, &full[s], 64 * h, it.kvHead, at.in, page);
            }
        }
        return true;
    };
    // the panels of one tile, int8
    auto requestPanels = [&](const PtItem &it, const At &at, const CUtensorMap *map, uint32_t &gs) {
        const uint32_t page = pageOf(at);
#pragma unroll
        for (int h = 0; h < L::kPanels; ++h, ++gs) {
            const uint32_t s = gs % (NS ? NS : 1u);
            if (gs >= NS && !pfWait<kCall>(&stEmpty[s], ((gs / (NS ? NS : 1u)) - 1u) & 1u, err, kDevErrEmptyWait)) return false;
            if (lane == 0) mbarExpectTx(&stFull[s], at.have * boxBytes);
            __syncwarp();
            if (lane < at.have) tmaLoad4D(smem + L::kStaging + s * L::kKvHalf + lane * boxBytes, map, &stFull[s], 128 * h, it.kvHead, at.in, page);
        }
        return true;
    };
    // The last release of every slot has to have arrived before the block leaves; where somebody gave up, the copies under way
    // still have to land.
    auto drain = [&](uint64_t *bar, uint32_t count, uint32_t N, uint32_t bit) {
        for (uint32_t back = 1; back <= N && back <= count; ++back)
            if (!pfWait<kCall>(&bar[(count - back) % N], ((count - back) / N) & 1u, err, bit)) return false;
        return true;
    };

    if (warp == 8) {
        // ------------------------------- producer -------------------------------
        uint32_t gk = 0, gs = 0, n = 0;
        PagedWalk w;
        // (heads apart: four whole prompts 316 -> 309 us; not where it would leave blocks without work)
        const bool some = w.prepare(p, tileRows * L::kQTiles, kPtOver, gridDim.x % p.c.nKV == 0u);
        gridDepWait();
        gridDepLaunch();
        if (lane == 0) pagedLeaveJoin(p, nullptr, 0u);
        bool ok = true, kept;
        if (w.start(p, some, kept)) do {
            uint32_t joins;
            const PtItem it = ptItem<kOne>(p, w, joins);
            if (lane == 0) {
                items[n % kPtItems] = it;
                mbarArrive(&itemFull[n % kPtItems]);
                if (joins != 0u) pagedLeaveJoin(p, &w, joins);
            }
            ++n;
            // the query tiles are free once the last score products of the previous item are complete
            if (n > 1u)
                ok = pfWait<kCall>(&qFree[0], n & 1u, err, kDevErrEmptyWait) && (kOne || pfWait<kCall>(&qFree[1], n & 1u, err, kDevErrEmptyWait));
            if (!ok) break;
            if (lane == 0) {
                const uint32_t qTiles = it.rowsB != 0u ? 2u : 1u;
                mbarExpectTx(qFull, qTiles * L::kHalves * tileRows * 128u);
                for (uint32_t x = 0; x < qTiles; ++x)
#pragma unroll
                    for (int h = 0; h < L::kHalves; ++h)
                        tmaLoad3D(smem + L::kQ + x * L::kQTile + h * L::kQHalf, &tmQ, qFull, 64 * h, w.kvHead * p.group,
                                  w.s.token0 + it.m0 / p.group + x * p.tileTokens);
            }
            __syncwarp();
            if constexpr (I8) {  // K two tiles ahead of V, panel by panel to the converters
                const int32_t *table = tableOf(it);
                At a0 = look(it, table, 0), a1 = look(it, table, 1), a2 = look(it, table, 2);
                ok = requestPanels(it, a0, &tmK, gs) && (it.nTiles < 2u || requestPanels(it, a1, &tmK, gs));
                for (uint32_t j = 0; ok && j < it.nTiles; ++j) {
                    const At a3 = look(it, table, j + 3u);
                    ok = (j + 2u >= it.nTiles || requestPanels(it, a2, &tmK, gs)) && requestPanels(it, a0, &tmV, gs);
                    a0 = a1, a1 = a2, a2 = a3;
                }
            } else {
                ok = requestTiles(it, &tmK, L::kK, kFull, kEmpty, gk, NK);
            }
        } while (ok && w.next(p));
        if (lane == 0) {
            items[n % kPtItems].nTiles = 0u;
            mbarArrive(&itemFull[n % kPtItems]);
        }
        if (ok && n != 0u)  // the query tiles' last release, like those of the slots
            ok = pfWait<kCall>(&qFree[0], (n - 1u) & 1u, err, kDevErrEmptyWait) && (kOne || pfWait<kCall>(&qFree[1], (n - 1u) & 1u, err, kDevErrEmptyWait));
        if (!ok && n != 0u) pfWait<kCall>(qFull, (n - 1u) & 1u, err, kDevErrFullWait);
        if constexpr (I8) {
            if (!ok || !drain(stEmpty, gs, NS ? NS : 1u, kDevErrEmptyWait)) drain(stFull, gs, NS ? NS : 1u, kDevErrFullWait);
        } else if (!ok || !drain(kEmpty, gk, NK, kDevErrEmptyWait)) {
            drain(kFull, gk, NK, kDevErrFullWait);
        }
    } else if (!I8 && warp == 13) {
        // ---------------------- producer of V (page by page, one warp's requests are late) ----------------------
        uint32_t gv = 0;
        bool ok = true;
        const PtItem *at;
        for (uint32_t n = 0; ok && takeItem(n, at); ++n) {
            const PtItem it = *at;
            ok = requestTiles(it, &tmV, L::kV, vFull, vEmpty, gv, NV);
        }
        if (!ok || !drain(vEmpty, gv, NV, kDevErrEmptyWait)) drain(vFull, gv, NV, kDevErrFullWait);
    } else if (I8 && warp >= 13) {
        // ------------------------------ converters -----------------------------------
        // Panels of 64 rows x 128 int8 in the order of the producer's requests, one warp each in turn, into two fp16 halves: rows of 64 dims
        // under the same 128-byte swizzle.  K's converter of a tile brings its scales, and zero for V's past the sequence: what stands
        // there is no number that a probability of 0 could be multiplied with.
        const uint32_t me = warp - 13u;
        uint32_t gs = 0, gk = 0, gv = 0;
        bool ok = true;
        const PtItem *at;
        for (uint32_t n = 0; ok && takeItem(n, at); ++n) {
            const PtItem it = *at;
            const int32_t *table = p.c.pages + static_cast<size_t>(it.seq) * p.c.pagesPerSeq;
            auto convert = [&](uint32_t j, bool isK) {
                uint32_t &g = isK ? gk : gv;
                const uint32_t N = isK ? NK : NV, d = g % N;
                uint64_t *full = isK ? kFull : vFull, *empty = isK ? kEmpty : vEmpty;
#pragma unroll
                for (int h = 0; h < L::kPanels; ++h, ++gs) {
                    if (gs % 3u != me) continue;
                    const uint32_t s = gs % (NS ? NS : 1u);
                    if (g >= N && !pfWait<kCall>(&empty[d], ((g / N) - 1u) & 1u, err, kDevErrEmptyWait)) return false;
                    if (isK && h == 0) {
                        // (a slot's last tile has been through the softmax: its score product was issued 16 - NK tiles ago)
                        float *sc = reinterpret_cast<float *>(smem + L::kScale) + (g % kPtScaleSlots) * kPtScales;
                        const uint32_t row0 = (it.t0 + j) * BN;
                        uint32_t top = 0u;
#pragma unroll
                        for (uint32_t u = 0; u < 2; ++u) {
                            const uint32_t key = lane + 32u * u, row = row0 + key;
                            float a = 0.0f, b = 0.0f;
                            if (row < it.len) {
                                const uint32_t slot = row / p.c.pageRows;
                                uint32_t page = static_cast<uint32_t>(__ldg(table + slot));
                                if (page >= p.c.numPages) page = 0;
                                const size_t at = (static_cast<size_t>(page) * p.c.pageRows + (row - slot * p.c.pageRows)) * p.c.nKV + it.kvHead;
                                a = __ldg(p.ks + at), b = __ldg(p.vs + at);
                            }
                            sc[key] = a, sc[64u + key] = b;
                            top = max(top, __float_as_uint(b) & 0x7fffffffu);
                        }
                        top = __reduce_max_sync(0xffffffffu, top);
                        // 2^that is above every scale; bounded below, see kPtLeastScale
                        if (lane == 0) sc[128] = static_cast<float>(max(static_cast<int>(top >> 23) - 126, kPtLeastScale));
                    }
                    if (!pfWait<kCall>(&stFull[s], (gs / (NS ? NS : 1u)) & 1u, err, kDevErrFullWait)) return false;
                    const uint32_t src = smemAddr(smem + L::kStaging + s * L::kKvHalf), dst = smemAddr(smem + (isK ? L::kK : L::kV) + d * L::kKvTile + 2 * h * L::kKvHalf);
#pragma unroll 4
                    for (uint32_t i = 0; i < 16u; ++i) {
                        const uint32_t row = (lane & 7u) + 8u * (i >> 1), q = (lane >> 3) + 4u * (i & 1u), x = row & 7u;
                        const uint4 v = ldShared4(src + row * 128u + ((q ^ x) << 4));
                        const uint32_t a[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
                        const uint32_t out = dst + (q >> 2) * L::kKvHalf + row * 128u, c = 2u * (q & 3u);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(out + ((c ^ x) << 4)), "r"(bytesLo(a[0])), "r"(bytesHi(a[0])), "r"(bytesLo(a[1])), "r"(bytesHi(a[1])) : "memory");
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(out + (((c + 1u) ^ x) << 4)), "r"(bytesLo(a[2])), "r"(bytesHi(a[2])), "r"(bytesLo(a[3])), "r"(bytesHi(a[3])) : "memory");
                    }
                    fenceProxyAsync();  // the tensor cores read what this warp wrote; TMA writes next what it read
                    __syncwarp();
                    if (lane == 0) {
                        mbarArrive(&full[d]);
                        mbarArrive(&stEmpty[s]);
                    }
                }
                ++g;
                return true;
            };
            ok = convert(0, true) && (it.nTiles < 2u || convert(1, true));
            for (uint32_t j = 0; ok && j < it.nTiles; ++j) ok = (j + 2u >= it.nTiles || convert(j + 2u, true)) && convert(j, false);
        }
    } else if (warp >= 9 && warp < 13) {
        // ------------------------------- MMA issuers -------------------------------
        // t counts the tiles of X over all items; tile t uses score buffer t % 2, which P(t - 2) has to have left (kAhead: the softmax
        // threads have to have read S(t - 1)).  A tile that is not X's is released all the same, once it is there: a warp that ran ahead would
        // hand in the release of a later round.
        const uint32_t x = (warp - 9u) & 1u;
        const bool pvRole = warp >= 11u;
        constexpr uint32_t idQK = umaInstrDescF16(kPagedTile, BN, 0, 0);
        constexpr uint32_t idPV = umaInstrDescF16(kPagedTile, HD, 0, 1);
        const uint64_t dQ0 = umaSmemDesc(smemAddr(smem + L::kQ), 16, 1024);
        const uint64_t dK0 = umaSmemDesc(smemAddr(smem + L::kK), 16, 1024);
        const uint64_t dV0 = umaSmemDesc(smemAddr(smem + L::kV), L::kKvHalf, 1024);
        const uint32_t tO = tmemBase + 128u * x, tS0 = tmemBase + 256u + 128u * x;
        uint32_t g = 0, t = 0;
        bool ok = !(kOne && x == 1u);
        const PtItem *at;
        for (uint32_t n = 0; ok && takeItem(n, at); ++n) {
            const PtItem it = *at;
            const uint32_t myTiles = x == 0 ? it.nA : it.nB;
            const uint64_t dQ = descAdvance(dQ0, it.split ? 0u : x * L::kQTile);
            uint32_t tt = t;
            for (uint32_t j = 0; ok && j < it.nTiles; ++j) {
                const uint32_t gg = g + j;
                const bool mine = it.mine(x, j);
                if (!pvRole) {
                    const uint32_t s = gg % NK;
                    if (mine && tt == t) ok = pfWait<kCall>(qFull, n & 1u, err, kDevErrFullWait);
                    ok = ok && pfWait<kCall>(&kFull[s], (gg / NK) & 1u, err, kDevErrFullWait);
                    if (mine) {
                        if (kAhead) {
                            if (ok && tt >= 1u) ok = pfWait<kCall>(&sFree[x], (tt - 1u) & 1u, err, kDevErrMmaWait);
                        } else if (ok && tt >= 2u) {
                            ok = pfWait<kCall>(&pvBuf[2u * x + (tt & 1u)], ((tt - 2u) >> 1) & 1u, err, kDevErrMmaWait);
                        }
                        if (!ok) break;
                        tcFenceAfter();
                        const uint64_t dK = descAdvance(dK0, s * L::kKvTile);
                        if (electOne()) {
#pragma unroll
                            for (uint32_t ks = 0; ks < HD / 16; ++ks)
                                umaMmaSS(tS0 + (kAhead ? 0u : 64u * (tt & 1u)), descAdvance(dQ, (ks >> 2) * L::kQHalf + (ks & 3u) * 32u),
                                         descAdvance(dK, (ks >> 2) * L::kKvHalf + (ks & 3u) * 32u), idQK, ks > 0 ? 1u : 0u);
                            umaCommit(&sFull[kAhead ? x : 2u * x + (tt & 1u)]);
                            if (tt + 1u == t + myTiles) umaCommit(&qFree[x]);
                            umaCommit(&kEmpty[s]);
                        }
                        ++tt;
                    } else if (ok && electOne()) {
                        umaCommit(&kEmpty[s]);
                    }
                    __syncwarp();
                } else {
                    const uint32_t s = gg % NV;
                    ok = pfWait<kCall>(&vFull[s], (gg / NV) & 1u, err, kDevErrFullWait);
                    if (mine) {
                        const uint32_t row0 = (it.t0 + j) * BN;
                        if (!I8 && ok && row0 + BN > it.len) {
                            // rows past the sequence: zeros, whatever the pages (or an earlier tile) left there
                            const uint32_t keep = it.len > row0 ? it.len - row0 : 0u;
                            const uint32_t base = smemAddr(smem + L::kV + s * L::kKvTile);
                            for (uint32_t i = lane; i < (BN - keep) * 8u * L::kHalves; i += 32u) {
                                const uint32_t chunk = i & 7u, row = keep + (i >> 3) % (BN - keep), h = (i >> 3) / (BN - keep);
                                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + h * L::kKvHalf + row * 128u + chunk * 16u), "r"(0u) : "memory");
                            }
                            fenceProxyAsync();
                            __syncwarp();
                        }
                        ok = ok && pfWait<kCall>(&pFull[2u * x + (tt & 1u)], (tt >> 1) & 1u, err, kDevErrMmaWait);
                        if (!ok) break;
                        tcFenceAfter();
                        const uint64_t dV = descAdvance(dV0, s * L::kKvTile);
                        const uint32_t tP = tS0 + (kAhead ? 64u + 32u * (tt & 1u) : 64u * (tt & 1u));
                        if (electOne()) {
#pragma unroll
                            for (uint32_t ks = 0; ks < BN / 16; ++ks)  // 16 rows per step: 8 columns of fp16 P, 2 KB of V
                                umaMmaTS(tO, tP + ks * 8u, descAdvance(dV, ks * 2048u), idPV, (tt > t || ks > 0) ? 1u : 0u);
                            umaCommit(&pvBuf[2u * x + (tt & 1u)]);
                            if (!kAhead) umaCommit(&pvDone[x]);
                            umaCommit(&vEmpty[s]);
                        }
                        ++tt;
                    } else if (ok && electOne()) {
                        umaCommit(&vEmpty[s]);
                    }
                    __syncwarp();
                }
            }
            // A half without tiles hands in its phase of qFree, too, behind the item's last K tile and the query tiles (a
            // parity wait cannot tell a phase that it skipped from the one before).
            if (!pvRole && myTiles == 0u && ok) {
                ok = pfWait<kCall>(qFull, n & 1u, err, kDevErrFullWait);
                if (ok && electOne()) umaCommit(&qFree[x]);
                __syncwarp();
            }
            t += myTiles;
            g += it.nTiles;
        }
        if (pvRole && ok) {
            // the last two buffer commits have to land before the block leaves
            for (uint32_t tt = t >= 2u ? t - 2u : 0u; tt < t; ++tt)
                if (!pfWait<kCall>(&pvBuf[2u * x + (tt & 1u)], (tt >> 1) & 1u, err, kDevErrMmaWait)) break;
        }
        // ... and the last releases of the slots.  Over int8 pages these warps wait for them: a converter knows of its own panels only, and a
        // parity wait on a slot whose last tile is not in yet would find an older phase.  (These have waited for every tile.)
        if (I8 && ok && x == 0u) {
            if (pvRole) drain(vEmpty, g, NV, kDevErrEmptyWait);
            else drain(kEmpty, g, NK, kDevErrEmptyWait);
        }
    } else if (!(kOne && warp >= 4)) {
        // --------------------------------- softmax ---------------------------------
        const uint32_t x = warp >> 2;                         // which query tile this warpgroup owns
        const uint32_t row = (warp & 3u) * 32u + lane;        // row of that tile = TMEM lane
        const uint32_t laneBase = ((warp & 3u) * 32u) << 16;  // TMEM lane field
        const uint32_t tO = tmemBase + 128u * x;
        float2 *exch = reinterpret_cast<float2 *>(smem + L::kExch);
        uint32_t t = 0, nSplit = 0, g = 0;  // tiles of X, items of one tile, KV tiles so far
        bool ok = true;
        auto pvWait = [&](uint32_t tile) {  // the P.V product of that tile is complete
            return kAhead ? pfWait<kCall>(&pvBuf[2u * x + (tile & 1u)], (tile >> 1) & 1u, err, kDevErrMmaWait)
                          : pfWait<kCall>(&pvDone[x], tile & 1u, err, kDevErrMmaWait);
        };
        const PtItem *at;
        for (uint32_t n = 0; ok && takeItem(n, at); ++n) {
            const PtItem &it = *at;
            const uint32_t g0 = g;
            g += it.nTiles;
            const uint32_t myTiles = x == 0 ? it.nA : it.nB;
            const bool split = it.split != 0u;
            const uint32_t tileRow0 = split ? 0u : x * tileRows, t0 = it.t0;  // the tile's first row inside the item
            int32_t pos, pos0;                                                // the last cache row that the query row (the tile's first row) sees
            {
                const uint32_t first = it.m0 + tileRow0;
                pos = it.before + static_cast<int32_t>((first + row) / p.group);
                pos0 = it.before + static_cast<int32_t>(first / p.group);
            }
            float m = kNegBig, l = 0.0f;
            for (uint32_t j = 0; j < myTiles; ++j) {
                const uint32_t tt = t + j, b = tt & 1u;
                const uint32_t jj = split ? 2u * j + x : j;
                const int32_t kt = static_cast<int32_t>(t0 + jj);  // KV tile
                const float4 *sc = reinterpret_cast<const float4 *>(smem + L::kScale) + ((g0 + jj) % kPtScaleSlots) * (kPtScales / 4);
                const uint32_t tS = tmemBase + 256u + 128u * x + (kAhead ? 0u : 64u * b), tP = kAhead ? tS + 64u + 32u * b : tS;
                if (!pfWait<kCall>(&sFull[kAhead ? x : 2u * x + b], (kAhead ? tt : tt >> 1) & 1u, err, kDevErrMmaWait)) {
                    ok = false;
                    break;
                }
                tcFenceAfter();
                uint32_t r[NC][32];  // the scores of this row
#pragma unroll
                for (int c = 0; c < NC; ++c) tmemLd32(tS + laneBase + 32u * c, r[c]);
                tmemLdWait();
                if (kAhead) {
                    tcFenceBefore();
                    __syncwarp();
                    if (lane == 0) mbarArrive(&sFree[x]);
                }
                if constexpr (I8) {
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 k = sc[8 * c + i / 4];
                            const float2 a = __fmul2_rn(make_float2(__uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1])), make_float2(k.x, k.y));
                            const float2 b = __fmul2_rn(make_float2(__uint_as_float(r[c][i + 2]), __uint_as_float(r[c][i + 3])), make_float2(k.z, k.w));
                            r[c][i] = __float_as_uint(a.x), r[c][i + 1] = __float_as_uint(a.y), r[c][i + 2] = __float_as_uint(b.x), r[c][i + 3] = __float_as_uint(b.y);
                        }
                }
                if (kPtBN * kt + (kPtBN - 1) > pos0) {  // causal edge
                    const int32_t first = kPtBN * kt - pos;
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (first + c * 32 + i > 0) r[c][i] = 0xff800000u;  // -inf
                }
                float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            mxs[u] = max3(mxs[u], __uint_as_float(r[c][i + 2 * u]), __uint_as_float(r[c][i + 2 * u + 1]));
                const float mx = fmaxf(fmaxf(mxs[0], mxs[1]), fmaxf(mxs[2], mxs[3])) * p.scaleLog2 +  // scale > 0: max commutes with it
                                 (I8 ? reinterpret_cast<const float *>(sc)[128] : 0.0f);
                const float mNew = mx > m + kPtLazyLog2 ? mx : m;
                const bool rescale = j > 0 && __any_sync(0xffffffffu, mNew != m);
                float alpha = 1.0f;
                // The products of tile t - 2 are complete: its probabilities' buffer may be written, and a wait for tile t - 1 below
                // cannot take an older phase of its barrier for the one it means (a parity wait tells the current phase from the one
                // before it only).  Without kAhead the score product of this tile has waited for them.
                if (kAhead) {
                    if (tt >= 2u && !pfWait<kCall>(&pvBuf[2u * x + b], ((tt - 2u) >> 1) & 1u, err, kDevErrMmaWait)) {
                        ok = false;
                        break;
                    }
                    tcFenceAfter();
                }
                // O may only be touched between two of its P.V products.  Without kAhead the wait goes by a barrier that completes a phase per tile;
                // the last step takes it in any case, so that the wait behind the loop does not find the barrier two behind.
                if (kAhead ? rescale : j > 0 && (rescale || j + 1u == myTiles)) {
                    if (!pvWait(tt - 1u)) {
                        ok = false;
                        break;
                    }
                    tcFenceAfter();
                }
                if (rescale) {
                    alpha = fastExp2(m - mNew);
#pragma unroll 1
                    for (uint32_t c = 0; c < HD / 32; ++c) {
                        uint32_t o[32];
                        tmemLd32(tO + laneBase + c * 32u, o);
                        tmemLdWait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmemSt32(tO + laneBase + c * 32u, o);
                    }
                    tmemStWait();
                }
                m = mNew;
                const float2 scale2 = make_float2(p.scaleLog2, p.scaleLog2), negM2 = make_float2(kPtOff - m, kPtOff - m);
                float psum = 0.0f;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    uint32_t h[16];
                    float2 sum2 = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 x2 = __ffma2_rn(make_float2(__uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1])), scale2, negM2);
                        const float2 p2 = make_float2(fastExp2(x2.x), fastExp2(x2.y));
                        sum2 = __fadd2_rn(sum2, p2);
                        if constexpr (I8) {
                            const float2 v = reinterpret_cast<const float2 *>(sc + 16)[16 * c + i], x = __fmul2_rn(p2, v);
                            h[i] = packHalf2(x.x, x.y);
                        } else {
                            h[i] = packHalf2(p2.x, p2.y);
                        }
                    }
                    psum += sum2.x + sum2.y;
                    tmemSt16(tP + laneBase + c * 16u, h);
                }
                l = l * alpha + psum;
                tmemStWait();
                tcFenceBefore();
                __syncwarp();
                if (lane == 0) mbarArrive(&pFull[2u * x + b]);
            }
            ok = ok && (myTiles == 0u || pvWait(t + myTiles - 1u));
            if (!ok) break;
            // Items of one query tile: each half leaves (m, l) of its rows for the other one and stores half of the dims, out of both
            // accumulators (they lie in the same TMEM lanes).
            float M = m, lAll = l, wMine = 1.0f, wOther = 0.0f;
            if (split) {
                exch[x * kPagedTile + row] = make_float2(m, l);
                tcFenceBefore();
                mbarArrive(exFull);
                ok = pfWait<kCall>(exFull, nSplit & 1u, err, kDevErrMmaWait);
                if (!ok) break;
                tcFenceAfter();
                const float2 o = exch[(x ^ 1u) * kPagedTile + row];
                M = fmaxf(m, o.x), wMine = fastExp2(m - M), wOther = fastExp2(o.x - M);
                lAll = fmaf(wMine, l, wOther * o.y);
            } else {
                tcFenceAfter();
            }
            const bool other = split && (x == 0u ? it.nB : it.nA) != 0u, own = myTiles != 0u;  // accumulators that were written
            const bool whole = it.whole != 0u;
            const uint32_t myRows = split || x == 0u ? it.rowsA : it.rowsB;
            const float inv = whole ? (lAll == 0.0f ? 0.0f : 1.0f / lAll) : 1.0f;
            wMine *= inv, wOther *= inv;
            constexpr uint32_t kChunks = HD / 32;
            const uint32_t k0 = split ? x * (kChunks / 2) : 0u, k1 = split ? k0 + kChunks / 2 : kChunks;
            const uint32_t local = tileRow0 + row;  // row of the item
            const uint32_t mr = tileRows * L::kQTiles;
            float *part = p.parts + (2u * static_cast<size_t>(blockIdx.x) + it.part) * pagedSlot(mr, HD);
            if (!whole && row < myRows && (!split || x == 0u)) part[mr * HD + local] = M, part[mr * HD + mr + local] = lAll;
            const uint32_t rr = it.m0 + local, tok = rr / p.group;
            __half *orow = static_cast<__half *>(p.out) + (static_cast<size_t>(it.token0 + tok) * p.nHeads + it.kvHead * p.group + (rr - tok * p.group)) * HD;
#pragma unroll 1
            for (uint32_t c = k0; c < k1; ++c) {
                uint32_t o[32];
                if (own) {
                    tmemLd32(tO + laneBase + c * 32u, o);
                    tmemLdWait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * wMine);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0u;
                }
                if (other) {
                    uint32_t o2[32];
                    tmemLd32(tmemBase + 128u * (x ^ 1u) + laneBase + c * 32u, o2);
                    tmemLdWait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(fmaf(__uint_as_float(o2[i]), wOther, __uint_as_float(o[i])));
                }
                if (row < myRows && !whole) {
                    // 32 bytes per store: a thread owns its row
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        stGlobalV8(part + static_cast<size_t>(local) * HD + c * 32 + 8 * i, __uint_as_float(o[8 * i]), __uint_as_float(o[8 * i + 1]),
                                   __uint_as_float(o[8 * i + 2]), __uint_as_float(o[8 * i + 3]), __uint_as_float(o[8 * i + 4]), __uint_as_float(o[8 * i + 5]),
                                   __uint_as_float(o[8 * i + 6]), __uint_as_float(o[8 * i + 7]));
                } else if (row < myRows) {
                    uint32_t h[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) h[i] = packHalf2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
#pragma unroll
                    for (int i = 0; i < 16; i += 8) {
                        if (!p.out32) {
                            *reinterpret_cast<uint4 *>(orow + c * 32 + 2 * i) = make_uint4(h[i], h[i + 1], h[i + 2], h[i + 3]);
                            *reinterpret_cast<uint4 *>(orow + c * 32 + 2 * i + 8) = make_uint4(h[i + 4], h[i + 5], h[i + 6], h[i + 7]);
                            continue;
                        }
                        stGlobalV8(reinterpret_cast<float *>(orow + c * 32 + 2 * i), __uint_as_float(h[i]), __uint_as_float(h[i + 1]), __uint_as_float(h[i + 2]),
                                   __uint_as_float(h[i + 3]), __uint_as_float(h[i + 4]), __uint_as_float(h[i + 5]), __uint_as_float(h[i + 6]), __uint_as_float(h[i + 7]));
                    }
                }
            }
            if (split) {
                // the next item's first P.V product may overwrite an accumulator once both halves have read it
                tcFenceBefore();
                mbarArrive(exRead);
                ok = pfWait<kCall>(exRead, nSplit & 1u, err, kDevErrMmaWait);
                ++nSplit;
            } else {
                tcFenceBefore();
            }
            t += myTiles;
        }
    }
    __syncthreads();
    if (warp == 0) tmemDealloc(tmemBase, 512);
}

template <int HD, bool I8>
static int launchTiles(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const PagedAttnParams &p, cudaStream_t st, uint32_t *blocks) {
    using L = PtL<HD, I8>;
    static bool attrDone[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attrDone[dev]) {
        TC_CUDA_OK(cudaFuncSetAttribute((pagedTilesKernel<HD, I8>), cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal));
        attrDone[dev] = true;
    }
    *blocks = std::min(numSMs(), kPagedSMs);
    return launchDependent(pagedTilesKernel<HD, I8>, dim3(*blocks), L::kThreads, L::kTotal, st, 1, q, k, v, p);
}

int pagedAttnTiles(const tc_paged_kv *c, const PagedAttnParams &p, cudaStream_t st, uint32_t *blocks) {
    CUtensorMap q, k, v;
    int rc = pagedMaps(c, p.box, &k, &v);
    if (rc != TC_OK) return rc;
    TensorMapKey key;
    memset(&key, 0, sizeof(key));
    key.base = p.q;
    key.dims[0] = c->hd, key.dims[1] = p.nHeads, key.dims[2] = c->tokens;
    key.strides[0] = static_cast<uint64_t>(c->hd) * 2;
    key.strides[1] = key.strides[0] * p.nHeads;
    key.box[0] = 64, key.box[1] = p.group, key.box[2] = p.tileTokens;
    key.rank = 3, key.elemBytes = 2, key.swizzle = 3;
    rc = getTensorMap(key, &q);
    if (rc != TC_OK) return rc;
    if (c->kvI8) return c->hd == 128 ? launchTiles<128, true>(q, k, v, p, st, blocks) : launchTiles<256, true>(q, k, v, p, st, blocks);
    if (c->hd == 64) return launchTiles<64, false>(q, k, v, p, st, blocks);
    return c->hd == 128 ? launchTiles<128, false>(q, k, v, p, st, blocks) : launchTiles<256, false>(q, k, v, p, st, blocks);
}

}  // namespace tc
