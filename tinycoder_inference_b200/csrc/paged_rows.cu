// paged_rows.cu -- f32 attention of more than 16 query rows per kv head over fp16 pages of head_dim 64 and 128 (chunks and prompts whose
// caller wants f32 results).
//
// The work, the ring and the partials are paged_attn.cuh's.  Here the query rows are on the M side of mma.sync m16n8k16: the
// instruction's 16 rows are 8 query rows twice, the upper half with the leading 11 bits of q (then of p), the lower one with what is left of
// it, and the two halves of a sum lie in the same thread.  That holds 21 bits and more of q and p and the exact values of K and V; a sum
// in the tensor unit, whose additions cut off, has at most hd / 16 products before it joins f32 registers.  Four warps
// take 8 query rows of an item each and all 64 rows of a tile: with several items per kv head the cache comes from L2, and what bounds
// the kernel is the tensor pipe at two products per term and the additions between them: 512 rows behind 3584 of 28 / 4 / 128 take
// 212 us, 133 TFLOP/s of terms (mma.sync alone 275).  With the rows on the N side (paged_steps.cu) the same call takes 250, with 17 - 64 rows 5 - 20 %
// more; at head_dim 256 and over int8 pages, whose rows this kernel would convert once per warp, that form is the faster one (3 - 8
// tokens of 16 / 2 / 256 over int8 pages: 74 - 132 us here, 60 - 100 there).
#include <algorithm>

#include "paged_attn.cuh"

namespace tc {

// p is held as 2^13 p: its fp16 pair keeps 11 + 11 bits down to p = 2^-15, the upper half's 11 down to 2^-27, and is off by 2^-38 at most
constexpr float kPrOff = 13.0f;

template <int HD>
struct PrL {
    static constexpr bool kI8 = false;
    static constexpr int NW = 4, kThreads = 160, kBlocks = 2, MR = 8 * NW;
    static constexpr int kPanels = HD / 64;                 // 128-byte columns of a row
    static constexpr int kPanel = int(kPaTile) * 128;
    static constexpr int kMat = kPanels * kPanel;
    static constexpr int kStage = 2 * kMat;
    static constexpr int NST = HD == 64 ? 5 : 3;
    static constexpr int kScales = NST * kStage;            // (none)
    static constexpr int kBuf = kScales;                    // [warp][8][36] f32
    static constexpr int kItems = kBuf + NW * 8 * 36 * 4;
    static constexpr int kBars = (kItems + int(kPaItems * sizeof(PaItem)) + 7) / 8 * 8;
    static constexpr int kTotal = kBars + (2 * NST + int(kPaItems)) * 8 + 1024;
    static_assert(NST + 2 <= int(kPaItems), "items");
    static_assert(kBlocks * (kTotal + 1024) <= 228 * 1024, "shared memory of an SM");
    static_assert(size_t(2) * kPagedSMs * kBlocks * pagedSlot(MR, HD) <= kTilesParts && kBlocks <= 2, "the workspace's room");
};

template <int HD>
__global__ void __launch_bounds__(PrL<HD>::kThreads, PrL<HD>::kBlocks)
pagedRowsKernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedAttnParams p) {
    using L = PrL<HD>;
    constexpr uint32_t NST = L::NST, MR = L::MR;
    extern __shared__ uint8_t smemRaw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::kBars), *empty = full + NST, *itemFull = empty + NST;
    PaItem *items = reinterpret_cast<PaItem *>(smem + L::kItems);
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < NST; ++i) {
            mbarInit(&full[i], 1);
            mbarInit(&empty[i], L::NW);
        }
        for (uint32_t i = 0; i < kPaItems; ++i) mbarInit(&itemFull[i], 1);
        fenceBarrierInit();
        tmaPrefetchDesc(&tmK);
        tmaPrefetchDesc(&tmV);
    }
    __syncthreads();
    if (warp == L::NW) {
        pagedProduce<L>(p, tmK, tmV, smem, full, empty, itemFull, items);
        return;
    }
    gridDepWait();
    gridDepLaunch();

    const uint32_t c = lane & 3u, n8 = lane >> 2;
    constexpr int NT = int(kPaTile) / 8, KK = int(kPaTile) / 16, NJ = HD / 8, NS = HD / 16;  // score tiles, their pairs, output tiles, steps of q . K
    float *buf = reinterpret_cast<float *>(smem + L::kBuf) + warp * (8u * 36u);
    uint32_t g = 0;  // tiles so far
    bool ok = true;
    for (uint32_t n = 0;; ++n) {
        // The producer hands in the end of the run whatever becomes of its waits, each of which is bounded: this one only has to be longer.
        for (uint32_t i = 0; i < (1u << 20) && !mbarTryWait(&itemFull[n % kPaItems], (n / kPaItems) & 1u); ++i) {}
        const PaItem it = items[n % kPaItems];
        if (it.nTiles == 0u) break;
        // q as A operands: row n8 (upper half) and what is left of it (lower half), in the order of dims that a thread's 16-byte loads of K have
        const uint32_t rr = it.m0 + 8u * warp + n8;
        const bool valid = rr < it.rows;
        const int32_t vis = valid ? it.before + static_cast<int32_t>(rr / p.group) + 1 : 0x7fffffff;  // cache rows that the query row sees
        uint32_t qa[NS][4];
        const float rowScale = p.scaleLog2 * pagedQuery<NS>(p, it, rr, valid, HD, [&](int st) { return 64 * (st / 4) + 16 * static_cast<int>(c) + 4 * (st % 4); },
                                                            [&](int st, const uint32_t(&w)[4]) { qa[st][0] = w[0], qa[st][1] = w[2], qa[st][2] = w[1], qa[st][3] = w[3]; });
        const int32_t leastVis = __reduce_min_sync(0xffffffffu, vis);
        float m = -INFINITY, l = 0.0f, o[NJ][2];
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[j][0] = o[j][1] = 0.0f;

        const uint32_t t0 = it.t0, t1 = t0 + it.nTiles;
        for (uint32_t t = t0; t < t1; ++t, ++g) {
            const uint32_t st = g % NST;
            ok = ok && pfWait<true>(&full[st], (g / NST) & 1u, p.c.err, kDevErrFullWait);
            if (!ok) break;
            const uint32_t sK = smemAddr(smem + st * L::kStage), sV = sK + L::kMat;
            const int32_t tile0 = static_cast<int32_t>(t * kPaTile), left = static_cast<int32_t>(it.len) - tile0;  // rows of the tile that exist
            float s[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float d[4] = {0.f, 0.f, 0.f, 0.f};
                const uint32_t key = 8u * nt + n8;
#pragma unroll
                for (int h = 0; h < L::kPanels; ++h) {
                    const uint32_t row = sK + h * L::kPanel + key * 128u;
                    const uint4 a = ldShared4(row + (((2u * c) ^ n8) << 4)), b = ldShared4(row + (((2u * c + 1u) ^ n8) << 4));
                    const uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t(&A)[4] = qa[4 * h + i];
                        mmaF16(d, A[0], A[1], A[2], A[3], v[2 * i], v[2 * i + 1]);
                    }
                }
                s[nt][0] = (d[0] + d[2]) * rowScale, s[nt][1] = (d[1] + d[3]) * rowScale;
            }
            if (tile0 + static_cast<int32_t>(kPaTile) > leastVis) {  // (whatever a masked place holds, a select takes it out)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (tile0 + static_cast<int32_t>(8u * nt + 2u * c) + e >= vis) s[nt][e] = -INFINITY;
            }
            float mx = m;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mx = fmaxf(mx, fmaxf(s[nt][0], s[nt][1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float mu = mx == -INFINITY ? 0.0f : mx, alpha = fastExp2(m - mu);
            m = mx;
            float sum = 0.0f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[nt][e] = fastExp2(s[nt][e] - mu + kPrOff);
                    sum += s[nt][e];
                }
            l = fmaf(l, alpha, sum);
            if (left < static_cast<int32_t>(kPaTile)) {
                // rows past the sequence: what stands there is no number that 0 could be multiplied with.  (Every warp clears them for itself.)
                for (int32_t i = static_cast<int32_t>(lane); i < int(kPaTile) * 8 * L::kPanels; i += 32) {
                    const int32_t key = i % int(kPaTile), chunk = i / int(kPaTile);
                    if (key >= left)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sV + (chunk / 8) * L::kPanel + key * 128 + (chunk % 8) * 16), "r"(0u) : "memory");
                }
                fenceProxyAsync();  // (TMA writes this room next)
                __syncwarp();
            }
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                float h[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) splitHalf(s[2 * kk + i / 2][i % 2], h[i], lo[i]);
                const uint32_t pa[4] = {packHalf2(h[0], h[1]), packHalf2(lo[0], lo[1]), packHalf2(h[2], h[3]), packHalf2(lo[2], lo[3])};
                const float a = kk == 0 ? alpha : 1.0f;
                const uint32_t key = 16u * kk + ((lane >> 3) & 1u) * 8u + (lane & 7u);
                auto product = [&](int j, uint32_t b0, uint32_t b1) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
                    mmaF16(d, pa[0], pa[1], pa[2], pa[3], b0, b1);
                    o[j][0] = fmaf(o[j][0], a, d[0] + d[2]), o[j][1] = fmaf(o[j][1], a, d[1] + d[3]);
                };
#pragma unroll
                for (int j = 0; j < NJ; j += 2) {
                    const uint32_t chunk = j + (lane >> 4);
                    uint32_t r0, r1, r2, r3;
                    ldmatrixX4Trans(r0, r1, r2, r3, sV + (chunk >> 3) * L::kPanel + key * 128u + (((chunk & 7u) ^ (key & 7u)) << 4));
                    product(j, r0, r1);
                    product(j + 1, r2, r3);
                }
            }
            uint32_t used = 0u;
#pragma unroll
            for (int j = 0; j < NJ; ++j) used ^= __float_as_uint(o[j][0]);
            releaseStage(&empty[st], used, p.zero);
        }
        // ---- the rows out, or into the item's partial ----
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const bool whole = it.whole != 0u;
        float *part = p.parts + (2u * static_cast<size_t>(blockIdx.x) + it.part) * pagedSlot(MR, HD);
        const float f = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
        if (!whole && c == 0) part[MR * HD + 8u * warp + n8] = m, part[MR * HD + MR + 8u * warp + n8] = l;
#pragma unroll
        for (int pass = 0; pass < NJ / 4; ++pass) {  // 32 dims at a time, so that a row leaves in whole lines
            __syncwarp();
#pragma unroll
            for (int jj = 0; jj < 4; ++jj)
#pragma unroll
                for (int e = 0; e < 2; ++e) buf[n8 * 36u + jj * 8u + 2u * c + e] = o[4 * pass + jj][e] * f;
            __syncwarp();
            for (uint32_t i = lane; i < 64u; i += 32u) {
                const uint32_t row = i >> 3, dim = 32u * pass + 4u * (i & 7u), local = 8u * warp + row, r = it.m0 + local;
                const float4 x = *reinterpret_cast<const float4 *>(buf + row * 36u + 4u * (i & 7u));
                if (r >= it.rows) continue;
                if (whole) pagedStore(p, HD, it.token0, it.kvHead, r, dim, x);
                else __stcg(reinterpret_cast<float4 *>(part + local * HD + dim), x);
            }
        }
        __syncwarp();
    }
}

template <int HD>
static int launchRows(const CUtensorMap &k, const CUtensorMap &v, const PagedAttnParams &p, cudaStream_t st, uint32_t *blocks) {
    using L = PrL<HD>;
    static bool attrDone[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attrDone[dev]) {
        TC_CUDA_OK(cudaFuncSetAttribute(pagedRowsKernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal));
        attrDone[dev] = true;
    }
    *blocks = std::min(numSMs(), kPagedSMs) * L::kBlocks;
    return launchDependent(pagedRowsKernel<HD>, dim3(*blocks), L::kThreads, L::kTotal, st, 1, k, v, p);
}

int pagedAttnRows(const tc_paged_kv *c, const PagedAttnParams &p, cudaStream_t st, uint32_t *blocks) {
    CUtensorMap k, v;
    const int rc = pagedMaps(c, p.box, &k, &v);
    if (rc != TC_OK) return rc;
    return c->hd == 64 ? launchRows<64>(k, v, p, st, blocks) : launchRows<128>(k, v, p, st, blocks);
}

}  // namespace tc
