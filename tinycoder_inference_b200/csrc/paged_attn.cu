// paged_attn.cu -- attention of few query rows per kv head over a paged cache: decode steps, drafts, short chunks, and every call
// that wants f32 results.
//
//   o[t, h] = sum_j p_j V[j] / sum_j p_j,   p_j = exp(q[t, h] . K[j] / sqrt(hd) - m),   j <= pos(t),
//
// in one pass over the rows with a running maximum and sum.  What bounds it is the cache: each of its bytes is read once per item
// (paged_attn.cuh), and mma.sync m16n8k16 is fed from registers fast enough for that.  A block has a producer warp, which looks up
// pages and requests tiles of 64 rows of K and V by TMA into a ring (128-byte swizzle; the scales of an int8 store by cp.async), and
// four consumer warps: WM groups of query rows, each split over 4 / WM shares of a tile's rows.  Every warp keeps its own
// maxima, sums and accumulators over the run; the shares meet at the end of an item.
//
// PAIR: an instruction's 16 rows are 8 query rows twice, the upper half with the leading 11 bits of q (then of p), the lower one with
// what is left of it; the two halves of a sum lie in the same thread.  That holds 21 bits and more of q and p, exact values of K
// and V (fp16, or int8 as fp16 integers whose scale comes after the product), and sums of at most hd / 16 + 4 products in the tensor
// unit, whose additions cut off, before they join f32 registers.  It is what f32 results take, and calls of at most 8 rows, whose
// lower half would be idle.
//
// int8 -> fp16: byte ^ 0x80 in the low bits of 0x6400 is 1024 + 128 + x, minus 1152 is x, exactly.  The dims of q . K and of the output are
// taken in the order in which a thread's 16-byte loads of the swizzled tile deliver them (free of bank conflicts), not in the matrix order.
#include <algorithm>
#include <cstring>

#include "paged_attn.cuh"

namespace tc {

constexpr float kPaOff = 13.0f;  // p is held as 2^13 p: its fp16 pair keeps 11 + 11 bits down to p = 2^-27

template <int HD, bool I8, bool PAIR, int WM>
struct PaL {
    static constexpr bool kI8 = I8;
    static constexpr int NW = HD == 256 && WM > 1 ? 8 : 4;          // consumer warps; a producer beside them
    // 8 consumer warps: a warpgroup for the producer, whose registers go to theirs (232 x 256 + 40 x 128 = 168 x 384, what the block is
    // launched with)
    static constexpr bool kSplitRegs = NW == 8;
    static constexpr int kThreads = kSplitRegs ? 384 : 32 * (NW + 1);
    static constexpr int WK = NW / WM, KS = int(kPaTile) / WK;      // shares of a tile; rows of a share
    static constexpr int RW = PAIR ? 8 : 16;                       // query rows of a warp
    static constexpr int MR = WM * RW;
    static constexpr int kPanels = HD * (I8 ? 1 : 2) / 128;        // 128-byte columns of a row
    static constexpr int kPanel = int(kPaTile) * 128;
    static constexpr int kMat = kPanels * kPanel;
    static constexpr int kStage = 2 * kMat;
    // as many stages as leave room for two blocks per SM (head_dim 256: one)
    static constexpr int NST = HD == 256 ? (I8 ? 6 : 3) : (kStage == 16384 ? 5 : 3);
    static constexpr int kScales = NST * kStage;                   // [stage][K, V][64]
    static constexpr int kBuf = kScales + (I8 ? NST * 512 : 0);    // [warp][16][36] f32
    static constexpr int kMl = kBuf + NW * 16 * 36 * 4;            // [warp][16] (m, l)
    static constexpr int kItems = kMl + NW * 16 * 8;
    static constexpr int kBars = kItems + int(kPaItems * sizeof(PaItem));
    static constexpr int kTotal = kBars + (2 * NST + int(kPaItems)) * 8 + 1024;
    static_assert(NST + 2 <= int(kPaItems), "items");
    static constexpr int kBlocks = HD == 256 ? 1 : 2;
    static_assert(kBlocks * (kTotal + 1024) <= 228 * 1024, "shared memory of an SM");
};

// The partials of the items that several blocks had a part in: block (i, y) takes item i's rows y, y + gridDim.y, ... (in steps of 8 / W).
// W warps share a row, each a W-th of its partials: few rows of many parts (a step of one long session: 74) are as much a chain of loads
// as many rows of two.
template <int HD>
__global__ void __launch_bounds__(256) pagedMergeKernel(const __grid_constant__ PagedAttnParams p, const float *partsB, const PagedJoin *joinsB, uint32_t blocksA) {
    constexpr int V = HD / 128 ? HD / 128 : 1;  // float4 of a lane
    __shared__ float4 sAcc[8][V * 32];
    __shared__ float2 sMl[8];
    gridDepWait();
    gridDepLaunch();
    const bool second = blockIdx.x >= blocksA;  // (the tiles kernel's)
    const uint32_t from = second ? blockIdx.x - blocksA : blockIdx.x;
    const PagedJoin j = (second ? joinsB : p.joins)[from];
    if (j.count == 0u) return;
    const float *parts = second ? partsB : p.parts;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const size_t slot = pagedSlot(j.mr, HD);
    auto part = [&](uint32_t c) { return parts + (2u * static_cast<size_t>(from + c) + (c == 0u ? 1u : 0u)) * slot; };
    const uint32_t W = j.count <= 8u ? 1u : j.count <= 16u ? 2u : j.count <= 32u ? 4u : 8u, perPass = 8u / W, mine = warp % W;
    const uint32_t rows = min(j.mr, j.rows - j.row0);
    for (uint32_t i0 = blockIdx.y * perPass; i0 < rows; i0 += gridDim.y * perPass) {
        const uint32_t i = i0 + warp / W;
        float M = -INFINITY, L = 0.0f;
        float4 acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < rows) {
            // 32 W partials at a time; the first accumulators are under way before the maxima that weigh them
            constexpr uint32_t A = HD == 256 ? 4 : 8;
            for (uint32_t cb = mine; cb < j.count; cb += 32u * W) {
                const uint32_t n = min(32u, (j.count - cb + W - 1u) / W);
                auto load = [&](uint32_t c, float4(&x)[V]) {
                    const float4 *a = reinterpret_cast<const float4 *>(part(cb + W * c) + static_cast<size_t>(i) * HD);
#pragma unroll
                    for (int v = 0; v < V; ++v) x[v] = HD >= 128 || lane < HD / 4u ? a[v * 32 + lane] : make_float4(0.f, 0.f, 0.f, 0.f);
                };
                float4 x[A][V];
#pragma unroll
                for (uint32_t u = 0; u < A; ++u)
                    if (u < n) load(u, x[u]);
                float m = -INFINITY, l = 0.0f;
                if (lane < n) m = part(cb + W * lane)[j.mr * HD + i], l = part(cb + W * lane)[j.mr * HD + j.mr + i];
                float top = fmaxf(m, M);
#pragma unroll
                for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const float Mu = top == -INFINITY ? 0.0f : top, keep = fastExp2(M - Mu), wc = fastExp2(m - Mu);  // (-inf: 0)
                M = top;
                L = fmaf(L, keep, wc * l);
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v].x *= keep, acc[v].y *= keep, acc[v].z *= keep, acc[v].w *= keep;
                for (uint32_t c0 = 0; c0 < n; c0 += A) {
#pragma unroll
                    for (uint32_t u = 0; u < A; ++u) {
                        if (c0 + u >= n) break;
                        if (c0 > 0u) load(c0 + u, x[u]);
                    }
#pragma unroll
                    for (uint32_t u = 0; u < A; ++u) {
                        if (c0 + u >= n) break;
                        const float f = __shfl_sync(0xffffffffu, wc, c0 + u);
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            acc[v].x = fmaf(f, x[u][v].x, acc[v].x), acc[v].y = fmaf(f, x[u][v].y, acc[v].y);
                            acc[v].z = fmaf(f, x[u][v].z, acc[v].z), acc[v].w = fmaf(f, x[u][v].w, acc[v].w);
                        }
                    }
                }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        }
        if (W > 1u) {  // (the same for the whole block)
            if (lane == 0) sMl[warp] = make_float2(M, L);
#pragma unroll
            for (int v = 0; v < V; ++v) sAcc[warp][v * 32 + lane] = acc[v];
            __syncthreads();
            if (mine == 0u) {
                const float own = M;
                for (uint32_t w = 1; w < W; ++w) M = fmaxf(M, sMl[warp + w].x);
                const float Mu = M == -INFINITY ? 0.0f : M;
                const float f0 = fastExp2(own - Mu);
                L *= f0;
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v].x *= f0, acc[v].y *= f0, acc[v].z *= f0, acc[v].w *= f0;
                for (uint32_t w = 1; w < W; ++w) {
                    const float f = fastExp2(sMl[warp + w].x - Mu);
                    L = fmaf(f, sMl[warp + w].y, L);
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const float4 x = sAcc[warp + w][v * 32 + lane];
                        acc[v].x = fmaf(f, x.x, acc[v].x), acc[v].y = fmaf(f, x.y, acc[v].y);
                        acc[v].z = fmaf(f, x.z, acc[v].z), acc[v].w = fmaf(f, x.w, acc[v].w);
                    }
                }
            }
            __syncthreads();
        }
        if (mine != 0u || i >= rows) continue;
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // (nothing seen)
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (HD >= 128 || lane < HD / 4u)
                pagedStore(p, HD, j.token0, j.kvHead, j.row0 + i, (v * 32u + lane) * 4u, make_float4(acc[v].x * inv, acc[v].y * inv, acc[v].z * inv, acc[v].w * inv));
    }
}

template <int HD, bool I8, bool PAIR, int WM>
__global__ void __launch_bounds__((PaL<HD, I8, PAIR, WM>::kThreads), (PaL<HD, I8, PAIR, WM>::kBlocks))
pagedRowsKernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedAttnParams p) {
    using L = PaL<HD, I8, PAIR, WM>;
    constexpr uint32_t NST = L::NST, MR = L::MR, WK = L::WK;
    extern __shared__ uint8_t smemRaw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::kBars), *empty = full + NST, *itemFull = empty + NST;
    PaItem *items = reinterpret_cast<PaItem *>(smem + L::kItems);
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < NST; ++i) {
            mbarInit(&full[i], I8 ? 33 : 1);  // (int8: every lane of the producer brings scales)
            mbarInit(&empty[i], L::NW);
        }
        for (uint32_t i = 0; i < kPaItems; ++i) mbarInit(&itemFull[i], 1);
        fenceBarrierInit();
        tmaPrefetchDesc(&tmK);
        tmaPrefetchDesc(&tmV);
    }
    __syncthreads();
    uint32_t g = 0;  // tiles so far
    if constexpr (L::kSplitRegs) {
        if (warp >= L::NW) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        if (warp > L::NW) return;
    }

    if (warp == L::NW) {
        pagedProduce<L>(p, tmK, tmV, smem, full, empty, itemFull, items);
        return;
    }

    gridDepWait();
    gridDepLaunch();
    // --------------------------------- consumers ---------------------------------
    const uint32_t wm = warp / WK, wk = warp % WK, c = lane & 3u, n8 = lane >> 2;
    constexpr int NR = PAIR ? 1 : 2;      // query rows of a thread: n8 (and n8 + 8)
    constexpr int NT = L::KS / 8;         // 8-row score tiles of a share
    constexpr int KK = L::KS / 16;
    constexpr int NJ = HD / 8;            // 8-dim output tiles
    constexpr int OR = PAIR ? 2 : 4;
    constexpr int NS = HD / 16;           // 16-dim steps of q . K
    const uint32_t key0 = wk * L::KS;
    float *buf = reinterpret_cast<float *>(smem + L::kBuf);
    float2 *ml = reinterpret_cast<float2 *>(smem + L::kMl);
    auto groupSync = [&] {
        if (WK == 1) __syncwarp();
        else namedBarSync(1u + wm, WK * 32u);
    };
    bool ok = true;  // (a warp that gave up still takes its items and meets the others at their barriers)
    for (uint32_t n = 0;; ++n) {
        // The producer hands in the end of the run whatever becomes of its waits, each of which is bounded: this one only has to be longer.
        for (uint32_t i = 0; i < (1u << 20) && !mbarTryWait(&itemFull[n % kPaItems], (n / kPaItems) & 1u); ++i) {}
        const PaItem it = items[n % kPaItems];
        if (it.nTiles == 0u) break;
        // q as A operands
        uint32_t qa[NS][4];
        float rowScale[NR];
        int32_t vis[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const uint32_t rr = it.m0 + wm * L::RW + n8 + 8u * r;
            const bool valid = rr < it.rows;
            const uint32_t tok = it.token0 + rr / p.group, head = it.kvHead * p.group + rr % p.group;
            vis[r] = valid ? it.before + static_cast<int32_t>(rr / p.group) + 1 : 0;
            rowScale[r] = p.scaleLog2;
            const size_t base = (static_cast<size_t>(tok) * p.nHeads + head) * HD;
            auto dim = [&](int st) { return I8 ? 128 * (st / 8) + 32 * static_cast<int>(c) + 4 * (st % 8) : 64 * (st / 4) + 16 * static_cast<int>(c) + 4 * (st % 4); };
            if (p.half) {
#pragma unroll
                for (int st = 0; st < NS; ++st) {
                    uint2 x = make_uint2(0u, 0u);
                    if (valid) x = __ldg(reinterpret_cast<const uint2 *>(static_cast<const __half *>(p.q) + base + dim(st)));
                    qa[st][r] = x.x, qa[st][2 + r] = x.y;
                    if (PAIR) qa[st][1] = qa[st][3] = 0u;
                }
            } else if constexpr (PAIR) {
                float4 x[NS];
                float top = 0.0f;
#pragma unroll
                for (int st = 0; st < NS; ++st) {
                    x[st] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (valid) x[st] = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(p.q) + base + dim(st)));
                    top = fmaxf(top, fmaxf(fmaxf(fabsf(x[st].x), fabsf(x[st].y)), fmaxf(fabsf(x[st].z), fabsf(x[st].w))));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // the row's largest goes to [2^10, 2^11), so that what the upper half leaves is a normal fp16 number
                float up = 1.0f;
                if (top > 0.0f && top < INFINITY) {
                    const int e = min(126, max(-116, static_cast<int>(__float_as_uint(top) >> 23) - 127));
                    up = __uint_as_float(static_cast<uint32_t>(127 + 10 - e) << 23);
                    rowScale[r] = p.scaleLog2 * __uint_as_float(static_cast<uint32_t>(127 - 10 + e) << 23);
                }
#pragma unroll
                for (int st = 0; st < NS; ++st) {
                    float h[4], l[4];
                    splitHalf(x[st].x * up, h[0], l[0]);
                    splitHalf(x[st].y * up, h[1], l[1]);
                    splitHalf(x[st].z * up, h[2], l[2]);
                    splitHalf(x[st].w * up, h[3], l[3]);
                    qa[st][0] = packHalf2(h[0], h[1]), qa[st][1] = packHalf2(l[0], l[1]);
                    qa[st][2] = packHalf2(h[2], h[3]), qa[st][3] = packHalf2(l[2], l[3]);
                }
            }
        }
        int32_t leastVis = vis[0];
        if (NR == 2) leastVis = min(leastVis, vis[NR - 1]);
        leastVis = __reduce_min_sync(0xffffffffu, leastVis);
        float m[NR], l[NR], o[NJ][OR];
        int vexp = -126;  // int8: the accumulators hold V 2^-vexp
#pragma unroll
        for (int r = 0; r < NR; ++r) m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < OR; ++e) o[j][e] = 0.0f;

        const uint32_t t0 = it.t0, t1 = t0 + it.nTiles;
        for (uint32_t t = t0; t < t1; ++t, ++g) {
            const uint32_t st = g % NST;
            ok = ok && pfWait<true>(&full[st], (g / NST) & 1u, p.c.err, kDevErrFullWait);
            if (!ok) break;
            const uint32_t sK = smemAddr(smem + st * L::kStage), sV = sK + L::kMat;
            const float *sc = reinterpret_cast<const float *>(smem + L::kScales) + st * 128u;
            const int32_t left = static_cast<int32_t>(it.len) - static_cast<int32_t>(t * kPaTile);  // rows of the tile that exist
            float s[NT][2 * NR];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float d[4] = {0.f, 0.f, 0.f, 0.f};
                const uint32_t key = key0 + 8u * nt + n8, x = key & 7u;
#pragma unroll
                for (int h = 0; h < L::kPanels; ++h) {
                    const uint32_t row = sK + h * L::kPanel + key * 128u;
                    const uint4 a = ldShared4(row + (((2u * c) ^ x) << 4)), b = ldShared4(row + (((2u * c + 1u) ^ x) << 4));
                    const uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                    if constexpr (I8) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint32_t u = v[i] ^ 0x80808080u;
                            const uint32_t(&A)[4] = qa[8 * h + i];
                            mmaF16(d, A[0], A[1], A[2], A[3], bytesLo(u), bytesHi(u));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t(&A)[4] = qa[4 * h + i];
                            mmaF16(d, A[0], A[1], A[2], A[3], v[2 * i], v[2 * i + 1]);
                        }
                    }
                }
                float k0 = 1.0f, k1 = 1.0f;
                if constexpr (I8) {
                    const float2 k = *reinterpret_cast<const float2 *>(sc + key0 + 8u * nt + 2u * c);
                    k0 = k.x, k1 = k.y;
                }
                if constexpr (PAIR) {
                    s[nt][0] = (d[0] + d[2]) * (k0 * rowScale[0]), s[nt][1] = (d[1] + d[3]) * (k1 * rowScale[0]);
                } else {
                    s[nt][0] = d[0] * (k0 * rowScale[0]), s[nt][1] = d[1] * (k1 * rowScale[0]);
                    s[nt][2] = d[2] * (k0 * rowScale[NR - 1]), s[nt][3] = d[3] * (k1 * rowScale[NR - 1]);
                }
            }
            const int32_t tile0 = static_cast<int32_t>(t * kPaTile);
            if (tile0 + static_cast<int32_t>(kPaTile) > leastVis) {  // (whatever a masked place holds, a select takes it out)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2 * NR; ++e)
                        if (tile0 + static_cast<int32_t>(key0 + 8u * nt + 2u * c) + (e & 1) >= vis[e >> 1]) s[nt][e] = -INFINITY;
            }
            float alpha[NR], mu[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float mx = -INFINITY;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mx = fmaxf(mx, fmaxf(s[nt][2 * r], s[nt][2 * r + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                mx = fmaxf(mx, m[r]);
                mu[r] = mx == -INFINITY ? 0.0f : mx;
                alpha[r] = fastExp2(m[r] - mu[r]);
                m[r] = mx;
                float sum = 0.0f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 2 * r; e < 2 * r + 2; ++e) {
                        s[nt][e] = fastExp2(s[nt][e] - mu[r] + kPaOff);
                        sum += s[nt][e];
                    }
                l[r] = fmaf(l[r], alpha[r], sum);
            }
            if constexpr (I8) {
                // p times the scale of V's row, relative to a power of two no smaller than any scale so far
                float2 v[NT];
                uint32_t top = 0u;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int32_t key = static_cast<int32_t>(key0 + 8u * nt + 2u * c);
                    v[nt] = *reinterpret_cast<const float2 *>(sc + 64u + key);
                    if (key >= left) v[nt].x = 0.0f;
                    if (key + 1 >= left) v[nt].y = 0.0f;
                    top = max(top, max(__float_as_uint(v[nt].x) & 0x7fffffffu, __float_as_uint(v[nt].y) & 0x7fffffffu));
                }
                top = __reduce_max_sync(0xffffffffu, top);
                const int e = max(vexp, min(126, static_cast<int>(top >> 23) - 126));
                const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                if (e != vexp) {
                    const float f = fastExp2(static_cast<float>(vexp - e));
#pragma unroll
                    for (int r = 0; r < NR; ++r) alpha[r] *= f;
                    vexp = e;
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < NR; ++r) s[nt][2 * r] *= v[nt].x * down, s[nt][2 * r + 1] *= v[nt].y * down;
            } else if (left < static_cast<int32_t>(kPaTile)) {
                // rows past the sequence: what stands there is no number that 0 could be multiplied with
                for (int32_t i = static_cast<int32_t>(lane); i < L::KS * 8 * L::kPanels; i += 32) {
                    const int32_t key = static_cast<int32_t>(key0) + i % L::KS, chunk = i / L::KS;
                    if (key >= left)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sV + (chunk / 8) * L::kPanel + key * 128 + (chunk % 8) * 16), "r"(0u) : "memory");
                }
                fenceProxyAsync();  // (TMA writes this room next)
                __syncwarp();
            }
            if constexpr (!PAIR) {
                const bool scale = alpha[0] != 1.0f || alpha[NR - 1] != 1.0f;
                if (__any_sync(0xffffffffu, scale)) {
#pragma unroll
                    for (int j = 0; j < NJ; ++j) o[j][0] *= alpha[0], o[j][1] *= alpha[0], o[j][OR - 2] *= alpha[NR - 1], o[j][OR - 1] *= alpha[NR - 1];
                }
            }
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                uint32_t pa[4];
                if constexpr (PAIR) {
                    float h[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) splitHalf(s[2 * kk + i / 2][i % 2], h[i], lo[i]);
                    pa[0] = packHalf2(h[0], h[1]), pa[1] = packHalf2(lo[0], lo[1]);
                    pa[2] = packHalf2(h[2], h[3]), pa[3] = packHalf2(lo[2], lo[3]);
                } else {
                    pa[0] = packHalf2(s[2 * kk][0], s[2 * kk][1]), pa[1] = packHalf2(s[2 * kk][2 * NR - 2], s[2 * kk][2 * NR - 1]);
                    pa[2] = packHalf2(s[2 * kk + 1][0], s[2 * kk + 1][1]), pa[3] = packHalf2(s[2 * kk + 1][2 * NR - 2], s[2 * kk + 1][2 * NR - 1]);
                }
                auto product = [&](int j, uint32_t b0, uint32_t b1) {
                    if constexpr (PAIR) {
                        float d[4] = {0.f, 0.f, 0.f, 0.f};
                        mmaF16(d, pa[0], pa[1], pa[2], pa[3], b0, b1);
                        const float a = kk == 0 ? alpha[0] : 1.0f;
                        o[j][0] = fmaf(o[j][0], a, d[0] + d[2]), o[j][1] = fmaf(o[j][1], a, d[1] + d[3]);
                    } else {
                        mmaF16(reinterpret_cast<float(&)[4]>(o[j]), pa[0], pa[1], pa[2], pa[3], b0, b1);
                    }
                };
                if constexpr (I8) {
                    const uint32_t k = key0 + 16u * kk + 2u * c;
#pragma unroll
                    for (int h = 0; h < L::kPanels; ++h) {
                        auto load = [&](uint32_t key) { return ldShared4(sV + h * L::kPanel + key * 128u + ((n8 ^ (key & 7u)) << 4)); };
                        const uint4 a0 = load(k), a1 = load(k + 1u), b0 = load(k + 8u), b1 = load(k + 9u);
                        const uint32_t A0[4] = {a0.x, a0.y, a0.z, a0.w}, A1[4] = {a1.x, a1.y, a1.z, a1.w};
                        const uint32_t B0[4] = {b0.x, b0.y, b0.z, b0.w}, B1[4] = {b1.x, b1.y, b1.z, b1.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            // dims 4 i .. 4 i + 3 of the thread's 16, of two rows each
                            const uint32_t al = __byte_perm(A0[i], A1[i], 0x5140) ^ 0x80808080u, ah = __byte_perm(A0[i], A1[i], 0x7362) ^ 0x80808080u;
                            const uint32_t bl = __byte_perm(B0[i], B1[i], 0x5140) ^ 0x80808080u, bh = __byte_perm(B0[i], B1[i], 0x7362) ^ 0x80808080u;
                            product(16 * h + 4 * i, bytesLo(al), bytesLo(bl));
                            product(16 * h + 4 * i + 1, bytesHi(al), bytesHi(bl));
                            product(16 * h + 4 * i + 2, bytesLo(ah), bytesLo(bh));
                            product(16 * h + 4 * i + 3, bytesHi(ah), bytesHi(bh));
                        }
                    }
                } else {
                    const uint32_t key = key0 + 16u * kk + ((lane >> 3) & 1u) * 8u + (lane & 7u), x = key & 7u;
#pragma unroll
                    for (int j = 0; j < NJ; j += 2) {
                        const uint32_t chunk = j + (lane >> 4);
                        uint32_t r0, r1, r2, r3;
                        ldmatrixX4Trans(r0, r1, r2, r3, sV + (chunk >> 3) * L::kPanel + key * 128u + (((chunk & 7u) ^ x) << 4));
                        product(j, r0, r1);
                        product(j + 1, r2, r3);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbarArrive(&empty[st]);
        }
        // ---- the shares of a row group, then the blocks of the item ----
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
        float f[NR], M[NR], sum[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) M[r] = m[r], sum[r] = l[r];
        if (WK > 1) {
#pragma unroll
            for (int r = 0; r < NR; ++r)
                if (c == 0) ml[warp * 16u + n8 + 8u * r] = make_float2(m[r], l[r]);
            groupSync();
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float2 x[WK];
                M[r] = -INFINITY, sum[r] = 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < WK; ++i) x[i] = ml[(wm * WK + i) * 16u + n8 + 8u * r], M[r] = fmaxf(M[r], x[i].x);
#pragma unroll
                for (uint32_t i = 0; i < WK; ++i) sum[r] = fmaf(fastExp2(x[i].x - (M[r] == -INFINITY ? 0.0f : M[r])), x[i].y, sum[r]);
            }
        }
        const bool whole = it.whole != 0u;
        float *part = p.parts + (2u * static_cast<size_t>(blockIdx.x) + it.part) * pagedSlot(MR, HD);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const float Mu = M[r] == -INFINITY ? 0.0f : M[r];
            f[r] = fastExp2(m[r] - Mu) * (whole ? (M[r] == -INFINITY ? 0.0f : 1.0f / sum[r]) : 1.0f);
            if (I8) f[r] *= __uint_as_float(static_cast<uint32_t>(127 + vexp) << 23);
            if (!whole && wk == 0 && c == 0) {
                const uint32_t i = wm * L::RW + n8 + 8u * r;
                part[MR * HD + i] = M[r], part[MR * HD + MR + i] = sum[r];
            }
        }
        constexpr int PJ = 4;  // output tiles of a pass: 32 dims
#pragma unroll
        for (int pass = 0; pass < NJ / PJ; ++pass) {
            if (pass > 0) groupSync();
            float *b = buf + warp * (16u * 36u);
#pragma unroll
            for (int jj = 0; jj < PJ; ++jj) {
                const int j = pass * PJ + jj;
#pragma unroll
                for (int e = 0; e < OR; ++e) {
                    const int r = e >> 1;
                    const uint32_t col = 2u * c + (e & 1);
                    b[(n8 + 8u * r) * 36u + (I8 ? col * 4u + jj : jj * 8u + col)] = o[j][e] * f[r];
                }
            }
            groupSync();
            for (uint32_t i = wk * 32u + lane; i < L::RW * 8u; i += WK * 32u) {
                const uint32_t row = i >> 3, q4 = i & 7u;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (uint32_t k = 0; k < WK; ++k) {
                    const float4 y = *reinterpret_cast<const float4 *>(buf + (wm * WK + k) * (16u * 36u) + row * 36u + q4 * 4u);
                    x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
                }
                const uint32_t dim = I8 ? 128u * (pass / 4) + 16u * q4 + 4u * (pass % 4) : 32u * pass + 4u * q4;
                const uint32_t local = wm * L::RW + row, r = it.m0 + local;
                if (r >= it.rows) continue;
                if (whole) pagedStore(p, HD, it.token0, it.kvHead, r, dim, x);
                else __stcg(reinterpret_cast<float4 *>(part + local * HD + dim), x);
            }
        }
        groupSync();
    }
}

static uint32_t pagedRowsBlocks(uint32_t hd) { return std::min(numSMs(), kPagedSMs) * (hd == 256 ? 1 : 2); }
template <int HD, bool I8, bool PAIR, int WM>
static int launchPagedRows(const CUtensorMap &k, const CUtensorMap &v, const PagedAttnParams &p, cudaStream_t st) {
    using L = PaL<HD, I8, PAIR, WM>;
    auto kern = pagedRowsKernel<HD, I8, PAIR, WM>;
    static bool attrDone[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attrDone[dev]) {
        TC_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal));
        attrDone[dev] = true;
    }
    const uint32_t blocks = pagedRowsBlocks(HD);
    return launchDependent(kern, dim3(blocks), L::kThreads, L::kTotal, st, 1, k, v, p);
}

int pagedMaps(const tc_paged_kv *c, uint32_t box, CUtensorMap *k, CUtensorMap *v) {
    const uint32_t e = c->kvI8 ? 1 : 2;
    TensorMapKey key;
    memset(&key, 0, sizeof(key));
    key.dims[0] = c->hd, key.dims[1] = c->nKV, key.dims[2] = c->pageRows, key.dims[3] = c->numPages;
    key.strides[0] = static_cast<uint64_t>(c->hd) * e;
    key.strides[1] = key.strides[0] * c->nKV;
    key.strides[2] = key.strides[1] * c->pageRows;
    key.box[0] = 128 / e, key.box[1] = 1, key.box[2] = box, key.box[3] = 1;
    key.rank = 4, key.elemBytes = e, key.swizzle = 3;
    key.promote128 = c->hd * e == 128;  // (256 would bring a row of the next kv head, which another block asks for much later)
    key.base = c->k;
    const int rc = getTensorMap(key, k);
    if (rc != TC_OK) return rc;
    key.base = c->v;
    return getTensorMap(key, v);
}

// rows: how many query rows per kv head a sequence brings as a rule, for the choice of a form; any number is right
static int pagedAttnRows(const tc_paged_kv *c, const PagedAttnParams &p, uint32_t rows, cudaStream_t st, uint32_t *blocks) {
    if (rows <= pagedStepRows(c)) return pagedAttnSteps(c, p, rows, st, blocks);
    CUtensorMap k, v;
    const int rc = pagedMaps(c, p.box, &k, &v);
    if (rc != TC_OK) return rc;
    *blocks = pagedRowsBlocks(c->hd);
    const int wm = !p.half || rows > 32 ? 4 : 2;  // (f32 results: the forms of fewer rows are paged_steps.cu's)
#define TC_PAGED_ROWS(HD, I8) \
    (!p.half ? launchPagedRows<HD, I8, true, 4>(k, v, p, st) : wm == 2 ? launchPagedRows<HD, I8, false, 2>(k, v, p, st) : launchPagedRows<HD, I8, false, 4>(k, v, p, st))
    if (c->kvI8) return c->hd == 128 ? TC_PAGED_ROWS(128, true) : TC_PAGED_ROWS(256, true);
    if (c->hd == 64) return TC_PAGED_ROWS(64, false);
    return c->hd == 128 ? TC_PAGED_ROWS(128, false) : TC_PAGED_ROWS(256, false);
#undef TC_PAGED_ROWS
}

// Query rows per kv head from which on a call's sequences are tiles of the tensor cores; in such a call, what the rows kernel keeps.
constexpr uint32_t kTilesFrom = 64, kRowsBeside = 16;

}  // namespace tc

extern "C" {

int tc_attn_paged_workspace_bytes(size_t *bytes) {
    using namespace tc;
    TC_REQUIRE(bytes != nullptr, TC_EINVAL, "paged attention: null pointer");
    *bytes = kPagedWorkspace;
    return TC_OK;
}

int tc_attn_paged(const tc_paged_kv *c, const void *q, void *out, int half, uint32_t nHeads, uint32_t maxTokens, float invSqrt,
                  void *workspace, size_t workspaceBytes, tc_stream stream) {
    using namespace tc;
    const int rc = pagedCheck(c, "paged attention");
    if (rc != TC_OK) return rc;
    TC_REQUIRE(nHeads > 0 && nHeads % c->nKV == 0, TC_EINVAL, "paged attention: %u q heads over %u kv heads", nHeads, c->nKV);
    TC_REQUIRE(nHeads / c->nKV <= 128, TC_EUNSUPPORTED, "paged attention: %u q heads per kv head (at most 128)", nHeads / c->nKV);
    TC_REQUIRE(static_cast<uint64_t>(c->tokens) * nHeads <= 0x7fffffffull, TC_EUNSUPPORTED, "paged attention: too many query rows");
    TC_REQUIRE(invSqrt > 0.0f && invSqrt < INFINITY, TC_EINVAL, "paged attention: scale");
    if (c->tokens == 0) return TC_OK;
    TC_REQUIRE(q != nullptr && out != nullptr && workspace != nullptr, TC_EINVAL, "paged attention: null pointer");
    TC_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15u) == 0,
               TC_EINVAL, "paged attention: alignment (16 bytes)");
    TC_REQUIRE(workspaceBytes >= kPagedWorkspace, TC_EWORKSPACE, "paged attention: %zu bytes of workspace, %zu needed", workspaceBytes, kPagedWorkspace);
    unsigned int *err = devErrorWord();
    TC_REQUIRE(err != nullptr, TC_ECUDA, "no CUDA device");
    const uint32_t most = c->starts != nullptr ? c->tokens : c->tokens / c->batch;
    if (maxTokens == 0 || maxTokens > most) maxTokens = most;
    const uintptr_t base = (reinterpret_cast<uintptr_t>(workspace) + 31) & ~uintptr_t(31);
    PagedAttnParams p;
    p.c = pagedView(c, err);
    p.q = q, p.out = out, p.ks = c->ks, p.vs = c->vs;
    p.parts = reinterpret_cast<float *>(base);
    float *const partsB = p.parts + kRowsParts;
    p.joins = reinterpret_cast<PagedJoin *>(partsB + kTilesParts);
    PagedJoin *const joinsB = p.joins + 3 * kPagedSMs;
    p.nHeads = nHeads, p.group = nHeads / c->nKV;
    p.box = 64;
    while (c->pageRows % p.box != 0) p.box /= 2;
    p.tileTokens = kPagedTile / p.group;
    p.out32 = (reinterpret_cast<uintptr_t>(out) & 31u) == 0;
    p.scaleLog2 = invSqrt * kLog2e;
    p.half = half != 0;
    const uint32_t rows = maxTokens * p.group;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Sequences with many query rows go to the tensor cores' tiles, the others of the call to the rows kernel.
    const bool tiles = half && rows > kTilesFrom;
    const bool rowsToo = !tiles || (c->starts != nullptr && c->batch > 1);
    uint32_t blocksA = 0;
    if (rowsToo) {
        p.minRows = 1, p.maxRows = tiles ? kRowsBeside : 0xffffffffu;
        const int ra = pagedAttnRows(c, p, tiles ? kRowsBeside : rows, st, &blocksA);
        if (ra != TC_OK) return ra;
    }
    if (tiles) {
        PagedAttnParams b = p;
        b.parts = partsB, b.joins = joinsB;
        b.minRows = rowsToo ? kRowsBeside + 1 : 1, b.maxRows = 0xffffffffu;
        const int rb = pagedAttnTiles(c, b, st);
        if (rb != TC_OK) return rb;
    }
    const dim3 grid(blocksA + (tiles ? std::min(numSMs(), kPagedSMs) : 0), 8);
    auto merge = c->hd == 64 ? pagedMergeKernel<64> : c->hd == 128 ? pagedMergeKernel<128> : pagedMergeKernel<256>;
    return launchDependent(merge, grid, 256, 0, st, 1, p, static_cast<const float *>(partsB), static_cast<const PagedJoin *>(joinsB), blocksA);
}

}  // extern "C"
