// paged_steps.cu -- attention of few query rows per kv head over a paged cache: decode steps and drafts, and what f32 queries have of more
// over int8 pages and at head_dim 256, 16 rows an item.
//
// The work, the ring and the partials are paged_attn.cuh's; the products have the cache rows on the M side of mma.sync m16n8k16: S^T = K Q^T
// (16 cache rows x 8 query rows) and O^T += V^T P^T (16 dims x 8 query rows), so that 8 query rows fill an instruction and an
// int8 row is turned into fp16 once for all of a block's query rows.  A warp takes 16 of a tile's 64 rows.  What bounds it is the cache for fp16
// pages; over int8 ones no unit by itself but a warp's chain per tile, the conversions in it (two byte permutes, half an exclusive-or and an
// fp16 subtraction per two values).
//   * P^T is S^T's accumulator through movmatrix: a thread has keys n8, n8 + 8 of query rows 2 c, 2 c + 1 and needs keys 2 c, 2 c + 1 of row n8.
//   * The running maximum is lazy: a vote finds whether any score is 2^8 (f32 results: 2^2) above it, and only then do the lanes exchange
//     maxima and rescale.
// Measured (warm graph, tokens of one step): fp16 pages 64 sessions of 40 / 8 / 128 6.5 TB/s, of 40 / 8 / 64 5.8, int8 pages 32 sessions of
// 512 - 32768 rows of 28 / 4 / 128 5.5 TB/s, with the ALU pipe and the issue slots half busy.  One session of 8191 int8 rows
// takes 15.5 us, two thirds of it the way from launch to launch.
//   * EXACT (f32 results): q and p as fp16 pairs, hi and lo in two products; the products of a tile are summed by themselves and join f32 registers,
//     since the tensor unit cuts off what an addition shifts out.  fp16 results accumulate in the instruction: some 2^-25 of
//     the sum lost per tile (a warp's 16 rows), 2^-14 behind 113000 rows of one block.
#include <algorithm>

#include "paged_attn.cuh"

namespace tc {

// p is held as 2^off p, at most 2^(off + lag) = 2^15: the smallest step of fp16 is 2^-24, so a weight is off by 2^-(25 + off) of the row's
// largest at most, over int8 pages (p times a scale relative to at most twice the largest) by twice that.  An f32 result may consist of
// small weights alone, where the large ones meet V = 0: 2^-38 instead of 2^-32 costs more frequent rescales.
template <bool EXACT>
struct PsRange {
    static constexpr float off = EXACT ? 13.0f : 7.0f, lag = EXACT ? 2.0f : 8.0f;
};

template <int HD, bool I8, bool EXACT, int NT>
struct PsL {
    static constexpr bool kI8 = I8;
    static constexpr int NW = 4, kThreads = 160, MR = 8 * NT;
    static constexpr int kPanels = HD * (I8 ? 1 : 2) / 128;
    static constexpr int kPanel = int(kPaTile) * 128;
    static constexpr int kMat = kPanels * kPanel;
    static constexpr int kStage = 2 * kMat;
    static constexpr bool kQRegs = NT == 1 && !(HD == 256 && EXACT);           // q in registers, else in shared memory
    // (in registers head_dim 256 with f32 results spills at two blocks per SM: 64 sessions of 16 / 2 / 256 over int8 pages 79 us, one block
    // 72, two with q in shared memory 64)
    static constexpr int kBlocks = HD == 256 ? (I8 && NT == 1 ? 2 : 1) : kStage == 16384 && NT == 1 ? 3 : 2;
    static constexpr int NST = kStage == 65536 ? (NT > 1 ? 2 : 3) : kStage == 32768 ? (kBlocks == 1 ? 5 : NT > 1 ? 2 : 3) : kBlocks == 3 ? (HD == 64 ? 4 : 3) : 5;
    static constexpr int NS = HD / 16;
    static constexpr int kScales = NST * kStage;                              // [stage][K, V][64]
    static constexpr int kQ = kScales + (I8 ? NST * 512 : 0);                 // NT > 1: [n tile][step][lane] hi (lo) pairs
    static constexpr int kBuf = kQ + (kQRegs ? 0 : NT * NS * 32 * (EXACT ? 16 : 8));
    static constexpr int kPass = NT == 1 && I8 && HD == 128 ? 128 : 32;      // dims that the warps put together at a time
    static constexpr int kMl = kBuf + NW * MR * (kPass + 4) * 4;              // [warp][row] (m, l)
    static constexpr int kRowScale = kMl + NW * MR * 8;
    static constexpr int kItems = kRowScale + MR * 4;
    static constexpr int kBars = (kItems + int(kPaItems * sizeof(PaItem)) + 7) / 8 * 8;
    static constexpr int kTotal = kBars + (2 * NST + int(kPaItems)) * 8 + 1024;
    static_assert(NST + 2 <= int(kPaItems), "items");
    static_assert(kBlocks * (kTotal + 1024) <= 228 * 1024, "shared memory of an SM");
    static_assert(size_t(2) * kPagedSMs * kBlocks * pagedSlot(MR, HD) <= kStepsParts && kBlocks <= 3, "the workspace's room");
};

template <int HD, bool I8, bool EXACT, int NT>
__global__ void __launch_bounds__((PsL<HD, I8, EXACT, NT>::kThreads), (PsL<HD, I8, EXACT, NT>::kBlocks))
pagedStepsKernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedAttnParams p) {
    using L = PsL<HD, I8, EXACT, NT>;
    constexpr uint32_t NST = L::NST, MR = L::MR;
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
    if (warp == L::NW) {
        pagedProduce<L>(p, tmK, tmV, smem, full, empty, itemFull, items);
        return;
    }

    gridDepWait();
    gridDepLaunch();

    const uint32_t c = lane & 3u, n8 = lane >> 2, key0 = warp * 16u;
    constexpr int NS = L::NS, NM = HD / 16, QW = EXACT ? 4 : 2;  // steps of q . K; 16-dim output tiles; registers of a step's q
    constexpr bool kQRegs = L::kQRegs;
    float *buf = reinterpret_cast<float *>(smem + L::kBuf), *rowScaleS = reinterpret_cast<float *>(smem + L::kRowScale);
    float2 *ml = reinterpret_cast<float2 *>(smem + L::kMl);
    uint32_t *qS = reinterpret_cast<uint32_t *>(smem + L::kQ);
    uint32_t g = 0;
    bool ok = true;  // (a warp that gave up still takes its items and meets the others at their barriers)
    for (uint32_t n = 0;; ++n) {
        // The producer hands in the end of the run whatever becomes of its waits, each of which is bounded: this one only has to be longer.
        for (uint32_t i = 0; i < (1u << 20) && !mbarTryWait(&itemFull[n % kPaItems], (n / kPaItems) & 1u); ++i) {}
        const PaItem it = items[n % kPaItems];
        if (it.nTiles == 0u) break;

        // ---- q as B operands: thread (n8, c) holds four dims of row n8 a step, in the order of its 16-byte loads of K ----
        uint32_t qr[kQRegs ? NS : 1][QW];
        float rowScale[2 * NT];
        auto loadQ = [&](uint32_t nt, auto &&put) {
            const uint32_t rr = it.m0 + 8u * nt + n8;
            const bool valid = rr < it.rows;
            auto dim = [&](int st) { return I8 ? 128 * (st / 8) + 32 * static_cast<int>(c) + 4 * (st % 8) : 64 * (st / 4) + 16 * static_cast<int>(c) + 4 * (st % 4); };
            if constexpr (EXACT) {
                return p.scaleLog2 * pagedQuery<NS>(p, it, rr, valid, HD, dim, put);
            } else {
                const uint32_t tok = it.token0 + rr / p.group, head = it.kvHead * p.group + rr % p.group;
                const __half *src = static_cast<const __half *>(p.q) + (static_cast<size_t>(tok) * p.nHeads + head) * HD;
#pragma unroll
                for (int st = 0; st < NS; ++st) {
                    uint2 x = make_uint2(0u, 0u);
                    if (valid) x = __ldg(reinterpret_cast<const uint2 *>(src + dim(st)));
                    const uint32_t w[2] = {x.x, x.y};
                    put(st, w);
                }
                return p.scaleLog2;
            }
        };
        if constexpr (kQRegs) {
            const float s = loadQ(0, [&](int st, const uint32_t(&w)[QW]) {
#pragma unroll
                for (int i = 0; i < QW; ++i) qr[st][i] = w[i];
            });
            rowScale[0] = __shfl_sync(0xffffffffu, s, 8u * c), rowScale[1] = __shfl_sync(0xffffffffu, s, 8u * c + 4u);
        } else {
            for (uint32_t nt = warp; nt < NT; nt += 4u) {
                const float s = loadQ(nt, [&](int st, const uint32_t(&w)[QW]) {
                    uint32_t *d = qS + ((nt * NS + st) * 32u + lane) * QW;
                    if constexpr (EXACT) *reinterpret_cast<uint4 *>(d) = make_uint4(w[0], w[1], w[QW - 2], w[QW - 1]);
                    else *reinterpret_cast<uint2 *>(d) = make_uint2(w[0], w[1]);
                });
                if (c == 0) rowScaleS[8u * nt + n8] = s;
            }
            namedBarSync(1, 128);
#pragma unroll
            for (int r = 0; r < 2 * NT; ++r) rowScale[r] = rowScaleS[8 * (r / 2) + 2 * c + (r & 1)];
        }
        // rows of a thread: r = 2 nt + e is query row 8 nt + 2 c + e; cache rows that it sees (rows that do not exist: all, unused)
        int32_t vis[2 * NT], leastVis = 0x7fffffff;
#pragma unroll
        for (int r = 0; r < 2 * NT; ++r) {
            const uint32_t rr = it.m0 + 8u * (r / 2) + 2u * c + (r & 1);
            vis[r] = rr < it.rows ? it.before + static_cast<int32_t>(rr / p.group) + 1 : 0x7fffffff;
            leastVis = min(leastVis, vis[r]);
        }
        leastVis = __reduce_min_sync(0xffffffffu, leastVis);
        float m[2 * NT], l[2 * NT], o[NT][NM][4];
        int vexp = -126;  // int8: the accumulators hold V 2^-vexp
        float down = __uint_as_float(253u << 23), most = __uint_as_float(1u << 23);
#pragma unroll
        for (int r = 0; r < 2 * NT; ++r) m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < NM; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][j][e] = 0.0f;

        const uint32_t t0 = it.t0, t1 = t0 + it.nTiles;
        for (uint32_t t = t0; t < t1; ++t, ++g) {
            const uint32_t st = g % NST;
            ok = ok && pfWait<true>(&full[st], (g / NST) & 1u, p.c.err, kDevErrFullWait);
            if (!ok) break;
            const uint32_t sK = smemAddr(smem + st * L::kStage), sV = sK + L::kMat;
            const float *sc = reinterpret_cast<const float *>(smem + L::kScales) + st * 128u + key0;
            const int32_t tile0 = static_cast<int32_t>(t * kPaTile);
            const int32_t left = static_cast<int32_t>(it.len) - tile0 - static_cast<int32_t>(key0);  // of the warp's rows those that exist
            // ---- S^T: element e of an accumulator is cache row n8 + 8 (e >> 1), query row 2 c + (e & 1) ----
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[nt][e] = 0.0f;
            auto score = [&](int step, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    uint32_t w[QW];
                    if constexpr (kQRegs) {
#pragma unroll
                        for (int i = 0; i < QW; ++i) w[i] = qr[step][i];
                    } else {
                        const uint32_t *d = qS + ((nt * NS + step) * 32u + lane) * QW;
                        if constexpr (EXACT) {
                            const uint4 x = *reinterpret_cast<const uint4 *>(d);
                            w[0] = x.x, w[1] = x.y, w[QW - 2] = x.z, w[QW - 1] = x.w;
                        } else {
                            const uint2 x = *reinterpret_cast<const uint2 *>(d);
                            w[0] = x.x, w[1] = x.y;
                        }
                    }
                    mmaF16(s[nt], a0, a1, a2, a3, w[0], w[1]);
                    if constexpr (EXACT) mmaF16(s[nt], a0, a1, a2, a3, w[QW - 2], w[QW - 1]);
                }
            };
            {
                const uint32_t x = n8, rowA = (key0 + n8) * 128u, rowB = rowA + 8u * 128u;  // (key0 and 8 leave the swizzle's row as it is)
                const uint32_t ch0 = ((2u * c) ^ x) << 4, ch1 = ((2u * c + 1u) ^ x) << 4;
#pragma unroll
                for (int h = 0; h < L::kPanels; ++h) {
                    const uint32_t base = sK + h * L::kPanel;
                    const uint4 a = ldShared4(base + rowA + ch0), b = ldShared4(base + rowA + ch1);
                    const uint4 d = ldShared4(base + rowB + ch0), e = ldShared4(base + rowB + ch1);
                    const uint32_t va[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, vb[8] = {d.x, d.y, d.z, d.w, e.x, e.y, e.z, e.w};
                    if constexpr (I8) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint32_t ua = va[i] ^ 0x80808080u, ub = vb[i] ^ 0x80808080u;
                            score(8 * h + i, bytesLo(ua), bytesLo(ub), bytesHi(ua), bytesHi(ub));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) score(4 * h + i, va[2 * i], vb[2 * i], va[2 * i + 1], vb[2 * i + 1]);
                    }
                }
            }
            float k0 = 1.0f, k1 = 1.0f;
            if constexpr (I8) k0 = sc[n8], k1 = sc[n8 + 8u];
            bool ahead = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[nt][e] *= (e >> 1 ? k1 : k0) * rowScale[2 * nt + (e & 1)];
            if (tile0 + static_cast<int32_t>(kPaTile) > leastVis) {  // (whatever a masked place holds, a select takes it out)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (tile0 + static_cast<int32_t>(key0 + n8 + 8u * (e >> 1)) >= vis[2 * nt + (e & 1)]) s[nt][e] = -INFINITY;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) ahead = ahead || s[nt][e] > m[2 * nt + (e & 1)] + PsRange<EXACT>::lag;
            if (__any_sync(0xffffffffu, ahead)) {
#pragma unroll
                for (int r = 0; r < 2 * NT; ++r) {
                    float mx = fmaxf(s[r / 2][r & 1], s[r / 2][2 + (r & 1)]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    mx = fmaxf(mx, m[r]);
                    const float alpha = fastExp2(m[r] - (mx == -INFINITY ? 0.0f : mx));
                    m[r] = mx, l[r] *= alpha;
#pragma unroll
                    for (int j = 0; j < NM; ++j) o[r / 2][j][r & 1] *= alpha, o[r / 2][j][2 + (r & 1)] *= alpha;
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float mr = m[2 * nt + (e & 1)];
                    s[nt][e] = fastExp2(s[nt][e] - ((mr == -INFINITY ? 0.0f : mr) - PsRange<EXACT>::off));
                    l[2 * nt + (e & 1)] += s[nt][e];
                }
            if constexpr (I8) {
                // p times the scale of V's row, relative to a power of two no smaller than any scale so far
                float v0 = sc[64u + n8], v1 = sc[64u + n8 + 8u];
                if (static_cast<int32_t>(n8) >= left) v0 = 0.0f;
                if (static_cast<int32_t>(n8) + 8 >= left) v1 = 0.0f;
                const uint32_t top = max(__float_as_uint(v0) & 0x7fffffffu, __float_as_uint(v1) & 0x7fffffffu);
                if (__any_sync(0xffffffffu, top >= __float_as_uint(most))) {
                    const int e = max(vexp, min(126, static_cast<int>(__reduce_max_sync(0xffffffffu, top) >> 23) - 126));
                    const float f = fastExp2(static_cast<float>(vexp - e));
                    vexp = e, down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23), most = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < NM; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[nt][j][i] *= f;
                }
                v0 *= down, v1 *= down;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][0] *= v0, s[nt][1] *= v0, s[nt][2] *= v1, s[nt][3] *= v1;
            } else if (left < 16) {
                // rows past the sequence: what stands there is no number that 0 could be multiplied with
                for (int32_t i = static_cast<int32_t>(lane); i < 16 * 8 * L::kPanels; i += 32) {
                    const int32_t key = i & 15, chunk = i >> 4;
                    if (key >= left)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sV + (chunk / 8) * L::kPanel + (key0 + key) * 128 + (chunk % 8) * 16), "r"(0u) : "memory");
                }
                fenceProxyAsync();  // (TMA writes this room next)
                __syncwarp();
            }
            // ---- P^T as B operands, then O^T ----
            uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if constexpr (EXACT) {
                    float h[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) splitHalf(s[nt][e], h[e], lo[e]);
                    ph[nt][0] = movmatrixTrans(packHalf2(h[0], h[1])), ph[nt][1] = movmatrixTrans(packHalf2(h[2], h[3]));
                    pl[nt][0] = movmatrixTrans(packHalf2(lo[0], lo[1])), pl[nt][1] = movmatrixTrans(packHalf2(lo[2], lo[3]));
                } else {
                    ph[nt][0] = movmatrixTrans(packHalf2(s[nt][0], s[nt][1])), ph[nt][1] = movmatrixTrans(packHalf2(s[nt][2], s[nt][3]));
                }
            }
            auto product = [&](int j, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if constexpr (EXACT) {
                        float d[4] = {0.f, 0.f, 0.f, 0.f};
                        mmaF16(d, a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
                        mmaF16(d, a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[nt][j][e] += d[e];
                    } else {
                        mmaF16(o[nt][j], a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
                    }
                }
            };
            if constexpr (I8) {
                const uint32_t k = key0 + 2u * c;
#pragma unroll
                for (int h = 0; h < L::kPanels; ++h) {
                    auto load = [&](uint32_t key) { return ldShared4(sV + h * L::kPanel + key * 128u + ((n8 ^ (key & 7u)) << 4)); };
                    const uint4 a0 = load(k), a1 = load(k + 1u), b0 = load(k + 8u), b1 = load(k + 9u);
                    const uint32_t A0[4] = {a0.x, a0.y, a0.z, a0.w}, A1[4] = {a1.x, a1.y, a1.z, a1.w};
                    const uint32_t B0[4] = {b0.x, b0.y, b0.z, b0.w}, B1[4] = {b1.x, b1.y, b1.z, b1.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // dims 4 i .. 4 i + 3 of the thread's 16: rows n8 and n8 + 8 of an output tile are two of them
                        const uint32_t al = __byte_perm(A0[i], A1[i], 0x5140) ^ 0x80808080u, ah = __byte_perm(A0[i], A1[i], 0x7362) ^ 0x80808080u;
                        const uint32_t bl = __byte_perm(B0[i], B1[i], 0x5140) ^ 0x80808080u, bh = __byte_perm(B0[i], B1[i], 0x7362) ^ 0x80808080u;
                        product(8 * h + 2 * i, bytesLo(al), bytesHi(al), bytesLo(bl), bytesHi(bl));
                        product(8 * h + 2 * i + 1, bytesLo(ah), bytesHi(ah), bytesLo(bh), bytesHi(bh));
                    }
                }
            } else {
                const uint32_t key = key0 + ((lane >> 3) & 1u) * 8u + (lane & 7u), x = key & 7u;
#pragma unroll
                for (int j = 0; j < NM; ++j) {
                    const uint32_t chunk = 2u * j + (lane >> 4);
                    uint32_t r0, r1, r2, r3;
                    ldmatrixX4Trans(r0, r1, r2, r3, sV + (chunk >> 3) * L::kPanel + key * 128u + (((chunk & 7u) ^ x) << 4));
                    product(j, r0, r2, r1, r3);
                }
            }
            uint32_t used = 0u;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < NM; ++j) used ^= __float_as_uint(o[nt][j][0]);
            releaseStage(&empty[st], used, p.zero);
        }

        // ---- the four warps' shares ----
#pragma unroll
        for (int r = 0; r < 2 * NT; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 4);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 8);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 16);
            if (n8 == 0) ml[warp * MR + 8u * (r / 2) + 2u * c + (r & 1)] = make_float2(m[r], l[r]);
        }
        namedBarSync(1, 128);
        const bool whole = it.whole != 0u;
        float *part = p.parts + (2u * static_cast<size_t>(blockIdx.x) + it.part) * pagedSlot(MR, HD);
        float f[2 * NT];
#pragma unroll
        for (int r = 0; r < 2 * NT; ++r) {
            const uint32_t row = 8u * (r / 2) + 2u * c + (r & 1);
            float2 x[4];
            float M = -INFINITY, sum = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) x[i] = ml[i * MR + row], M = fmaxf(M, x[i].x);
            const float Mu = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) sum = fmaf(fastExp2(x[i].x - Mu), x[i].y, sum);
            f[r] = fastExp2(m[r] - Mu) * (whole ? (M == -INFINITY ? 0.0f : 1.0f / sum) : 1.0f);
            if (I8) f[r] *= __uint_as_float(static_cast<uint32_t>(127 + vexp) << 23);
            if (!whole && warp == 0 && n8 == 0) part[MR * HD + row] = M, part[MR * HD + MR + row] = sum;
        }
        // kPass dims at a time through shared memory
        constexpr int PW = L::kPass, PT = PW / 16;  // 16-dim tiles of a pass
        constexpr uint32_t kRow = PW + 4;
#pragma unroll
        for (int pass = 0; pass < NM / PT; ++pass) {
            if (pass > 0) namedBarSync(1, 128);
            float *b = buf + warp * (MR * kRow);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int jj = 0; jj < PT; ++jj)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // int8: a pass of 32 dims has four of each 16 (a thread's quads), one of 128 has all of a panel
                        const uint32_t col = !I8       ? 16u * jj + 8u * (e >> 1) + n8
                                             : PW == 32 ? n8 * 4u + 2u * jj + (e >> 1)
                                                        : n8 * 16u + 2u * jj + (e >> 1);
                        b[(8u * nt + 2u * c + (e & 1)) * kRow + col] = o[nt][PT * pass + jj][e] * f[2 * nt + (e & 1)];
                    }
            namedBarSync(1, 128);
            for (uint32_t i = threadIdx.x; i < MR * (PW / 4); i += 128u) {
                const uint32_t row = i / (PW / 4), q4 = i % (PW / 4), r = it.m0 + row;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) {
                    const float4 y = *reinterpret_cast<const float4 *>(buf + k * (MR * kRow) + row * kRow + q4 * 4u);
                    x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
                }
                const uint32_t dim = I8 && PW == 32 ? 128u * (pass / 4) + 16u * q4 + 4u * (pass % 4) : PW * pass + 4u * q4;
                if (r >= it.rows) continue;
                if (whole) pagedStore(p, HD, it.token0, it.kvHead, r, dim, x);
                else __stcg(reinterpret_cast<float4 *>(part + row * HD + dim), x);
            }
        }
        namedBarSync(1, 128);
    }
}

template <int HD, bool I8, bool EXACT, int NT>
static int launchSteps(const CUtensorMap &k, const CUtensorMap &v, const PagedAttnParams &p, cudaStream_t st, uint32_t *blocks) {
    using L = PsL<HD, I8, EXACT, NT>;
    auto kern = pagedStepsKernel<HD, I8, EXACT, NT>;
    static bool attrDone[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attrDone[dev]) {
        TC_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal));
        attrDone[dev] = true;
    }
    *blocks = std::min(numSMs(), kPagedSMs) * L::kBlocks;
    return launchDependent(kern, dim3(*blocks), L::kThreads, L::kTotal, st, 1, k, v, p);
}

int pagedAttnSteps(const tc_paged_kv *c, const PagedAttnParams &p, uint32_t rows, cudaStream_t st, uint32_t *blocks) {
    CUtensorMap k, v;
    const int rc = pagedMaps(c, p.box, &k, &v);
    if (rc != TC_OK) return rc;
    // One group of 8 query rows an item or two: two share a converted tile, one leaves room for twice the warps.  Drafts of 16 - 48
    // rows of 16 / 2 / 256 with f32 results: int8 pages 63 us with two, 58 with one; fp16 pages 77 and 79.
    const bool one = rows <= 8 || (rows <= 64 && c->kvI8 && c->hd == 256 && !p.half);
#define TC_PAGED_NT(HD, I8, EXACT) (one ? launchSteps<HD, I8, EXACT, 1>(k, v, p, st, blocks) : launchSteps<HD, I8, EXACT, 2>(k, v, p, st, blocks))
#define TC_PAGED_STEPS(HD, I8) (p.half ? TC_PAGED_NT(HD, I8, false) : TC_PAGED_NT(HD, I8, true))
    if (c->kvI8) return c->hd == 128 ? TC_PAGED_STEPS(128, true) : TC_PAGED_STEPS(256, true);
    if (c->hd == 64) return TC_PAGED_STEPS(64, false);
    return c->hd == 128 ? TC_PAGED_STEPS(128, false) : TC_PAGED_STEPS(256, false);
#undef TC_PAGED_STEPS
#undef TC_PAGED_NT
}

}  // namespace tc
