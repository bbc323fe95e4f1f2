// paged_kv.cu -- the paged K/V cache's writer and reader, and the checks that all calls over such a cache share.
//
// Write: K' = rot(K, pos), V' = V of every new token into the row of its page, as fp16 or as int8 with a scale per row and kv
// head (scale = amax / 127, 1 where amax is 0; byte = round to even of x / scale), and q' = rot(q, pos) to f32 or fp16.  The
// arithmetic is kvAppendKernel's and kvQuantKernel's, bit for bit.  Read: the same rows back, byte x scale, as f32 or fp16.
// Both stream: HBM bounds the prompts, the chain starts -> lens -> page -> row the single tokens, so the rows that do
// not depend on it are requested ahead of it.
#include "paged.cuh"
#include "tc_tcgen05.cuh"

namespace tc {

int pagedCheck(const tc_paged_kv *c, const char *what) {
    TC_REQUIRE(c != nullptr, TC_EINVAL, "%s: null descriptor", what);
    TC_REQUIRE(c->k != nullptr && c->v != nullptr && c->pages != nullptr && c->lens != nullptr, TC_EINVAL, "%s: null pointer", what);
    TC_REQUIRE(!c->kvI8 || (c->ks != nullptr && c->vs != nullptr), TC_EINVAL, "%s: an int8 cache needs its scales", what);
    TC_REQUIRE(c->batch > 0 && c->pagesPerSeq > 0 && c->numPages > 0 && c->pageRows > 0 && c->nKV > 0, TC_EINVAL, "%s: empty cache", what);
    TC_REQUIRE(c->hd == 128 || c->hd == 256 || (c->hd == 64 && !c->kvI8), TC_EUNSUPPORTED,
               "%s: head_dim %u (fp16 pages take 64, 128 and 256, int8 pages 128 and 256)", what, c->hd);
    TC_REQUIRE(c->pageRows % 8 == 0, TC_EUNSUPPORTED, "%s: %u rows a page (a multiple of 8 is needed)", what, c->pageRows);
    TC_REQUIRE(c->nKV <= 65535u && c->pageRows <= (1u << 20) && c->numPages <= 0x7fffffffu && c->batch <= (1u << 20) && c->tokens <= 0x7fffffffu &&
                       static_cast<uint64_t>(c->pagesPerSeq) * c->pageRows <= 0x7fffff00ull,
               TC_EUNSUPPORTED, "%s: too many rows", what);
    TC_REQUIRE(c->starts != nullptr || c->tokens % c->batch == 0, TC_EINVAL, "%s: %u tokens do not divide by %u sequences: starts is needed", what,
               c->tokens, c->batch);
    TC_REQUIRE(((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15u) == 0, TC_EINVAL, "%s: pool alignment", what);
    return TC_OK;
}

PagedView pagedView(const tc_paged_kv *c, unsigned int *err) {
    return PagedView{c->pages, c->lens, c->starts, c->batch, c->pagesPerSeq, c->numPages, c->pageRows, c->nKV,
                     c->tokens, c->starts != nullptr ? 0u : c->tokens / c->batch, err};
}

// ---------------------------------------------------------------------------
// write
// ---------------------------------------------------------------------------
struct PagedWriteParams {
    PagedView c;
    void *kc, *vc;
    float *ks, *vs;
    const float *k, *v;
    float *q;
    void *qOut;
    const float *cosT, *sinT;
    uint32_t nHeads, tableRows, unitsPerToken;
    int qHalf;
};

// A row (a q, K or V head of a token) belongs to HD / 8 lanes; a lane holds four pairs (j .. j + 3 with their partners HD / 2
// further on), so the rotation needs no exchange and a row's largest is a few shuffles away.  A group of lanes takes U rows of one token:
// it looks the token up once and has 2 U loads under way.
template <int HD, bool I8, int U>
__global__ void __launch_bounds__(256) pagedWriteKernel(const __grid_constant__ PagedWriteParams p) {
    constexpr uint32_t G = HD / 8, kHalf4 = HD / 8;  // lanes of a row; float4 of half a row
    const uint32_t unit = blockIdx.x * (256u / G) + threadIdx.x / G;
    const uint32_t i = threadIdx.x & (G - 1u);
    const uint32_t t = unit / p.unitsPerToken, first = (unit - t * p.unitsPerToken) * U;
    const uint32_t rows = p.nHeads + 2u * p.c.nKV;
    gridDepWait();  // (no gridDepLaunch: int8 rows have to be in memory before a later grid may look)
    if (t >= p.c.tokens) return;
    float4 x0[U], x1[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t r = first + u;
        if (r >= rows) continue;
        const float *src = r < p.nHeads                ? p.q + (static_cast<size_t>(t) * p.nHeads + r) * HD
                           : r < p.nHeads + p.c.nKV ? p.k + (static_cast<size_t>(t) * p.c.nKV + (r - p.nHeads)) * HD
                                                    : p.v + (static_cast<size_t>(t) * p.c.nKV + (r - p.nHeads - p.c.nKV)) * HD;
        x0[u] = reinterpret_cast<const float4 *>(src)[i];
        x1[u] = reinterpret_cast<const float4 *>(src)[i + kHalf4];
    }
    uint32_t seq;
    int64_t pos;
    if (!findToken<G>(p.c, t, seq, pos)) return;
    const bool needRow = first + U > p.nHeads;
    size_t row = 0;
    const bool held = needRow && pagedRow(p.c, seq, pos, row);
    float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool turn = p.cosT != nullptr, inTable = pos >= 0 && pos < static_cast<int64_t>(p.tableRows);
    if ((needRow && !held) || (turn && !inTable)) {  // no page for the row, or no angle for the position: reported, nothing stored
        if (i == 0) atomicOr(p.c.err, kDevErrRowBound);
        if (turn && !inTable) return;
    }
    if (turn) {
        c = __ldg(reinterpret_cast<const float4 *>(p.cosT) + static_cast<size_t>(pos) * kHalf4 + i);
        s = __ldg(reinterpret_cast<const float4 *>(p.sinT) + static_cast<size_t>(pos) * kHalf4 + i);
    }
    auto half4 = [](const float4 &x) { return make_uint2(packHalf2(x.x, x.y), packHalf2(x.z, x.w)); };
    auto rot = [](float &a, float &b, float cc, float ss) {
        const float y = fmaf(a, cc, -__fmul_rn(b, ss));
        b = fmaf(a, ss, __fmul_rn(b, cc));
        a = y;
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t r = first + u;
        if (r >= rows) continue;  // (the same for all lanes of a group)
        const bool isQ = r < p.nHeads, isV = r >= p.nHeads + p.c.nKV;
        if (turn && !isV) {
            rot(x0[u].x, x1[u].x, c.x, s.x);
            rot(x0[u].y, x1[u].y, c.y, s.y);
            rot(x0[u].z, x1[u].z, c.z, s.z);
            rot(x0[u].w, x1[u].w, c.w, s.w);
        }
        if (isQ) {
            const size_t at = (static_cast<size_t>(t) * p.nHeads + r) * (HD / 4) + i;
            if (p.qHalf) {
                static_cast<uint2 *>(p.qOut)[at] = half4(x0[u]);
                static_cast<uint2 *>(p.qOut)[at + kHalf4] = half4(x1[u]);
            } else {
                static_cast<float4 *>(p.qOut)[at] = x0[u];
                static_cast<float4 *>(p.qOut)[at + kHalf4] = x1[u];
            }
            continue;
        }
        const size_t rowHead = row * p.c.nKV + (r - p.nHeads - (isV ? p.c.nKV : 0u));
        void *pool = isV ? p.vc : p.kc;
        if constexpr (I8) {
            auto amax4 = [](const float4 &x) { return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))); };
            const uint32_t lane = threadIdx.x & 31u;
            const uint32_t mask = G == 32 ? 0xffffffffu : ((1u << (G & 31u)) - 1u) << (lane & ~(G - 1u));
            float m = fmaxf(amax4(x0[u]), amax4(x1[u]));
#pragma unroll
            for (uint32_t o = G / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(mask, m, o));
            const float sc = m > 0.0f ? __fdiv_rn(m, 127.0f) : 1.0f;
            auto q8 = [&](float x) -> uint32_t {
                int v = __float2int_rn(__fdiv_rn(x, sc));
                v = v < -128 ? -128 : (v > 127 ? 127 : v);
                return static_cast<uint32_t>(v) & 0xffu;
            };
            auto pack = [&](const float4 &x) { return q8(x.x) | (q8(x.y) << 8) | (q8(x.z) << 16) | (q8(x.w) << 24); };
            if (!held) continue;
            if (i == 0) (isV ? p.vs : p.ks)[rowHead] = sc;
            uint32_t *d = static_cast<uint32_t *>(pool) + rowHead * (HD / 4) + i;
            d[0] = pack(x0[u]);
            d[kHalf4] = pack(x1[u]);
        } else {
            if (!held) continue;
            uint2 *d = static_cast<uint2 *>(pool) + rowHead * (HD / 4) + i;
            d[0] = half4(x0[u]);
            d[kHalf4] = half4(x1[u]);
        }
    }
}

// ---------------------------------------------------------------------------
// read
// ---------------------------------------------------------------------------
struct PagedReadParams {
    PagedView c;
    const void *kc, *vc;
    const float *ks, *vs;
    void *kOut, *vOut;
    uint32_t out32;  // the outputs are 32-byte aligned
};

// 16 bytes of a store row as f32 or fp16 values from element `at` on
template <bool I8, bool HALF>
__device__ __forceinline__ void pagedPut(void *out, size_t at, const uint4 &raw, float sc, bool out32) {
    constexpr uint32_t E = I8 ? 16 : 8;
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (!I8 && HALF) {
        *reinterpret_cast<uint4 *>(static_cast<__half *>(out) + at) = raw;
    } else {
        float f[E];
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) {
            if constexpr (I8) f[e] = static_cast<float>(static_cast<int8_t>((w[e / 4] >> (8 * (e % 4))) & 0xffu)) * sc;
            else f[e] = __half2float(__ushort_as_half(static_cast<unsigned short>((w[e / 2] >> (16 * (e % 2))) & 0xffffu)));
        }
        constexpr uint32_t N = HALF ? E / 2 : E;  // words
        uint32_t o[N];
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) o[i] = HALF ? packHalf2(f[2 * i], f[2 * i + (HALF ? 1 : 0)]) : __float_as_uint(f[i]);
        uint32_t *d = HALF ? reinterpret_cast<uint32_t *>(static_cast<__half *>(out) + at) : reinterpret_cast<uint32_t *>(static_cast<float *>(out) + at);
        // 32 bytes a store, whole sectors: 16 bytes at a stride of 32 take 46 us for what these take 36 (60000 int8 rows of 4 x 128 to fp16)
#pragma unroll
        for (uint32_t i = 0; i < N; i += 8) {
            if (N >= 8 && out32) {
                stGlobalV8(reinterpret_cast<float *>(d + i), __uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]),
                           __uint_as_float(o[i + (N >= 8 ? 4 : 0)]), __uint_as_float(o[i + (N >= 8 ? 5 : 1)]), __uint_as_float(o[i + (N >= 8 ? 6 : 2)]),
                           __uint_as_float(o[i + (N >= 8 ? 7 : 3)]));
            } else {
#pragma unroll
                for (uint32_t k = i; k < i + 8 && k < N; k += 4) *reinterpret_cast<uint4 *>(d + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
            }
        }
    }
}

// A lane takes 16 bytes of a store row (16 int8 or 8 fp16 values), a group of lanes the row.  For few rows, where the chain
// starts -> lens -> page -> row is all there is.
template <int HD, bool I8, bool HALF>
__global__ void __launch_bounds__(256) pagedReadKernel(const __grid_constant__ PagedReadParams p) {
    constexpr uint32_t E = I8 ? 16 : 8, G = HD / E;  // values of a lane; lanes of a row
    const uint32_t unit = blockIdx.x * (256u / G) + threadIdx.x / G;
    const uint32_t i = threadIdx.x & (G - 1u);
    const uint32_t rows = 2u * p.c.nKV, t = unit / rows, r = unit - t * rows;  // row r of token t: K heads, then V heads
    gridDepWait();
    gridDepLaunch();
    if (t >= p.c.tokens) return;
    uint32_t seq;
    int64_t pos;
    if (!findToken<G>(p.c, t, seq, pos)) return;
    size_t row = 0;
    const bool held = pagedRow(p.c, seq, pos, row), isV = r >= p.c.nKV;
    if (!held && i == 0) atomicOr(p.c.err, kDevErrRowBound);
    const uint32_t head = isV ? r - p.c.nKV : r;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);  // a row without a page reads as zero
    float sc = 0.0f;
    if (held) {
        const size_t rowHead = row * p.c.nKV + head;
        raw = __ldg(static_cast<const uint4 *>(isV ? p.vc : p.kc) + rowHead * G + i);
        if (I8) sc = __ldg((isV ? p.vs : p.ks) + rowHead);
    }
    pagedPut<I8, HALF>(isV ? p.vOut : p.kOut, ((static_cast<size_t>(t) * p.c.nKV + head) * G + i) * E, raw, sc, p.out32 != 0u);
}

// The same for many rows: a block takes kReadTokens tokens.  One warp looks them up, a lane each, and leaves their rows in shared memory; then
// every thread has U loads under way that wait for nothing else.  (A group of lanes that looks its own token up every four rows spends
// more than half of its time on that chain: 60000 rows of 4 x 128 int8 to fp16 43 us.)
constexpr uint32_t kReadTokens = 32;
template <int HD, bool I8, bool HALF>
__global__ void __launch_bounds__(256) pagedReadManyKernel(const __grid_constant__ PagedReadParams p) {
    constexpr uint32_t E = I8 ? 16 : 8, G = HD / E, U = 4;
    __shared__ int64_t rowS[kReadTokens];  // -1: no page; -2: of no sequence
    gridDepWait();
    gridDepLaunch();
    const uint32_t t0 = blockIdx.x * kReadTokens;
    if (threadIdx.x < kReadTokens) {
        const uint32_t t = t0 + threadIdx.x;
        int64_t at = -2;
        if (t < p.c.tokens) {
            uint32_t b = 0, n = p.c.batch, end, first = 0;
            if (p.c.starts == nullptr) {
                b = t / p.c.perSeq, end = (b + 1u) * p.c.perSeq;
            } else {
                while (n > 1u) {  // the last sequence that does not start behind t
                    const uint32_t half = n / 2u;
                    const bool right = __ldg(p.c.starts + b + half) <= t;
                    b += right ? half : 0u, n = right ? n - half : half;
                }
                end = __ldg(p.c.starts + b + 1u);
                if (b == 0u) first = __ldg(p.c.starts);
            }
            if (t >= first && t < end) {
                size_t row;
                at = pagedRow(p.c, b, static_cast<int64_t>(__ldg(p.c.lens + b)) - static_cast<int64_t>(end - t), row) ? static_cast<int64_t>(row) : -1;
                if (at < 0) atomicOr(p.c.err, kDevErrRowBound);
            }
        }
        rowS[threadIdx.x] = at;
    }
    __syncthreads();
    const uint32_t perToken = 2u * p.c.nKV * G, units = min(kReadTokens, p.c.tokens - t0) * perToken;
    for (uint32_t u0 = threadIdx.x; u0 < units; u0 += U * 256u) {
        uint4 raw[U];
        float sc[U];
        uint32_t tok[U], rest[U];
#pragma unroll
        for (uint32_t k = 0; k < U; ++k) {
            const uint32_t u = u0 + k * 256u;
            raw[k] = make_uint4(0u, 0u, 0u, 0u), sc[k] = 0.0f;
            tok[k] = u / perToken, rest[k] = u - tok[k] * perToken;
            if (u >= units) continue;
            const int64_t row = rowS[tok[k]];
            if (row < 0) continue;
            const uint32_t r = rest[k] / G, head = r >= p.c.nKV ? r - p.c.nKV : r;
            const size_t rowHead = static_cast<size_t>(row) * p.c.nKV + head;
            raw[k] = __ldg(static_cast<const uint4 *>(r >= p.c.nKV ? p.vc : p.kc) + rowHead * G + rest[k] % G);
            if (I8) sc[k] = __ldg((r >= p.c.nKV ? p.vs : p.ks) + rowHead);
        }
#pragma unroll
        for (uint32_t k = 0; k < U; ++k) {
            if (u0 + k * 256u >= units || rowS[tok[k]] == -2) continue;
            const uint32_t r = rest[k] / G, head = r >= p.c.nKV ? r - p.c.nKV : r;
            pagedPut<I8, HALF>(r >= p.c.nKV ? p.vOut : p.kOut, ((static_cast<size_t>(t0 + tok[k]) * p.c.nKV + head) * G + rest[k] % G) * E, raw[k], sc[k], p.out32 != 0u);
        }
    }
}

// blocks of 256 threads for `units` groups of `lanes` lanes
static int pagedGrid(uint64_t units, uint32_t lanes, uint32_t *blocks) {
    TC_REQUIRE(units < 0xffffff00ull, TC_EUNSUPPORTED, "paged rows: too many");
    const uint64_t n = (units * lanes + 255) / 256;
    *blocks = static_cast<uint32_t>(n);
    return TC_OK;
}

// Rows a group takes: one while the call is too small to fill the SMs otherwise, four beyond.
constexpr int kManyRows = 4;
static bool manyRows(uint64_t rows, uint32_t lanes) { return rows * lanes >= static_cast<uint64_t>(numSMs()) * 2048u * kManyRows; }

}  // namespace tc

extern "C" {

int tc_paged_kv_write(const tc_paged_kv *c, const float *k, const float *v, float *q, void *qOut, int qHalf, uint32_t nHeads,
                      const float *cosT, const float *sinT, uint32_t tableRows, tc_stream stream) {
    using namespace tc;
    const int rc = pagedCheck(c, "paged write");
    if (rc != TC_OK) return rc;
    TC_REQUIRE((cosT == nullptr) == (sinT == nullptr), TC_EINVAL, "paged write: cosT and sinT come together");
    if (q == nullptr) nHeads = 0;
    TC_REQUIRE(q == nullptr || (qOut != nullptr && nHeads > 0 && nHeads <= 65535u), TC_EINVAL, "paged write: q without a place or heads");
    TC_REQUIRE(q == nullptr || !qHalf || static_cast<const void *>(q) != qOut, TC_EINVAL, "paged write: fp16 q cannot replace f32 q in place");
    if (c->tokens == 0) return TC_OK;
    TC_REQUIRE(k != nullptr && v != nullptr, TC_EINVAL, "paged write: null pointer");
    uintptr_t align = 0;
    for (const void *a : {static_cast<const void *>(k), static_cast<const void *>(v), static_cast<const void *>(q), static_cast<const void *>(qOut),
                          static_cast<const void *>(cosT), static_cast<const void *>(sinT)})
        align |= reinterpret_cast<uintptr_t>(a);
    TC_REQUIRE((align & 15u) == 0, TC_EINVAL, "paged write: alignment (16 bytes)");
    unsigned int *err = devErrorWord();
    TC_REQUIRE(err != nullptr, TC_ECUDA, "no CUDA device");
    PagedWriteParams p{pagedView(c, err), c->k, c->v, c->ks, c->vs, k, v, q, qOut, cosT, sinT, nHeads, tableRows, 0, qHalf};
    const uint32_t rows = nHeads + 2 * c->nKV, lanes = c->hd / 8;
    const bool many = manyRows(static_cast<uint64_t>(c->tokens) * rows, lanes);
    p.unitsPerToken = many ? (rows + kManyRows - 1) / kManyRows : rows;
    uint32_t blocks;
    const int gc = pagedGrid(static_cast<uint64_t>(c->tokens) * p.unitsPerToken, lanes, &blocks);
    if (gc != TC_OK) return gc;
    auto pick = [&](auto one, auto four) { return launchDependent(many ? four : one, dim3(blocks), 256, 0, static_cast<cudaStream_t>(stream), 1, p); };
    if (c->kvI8) {
        if (c->hd == 128) return pick(pagedWriteKernel<128, true, 1>, pagedWriteKernel<128, true, kManyRows>);
        return pick(pagedWriteKernel<256, true, 1>, pagedWriteKernel<256, true, kManyRows>);
    }
    if (c->hd == 64) return pick(pagedWriteKernel<64, false, 1>, pagedWriteKernel<64, false, kManyRows>);
    if (c->hd == 128) return pick(pagedWriteKernel<128, false, 1>, pagedWriteKernel<128, false, kManyRows>);
    return pick(pagedWriteKernel<256, false, 1>, pagedWriteKernel<256, false, kManyRows>);
}

int tc_paged_kv_read(const tc_paged_kv *c, void *kOut, void *vOut, int outHalf, tc_stream stream) {
    using namespace tc;
    const int rc = pagedCheck(c, "paged read");
    if (rc != TC_OK) return rc;
    if (c->tokens == 0) return TC_OK;
    TC_REQUIRE(kOut != nullptr && vOut != nullptr, TC_EINVAL, "paged read: null pointer");
    TC_REQUIRE(((reinterpret_cast<uintptr_t>(kOut) | reinterpret_cast<uintptr_t>(vOut)) & 15u) == 0, TC_EINVAL, "paged read: alignment (16 bytes)");
    unsigned int *err = devErrorWord();
    TC_REQUIRE(err != nullptr, TC_ECUDA, "no CUDA device");
    PagedReadParams p{pagedView(c, err), c->k, c->v, c->ks, c->vs, kOut, vOut, 0};
    p.out32 = ((reinterpret_cast<uintptr_t>(kOut) | reinterpret_cast<uintptr_t>(vOut)) & 31u) == 0;
    const uint32_t rows = 2 * c->nKV, lanes = c->hd / (c->kvI8 ? 16 : 8);
    const bool many = manyRows(static_cast<uint64_t>(c->tokens) * rows, lanes);
    uint32_t blocks = (c->tokens + kReadTokens - 1) / kReadTokens;
    const int gc = many ? TC_OK : pagedGrid(static_cast<uint64_t>(c->tokens) * rows, lanes, &blocks);
    if (gc != TC_OK) return gc;
    auto go = [&](auto kern) { return launchDependent(kern, dim3(blocks), 256, 0, static_cast<cudaStream_t>(stream), 1, p); };
#define TC_PAGED_READ(HD, I8) \
    (many ? (outHalf ? go(pagedReadManyKernel<HD, I8, true>) : go(pagedReadManyKernel<HD, I8, false>)) \
          : (outHalf ? go(pagedReadKernel<HD, I8, true>) : go(pagedReadKernel<HD, I8, false>)))
    if (c->kvI8) return c->hd == 128 ? TC_PAGED_READ(128, true) : TC_PAGED_READ(256, true);
    if (c->hd == 64) return TC_PAGED_READ(64, false);
    return c->hd == 128 ? TC_PAGED_READ(128, false) : TC_PAGED_READ(256, false);
#undef TC_PAGED_READ
}

}  // extern "C"
