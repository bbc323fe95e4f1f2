// paged_attn.cu -- attention over a paged K/V cache: the entry point, which of the kernels takes what, and the launch that joins
// what several blocks had a part in.
//
//   o[t, h] = sum_j p_j V[j] / sum_j p_j,   p_j = exp(q[t, h] . K[j] / sqrt(hd) - m),   j <= pos(t),
//
// in one pass over the rows with a running maximum and sum: paged_steps.cu for few query rows per kv head, paged_tiles.cu (tcgen05, fp16 queries) and
// paged_rows.cu (f32 queries) for many.  A call whose sequences differ launches two of them, each of which leaves the other's sequences
// alone.
#include <algorithm>
#include <cstring>

#include "paged_attn.cuh"

namespace tc {

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
    auto part = [&](uint32_t c) { return parts + (2u * static_cast<size_t>(from + c * j.groups) + (c == 0u ? 1u : 0u)) * slot; };
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

// A sequence of more query rows per kv head than this goes to the call's kernel for many rows: fp16 queries to the tiles of the tensor cores, f32
// ones to the rows kernel where that is faster; what is left, to the steps kernel.  Both sides measured, tokens of 32 (16) sessions behind
// 1000 - 6000 rows.  Tiles against steps, fp16 pages: 21 rows of head_dim 128 53 us against 87, 24 of 256 32 against 50; int8 pages: 21 rows of 128 90 against 70
// and 24 of 256 45 and 44, 35 of 128 92 against 100, 40 of 256 46 against 57.  For f32 see paged_rows.cu.
static uint32_t fewRows(const tc_paged_kv *c, bool half) { return half && c->kvI8 ? 32u : 16u; }
static bool hasRowsForm(const tc_paged_kv *c) { return !c->kvI8 && c->hd < 256; }

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
    if (maxTokens == 0 || maxTokens > most || c->starts == nullptr) maxTokens = most;
    const uintptr_t base = (reinterpret_cast<uintptr_t>(workspace) + 31) & ~uintptr_t(31);
    PagedAttnParams p;
    p.c = pagedView(c, err);
    p.q = q, p.out = out, p.ks = c->ks, p.vs = c->vs;
    p.parts = reinterpret_cast<float *>(base);
    float *const partsB = p.parts + kStepsParts;
    p.joins = reinterpret_cast<PagedJoin *>(partsB + kTilesParts);
    PagedJoin *const joinsB = p.joins + 3 * kPagedSMs;
    p.nHeads = nHeads, p.group = nHeads / c->nKV;
    p.box = 64;
    while (c->pageRows % p.box != 0) p.box /= 2;
    p.tileTokens = kPagedTile / p.group;
    p.out32 = (reinterpret_cast<uintptr_t>(out) & 31u) == 0;
    p.scaleLog2 = invSqrt * kLog2e;
    p.half = half != 0;
    p.zero = 0;
    const uint32_t rows = maxTokens * p.group;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uint32_t few = fewRows(c, half != 0);
    const bool many = rows > few && (half || hasRowsForm(c));
    uint32_t blocksA = 0, blocksB = 0;
    // Over fp16 pages the form for many rows takes the call's short sequences along: single tokens stream at 4.9 TB/s there, and a
    // launch without work is 4 us.  Over int8 pages its rate for them is a quarter of the steps kernel's.
    if (!many || (c->kvI8 && c->starts != nullptr && c->batch > 1)) {
        p.minRows = 1, p.maxRows = many ? few : 0xffffffffu;
        const int ra = pagedAttnSteps(c, p, many ? few : rows, st, &blocksA);
        if (ra != TC_OK) return ra;
    }
    if (many) {
        PagedAttnParams b = p;
        b.parts = partsB, b.joins = joinsB;
        b.minRows = blocksA != 0u ? few + 1 : 1, b.maxRows = 0xffffffffu;
        const int rb = half ? pagedAttnTiles(c, b, st, &blocksB) : pagedAttnRows(c, b, st, &blocksB);
        if (rb != TC_OK) return rb;
    }
    const dim3 grid(blocksA + blocksB, 8);  // (an empty block costs: 16 and 32 along y take 3 and 10 us more for a step, and win nothing for prompts)
    auto merge = c->hd == 64 ? pagedMergeKernel<64> : c->hd == 128 ? pagedMergeKernel<128> : pagedMergeKernel<256>;
    return launchDependent(merge, grid, 256, 0, st, 1, p, static_cast<const float *>(partsB), static_cast<const PagedJoin *>(joinsB), blocksA);
}

}  // extern "C"
