// What the kernels of attention over a paged cache share: their parameters, the parts of the work that a CTA takes, and what it leaves for the kernel that joins them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace gpuk {
namespace {

constexpr int kRows = 128;                       // of a tile
constexpr int kKeys = 64;                        // of a block
constexpr int kCtasPerSm = 2;
constexpr int kTileCost = 4 * kKeys;             // what a tile costs beside its keys, in keys: its queries, its outputs, the first scores
constexpr int kGrain = 2 * kKeys;                // no tile is cut nearer than that to its end, or than kFront to its beginning
constexpr int kFront = 3 * kKeys;
constexpr int kPerCta = 256;                     // keys for which a call takes another CTA
constexpr int kSmall = 6;                        // tiles of a sixth of a CTA's share are not cut
constexpr float kLowest = -3.4e38f;              // a maximum before any key ...
constexpr float kSeen = -3.3e38f;                // ... and where all scores are -infinity: finite both, and below any score behind them

// Blocks [first, first + blocks) of the keys of a tile: what a CTA does at a time.
struct alignas(16) Segment {
    int request, start, n, ctx;                  // its first row in q, new and cached tokens
    int tok0, kvh;                               // the tile's first token
    int first, blocks;                           // no blocks: the end
    int slot;                                    // of the partial results; -1: the whole tile
};
struct Request {
    int start, n, ctx, tiles;
    bool over;      // more tokens than the table's row holds: its tiles are not cut
};
// Where a CTA begins: weight `pos` of a tile; and its borders on the line of all tiles.
struct Start {
    Request r;
    int request, kvh, tile, ctas;
    int64_t pos, x[2];
};

struct PagedAttentionParams {
    const int32_t *tables, *lens, *starts, *masks;
    const void *q, *k, *v;
    void *out;
    int64_t q_token, q_head, table_stride, page_stride, head_stride, row_stride, num_pages;
    int64_t out_token, out_head;
    int batch, tokens, kv_heads, group, tile_tokens, words;
    uint32_t tile_inverse;                       // 2^32 / tile_tokens, rounded up
    int width, page_shift;                       // of a row of the table, and log2 of a page's tokens
    int row_groups;                              // of 32, of a tile
    int may_split, out_sectors;                  // rows of the outputs lie on borders of 32 bytes
    float scale_log2;
    int *status;
    // of the partial results, for `ctas` CTAs: see Joint, [2 * ctas][HD / 4][128][4] outputs (a warp's rows side by side), [2 * ctas][2][128] maxima and sums
    struct Joint *joints;
    float *partial, *stats;
};
// What the second kernel learns from each CTA of the first.
struct alignas(16) Joint {
    Segment open;                                // a tile that begins in the CTA and goes on behind it (slot -1: none)
    int head;                                    // the CTA takes: 0 nothing, 1 a part of such a tile and nothing else, 2 the last part of one, 3 begins with a tile
    int ctas;                                    // that take part
};

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint64_t policy_once() {      // what is read leaves L2 first
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
template <typename T>
struct Half;
template <>
struct Half<__nv_bfloat16> {
    static constexpr int kFormat = 1;
    static constexpr uint32_t kExponent = 0x7f807f80u;
    static constexpr float kBias = 0.f, kLag = 8.f;
    __device__ static uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    __device__ static float round(float x) { return __uint_as_float(pack(0.f, x)); }      // the upper half, and nothing below
};
template <>
struct Half<__half> {
    static constexpr int kFormat = 0;
    static constexpr uint32_t kExponent = 0x7c007c00u;
    static constexpr float kBias = 8.f, kLag = 7.f;      // 2^15 at most
    __device__ static uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    __device__ static float round(float x) { return __half2float(__float2half_rn(x)); }
};
// ---- which parts of which tiles a CTA takes ---------------------------------------------------------
// Tiles lie one after another, by request, kv head and token, each as long as the keys that it sees and kTileCost more.  A CTA takes an equal share of that line; where a border comes
// near an end of a tile it goes to that end.
__device__ __forceinline__ int64_t room_of(const PagedAttentionParams &p) { return static_cast<int64_t>(p.width) << p.page_shift; }
__device__ __forceinline__ Request request_of(const PagedAttentionParams &p, int i) {
    Request r;
    r.start = min(max(p.starts[i], 0), p.tokens);
    r.n = min(max(p.starts[i + 1], r.start), p.tokens) - r.start;
    r.ctx = static_cast<int>(min(static_cast<int64_t>(max(p.lens[i], 0)), room_of(p)));
    r.tiles = static_cast<int>(p.tile_tokens == 1 ? r.n : __umulhi(r.n + p.tile_tokens - 1, p.tile_inverse));      // exact below 2^32 / tile_tokens
    r.over = static_cast<int64_t>(r.ctx) + r.n > room_of(p);
    return r;
}
// Keys that some row of a tile sees.
__device__ __forceinline__ int64_t keys_of(const PagedAttentionParams &p, const Request &r, int tile) {
    const int64_t most = static_cast<int64_t>(r.ctx) + (p.masks ? static_cast<int64_t>(r.n) : min(static_cast<int64_t>(r.n), static_cast<int64_t>(tile + 1) * p.tile_tokens));
    return min(most, room_of(p));
}
// The weight of a tile, and of those in front of one.
__device__ __forceinline__ int64_t weight_of(const PagedAttentionParams &p, const Request &r, int tile) { return kTileCost + (r.over ? room_of(p) : keys_of(p, r, tile)); }
__device__ __forceinline__ int64_t weight_before(const PagedAttentionParams &p, const Request &r, int tile) {
    if (r.tiles == 0) return 0;
    if (p.masks || r.over) return tile * (kTileCost + min(static_cast<int64_t>(r.ctx) + r.n, room_of(p)));
    const int64_t whole = min(tile, r.tiles - 1), w = whole * (kTileCost + r.ctx) + p.tile_tokens * (whole * (whole + 1) / 2);
    return tile < r.tiles || tile == 0 ? w : w + kTileCost + r.ctx + r.n;
}
// Sums over the lanes up to this one.
__device__ __forceinline__ int64_t warp_scan(int64_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}

// One warp for each of a CTA's two borders; lane l looks after a run of the requests.  Quotients are estimated in fp32 and put right, which is faster than dividing 64 bits.
__device__ void find_border(const PagedAttentionParams &p, Start *out, int side) {
    const int lane = threadIdx.x & 31, per = (p.batch + 31) / 32, lo = min(lane * per, p.batch), hi = min(lo + per, p.batch);
    int64_t weight = 0, tiles = 0, most = 0;
    Request r = {};
    for (int i = lo; i < hi; ++i) {
        r = request_of(p, i);
        if (r.tiles) most = max(most, weight_of(p, r, r.tiles - 1));
        weight += weight_before(p, r, r.tiles) * p.kv_heads, tiles += static_cast<int64_t>(r.tiles) * p.kv_heads;
    }
    const int64_t upto = warp_scan(weight, lane), all = __shfl_sync(0xffffffffu, upto, 31), before = upto - weight;
    // enough borders for each tile to have a CTA of its own where there are few
    const int few = __reduce_add_sync(0xffffffffu, static_cast<int>(min(tiles, static_cast<int64_t>(1 << 20))));
    const int ctas = static_cast<int>(max(min(static_cast<int64_t>(gridDim.x), 2 * few + all / kPerCta), static_cast<int64_t>(1)));
    const int border = static_cast<int>(blockIdx.x) + side;
    const int64_t share = static_cast<int64_t>(static_cast<float>(all) * (1.00001f / ctas)) + 1;      // the last CTA's is a little shorter
    const int64_t raw = min(all, border * share);
    // Tiles are left whole where each has a CTA and none is much more than a share, and where the largest is a kSmall-th of a share or less: what parts cost is more than what a more even end gains.
    // 64 / 8 heads, with and without cuts: single tokens of 32 x 2049 keys 51.5 and 48.3 us, of 256 x 2049 372 and 356, 64 trees of 32 behind 2048 223 and 217, 8 prompts of 2048 behind 2048 1586 and 1599.
    // At a third of a share a prompt of 4096 takes 255 with cuts and 280 without.
    const int64_t largest = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(min(most, static_cast<int64_t>(0x7fffffff))));
    const bool cut = p.may_split && !(few <= static_cast<int>(gridDim.x) && 2 * largest <= 3 * share) && kSmall * largest > share;
    if (lane == 0) out->x[side] = all, out->ctas = ctas;      // the line's end, unless a lane below has the border
    __syncwarp();
    if (raw >= all || raw < before || raw >= upto) return;
    int64_t base = before;
    for (int i = lo; i < hi; ++i) {
        if (per > 1) r = request_of(p, i);
        const int64_t head = weight_before(p, r, r.tiles), here = head * p.kv_heads;
        if (raw >= base + here) {
            base += here;
            continue;
        }
        int64_t at = raw - base, first = 0;
        int kvh = min(p.kv_heads - 1, static_cast<int>(__fdividef(static_cast<float>(at), static_cast<float>(head)))), tile = 0;
        while (kvh > 0 && kvh * head > at) --kvh;
        while (kvh + 1 < p.kv_heads && (kvh + 1) * head <= at) ++kvh;
        at -= kvh * head;
        if (r.tiles > 1) {      // weight_before(tile) <= at < weight_before(tile + 1): a line, or a parabola with half a tile's tokens to the square
            const float slope = kTileCost + r.ctx + (p.masks || r.over ? static_cast<float>(r.n) : 0.5f * p.tile_tokens), bend = p.masks || r.over ? 0.f : 0.5f * p.tile_tokens;
            tile = min(r.tiles - 1, static_cast<int>(bend == 0.f ? static_cast<float>(at) / slope : (sqrtf(slope * slope + 4.f * bend * at) - slope) / (2.f * bend)));
            while (tile > 0 && weight_before(p, r, tile) > at) --tile;
            while (tile + 1 < r.tiles && weight_before(p, r, tile + 1) <= at) ++tile;
            first = weight_before(p, r, tile);
        }
        const int64_t size = weight_of(p, r, tile);
        int64_t pos = at - first;
        if (!cut || r.over || pos < kTileCost + kFront) pos = 0;
        else if (size - pos < kGrain) pos = size;
        else pos = pos / kKeys * kKeys;      // the borders of blocks, behind the tile's cost
        out->x[side] = base + kvh * head + first + pos;
        if (side == 0) out->r = r, out->request = i, out->kvh = kvh, out->tile = tile, out->pos = pos;
        return;
    }
}

// The segments of a CTA one after another.
struct Walk {
    Request r;
    int request, kvh, tile, index;
    int64_t pos, left;
    __device__ explicit Walk(const Start &s) : r(s.r), request(s.request), kvh(s.kvh), tile(s.tile), index(0), pos(s.pos), left(s.x[1] - s.x[0]) {}
    __device__ bool next(const PagedAttentionParams &p, Segment *out, bool *begins, bool *ends) {
        if (left <= 0) return false;
        int64_t size = weight_of(p, r, tile);
        while (pos >= size) {      // at a tile's end, to the next
            pos = 0;
            if (++tile >= r.tiles) {
                tile = 0;
                if (++kvh >= p.kv_heads) {
                    kvh = 0;
                    do {
                        if (++request >= p.batch) return false;      // cannot be: the weights say that there is more
                        r = request_of(p, request);
                    } while (r.tiles == 0);
                }
            }
            size = weight_of(p, r, tile);
        }
        const int64_t take = min(size - pos, left), end = pos + take;
        const int all = static_cast<int>((keys_of(p, r, tile) + kKeys - 1) / kKeys);
        auto block_at = [&](int64_t w) { return w <= kTileCost ? 0 : static_cast<int>(min((w - kTileCost + kKeys - 1) / kKeys, static_cast<int64_t>(all))); };
        *begins = pos == 0, *ends = end == size;
        const int first = *begins ? 0 : block_at(pos), last = *ends ? all : block_at(end);
        *out = {request, r.start, r.n, r.ctx, tile * p.tile_tokens, kvh, first, last - first, -1};
        if (!*begins || !*ends) out->slot = 2 * static_cast<int>(blockIdx.x) + (*begins && index > 0);
        pos = end, left -= take, ++index;
        return true;
    }
};

}  // namespace

// The kernel for single tokens (paged_decode.cu), its shared memory, and how many query heads a kv head may have for it.
constexpr int kDecodeThreads = 128, kDecodeGroup = 16;
const void *paged_decode_of(int dtype, int head_dim, int *smem);

}  // namespace gpuk
