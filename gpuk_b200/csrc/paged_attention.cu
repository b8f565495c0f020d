// Attention of a ragged batch of new tokens over pages of a KV cache: single tokens, trees of drafted tokens and prompts, heads of 64 and 128, bf16 and fp16.
//
// A request has `ctx` cached tokens and `n` new ones, whose keys and values are in its pages already.  A new token sees the cached ones and, of the new ones, those up to
// itself or those that its bits in `masks` name (in a tree: its ancestors and itself).
//
// One kernel for all of them.  The rows of a tile are pairs of a token and a query head of one kv head's group, tokens outermost: 128 rows are 128 / group tokens, so that a page
// is read once for a tree of that many nodes, and up to 128 rows cost the tensor pipe less than the page costs HBM (128 operations a byte; the pipe has 250 for each that
// HBM delivers).  Single tokens leave most rows idle, and warps without a row only keep the barriers going.
//
//   * scores of 64 keys go to one of two buffers in tensor memory, so that the next block's are multiplied while a thread per row works on this one's; the probabilities
//     go back into the same columns, from where they are the first operand of O += P V.  256 columns and 113 KiB a CTA: two CTAs an SM hide each other's waits.
//   * pages come by TMA through a ring of 8 or 16 KiB slots; a block of 64 keys is one box of a large page or several small ones, whose numbers the copying warp
//     reads from the table a block ahead.  Numbers outside the pool and pages behind the last key read as zeros.
//   * the keys of a tile are cut into parts where the tiles alone do not fill the GPU.  Each CTA works that out from the lengths on the device, the same way, so the host need not
//     know them; parts leave sums, maxima and outputs in fp32, and a second kernel joins them in order.  The same inputs give the same bits.
//   * only blocks that some row sees in part are masked.  There a value that is no finite number would spoil the rows that do not see it (0 * inf), so it is taken out of shared memory
//     before the product, and the rows that do see it add it at the end.
//
// fp32 scores, maxima, sums and outputs.  Probabilities are rounded to the operands' type for the second product; in fp16 they are held times 2^10, so that small
// ones do not fall under its smallest numbers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/gpuk_b200.h"
#include "launch.cuh"
#include "linear.cuh"
#include "tensor_core.cuh"

namespace gpuk {
namespace {

constexpr int kRows = 128;                       // of a tile
constexpr int kKeys = 64;                        // of a block
constexpr int kThreads = kRows + 64;             // a thread per row, a warp that multiplies, one that copies
constexpr int kSpanBytes = kKeys * 128;          // 64 rows of one swizzle span (64 values)
constexpr int kQSpanBytes = kRows * 128;
constexpr int kColumns = 256;                    // two score buffers of 64, up to 128 of outputs
constexpr int kOut = 2 * kKeys;                  // first column of the outputs
constexpr int kMaskedBlocks = 8;                 // that a tile can have
constexpr int kMinPart = 4;                      // blocks of a part
constexpr int kCtasPerSm = 2;

constexpr float kLowest = -3.4e38f;              // a maximum before any key ...
constexpr float kSeen = -3.3e38f;                // ... and where all scores are -infinity: finite both, and below any score behind them

template <int HD>
constexpr int kSlotsOf = HD == 128 ? 5 : 10;

struct alignas(16) Unit {                        // what a CTA of the first kernel does, or a joined tile
    int request, start, n, ctx;                  // its first row in q, new and cached tokens
    int tile, kvh;
    int part, parts, first, last;                // blocks [first, last)
    int slot;                                    // of the partial results, where there are parts
    int found;
};

// A wait tells a phase of a barrier from the one before and the one behind it, not from the next but one.  Scores and products have two barriers in turn, since a row's thread may
// come to block j when product j - 2 is the last that is known to be complete, and to its end when the last product is.
template <int HD>
struct Smem {
    alignas(1024) unsigned char q[HD / 64 * kQSpanBytes];
    alignas(1024) unsigned char ring[kSlotsOf<HD>][HD / 64 * kSpanBytes];
    uint64_t q_full, full[kSlotsOf<HD>], empty[kSlotsOf<HD>], s_full[2], p_full[2], o_done[2], drained;
    Unit unit;
    uint32_t tmem;
    uint32_t poison[kMaskedBlocks * 2];          // keys of the masked blocks with a value that is no finite number
};

struct PagedAttentionParams {
    const int32_t *tables, *lens, *starts, *masks;
    const void *v;
    void *out;
    int64_t table_stride, page_stride, head_stride, row_stride, num_pages;
    int64_t out_token, out_head;
    int batch, tokens, kv_heads, group, tile_tokens, words;
    int width, page_shift;                       // of a row of the table, and log2 of a page's tokens
    int target;                                  // CTAs that run at once
    int may_split;
    float scale_log2;
    int *status;
    int *units;                                  // count, then a Unit of each tile that is joined
    float *partial;                              // [slot][128][HD], [slot][2][128]: outputs, then maxima and sums
    int max_slots;
};

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
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
};
// Whether one of the two halves is an infinity or NaN: all bits of its exponent are set.
__device__ __forceinline__ bool any_not_finite(uint32_t w, uint32_t exponent) {
    const uint32_t x = (w & exponent) ^ exponent;      // a zero half
    return ((x - 0x00010001u) & ~x & 0x80008000u) != 0;
}

// ---- which part of which tile a CTA takes ---------------------------------------------------------
struct Request {
    int start, n, ctx, tiles, blocks;
};
__device__ __forceinline__ Request request_of(const PagedAttentionParams &p, int i) {
    Request r;
    r.start = min(max(p.starts[i], 0), p.tokens);
    r.n = min(max(p.starts[i + 1], r.start), p.tokens) - r.start;
    const int64_t room = static_cast<int64_t>(p.width) << p.page_shift;      // what the row of the table can hold
    r.ctx = static_cast<int>(min(static_cast<int64_t>(max(p.lens[i], 0)), room));
    const int64_t end = min(static_cast<int64_t>(r.ctx) + r.n, room);
    r.tiles = (r.n + p.tile_tokens - 1) / p.tile_tokens;
    r.blocks = static_cast<int>((end + kKeys - 1) / kKeys);
    return r;
}
__device__ __forceinline__ int64_t warp_sum(int64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ int64_t warp_before(int64_t v, int lane) {
    int64_t s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
    }
    return s - v;
}

// One warp.  Lane l looks after a run of the requests; parts of `cut` blocks, the fewest with which all parts run at once.
__device__ void find_unit(const PagedAttentionParams &p, Unit *u, int item) {
    const int lane = threadIdx.x & 31, per = (p.batch + 31) / 32, lo = min(lane * per, p.batch), hi = min(lo + per, p.batch);
    const int kvh = item % p.kv_heads, rest = item / p.kv_heads;
    int cut = 1 << 30;
    if (p.may_split) {
        int64_t work = 0;
        int most = 0;
        for (int i = lo; i < hi; ++i) {
            const Request r = request_of(p, i);
            work += static_cast<int64_t>(r.tiles) * r.blocks;
            if (r.tiles) most = max(most, r.blocks);
        }
        work = warp_sum(work) * p.kv_heads;
        most = __reduce_max_sync(0xffffffffu, most);
        cut = static_cast<int>(max(static_cast<int64_t>(kMinPart), (work + p.target - 1) / p.target));
        for (int tries = 0; tries < 6 && cut < most; ++tries) {
            int64_t items = 0;
            for (int i = lo; i < hi; ++i) {
                const Request r = request_of(p, i);
                items += static_cast<int64_t>(r.tiles) * ((r.blocks + cut - 1) / cut);
            }
            if (warp_sum(items) * p.kv_heads <= p.target) break;
            cut += cut / 4 + 1;
        }
    }
    int64_t items = 0, joined = 0, tiles = 0;      // of this lane's requests: CTAs per kv head, those of tiles in parts, such tiles
    for (int i = lo; i < hi; ++i) {
        const Request r = request_of(p, i);
        const int parts = max(1, (r.blocks + cut - 1) / cut);
        items += static_cast<int64_t>(r.tiles) * parts;
        if (parts > 1) joined += static_cast<int64_t>(r.tiles) * parts, tiles += r.tiles;
    }
    int64_t before = warp_before(items, lane), joined_before = warp_before(joined, lane), tiles_before = warp_before(tiles, lane);
    if (p.may_split && item == 0) {
        const int64_t all = warp_sum(tiles) * p.kv_heads;
        if (lane == 0) p.units[0] = static_cast<int>(all);
    }
    const bool mine = rest >= before && rest < before + items;
    if (lane == 0) u->found = 0;
    __syncwarp();
    if (!mine) return;
    for (int i = lo; i < hi; ++i) {
        const Request r = request_of(p, i);
        const int parts = max(1, (r.blocks + cut - 1) / cut);
        const int64_t here = static_cast<int64_t>(r.tiles) * parts;
        if (rest < before + here) {
            const int at = static_cast<int>(rest - before);
            Unit v;
            v.request = i, v.start = r.start, v.n = r.n, v.ctx = r.ctx, v.kvh = kvh;
            v.tile = r.tiles - 1 - at / parts;      // the tiles that see most come first
            v.part = at % parts, v.parts = parts;
            // keys that some row of the tile sees
            const int64_t end = min(static_cast<int64_t>(r.ctx) + (p.masks ? r.n : min(r.n, (v.tile + 1) * p.tile_tokens)), static_cast<int64_t>(p.width) << p.page_shift);
            const int blocks = static_cast<int>((end + kKeys - 1) / kKeys);
            v.first = static_cast<int>(min(static_cast<int64_t>(v.part) * cut, static_cast<int64_t>(blocks)));
            v.last = static_cast<int>(min(static_cast<int64_t>(v.first) + cut, static_cast<int64_t>(blocks)));
            v.slot = 0;
            v.found = 1;
            if (parts > 1) {
                const int64_t tile = (tiles_before + v.tile) * p.kv_heads + kvh;
                const int64_t slot = joined_before * p.kv_heads + (static_cast<int64_t>(v.tile) * p.kv_heads + kvh) * parts + v.part;
                if (slot - v.part + parts > p.max_slots || tile >= p.target) {      // cannot be: the parts of joined tiles are at most twice the target
                    *p.status = 1;
                    v.found = 0;
                }
                v.slot = static_cast<int>(slot);
                if (v.part == 0 && v.found) reinterpret_cast<Unit *>(p.units + 4)[tile] = v;
            }
            *u = v;
            return;
        }
        before += here;
        if (parts > 1) joined_before += here, tiles_before += r.tiles;
    }
}

// Bits [at, at + 64) of a row of mask words, zeros outside.
__device__ __forceinline__ uint64_t mask_bits(const int32_t *row, int words, int at) {
    const int w = at >> 5, s = at & 31;
    const uint32_t a = w < words ? row[w] : 0, b = w + 1 < words ? row[w + 1] : 0, c = w + 2 < words ? row[w + 2] : 0;
    return static_cast<uint64_t>(__funnelshift_r(a, b, s)) | static_cast<uint64_t>(__funnelshift_r(b, c, s)) << 32;
}
// Which keys of block `base` a row sees: cached ones, and of the new ones those up to token `tok` or those in its mask.
__device__ __forceinline__ uint64_t seen_of(const PagedAttentionParams &p, const Unit &u, int tok, int base) {
    const int old = min(max(u.ctx - base, 0), kKeys);      // keys of the block in front of the new ones
    const uint64_t cached = old == kKeys ? ~0ull : (1ull << old) - 1;
    if (old == kKeys) return cached;
    const int rel = base + old - u.ctx;
    const int most = min(p.masks ? u.n - rel : tok + 1 - rel, kKeys - old);
    uint64_t fresh = most <= 0 ? 0 : most == 64 ? ~0ull : (1ull << most) - 1;
    if (p.masks && fresh) fresh &= mask_bits(p.masks + static_cast<int64_t>(u.start + tok) * p.words, p.words, rel);
    return cached | fresh << old;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) paged_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                                                                               const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PagedAttentionParams p) {
    constexpr int kSpans = HD / 64, kSlots = kSlotsOf<HD>, kBlockBytes = kSpans * kSpanBytes;
    extern __shared__ __align__(1024) unsigned char dyn[];
    Smem<HD> &sm = *reinterpret_cast<Smem<HD> *>(dyn);
    const int tid = threadIdx.x, warp = tid >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 0) find_unit(p, &sm.unit, blockIdx.x);
    if (tid == kRows) {
        mbar_init(&sm.q_full, 1), mbar_init(&sm.drained, 1);
        for (int s = 0; s < kSlots; ++s) mbar_init(&sm.full[s], 1), mbar_init(&sm.empty[s], 1);
        for (int b = 0; b < 2; ++b) mbar_init(&sm.s_full[b], 1), mbar_init(&sm.p_full[b], kRows), mbar_init(&sm.o_done[b], 1);
        mbar_init_fence();
    }
    if (tid >= kRows + 32 && tid < kRows + 32 + kMaskedBlocks * 2) sm.poison[tid - kRows - 32] = 0;
    __syncthreads();
    const Unit u = sm.unit;
    if (!u.found) return;
    if (warp == kRows / 32) tmem_alloc<kColumns>(&sm.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // behind the allocation: no CTA that follows takes columns one of this grid waits for
    const uint32_t tm = sm.tmem;
    const int blocks = u.last - u.first, tok0 = u.tile * p.tile_tokens;
    // keys from here on are not seen by every row, or are no keys
    const int64_t limit = p.masks ? u.ctx : static_cast<int64_t>(u.ctx) + tok0 + 1;
    const int first_masked = max(u.first, static_cast<int>(limit / kKeys));
    bool ok = (smem_addr(dyn) & 1023u) == 0;

    if (warp == kRows / 32 + 1) {      // copies: Q, then K of the first block, and K of the next block before V of each
        const int lane = tid & 31;
        if (ok && blocks > 0) {
            const uint64_t once = policy_evict_first();
            if (lane == 0) {
                mbar_expect_bytes(&sm.q_full, kSpans * p.tile_tokens * p.group * 128);
                for (int h = 0; h < kSpans; ++h) tma_load_3d(smem_addr(sm.q) + h * kQSpanBytes, &qmap, h * 64, u.kvh * p.group, u.start + tok0, &sm.q_full);
            }
            const int rows = min(1 << p.page_shift, kKeys), boxes = kKeys / rows;
            const int32_t *table = p.tables + u.request * p.table_stride;
            // the page of this lane's box in block j; one outside the pool, which reads as zeros, where there is none
            auto page_of = [&](int j) {
                const int64_t key = static_cast<int64_t>(u.first + j) * kKeys + lane * rows;
                const int64_t end = static_cast<int64_t>(u.ctx) + u.n;
                return lane < boxes && j < blocks && key < end && (key >> p.page_shift) < p.width ? table[key >> p.page_shift] : -1;
            };
            int page_k = page_of(0), page_next = page_of(1), page_v = page_k;
            int filled = 0;
            auto load = [&](const CUtensorMap *map, int j, int page) {
                const int s = filled % kSlots;
                if (!mbar_wait(&sm.empty[s], ((filled / kSlots) & 1) ^ 1)) return false;
                if (lane == 0) mbar_expect_bytes(&sm.full[s], kBlockBytes);
                __syncwarp();
                if (lane < boxes) {
                    const int inside = (u.first + j) * kKeys & ((1 << p.page_shift) - 1);
                    for (int h = 0; h < kSpans; ++h)
                        tma_load_4d(smem_addr(sm.ring[s]) + h * kSpanBytes + lane * rows * 128, map, h * 64, rows == kKeys ? inside : 0, u.kvh, page, &sm.full[s], once);
                }
                ++filled;
                return true;
            };
            ok = load(&kmap, 0, page_k);
            for (int j = 0; ok && j < blocks; ++j) {
                page_v = page_k, page_k = page_next, page_next = page_of(j + 2);
                if (j + 1 < blocks) ok = load(&kmap, j + 1, page_k);
                if (ok) ok = load(&vmap, j, page_v);
            }
            // nobody leaves with copies in flight
            ok = mbar_wait(&sm.q_full, 0) && ok;
            for (int i = max(0, filled - kSlots); i < filled; ++i) ok = mbar_wait(&sm.full[i % kSlots], (i / kSlots) & 1) && ok;
        }
    } else if (warp == kRows / 32) {   // multiplications
        if ((tid & 31) == 0 && ok && blocks > 0) {
            constexpr uint32_t s_desc = mma_desc(Half<T>::kFormat, Half<T>::kFormat, kRows, kKeys), o_desc = mma_desc(Half<T>::kFormat, Half<T>::kFormat, kRows, HD, true);
            const int loads = 2 * blocks;
            auto k_at = [&](int j) { return j == 0 ? 0 : 2 * j - 1; };
            auto v_at = [&](int j) { return j + 1 < blocks ? 2 * j + 2 : loads - 1; };
            auto slot = [&](int i) { return smem_addr(sm.ring[i % kSlots]); };
            auto wait_slot = [&](int i) { return mbar_wait(&sm.full[i % kSlots], (i / kSlots) & 1); };
            // only a slot that the copies wait for: nothing may arrive in shared memory behind the CTA's end
            auto release = [&](int i) {
                if (i + kSlots < loads) tc_commit(&sm.empty[i % kSlots]);
            };
            auto scores = [&](int j) {
                const uint32_t q = smem_addr(sm.q), k = slot(k_at(j));
#pragma unroll
                for (int d = 0; d < HD / 16; ++d)
                    tc_mma_f16(tm + (j & 1) * kKeys, kmajor_desc<128>(q + (d / 4) * kQSpanBytes + (d % 4) * 32), kmajor_desc<128>(k + (d / 4) * kSpanBytes + (d % 4) * 32), s_desc,
                               d > 0);
                tc_commit(&sm.s_full[j & 1]);
                release(k_at(j));
            };
            ok = mbar_wait(&sm.q_full, 0) && wait_slot(0);
            tc_fence_after();
            if (ok) scores(0);
            for (int j = 0; ok && j < blocks; ++j) {
                if (j + 1 < blocks) {
                    ok = wait_slot(k_at(j + 1));
                    tc_fence_after();
                    if (!ok) break;
                    scores(j + 1);      // into the buffer of P(j - 1), whose product is in front of it
                }
                ok = wait_slot(v_at(j)) && mbar_wait(&sm.p_full[j & 1], (j >> 1) & 1);
                tc_fence_after();
                if (!ok) break;
                const uint32_t v = slot(v_at(j));
#pragma unroll
                for (int k = 0; k < kKeys / 16; ++k)
                    tc_mma_f16_ts(tm + kOut, tm + (j & 1) * kKeys + k * 8, mnmajor_desc(v + k * 16 * 128, kSpanBytes), o_desc, j > 0 || k > 0);
                tc_commit(&sm.o_done[j & 1]);
                release(v_at(j));
            }
            if (!ok) {      // a wait gave up: the row threads do not wait for what was issued, and the tensor memory is about to be freed
                tc_commit(&sm.drained);
                mbar_wait(&sm.drained, 0);
            }
        }
    } else {                           // a row's thread
        const int tok = tok0 + tid / p.group, head = u.kvh * p.group + tid % p.group;
        const bool valid = tid < p.tile_tokens * p.group && tok < u.n;
        const bool busy = __any_sync(0xffffffffu, valid);
        const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16, o_at = tm + lanes + kOut;
        float m = kLowest, l = 0.f;
        for (int j = 0; j < blocks && ok; ++j) {
            const int block = u.first + j;
            if (block >= first_masked) {
                // values that are none, or that a row may not see and that are no finite numbers, become zeros
                const int i = j + 1 < blocks ? 2 * j + 2 : 2 * blocks - 1;
                ok = mbar_wait(&sm.full[i % kSlots], (i / kSlots) & 1) && ok;
                uint4 *v = reinterpret_cast<uint4 *>(sm.ring[i % kSlots]);
                const int64_t keys = min(static_cast<int64_t>(u.ctx) + u.n, static_cast<int64_t>(p.width) << p.page_shift) - static_cast<int64_t>(block) * kKeys;
                bool changed = false;
#pragma unroll
                for (int c = 0; c < kBlockBytes / 16 / kRows; ++c) {
                    const int at = c * kRows + tid, key = (at & (kSpanBytes / 16 - 1)) / 8;
                    if (key >= keys) {
                        v[at] = make_uint4(0, 0, 0, 0);
                        changed = true;
                        continue;
                    }
                    uint4 x = v[at];
                    uint32_t w[4] = {x.x, x.y, x.z, x.w};
                    constexpr uint32_t e = Half<T>::kExponent;
                    if (any_not_finite(w[0], e) || any_not_finite(w[1], e) || any_not_finite(w[2], e) || any_not_finite(w[3], e)) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            if ((w[k] & e & 0xffffu) == (e & 0xffffu)) w[k] &= 0xffff0000u;
                            if ((w[k] & e & 0xffff0000u) == (e & 0xffff0000u)) w[k] &= 0xffffu;
                        }
                        v[at] = make_uint4(w[0], w[1], w[2], w[3]);
                        const int bit = (block - first_masked) * kKeys + key;
                        if (bit < kMaskedBlocks * 64) atomicOr(&sm.poison[bit >> 5], 1u << (bit & 31));
                        changed = true;
                    }
                }
                if (changed) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            ok = mbar_wait(&sm.s_full[j & 1], (j >> 1) & 1) && ok;      // idle warps too: nobody arrives twice in a phase
            __syncwarp();
            if (busy) {
                tc_fence_after();
                const uint32_t s_at = tm + lanes + (j & 1) * kKeys;
                uint32_t s[2][32];
                tmem_ld32(s[0], s_at);
                tmem_ld32(s[1], s_at + 32);
                tmem_wait_ld();
                bool some = true;
                if (block >= first_masked) {
                    const uint64_t seen = valid ? seen_of(p, u, tok, block * kKeys) : ~0ull;
                    some = seen != 0;
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (!(seen >> i & 1)) s[i / 32][i % 32] = 0xff800000u;
                }
                float mx[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    mx[c] = __uint_as_float(s[c / 2][(c & 1) * 16]);
#pragma unroll
                    for (int i = 1; i < 16; ++i) mx[c] = fmaxf(mx[c], __uint_as_float(s[c / 2][(c & 1) * 16 + i]));
                }
                float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
                if (some) top = fmaxf(top, kSeen);
                const bool grown = top > m + Half<T>::kLag;
                if (j == 0) {
                    m = fmaxf(top, kLowest);
                } else if (__any_sync(0xffffffffu, grown)) {
                    ok = mbar_wait(&sm.o_done[(j - 1) & 1], ((j - 1) >> 1) & 1) && ok;
                    __syncwarp();
                    tc_fence_after();
                    const float f = grown ? exp2_fast(m - top) : 1.f;
                    if (grown) m = top, l *= f;
#pragma unroll
                    for (int c = 0; c < HD; c += 16) {
                        float o[16];
                        tmem_ld16(o, o_at + c);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] *= f;
                        tmem_st16(o_at + c, o);
                    }
                }
                const float shift = Half<T>::kBias - m;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                uint32_t pk[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float a = exp2_fast(fmaf(__uint_as_float(s[i / 16][2 * (i % 16)]), p.scale_log2, shift));
                    const float c = exp2_fast(fmaf(__uint_as_float(s[i / 16][2 * (i % 16) + 1]), p.scale_log2, shift));
                    sum[i & 1] += a, sum[2 + (i & 1)] += c;
                    pk[i] = Half<T>::pack(a, c);
                }
                tmem_st32(s_at, pk);
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_st();
                tc_fence_before();
            }
            mbar_arrive(&sm.p_full[j & 1]);
        }
        if (blocks > 0 && ok) {
            ok = mbar_wait(&sm.o_done[(blocks - 1) & 1], ((blocks - 1) >> 1) & 1) && ok;
            tc_fence_after();
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (busy) {
            uint32_t poison = 0;
            for (int i = 0; i < kMaskedBlocks * 2; ++i) poison |= sm.poison[i];
            const bool whole = u.parts == 1;
            // a row that saw no key is zeros; one whose scores are all -infinity is NaN, as a softmax has it
            const float r = l == 0.f ? (m > kLowest ? __int_as_float(0x7fffffff) : 0.f) : 1.f / l;
            T *out = static_cast<T *>(p.out) + static_cast<int64_t>(u.start + tok) * p.out_token + head * p.out_head;
            float *part = p.partial + (static_cast<int64_t>(u.slot) * kRows + tid) * HD;
            if (valid && !whole) {
                float *stats = p.partial + static_cast<int64_t>(p.max_slots) * kRows * HD + static_cast<int64_t>(u.slot) * 2 * kRows + tid;
                stats[0] = m, stats[kRows] = l;
            }
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                __syncwarp();
                if (blocks > 0) {
                    tmem_ld32(o, o_at + c * 32);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
                if (poison && valid) {
                    for (int b = 0; b < kMaskedBlocks * 2; ++b)
                        for (uint32_t bits = sm.poison[b]; bits; bits &= bits - 1) {
                            const int bit = b * 32 + __ffs(bits) - 1, block = first_masked + bit / kKeys, key = block * kKeys + bit % kKeys;
                            if (!(seen_of(p, u, tok, block * kKeys) >> (bit % kKeys) & 1)) continue;
                            const int64_t page = p.tables[u.request * p.table_stride + (key >> p.page_shift)];
                            const T *v = static_cast<const T *>(p.v) + page * p.page_stride + u.kvh * p.head_stride + (key & ((1 << p.page_shift) - 1)) * p.row_stride + c * 32;
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                const float x = static_cast<float>(v[i]);
                                if (!isfinite(x)) o[i] = __float_as_uint(__uint_as_float(o[i]) + x);
                            }
                        }
                }
                if (valid && whole) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = Half<T>::pack(__uint_as_float(o[8 * i + 2 * e]) * r, __uint_as_float(o[8 * i + 2 * e + 1]) * r);
                        reinterpret_cast<uint4 *>(out)[c * 4 + i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else if (valid) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) reinterpret_cast<uint4 *>(part)[c * 8 + i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
            }
        }
    }
    if (!ok) *p.status = 1;
    tc_fence_before();
    __syncthreads();
    if (warp == kRows / 32) {
        tc_fence_after();
        tmem_free<kColumns>(tm);
    }
}

// Parts of a tile joined, a warp per row: weights from the parts' maxima, sums in the order of the parts.
constexpr int kJoinThreads = 256;
template <typename T, int HD>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ PagedAttentionParams p) {
    constexpr int kVec = HD / 32;      // values a lane
    grid_dependency_sync();
    const int lane = threadIdx.x & 31;
    const int64_t rows = static_cast<int64_t>(p.units[0]) * kRows;
    for (int64_t at = blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5); at < rows; at += static_cast<int64_t>(gridDim.x) * (kJoinThreads / 32)) {
        const Unit u = reinterpret_cast<const Unit *>(p.units + 4)[at / kRows];
        const int row = static_cast<int>(at % kRows), tok = u.tile * p.tile_tokens + row / p.group;
        if (row >= p.tile_tokens * p.group || tok >= u.n) continue;
        const float *stats = p.partial + static_cast<int64_t>(p.max_slots) * kRows * HD + static_cast<int64_t>(u.slot) * 2 * kRows + row;
        const float *part = p.partial + (static_cast<int64_t>(u.slot) * kRows + row) * HD + lane * kVec;
        float top = kLowest;
        for (int s = lane; s < u.parts; s += 32) top = fmaxf(top, stats[s * 2 * kRows]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float acc[kVec] = {}, total = 0.f;
#pragma unroll 4
        for (int s = 0; s < u.parts; ++s) {
            const float w = exp2f(stats[s * 2 * kRows] - top);
            total += w * stats[s * 2 * kRows + kRows];
#pragma unroll
            for (int i = 0; i < kVec; ++i) acc[i] += w * part[static_cast<int64_t>(s) * kRows * HD + i];
        }
        const float r = total == 0.f ? (top > kLowest ? __int_as_float(0x7fffffff) : 0.f) : 1.f / total;
        uint32_t *out = reinterpret_cast<uint32_t *>(static_cast<T *>(p.out) + static_cast<int64_t>(u.start + tok) * p.out_token +
                                                     (u.kvh * p.group + row % p.group) * p.out_head + lane * kVec);
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) out[i] = Half<T>::pack(acc[2 * i] * r, acc[2 * i + 1] * r);
    }
}

struct Kernels {
    const void *attend, *join;
    int smem;
};
template <typename T, int HD>
Kernels kernels_of() {
    return {reinterpret_cast<const void *>(&paged_attention_kernel<T, HD>), reinterpret_cast<const void *>(&join_kernel<T, HD>), static_cast<int>(sizeof(Smem<HD>))};
}
Kernels kernels_of(int dtype, int head_dim) {
    if (dtype == GPUK_DTYPE_BF16) return head_dim == 128 ? kernels_of<__nv_bfloat16, 128>() : kernels_of<__nv_bfloat16, 64>();
    return head_dim == 128 ? kernels_of<__half, 128>() : kernels_of<__half, 64>();
}

// What a call is cut into at most.
struct Shape {
    int group, tile_tokens, target, may_split;
    int64_t tiles;      // times kv heads
    int64_t grid, slots, bytes;
};
Shape shape_of(int batch, int tokens, int heads, int kv_heads, int head_dim, int64_t max_len, int sms) {
    Shape s = {};
    s.group = heads / kv_heads;
    s.tile_tokens = kRows / s.group;
    s.target = sms * kCtasPerSm;
    // sum of ceil(n / t) <= floor(sum of n / t) + requests with new tokens
    const int64_t full = tokens / s.tile_tokens, some = batch < tokens ? batch : tokens;
    s.tiles = (full + some < tokens ? full + some : tokens) * kv_heads;
    s.may_split = max_len > kMinPart * kKeys;
    // a part has at least work / target blocks: all parts are at most tiles + target, those of tiles in parts at most 2 * target
    s.grid = s.tiles + (s.may_split ? s.target : 0);
    s.slots = s.may_split ? 2 * s.target : 0;
    s.bytes = s.may_split ? 16 + s.target * static_cast<int64_t>(sizeof(Unit)) + s.slots * kRows * (head_dim + 2) * 4 : 0;
    return s;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_shape(const gpuk_pages *pages, int batch, int tokens, int heads, int64_t max_len) {
    if (!pages) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: no pages");
    if (batch < 0 || tokens < 0 || heads <= 0 || pages->kv_heads <= 0 || pages->num_pages < 0 || max_len < 0)
        return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: bad sizes");
    if (pages->dtype != GPUK_DTYPE_BF16 && pages->dtype != GPUK_DTYPE_F16) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: built for bf16 and fp16");
    if (pages->head_dim != 64 && pages->head_dim != 128) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: built for heads of 64 and 128 (got %d)", pages->head_dim);
    if (heads % pages->kv_heads || heads / pages->kv_heads > kRows)
        return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: a whole number of query heads per kv head, at most %d (got %d / %d)", kRows, heads, pages->kv_heads);
    return GPUK_OK;
}

}  // namespace

cudaError_t paged_attention_setup() {
    cudaError_t e = cudaSuccess;
    for (int dtype : {GPUK_DTYPE_BF16, GPUK_DTYPE_F16})
        for (int hd : {64, 128}) {
            const Kernels k = kernels_of(dtype, hd);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(k.attend, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem);
        }
    return e;
}

}  // namespace gpuk

using namespace gpuk;

extern "C" int gpuk_paged_attention_workspace(const gpuk_pages *pages, int batch, int tokens, int heads, int64_t max_len, int64_t *bytes) {
    if (!bytes) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: null pointer");
    *bytes = 0;
    int rc = check_shape(pages, batch, tokens, heads, max_len);
    if (rc != GPUK_OK) return rc;
    if (batch == 0 || tokens == 0) return GPUK_OK;
    const DecodeDevice *d = nullptr;
    rc = decode_device(&d);
    if (rc != GPUK_OK) return rc;
    *bytes = shape_of(batch, tokens, heads, pages->kv_heads, pages->head_dim, max_len, d->sms).bytes;
    return GPUK_OK;
}

extern "C" int gpuk_paged_attention(const void *q, int64_t q_token_stride, int64_t q_head_stride, const gpuk_pages *pages, const int32_t *tables, int64_t table_stride, int table_width,
                                    const int32_t *lens, const int32_t *starts, const int32_t *masks, int mask_words, void *out, int64_t out_token_stride, int64_t out_head_stride,
                                    int batch, int tokens, int heads, int64_t max_len, float scale, void *workspace, int64_t workspace_bytes, void *stream) {
    int rc = check_shape(pages, batch, tokens, heads, max_len);
    if (rc != GPUK_OK) return rc;
    if (table_width < 0 || mask_words < 0 || (masks && mask_words == 0)) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: bad sizes");
    if (!(scale > 0.f) || std::isinf(scale)) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: the scale must be a positive number");
    const int p2 = pages->page_size;
    if (p2 < 8 || (p2 & (p2 - 1)) || p2 > 65536) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: pages of %d tokens; built for powers of two from 8 to 65536", p2);
    if (masks && mask_words > 8) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: masks of %d words; built for at most 8 (256 new tokens of a request)", mask_words);
    if (static_cast<int64_t>(table_width) * p2 > 0x7fffff00ll) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: a table of %d pages is too wide", table_width);
    if (batch == 0 || tokens == 0) return GPUK_OK;
    if (!q || !lens || !starts || !out || (table_width > 0 && !tables)) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: null pointer");
    if (pages->num_pages == 0 || table_width == 0 || !pages->k || !pages->v) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: no pages");
    if (pages->num_pages > 0x7fffffffll) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: too many pages");
    if (!aligned16(q) || !aligned16(pages->k) || !aligned16(pages->v) || !aligned16(out)) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: pointers must be 16-byte aligned");
    for (int64_t s : {q_token_stride, q_head_stride, pages->page_stride, pages->head_stride, pages->row_stride, out_token_stride, out_head_stride})
        if (s <= 0 || s % 8 || s >= (1ll << 38)) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: strides must be positive multiples of 8 values");
    const DecodeDevice *d = nullptr;
    rc = decode_device(&d);
    if (rc != GPUK_OK) return rc;
    Shape s = shape_of(batch, tokens, heads, pages->kv_heads, pages->head_dim, max_len, d->sms);
    if (s.grid > 0x7fffffffll) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: too many tokens");
    if (s.may_split && (!workspace || workspace_bytes < s.bytes || !aligned16(workspace)))
        return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: needs a workspace of %lld bytes, 16-byte aligned", static_cast<long long>(s.bytes));
    const int hd = pages->head_dim;
    const CUtensorMapDataType type = pages->dtype == GPUK_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap qmap, kmap, vmap;
    const uint64_t q_sizes[3] = {static_cast<uint64_t>(hd), static_cast<uint64_t>(heads), static_cast<uint64_t>(tokens)};
    const uint64_t q_strides[2] = {static_cast<uint64_t>(q_head_stride) * 2, static_cast<uint64_t>(q_token_stride) * 2};
    const uint32_t q_box[3] = {64, static_cast<uint32_t>(s.group), static_cast<uint32_t>(s.tile_tokens)};
    const uint64_t sizes[4] = {static_cast<uint64_t>(hd), static_cast<uint64_t>(p2), static_cast<uint64_t>(pages->kv_heads), static_cast<uint64_t>(pages->num_pages)};
    const uint64_t strides[3] = {static_cast<uint64_t>(pages->row_stride) * 2, static_cast<uint64_t>(pages->head_stride) * 2, static_cast<uint64_t>(pages->page_stride) * 2};
    const uint32_t box[4] = {64, static_cast<uint32_t>(p2 < kKeys ? p2 : kKeys), 1, 1};
    int e = encode_map(&qmap, type, q, 3, q_sizes, q_strides, q_box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!e) e = encode_map(&kmap, type, pages->k, 4, sizes, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!e) e = encode_map(&vmap, type, pages->v, 4, sizes, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (e) return set_last_error(GPUK_ERR_CUDA, "paged_attention: the driver refused a tensor map (%d)", e);
    int shift = 0;
    while ((1 << shift) < p2) ++shift;
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    PagedAttentionParams p = {tables, lens, starts, masks, pages->v, out, table_stride, pages->page_stride, pages->head_stride, pages->row_stride, pages->num_pages,
                              out_token_stride, out_head_stride, batch, tokens, pages->kv_heads, s.group, s.tile_tokens, mask_words, table_width, shift, s.target, s.may_split,
                              scale * 1.4426950408889634f, d->status, reinterpret_cast<int *>(ws), reinterpret_cast<float *>(ws + 16 + s.target * sizeof(Unit)),
                              static_cast<int>(s.slots)};
    const Kernels k = kernels_of(pages->dtype, hd);
    void *args[] = {&qmap, &kmap, &vmap, &p};
    cudaError_t err = launch_kernel(k.attend, static_cast<int>(s.grid), kThreads, 1, false, args, static_cast<cudaStream_t>(stream), k.smem);
    if (err == cudaSuccess && s.may_split) {
        void *join_args[] = {&p};
        err = launch_kernel(k.join, 4 * d->sms, kJoinThreads, 1, false, join_args, static_cast<cudaStream_t>(stream));
    }
    if (err != cudaSuccess) return set_last_error(GPUK_ERR_CUDA, "paged_attention: launch failed: %s", cudaGetErrorString(err));
    return GPUK_OK;
}
