// Attention of a ragged batch of new tokens over pages of a KV cache: trees of drafted tokens, prompts and single tokens, heads of 64 and 128, bf16 and fp16.
//
// A request has `ctx` cached tokens and `n` new ones, whose keys and values are in its pages already.  A new token sees the cached ones and, of the new ones, those up to
// itself or those that its bits in `masks` name (in a tree: its ancestors and itself).  softmax(scale * q k^T) v, with a running maximum and sum over blocks of 64 keys.
//
// The rows of a tile are pairs of a token and a query head of one kv head's group, tokens outermost: 128 rows are 128 / group tokens, so that a page is read once for a tree of
// that many nodes, and up to 128 rows cost the tensor pipe less than the page costs HBM (128 operations a byte; the pipe has 250 for each that HBM delivers).  Calls
// whose requests have a token each, so that tiles would be nearly empty, go to paged_decode.cu: single_tokens below says which.
//
//   * scores go to one of two buffers in tensor memory, so that the next block's are multiplied while a thread per row works on this one's; the probabilities go back into the
//     same columns, from where they are the first operand of O += P V.  256 columns and 113 KiB a CTA: two CTAs an SM hide each other's waits.
//   * O is rescaled only where a row's maximum has grown by more than 2^8 (fp16: 2^7) since it was last: otherwise some row of a warp has a new maximum in nearly every block, and each
//     time 128 columns go through registers (prompts below 240 us in place of 190, trees 58.6 in place of 50.6).  The largest weight is then no longer 1, which the operands' type holds, and is
//     rounded like the others: the error against float64 is 2.12e-3 in place of 1.96e-3 for the prompts, 2.28e-3 in place of 2.03e-3 for the trees (1.65e-3 is the result's rounding alone).
//     The largest weight of each block counts in the sum as it is multiplied, so that a row which it dominates is moved by the result's rounding alone (without that 2.16e-3 and 2.32e-3, 0.3 % less
//     time; with all weights summed so 2.11e-3 and 2.29e-3, 3.7 and 1.2 % more).
//   * pages come by TMA through a ring of 8 or 16 KiB slots; a block of 64 keys is one box of a large page or several small ones.  The copying warp reads the table 32 boxes at a time, the
//     next 32 on their way.  Numbers outside the pool and pages behind the last key read as zeros.
//   * every CTA takes an equal share of all tiles' keys, found from the lengths on the device, so the host need not know them.  A tile that several share leaves sums, maxima and outputs
//     in fp32, and a second kernel joins them in order: the same inputs give the same bits.
//   * only blocks that some row sees in part are masked.  There a value that is no finite number would spoil the rows that do not see it (0 * inf), so it is taken out of shared memory
//     before the product, and the rows that do see it add it at the end.
//
// fp32 scores, maxima, sums and outputs.  Probabilities are rounded to the operands' type for the second product; in fp16 they are held times 2^8, so that small
// ones do not fall under its smallest numbers.
//
// Measured (64 / 8 heads of 128, pages of 16 and 64): 2 prompts of 2048 behind 0 and 1000 cached tokens, with 4 single tokens, 224 us a pass among others, where the power limit
// holds the clock: 800 TFLOP/s of what the masks leave, 0.48 of the measured bf16 rate; 190 in the first milliseconds.  8 trees of 33 to 64 nodes over 2000 keys 58, and 50.5 where three states in turn
// leave their pages in L2; 13 nodes over 31 000 keys of 32 / 8 heads of 64, 29.  What bounds it: for prompts the tensor pipe, which takes as long for a product with 64 columns
// as for one with 128, so that the scores of 64 keys cost as much as their 128 outputs twice over (half the score products left out of a copy: 138 us where it took 186; the exponentials left out: 169).  Blocks of 128 keys
// with two score buffers would need 384 columns a CTA, and so one CTA an SM; with one buffer nothing is multiplied while the rows work on it, and the prompts took 220; one CTA an SM with three
// buffers, whose row threads take the blocks in turn with a second 128, takes 320 (long prompts 1.2 times as long), since nothing hides a tile's start and end.  For trees and one long context some
// 9 us of a call are the start of its CTAs, the parts' outputs and the join.  An exponential by polynomial for a quarter of the scores, and two threads a row, did not help: neither unit is the bound.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/gpuk_b200.h"
#include "launch.cuh"
#include "linear.cuh"
#include "paged_share.cuh"
#include "tensor_core.cuh"

namespace gpuk {
namespace {

constexpr int kThreads = kRows + 64;             // a thread per row, a warp that multiplies, one that copies
constexpr int kSpanBytes = kKeys * 128;          // 64 rows of one swizzle span (64 values)
constexpr int kQSpanBytes = kRows * 128;
constexpr int kColumns = 256;                    // two score buffers of 64, up to 128 of outputs
constexpr int kOut = 2 * kKeys;                  // first column of the outputs
constexpr int kMaskedBlocks = 8;                 // that a tile can have
constexpr int kFewTiles = 4;                     // of a request, whose pages are not kept in L2
constexpr int kQueue = 4;                        // segments that are described at a time


template <int HD>
constexpr int kSlotsOf = HD == 128 ? 5 : 10;

// A wait tells a phase of a barrier from the one before and the one behind it, not from the next but one.  Scores, products and queries have two barriers in turn, since a row's thread
// may come to block j when product j - 2 is the last that is known to be complete, and to its end when the last product is.
template <int HD>
struct Smem {
    alignas(1024) unsigned char q[HD / 64 * kQSpanBytes];
    alignas(1024) unsigned char ring[kSlotsOf<HD>][HD / 64 * kSpanBytes];
    uint64_t q_full[2], q_empty, full[kSlotsOf<HD>], empty[kSlotsOf<HD>], s_full[2], p_full[2], o_done[2], together, drained;
    Segment queue[kQueue];
    Start start;
    uint32_t tmem, gave_up;                      // gave_up: some wait has
    uint32_t poison[3][kMaskedBlocks * 2];       // keys of the masked blocks with a value that is no finite number, of a segment, the next and the one before
};

// Nonzero where one of the two halves is an infinity or NaN: all bits of its exponent are set.
__device__ __forceinline__ uint32_t not_finite(uint32_t w, uint32_t exponent) {
    const uint32_t x = (w & exponent) ^ exponent;      // a zero half
    return (x - 0x00010001u) & ~x & 0x80008000u;
}
// 32 bytes, a whole sector: a warp's rows lie apart, and each store of theirs is a sector a row.
__device__ __forceinline__ void store_sector(void *to, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Barriers by their address in shared memory: the warps that copy and multiply are bound by the instructions between two waits.
// A wait gives up after some two seconds, each lane by its own clock, or soon where another has: `gave_up` is in shared memory.  What follows a wait (shuffles, loads of tensor memory) is for
// whole warps, and a lane that left its warp's way would leave the others in it for good.  So a row's lane goes on as if its wait were over, and so do all others behind it, to the end of
// the segment; the copying lanes go on without copying; and from one segment to the next warps go by a vote.  What comes out then means nothing, which the status says.
// (A vote behind each wait, in the multiplying warp's way, takes 1 us of 50 for trees of drafts, 2 of 190 for prompts.)
__device__ __forceinline__ bool wait_at(uint32_t bar, uint32_t parity, uint32_t gave_up) {
    uint64_t began = 0;
    for (uint32_t spin = 1;; ++spin) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if (spin % 128 == 0) {
            uint64_t now;
            asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(ok) : "r"(gave_up) : "memory");
            if (ok) return false;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (began == 0) began = now;
            else if (now - began > 2000000000ull) break;
        }
    }
    asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(gave_up), "r"(1) : "memory");
    return false;
}
__device__ __forceinline__ bool vote(bool ok) { return __all_sync(0xffffffffu, ok) != 0; }
__device__ __forceinline__ void arrive_at(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void expect_at(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ void commit_at(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// One lane of a warp that is together.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// Bits [at, at + 64) of a row of mask words, zeros outside.
__device__ __forceinline__ uint64_t mask_bits(const int32_t *row, int words, int at) {
    const int w = at >> 5, s = at & 31;
    const uint32_t a = w < words ? row[w] : 0, b = w + 1 < words ? row[w + 1] : 0, c = w + 2 < words ? row[w + 2] : 0;
    return static_cast<uint64_t>(__funnelshift_r(a, b, s)) | static_cast<uint64_t>(__funnelshift_r(b, c, s)) << 32;
}
// Which keys of block `base` a row sees: cached ones, and of the new ones those up to token `tok` or those in its mask.
__device__ __forceinline__ uint64_t seen_of(const PagedAttentionParams &p, const Segment &u, int tok, int base) {
    const int old = min(max(u.ctx - base, 0), kKeys);      // keys of the block in front of the new ones
    const uint64_t cached = old == kKeys ? ~0ull : (1ull << old) - 1;
    if (old == kKeys) return cached;
    const int rel = base + old - u.ctx;
    const int room = static_cast<int>(min(room_of(p) - base - old, static_cast<int64_t>(kKeys - old)));      // tokens behind the table's row have no keys
    const int most = min(p.masks ? u.n - rel : tok + 1 - rel, room);
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
    if (tid == kRows + 32) prefetch_map(&qmap), prefetch_map(&kmap), prefetch_map(&vmap);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp < 2) find_border(p, &sm.start, warp);
    if (warp == kRows / 32) tmem_alloc<kColumns>(&sm.tmem);
    if (tid == kRows) {
        for (int b = 0; b < 2; ++b) mbar_init(&sm.q_full[b], 1), mbar_init(&sm.s_full[b], 1), mbar_init(&sm.p_full[b], kRows / 32), mbar_init(&sm.o_done[b], 1);
        for (int s = 0; s < kSlots; ++s) mbar_init(&sm.full[s], 1), mbar_init(&sm.empty[s], 1);
        mbar_init(&sm.q_empty, 1), mbar_init(&sm.together, kRows / 32), mbar_init(&sm.drained, 1);
        sm.gave_up = 0;
        mbar_init_fence();
    }
    if (tid >= kRows + 32)
        for (int i = tid - kRows - 32; i < 3 * kMaskedBlocks * 2; i += 32) sm.poison[0][i] = 0;
    tc_fence_before();
    __syncthreads();
    if (sm.start.x[1] <= sm.start.x[0]) {      // a border that went to an end of its tile, or fewer CTAs than there are
        if (tid == 0 && p.may_split) p.joints[blockIdx.x].open.slot = -1, p.joints[blockIdx.x].head = 0, p.joints[blockIdx.x].ctas = sm.start.ctas;
        if (warp == kRows / 32) tmem_free<kColumns>(sm.tmem);
        return;
    }
    tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // behind the allocation: no CTA that follows takes columns one of this grid waits for
    const uint32_t tm = sm.tmem;
    const bool aligned = (smem_addr(dyn) & 1023u) == 0;
    bool ok = aligned;

    const uint32_t full = smem_addr(sm.full), empty = smem_addr(sm.empty), q_full = smem_addr(sm.q_full), s_full = smem_addr(sm.s_full), p_full = smem_addr(sm.p_full),
                   o_done = smem_addr(sm.o_done), q_empty = smem_addr(&sm.q_empty), gave_up = smem_addr(&sm.gave_up);
    auto wait = [&](uint32_t bar, uint32_t parity) { return wait_at(bar, parity, gave_up); };
    auto all_well = [&]() { return *static_cast<volatile uint32_t *>(&sm.gave_up) == 0; };

    if (warp == kRows / 32 + 1) {      // copies: of a segment K of the first block, Q, and K of the next block before V of each
        const int lane = tid & 31;
        const int rows = min(1 << p.page_shift, kKeys), box_shift = min(p.page_shift, 6), boxes = kKeys >> box_shift, batch_blocks = 32 >> (6 - box_shift);
        Walk walk(sm.start);
        const uint64_t once = policy_evict_first(), again = policy_evict_normal();
        Joint joint;
        joint.open.slot = -1, joint.head = 3, joint.ctas = sm.start.ctas;
        int segments = 0, slot = 0, filled = 0;
        uint32_t phase = 1;      // a fresh slot counts as released
        Segment u;
        bool begins, ends;
        while (ok && walk.next(p, &u, &begins, &ends)) {
            if (!begins) joint.head = ends ? 2 : 1;
            if (begins && !ends) joint.open = u;
            // What few tiles read leaves L2 first, which is 10 % of a batch of single tokens (32 x 30 to 4000 keys: 42.7 / 47.3 us); a prompt's tiles read the same pages again and
            // again (2 x 2048 tokens: 186 / 211 us the other way).
            const uint64_t policy = walk.r.tiles <= kFewTiles ? once : again;
            const int32_t *table = p.tables + u.request * p.table_stride;
            // Pages by 32 boxes, a lane for each, and the next 32 on their way; one outside the pool, which reads as zeros, where there is none.
            const int end = static_cast<int>(min(min(static_cast<int64_t>(u.ctx) + u.n, room_of(p)), (static_cast<int64_t>(u.first) + u.blocks) * kKeys));
            auto pages_from = [&](int j) {
                const int64_t key = (static_cast<int64_t>(u.first) + j) * kKeys + (lane << box_shift);
                return key < end ? table[key >> p.page_shift] : -1;
            };
            int pages = pages_from(0), pages_next = batch_blocks < u.blocks ? pages_from(batch_blocks) : -1, left = batch_blocks, from = 0;
            const int inside_mask = rows == kKeys ? (1 << p.page_shift) - 1 : 0;
            auto load = [&](const CUtensorMap *map, int j, int page) {
                const uint32_t bar = full + 8 * slot;
                ok &= wait(empty + 8 * slot, phase);
                if (lane == 0 && ok) expect_at(bar, kBlockBytes);
                __syncwarp();
                if (lane < boxes && ok) {
                    const int inside = (u.first + j) * kKeys & inside_mask;
                    const uint32_t to = smem_addr(sm.ring) + slot * kBlockBytes + (lane << box_shift) * 128;
#pragma unroll
                    for (int h = 0; h < kSpans; ++h) tma_load_4d(to + h * kSpanBytes, map, h * 64, inside, u.kvh, page, &sm.full[slot], policy);
                }
                filled += ok;
                if (++slot == kSlots) slot = 0, phase ^= 1u;
            };
            // the pages of the next block
            auto next_page = [&](int j) {
                if (left == 0) {
                    pages = pages_next, left = batch_blocks, from = 0;
                    pages_next = j + batch_blocks < u.blocks ? pages_from(j + batch_blocks) : -1;
                }
                const int page = __shfl_sync(0xffffffffu, pages, (from + lane) & 31);
                from += boxes, --left;
                return page;
            };
            auto load_q = [&]() {
                if (lane == 0) {
                    sm.queue[segments % kQueue] = u;
                    expect_at(q_full + 8 * (segments & 1), kSpans * p.tile_tokens * p.group * 128);
#pragma unroll
                    for (int h = 0; h < kSpans; ++h) tma_load_3d(smem_addr(sm.q) + h * kQSpanBytes, &qmap, h * 64, u.kvh * p.group, u.start + u.tok0, &sm.q_full[segments & 1]);
                }
            };
            if (segments == 0) load_q();      // the first keys wait for the table, those of later segments for nothing
            int page_k = next_page(0);
            load(&kmap, 0, page_k);
            if (segments > 0) {
                ok &= wait(q_empty, (segments - 1) & 1);
                ok = vote(ok && all_well());
                if (!ok) break;
                load_q();
            }
            ++segments;
            for (int j = 0; j < u.blocks; ++j) {
                const int page_v = page_k;
                if (j + 1 < u.blocks) {
                    page_k = next_page(j + 1);
                    load(&kmap, j + 1, page_k);
                }
                load(&vmap, j, page_v);
            }
            ok = vote(ok);
        }
        if (lane == 0 && p.may_split) p.joints[blockIdx.x] = joint;
        // the end, behind the last segment's scores; and nobody leaves with copies in flight or releases to come
        if (ok && segments > 0) ok = wait(q_empty, (segments - 1) & 1);
        if (ok && lane == 0) {
            sm.queue[segments % kQueue].blocks = 0;
            arrive_at(q_full + 8 * (segments & 1));
        }
        if (!ok && segments > 0) mbar_wait(&sm.q_full[(segments - 1) & 1], ((segments - 1) >> 1) & 1);
        for (int i = max(0, filled - kSlots); i < filled; ++i) {
            if (ok) ok = wait(empty + 8 * (i % kSlots), (i / kSlots) & 1);
            if (!ok && !mbar_wait(&sm.full[i % kSlots], (i / kSlots) & 1)) break;      // not released: landed at least, however long others have waited
        }
    } else if (warp == kRows / 32) {   // multiplications: K and V of the ring are used in the order in which they were copied
        // The whole warp goes through the loop and one lane issues, so that descriptors stay in uniform registers: a lane on its own took 80 cycles an instruction.
        constexpr uint32_t s_desc = mma_desc(Half<T>::kFormat, Half<T>::kFormat, kRows, kKeys), o_desc = mma_desc(Half<T>::kFormat, Half<T>::kFormat, kRows, HD, true);
        const uint64_t q_at = kmajor_desc<128>(smem_addr(sm.q)), k_at = kmajor_desc<128>(smem_addr(sm.ring)), v_at = mnmajor_desc(smem_addr(sm.ring), kSpanBytes);
        const uint32_t out_at = __shfl_sync(0xffffffffu, tm, 0) + kOut, scores_at = out_at - kOut;
        int slot = 0;
        uint32_t phase = 0, t = 0;      // of the ring; blocks so far
        auto wait_all = [&](uint32_t bar, uint32_t parity) { return vote(wait(bar, parity)); };
        auto taken = [&]() {
            if (++slot == kSlots) slot = 0, phase ^= 1u;
        };
        auto scores = [&](uint32_t t, bool last) {
            const uint64_t k = k_at + slot * (kBlockBytes / 16);
            const uint32_t to = scores_at + (t & 1) * kKeys;
            if (elect_one()) {
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) tc_mma_f16(to, q_at + ((d / 4) * kQSpanBytes + (d % 4) * 32) / 16, k + ((d / 4) * kSpanBytes + (d % 4) * 32) / 16, s_desc, d > 0);
                commit_at(s_full + 8 * (t & 1));
                commit_at(empty + 8 * slot);
                if (last) commit_at(q_empty);
            }
            taken();
        };
        for (uint32_t segment = 0; ok; ++segment) {
            ok = wait_all(q_full + 8 * (segment & 1), (segment >> 1) & 1);
            if (!ok) break;
            const int blocks = __shfl_sync(0xffffffffu, sm.queue[segment % kQueue].blocks, 0);
            if (blocks == 0) break;
            ok = wait_all(full + 8 * slot, phase);
            tc_fence_after();
            if (ok) scores(t, blocks == 1);
            for (int j = 0; ok && j < blocks; ++j, ++t) {
                if (j + 1 < blocks) {
                    ok = wait_all(full + 8 * slot, phase);
                    tc_fence_after();
                    if (!ok) break;
                    scores(t + 1, j + 2 == blocks);      // into the buffer of P(t - 1), whose product is in front of it
                }
                ok = wait_all(full + 8 * slot, phase) && wait_all(p_full + 8 * (t & 1), (t >> 1) & 1);
                tc_fence_after();
                if (!ok) break;
                const uint64_t v = v_at + slot * (kBlockBytes / 16);
                const uint32_t probabilities = scores_at + (t & 1) * kKeys;
                if (elect_one()) {
                    tc_mma_f16_ts(out_at, probabilities, v, o_desc, j > 0);
#pragma unroll
                    for (int k = 1; k < kKeys / 16; ++k) tc_mma_f16_ts(out_at, probabilities + k * 8, v + k * 16 * 128 / 16, o_desc, true);
                    commit_at(o_done + 8 * (t & 1));
                    commit_at(empty + 8 * slot);
                }
                taken();
            }
        }
        // where a wait gave up, here or in a row's warp, nobody has waited for what was issued last, and the tensor memory is about to be freed
        if (elect_one()) tc_commit(&sm.drained);
        mbar_wait(&sm.drained, 0);
    } else {                           // a row's thread
        const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16, o_at = tm + lanes + kOut;
        const f32x2 scale2 = f2_splat(p.scale_log2);
        const int row_tok = tid / p.group, row_head = tid - row_tok * p.group;
        int t = 0, fill = 0;
        for (int segment = 0; aligned; ++segment) {
            if (!vote(wait(q_full + 8 * (segment & 1), (segment >> 1) & 1) && all_well())) break;
            const Segment u = sm.queue[segment % kQueue];
            if (u.blocks == 0) break;
            const int tok = u.tok0 + row_tok;
            const bool valid = tid < p.tile_tokens * p.group && tok < u.n;
            const bool busy = __any_sync(0xffffffffu, valid);
            // blocks from here on hold keys that some row does not see, or none: a tile may begin behind the end of the table's row, inside whose last block the keys end
            const int64_t limit = p.masks ? u.ctx : min(static_cast<int64_t>(u.ctx) + u.tok0 + 1, room_of(p));
            const int first_masked = max(u.first, static_cast<int>(limit / kKeys));
            uint32_t *poison = sm.poison[segment % 3];
            if (tid < kMaskedBlocks * 2) sm.poison[(segment + 1) % 3][tid] = 0;      // read last before the barrier of the segment in front
            float m = kLowest, l = 0.f;
            for (int j = 0; j < u.blocks; ++j, ++t) {
                const int block = u.first + j;
                wait(s_full + 8 * (t & 1), (t >> 1) & 1);      // idle warps too: nobody arrives twice in a phase
                __syncwarp();
                if (busy) {
                    tc_fence_after();
                    const uint32_t s_at = tm + lanes + (t & 1) * kKeys;
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
                    auto score = [&](int i) { return __uint_as_float(s[i / 32][i % 32]); };
                    float mx[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        mx[c] = fmaxf(score(16 * c), score(16 * c + 1));
#pragma unroll
                        for (int i = 2; i < 16; i += 2) mx[c] = max3(mx[c], score(16 * c + i), score(16 * c + i + 1));
                    }
                    const float largest = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
                    float top = largest * p.scale_log2;
                    if (some) top = fmaxf(top, kSeen);
                    const bool grown = top > m + Half<T>::kLag;
                    if (j == 0) {
                        m = fmaxf(top, kLowest);
                    } else if (__any_sync(0xffffffffu, grown)) {
                        wait(o_done + 8 * ((t - 1) & 1), ((t - 1) >> 1) & 1);
                        __syncwarp();
                        tc_fence_after();
                        const float f = grown ? exp2_fast(m - top) : 1.f;
                        if (grown) m = top, l *= f;
#pragma unroll 1
                        for (int c = 0; c < HD; c += 16) {
                            float o[16];
                            tmem_ld16(o, o_at + c);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] *= f;
                            tmem_st16(o_at + c, o);
                        }
                    }
                    const f32x2 shift2 = f2_splat(Half<T>::kBias - m);
                    // the block's largest weight counts as it is multiplied, so that its rounding moves no row that it dominates
                    const float heaviest = exp2_fast(fmaf(largest, p.scale_log2, Half<T>::kBias - m));
                    l += Half<T>::round(heaviest) - heaviest;
                    f32x2 sum[2] = {0, 0};
                    uint32_t pk[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float a, c;
                        f2_split(f2_fma(f2_make_bits(s[i / 16][2 * (i % 16)], s[i / 16][2 * (i % 16) + 1]), scale2, shift2), a, c);
                        a = exp2_fast(a), c = exp2_fast(c);
                        sum[i & 1] = f2_add(sum[i & 1], f2_make(a, c));
                        pk[i] = Half<T>::pack(a, c);
                    }
                    tmem_st32(s_at, pk);
                    l += f2_sum(f2_add(sum[0], sum[1]));
                    tmem_wait_st();
                    tc_fence_before();
                }
                if (block >= first_masked) {
                    // values that are none, or that a row may not see and that are no finite numbers, become zeros
                    const int i = fill + (j + 1 < u.blocks ? 2 * j + 2 : 2 * j + 1);
                    wait(full + 8 * (i % kSlots), (i / kSlots) & 1);
                    uint4 *v = reinterpret_cast<uint4 *>(sm.ring[i % kSlots]);
                    const int keys = static_cast<int>(min(min(static_cast<int64_t>(u.ctx) + u.n, room_of(p)) - static_cast<int64_t>(block) * kKeys, static_cast<int64_t>(kKeys)));
                    constexpr uint32_t e = Half<T>::kExponent;
                    constexpr int kMine = kBlockBytes / 16 / kRows;
                    uint4 x[kMine];
#pragma unroll
                    for (int c = 0; c < kMine; ++c) x[c] = v[c * kRows + tid];
                    uint32_t odd = keys < kKeys;
#pragma unroll
                    for (int c = 0; c < kMine; ++c) odd |= not_finite(x[c].x, e) | not_finite(x[c].y, e) | not_finite(x[c].z, e) | not_finite(x[c].w, e);
                    const bool changed = odd != 0;
                    if (changed) {
#pragma unroll
                        for (int c = 0; c < kMine; ++c) {
                            const int at = c * kRows + tid, key = (at & (kSpanBytes / 16 - 1)) / 8;
                            uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
                            if (key >= keys) {
                                v[at] = make_uint4(0, 0, 0, 0);
                            } else if (not_finite(w[0], e) | not_finite(w[1], e) | not_finite(w[2], e) | not_finite(w[3], e)) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    if ((w[k] & e & 0xffffu) == (e & 0xffffu)) w[k] &= 0xffff0000u;
                                    if ((w[k] & e & 0xffff0000u) == (e & 0xffff0000u)) w[k] &= 0xffffu;
                                }
                                v[at] = make_uint4(w[0], w[1], w[2], w[3]);
                                const int bit = (block - first_masked) * kKeys + key;
                                if (bit < kMaskedBlocks * 64) atomicOr(&poison[bit >> 5], 1u << (bit & 31));
                            }
                        }
                    }
                    if (changed) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                __syncwarp();
                if ((tid & 31) == 0) arrive_at(p_full + 8 * (t & 1));
            }
            fill += 2 * u.blocks;
            wait(o_done + 8 * ((t - 1) & 1), ((t - 1) >> 1) & 1);
            tc_fence_after();
            // all rows' warps have come here, or one of them has given up: a named barrier would wait for it without end
            __syncwarp();
            if ((tid & 31) == 0) arrive_at(smem_addr(&sm.together));
            wait(smem_addr(&sm.together), segment & 1);
            if (busy) {
                uint32_t any = 0;
#pragma unroll
                for (int i = 0; i < kMaskedBlocks * 2; ++i) any |= poison[i];
                const bool whole = u.slot < 0;
                // a row that saw no key is zeros; one whose scores are all -infinity is NaN, as a softmax has it
                const float r = l == 0.f ? (m > kLowest ? __int_as_float(0x7fffffff) : 0.f) : 1.f / l;
                const int head = u.kvh * p.group + row_head;
                T *out = static_cast<T *>(p.out) + static_cast<int64_t>(u.start + tok) * p.out_token + head * p.out_head;
                uint4 *part = reinterpret_cast<uint4 *>(p.partial) + static_cast<int64_t>(u.slot) * (HD / 4) * kRows + tid;
                if (valid && !whole) {
                    float *stats = p.stats + static_cast<int64_t>(u.slot) * 2 * kRows + tid;
                    stats[0] = m, stats[kRows] = l;
                }
#pragma unroll 1
                for (int c = 0; c < HD / 32; ++c) {
                    uint32_t o[32];
                    __syncwarp();
                    tmem_ld32(o, o_at + c * 32);
                    tmem_wait_ld();
                    if (any && valid) {
                        for (int b = 0; b < kMaskedBlocks * 2; ++b)
                            for (uint32_t bits = poison[b]; bits; bits &= bits - 1) {
                                const int bit = b * 32 + __ffs(bits) - 1, block = first_masked + bit / kKeys, key = block * kKeys + bit % kKeys;
                                if (!(seen_of(p, u, tok, block * kKeys) >> (bit % kKeys) & 1)) continue;
                                const int64_t page = p.tables[u.request * p.table_stride + (key >> p.page_shift)];
                                if (page < 0 || page >= p.num_pages) continue;      // read as zeros: only behind a wait that gave up can there have been anything else
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
                        for (int i = 0; i < 2; ++i) {
                            uint32_t w[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) w[e] = Half<T>::pack(__uint_as_float(o[16 * i + 2 * e]) * r, __uint_as_float(o[16 * i + 2 * e + 1]) * r);
                            if (p.out_sectors) {
                                store_sector(out + c * 32 + i * 16, w);
                            } else {
                                reinterpret_cast<uint4 *>(out)[c * 4 + 2 * i] = make_uint4(w[0], w[1], w[2], w[3]);
                                reinterpret_cast<uint4 *>(out)[c * 4 + 2 * i + 1] = make_uint4(w[4], w[5], w[6], w[7]);
                            }
                        }
                    } else if (valid) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) part[(c * 8 + i) * kRows] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
            }
        }
        // the product before the last has been counted too before the CTA ends
        if (t > 1) wait(o_done + 8 * (t & 1), ((t - 2) >> 1) & 1);
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && !(aligned && all_well())) *p.status = 1;
    if (warp == kRows / 32) {
        tc_fence_after();
        tmem_free<kColumns>(tm);
    }
}

// Parts of a tile joined: the one that the CTA where the tile begins left, and those of the CTAs behind it up to the tile's last, in that order.  A CTA takes 32 rows of a tile, a lane
// for each; its warps read the statistics of as many parts at a time, and then each its share of the values of all parts.
constexpr int kJoinWarps = 8, kJoinParts = 32;
template <typename T, int HD>
__global__ void __launch_bounds__(kJoinWarps * 32, 3) join_kernel(const __grid_constant__ PagedAttentionParams p) {
    constexpr int kVecs = HD / 4 / kJoinWarps, kAhead = 8 / kVecs;      // vectors of four that a lane sums up, and parts of them that it reads at a time
    __shared__ float maxima[kJoinParts][32], sums[kJoinParts][32];
    __shared__ int slots[kJoinParts];
    grid_dependency_sync();
    const int cta = blockIdx.x / p.row_groups, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ctas = p.joints[0].ctas;
    if (cta >= ctas) return;
    const Segment u = p.joints[cta].open;
    const int row = blockIdx.x % p.row_groups * 32 + lane, tok = u.tok0 + row / p.group;
    const bool valid = u.slot >= 0 && row < p.tile_tokens * p.group && tok < u.n;
    if (!__any_sync(0xffffffffu, valid)) return;      // the same in all warps
    const float4 *partial = reinterpret_cast<const float4 *>(p.partial) + warp * kVecs * kRows + row;
    float top = kLowest, total = 0.f;
    float4 acc[kVecs] = {};
    for (int next = cta; next < ctas; next += 32) {      // 32 CTAs at a time, a lane for each
        const int c = next + lane;
        const int head = c >= ctas ? 0 : c == cta ? 1 : p.joints[c].head;
        const uint32_t over = __ballot_sync(0xffffffffu, c >= ctas || head >= 2);
        const int reach = over ? __ffs(over) : 32;
        const bool mine = lane < reach && (head == 1 || head == 2);
        const uint32_t parts = __ballot_sync(0xffffffffu, mine);
        const int count = __popc(parts);
        __syncthreads();      // the last 32 have been read
        if (warp == 0 && mine) slots[__popc(parts & ((1u << lane) - 1))] = c == cta ? u.slot : 2 * c;
        __syncthreads();
#pragma unroll 2
        for (int i = warp; i < count; i += kJoinWarps) {
            const float *stats = p.stats + static_cast<int64_t>(slots[i]) * 2 * kRows + row;
            maxima[i][lane] = stats[0], sums[i][lane] = stats[kRows];
        }
        __syncthreads();
        float high = top;
        for (int i = 0; i < count; ++i) high = fmaxf(high, maxima[i][lane]);
        const float fade = exp2f(top - high);
        top = high, total *= fade;
#pragma unroll
        for (int k = 0; k < kVecs; ++k) acc[k].x *= fade, acc[k].y *= fade, acc[k].z *= fade, acc[k].w *= fade;
        for (int i = 0; i < count; i += kAhead) {
            float4 v[kAhead][kVecs];
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
#pragma unroll
                for (int k = 0; k < kVecs; ++k) v[a][k] = partial[(static_cast<int64_t>(slots[min(i + a, count - 1)]) * (HD / 4) + k) * kRows];
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
                if (i + a < count) {
                    const float w = exp2f(maxima[i + a][lane] - top);
                    total += w * sums[i + a][lane];
#pragma unroll
                    for (int k = 0; k < kVecs; ++k) acc[k].x += w * v[a][k].x, acc[k].y += w * v[a][k].y, acc[k].z += w * v[a][k].z, acc[k].w += w * v[a][k].w;
                }
        }
        if (over) break;
    }
    if (!valid) return;
    const float r = total == 0.f ? (top > kLowest ? __int_as_float(0x7fffffff) : 0.f) : 1.f / total;
    uint2 *out = reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + static_cast<int64_t>(u.start + tok) * p.out_token + (u.kvh * p.group + row % p.group) * p.out_head) + warp * kVecs;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) out[k] = make_uint2(Half<T>::pack(acc[k].x * r, acc[k].y * r), Half<T>::pack(acc[k].z * r, acc[k].w * r));
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
    int group, tile_tokens, may_split;
    int64_t grid, bytes;
};
// `single`: single tokens, or without a bound on a request's new ones no more of them than requests, and so in all likelihood one for each.  Both kernels give the formula's result whatever the
// requests have; for single tokens the one that is built for them takes 4 x 100 to 300 keys of 16 / 4 heads in 6.6 us instead of 9.7, 32 x 30 to 4000 of 64 / 8 in 39.4 instead of 42.7.  For many tokens of a few of the
// requests it is the other way round: 64 of one behind 2000 keys 64 us, 23 by the tensor-core kernel; 8 behind nothing 4.8 and 6.9.
Shape shape_of(int batch, int tokens, int heads, int kv_heads, int head_dim, int64_t max_len, int sms, bool single) {
    Shape s = {};
    s.group = heads / kv_heads;
    s.tile_tokens = single ? 1 : kRows / s.group;
    // sum of ceil(n / t) <= floor(sum of n / t) + requests with new tokens
    const int64_t full = tokens / s.tile_tokens, some = batch < tokens ? batch : tokens;
    const int64_t tiles = (full + some < tokens ? full + some : tokens) * kv_heads;
    s.may_split = max_len >= kFront + kGrain;      // shorter tiles are never cut
    const int64_t most = static_cast<int64_t>(sms) * kCtasPerSm, want = 2 * tiles + tiles * (max_len + kTileCost) / kPerCta;
    s.grid = single && !s.may_split ? tiles : tiles >= most || want >= most ? most : want;
    s.bytes = s.may_split ? s.grid * (static_cast<int64_t>(sizeof(Joint)) + 2ll * kRows * (head_dim + 2) * 4) : 0;
    return s;
}

int row_groups_of(const Shape &s) { return (s.tile_tokens * s.group + 31) / 32; }
bool single_tokens(int batch, int tokens, int max_new, int heads, int kv_heads, bool masks) {
    return !masks && (max_new ? max_new == 1 : tokens <= batch) && heads / kv_heads <= kDecodeGroup;
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
            int smem = 0;
            const void *decode = paged_decode_of(dtype, hd, &smem);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(decode, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
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
    // of the kernel that needs more: which one a call takes depends on its masks and on max_new too
    for (bool single : {false, true}) {
        if (single && !single_tokens(batch, tokens, 1, heads, pages->kv_heads, false)) continue;
        const int64_t need = shape_of(batch, tokens, heads, pages->kv_heads, pages->head_dim, max_len, d->sms, single).bytes;
        if (need > *bytes) *bytes = need;
    }
    return GPUK_OK;
}

extern "C" int gpuk_paged_attention(const void *q, int64_t q_token_stride, int64_t q_head_stride, const gpuk_pages *pages, const int32_t *tables, int64_t table_stride, int table_width,
                                    const int32_t *lens, const int32_t *starts, const int32_t *masks, int mask_words, void *out, int64_t out_token_stride, int64_t out_head_stride,
                                    int batch, int tokens, int heads, int64_t max_len, int max_new, float scale, void *workspace, int64_t workspace_bytes, void *stream) {
    int rc = check_shape(pages, batch, tokens, heads, max_len);
    if (rc != GPUK_OK) return rc;
    if (table_width < 0 || mask_words < 0 || max_new < 0 || (masks && mask_words == 0)) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: bad sizes");
    if (!(scale > 0.f) || std::isinf(scale)) return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: the scale must be a positive number");
    const int p2 = pages->page_size;
    if (p2 < 8 || (p2 & (p2 - 1)) || p2 > 65536) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: pages of %d tokens; built for powers of two from 8 to 65536", p2);
    if (masks && mask_words > 8) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: masks of %d words; built for at most 8 (256 new tokens of a request)", mask_words);
    if (static_cast<int64_t>(table_width) * p2 > 0x7fffff00ll) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: a table of %d pages is too wide", table_width);
    if (tokens > 1 << 24) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: %d new tokens; built for at most 2^24", tokens);
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
    const bool single = single_tokens(batch, tokens, max_new, heads, pages->kv_heads, masks != nullptr);
    const Shape s = shape_of(batch, tokens, heads, pages->kv_heads, pages->head_dim, max_len, d->sms, single);
    if (s.grid * row_groups_of(s) > 0x7fffffffll) return set_last_error(GPUK_ERR_UNSUPPORTED, "paged_attention: too many tokens");
    if (s.may_split && (!workspace || workspace_bytes < s.bytes || !aligned16(workspace)))
        return set_last_error(GPUK_ERR_INVALID_ARGUMENT, "paged_attention: needs a workspace of %lld bytes, 16-byte aligned", static_cast<long long>(s.bytes));
    const int hd = pages->head_dim;
    int shift = 0;
    while ((1 << shift) < p2) ++shift;
    Joint *joints = static_cast<Joint *>(workspace);
    float *partial = reinterpret_cast<float *>(joints + s.grid);
    PagedAttentionParams p = {tables, lens, starts, masks, q, pages->k, pages->v, out, q_token_stride, q_head_stride, table_stride, pages->page_stride, pages->head_stride, pages->row_stride, pages->num_pages,
                              out_token_stride, out_head_stride, batch, tokens, pages->kv_heads, s.group, s.tile_tokens, mask_words, static_cast<uint32_t>(((1ull << 32) + s.tile_tokens - 1) / s.tile_tokens), table_width, shift, row_groups_of(s), s.may_split,
                              (reinterpret_cast<uintptr_t>(out) | out_token_stride * 2 | out_head_stride * 2) % 32 == 0,
                              scale * 1.4426950408889634f, d->status, joints, partial, partial + s.grid * 2 * kRows * hd};
    const Kernels k = kernels_of(pages->dtype, hd);
    cudaError_t err;
    if (single) {
        int smem = 0;
        const void *decode = paged_decode_of(pages->dtype, hd, &smem);
        void *args[] = {&p};
        err = launch_kernel(decode, static_cast<int>(s.grid), kDecodeThreads, 1, false, args, static_cast<cudaStream_t>(stream), smem);
    } else {
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
        void *args[] = {&qmap, &kmap, &vmap, &p};
        err = launch_kernel(k.attend, static_cast<int>(s.grid), kThreads, 1, false, args, static_cast<cudaStream_t>(stream), k.smem);
    }
    if (err == cudaSuccess && s.may_split) {
        void *join_args[] = {&p};
        err = launch_kernel(k.join, static_cast<int>(s.grid) * p.row_groups, kJoinWarps * 32, 1, false, join_args, static_cast<cudaStream_t>(stream));
    }
    if (err != cudaSuccess) return set_last_error(GPUK_ERR_CUDA, "paged_attention: launch failed: %s", cudaGetErrorString(err));
    return GPUK_OK;
}
